"""GPU: products with weights of 4 bits whose every step is exact, so that the result is the exact one rounded once and nothing that is left out or counted twice hides
below a tolerance.

Rows are whole numbers, zero points too, scales are 1/2, 1, 2 or -1.  Then codes less their zero points, weights in any of the types and all products are exact, and so is each sum of
them as long as the sum of their sizes, counted in halves, is below 2^24 (asserted): whatever the order, no partial sum has more than fp32's 24 bits.  In the kernel for
few rows a group's sum has 16 + code in place of code - zero, at most 31 of a row's value each: 4096 k of them are below 2^24 as well.  fp32 rows have a value with 18 bits, all
three parts of which count."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(inner, out, group, dtype, zeros, gen):
    groups = (inner + group - 1) // group
    codes = torch.randint(0, 16, (out, inner), device="cuda", generator=gen, dtype=torch.uint8)
    scales = torch.tensor([0.5, 1.0, 2.0, -1.0], device="cuda")[torch.randint(0, 4, (out, groups), device="cuda", generator=gen)].to(dtype)
    zero = torch.randint(0, 16, (out, groups), device="cuda", generator=gen).to(dtype) if zeros else None
    at = torch.arange(inner, device="cuda") // group
    w = (codes.double() - (zero.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    return codes, scales, zero, w


def _rows(rows, inner, dtype, gen):
    top = 3 if inner <= 100_000 else 1
    x = torch.randint(-top, top + 1, (rows, inner), device="cuda", generator=gen).float()
    if dtype == torch.float32:
        at = torch.randint(0, inner, (rows, 1), device="cuda", generator=gen)
        x.scatter_(1, at, torch.where(x.gather(1, at) < 0, -1.0, 1.0) * (2 ** 17 + 1))
    return x.to(dtype)


SIZES = [(16384, 512, 64), (16385, 200, 32), (16384, 130, 4096), (40000, 64, 128), (4096, 1000, 64), (7997, 300, 256), (1000, 2000, 32), (129, 70, 64), (512, 9000, 64), (31, 17, 32)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("inner,out,group", SIZES)
def test_whole_numbers(inner, out, group, dtype, zeros):
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit, check_status
    gen = torch.Generator("cuda").manual_seed(inner + out)
    codes, scales, zero, w = _case(inner, out, group, dtype, zeros, gen)
    packed = castle_pack_4bit(codes)
    for rows in (1, 2, 5, 8, 9, 11, 16, 17, 25, 32, 33, 48, 100, 300):
        x = _rows(rows, inner, dtype, gen)
        assert 2 * (x.double().abs() @ w.abs().t()).max().item() < 2 ** 24
        y, exact = castle_linear_4bit(x, packed, scales, zero, group), torch.einsum("rk,nk->rn", x.double(), w)
        assert torch.equal(y, exact.to(dtype)), (rows, (y.double() - exact).abs().max().item())
    check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_widest_rows(dtype):
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit, check_status
    gen = torch.Generator("cuda").manual_seed(1)
    codes, scales, zero, w = _case(600_001, 20, 64, dtype, True, gen)
    packed = castle_pack_4bit(codes)
    for rows in (1, 3, 9, 17, 32, 40):
        x = _rows(rows, 600_001, dtype, gen)
        assert 2 * (x.double().abs() @ w.abs().t()).max().item() < 2 ** 24
        assert torch.equal(castle_linear_4bit(x, packed, scales, zero), torch.einsum("rk,nk->rn", x.double(), w).to(dtype))
    check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
def test_the_gradient_of_one_output_is_its_weights(dtype, zeros):
    """Rows of a unit matrix as the gradient: the weights at full width, each the exact one (sums of it and zeros)."""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(2)
    for inner, out, group in ((700, 90, 32), (4096, 64, 128), (1001, 300, 64), (5, 3, 32)):
        codes, scales, zero, w = _case(inner, out, group, dtype, zeros, gen)
        x = torch.zeros(out, inner, device="cuda", dtype=dtype, requires_grad=True)
        y = castle_linear_4bit(x, castle_pack_4bit(codes), scales, zero, group)
        (dx,) = torch.autograd.grad(y, [x], torch.eye(out, device="cuda", dtype=dtype))
        assert torch.equal(dx, w.to(dtype))
