"""GPU: token lookup and its table's gradient against the definition in 64 bits.

Tolerances, with u = 2^-24 (fp32) and h = half a step of the type: y = scale w is off by the rounding of scale and of the
product (u each) and the result's (h).  A gradient is a sum of k values in fp32, off by at most k u times the sum of their sizes,
then scaled (2 u) and rounded (h).  fp16 results below its normal numbers are off by half of its smallest step instead."""
import pytest
import torch

from lookahead_keys_attention_b200 import castle_embedding, check_status, release_workspaces

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def check(tokens, weight, grad, scale, padding=None):
    """One call and its gradient; returns the gradient."""
    dtype = weight.dtype
    w = weight.detach().requires_grad_()
    y = castle_embedding(tokens, w, scale, padding)
    (dw,) = torch.autograd.grad(y, [w], grad)
    check_status()
    assert y.dtype == dtype and y.shape == (*tokens.shape, weight.shape[1]) and dw.shape == weight.shape and dw.dtype == dtype
    t = tokens.reshape(-1).long()
    want = weight.double()[t].reshape(y.shape) * scale
    assert bool(((y.double() - want).abs() <= (half_step(dtype) + 2 * U) * want.abs() + least(dtype)).all())
    g = grad.double().reshape(-1, weight.shape[1])
    keep = torch.ones_like(t, dtype=torch.bool) if padding is None else t != padding % weight.shape[0]
    ref = torch.zeros_like(weight, dtype=torch.float64).index_add_(0, t[keep], g[keep]) * scale
    size = torch.zeros_like(ref).index_add_(0, t[keep], g[keep].abs()) * abs(scale)
    k = torch.bincount(t[keep], minlength=weight.shape[0])[:, None] + 3
    tol = half_step(dtype) * ref.abs() + k * U * size * (1 + half_step(dtype)) + least(dtype)
    bad = (dw.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} gradients off, worst {((dw.double() - ref).abs() - tol).max().item():.3e}"
    return dw


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,dim,vocab", [(1, 64, 100), (8, 512, 256), (1, 1, 1), (33, 7, 5), (1000, 129, 131), (1025, 1032, 3001), (4099, 1000, 50021),
                                         (257, 2056, 1537), (65, 8192, 149)])
def test_sizes(dtype, n, dim, vocab):
    gen = torch.Generator("cuda").manual_seed(n)
    t = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    w = torch.randn(vocab, dim, device="cuda", generator=gen).to(dtype)
    g = torch.randn(n, dim, device="cuda", generator=gen).to(dtype)
    check(t, w, g, dim ** 0.5)


@pytest.mark.parametrize("n,runs", [(5000, [5000]), (5000, [1, 2500, 1, 2498]), (4096, [16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 3391]), (300000, [299999, 1])])
def test_rows_with_many_tokens(n, runs):
    """Runs whose pieces begin and end at, before and behind the places where long rows are cut."""
    assert sum(runs) == n
    gen = torch.Generator("cuda").manual_seed(3)
    t = torch.cat([torch.full((r,), 3 * i + 1, dtype=torch.int64) for i, r in enumerate(runs)])
    t = t[torch.randperm(n, generator=torch.Generator().manual_seed(1))].cuda()
    w = torch.randn(3 * len(runs) + 5, 40, device="cuda", generator=gen)
    g = torch.randn(n, 40, device="cuda", generator=gen)
    a = check(t, w, g, 1.0)
    release_workspaces()
    assert torch.equal(a, check(t, w, g, 1.0))   # the same order of additions in every call
    check(t.int(), w.bfloat16(), g.bfloat16(), 0.5)


@pytest.mark.parametrize("padding", [None, 0, 4, -1])
def test_padding_has_no_gradient(padding):
    gen = torch.Generator("cuda").manual_seed(5)
    t = torch.randint(0, 6, (7, 50), device="cuda", generator=gen)
    w = torch.randn(6, 24, device="cuda", generator=gen).bfloat16()
    dw = check(t, w, torch.randn(7, 50, 24, device="cuda", generator=gen).bfloat16(), 2.0, padding)
    if padding is not None:
        assert not bool(dw[padding].any())
    all_padding = torch.full((9,), 4, device="cuda")
    assert not bool(check(all_padding, w, torch.ones(9, 24, device="cuda").bfloat16(), 1.0, 4).any())


def test_strides():
    gen = torch.Generator("cuda").manual_seed(6)
    w = torch.randn(90, 3, 64, device="cuda", generator=gen).half()
    t = torch.randint(0, 90, (12, 20), device="cuda", generator=gen)
    g = torch.randn(10, 12, 64, device="cuda", generator=gen).half()
    check(t[:, ::2].t(), w[:, 1], g, 1.5)                                     # rows of a table inside another one, tokens across
    check(t.t()[::2], w[:, 2, :63], g[..., :63], 1.5)                          # not at 16-byte boundaries
    check(t[:, ::2].t(), w[:, 0].t().contiguous().t(), g, 1.0)                 # down the columns
    check(t[:, ::2].t(), w[:, 1], g[:1, :1, :1].expand(10, 12, 64), 1.0)       # a gradient that repeats one value (of a sum)
    check(t[:, ::2].t(), w[:, 1], g.transpose(0, 1).contiguous().transpose(0, 1), 1.0)


def test_no_tokens():
    w = torch.randn(5, 8, device="cuda", requires_grad=True)
    y = castle_embedding(torch.empty(2, 0, dtype=torch.int64, device="cuda"), w)
    assert y.shape == (2, 0, 8)
    y.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.parametrize("bad", [-1, 100, 2 ** 40])
def test_a_token_outside_the_vocabulary_is_reported(bad):
    w = torch.randn(100, 72, device="cuda", requires_grad=True)
    t = torch.arange(50, device="cuda")
    t[7] = bad
    y = castle_embedding(t, w)
    assert bool(y[7].isnan().all()) and torch.equal(y[:7], w[:7]) and torch.equal(y[8:], w[8:50])
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        check_status()
    y.backward(torch.ones_like(y))
    want = torch.zeros_like(w)
    want[:50] = 1
    want[7] = 0
    assert torch.equal(w.grad, want)
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        check_status()
    check_status()


def test_values_that_are_not_numbers_stay_in_their_rows():
    w = torch.randn(10, 40, device="cuda", requires_grad=True)
    t = torch.tensor([1, 2, 3, 2, 9], device="cuda")
    g = torch.ones(5, 40, device="cuda")
    g[0, 3], g[4] = float("nan"), float("inf")
    (dw,) = torch.autograd.grad(castle_embedding(t, w, 2.0, padding_idx=9), [w], g)
    assert bool(dw[1, 3].isnan()) and int((~dw.isfinite()).sum()) == 1
    assert bool((dw[2] == 4).all()) and bool((dw[3] == 2).all()) and not bool(dw[9].any())


def test_refusals():
    w = torch.randn(10, 8, device="cuda")
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    for args in [(t.float(), w), (t.short(), w), (t, w.double()), (t, w[0]), (t, w[:0]), (t.cpu(), w), (t, w.cpu())]:
        with pytest.raises(RuntimeError, match="castle_embedding"):
            castle_embedding(*args)
    for padding in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            castle_embedding(t, w, padding_idx=padding)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        castle_embedding(t, torch.autograd.forward_ad.make_dual(w, w))


def test_gradient_against_differences():
    """The result is linear in the table, so a difference of two results is the gradient's product with the step."""
    gen = torch.Generator("cuda").manual_seed(9)
    w = torch.randn(20, 16, device="cuda", generator=gen, requires_grad=True)
    t = torch.randint(0, 20, (64,), device="cuda", generator=gen)
    g, step = (torch.randn(s, 16, device="cuda", generator=gen) for s in (64, 20))
    (dw,) = torch.autograd.grad(castle_embedding(t, w, 3.0), [w], g)
    moved = (castle_embedding(t, w + step, 3.0).double() - castle_embedding(t, w, 3.0).double()) * g.double()
    size = (g.abs().double() * 3 * (w[t].abs() + step[t].abs()).double()).sum()
    assert abs(moved.sum() - (dw.double() * step.double()).sum()) <= 16 * U * size
