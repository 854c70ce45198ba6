"""GPU: products with weights of 4 bits, against their definition in 64 bits.

Tolerances.  The codes less eight are exact operands and so are the rows (fp32 rows in three parts), so a group's sum of products is off by its fp32
additions alone: at most 2^-23 of the sum of the products' sizes for each of the k (128 products are added in sixteens, with some bits less than
fp32's kept of the smaller ones: 2^-22), then the zero points' part, (8 - z) times the sum of x, by as much of its own, and
the groups' sums another in + 16 roundings.  For 16-bit rows a code enters as 16 + code and 16 + z times the sum of x is taken off, sums that are at most six times
larger.  The result is rounded once: eps / 2.  Products with many rows have each weight rounded as well, once, or twice with zero points: eps / 2
or eps of the products' sizes, and add all in fp32, with in roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}


def _weight(out, inner, group, dtype, zeros, gen):
    groups = (inner + group - 1) // group
    codes = torch.randint(0, 16, (out, inner), device="cuda", generator=gen, dtype=torch.uint8)
    scales = torch.empty(out, groups, device="cuda").uniform_(-0.2, 0.3, generator=gen).to(dtype)
    zero = torch.empty(out, groups, device="cuda").uniform_(-1, 16, generator=gen).to(dtype) if zeros else None
    at = torch.arange(inner, device="cuda") // group
    w = (codes.double() - (zero.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    parts = codes.double() - 8, scales.double()[:, at], (8 - zero.double()[:, at]) if zeros else torch.zeros(1, 1, dtype=torch.float64, device="cuda")
    return codes, scales, zero, w, parts


def _check(y, x, w, parts, eps, rounded_weights):
    exact = torch.einsum("rk,nk->rn", x.double(), w)
    xa = x.double().abs()
    code, scale, zero = parts
    large = 16 + 16 if eps > 2.0 ** -23 else 0
    sizes = torch.einsum("rk,nk->rn", xa, ((code.abs() + zero.abs() + large) * scale.abs()).expand_as(w))
    tol = eps / 2 * exact.abs() + (2.0 ** -22 + (x.shape[-1] / 32 + 16) * 2.0 ** -24) * sizes + 1e-30
    if rounded_weights:
        tol = tol + eps * torch.einsum("rk,nk->rn", xa, w.abs()) + x.shape[-1] * 2.0 ** -24 * sizes
    off = (y.double() - exact).abs() - tol
    assert off.max().item() <= 0, f"{off.max().item():.3e} above the tolerance, largest {exact.abs().max().item():.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128, 512])
def test_against_the_definition(dtype, zeros, group):
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(group)
    for inner, out in ((512, 96), (64, 17), (1000, 333), (129, 2048), (4096, 40), (2176, 5000), (1, 1), (31, 16), (9000, 130)):
        codes, scales, zero, w, parts = _weight(out, inner, group, dtype, zeros, gen)
        packed = castle_pack_4bit(codes)
        for rows in (1, 2, 3, 8, 9, 17, 32, 33, 50):
            x = torch.randn(rows, inner, device="cuda", generator=gen).to(dtype)
            x[:, ::7] *= 20
            y = castle_linear_4bit(x, packed, scales, zero, group_size=group)
            assert y.shape == (rows, out) and y.dtype == dtype
            _check(y, x, w, parts, EPS[dtype], True)
            if rows <= (2 if dtype == torch.float32 else 8) and inner <= 4096:
                _check(y, x, w, parts, EPS[dtype], False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_and_tiles(dtype):
    """More row tiles than a CTA leaves at a time, wide rows shared out among the CTAs of a cluster."""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(1)
    for inner, out, rows in ((512, 50021, 3), (1000, 333, 65), (300, 130, 257), (4096, 1000, 777), (1100, 4096, 777), (2048, 9472, 500), (640, 4700, 1024), (129, 17, 1000), (256, 300, 5000), (7, 9, 100), (128, 70000, 20), (16384, 512, 8), (16384, 2500, 17), (12000, 48, 1), (1024, 4096, 300), (40000, 100, 5), (40000, 64, 32)):
        codes, scales, zero, w, parts = _weight(out, inner, 64, dtype, True, gen)
        x = torch.randn(rows, inner, device="cuda", generator=gen).to(dtype)
        y = castle_linear_4bit(x, castle_pack_4bit(codes), scales, zero)
        _check(y, x, w, parts, EPS[dtype], True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
def test_the_width_shared_out(dtype, zeros):
    """Weights of few tiles, whose width the CTAs of clusters share out: of two, four and eight, in even and odd shares, groups that end inside one."""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(8)
    for inner, out, rows, group in ((4096, 4096, 40, 64), (8000, 200, 500, 32), (7997, 1000, 500, 256), (16384, 512, 48, 64), (16384, 17, 33, 4096), (8192, 1024, 100, 128),
                                    (1153, 130, 70, 32), (1100, 100, 1000, 64), (4096, 4096, 200, 64), (5000, 2100, 300, 64), (6000, 8192, 60, 128)):
        codes, scales, zero, w, parts = _weight(out, inner, group, dtype, zeros, gen)
        packed, x = castle_pack_4bit(codes), torch.randn(rows, inner, device="cuda", generator=gen).to(dtype)
        y = castle_linear_4bit(x, packed, scales, zero, group)
        _check(y, x, w, parts, EPS[dtype], True)
        assert all(torch.equal(castle_linear_4bit(x, packed, scales, zero, group), y) for _ in range(3))


def test_fp32_rows_in_turns():
    """Five or ten at a time, the last turn with fewer, and from how many on at full width."""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(9)
    for inner, out, group in ((4097, 3000, 64), (4096, 2000, 32), (9000, 1100, 128), (1000, 9000, 64)):
        codes, scales, zero, w, parts = _weight(out, inner, group, torch.float32, True, gen)
        packed = castle_pack_4bit(codes)
        for rows in (5, 6, 10, 11, 21, 33, 47, 90):
            x = torch.randn(rows, inner, device="cuda", generator=gen)
            _check(castle_linear_4bit(x, packed, scales, zero, group), x, w, parts, EPS[torch.float32], True)


def test_more_rows_than_a_launch_has_and_the_widest():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(7)
    codes, scales, zero, w, parts = _weight(40, 16, 64, torch.bfloat16, True, gen)
    x = torch.randn(65535 * 32 * 2 + 77, 16, device="cuda", generator=gen).bfloat16()
    y = castle_linear_4bit(x, castle_pack_4bit(codes), scales, zero)
    for part in (slice(0, 1000), slice(65535 * 32 - 500, 65535 * 32 + 500), slice(65535 * 64 - 500, None)):
        _check(y[part], x[part], w, parts, EPS[torch.bfloat16], True)
    codes, scales, zero, w, parts = _weight(20, 600_001, 64, torch.bfloat16, False, gen)
    for rows in (1, 3, 40):
        x = torch.randn(rows, 600_001, device="cuda", generator=gen).bfloat16()
        _check(castle_linear_4bit(x, castle_pack_4bit(codes), scales), x, w, parts, EPS[torch.bfloat16], True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_strides_and_shapes(dtype):
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(2)
    codes, scales, zero, w, parts = _weight(70, 300, 64, dtype, True, gen)
    packed = castle_pack_4bit(codes)
    base = torch.randn(4, 3, 700, device="cuda", generator=gen).to(dtype)
    many = torch.randn(30, 5, 700, device="cuda", generator=gen).to(dtype)
    for x in (many[..., :300], many[..., 3:303], many[..., ::2][..., :300], many.transpose(0, 1)[..., 1:301], many[:, 2:3, 8:308].expand(30, 4, 300)):
        _check(castle_linear_4bit(x, packed, scales, zero).reshape(-1, 70), x.reshape(-1, 300), w, parts, EPS[dtype], True)
    for x in (base[0, 0, :300], base[:, 1, 5:305], base[..., ::2][..., :300], base[:, :, 399:699], base[:0, :, :300], base.transpose(0, 1)[:, :, 1:301]):
        y = castle_linear_4bit(x, packed, scales, zero)
        assert y.shape == (*x.shape[:-1], 70) and y.is_contiguous()
        if x.numel():
            _check(y.reshape(-1, 70), x.reshape(-1, 300), w, parts, EPS[dtype], False)
    spread = torch.zeros(70, 2 * scales.shape[1], device="cuda", dtype=dtype)
    spread[:, ::2] = scales
    assert torch.equal(castle_linear_4bit(base[0, :, :300], packed, spread[:, ::2], zero), castle_linear_4bit(base[0, :, :300], packed, scales, zero))


def test_fp32_rows_of_all_sizes():
    """The three parts of a row hold all its bits, down to where the last part's leave the type's range, and infinities and NaN stay what they are."""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(3)
    codes, scales, _, w, parts = _weight(64, 256, 64, torch.float32, False, gen)
    packed = castle_pack_4bit(codes)
    for size in (1e-20, 1.0, 1e30):
        x = torch.randn(2, 256, device="cuda", generator=gen) * size
        _check(castle_linear_4bit(x, packed, scales), x, w, parts, EPS[torch.float32], False)
    x = torch.zeros(3, 256, device="cuda")
    x[0, 7], x[1, 9] = float("inf"), float("nan")
    x[2, 5] = torch.finfo(torch.float32).max / 4096
    y = castle_linear_4bit(x, packed, scales)
    sign = (codes[:, 7].double() - 8) * scales[:, 0].double()
    assert bool((y[0][sign != 0] == torch.where(sign > 0, torch.inf, -torch.inf)[sign != 0].float()).all()) and bool(y[0][sign == 0].isnan().all())
    assert bool(y[1].isnan().all()) and bool(y[2].isfinite().all())
    _check(y[2:], x[2:], w, parts, EPS[torch.float32], False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_near_the_types_ends(dtype, zeros):
    """Finite results of rows whose groups' sums, before their scales, are beyond fp32's range; and rows far below one.  (Small ones: what products with codes
    lose below fp32's smallest normal number, 2^-149 each of 2^-16 of them, is 2^-133 of a scale a product.)"""
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(6)
    codes, scales, zero, w, parts = _weight(100, 640, 64, dtype, zeros, gen)
    for top, factor in ((torch.finfo(dtype).max, 2.0 ** -16), (1e-32, 1.0)):
        small, part = (scales.float() * factor).to(dtype), (parts[0], parts[1] * factor, parts[2])   # (exact: a power of two)
        for rows in (1, 3, 8):
            x = ((torch.rand(rows, 640, device="cuda", generator=gen) * 0.5 + 0.5) * top).to(dtype)
            y = castle_linear_4bit(x, castle_pack_4bit(codes), small, zero)
            assert bool(y.isfinite().all())
            lift = 1.0 / (x.double().abs().max() * factor)                                           # (the tolerance's constant is for results near one)
            _check(y.double() * lift, x.double() * lift, w * factor, part, EPS[dtype], rows > 2)


def test_a_row_does_not_change_another():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(4)
    codes, scales, zero, _, _ = _weight(500, 1024, 32, torch.bfloat16, True, gen)
    packed = castle_pack_4bit(codes)
    x = torch.randn(8, 1024, device="cuda", generator=gen).bfloat16()
    y = castle_linear_4bit(x, packed, scales, zero, 32)
    assert all(torch.equal(castle_linear_4bit(x, packed, scales, zero, 32), y) for _ in range(5))
    z = x.clone()
    z[3] = float("nan")
    other = castle_linear_4bit(z, packed, scales, zero, 32)
    keep = [i for i in range(8) if i != 3]
    assert torch.equal(other[keep], y[keep]) and bool(other[3].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,inner,out,zeros", [(1, 128, 64, False), (5, 300, 130, True), (100, 1000, 513, True)])
def test_gradient_of_the_rows(dtype, rows, inner, out, zeros):
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit
    gen = torch.Generator("cuda").manual_seed(5)
    codes, scales, zero, w, _ = _weight(out, inner, 64, dtype, zeros, gen)
    packed = castle_pack_4bit(codes)
    x = torch.randn(rows, inner, device="cuda", generator=gen).to(dtype).requires_grad_()
    g = torch.randn(rows, out, device="cuda", generator=gen).to(dtype)
    y = castle_linear_4bit(x, packed, scales, zero)
    (dx,) = torch.autograd.grad(y, [x], g, retain_graph=True)
    exact = g.double() @ w
    tol = EPS[dtype] / 2 * exact.abs() + (EPS[dtype] / 2 + (out + 8) * 2.0 ** -24) * (g.double().abs() @ w.abs()) + 1e-30
    assert bool(((dx.double() - exact).abs() <= tol).all()) and dx.dtype == dtype
    (again,) = torch.autograd.grad(y, [x], g.t().contiguous().t())
    assert torch.equal(again, dx)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, [x], g)      # (released)
    if dtype == torch.float32:              # differences: the product is linear, so they are the gradient
        d = torch.randn_like(x)
        with torch.no_grad():
            change = (castle_linear_4bit(x + d, packed, scales, zero) - castle_linear_4bit(x - d, packed, scales, zero)).double()
        assert torch.allclose((change / 2 * g.double()).sum(), (dx.double() * d.double()).sum(), rtol=1e-4, atol=1e-3)


def test_second_derivatives_are_refused():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_quantize_4bit
    codes, scales, _ = castle_quantize_4bit(torch.randn(64, 64, device="cuda"))
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(castle_linear_4bit(x, codes, scales).square().sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        dx.sum().backward()


def test_under_autocast():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_quantize_4bit
    w = torch.randn(200, 256, device="cuda")
    codes, scales, zeros = castle_quantize_4bit(w, zeros=True)
    for rows in (4, 200):
        x = torch.randn(rows, 256, device="cuda").bfloat16().requires_grad_()
        with torch.autocast("cuda", dtype=torch.float16):
            y = castle_linear_4bit(x, codes, scales, zeros)
            (dx,) = torch.autograd.grad(y.float().sum(), [x])
        want = castle_linear_4bit(x.detach(), codes, scales.bfloat16(), zeros.bfloat16())
        assert y.dtype == dx.dtype == torch.bfloat16 and torch.equal(y, want)


def test_quantized_weights_are_the_nearest():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_quantize_4bit
    for zeros in (False, True):
        for k, group in ((256, 64), (200, 64), (100, 128)):
            w = torch.randn(40, k, device="cuda") * torch.rand(40, 1, device="cuda")
            w[3, :64] = 0
            w[4, :64] = 0.25
            codes, scales, zp = castle_quantize_4bit(w, group, zeros)
            back = castle_linear_4bit(torch.eye(k, device="cuda"), codes, scales, zp, group).t()
            at = torch.arange(k, device="cuda") // group
            step = scales[:, at]
            # half a step inside the range, plus what the zero point's or the extremes' rounding takes (fp32: 16 units of 2^-23 of 15 steps)
            assert bool(((back - w).abs() <= step * (0.5 + 1e-4)).all())


def test_refusals():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit, castle_quantize_4bit
    codes, scales, zeros = castle_quantize_4bit(torch.randn(32, 128, device="cuda").bfloat16(), zeros=True)
    x = torch.randn(2, 128, device="cuda").bfloat16()
    for call in (lambda: castle_linear_4bit(x[:, :60], codes, scales), lambda: castle_linear_4bit(x.float(), codes, scales), lambda: castle_linear_4bit(x, codes, scales, zeros[:, :1]),
                 lambda: castle_linear_4bit(x, codes.long(), scales), lambda: castle_linear_4bit(x, codes, scales, group_size=48), lambda: castle_linear_4bit(x, codes, scales, group_size=128),
                 lambda: castle_linear_4bit(x.cpu(), codes, scales), lambda: castle_linear_4bit(x, codes.cpu(), scales), lambda: castle_linear_4bit(x.double(), codes, scales),
                 lambda: castle_linear_4bit(x, codes, scales.requires_grad_())):
        with pytest.raises(RuntimeError, match="castle_linear_4bit"):
            call()
    for call in (lambda: castle_pack_4bit(x), lambda: castle_pack_4bit(codes[0]), lambda: castle_quantize_4bit(x, 48), lambda: castle_quantize_4bit(codes)):
        with pytest.raises(ValueError):
            call()


def test_captured_and_on_streams():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_quantize_4bit
    w = torch.randn(3000, 2048, device="cuda").bfloat16()
    codes, scales, _ = castle_quantize_4bit(w)
    xs = [torch.randn(r, 2048, device="cuda").bfloat16() for r in (1, 8, 20, 60, 500)]
    want = [castle_linear_4bit(x, codes, scales) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = []
    for x, s in zip(xs, streams):
        with torch.cuda.stream(s):
            outs.append(castle_linear_4bit(x, codes, scales))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    for x, y in zip(xs[:4], want):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = castle_linear_4bit(x, codes, scales)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)
