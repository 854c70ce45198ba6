"""GPU: layer norm and its gradients against the definition in 64 bits, and the layer that has it in front.

Tolerances, with u = 2^-24 and h = half a step of the type.  A sum over a row is a chain of at most c = 24 + dim / 256 additions
in fp32 (16 or dim / 256 of a thread, then trees and the warps), so it is off by c u times the sum of the sizes.  So the mean is
off by d = c u mean|x|, the normalised value n by e = 2 r d + (c + 8) u |n| (the difference, the variance's sum, the root, two
products); y by |w| e + 2 u |n w| + u |y| and its rounding h |y|.  The gradients follow from their formulas in the same way."""
import pytest
import torch

from lookahead_keys_attention_b200 import Castle, castle_layer_norm, check_status

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def least(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


def within(got, want, tol, dtype, what):
    tol = tol * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * want.abs() + least(dtype)
    excess = ((got.double() - want).abs() - tol).max().item()
    assert got.dtype == dtype and got.shape == want.shape and excess <= 0, f"{what}: {excess:.3e} beyond the tolerance"


def check(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = castle_layer_norm(*leaves, eps)
    grads = list(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    check_status()
    dim, dtype = x.shape[-1], x.dtype
    c, cr = 24 + dim / 256, x.numel() // dim + 8
    X, DY = x.double().reshape(-1, dim), dy.double().reshape(-1, dim)
    W = torch.ones_like(X[0]) if w is None else w.double()
    B = torch.zeros_like(X[0]) if b is None else b.double()
    def mean(t):
        return t.mean(1, keepdim=True)
    m = mean(X)
    r = 1 / torch.sqrt(mean((X - m) ** 2) + eps)
    n = (X - m) * r
    e = 2 * r * c * U * mean(X.abs()) + (c + 8) * U * n.abs()
    Y = n * W + B
    within(y.reshape(-1, dim), Y, W.abs() * e + 2 * U * (n * W).abs() + U * Y.abs(), dtype, "y")
    g = DY * W
    mg, mgn = mean(g), mean(g * n)
    dx = r * (g - mg - n * mgn)
    off = (4 * U * (g.abs() + mg.abs() + (n * mgn).abs()) + (c + 2) * U * (mean(g.abs()) + n.abs() * mean((g * n).abs()))
           + e * mgn.abs() + n.abs() * mean(g.abs() * e))
    within(grads.pop(0).reshape(-1, dim), dx, r * off + (c + 8) * U * dx.abs(), dtype, "dx")
    if w is not None:
        within(grads.pop(0), (DY * n).sum(0), (cr * U * (DY * n).abs() + DY.abs() * e).sum(0), dtype, "dweight")
    if b is not None:
        within(grads.pop(0), DY.sum(0), cr * U * DY.abs().sum(0), dtype, "dbias")


def case(rows, dim, dtype, seed=0, offset=0.5, affine="both"):
    gen = torch.Generator("cuda").manual_seed(seed)
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    x = (rand(rows, dim) * 2 + offset * rand(rows, 1)).to(dtype)
    w = (1 + 0.3 * rand(dim)).to(dtype) if affine != "none" else None
    b = rand(dim).to(dtype) if affine == "both" else None
    return x, w, b, rand(rows, dim).to(dtype)


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("rows,dim", [(1, 8), (2, 512), (1, 1), (3, 7), (37, 256), (100, 257), (301, 504), (64, 512), (65, 1000), (33, 1024), (17, 1333), (40, 2048),
                                      (19, 3001), (700, 4096), (9, 4104), (5, 8192), (301, 8191), (6, 8200), (4, 16384), (3, 20001)])
def test_sizes(dtype, rows, dim):
    check(*case(rows, dim, dtype, rows + dim))


@pytest.mark.parametrize("affine", ["none", "weight"])
@pytest.mark.parametrize("rows,dim", [(50, 512), (50, 1333), (20, 9000)])
def test_without_weight_or_bias(rows, dim, affine):
    check(*case(rows, dim, torch.bfloat16, 1, affine=affine))


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (0, 1), (1, 2), (0, 2)])
@pytest.mark.parametrize("rows,dim", [(70, 512), (40, 5000)])
def test_some_of_the_gradients(rows, dim, wanted):
    x, w, b, dy = case(rows, dim, torch.float32, 2)
    leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
    some = torch.autograd.grad(castle_layer_norm(*leaves), [leaves[i] for i in wanted], dy)
    all_leaves = [t.clone().double().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(all_leaves[0], (dim,), all_leaves[1], all_leaves[2], 1e-5)
    ref = torch.autograd.grad(y, all_leaves, dy.double())
    for i, g in zip(wanted, some):
        # sizes are of the order of one (dx) or of the root of the rows' number: chains of 24 + dim / 256 and `rows` additions
        assert (g.double() - ref[i]).abs().max() <= 64 * (24 + dim / 256 + rows) * U * ref[i].abs().max()


def test_rows_with_an_offset_keep_their_spread():
    x, w, b, dy = case(40, 1000, torch.float32, 3, offset=0.0)
    check(x + 4096, w, b, dy)


def test_constant_rows_and_zero_rows():
    x, w, b, dy = case(20, 512, torch.float32, 4)
    x[3], x[5] = 0.0, 2.0
    check(x, w, b, dy, eps=1e-3)
    assert torch.equal(castle_layer_norm(x, w, b, 1e-3)[3], b) and torch.equal(castle_layer_norm(x, w, b, 1e-3)[5], b)


def test_rows_that_are_not_numbers_stay_alone():
    for dim in (512, 1333, 9000):
        x, w, b, dy = case(30, dim, torch.bfloat16, 5)
        y = castle_layer_norm(x, w, b)
        x[4, 1], x[9, 0] = float("nan"), float("inf")
        leaf = x.requires_grad_()
        z = castle_layer_norm(leaf, w, b)
        (dx,) = torch.autograd.grad(z, [leaf], dy)
        others = [i for i in range(30) if i not in (4, 9)]
        assert torch.equal(z[others], y[others]) and bool(z[4].isnan().all()) and bool(z[9].isnan().all())
        assert bool(dx[others].isfinite().all()) and bool(dx[4].isnan().all())


def test_strides():
    x, w, b, dy = case(24 * 5, 512, torch.float16, 6)
    big = torch.randn(24, 9, 520, device="cuda").half()
    check(big[:, 3, :512], w, b, dy[:24])                                     # rows of a larger tensor, at 16-byte boundaries
    check(big[:, 3, 1:513], w, b, dy[:24])                                    # and not
    check(big[:, 2:7, :512], w, b, dy.view(24, 5, 512))                       # no single stride: copied
    check(x.view(24, 5, 512).transpose(0, 1), w, b, dy.view(5, 24, 512))
    check(x.t().contiguous().t(), w, b, dy)
    check(x, w, b, dy[:1].expand(120, 512))                                   # a repeated gradient row
    check(x, w, b, dy[:1, :1].expand(120, 512))                               # the gradient of a sum
    check(big[0, 0, :512], w, b, dy[0])                                       # one row as a vector
    check(big[:, 0, ::2][:, :256], w[::2].contiguous(), b[::2], dy[:24, ::2])


def test_no_rows():
    w, b = (torch.randn(16, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.empty(0, 3, 16, device="cuda", requires_grad=True)
    y = castle_layer_norm(x, w, b)
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and not bool(w.grad.any()) and not bool(b.grad.any())


def test_the_weights_gradients_are_the_same_from_call_to_call():
    x, w, b, dy = case(5000, 512, torch.bfloat16, 7)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(castle_layer_norm(*leaves), leaves, dy)
    for _ in range(3):
        again = torch.autograd.grad(castle_layer_norm(*leaves), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_refusals():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(16, device="cuda")
    for args in [(x.double(),), (x, w.half()), (x, w[:8]), (x, w, w[None]), (x.cpu(),), (x, w.cpu()), (x[:, :0],), (x[0, 0],)]:
        with pytest.raises(RuntimeError, match="castle_layer_norm"):
            castle_layer_norm(*args)
    leaf = x.requires_grad_()
    (g,) = torch.autograd.grad(castle_layer_norm(leaf).sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                    # no second derivative


def test_gradient_against_differences():
    """Along a random direction, by central differences of the 64-bit sum of the fp32 results."""
    x, w, b, dy = case(8, 96, torch.float32, 8)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(castle_layer_norm(*leaves), leaves, dy)
    gen = torch.Generator("cuda").manual_seed(1)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        step = torch.randn(leaf.shape, device="cuda", generator=gen)
        h = 2.0 ** -7
        def at(s):
            moved = [t.detach() + s * h * step if j == i else t.detach() for j, t in enumerate(leaves)]
            return (castle_layer_norm(*moved).double() * dy.double()).sum()
        slope, want = (at(1) - at(-1)) / (2 * h), (grad.double() * step.double()).sum()
        # third derivatives of a normalised row are of the order of one per value: h^2; roundings: (c + 16) u per value / h
        bound = (h * h + 50 * U / h) * (dy.abs().double() * (1 + step.abs().double().amax()) ** 3 * 2).sum()
        assert abs(slope - want) <= bound


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("bias", [True, False])
def test_a_layer_with_a_layer_norm(dtype, bias):
    """`Castle(prenorm="layer")`: the native layer against the same layer with its submodules called as modules.  Both round the norm
    and the projections to the type at the same places and add in different orders, so each of them is as far from the exact result
    as the types' steps say: the difference of their norms' ratios is bounded by eight steps (outputs) and sixteen (gradients)."""
    torch.manual_seed(0)
    m = Castle(256, heads=4, prenorm="layer").cuda()
    torch.nn.init.normal_(m.norm.weight, 1.0, 0.2)
    if bias:
        torch.nn.init.normal_(m.norm.bias)
    else:
        m.norm.bias = None
    m = m.to(dtype)
    assert m._plain_layer() is not None
    x = torch.randn(2, 300, 256, device="cuda").to(dtype).requires_grad_()
    g = torch.randn(2, 300, 256, device="cuda").to(dtype)
    out = m(x)
    grads = torch.autograd.grad(out, [x, *m.parameters()], g)
    handle = m.norm.register_forward_hook(lambda *a: None)
    assert m._plain_layer() is None
    out_m = m(x)
    grads_m = torch.autograd.grad(out_m, [x, *m.parameters()], g)
    handle.remove()
    check_status()
    step = max(torch.finfo(dtype).eps, torch.finfo(torch.float16).eps)   # the core's operands have 16 bits
    def far(a, b):
        return ((a.double() - b.double()).norm() / b.double().norm()).item()
    assert far(out, out_m) <= 8 * step
    assert len(grads) == (5 if bias else 4)
    for (name, _), a, b in zip([("x", None), *m.named_parameters()], grads, grads_m):
        assert a.dtype == dtype and a.shape == b.shape and far(a, b) <= 16 * step, name
    # a prompt and single tokens behind it
    with torch.no_grad():
        whole = m(x)
        first, cache = m(x[:, :290], return_next_cache=True)
        tokens = []
        for t in range(290, 300):
            o, cache = m(x[:, t:t + 1], cache=cache)
            tokens.append(o)
    check_status()
    assert far(torch.cat([first, *tokens], 1), whole) <= 8 * step


def test_a_layer_norm_put_in_another_norms_place_is_called():
    m = Castle(64, heads=2, dim_head=32, prenorm=True).cuda()
    m.norm = torch.nn.LayerNorm(64).cuda()
    assert m._plain_layer() is None
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert Castle(64, heads=2, dim_head=32, prenorm="layer").cuda()(torch.randn(1, 9, 64, device="cuda")).dtype == torch.bfloat16
    assert set(Castle(64, prenorm="layer").state_dict()) == {"norm.weight", "norm.bias", "to_all_qkv.weight", "combine_heads.weight"}


def test_only_some_parameters_of_a_layer_learn():
    torch.manual_seed(1)
    m = Castle(128, heads=2, prenorm="layer").cuda().bfloat16()
    x = torch.randn(2, 50, 128, device="cuda").bfloat16()
    g = torch.randn(2, 50, 128, device="cuda").bfloat16()
    full = dict(zip([n for n, _ in m.named_parameters()], torch.autograd.grad(m(x), list(m.parameters()), g)))
    for names in (["norm.bias"], ["norm.weight"], ["norm.bias", "combine_heads.weight"], ["to_all_qkv.weight"]):
        for n, p in m.named_parameters():
            p.requires_grad_(n in names)
        got = torch.autograd.grad(m(x), [dict(m.named_parameters())[n] for n in names], g)
        for n, t in zip(names, got):
            assert ((t.float() - full[n].float()).norm() / full[n].float().norm()).item() <= 16 * 2.0 ** -8, n
