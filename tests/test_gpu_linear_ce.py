"""GPU: cross entropy of a linear head and its gradients against the definition in 64 bits.

Tolerances, with u = 2^-24, h half a step of the type and s = 2^-22 for one addition in the tensor cores (which may cut what they add).
A logit sums its products 16 at a time: off by a = (steps + 4) s times the sum of their sizes, steps = dim / 16 (fp32: six times as many,
and the left-out products, 4 u).  A loss is off by twice the largest of these (the target's and the log-sum-exp's) and by what the
exponentials are off: 2^-21 each, their sum's 300 u, and the argument's rounding, 4 u per unit of the logits' spread.  Call
the latter three b.  The logits' gradient G is then off by (a + b) of p and by its rounding h |G| (fp32: 2 u), and the gradients by
the sum of these with |W| (or |x|), by the additions, (terms / 16 + 64) s, and their own rounding h.  These add sizes and allow
for every rounding to fall the same way; roundings that fall at random, two in a row of at most half a step, have a mean
square of at most (2/3) h^2, so the norm of the error is also held below h times the norm of the result (16-bit types)."""
import pytest
import torch

from lookahead_keys_attention_b200 import castle_linear_cross_entropy, check_status

pytestmark = pytest.mark.gpu
U, S = 2.0 ** -24, 2.0 ** -22
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def case(n, dim, vocab, dtype, ignored=0.0, seed=0, spread=2.0):
    gen = torch.Generator("cuda").manual_seed(seed + 7 * n + vocab)
    w = (torch.randn(vocab, dim, device="cuda", generator=gen) * spread * dim ** -0.5).to(dtype)
    x = torch.randn(n, dim, device="cuda", generator=gen).to(dtype)
    t = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    t[torch.rand(n, device="cuda", generator=gen) < ignored] = -100
    return x, w, t


def check(x, w, t, reduction="mean", up=None, norms=True):
    """One call and its gradients against the formulas; the whole logits are formed in 64 bits."""
    dtype, n, dim, vocab = x.dtype, x.shape[0], x.shape[1], w.shape[0]
    xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = castle_linear_cross_entropy(xl, wl, t, reduction=reduction)
    if up is None:
        up = torch.full((), 3.0, device="cuda") if reduction != "none" else torch.linspace(-2, 3, n, device="cuda")
    dx, dw = torch.autograd.grad(loss, [xl, wl], up)
    check_status()
    assert loss.dtype == torch.float32 and loss.shape == up.shape and dx.shape == x.shape and dw.shape == w.shape and dx.dtype == dw.dtype == dtype

    h = half_step(dtype)
    rows = (t != -100).nonzero()[:, 0]
    k = torch.arange(len(rows), device="cuda")
    X, W, T = x.double()[rows], w.double(), t[rows].long()
    z, size = X @ W.t(), X.abs() @ W.abs().t()
    steps = dim / 16 * (6 if dtype == torch.float32 else 1)
    a = ((steps + 4) * S + (4 * U if dtype == torch.float32 else 0)) * size.amax(1, keepdim=True)
    lse = z.logsumexp(1, keepdim=True)
    b = 2.0 ** -21 + 300 * U + 4 * U * (z.amax(1, keepdim=True) - z.amin(1, keepdim=True) + lse.abs())
    each = torch.zeros(n, dtype=torch.float64, device="cuda")
    each[rows] = (lse - z.gather(1, T[:, None]))[:, 0]
    tol = torch.zeros_like(each)
    tol[rows] = (2 * a + b)[:, 0]
    if reduction == "none":
        assert bool(((loss.double() - each).abs() <= tol + 2 * U * each.abs()).all())
    else:
        div = max(len(rows), 1) if reduction == "mean" else 1
        assert abs(loss.item() - each.sum().item() / div) <= tol.sum().item() / div + 4 * U * each.abs().sum().item() / div

    c = up.double().expand(n)[rows][:, None] / (len(rows) if reduction == "mean" else 1)
    p = (z - lse).exp()
    del z, size
    off = p * (2 * a + 2 * b + 4 * U) * c.abs()
    G = p
    G[k, T] -= 1
    G *= c
    ho = h if dtype != torch.float32 else 2 * U
    off += ho * G.abs() + (2.0 ** -24 * 2.0 ** -14 * 2 * c.abs().max() if dtype == torch.float16 else 0)   # fp16 below its normal numbers
    # A probability below 2^-126, the smallest normal number of fp32, is taken as zero (an exponential that flushes to zero): G is off by up
    # to 2^-126 |c|, and by as much again where a part of it in the operands' type is below that.
    off += 2 * 2.0 ** -126 * c.abs().max()
    def within(got, want, tol, what):
        tol = tol * (1 + 2 * h) + h * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        excess = ((got.double() - want).abs() - tol).max().item()
        assert excess <= 0, f"{what}: {excess:.3e} beyond the tolerance"
        if norms and dtype != torch.float32 and want.norm() > 0:
            far = ((got.double() - want).norm() / want.norm()).item()
            assert far <= h, f"{what}: {far:.3e} of its norm"
    want = torch.zeros(n, dim, dtype=torch.float64, device="cuda")
    want[rows] = G @ W
    tol = torch.zeros_like(want)
    extra = (vocab / 16 * (6 if dtype == torch.float32 else 1) + 64) * S
    tol[rows] = (off + extra * G.abs()) @ W.abs()
    within(dx, want, tol, "dx")
    assert not bool(dx[t == -100].any())
    extra = (len(rows) / 16 * (6 if dtype == torch.float32 else 1) + 64) * S
    within(dw, G.t() @ X, (off + extra * G.abs()).t() @ X.abs(), "dweight")
    return loss, dx, dw


SIZES = [(1, 64, 100), (1, 8, 1), (2, 1, 3), (5, 3, 17), (37, 72, 300), (128, 64, 256), (129, 512, 257), (197, 512, 256), (300, 520, 1000), (1000, 136, 5003),
         (513, 1333, 771), (4200, 64, 129), (3, 2048, 20000), (257, 8192, 300)]


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,dim,vocab", SIZES)
def test_sizes(n, dim, vocab, dtype):
    check(*case(n, dim, vocab, dtype), norms=n * vocab > 1000)


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("ignored", [0.0, 0.4, 0.99])
def test_reductions_and_ignored_targets(reduction, ignored, dtype):
    x, w, t = case(700, 136, 1003, dtype, ignored)
    t[5] = 1002
    check(x, w, t, reduction)
    check(x, w, t.int(), reduction)


@pytest.mark.parametrize("n,dim,vocab,dtype", [(8200, 64, 70000, torch.bfloat16), (8200, 64, 30000, torch.float32), (16, 4096, 50000, torch.float32)])
def test_a_vocabulary_in_pieces(n, dim, vocab, dtype):
    """More columns than one piece of the scratch takes: in the backward, there in fp32's three parts, and in an fp32 forward."""
    check(*case(n, dim, vocab, dtype, 0.1))


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,dim,vocab", [(40, 21, 500), (300, 107, 513), (4200, 301, 1700), (1700, 301, 4200), (600, 260, 2000), (8200, 65, 70000)])
def test_rows_at_odd_places(n, dim, vocab, dtype):
    """Rows that begin at every place in 16 bytes: read and written in parts, whole tiles, shared ones and several pieces of a vocabulary."""
    if vocab == 70000 and dtype == torch.float32:
        vocab = 30000
    check(*case(n, dim, vocab, dtype, 0.1))


def test_nothing_to_learn():
    for reduction in ("mean", "sum", "none"):
        x, w, t = case(300, 64, 500, torch.bfloat16)
        t[:] = -100
        x, w = x.requires_grad_(), w.requires_grad_()
        loss = castle_linear_cross_entropy(x, w, t, reduction=reduction)
        assert bool(loss.isnan()) if reduction == "mean" else not bool(loss.any())
        dx, dw = torch.autograd.grad(loss, [x, w], torch.ones_like(loss))
        assert not bool(dx.any()) and not bool(dw.any())      # a batch without targets moves nothing
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.randn(10, 64, device="cuda", requires_grad=True)
    loss = castle_linear_cross_entropy(x, w, torch.empty(0, dtype=torch.int64, device="cuda"), reduction="sum")
    loss.backward()
    assert loss.item() == 0 and x.grad.shape == (0, 64) and not bool(w.grad.any())
    check_status()


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_what_ignored_rows_hold_reaches_nothing(dtype):
    x, w, t = case(400, 72, 300, dtype, 0.3, seed=1)
    t[399], t[0] = -100, -100
    clean = check(x, w, t)
    x = x.clone()
    skip = (t == -100).nonzero()[:, 0]
    x[skip[::2]], x[skip[1::2]] = float("nan"), float("inf")
    x[skip[0]] = torch.finfo(dtype).min
    again = check_values(x, w, t)
    assert all(torch.equal(a, b) for a, b in zip(clean, again))


def check_values(x, w, t, reduction="mean", up=3.0):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = castle_linear_cross_entropy(x, w, t, reduction=reduction)
    return (loss, *torch.autograd.grad(loss, [x, w], torch.full_like(loss, up)))


def test_rows_that_are_not_numbers_stay_alone():
    x, w, t = case(300, 64, 500, torch.bfloat16)
    clean, dx0, _ = check_values(x, w, t, "none", 1.0)
    x = x.clone()
    x[7, 3], x[200] = float("nan"), float("inf")
    loss, dx, dw = check_values(x, w, t, "none", 1.0)
    others = [i for i in range(300) if i not in (7, 200)]
    assert torch.equal(loss[others], clean[others]) and bool(loss[[7, 200]].isnan().all()) and torch.equal(dx[others], dx0[others])
    assert bool(dx[7].isnan().all()) and bool(dw.isnan().any())
    check_status()


def test_large_and_far_apart_logits():
    """Logits in the thousands: probabilities of one and of nothing."""
    x, w, t = case(200, 64, 300, torch.float32, spread=200.0)
    loss, dx, dw = check(x, w, t, "none")
    assert bool(loss.isfinite().all()) and bool(dx.isfinite().all())
    check(x.bfloat16(), w.bfloat16(), t)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-6, 1.0, 1e4, 1e30])
def test_upstream_gradients_of_any_size(scale):
    """bf16 has the range of fp32: small and large upstream gradients lose nothing."""
    x, w, t = case(200, 64, 300, torch.bfloat16)
    _, dx1, dw1 = check_values(x, w, t, "sum", 1.0)
    _, dx, dw = check_values(x, w, t, "sum", scale)
    for a, b in ((dx, dx1), (dw, dw1)):
        want = b.double() * scale
        # one rounding of b, one of a, and of G where scale is no power of two
        assert ((a.double() - want).norm() <= 3 * half_step(torch.bfloat16) * want.norm()).item()


def test_fp16_probabilities_keep_their_precision():
    """Gradients of a loss with a loss scale, in fp16: most of G's entries are far below fp16's normal numbers."""
    x, w, t = case(500, 128, 20000, torch.float16, spread=1.0)
    check(x, w, t, "mean", up=torch.full((), 2.0 ** 14, device="cuda"))
    check(x, w, t, "none", up=torch.logspace(-3, 1, 500, device="cuda"))


@pytest.mark.parametrize("bad", [-1, 500, 2 ** 40])
def test_a_target_outside_the_vocabulary_is_reported(bad):
    x, w, t = case(300, 64, 500, torch.bfloat16)
    t[100] = bad
    assert bool(castle_linear_cross_entropy(x, w, t).isnan())
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        check_status()
    loss, dx, dw = check_values(x, w, t, "none", 1.0)
    assert int(loss.isnan().sum()) == 1 and bool(loss[100].isnan()) and bool(dx.isfinite().all()) and not bool(dx[100].any()) and bool(dw.isfinite().all())
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        check_status()
    assert castle_linear_cross_entropy(x, w, t, ignore_index=bad).isfinite()
    check_status()


def test_a_class_can_be_ignored():
    """As a padding token's number is."""
    x, w, t = case(300, 64, 50, torch.float32)
    a = check_values(x, w, t.where(t != 7, -100))
    loss = castle_linear_cross_entropy(x, w, t, ignore_index=7)
    assert torch.equal(loss, a[0])


def test_strides():
    x, w, t = case(24 * 10, 64, 300, torch.bfloat16)
    def same(a, wt, tt):
        got, want = check_values(a, wt, tt, "sum", 1.0), check_values(a.contiguous(), wt.contiguous(), tt.contiguous(), "sum", 1.0)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    big = torch.randn(24, 10, 3, 72, device="cuda").bfloat16()
    table = torch.randn(300, 2, 72, device="cuda").bfloat16()
    same(big[:, :, 1, :64], w, t.view(24, 10))                                    # rows with a stride
    same(big[:, :, 1, 1:65], w, t.view(24, 10))                                   # not at 16-byte boundaries
    same(big[:, 2:7, 0, :64], table[:, 1, :64], t.view(24, 10)[:, 2:7])           # rows without a single stride, a strided table
    same(big[:, 2:7, 0, :64], table[:, 1, 3:67], t.view(24, 10)[:, 2:7])
    same(big[:, :, 0, :64].transpose(0, 1), w.t().contiguous().t(), t.view(24, 10).t())
    same(big[:1, :1, 0, :64].expand(24, 10, 64), w, t.view(24, 10))               # one row repeated
    same(x[0], w, t[0])                                                           # one row as a vector
    up = torch.full((1, 1), 0.5, device="cuda").expand(24, 10)
    x3 = x.view(24, 10, 64).requires_grad_()
    a = torch.autograd.grad(castle_linear_cross_entropy(x3, w, t.view(24, 10), reduction="none"), [x3], up)[0]
    b = torch.autograd.grad(castle_linear_cross_entropy(x3, w, t.view(24, 10), reduction="sum"), [x3], up[0, 0])[0]
    assert torch.equal(a, b)


def test_only_one_gradient():
    x, w, t = case(300, 136, 700, torch.bfloat16, 0.2)
    _, dx, dw = check_values(x, w, t)
    for i, want in ((0, dx), (1, dw)):
        leaves = [x.clone().requires_grad_(i == 0), w.clone().requires_grad_(i == 1)]
        (got,) = torch.autograd.grad(castle_linear_cross_entropy(*leaves, t), [leaves[i]], torch.full((), 3.0, device="cuda"))
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("reduction,up", [("mean", 3.0), ("sum", 1.7), ("none", None)])
def test_dx_of_rows_that_have_not_learnt(reduction, up, dtype):
    """A row's gradient is the target's row of the weight but for little; its coefficient and that entry of G are exact or made up for, so
    what is left is the result's rounding: a mean square of at most h^2 / 3, here with a tenth on top for the other entries of G."""
    n, dim, vocab = 300, 256, 20000
    x, w, t = case(n, dim, vocab, dtype, spread=0.5)
    up = torch.linspace(0.3, 2.9, n, device="cuda") if up is None else torch.full((), up * (n if reduction == "mean" else 1), device="cuda")
    xl = x.requires_grad_()
    (dx,) = torch.autograd.grad(castle_linear_cross_entropy(xl, w, t, reduction=reduction), [xl], up)
    G = torch.softmax(x.double() @ w.double().t(), 1)
    G[torch.arange(n, device="cuda"), t] -= 1
    want = (up.double().expand(n)[:, None] / (n if reduction == "mean" else 1) * G) @ w.double()
    assert ((dx.double() - want).norm() <= 1.1 * half_step(dtype) / 3 ** 0.5 * want.norm()).item()


def test_the_same_from_call_to_call():
    x, w, t = case(3000, 256, 5001, torch.bfloat16, 0.2)
    first = check_values(x, w, t)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, check_values(x, w, t)))


def test_refusals():
    x, w, t = case(8, 16, 30, torch.bfloat16)
    for args in [(x.double(), w.double(), t), (x, w.float(), t), (x, w[:, :8], t), (x, w[0], t), (x, w[:0], t), (x, w, t[:7]), (x, w, t.float()), (x.cpu(), w, t),
                 (x, w.cpu(), t), (x, w, t.cpu()), (x[0, 0], w, t[0])]:
        with pytest.raises(RuntimeError, match="castle_linear_cross_entropy"):
            castle_linear_cross_entropy(*args)
    with pytest.raises(ValueError, match="reduction"):
        castle_linear_cross_entropy(x, w, t, reduction="max")
    leaf = x.requires_grad_()
    (g,) = torch.autograd.grad(castle_linear_cross_entropy(leaf, w, t), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_gradient_against_differences():
    """Along random directions, by central differences of the fp32 losses (64-bit sums)."""
    x, w, t = case(40, 32, 60, torch.float32)
    loss, dx, dw = check_values(x, w, t, "sum", 1.0)
    gen = torch.Generator("cuda").manual_seed(1)
    for which, grad in ((0, dx), (1, dw)):
        step = torch.randn(grad.shape, device="cuda", generator=gen)
        e = 2.0 ** -8
        def at(s):
            moved = [x + s * e * step, w] if which == 0 else [x, w + s * e * step]
            return castle_linear_cross_entropy(*moved, t, reduction="none").double().sum()
        slope, want = (at(1) - at(-1)) / (2 * e), (grad.double() * step.double()).sum()
        # a row's third derivative is below (twice the spread of its logits' derivatives)^3; e^2 / 6 of it, and 100 u per loss / e
        moves = (step.double() @ w.double().t()) if which == 0 else (x.double() @ step.double().t())
        bound = e * e / 6 * ((moves.amax(1) - moves.amin(1)) ** 3).sum() + 40 * 100 * U * 10 / e
        assert abs(slope - want) <= bound
