"""The losses and gradients of the head's cross entropy hold 32 bits where they say so: norms of the errors, in which single roundings do not add up as
they do in the bounds of single values.

With u = 2^-24, logits z of spread 2, log-sum-exps up to 12, and roundings that fall at random (0.3 of a step each, squares added):

* a logit's blocks of 24 (fp32) or 32 (16 bits) additions in the tensor cores, each of which cuts half a step of a sum that grows from nothing: at most 16 u
  of a block's size, blocks of either sign, so 16 u of the products' root of squares: 2 u 16 at random places, some 2e-6; and a row's
  loss is between 6 and 12: its norm is off by less than 2^-21 in 16 bits; in fp32 with its shorter blocks by less than 2^-22.
* fp32 gradients: an exponential 2^-22.5, its argument's two roundings where most of a probability lies (within 8 of the log-sum-exp) 5 u, the
  log-sum-exp's 5 u, a logit's 8 u: together below 12 u of their norm.

One product of parts less than six, a part of G less, two parts that changed places or accumulators that are not emptied are off by more; the first test
says how much, in 64 bits, with each of these mistakes in turn."""
import pytest
import torch

U = 2.0 ** -24
LOSS_F32, LOSS_16, GRAD_F32 = 2.0 ** -22, 2.0 ** -21, 12 * U
SIX = [(0, 2), (2, 0), (1, 1), (0, 1), (1, 0), (0, 0)]


def case(n, dim, vocab, dtype, device, seed=0):
    gen = torch.Generator(device).manual_seed(seed + 7 * n + vocab)
    w = (torch.randn(vocab, dim, device=device, generator=gen) * 2 * dim ** -0.5).to(dtype)
    x = torch.randn(n, dim, device=device, generator=gen).to(dtype)
    return x, w, torch.randint(0, vocab, (n,), device=device, generator=gen)


def far(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def parts(v):
    a = v.bfloat16().float()
    b = (v - a).bfloat16().float()
    return [t.double() for t in (a, b, (v - a - b).bfloat16().float())]


@pytest.mark.parametrize("mistake", ["none", "products 1 1", "products 0 2", "products 2 0", "three products", "one product", "changed places", "two parts of G"])
@pytest.mark.parametrize("n,dim,vocab", [(37, 72, 300), (129, 512, 257), (600, 64, 300)])
def test_the_bounds_see_a_missing_part(n, dim, vocab, mistake):
    terms = {"products 1 1": [t for t in SIX if t != (1, 1)], "products 0 2": [t for t in SIX if t != (0, 2)], "products 2 0": [t for t in SIX if t != (2, 0)],
             "three products": SIX[3:], "one product": SIX[5:], "changed places": [(0, 2), (2, 0), (1, 1), (0, 1), (0, 1), (0, 0)]}.get(mistake, SIX)
    x, w, t = case(n, dim, vocab, torch.float32, "cpu")
    k = torch.arange(n)
    def product(a, b):
        return sum(a[i] @ b[j] for i, j in terms)
    def results(z, dx_of, dw_of):
        g = z.softmax(1)
        g[k, t] -= 1
        return z.logsumexp(1) - z[k, t], dx_of(g), dw_of(g)
    X, W = parts(x), parts(w)
    G = lambda g: [p * (i < 2 or mistake != "two parts of G") for i, p in enumerate(parts(g.float()))]
    got = results(product(X, [p.t() for p in W]), lambda g: product(G(g), W), lambda g: product([p.t() for p in G(g)], X))
    want = results(x.double() @ w.double().t(), lambda g: g @ w.double(), lambda g: g.t() @ x.double())
    off = [far(a, b) for a, b in zip(got, want)]
    if mistake == "none":
        assert off[0] <= LOSS_F32 / 16 and max(off[1:]) <= GRAD_F32 / 16
    else:
        assert max(off[1:]) > GRAD_F32 and (off[0] > LOSS_F32 or mistake == "two parts of G")


def exact(x, w, t):
    z = x.double() @ w.double().t()
    k = torch.arange(len(t), device=x.device)
    loss = z.logsumexp(1) - z[k, t]
    g = z.softmax(1)
    g[k, t] -= 1
    return loss, g @ w.double(), g.t() @ x.double()


# single CTAs with all parts in a stage, with one; pairs; rows and widths that end inside a tile; shared tiles of dx, of dW; pieces in the backward, in the forward
@pytest.mark.gpu
@pytest.mark.parametrize("n,dim,vocab", [(37, 72, 300), (129, 512, 257), (197, 512, 256), (300, 520, 1000), (1000, 1333, 771), (2048, 512, 3000), (2000, 136, 3001),
                                         (4200, 64, 129), (600, 260, 20000), (257, 8192, 300), (8200, 64, 30000), (64, 4096, 50000)])
def test_fp32(n, dim, vocab):
    from lookahead_keys_attention_b200 import castle_linear_cross_entropy, check_status
    x, w, t = case(n, dim, vocab, torch.float32, "cuda")
    leaves = [v.requires_grad_() for v in (x, w)]
    loss = castle_linear_cross_entropy(*leaves, t, reduction="none")
    got = (loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones_like(loss)))
    check_status()
    for what, a, b, most in zip(("losses", "dx", "dweight"), got, exact(x.detach(), w.detach(), t), (LOSS_F32, GRAD_F32, GRAD_F32)):
        assert far(a, b) <= most, f"{what}: {far(a, b):.2e} of its norm"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("n,dim,vocab", [(300, 512, 1000), (300, 576, 1000), (129, 1333, 771), (500, 4096, 3000), (3000, 4096, 5003), (64, 8192, 1000)])
def test_losses_of_16_bit_rows(n, dim, vocab, dtype):
    from lookahead_keys_attention_b200 import castle_linear_cross_entropy, check_status
    x, w, t = case(n, dim, vocab, dtype, "cuda")
    loss = castle_linear_cross_entropy(x, w, t, reduction="none")
    check_status()
    z = x.double() @ w.double().t()
    assert far(loss, z.logsumexp(1) - z[torch.arange(n, device="cuda"), t]) <= LOSS_16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_a_forward_of_16_bit_rows_in_pieces(dtype):
    """65536 rows leave a forward's scratch for 262144 columns at a time: the second piece reads the weight where it lies from its own first row on, and joins the
    first one's maxima, sums and target logits.  Targets on either side of the border and next to it; the logits of a sample of rows in 64 bits.  (Eight
    products make a logit: off by 2 u of it, a loss by 2^-21 of an exponential, 300 u of their sum and 4 u of the log-sum-exp.)"""
    from lookahead_keys_attention_b200 import castle_linear_cross_entropy, check_status
    n, dim, vocab, border = 65536, 8, 300001, 262144
    x, w, t = case(n, dim, vocab, dtype, "cuda")
    t[:6] = torch.tensor([border - 1, border, 0, vocab - 1, border + 255, border - 256], device="cuda")
    t[100:200] = -100
    xl, wl = x.requires_grad_(), w.requires_grad_()
    loss = castle_linear_cross_entropy(xl, wl, t, reduction="none")
    mean = castle_linear_cross_entropy(x.detach(), w.detach(), t)
    check_status()
    rows = torch.cat([torch.arange(6), torch.arange(200, n, 331)]).cuda()
    assert bool((t[rows] < border).any()) and bool((t[rows] >= border).any())
    z = x[rows].double() @ w.double().t()
    lse = z.logsumexp(1)
    want = lse - z[torch.arange(len(rows), device="cuda"), t[rows]]
    tol = 4 * U * z.abs().amax(1) + 2.0 ** -21 + 300 * U + 4 * U * lse.abs() + 2 * U * want.abs()
    assert bool(((loss[rows].double() - want).abs() <= tol).all())
    assert not bool(loss[100:200].any())
    assert abs(mean.double() - loss.double().sum() / (n - 100)) <= 2 * U * mean
    (dx,) = torch.autograd.grad(loss, [xl], torch.ones_like(loss))      # (37 pieces)
    check_status()
    p = z.softmax(1)
    p[torch.arange(len(rows), device="cuda"), t[rows]] -= 1
    assert far(dx[rows], p @ w.double()) <= torch.finfo(dtype).eps / 2
