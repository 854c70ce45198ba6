"""GPU: the sums in the tensor cores of the head's cross entropy, where the general tolerances (worst cases of all additions) are too wide to see them.

With u = 2^-24 and h half a step of the type."""
import pytest
import torch

from lookahead_keys_attention_b200 import castle_linear_cross_entropy, check_status

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
@pytest.mark.parametrize("n,dim,vocab", [(64, 8192, 1000), (200, 4096, 700), (1000, 4096, 20000), (40, 512, 300)])
def test_learnt_rows_have_probabilities_that_add_up(n, dim, vocab, dtype):
    """The gradient's logits are the same sums in the same order as those behind the log-sum-exp, so a row's probabilities add up to one: off by 2^-21 of
    an exponential, 300 u of their sum, and u |lse|, by which the log-sum-exp is rounded.  A column of ones in the weight has the row's sum of G as its
    dx: to the above comes h of the probabilities beside the target's (whose rounding is made up for; fp32: 2 u), and what adding them loses.
    Logits have an offset of some 50, as nothing in a loss holds them near zero; targets have about 0.999 of the probability, so G's entries are
    small differences.  (Sums of the whole contraction, not emptied on the way, were off by 3e-4 to
    1.6e-3 in 16 bits.)"""
    gen = torch.Generator("cuda").manual_seed(dim)
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    common, noise = rand(dim), rand(vocab, dim)
    noise -= (noise @ common)[:, None] * common / (common @ common)
    w = (2 * noise + common) * dim ** -0.5
    t = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    need = 7.0 + torch.log(torch.tensor(float(vocab)))
    x = 2 * noise[t] * (need / 4 * dim ** -0.5) + common * (50 * dim ** -0.5)
    w[:, 1] = 1.0
    x[:, 1] = 0.0
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    loss = castle_linear_cross_entropy(x, w, t, reduction="sum")
    (dx,) = torch.autograd.grad(loss, [x])
    check_status()
    z = x.double() @ w.double().t()
    lse = z.logsumexp(1)
    p = (z[torch.arange(n, device="cuda"), t] - lse).exp()
    assert 0.99 < p.median().item() < 0.99999 and z.amax() > 40
    h = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2 * U
    tol = 2.0 ** -21 + 300 * U + U * lse.abs() + h * (1 - p) + (vocab / 16 * (6 if dtype == torch.float32 else 1) + 64) * 2.0 ** -22 * 2 * (1 - p)
    off = dx[:, 1].double().abs()
    assert bool((off <= tol).all()), f"{off.max().item():.2e} beyond {tol.min().item():.2e}"


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_rows_of_the_types_lowest_value(dtype, sign):
    """Finite numbers however large have finite parts: a row with the type's lowest value in it (or the largest) has logits of some 1e37 and the loss and
    gradients that go with them, and the other rows keep theirs.  Losses: (32 + 8) additions of 2 u and the largest logit's rounding, 2^-18
    at most; gradients of such a row: one weight's row less another's, or the row itself, off by the type's rounding h and, in fp32, 4 u."""
    n, dim, vocab = 200, 64, 300
    gen = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(n, dim, device="cuda", generator=gen).to(dtype)
    w = (torch.randn(vocab, dim, device="cuda", generator=gen) * 0.1).to(dtype)
    t = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    far = torch.finfo(dtype).max * sign
    def call(x):
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = castle_linear_cross_entropy(xl, wl, t, reduction="none")
        return (loss.detach(), *torch.autograd.grad(loss, [xl, wl], torch.ones(n, device="cuda")))
    loss0, dx0, dw0 = call(x)
    x[7, 5] = far
    loss, dx, dw = call(x)
    check_status()
    z = x[7].double() @ w.double().t()
    want = z.amax() - z[t[7]]
    assert want > 1e36 and abs(loss[7].double() - want) <= 2.0 ** -18 * want
    others = [i for i in range(n) if i != 7]
    assert torch.equal(loss[others], loss0[others]) and torch.equal(dx[others], dx0[others])
    h = max(torch.finfo(dtype).eps / 2, 4 * U)
    top = int(z.argmax())
    row = w[top].double() - w[t[7]].double()
    assert bool(((dx[7].double() - row).abs() <= 2 * h * row.abs() + 4 * U * w[t[7]].double().abs()).all())
    assert bool(dw.isfinite().all())
    for v, g in ((top, 1.0), (int(t[7]), -1.0)):
        assert abs(dw[v, 5].double() - g * far) <= 2 * h * abs(far)
