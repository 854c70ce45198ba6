"""GPU: second derivatives are refused where a gradient is used in another loss (create_graph), not taken for zero: a penalty on a gradient would
silently lose its share of the operator's inputs.  First derivatives under create_graph are the same as without."""
import pytest
import torch

from lookahead_keys_attention_b200 import Castle, castle_attention, castle_attention_packed, castle_embedding, castle_layer_norm, castle_linear_cross_entropy

pytestmark = pytest.mark.gpu


def leaf(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).requires_grad_()


def operators():
    """name: (operator, its differentiable inputs)"""
    t = torch.arange(12, device="cuda") % 7
    return {"castle_embedding": (lambda w: castle_embedding(t, w, 2.0), [leaf(30, 16)]),
            "castle_layer_norm": (castle_layer_norm, [leaf(12, 16), leaf(16, seed=1), leaf(16, seed=2)]),
            "castle_linear_cross_entropy": (lambda x, w: castle_linear_cross_entropy(x, w, t, reduction="none"), [leaf(12, 16), leaf(30, 16, seed=1)])}


def refused(make, leaves, name):
    """make(): the operator's result and an upstream gradient."""
    out, up = make()
    plain = torch.autograd.grad(out, leaves, up.detach())
    out, up = make()
    first = torch.autograd.grad(out, leaves, up, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, first))
    penalty = sum((g.float() ** 2).sum() for g in first)
    with pytest.raises(RuntimeError, match=f"{name}: second derivatives are not implemented"):
        (out.float().sum() + penalty).backward()                 # something else in the loss has a graph
    return first


@pytest.mark.parametrize("name", ["castle_embedding", "castle_layer_norm", "castle_linear_cross_entropy"])
def test_a_penalty_on_the_gradient_is_refused(name):
    op, leaves = operators()[name]
    scale = leaf(1, seed=9)
    def make():
        out = op(*leaves)
        return out, torch.ones_like(out) * scale                 # an upstream gradient that has a graph
    refused(make, leaves, name)
    if name != "castle_embedding":                               # (whose gradient depends on the upstream one alone)
        def constant():
            out = op(*leaves)
            return out, torch.ones_like(out)
        for i, g in enumerate(refused(constant, leaves, name)):
            assert g.requires_grad
            with pytest.raises(RuntimeError, match="second derivatives"):
                torch.autograd.grad(g.sum(), leaves[:1], retain_graph=True)


def test_what_does_not_need_them_goes_on():
    """A gradient kept with its graph, a penalty on another gradient, and an upstream gradient that leads nowhere."""
    for name, (op, leaves) in operators().items():
        other = leaf(5, seed=4)
        out = op(*leaves).sum() + (other ** 3).sum()
        (g,) = torch.autograd.grad(out, [other], create_graph=True)
        (g ** 2).sum().backward()
        assert torch.allclose(other.grad, 36 * other.detach() ** 3)
        out = op(*leaves).sum()
        out.backward(create_graph=True)
        want = torch.autograd.grad(op(*leaves).sum(), leaves)
        assert all(torch.equal(l.grad, w) for l, w in zip(leaves, want))
        for l in leaves:
            l.grad = None
    t, w = torch.arange(12, device="cuda"), leaf(30, 16)
    (dw,) = torch.autograd.grad(castle_embedding(t, w).sum(), [w], create_graph=True)
    assert not dw.requires_grad


def test_a_traced_operator_refuses_them_too():
    t = torch.arange(12, device="cuda")
    x, w = leaf(12, 16), leaf(30, 16, seed=1)
    traced = torch.jit.trace(lambda x, w: castle_linear_cross_entropy(x, w, t), (x, w), check_trace=False)
    (dx,) = torch.autograd.grad(traced(x, w), [x], create_graph=True)
    assert torch.equal(dx, torch.autograd.grad(castle_linear_cross_entropy(x, w, t), [x])[0])
    with pytest.raises(RuntimeError, match="second derivatives"):
        ((dx ** 2).sum() + w.sum()).backward()


def test_attention_refuses_them():
    six = [leaf(2, 2, 40, 64, seed=i) for i in range(6)]
    packed = leaf(2, 40, 6, 2, 64)
    for op, leaves in ((lambda *v: castle_attention(*v, 0.125), six), (lambda v: castle_attention_packed(v, 0.125), [packed])):
        for up in (1.0, leaf(1, seed=9)):
            def make():
                out = op(*leaves)
                return out, torch.ones_like(out) * up
            refused(make, leaves, "castle_attention")


@pytest.mark.parametrize("prenorm", [False, True, "layer"])
def test_a_layer_refuses_them(prenorm):
    torch.manual_seed(0)
    m = Castle(64, heads=2, dim_head=64, prenorm=prenorm).cuda()
    x = leaf(2, 40, 64)
    def make():
        out = m(x)
        return out, torch.ones_like(out)
    refused(make, [x, *m.parameters()], "Castle")
    for p in m.parameters():                                     # one that learns is enough: another's gradient depends on it
        p.requires_grad_(False)
    refused(make, [x], "Castle")
    handle = m.combine_heads.register_forward_hook(lambda *a: None)   # the submodules as modules, around the core's own node
    (g,) = torch.autograd.grad(m(x).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="castle_attention: second derivatives"):
        ((g ** 2).sum() + x.sum()).backward()
    handle.remove()
    out = m(x)
    (g,) = torch.autograd.grad(out, [x], torch.ones_like(out))   # without create_graph nothing is added
    assert not g.requires_grad
