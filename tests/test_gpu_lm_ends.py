"""GPU: the operators around a language model's layers as they are used together, captured, on several streams and threads, under what
autograd offers, and with offsets beyond 32 bits."""
import threading

import pytest
import torch
import torch.nn.functional as F

from lookahead_keys_attention_b200 import (Castle, castle_embedding, castle_layer_norm, castle_linear_cross_entropy, check_status, release_workspaces)

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class Model(torch.nn.Module):
    """Tokens, two layers, a final norm and the loss, with one table at both ends; `own`: with this package's operators."""

    def __init__(self, vocab, dim, heads, own):
        super().__init__()
        self.own, self.scale = own, dim ** 0.5
        self.table = torch.nn.Parameter(torch.randn(vocab, dim) * dim ** -0.5)
        self.layers = torch.nn.ModuleList([Castle(dim, heads=heads, prenorm="layer") for _ in range(2)])
        self.norm = torch.nn.LayerNorm(dim)

    def forward(self, tokens, targets):
        if self.own:
            h = castle_embedding(tokens, self.table, scale=self.scale, padding_idx=0)
        else:
            h = (F.embedding(tokens, self.table, padding_idx=0).float() * self.scale).to(self.table.dtype)
        for layer in self.layers:
            h = layer(h) + h
        if self.own:
            h = castle_layer_norm(h, self.norm.weight, self.norm.bias, self.norm.eps)
            return castle_linear_cross_entropy(h, self.table, targets)
        return F.cross_entropy((self.norm(h).float() @ self.table.float().t()).flatten(0, 1), targets.flatten())


def batch(vocab, b=3, n=150, seed=0):
    gen = torch.Generator("cuda").manual_seed(seed)
    ids = torch.randint(0, vocab, (b, n + 1), device="cuda", generator=gen)
    x, y = ids[:, :-1], ids[:, 1:].clone()
    y[0, 100:] = -100
    return x, y


@pytest.mark.parametrize("dtype", TYPES.values(), ids=TYPES.keys())
def test_a_training_step(dtype):
    """Against the same model with torch's operators around the layers.  Each result of an operator is rounded to the type once in either
    (half a step, and the layers' operands have 16 bits in any case); a gradient passes some ten such results: differences in the
    norm of at most ten steps of the type."""
    torch.manual_seed(0)
    own = Model(307, 128, 2, True).cuda().to(dtype)
    torch.manual_seed(0)
    ref = Model(307, 128, 2, False).cuda().to(dtype)
    x, y = batch(307)
    losses = [m(x, y) for m in (own, ref)]
    up = 1024.0 if dtype == torch.float16 else 1.0
    grads = [torch.autograd.grad(l * up, list(m.parameters())) for l, m in zip(losses, (own, ref))]
    check_status()
    step = max(torch.finfo(dtype).eps, 2.0 ** -10)
    assert abs(losses[0].item() - losses[1].item()) <= 10 * step
    for (name, _), a, b in zip(own.named_parameters(), *grads):
        far = ((a.double() - b.double()).norm() / b.double().norm()).item()
        assert far <= 10 * step, f"{name}: {far:.2e}"


def test_a_captured_training_step():
    torch.manual_seed(0)
    m = Model(307, 128, 2, True).cuda().bfloat16()
    x, y = batch(307)
    def step(x, y):
        loss = m(x, y)
        return (loss.detach(), *torch.autograd.grad(loss, list(m.parameters())))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, y)
    for seed in (1, 2):
        nx, ny = batch(307, seed=seed)
        x.copy_(nx)
        y.copy_(ny)
        graph.replay()
        got = [t.clone() for t in out]
        want = step(nx, ny)
        check_status()
        # the projections of a capture are the library's, eager ones this package's: other orders of addition, ten steps as above
        for a, b in zip(got, want):
            assert ((a.double() - b.double()).norm() <= 10 * 2.0 ** -7 * b.double().norm()).item()


def ops(seed):
    """Each operator's training call with inputs of its own: a function that returns its results."""
    gen = torch.Generator("cuda").manual_seed(seed)
    def rand(*s):
        return torch.randn(*s, device="cuda", generator=gen).bfloat16().requires_grad_()
    t = torch.randint(0, 501, (900,), device="cuda", generator=gen)
    y = t.clone()
    y[::3] = -100
    table, x, w, b, g = rand(501, 264), rand(900, 264), rand(264), rand(264), rand(900, 264).detach()
    def embed():
        out = castle_embedding(t, table, 2.0)
        return (out.detach(), *torch.autograd.grad(out, [table], g))
    def norm():
        out = castle_layer_norm(x, w, b)
        return (out.detach(), *torch.autograd.grad(out, [x, w, b], g))
    def loss():
        out = castle_linear_cross_entropy(x, table, y)
        return (out.detach(), *torch.autograd.grad(out, [x, table]))
    return {"embed": embed, "norm": norm, "loss": loss}


@pytest.mark.parametrize("name", ["embed", "norm", "loss"])
def test_graphs_of_one_stream_replay_in_any_order(name):
    """Two graphs with scratch of their own, beside eager calls on the stream that they were captured on."""
    calls = [ops(i)[name] for i in range(2)]
    want = [c() for c in calls]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for c in calls:
            c()
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            out = c()
        graphs.append((g, out))
    for i in (1, 0, 0, 1):
        for t in graphs[i][1]:
            t.zero_()
        torch.cuda.synchronize()
        graphs[i][0].replay()
        with torch.cuda.stream(stream):
            eager = calls[1 - i]()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[1 - i]))
    check_status()


@pytest.mark.parametrize("name", ["embed", "norm", "loss"])
def test_streams_side_by_side(name):
    calls = [ops(i)[name] for i in range(3)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    check_status()


def test_threads_on_one_stream():
    sets = [ops(i) for i in range(3)]
    want = [{k: f() for k, f in s.items()} for s in sets]
    torch.cuda.synchronize()
    bad = []
    def work(i):
        for _ in range(10):
            for k, f in sets[i].items():
                got = f()
                torch.cuda.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i][k])):
                    bad.append((i, k))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    check_status()


def test_scratch_given_back_between_forward_and_backward():
    x, w, t = torch.randn(600, 64, device="cuda", requires_grad=True), torch.randn(900, 64, device="cuda", requires_grad=True), torch.arange(600, device="cuda")
    want = torch.autograd.grad(castle_linear_cross_entropy(x, w, t), [x, w])
    loss = castle_linear_cross_entropy(x, w, t)
    release_workspaces()
    dirt = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]
    del dirt
    got = torch.autograd.grad(loss, [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_what_autograd_offers():
    """Saved tensors on the CPU, recomputed activations, a second backward of a kept graph, an input changed after the forward."""
    from torch.utils.checkpoint import checkpoint
    for name in ("embed", "norm", "loss"):
        call = ops(5)[name]
        want = call()
        with torch.autograd.graph.save_on_cpu():
            assert all(torch.equal(a, b) for a, b in zip(call(), want))
    x = torch.randn(50, 64, device="cuda", requires_grad=True)
    w = torch.randn(300, 64, device="cuda", requires_grad=True)
    t = torch.arange(50, device="cuda")
    def head(x, w):
        return castle_linear_cross_entropy(castle_layer_norm(x, w[0], w[1]), w, t)
    want = torch.autograd.grad(head(x, w), [x, w])
    got = torch.autograd.grad(checkpoint(head, x, w, use_reentrant=False), [x, w])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    loss = head(x, w)
    first = torch.autograd.grad(loss, [x, w], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(loss, [x, w])))
    with pytest.raises(RuntimeError, match="second time|already been freed"):
        torch.autograd.grad(loss, [x, w])
    for f in (lambda v: castle_layer_norm(v).sum(), lambda v: castle_linear_cross_entropy(v, w, t)):
        v = (x * 1).detach().requires_grad_()
        moved = v * 1
        out = f(moved)
        with torch.no_grad():
            moved.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()


def test_hooks_that_change_a_saved_tensor_are_refused():
    x, w, t = torch.randn(20, 64, device="cuda", requires_grad=True), torch.randn(30, 64, device="cuda", requires_grad=True), torch.arange(20, device="cuda")
    for call in (lambda: castle_layer_norm(x, w[0]).sum(), lambda: castle_linear_cross_entropy(x, w, t), lambda: castle_embedding(t, w).sum()):
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: s[:-1] if s.dim() else s):
            out = call()
        with pytest.raises(RuntimeError, match="saved tensor"):
            out.backward()


def test_a_refused_saved_tensor_names_its_operator():
    x, w, t = torch.randn(20, 64, device="cuda", requires_grad=True), torch.randn(30, 64, device="cuda", requires_grad=True), torch.arange(20, device="cuda")
    for name, call in (("castle_layer_norm", lambda: castle_layer_norm(x, w[0]).sum()), ("castle_linear_cross_entropy", lambda: castle_linear_cross_entropy(x, w, t)),
                       ("castle_embedding", lambda: castle_embedding(t, w).sum())):
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, lambda s: s[:-1] if s.dim() else s):
            out = call()
        with pytest.raises(RuntimeError, match=name + ": a saved tensor came back"):
            out.backward()


def test_a_traced_forward():
    w = torch.randn(40, 64, device="cuda", requires_grad=True)
    def f(tokens, table):
        h = castle_layer_norm(castle_embedding(tokens, table, 3.0), table[0], table[1])
        return castle_linear_cross_entropy(h, table, tokens)
    t = torch.arange(30, device="cuda")
    traced = torch.jit.trace(f, (t, w), check_trace=False)
    other = (t + 7) % 40
    want, got = f(other, w), traced(other, w)
    assert torch.equal(want, got)
    assert torch.equal(torch.autograd.grad(want, [w])[0], torch.autograd.grad(got, [w])[0])


def test_batched_gradients_and_functional_transforms_are_refused():
    x = torch.randn(6, 16, device="cuda", requires_grad=True)
    y = castle_layer_norm(x)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, [x], torch.ones(3, 6, 16, device="cuda"), is_grads_batched=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: castle_layer_norm(v))(x.detach())


def test_lazily_negated_tensors_are_taken_with_their_sign():
    z = torch.randn(20, 64, dtype=torch.complex64, device="cuda")
    neg = z.conj().imag[..., :64]
    assert neg.is_neg()
    w, t = torch.randn(30, 64, device="cuda"), torch.arange(20, device="cuda")
    plain = neg.resolve_neg().contiguous()
    assert torch.equal(castle_layer_norm(neg), castle_layer_norm(plain))
    assert torch.equal(castle_linear_cross_entropy(neg, w, t), castle_linear_cross_entropy(plain, w, t))
    assert torch.equal(castle_embedding(t, neg), castle_embedding(t, plain))
    x = plain.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(castle_layer_norm(x), [x], neg)[0], torch.autograd.grad(castle_layer_norm(x), [x], plain)[0])


def test_under_autocast_and_inference_mode():
    x, w, t = torch.randn(20, 64, device="cuda"), torch.randn(30, 64, device="cuda"), torch.arange(20, device="cuda")
    want = castle_layer_norm(x), castle_linear_cross_entropy(x, w, t), castle_embedding(t, w)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = castle_layer_norm(x), castle_linear_cross_entropy(x, w, t), castle_embedding(t, w)
    with torch.inference_mode():
        also = castle_layer_norm(x), castle_linear_cross_entropy(x, w, t), castle_embedding(t, w)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, also))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_a_layers_rows_beside_parameters_of_32_bits_under_autocast(dtype):
    """Parameters are cast to the rows' type: bit for bit what a caller's own casts give, with gradients in the parameters' type.  Outside of autocast
    mixed types stay refused."""
    torch.manual_seed(0)
    layer, norm, table = Castle(64, heads=2, dim_head=32).cuda(), torch.nn.LayerNorm(64).cuda(), torch.randn(300, 64, device="cuda", requires_grad=True)
    torch.nn.init.normal_(norm.weight)
    x, t = torch.randn(2, 50, 64, device="cuda"), torch.randint(0, 300, (2, 50), device="cuda")
    leaves = [norm.weight, norm.bias, table]
    def loss(cast):
        h = castle_layer_norm(layer(x), cast(norm.weight), cast(norm.bias), norm.eps)
        assert h.dtype == dtype
        return castle_linear_cross_entropy(h, cast(table), t)
    with torch.autocast("cuda", dtype=dtype):
        got, want = loss(lambda p: p), loss(lambda p: p.to(dtype))
    assert torch.equal(got, want)
    for a, b, p in zip(torch.autograd.grad(got * 64, leaves), torch.autograd.grad(want * 64, leaves), leaves):
        assert a.dtype == p.dtype == torch.float32 and torch.equal(a, b) and bool(a.any())
    with torch.autocast("cuda", dtype=dtype):
        assert castle_layer_norm(x, norm.weight.to(dtype)).dtype == torch.float32      # rows of 32 bits stay so
        with pytest.raises(RuntimeError, match="castle_layer_norm"):
            castle_layer_norm(x, norm.weight.double())
    h = x.to(dtype)
    for call in (lambda: castle_layer_norm(h, norm.weight), lambda: castle_layer_norm(h, None, norm.bias), lambda: castle_linear_cross_entropy(h, table, t)):
        with pytest.raises(RuntimeError, match="type"):
            call()
    check_status()


def test_offsets_beyond_32_bits():
    """Elements behind the 2^31st of the table, of the rows and of the weight, against the same values in small tensors."""
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs some 40 GB")
    gen = torch.Generator("cuda").manual_seed(0)
    vocab, dim = 1_100_000, 2048                       # 2.25e9 elements
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(1000, dim, device="cuda", generator=gen).bfloat16()
    table[-1000:] = last
    t = torch.randint(0, 1000, (300,), device="cuda", generator=gen)
    g = torch.randn(300, dim, device="cuda", generator=gen).bfloat16()
    leaf, small = table.requires_grad_(), last.clone().requires_grad_()
    a, b = castle_embedding(t + vocab - 1000, leaf, 2.0), castle_embedding(t, small, 2.0)
    assert torch.equal(a, b)
    (da,), (db,) = torch.autograd.grad(a, [leaf], g), torch.autograd.grad(b, [small], g)
    assert torch.equal(da[-1000:], db) and not bool(da[:-1000].any())
    del da, db
    # the loss of a few rows against that table: all other logits are zero
    x = torch.randn(40, dim, device="cuda", generator=gen).bfloat16().requires_grad_()
    loss = castle_linear_cross_entropy(x, leaf, t[:40] + vocab - 1000, reduction="none")
    z = x.double() @ last.double().t()
    want = torch.log(z.exp().sum(1) + (vocab - 1000)) - z[torch.arange(40), t[:40]]
    assert bool(((loss.double() - want).abs() <= 1e-3).all())          # logits of 2048 products, off by 130 * 2^-22 of some 1600
    dx, dw = torch.autograd.grad(loss, [x, leaf], torch.ones(40, device="cuda"))
    p = z.exp() / (z.exp().sum(1, keepdim=True) + (vocab - 1000))
    p[torch.arange(40), t[:40]] -= 1
    assert ((dx.double() - p @ last.double()).norm() <= 2.0 ** -8 * (p @ last.double()).norm()).item()
    assert ((dw[-1000:].double() - p.t() @ x.double()).norm() <= 2.0 ** -8 * (p.t() @ x.double()).norm()).item()
    del table, leaf, dw, a, loss
    release_workspaces()
    rows, dim = 280_000, 8192                          # 2.29e9 elements
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(100, dim, device="cuda", generator=gen).bfloat16()
    x[-100:] = last
    y = castle_layer_norm(x)
    assert torch.equal(y[-100:], castle_layer_norm(last)) and not bool(y[:-100].any())
    del y
    w = torch.randn(70, dim, device="cuda", generator=gen).bfloat16()
    t = torch.full((rows,), -100, device="cuda")
    t[-100:] = torch.arange(100, device="cuda") % 70
    leaf = x.requires_grad_()
    loss = castle_linear_cross_entropy(leaf, w, t)
    assert torch.equal(loss, castle_linear_cross_entropy(last, w, t[-100:]))
    (dx,) = torch.autograd.grad(loss, [leaf])
    small = last.clone().requires_grad_()
    want = torch.autograd.grad(castle_linear_cross_entropy(small, w, t[-100:]), [small])[0]
    assert ((dx[-100:].double() - want.double()).norm() <= 2.0 ** -8 * want.double().norm()).item() and not bool(dx[:-100].any())
    check_status()
    release_workspaces()


def test_rows_longer_than_32_bits_are_refused():
    dim = 2 ** 32 + 8          # (8 in 32 bits; nothing of this size is laid out)
    x = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(4, dim)
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for call in (lambda: castle_embedding(t, x), lambda: castle_layer_norm(x), lambda: castle_linear_cross_entropy(x, x, t)):
        with pytest.raises(RuntimeError, match="4294967304 elements are not supported"):
            call()


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x, w, t = torch.randn(20, 64, device="cuda:1", requires_grad=True), torch.randn(30, 64, device="cuda:1", requires_grad=True), torch.arange(20, device="cuda:1")
    loss = castle_linear_cross_entropy(castle_layer_norm(castle_embedding(t, w) + x), w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert loss.device == dx.device == dw.device == x.device and bool(dx.isfinite().all())
    check_status()
