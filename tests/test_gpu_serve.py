"""GPU: paged caches and weights of 4 bits under the module, as a server uses them, beside the contiguous caches and the weights at full width."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


def _layers(count, dtype, dim=256, heads=4, dim_head=64, **kw):
    from lookahead_keys_attention_b200 import Castle
    torch.manual_seed(0)
    return nn.ModuleList([Castle(dim, heads=heads, dim_head=dim_head, **kw) for _ in range(count)]).cuda().to(dtype)


def _prompt(layers, x):
    caches = []
    for m in layers:
        o, c = m(x, return_next_cache=True)
        x = x + o
        caches.append(c)
    return x, caches


def _token(layers, x, caches):
    for i, m in enumerate(layers):
        o, caches[i] = m(x, cache=caches[i])
        x = x + o
    return x


def _paged_token(layers, x, batch):
    for i, m in enumerate(layers):
        o, c = m(x, cache=batch.layer(i))
        assert c.batch is batch
        x = x + o
    return x


# Both steps do the same arithmetic on the same caches in fp32; they add in other orders.  fp32: some hundred roundings of sums of size 1 to 10 through three
# layers and 40 tokens.  bf16: what a rounding that falls the other way changes, at most a few steps of 2^-8 of values up to 4 through the layers
CLOSE = {torch.float32: 2e-4, torch.bfloat16: 8e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, dict(prenorm=True, rotary_emb=True), dict(prenorm="layer"), dict(dim_head=32, heads=3, prenorm=True)], ids=str)
@torch.no_grad()
def test_sequences_of_different_lengths(dtype, kw):
    """Each sequence's tokens beside the same sequence alone over contiguous caches."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(3, dtype, **kw)
    cache = PagedCache(3, 64, layers[0].heads, layers[0].dim_head, 16, dtype=dtype)
    lengths, seqs, alone = [40, 2, 33, 15], [], []
    for n in lengths:
        _, c = _prompt(layers, torch.randn(1, n, 256, device="cuda").to(dtype))
        seqs.append(cache.add())
        for i in range(3):
            cache.write([seqs[-1]], i, c[i])
        alone.append(c)
    batch = cache.batch(seqs)
    for t in range(40):
        x = torch.randn(4, 1, 256, device="cuda").to(dtype)
        got = _paged_token(layers, x, batch)
        batch.advance()
        for b in range(4):
            want = _token(layers, x[b:b + 1], alone[b])
            assert (got[b] - want[0]).abs().max().item() <= CLOSE[dtype] * want.abs().max().item(), (t, b)
    check_status()
    assert [cache.length(q) for q in seqs] == [n + 40 for n in lengths] == batch.lengths.tolist()


@torch.no_grad()
def test_from_no_positions_at_all_and_large_batches():
    """Sequences that begin with their first token; batches that the token's own projections are too small for."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.bfloat16, prenorm=True)
    cache = PagedCache(2, 100, 4, 64, 16)
    batch = cache.batch([cache.add() for _ in range(40)])
    contiguous = [None, None]
    for t in range(20):
        x = torch.randn(40, 1, 256, device="cuda").bfloat16()
        got = _paged_token(layers, x, batch)
        want = _token(layers, x, contiguous)
        batch.advance()
        assert (got - want).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max()
    check_status()


@torch.no_grad()
def test_forks_go_their_own_ways():
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.float32, prenorm=True, rotary_emb=True)
    cache = PagedCache(2, 40, 4, 64, 16, dtype=torch.float32)
    x0 = torch.randn(1, 41, 256, device="cuda")
    first = cache.add()
    for i, c in enumerate(_prompt(layers, x0)[1]):
        cache.write([first], i, c)
    seqs = [first, *cache.fork(first, 2)]
    batch = cache.batch(seqs)
    same = torch.randn(1, 1, 256, device="cuda").expand(3, 1, 256)
    got = _paged_token(layers, same, batch)
    batch.advance()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    seqs.append(cache.fork(seqs[1])[0])
    batch.replace(seqs)
    tokens = [[same[:1]] for _ in range(3)]
    tokens.append(list(tokens[1]))
    for t in range(25):
        x = torch.randn(4, 1, 256, device="cuda")
        got = _paged_token(layers, x, batch)
        batch.advance()
        for b in range(4):
            tokens[b].append(x[b:b + 1])
    cache.compact()
    got = _paged_token(layers, x, batch)
    for b in range(4):                                        # each alone, from the prompt on
        caches = _prompt(layers, x0)[1]
        for v in tokens[b]:
            _token(layers, v, caches)
        want = _token(layers, x[b:b + 1], caches)
        assert (got[b] - want[0]).abs().max() <= CLOSE[torch.float32] * want.abs().max()
    check_status()


@torch.no_grad()
def test_a_freed_sequence_and_its_pages():
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(1, torch.bfloat16)
    cache = PagedCache(1, 8, 4, 64, 16)
    x = torch.randn(2, 30, 256, device="cuda").bfloat16()
    a, b = cache.add(), cache.add()
    cache.write([a, b], 0, _prompt(layers, x)[1][0])
    batch = cache.batch([a, b])
    cache.free(a)
    token = torch.randn(2, 1, 256, device="cuda").bfloat16()
    out, _ = layers[0](token, cache=batch.layer(0))
    assert not out[0].any() and bool(out[1].any()) and batch.seqs == [None, b]
    c = cache.add()                                           # takes a's pages
    cache.write([c], 0, _prompt(layers, x[1:])[1][0])
    batch.replace([c, b])
    out, _ = layers[0](token[1:].expand(2, 1, 256).contiguous(), cache=batch.layer(0))
    check_status()
    # (b has taken the other token in its place: its position was not counted, but its lookahead keys were moved)
    alone = _prompt(layers, x[1:])[1]
    want, _ = layers[0](token[1:], cache=alone[0])
    assert (out[0] - want[0]).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max()


@torch.no_grad()
def test_a_captured_token_serves_whoever_is_there():
    """One graph of a token through all layers, replayed as sequences grow, come and go, and pages move."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.bfloat16, prenorm=True, rotary_emb=True)
    cache = PagedCache(2, 60, 4, 64, 16)

    def new(n):
        x = torch.randn(1, n, 256, device="cuda").bfloat16()
        q, c = cache.add(), _prompt(layers, x)[1]
        for i in range(2):
            cache.write([q], i, c[i])
        return q, c

    (a, ca), (b, cb) = new(20), new(5)
    batch = cache.batch([a, b], size=4, width=8)
    x = torch.randn(4, 1, 256, device="cuda").bfloat16()
    spare = cache.fork(a)[0]
    warm = cache.batch([spare], size=4, width=8)
    _paged_token(layers, x, warm)
    del warm
    cache.free(spare)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = _paged_token(layers, x, batch)
    pointers = batch.table.data_ptr(), batch.lengths.data_ptr()
    who = [(0, ca), (1, cb)]
    for t in range(60):
        if t == 20:
            c, cc = new(33)
            batch.replace([b, None, c])
            cache.free(a)
            who = [(0, cb), (2, cc)]
        if t == 30:
            cache.compact()
        x.copy_(torch.randn(4, 1, 256, device="cuda"))
        graph.replay()
        batch.advance()
        for row, caches in who:
            want = _token(layers, x[row:row + 1], caches)
            assert (out[row] - want[0]).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max(), (t, row)
    assert pointers == (batch.table.data_ptr(), batch.lengths.data_ptr())
    check_status()


def test_what_the_module_refuses():
    from lookahead_keys_attention_b200 import PagedCache
    m = _layers(1, torch.bfloat16)[0]
    cache = PagedCache(1, 8, 4, 64, 16)
    batch = cache.batch([cache.add()])
    x = torch.randn(1, 2, 256, device="cuda").bfloat16()
    for bad in (x, x[:, :1].expand(2, 1, 256)):
        with pytest.raises(ValueError, match="one token"):
            m(bad, cache=batch.layer(0))
    with pytest.raises(RuntimeError, match="rows' type"):
        other = PagedCache(1, 8, 4, 64, 16, dtype=torch.float32)
        m(x[:, :1], cache=other.batch([other.add()]).layer(0))
    with pytest.raises(RuntimeError, match="heads"):
        other = PagedCache(1, 8, 2, 64, 16)
        m(x[:, :1], cache=other.batch([other.add()]).layer(0))


def test_no_gradient_flows_through_the_cached_step_but_the_last_projection_has_one():
    from lookahead_keys_attention_b200 import PagedCache
    m = _layers(1, torch.float32)[0]
    cache = PagedCache(1, 8, 4, 64, 16, dtype=torch.float32)
    batch = cache.batch([cache.add()])
    out, _ = m(torch.randn(1, 1, 256, device="cuda", requires_grad=True), cache=batch.layer(0))
    out.sum().backward()
    assert m.combine_heads.weight.grad is not None and m.to_all_qkv.weight.grad is None


class Model(nn.Module):
    """A byte model with 4-bit weights everywhere but in its table."""

    def __init__(self, layers, dim=256, heads=4):
        super().__init__()
        from lookahead_keys_attention_b200 import Castle
        self.table = nn.Parameter(torch.randn(256, dim) * dim ** -0.5)
        self.attn = nn.ModuleList([Castle(dim, heads=heads, prenorm=True, rotary_emb=True) for _ in range(layers)])
        self.ff = nn.ModuleList([nn.Sequential(nn.RMSNorm(dim), nn.Linear(dim, 4 * dim), nn.GELU(), nn.Linear(4 * dim, dim)) for _ in range(layers)])
        self.norm, self.head = nn.RMSNorm(dim), nn.Linear(dim, 256, bias=False)

    def forward(self, ids, caches=None, keep=False):
        from lookahead_keys_attention_b200 import castle_embedding
        h, new = castle_embedding(ids, self.table, scale=16.0), []
        for i, (a, f) in enumerate(zip(self.attn, self.ff)):
            o = a(h, cache=None if caches is None else caches[i], return_next_cache=keep or None)
            if isinstance(o, tuple):
                o, c = o
                new.append(c)
            h = h + o
            h = h + f(h)
        return self.head(self.norm(h)), new


@torch.no_grad()
def test_a_small_server():
    """Quantised weights, prompts of different lengths, forks, a batch that changes: every token's logits beside the same model over contiguous caches, one
    sequence at a time, from the same 4-bit weights."""
    from lookahead_keys_attention_b200 import Linear4bit, PagedCache, check_status
    torch.manual_seed(1)
    model = Model(2).cuda().bfloat16()
    full = model(torch.randint(0, 256, (1, 50), device="cuda"))[0]
    for a, f in zip(model.attn, model.ff):
        a.quantize_4bit(group_size=32, zeros=True)
        f[1], f[3] = Linear4bit.from_linear(f[1], 32), Linear4bit.from_linear(f[3], 32)
    model.head = Linear4bit.from_linear(model.head, 32)
    assert type(model.attn[0].to_all_qkv) is Linear4bit and full.shape == (1, 50, 256)
    cache = PagedCache(2, 60, 4, 64, 16)
    prompts = [torch.randint(0, 256, (1, n), device="cuda") for n in (30, 7, 16)]
    texts, seqs = [], []
    for p in prompts:
        logits, caches = model(p, keep=True)
        seqs.append(cache.add())
        for i, c in enumerate(caches):
            cache.write(seqs[-1:], i, c)
        texts.append(torch.cat((p, logits[:, -1:].argmax(-1)), 1))
    seqs += cache.fork(seqs[0], 2)
    texts += [texts[0].clone(), texts[0].clone()]
    texts[3][0, -1], texts[4][0, -1] = 5, 200
    batch = cache.batch(seqs)
    logits = []
    for t in range(20):
        ids = torch.cat([t[:, -1:] for t in texts])
        out, _ = model(ids, [batch.layer(i) for i in range(2)])
        batch.advance()
        logits.append(out)
        texts = [torch.cat((t, out[b, -1:].argmax(-1)[None]), 1) for b, t in enumerate(texts)]
    check_status()
    logits = torch.cat(logits, 1)
    for b, n in enumerate((30, 7, 16, 30, 30)):
        _, caches = model(texts[b][:, :n], keep=True)
        for t in range(20):
            want, caches = model(texts[b][:, n + t:n + t + 1], caches)
            assert (logits[b, t] - want[0, 0]).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max(), (b, t)


def test_a_quantised_layer_trains_what_is_in_front_of_it():
    """The gradient of the input of a layer with 4-bit projections, beside that of the same layer with the weights that the codes stand for."""
    from lookahead_keys_attention_b200 import Castle, castle_linear_4bit
    torch.manual_seed(2)
    m = Castle(256, heads=4, prenorm=True).cuda()
    q = Castle(256, heads=4, prenorm=True).cuda()
    q.load_state_dict(m.state_dict())
    q.quantize_4bit(32)
    for name in ("to_all_qkv", "combine_heads"):
        lin = getattr(q, name)
        getattr(m, name).weight.data = castle_linear_4bit(torch.eye(lin.in_features, device="cuda"), lin.codes, lin.scales, None, 32).t().contiguous()
    x = torch.randn(2, 100, 256, device="cuda")
    g = torch.randn(2, 100, 256, device="cuda")
    outs = []
    for layer in (m, q):
        v = x.clone().requires_grad_()
        y = layer(v)
        outs.append((y.detach(), torch.autograd.grad(y, [v, layer.norm.weight], g)))
    (y0, g0), (y1, g1) = outs
    # (the core's operands are fp16 in either; the projections differ by fp32 roundings)
    assert (y0 - y1).norm() <= 2e-3 * y0.norm() and all((a - b).norm() <= 4e-3 * a.norm() for a, b in zip(g0, g1))
    assert not any(p.requires_grad for p in q.to_all_qkv.parameters())


def test_threads_on_one_stream():
    """Steps and products of several host threads: what a call's launches share is the stream's, so they must not mix."""
    import threading
    from lookahead_keys_attention_b200 import PagedCache, check_status

    def server(seed, dtype, heads, quantised):
        layers = _layers(2, dtype, heads=heads, prenorm=True)
        if quantised:
            for m in layers:
                m.quantize_4bit(32, zeros=True)
        gen = torch.Generator("cuda").manual_seed(seed)
        xs = torch.randn(60, 3, 1, 256, device="cuda", generator=gen).to(dtype)

        @torch.no_grad()
        def go():
            cache = PagedCache(2, 60, heads, 64, 16, dtype=dtype)
            prompt = torch.ones(3, 37, 256, device="cuda", dtype=dtype)
            seqs = [cache.add() for _ in range(3)]
            for i, c in enumerate(_prompt(layers, prompt)[1]):
                cache.write(seqs, i, c)
            batch, outs = cache.batch(seqs), []
            for x in xs:
                outs.append(_paged_token(layers, x, batch))
                batch.advance()
            return torch.cat(outs, 1)

        return go

    work = [server(1, torch.bfloat16, 4, True), server(2, torch.float32, 8, False), server(3, torch.float16, 2, True), server(4, torch.bfloat16, 6, False)]
    want = [w() for w in work]
    torch.cuda.synchronize()
    got, errors = [None] * len(work), []

    def run(i):
        try:
            got[i] = work[i]()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    check_status()
    assert not errors, errors
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_traced_calls():
    from lookahead_keys_attention_b200 import Castle, Linear4bit, PagedCache, castle_copy_pages
    m = Linear4bit.from_linear(nn.Linear(64, 32).cuda(), 32)
    x = torch.randn(3, 64, device="cuda")
    traced = torch.jit.trace(m, (x,), check_trace=False)
    y = torch.randn(3, 64, device="cuda")
    assert torch.equal(traced(y), m(y))
    cache = PagedCache(1, 4, 2, 64, 16, dtype=torch.float32)
    batch = cache.batch([cache.add()])
    layer = Castle(64, heads=2).cuda()
    with pytest.raises(RuntimeError, match="traced"), torch.no_grad():
        torch.jit.trace(lambda v: layer(v, cache=batch.layer(0))[0], (torch.randn(1, 1, 64, device="cuda"),), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda v: castle_copy_pages(v, [0], [1]) or v, (torch.randn(4, 2, 16, 64, device="cuda"),), check_trace=False)


@torch.no_grad()
def test_under_a_default_device():
    """A server that makes everything on the GPU by default: the same tokens."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.bfloat16, prenorm=True)
    prompt, tokens = torch.randn(2, 30, 256, device="cuda").bfloat16(), torch.randn(5, 3, 1, 256, device="cuda").bfloat16()

    def serve():
        cache = PagedCache(2, 40, 4, 64, 16)
        a, b = cache.add(), cache.add()
        for i, c in enumerate(_prompt(layers, prompt)[1]):
            cache.write([a, b], i, c)
        c = cache.fork(b)[0]
        batch, outs = cache.batch([a, b, c]), []
        for x in tokens:
            outs.append(_paged_token(layers, x, batch))
            batch.advance()
        cache.free(a)
        cache.compact()
        cache.resize(30)
        outs.append(_paged_token(layers, tokens[0], batch))
        return torch.cat(outs, 1)

    want = serve()
    with torch.device("cuda"):
        got = serve()
    check_status()
    assert torch.equal(got, want)


@pytest.mark.parametrize("other", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_quantised_linear_under_autocast(dtype, other):
    """The types that a linear layer takes and gives; bit for bit the operator's result for rows and parameters in autocast's type."""
    from lookahead_keys_attention_b200 import Linear4bit, castle_linear_4bit
    torch.manual_seed(3)
    full = nn.Linear(192, 96).cuda().to(dtype)
    m = Linear4bit.from_linear(full, 64, zeros=True)
    for rows in ((3,), (2, 150)):
        for x_type in (torch.float32, torch.bfloat16, torch.float16):
            x, g = torch.randn(*rows, 192, device="cuda").to(x_type), torch.randn(*rows, 96, device="cuda").to(other)
            outs = []
            for layer in (full, m):
                v = x.clone().requires_grad_()
                with torch.autocast("cuda", dtype=other):
                    y = layer(v)
                outs.append((y, torch.autograd.grad(y, [v], g)[0]))
            (y0, dx0), (y1, dx1) = outs
            assert y1.dtype == y0.dtype == other and dx1.dtype == dx0.dtype == x_type and y1.shape == y0.shape
            want = castle_linear_4bit(x.to(other), m.codes, m.scales.to(other), m.zeros.to(other), 64) + m.bias.to(other)
            assert torch.equal(y1, want)


@torch.no_grad()
def test_a_quantised_model_under_autocast():
    """fp32 parameters, autocast's rows: caches of autocast's type, into pages and on from there, beside the same layers over contiguous caches."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.float32, prenorm=True)
    for m in layers:
        m.quantize_4bit(32)
    cache = PagedCache(2, 20, 4, 64, 16)
    a = cache.add()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        _, caches = _prompt(layers, torch.randn(1, 21, 256, device="cuda"))
        for i, c in enumerate(caches):
            assert all(t.dtype == torch.bfloat16 for t in c)
            cache.write([a], i, c)
        batch = cache.batch([a])
        for t in range(12):
            x = torch.randn(1, 1, 256, device="cuda")
            got, want = _paged_token(layers, x, batch), _token(layers, x, caches)
            batch.advance()
            assert got.dtype == want.dtype and (got - want).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max()
    check_status()


@torch.no_grad()
def test_sequences_leave_a_full_cache():
    """A captured token: the row of a sequence that no page is free for takes no part, the other goes on, and the first comes back with all its positions."""
    from lookahead_keys_attention_b200 import PagedCache, check_status
    layers = _layers(2, torch.bfloat16, prenorm=True)
    cache = PagedCache(2, 3, 4, 64, 16)
    a, b = cache.add(), cache.add()
    batch, alone, x = cache.batch([a, b], width=2), [[None] * 2, [None] * 2], torch.zeros(2, 1, 256, device="cuda").bfloat16()
    _paged_token(layers, x, batch)                                       # (not counted: nothing of it stays)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = _paged_token(layers, x, batch)

    def token(rows):
        x.copy_(torch.randn(2, 1, 256, device="cuda"))
        graph.replay()
        for row, who in enumerate(rows):
            if who is None:
                assert torch.equal(out[row], x[row])                     # (the layers' outputs are zero)
            else:
                want = _token(layers, x[row:row + 1], alone[who])
                assert (out[row] - want[0]).abs().max() <= CLOSE[torch.bfloat16] * want.abs().max()

    for t in range(16):
        token([0, 1])
        assert batch.advance(leave=True) == ([b] if t == 15 else [])
    for _ in range(4):
        token([0, None])
        assert batch.advance(leave=True) == []
    cache.free(a)
    batch.replace([None, b])
    for _ in range(9):
        token([None, 1])
        assert batch.advance(leave=True) == []
    check_status()
    assert cache.length(b) == 25
