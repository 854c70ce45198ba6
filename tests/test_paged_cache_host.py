"""CPU: the books of `PagedCache`, with the device's copies replaced by plain indexing: whatever is added, forked, freed, moved and continued, every
sequence reads its own rows, and no page that is written belongs to two."""
import random

import pytest
import torch

from lookahead_keys_attention_b200 import ops, serve


@pytest.fixture
def plain(monkeypatch):
    def copy_pages(pools, source, target):
        source, target = list(source), list(target)
        assert not set(source) & set(target) and len(set(target)) == len(target)
        for p in pools if isinstance(pools, list) else [pools]:
            p[target] = p[source].clone()

    def write_pages(U, qu, kc, vc, Up, qup, kcp, vcp, u_table, table, lengths):
        for b, n in enumerate(lengths.tolist()):
            for cache, pool, t in ((U, Up, u_table), (qu, qup, table), (kc, kcp, table), (vc, vcp, table)):
                for k in range(n):
                    pool[t[b, k // pool.shape[2]].long(), :, k % pool.shape[2]] = cache[b, :, k]

    monkeypatch.setattr(ops, "castle_copy_pages", copy_pages)
    monkeypatch.setattr(ops, "castle_write_pages", write_pages)


def _cache(**kw):
    return serve.PagedCache(**{**dict(layers=2, pages=40, heads=1, dim_head=16, page_size=16, dtype=torch.float64, device="cpu"), **kw})


def _step(batch, value):
    """What a token does to the pools, by the batch's tables: U of every row changes, a row is appended."""
    cache = batch.cache
    for layer in range(cache.layers):
        U, qu, kc, vc = batch.layer(layer).pools
        for b, n in enumerate(batch.lengths.tolist()):
            for k in range(max(n, 0)):
                U[batch.u_table[b, k // 16].long(), :, k % 16] += value[b]
            if n >= 0:
                U[batch.u_table[b, n // 16].long(), :, n % 16] = 0
                for i, p in enumerate((qu, kc, vc)):
                    p[batch.table[b, n // 16].long(), :, n % 16] = 10 * value[b] + i + 100 * layer


def _check(cache, model):
    """`model`: {sequence: (U's values, the appended rows')}"""
    held = {}
    for q, (u, rows) in model.items():
        s = cache._of(q)
        assert s.length == len(u) == cache.length(q)
        for k in range(s.length):
            for layer in range(cache.layers):
                U, qu, kc, vc = cache._pools(layer)
                assert bool((U[s.u_pages[k // 16], :, k % 16] == u[k]).all())
                for i, p in enumerate((qu, kc, vc)):
                    assert bool((p[s.pages[k // 16], :, k % 16] == 10 * rows[k] + i + 100 * layer).all())
        for p in s.u_pages:
            held[("u", p)] = held.get(("u", p), 0) + 1
        for n, p in enumerate(s.pages):
            held[("kv", p)] = held.get(("kv", p), 0) + 1
            assert cache._kv.held[p] == 1 or (n + 1) * 16 <= s.length      # what is shared is full
    assert all(v == 1 for (kind, _), v in held.items() if kind == "u")
    for pool, kind in ((cache._kv, "kv"), (cache._u, "u")):
        assert [held.get((kind, p), 0) for p in range(len(pool.held))] == pool.held
        assert sorted(pool.free) == [p for p, h in enumerate(pool.held) if h == 0]


@pytest.mark.parametrize("seed", range(6))
def test_whatever_happens(plain, seed):
    rng = random.Random(seed)
    cache, model, batch = _cache(), {}, None
    for _ in range(70):
        what = rng.choice(["prompt", "fork", "free", "step", "step", "step", "step", "compact", "resize", "replace"])
        if what == "prompt":
            n, count = rng.choice([0, 1, 15, 16, 17, 40]), rng.randint(1, 2)
            if count * (n // 16 + 1) > min(cache.free_pages()):
                continue
            seqs = [cache.add() for _ in range(count)]
            u = torch.randint(0, 9, (count, n)).double()
            rows = torch.randint(0, 9, (count, n)).double()
            for layer in range(2):
                wide = lambda v: v[:, None, :, None].expand(count, 1, n, 16)  # noqa: E731
                cache.write(seqs, layer, (wide(u), *(wide(10 * rows + i + 100 * layer) for i in range(3))))
            for i, q in enumerate(seqs):
                model[q] = (u[i].tolist(), rows[i].tolist())
        elif what == "fork" and model:
            q = rng.choice(list(model))
            try:
                new = cache.fork(q, rng.randint(1, 2))
            except RuntimeError:
                continue
            for f in new:
                model[f] = (list(model[q][0]), list(model[q][1]))
        elif what == "free" and model:
            q = rng.choice(list(model))
            cache.free(q)
            del model[q]
        elif what == "replace" and model:
            seqs = rng.sample(list(model), rng.randint(1, len(model)))
            seqs.insert(rng.randint(0, len(seqs)), None)
            try:
                if batch is None:
                    batch = cache.batch(seqs, size=4)
                else:
                    batch.replace(seqs)
            except RuntimeError:
                pass
        elif what == "step" and batch is not None:
            value = [rng.randint(1, 9) for _ in batch.seqs]
            assert [-1 if q is None else len(model[q][0]) for q in batch.seqs] == batch.lengths.tolist()
            _step(batch, value)
            try:
                batch.advance()
            except RuntimeError:
                for b, q in enumerate(batch.seqs):      # not counted: as if it had not been, but for U
                    if q is not None:
                        model[q] = ([v + value[b] for v in model[q][0]], model[q][1])
                victim = next((q for q in batch.seqs if q is not None), None)
                cache.free(victim)
                del model[victim]
                _check(cache, model)
                continue
            for b, q in enumerate(batch.seqs):
                if q is not None:
                    u, rows = model[q]
                    model[q] = ([v + value[b] for v in u] + [0], rows + [value[b]])
        elif what == "compact":
            used = cache.compact()
            assert all(h == 0 for h in cache._kv.held[used[0]:]) and all(h == 0 for h in cache._u.held[used[1]:])
        elif what == "resize":
            used = cache.compact()
            cache.resize(max(30, used[0]), max(30, used[1]))
        _check(cache, model)


def test_nothing_is_taken_where_not_all_is_there(plain):
    cache = _cache(pages=4)
    a = cache.add()
    z = torch.zeros(1, 1, 40, 16, dtype=torch.float64)
    cache.write([a], 0, (z, z, z, z))
    assert cache.free_pages() == (1, 1)
    with pytest.raises(RuntimeError, match="more pages needed"):
        cache.fork(a)
    b = cache.add()
    with pytest.raises(RuntimeError, match="more pages needed"):
        cache.write([b], 0, (z, z, z, z))
    assert cache.free_pages() == (1, 1) and cache.length(b) == 0
    batch = cache.batch([a])
    for _ in range(23):
        batch.advance()
    c = batch.lengths.tolist()
    with pytest.raises(RuntimeError, match="more pages needed"):
        batch.advance()
    assert batch.lengths.tolist() == c == [63] and cache.length(a) == 63


def test_a_forked_prompt_shares_its_full_pages(plain):
    cache = _cache()
    a = cache.add()
    z = torch.zeros(1, 1, 40, 16, dtype=torch.float64)
    cache.write([a], 0, (z, z, z, z))
    cache.fork(a, 3)
    assert cache.free_pages() == (40 - 2 - 4, 40 - 4 * 3)


def test_pages_that_forks_share_take_no_prompt(plain):
    cache = _cache()
    a = cache.add()
    z = torch.zeros(1, 1, 40, 16, dtype=torch.float64)
    cache.write([a], 0, (z, z, z, z))
    (b,) = cache.fork(a)
    for q in (a, b):
        with pytest.raises(ValueError, match="shares"):
            cache.write([q], 1, (z, z, z, z))
    cache.free(b)
    cache.write([a], 1, (z, z, z, z))


def test_a_prompt_that_was_not_written_is_not_counted(plain, monkeypatch):
    cache = _cache()
    a = cache.add()
    z = torch.zeros(1, 1, 40, 16, dtype=torch.float64)
    with monkeypatch.context() as m:
        def refuse(*_):
            raise RuntimeError("refused")
        m.setattr(ops, "castle_write_pages", refuse)
        with pytest.raises(RuntimeError, match="refused"):
            cache.write([a], 0, (z, z, z, z))
    assert cache.length(a) == 0
    cache.write([a], 0, (z[:, :, :20], z[:, :, :20], z[:, :, :20], z[:, :, :20]))
    assert cache.length(a) == 20
    cache.free(a)
    assert cache.free_pages() == (40, 40)


def test_a_fork_that_was_not_copied_keeps_no_pages(plain, monkeypatch):
    cache = _cache()
    a = cache.add()
    z = torch.zeros(1, 1, 40, 16, dtype=torch.float64)
    cache.write([a], 0, (z, z, z, z))
    before = cache.free_pages(), list(cache._kv.held), list(cache._u.held), list(cache._sequences)
    with monkeypatch.context() as m:
        def refuse(*_):
            raise RuntimeError("refused")
        m.setattr(ops, "castle_copy_pages", refuse)
        with pytest.raises(RuntimeError, match="refused"):
            cache.fork(a, 3)
    assert before == (cache.free_pages(), cache._kv.held, cache._u.held, list(cache._sequences))
    assert len(cache.fork(a, 3)) == 3


def test_made_in_inference_mode_and_used_outside(plain):
    with torch.inference_mode():
        cache = _cache()
        a = cache.add()
        z = torch.ones(1, 1, 15, 16, dtype=torch.float64)
        cache.write([a], 0, (z, z, z, z))
        batch = cache.batch([a])
    for _ in range(3):                                                  # over the end of a page
        batch.advance()
    assert batch.lengths.tolist() == [18]
    b = cache.fork(a)[0]
    batch.replace([b])
    with torch.inference_mode():
        batch.advance()
    assert batch.lengths.tolist() == [19] and cache.length(b) == 19 and cache.length(a) == 18
    cache.free(a)
    cache.compact()
    cache.resize(10)


def test_a_token_that_fills_the_last_page_is_counted(plain):
    """With `leave`: one page of 16 holds 16 positions, and only the sequence that has no place for its next token leaves the batch."""
    cache = _cache(pages=1)
    a = cache.add()
    batch = cache.batch([a])
    for t in range(16):
        _step(batch, [t + 1])
        assert batch.advance(leave=True) == ([a] if t == 15 else [])
    # a token's value is added to U of every row before it
    model = {a: ([sum(range(t + 2, 17)) for t in range(16)], list(range(1, 17)))}
    _check(cache, model)
    assert cache.length(a) == 16 and batch.seqs == [None] and batch.lengths.tolist() == [-1] and batch.advance(leave=True) == []
    with pytest.raises(RuntimeError, match="more pages needed"):
        batch.replace([a])
    cache.resize(2)
    batch.replace([a])
    _step(batch, [100])
    assert batch.advance() == [] and batch.lengths.tolist() == [17]
    model[a] = ([u + 100 for u in model[a][0]] + [0], model[a][1] + [100])
    _check(cache, model)


def test_the_others_go_on(plain):
    """Three sequences, pages for two of them: the third leaves with all its positions and comes back to the pages of one that is freed."""
    cache = _cache(pages=5)
    seqs = [cache.add() for _ in range(3)]
    model = {q: ([], []) for q in seqs}
    batch = cache.batch(seqs, size=4, width=3)
    tensors = batch.u_table, batch.table, batch.lengths

    def token(value, gone):
        who = list(batch.seqs)
        _step(batch, [value + i for i in range(4)])
        assert batch.advance(leave=True) == gone
        for i, q in enumerate(who):
            if q is not None:
                u, rows = model[q]
                model[q] = ([v + value + i for v in u] + [0], rows + [value + i])
        _check(cache, model)
        assert batch.lengths.tolist() == [-1 if q is None else len(model[q][0]) for q in batch.seqs]

    for t in range(15):
        token(t, [])
    token(15, [seqs[2]])                                                # 16 each; the two free pages are the first two's
    for t in range(5):
        token(20 + t, [])
    cache.free(seqs[0])
    del model[seqs[0]]
    batch.replace([seqs[2], seqs[1]])
    for t in range(12):
        token(30 + t, [])
    assert all(a is b for a, b in zip(tensors, (batch.u_table, batch.table, batch.lengths)))
    assert [cache.length(q) for q in seqs[1:]] == [33, 28]


def test_a_sequence_that_leaves_as_another_outgrows_the_tables(plain):
    cache = _cache(pages=4)
    a, b = cache.add(), cache.add()
    z = torch.zeros(1, 1, 31, 16, dtype=torch.float64)
    cache.write([a], 0, (z, z, z, z))
    z = z[:, :, :15]
    cache.write([b], 0, (z, z, z, z))
    batch = cache.batch([a, b])
    assert batch.table.shape == (2, 2) and cache.free_pages() == (1, 1)
    assert batch.advance(leave=True) == [b]
    assert batch.table.shape == (2, 3) and batch.lengths.tolist() == [32, -1] and batch.table[1].tolist() == [-1] * 3
    assert cache.length(a) == 32 and cache.length(b) == 16 and cache.batch([None], width=1).seqs == [None]
    cache.free(a)
    assert cache.batch([b]).lengths.tolist() == [16]


def test_under_another_default_device(plain):
    """Lists on their way to the cache's device begin on the host, whatever the default device is ("meta": one without values, which cannot be copied from)."""
    cache = _cache()
    a = cache.add()
    z = torch.ones(1, 1, 15, 16, dtype=torch.float64)
    with torch.device("meta"):
        cache.write([a], 0, (z, z, z, z))
        batch = cache.batch([a])
        for _ in range(3):                                              # over the end of a page
            batch.advance()
        (b,) = cache.fork(a)
        batch.replace([b, a])
        cache.free(b)
        cache.compact()
        cache.resize(10)
    assert batch.lengths.tolist() == [-1, 18] and all(t.device.type == "cpu" for t in (batch.u_table, batch.table, batch.lengths, cache.U, cache.kc))
    other = _cache()
    q = other.add()
    with torch.device("meta"):
        made = other.batch([q], size=2, width=3)
    assert made.table.device.type == made.lengths.device.type == "cpu" and made.lengths.tolist() == [0, -1]


def test_refusals(plain):
    for bad in (dict(layers=0), dict(pages=0), dict(u_pages=0), dict(page_size=8), dict(page_size=48), dict(dim_head=48)):
        with pytest.raises(ValueError):
            _cache(**bad)
    cache = _cache()
    a, b = cache.add(), cache.add()
    z = torch.zeros(1, 1, 4, 16, dtype=torch.float64)
    for bad in (lambda: cache.free(7), lambda: cache.fork(7), lambda: cache.length(7), lambda: cache.batch([7]), lambda: cache.batch([]), lambda: cache.batch([a, a]),
                lambda: cache.write([a, b], 0, (z, z, z, z)), lambda: cache.write([a], 2, (z, z, z, z)), lambda: cache.write([a], -1, (z, z, z, z)), lambda: cache.resize(0)):
        with pytest.raises(ValueError):
            bad()
    batch = cache.batch([a])
    for bad in (lambda: cache.batch([a, b]), lambda: cache.write([a], 0, (z, z, z, z)), lambda: batch.layer(2), lambda: batch.replace([a, a])):
        with pytest.raises(ValueError):
            bad()
    assert batch.seqs == [a]
    del batch
    cache.batch([a, b])


def test_linear_4bit_module():
    from lookahead_keys_attention_b200 import Linear4bit
    m = Linear4bit.from_linear(torch.nn.Linear(100, 30).bfloat16(), group_size=32, zeros=True).eval()
    assert m.codes.shape == (2, 512) and m.scales.shape == m.zeros.shape == (30, 4) and m.scales.dtype == torch.bfloat16 and not m.training
    other = Linear4bit(100, 30, True, 32, True, dtype=torch.bfloat16)
    other.load_state_dict(m.state_dict())
    assert all(torch.equal(a, b) for a, b in zip(other.state_dict().values(), m.state_dict().values())) and "group_size=32" in repr(other)
    assert [n for n, _ in m.named_parameters()] == ["bias"]
    with pytest.raises(ValueError):
        Linear4bit(10, 10, group_size=20)
