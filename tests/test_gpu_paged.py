"""GPU: the cached step over caches in pages, against its definition in 64 bits.

Tolerances.  A lookahead key is the sum of the old one and gate * vu in fp32, rounded once: half a step of its type, eps / 2 of its size, and the
gate's error times vu.  The gate is 1 / (1 + e^-z): z is a sum of d products in fp32 (d + 2 roundings of 2^-24 of the sum of their sizes), a quarter
of whose error reaches the gate, and __expf is off by 2 + 1.2 |z| units of 2^-23, of which at most 0.25 (2 + 1.2 |z|) 2^-23 < 2^-20 reach it (the
gate's slope makes up for large z).  Scores: two such sums, silu's slope is below 1.1, and su times the gate's error.  The result is a mean of the
values with weights e^score: an error e of every score moves it by at most 2 e max|v|; the weights have __expf's error (2^-20, as above), the running
sums n roundings, and the result one of its own type.  The scores of the definition are those of the lookahead keys as they are kept, so the
reference takes the kernel's (which are checked first)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -23}


class Case:
    """Sequences in pages of random order, tables with rubbish behind each last page."""

    def __init__(self, dtype, lengths, H, d, page, seed=0, layout="plain", std=1.0, tables="own"):
        gen = torch.Generator("cuda").manual_seed(seed)
        self.dtype, self.lengths, self.H, self.d, self.page, self.scale = dtype, lengths, H, d, page, d ** -0.5
        B = len(lengths)
        randn = lambda *s: torch.randn(*s, device="cuda", generator=gen).mul_(std).to(dtype)  # noqa: E731
        need = [max(n, 0) // page + 1 for n in lengths]
        width = max(need) + 1
        tables = []
        for _ in range(2):
            pages = sum(need) + 3
            order = torch.randperm(pages, generator=gen, device="cuda").int().cpu()
            t, at = torch.full((B, width), 2 ** 31 - 1, dtype=torch.int32), 0
            for b, n in enumerate(need):
                t[b, :n] = order[at:at + n]
                at += n
            tables.append((t.cuda(), pages))
        (self.u_table, u_pages), (self.table, pages) = tables
        self.pools = []
        for n in (u_pages, pages, pages, pages):
            if layout == "plain":
                self.pools.append(randn(n, H, page, d))
            elif layout == "layers":       # one of the layers of pages that hold them all
                self.pools.append(randn(n, 3, H, page, d)[:, 1])
            else:                          # heads first
                self.pools.append(randn(H, n, page, d).transpose(0, 1))
        packed = randn(B, 1, 6, H, d)
        self.new = [packed[:, :, i].transpose(1, 2) for i in (3, 4, 5, 0, 1, 2)] if layout != "plain" else [randn(B, H, 1, d) for _ in range(6)]
        self.lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def step(self):
        from lookahead_keys_attention_b200 import castle_paged_decode_step
        return castle_paged_decode_step(*self.new, *self.pools, self.u_table, self.table, self.lens, self.scale)

    def rows(self, i, b, count, pools):
        r = torch.arange(count, device="cuda")
        t = (self.u_table if i == 0 else self.table)[b].long()
        return pools[i][t[r // self.page], :, r % self.page].transpose(0, 1)      # (H, count, d)

    def check(self, before, out):
        """`before`: the pools as they were; the pools now and `out` against the definition."""
        eps = EPS[self.dtype]
        want = [p.clone() for p in before]
        for b, n in enumerate(self.lengths):
            new = [t[b, :, 0].double() for t in self.new]
            qc, kc, vc, qu, ku, vu = new
            if n < 0:
                assert bool((out[b] == 0).all())
                continue
            at = n // self.page, n % self.page
            for i, row in enumerate((torch.zeros_like(qu), qu, kc, vc)):
                want[i][(self.u_table if i == 0 else self.table)[b, at[0]].long(), :, at[1]] = row.to(self.dtype)
            u0, qus = self.rows(0, b, n, before).double(), self.rows(1, b, n, before).double()
            u1, ks, vs = self.rows(0, b, n, self.pools).double(), self.rows(2, b, n, before).double(), self.rows(3, b, n, before).double()
            z = torch.einsum("hnd,hd->hn", qus, ku) * self.scale
            z_err = (self.d + 3) * 2.0 ** -24 * torch.einsum("hnd,hd->hn", qus.abs(), ku.abs()) * self.scale
            exact_u = u0 + torch.sigmoid(z)[..., None] * vu[:, None]
            tol = (eps / 2 + 2.0 ** -23) * exact_u.abs() + (z_err / 4 + 2.0 ** -20)[..., None] * vu.abs()[:, None] + 1e-7
            bad = (u1 - exact_u).abs() - tol
            assert n == 0 or bad.max().item() <= 0, f"U of sequence {b}: {bad.max().item():.3e} above the tolerance"
            su, sc = torch.einsum("hnd,hd->hn", u1, qc) * self.scale, torch.einsum("hnd,hd->hn", ks, qc) * self.scale
            own = (qc * kc).sum(-1, keepdim=True) * self.scale
            s = torch.cat((sc - torch.nn.functional.silu(su), own), -1)
            err = (self.d + 3) * 2.0 ** -24 * self.scale * (torch.einsum("hnd,hd->hn", ks.abs(), qc.abs()) + 1.1 * torch.einsum("hnd,hd->hn", u1.abs(), qc.abs())) + su.abs() * 2.0 ** -20
            e = torch.cat((err, (self.d + 3) * 2.0 ** -24 * self.scale * (qc * kc).abs().sum(-1, keepdim=True)), -1).amax(-1)
            v = torch.cat((vs, vc[:, None]), 1)
            exact = torch.einsum("hn,hnd->hd", torch.softmax(s, -1), v)
            tol = eps / 2 * exact.abs() + (2 * e + 2.0 ** -19 + (n + 16) * 2.0 ** -24)[:, None] * v.abs().amax((1, 2))[:, None]
            off = (out[b, :, 0].double() - exact).abs() - tol
            assert off.max().item() <= 0, f"sequence {b} of {n} positions: {off.max().item():.3e} above the tolerance"
            t = self.u_table[b].long()
            r = torch.arange(n, device="cuda")
            want[0][t[r // self.page], :, r % self.page] = self.pools[0][t[r // self.page], :, r % self.page]   # (checked above)
        for i, name in enumerate(("U", "qu", "kc", "vc")):
            assert torch.equal(self.pools[i], want[i]), f"{name}: a row that is not the step's was written, or the appended one is not the token's"


def _run(c):
    from lookahead_keys_attention_b200 import check_status
    before = [p.clone() for p in c.pools]
    out = c.step()
    check_status()
    assert out.shape == (len(c.lengths), c.H, 1, c.d) and out.dtype == c.dtype
    c.check(before, out)
    return out


LENGTHS = {"one": [1], "zero": [0, 0], "few": [0, 1, 15, 16, 17, 31, 32, 33], "ragged": [777, -1, 3, 1200, 64, 0, -7, 255, 256], "long": [9001]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_against_the_definition(dtype, d, lengths):
    for page in (16, 64, 256):
        _run(Case(dtype, LENGTHS[lengths], 3, d, page, seed=d + page))


@pytest.mark.parametrize("layout", ["layers", "heads"])
@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 32), (torch.float32, 1024)])
def test_pools_and_rows_of_other_strides(layout, dtype, page):
    c = Case(dtype, [100, 2047, 5, 0], 5, 64, page, layout=layout)
    assert not c.pools[0].is_contiguous() and not c.new[0].is_contiguous()
    _run(c)


def test_many_sequences_of_many_pieces():
    """More pairs than there are CTAs, whole and cut ones, and batches beyond a CTA's threads."""
    _run(Case(torch.bfloat16, [16000 - 131 * i for i in range(48)], 8, 16, 128, std=0.5))
    _run(Case(torch.float16, [(i * 7) % 50 - 2 for i in range(700)], 2, 64, 16))


def test_a_step_after_the_other():
    """Tokens one after the other, beside the step over contiguous caches."""
    from lookahead_keys_attention_b200 import castle_decode_step, castle_paged_decode_step, check_status
    n, H, d, page = 30, 4, 64, 16
    c = Case(torch.float32, [n, n], H, d, page, seed=3)
    wide = torch.arange(8, dtype=torch.int32, device="cuda").repeat(2, 1)
    wide[1] += 8
    pools = [torch.randn(16, H, page, d, device="cuda") for _ in range(4)]
    bufs = [p.view(2, 8, H, page, d).transpose(1, 2).reshape(2, H, 8 * page, d).clone() for p in pools]
    lens = c.lens.clone()
    for t in range(n, n + 40):
        new = [torch.randn(2, H, 1, d, device="cuda") for _ in range(6)]
        a = castle_paged_decode_step(*new, *pools, wide, wide, lens, c.scale)
        b = castle_decode_step(*new, *bufs, t, c.scale)
        assert (a - b).abs().max() <= 2e-5
        lens += 1
    check_status()
    for p, q in zip(pools, bufs):
        assert (p.view(2, 8, H, page, d).transpose(1, 2).reshape(2, H, 8 * page, d) - q).abs().max() <= 2e-4


def test_shared_pages_are_read_and_left():
    c = Case(torch.bfloat16, [200, 200, 71], 4, 64, 32, seed=5)
    c.table[1, :6] = c.table[0, :6]      # 192 common positions
    c.table[2, :2] = c.table[0, :2]
    _run(c)


def test_same_bits_every_time_and_whatever_the_batch():
    """A sequence's result does not depend on who else is in the batch where it is cut the same way, nor on the run."""
    c = Case(torch.bfloat16, [5000, 12, 900], 8, 64, 64, seed=8)
    before = [p.clone() for p in c.pools]
    first = c.step()
    after = [p.clone() for p in c.pools]
    for _ in range(5):
        for p, q in zip(c.pools, before):
            p.copy_(q)
        assert torch.equal(c.step(), first) and all(torch.equal(p, q) for p, q in zip(c.pools, after))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_sequence_in_different_batches(dtype):
    """Who else is in the batch decides where a sequence is cut: its result is within the tolerance in each of them, its lookahead keys are the same bits."""
    from lookahead_keys_attention_b200 import check_status
    c = Case(dtype, [5000, 12, 900, 4097, 64], 8, 64, 64, seed=14)
    before, everyone, keys, outs = [p.clone() for p in c.pools], list(c.lengths), [], []
    for there in ([0, 1, 2, 3, 4], [0], [0, 1], [0, 3], [0, 2, 4]):
        c.lengths = [n if b in there else -1 for b, n in enumerate(everyone)]
        c.lens.copy_(torch.tensor(c.lengths, dtype=torch.int32))
        for p, q in zip(c.pools, before):
            p.copy_(q)
        out = c.step()
        check_status()
        c.check(before, out)
        keys.append(c.rows(0, 0, everyone[0], c.pools))
        outs.append(out[0])
    assert all(torch.equal(k, keys[0]) for k in keys)
    # fp32: two results of one sequence are apart by what joining in another order rounds, n + 16 roundings of each, and twice the weights' error, 2^-19 of the largest value
    largest = c.rows(3, 0, everyone[0] + 1, c.pools).abs().amax().item()
    if dtype == torch.float32:
        assert all((o - outs[0]).abs().max().item() <= 2 * (2.0 ** -19 + (everyone[0] + 16) * 2.0 ** -24) * largest for o in outs)


@pytest.mark.parametrize("bad", ["u", "kv", "new", "length"])
def test_places_outside_the_pools(bad):
    """NaN for the sequence, the others as they should be, nothing written outside; then the status, which is clear again after it."""
    from lookahead_keys_attention_b200 import check_status
    c = Case(torch.bfloat16, [300, 100, 40], 4, 64, 32, seed=9)
    before = [p.clone() for p in c.pools]
    if bad == "u":
        c.u_table[1, 1] = c.pools[0].shape[0]
    elif bad == "kv":
        c.table[1, 2] = -1
    elif bad == "new":
        c.table[1, 3] = 2 ** 31 - 1
    else:
        c.lens[1] = c.table.shape[1] * c.page
    out = c.step()
    with pytest.raises(RuntimeError, match="status 4"):
        check_status()
    check_status()
    assert bool(out[1].isnan().all()) and bool(out[[0, 2]].isfinite().all())
    good = Case(torch.bfloat16, [300, 100, 40], 4, 64, 32, seed=9)
    want = good.step()
    assert torch.equal(out[[0, 2]], want[[0, 2]])
    mine = good.table[1, :4].long() if bad != "length" else None
    for p, q, b in zip(c.pools[1:], good.pools[1:], before[1:]):
        keep = torch.ones(len(p), dtype=torch.bool, device="cuda")
        if mine is not None:
            keep[mine] = False
        else:
            keep[good.table[1, :4].long()] = False
            assert torch.equal(p[~keep], b[~keep])
        assert torch.equal(p[keep], q[keep])


def test_values_that_are_not_finite_stay_in_their_sequence():
    c = Case(torch.float16, [100, 100, 100], 2, 64, 16, seed=10)
    c.pools[2][c.table[1, 2].long(), 1, 3, 5] = float("nan")
    c.pools[2][c.table[2, 0].long(), 0, 0] = float("-inf")     # a score of minus infinity (or plus) in the first row
    c.new[0][2] = c.new[0][2].abs()
    out = c.step()
    assert bool(out[0].isfinite().all()) and bool(out[1, 0].isfinite().all()) and bool(out[1, 1].isnan().all())
    assert bool(out[2].isfinite().all())


@pytest.mark.parametrize("limit", [0, 1, 2, 5, 20, 100])
def test_rows_that_do_not_arrive_in_time(limit):
    """Waits for rows that give up after some polls: every pair has its whole result or NaN, the status says so, rows that did not arrive stay as they were, and the next
    step is right."""
    from lookahead_keys_attention_b200 import _lib, check_status
    lib = _lib.load()
    shape = torch.bfloat16, [900, 0, 40, 2500, 333], 4, 64, 32
    c, good = Case(*shape, seed=13), Case(*shape, seed=13)
    before = [p.clone() for p in c.pools]
    want = good.step()
    check_status()
    _lib.check(lib.castle_selftest_paged_polls(limit), "paged_polls")
    try:
        out = c.step()
    finally:
        _lib.check(lib.castle_selftest_paged_polls(-1), "paged_polls")
    lost = out.isnan().flatten(2)
    assert bool((lost.all(-1) == lost.any(-1)).all()) and torch.equal(out[~lost.any(-1)], want[~lost.any(-1)])
    if bool(lost.any()):
        with pytest.raises(RuntimeError, match="status 1"):
            check_status()
    if limit == 0:                                                       # none arrives
        rows = [0, 2, 3, 4]
        assert bool(lost[rows].all())
        spare = c.u_table[1, 0].long(), c.table[1, 0].long()
        for i, (p, q) in enumerate(zip(c.pools, before)):
            keep = torch.ones(len(p), dtype=torch.bool, device="cuda")
            keep[spare[min(i, 1)]] = False
            assert torch.equal(p[keep], q[keep])
    for p, q, w in zip(c.pools, before, good.pools):                     # a row is the one before or the one of the whole step
        assert bool(((p == q) | (p == w)).all())
        p.copy_(q)
    for _ in range(2):
        assert torch.equal(c.step(), want) and all(torch.equal(p, q) for p, q in zip(c.pools, good.pools))
        for p, q in zip(c.pools, before):
            p.copy_(q)
    check_status()


def test_places_beyond_32_bits():
    """Pools of more than 2^31 elements, pages at their ends."""
    from lookahead_keys_attention_b200 import castle_paged_decode_step, check_status
    H, d, page = 16, 128, 64
    pages = 2 ** 31 // (H * page * d) + 40
    pools = [torch.zeros(pages, H, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    c = Case(torch.bfloat16, [150, 90], H, d, page, seed=11)
    small = [p.clone() for p in c.pools]
    want = c.step()
    shift = pages - max(p.shape[0] for p in small)
    for big, s in zip(pools, small):
        big[shift:shift + len(s)] = s
    out = castle_paged_decode_step(*c.new, *pools, c.u_table + shift, c.table + shift, c.lens, c.scale)
    check_status()
    assert torch.equal(out, want)
    for big, s in zip(pools, c.pools):
        assert torch.equal(big[shift:shift + len(s)], s) and not big[:shift].any()


def test_a_captured_step_follows_lengths_and_tables():
    c = Case(torch.bfloat16, [70, 300, -1], 4, 64, 32, seed=12)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = c.step()
    for lengths in ([70, 300, -1], [64, -1, 10], [0, 31, 15]):
        c.lengths = lengths
        c.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        before = [p.clone() for p in c.pools]
        graph.replay()
        torch.cuda.synchronize()
        c.check(before, out)


def test_streams_beside_each_other():
    cases = [Case(torch.bfloat16, [3000 + 100 * i, 50, 700], 8, 64, 64, seed=20 + i) for i in range(3)]
    want = [Case(torch.bfloat16, [3000 + 100 * i, 50, 700], 8, 64, 64, seed=20 + i).step() for i in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            outs.append(c.step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,page", [(16, 16), (64, 64), (128, 1024)])
def test_prompts_into_pages(dtype, d, page):
    from lookahead_keys_attention_b200 import castle_write_pages, check_status
    for layout in ("plain", "layers", "heads"):
        c = Case(dtype, [1, 130, 2047, -1, 0, 64], 3, d, page, seed=d, layout=layout)
        caches = [torch.randn(6, 3, 2047, d, device="cuda").to(dtype) for _ in range(3)]
        caches.append(torch.randn(6, 2047, 3, d, device="cuda").to(dtype).transpose(1, 2))
        want = [p.clone() for p in c.pools]
        for b, n in enumerate(c.lengths):
            for i in range(4):
                r = torch.arange(max(n, 0), device="cuda")
                want[i][(c.u_table if i == 0 else c.table)[b].long()[r // page], :, r % page] = caches[i][b, :, :max(n, 0)].transpose(0, 1)
        castle_write_pages(*caches, *c.pools, c.u_table, c.table, c.lens)
        check_status()
        assert all(torch.equal(p, w) for p, w in zip(c.pools, want))


@pytest.mark.parametrize("bad", ["page", "long", "wide"])
def test_prompts_that_have_no_place(bad):
    from lookahead_keys_attention_b200 import castle_write_pages, check_status
    c = Case(torch.bfloat16, [40, 60], 2, 64, 16, seed=1)
    caches = [torch.randn(2, 2, 100, 64, device="cuda").bfloat16() for _ in range(4)]
    before = [p.clone() for p in c.pools]
    if bad == "page":
        c.table[0, 1], c.u_table[0, 1] = -1, 2 ** 31 - 1
    elif bad == "long":
        c.lens[0] = 101
    else:
        caches = [torch.randn(2, 2, 1000, 64, device="cuda").bfloat16() for _ in range(4)]
        c.lens[0] = c.table.shape[1] * 16 + 1
    castle_write_pages(*caches, *c.pools, c.u_table, c.table, c.lens)
    with pytest.raises(RuntimeError, match="status 4"):
        check_status()
    for i in range(4):
        assert torch.equal(c.rows(i, 1, 60, c.pools), caches[i][1, :, :60])
        t = (c.u_table if i == 0 else c.table)[0].long()
        if bad == "page":
            assert torch.equal(c.pools[i][t[0]], caches[i][0, :, :16]) and torch.equal(c.pools[i][t[2], :, :8], caches[i][0, :, 32:40])
        else:
            assert torch.equal(c.pools[i][t[:3]], before[i][t[:3]])


@pytest.mark.parametrize("pools,shape,dtype", [(1, (64, 8, 16, 64), torch.bfloat16), (30, (50, 2, 16, 16), torch.float32), (2, (2000, 1, 16, 16), torch.float16),
                                               (3, (9, 3, 8), torch.int32), (1, (7, 5, 1024, 128), torch.bfloat16)])
def test_copies_of_pages(pools, shape, dtype):
    from lookahead_keys_attention_b200 import castle_copy_pages
    ps = [torch.randint(-100, 100, shape, device="cuda").to(dtype) for _ in range(pools)]
    order = torch.randperm(shape[0])
    k = shape[0] // 2
    source, target = order[:k], order[k:2 * k]
    want = [p.clone() for p in ps]
    for w in want:
        w[target.cuda()] = w[source.cuda()]
    castle_copy_pages(ps, source.tolist(), target.int())
    assert all(torch.equal(p, w) for p, w in zip(ps, want))
    same = [torch.cat([source[:1]] * 3), order[k:k + 3]]      # one page to three places
    for w in want:
        w[same[1].cuda()] = w[same[0].cuda()]
    for p in ps:
        castle_copy_pages(p, *same)
    assert all(torch.equal(p, w) for p, w in zip(ps, want))
    castle_copy_pages(ps, [], [])


def test_copies_of_pages_of_other_strides():
    from lookahead_keys_attention_b200 import castle_copy_pages
    for make in (lambda: torch.randn(20, 3, 4, 16, 64, device="cuda")[:, 1], lambda: torch.randn(4, 20, 16, 64, device="cuda").transpose(0, 1)):
        ps = [make(), make()]
        want = [p.clone() for p in ps]
        for w in want:
            w[[5, 6]] = w[[19, 0]]
        whole = [p._base.clone() for p in ps]
        castle_copy_pages(ps, [19, 0], [5, 6])
        for p, w, b in zip(ps, want, whole):
            assert torch.equal(p, w)
            p[[5, 6]] = 0
            (b[[5, 6], 1] if b.dim() == 5 else b[:, [5, 6]]).zero_()
            if b.dim() == 5:
                b[[5, 6], 1] = 0
            else:
                b[:, [5, 6]] = 0
            assert torch.equal(p._base, b)


def test_copies_beyond_32_bits():
    from lookahead_keys_attention_b200 import castle_copy_pages
    pool = torch.zeros(2 ** 31 // 65536 + 3, 8, 64, 128, dtype=torch.bfloat16, device="cuda")
    last = pool.shape[0] - 1
    pool[last] = torch.randn(8, 64, 128, device="cuda").bfloat16()
    castle_copy_pages(pool, [last], [1])
    castle_copy_pages(pool, [1], [last - 1])
    assert torch.equal(pool[1], pool[last]) and torch.equal(pool[last - 1], pool[last]) and not pool[0].any() and not pool[2:last - 1].any()
