"""The operators of serving from a paged cache, as cases that can be timed and compared: the cached step of sequences of different
lengths, the pages' copies, and the products with 4-bit weights that a token's projections are.

A case's "kind" says which call it is:

    step      castle_paged_decode_step: a token for each of `batch` sequences of up to `n` positions
    copy      castle_copy_pages: `copied` pages of each of `pools` pools, as a fork or a compaction copies them
    write     castle_write_pages: a prompt's four caches into pages
    linear    castle_linear_4bit: `rows` rows times a (out, in) weight; where "train" is true the rows' gradient, too (adapters that
              are trained in front of frozen weights)

With `own` false `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _step(name, dtype, batch, heads, dim_head, n, page, ragged=True):
    return {"name": name, "kind": "step", "dtype": dtype, "batch": batch, "heads": heads, "dim_head": dim_head, "n": n, "page": page, "ragged": ragged}


def _copy(name, dtype, pools, heads, dim_head, page, pages, copied):
    return {"name": name, "kind": "copy", "dtype": dtype, "pools": pools, "heads": heads, "dim_head": dim_head, "page": page, "pages": pages, "copied": copied}


def _write(name, dtype, batch, heads, dim_head, n, page, ragged=False):
    return {"name": name, "kind": "write", "dtype": dtype, "batch": batch, "heads": heads, "dim_head": dim_head, "n": n, "page": page, "ragged": ragged}


def _linear(name, dtype, rows, inner, out, group, zeros=False, train=False):
    return {"name": name, "kind": "linear", "dtype": dtype, "rows": rows, "in": inner, "out": out, "group": group, "zeros": zeros, "train": train}


def listed():
    return [
        # Two short fp32 sequences (the README's heads and length): latency alone.
        _step("step_b2_128_fp32", "fp32", 2, 8, 64, 128, 16),
        # Sampling from a layer of the byte language model: a batch of ragged lengths up to its context.
        _step("step_lm_b16_1024", "bf16", 16, 8, 64, 1024, 32),
        # The decode benchmark's heads, 64 sequences of ragged lengths, 8.3 thousand positions on average.
        _step("step_b64_16411", "bf16", 64, 16, 128, 16411, 64),
        # One long sequence.
        _step("step_b1_131071_fp16", "fp16", 1, 16, 128, 131071, 128, ragged=False),
        # A short sequence of one layer is forked: two pages of its lookahead keys.
        _copy("copy_fork_2", "bf16", 1, 8, 64, 16, 64, 2),
        # A sequence of 8192 positions is forked in all 8 layers of a model.
        _copy("copy_fork_8_layers", "bf16", 8, 16, 128, 64, 512, 129),
        # A prompt of ragged length through a layer of the language model.
        _write("write_lm_197", "bf16", 1, 8, 64, 197, 32),
        # A long prompt, an odd number of positions.
        _write("write_8189_d128", "bf16", 2, 16, 128, 8189, 64),
        # A token's feed-forward projection in the language model.
        _linear("linear_1_512_2048", "bf16", 1, 512, 2048, 64),
        # A wide model's token.
        _linear("linear_1_4096_16384", "bf16", 1, 4096, 16384, 128),
        # The head over an odd vocabulary, a few sequences, zero points.
        _linear("linear_8_1000_50021_fp16", "fp16", 8, 1000, 50021, 32, zeros=True),
        # A ragged batch's rows through a wide projection, and their gradient.
        _linear("linear_train_777_4096", "bf16", 777, 4096, 4096, 64, train=True),
    ]


MOST_CACHE = 64 * 16 * 8300 * 128 * 2       # bytes of one cache of the largest listed step
MOST_COPY = 8 * 129 * 16 * 64 * 128 * 2     # bytes that the largest listed copy reads
MOST_WRITE = 2 * 16 * 8189 * 128 * 2        # bytes of one cache of the largest listed prompt
MOST_WEIGHT = 4096 * 16384                  # elements of the largest listed weight
MOST_PRODUCT = 777 * 4096 * 4096


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "copy", "write", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    heads, dim_head, page = _log_uniform(rng, 1, 32), rng.choice([16, 32, 64, 64, 128, 128]), rng.choice([16, 32, 64, 128, 256])
    if kind == "step":
        batch, n = _log_uniform(rng, 1, 256), _log_uniform(rng, 1, 131072)
        while batch * heads * n * dim_head * size > MOST_CACHE:
            batch, n = (batch + 1) // 2, max(1, n * 3 // 4)
        c = _step(None, dtype, batch, heads, dim_head, n, page, rng.random() < 0.8)
    elif kind == "copy":
        pools, copied = rng.choice([1, 1, 3, 8, 24]), _log_uniform(rng, 1, 1000)
        while pools * copied * heads * page * dim_head * size > MOST_COPY:
            copied, pools = max(1, copied // 2), (pools + 1) // 2
        c = _copy(None, dtype, pools, heads, dim_head, page, 2 * copied + rng.randint(0, copied), copied)
    elif kind == "write":
        batch, n = _log_uniform(rng, 1, 16), _log_uniform(rng, 1, 16384)
        while batch * heads * n * dim_head * size > MOST_WRITE:
            batch, n = (batch + 1) // 2, max(1, n * 3 // 4)
        c = _write(None, dtype, batch, heads, dim_head, n, page, rng.random() < 0.5)
    else:
        step = rng.choice([128, 64, 8, 1])
        rows, inner, out = rng.choice([1, 1, 1, _log_uniform(rng, 2, 64), _log_uniform(rng, 2, 2048)]), _log_uniform(rng, 64, 16384), _log_uniform(rng, 64, 131072)
        inner = max(64, inner // step * step)
        while inner * out > MOST_WEIGHT or rows * inner * out * (4 if dtype == "fp32" else 1) > MOST_PRODUCT:
            rows, out = (rows + 1) // 2, max(64, out * 3 // 4)
        c = _linear(None, dtype, rows, inner, out, rng.choice([32, 64, 64, 128, 256]), rng.random() < 0.4, rng.random() < 0.2)
    del c["name"]
    return c


def _randn(shape, dtype, gen, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _lengths(c):
    """Positions of each sequence: spread evenly between none and n, the last one n (a server's sequences are anywhere in their course)."""
    if not c["ragged"]:
        return [c["n"]] * c["batch"]
    golden = (5 ** 0.5 - 1) / 2
    return [int(c["n"] * (golden * (b + 1) % 1)) for b in range(c["batch"] - 1)] + [c["n"]]


def _tables(c, lengths, spare, gen):
    """Where each sequence's pages lie in a pool, in any order, -1 behind its last one; and the number of pages of the pool."""
    page = c["page"]
    need = [(n + spare + page - 1) // page for n in lengths]
    pages = sum(need) + sum(need) // 8 + 1
    table = torch.full((len(need), max(max(need), 1) + 2), -1, dtype=torch.int32)
    places = torch.randperm(pages, device="cuda", generator=gen).int().cpu()
    at = 0
    for b, count in enumerate(need):
        table[b, :count] = places[at:at + count]
        at += count
    return table.cuda(), pages


def _flat(c, lengths, *tables):
    """The pages that hold rows, one after the other: their sequence, which of its pages each is, and their places."""
    page = c["page"]
    counts = [(n + page - 1) // page for n in lengths]
    seq = torch.tensor([b for b, k in enumerate(counts) for _ in range(k)], dtype=torch.int64, device="cuda")
    nth = torch.tensor([i for k in counts for i in range(k)], dtype=torch.int64, device="cuda")
    return seq, nth, [t[seq, nth].long() for t in tables]


def prepare(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "linear":
        R, K, N, g = c["rows"], c["in"], c["out"], c["group"]
        groups = (K + g - 1) // g
        s["codes"] = torch.randint(0, 16, (N, K), dtype=torch.uint8, device="cuda", generator=gen)
        s["x"] = _randn((R, K), dtype, gen)
        s["x"][:, torch.randint(0, K, (1 + K // 500,), device="cuda", generator=gen)] *= 8.0    # a few large channels, as activations have them
        # weights of spread K^-1/2: codes spread over 16 steps, 4.6 of them the standard deviation
        s["scales"] = (torch.empty((N, groups), device="cuda").uniform_(0.5, 1.5, generator=gen) * (K ** -0.5 / 4.6)).to(dtype)
        s["grad"] = _randn((R, N), dtype, gen, 1e-2) if c["train"] else None
        s["x"].requires_grad_(c["train"])
        s["zeros"] = torch.empty((N, groups), device="cuda").uniform_(5.0, 10.0, generator=gen).round_().to(dtype) if c["zeros"] else None
        if own:
            import lookahead_keys_attention_b200 as castle
            s["packed"] = castle.castle_pack_4bit(s["codes"])
        return s
    H, d, page = c["heads"], c["dim_head"], c["page"]
    if c["kind"] == "copy":
        s["pools"] = [_randn((c["pages"], H, page, d), dtype, gen) for _ in range(c["pools"])]
        order = torch.randperm(c["pages"], device="cuda", generator=gen)
        s["source"], s["target"] = order[:c["copied"]].cpu(), order[c["copied"]:2 * c["copied"]].cpu()
        s["source_gpu"], s["target_gpu"] = s["source"].cuda(), s["target"].cuda()
        return s
    B, lengths = c["batch"], _lengths(c)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["u_table"], u_pages = _tables(c, lengths, 1, gen)
    s["table"], pages = _tables(c, lengths, 1, gen)
    # projections of unit-variance inputs; a lookahead key is a sum of up to n such rows with gates around 1/2
    s["pools"] = [_randn((p, H, page, d), dtype, gen, std) for p, std in
                  [(u_pages, 0.5 * max(1.0, c["n"]) ** 0.5 / 2), (pages, 3 ** -0.5), (pages, 3 ** -0.5), (pages, 3 ** -0.5)]]
    if c["kind"] == "step":
        s["new"] = [_randn((B, H, 1, d), dtype, gen, 3 ** -0.5) for _ in range(6)]
    else:
        s["caches"] = [_randn((B, H, c["n"], d), dtype, gen, 3 ** -0.5) for _ in range(4)]
    s["seq"], s["nth"], (s["u_flat"], s["flat"]) = _flat(c, lengths, s["u_table"], s["table"])
    last = s["lengths"].long()
    s["u_last"], s["last"] = (t.long().gather(1, (last // page)[:, None])[:, 0] for t in (s["u_table"], s["table"]))
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import lookahead_keys_attention_b200 as castle
    c = s["case"]
    if c["kind"] == "linear":
        y = castle.castle_linear_4bit(s["x"], s["packed"], s["scales"], s["zeros"], group_size=c["group"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, [s["x"]], s["grad"])[0]} if c["train"] else y
    if c["kind"] == "copy":
        castle.castle_copy_pages(s["pools"], s["source"], s["target"])
        return s["pools"]
    if c["kind"] == "write":
        castle.castle_write_pages(*s["caches"], *s["pools"], s["u_table"], s["table"], s["lengths"])
        return s["pools"]
    out = castle.castle_paged_decode_step(*s["new"], *s["pools"], s["u_table"], s["table"], s["lengths"], c["dim_head"] ** -0.5)
    return {"out": out, "pools": s["pools"]}


def _rows_of(s):
    """The number in its sequence of each row of the flat pages, (pages, 1, page), and whether it is one of the sequence's."""
    at = s["nth"][:, None] * s["case"]["page"] + torch.arange(s["case"]["page"], device="cuda")
    return at, (at < s["lengths"].long()[s["seq"]][:, None])[:, None]


def _run_plain(s):
    c = s["case"]
    with torch.no_grad():
        if c["kind"] == "linear":
            K, g = c["in"], c["group"]
            w = s["codes"].float()
            zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(g, 1)[:, :K]
            w = (w - zero) * s["scales"].float().repeat_interleave(g, 1)[:, :K]
            y = (s["x"].float() @ w.t()).to(s["x"].dtype)
            return {"y": y, "dx": (s["grad"].float() @ w).to(s["x"].dtype)} if c["train"] else y
        if c["kind"] == "copy":
            for p in s["pools"]:
                p[s["target_gpu"]] = p[s["source_gpu"]]
            return s["pools"]
        at, valid = _rows_of(s)
        seq, page = s["seq"], c["page"]
        if c["kind"] == "write":
            n = at.clamp(max=c["n"] - 1)
            for cache, pool, flat in zip(s["caches"], s["pools"], (s["u_flat"], s["flat"], s["flat"], s["flat"])):
                rows = cache.transpose(1, 2)[seq[:, None], n].transpose(1, 2)      # (pages, H, page, d)
                pool[flat] = torch.where(valid[..., None], rows, pool[flat])
            return s["pools"]
        scale, dtype, B, H = c["dim_head"] ** -0.5, s["pools"][0].dtype, c["batch"], c["heads"]
        qc, kc, vc, qu, ku, vu = (t[:, :, 0].float() for t in s["new"])          # (B, H, d)
        U_pool, qu_pool, kc_pool, vc_pool = s["pools"]
        gate = torch.sigmoid((qu_pool[s["flat"]].float() * (ku * scale)[seq][:, :, None]).sum(-1))
        U_old = U_pool[s["u_flat"]]
        U = (U_old.float() + gate[..., None] * vu[seq][:, :, None]).to(dtype)
        U_pool[s["u_flat"]] = torch.where(valid[..., None], U, U_old)
        q = (qc * scale)[seq][:, :, None]
        su = (U.float() * q).sum(-1)
        score = (kc_pool[s["flat"]].float() * q).sum(-1) - su * torch.sigmoid(su)
        score = torch.where(valid, score, -math.inf)                               # (pages, H, page)
        own_score = (qc * kc).sum(-1) * scale                                      # (B, H): the new row's
        width = s["table"].shape[1]
        most = torch.full((B, width, H), -math.inf, device="cuda")
        most[seq, s["nth"]] = score.amax(-1)
        most = torch.maximum(most.amax(1), own_score)
        e, e_own = torch.exp(score - most[seq][..., None]), torch.exp(own_score - most)
        total, acc = torch.zeros((B, width, H), device="cuda"), torch.zeros((B, width, H, c["dim_head"]), device="cuda")
        total[seq, s["nth"]] = e.sum(-1)
        acc[seq, s["nth"]] = (e[..., None] * torch.where(valid[..., None], vc_pool[s["flat"]], 0).float()).sum(2)
        out = (acc.sum(1) + e_own[..., None] * vc) / (total.sum(1) + e_own)[..., None]
        last = s["lengths"].long() % page
        U_pool[s["u_last"], :, last] = 0
        for pool, new in zip(s["pools"][1:], (s["new"][3], s["new"][1], s["new"][2])):
            pool[s["last"], :, last] = new[:, :, 0]
        return {"out": out[:, :, None].to(dtype), "pools": s["pools"]}


def exact(case, seed):
    """The definitions in 64 bits, a sequence at a time."""
    s, c = prepare(case, seed), case
    with torch.no_grad():
        if c["kind"] == "linear":
            group = torch.arange(c["in"], device="cuda") // c["group"]
            w = s["codes"].double() - (8.0 if s["zeros"] is None else s["zeros"].double()[:, group])
            w *= s["scales"].double()[:, group]
            y = torch.nn.functional.linear(s["x"].double(), w)
            return {"y": y, "dx": torch.einsum("rn,nk->rk", s["grad"].double(), w)} if c["train"] else y
        if c["kind"] == "copy":
            want = []
            for p in s["pools"]:
                from_ = torch.arange(c["pages"], device="cuda")
                from_[s["target_gpu"]] = s["source_gpu"]
                want.append(p.index_select(0, from_).double())
            return want
        page, lengths = c["page"], _lengths(c)
        pools = [p.double() for p in s["pools"]]
        tables = [s["u_table"].long(), s["table"].long(), s["table"].long(), s["table"].long()]

        def places(i, b, count):
            r = torch.arange(count, device="cuda")
            return tables[i][b][r // page], r % page

        if c["kind"] == "write":
            for b, n in enumerate(lengths):
                for i, cache in enumerate(s["caches"]):
                    p, r = places(i, b, n)
                    pools[i][p, :, r] = cache[b, :, :n].transpose(0, 1).double()
            return pools
        new = [t[:, :, 0].double() for t in s["new"]]
        scale, out = c["dim_head"] ** -0.5, []
        for b, n in enumerate(lengths):
            qc, kc, vc, qu, ku, vu = (t[b] for t in new)
            for i, row in enumerate((torch.zeros_like(qu), qu, kc, vc)):
                p, r = places(i, b, n + 1)
                pools[i][p[-1], :, r[-1]] = row
            rows = []
            for i in range(4):
                p, r = places(i, b, n + 1)
                rows.append(pools[i][p, :, r].transpose(0, 1))                     # (H, n + 1, d)
            U = rows[0][:, :n] + torch.sigmoid(torch.einsum("hnd,hd->hn", rows[1][:, :n], ku) * scale)[..., None] * vu[:, None]
            p, r = places(0, b, n)
            pools[0][p, :, r] = U.transpose(0, 1)
            # the scores are those of the lookahead keys as they are kept, in the caches' type
            su = torch.einsum("hnd,hd->hn", U.to(s["pools"][0].dtype).double(), qc) * scale
            score = torch.einsum("hnd,hd->hn", rows[2], qc) * scale
            score[:, :n] -= torch.nn.functional.silu(su)
            out.append(torch.einsum("hn,hnd->hd", torch.softmax(score, -1), rows[3]))
        return {"out": torch.stack(out)[:, :, None], "pools": pools}


def work(case):
    """Bytes with every input read and every output written once, and the flops that the definitions take.  A step reads four rows of
    each position and writes one; a product reads half a byte and a share of its group's parameters for each weight."""
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["kind"] == "linear":
        params = c["out"] * ((c["in"] + c["group"] - 1) // c["group"]) * (2 if c["zeros"] else 1)
        return {"bytes": c["out"] * c["in"] / 2 + size * (params + c["rows"] * (c["in"] + c["out"]) * (2 if c["train"] else 1)),
                "flops": 2 * c["rows"] * c["out"] * c["in"] * (2 if c["train"] else 1)}
    row = c["heads"] * c["dim_head"]
    if c["kind"] == "copy":
        return {"bytes": 2 * size * c["pools"] * c["copied"] * c["page"] * row, "flops": 0}
    rows = sum(_lengths(c))
    if c["kind"] == "write":
        return {"bytes": 8 * size * rows * row, "flops": 0}
    return {"bytes": size * row * (5 * rows + 11 * c["batch"]) + 8 * sum(n // c["page"] + 1 for n in _lengths(c)), "flops": 10 * rows * row}
