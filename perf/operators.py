"""The operators of a language model around its layers, as cases that can be timed and compared: the lookup of its
tokens, layer norm, and the cross entropy of its head, each with its gradient.

A case's "kind" says which call it is:

    embed          castle_embedding, forward only (serving)
    embed_train    castle_embedding, forward and the table's gradient
    norm           castle_layer_norm, forward only
    norm_train     castle_layer_norm, forward and all gradients
    loss           castle_linear_cross_entropy, forward only (scoring)
    loss_train     castle_linear_cross_entropy, forward and both gradients

"tokens" is the number of rows of the call.  With `own` false `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORED = -100


def _embed(name, dtype, tokens, dim, vocab, train, spread="zipf", padded=0.0):
    return {"name": name, "kind": "embed_train" if train else "embed", "dtype": dtype, "tokens": tokens, "dim": dim, "vocab": vocab,
            "spread": spread, "padded": padded}


def _norm(name, dtype, tokens, dim, train, affine="both"):
    return {"name": name, "kind": "norm_train" if train else "norm", "dtype": dtype, "tokens": tokens, "dim": dim, "affine": affine}


def _loss(name, dtype, tokens, dim, vocab, train, reduction="mean", ignored=0.0):
    return {"name": name, "kind": "loss_train" if train else "loss", "dtype": dtype, "tokens": tokens, "dim": dim, "vocab": vocab,
            "reduction": reduction, "ignored": ignored}


def listed():
    return [
        # The lookup of one token for each of a few sequences: serving, latency alone.
        _embed("embed_token_b8", "bf16", 8, 512, 256, False),
        # The byte language model's training step: 16 x 1024 tokens, 256 rows that each occur some 64 times.
        _embed("embed_train_bytes", "bf16", 16384, 512, 256, True, "uniform"),
        # A ragged batch, a word-piece vocabulary with the frequencies of text, a quarter of it padding.
        _embed("embed_train_50021_fp32", "fp32", 8191, 1000, 50021, True, padded=0.25),
        # A large vocabulary: most of the gradient's rows are zero.
        _embed("embed_train_131072", "bf16", 65536, 2048, 131072, True),
        # The norm of one token of a few sequences.
        _norm("norm_token_fp32", "fp32", 2, 512, False),
        # The norm in front of one layer of the byte language model, training.
        _norm("norm_train_lm_layer", "bf16", 16384, 512, True),
        # Odd in both sizes, without a bias.
        _norm("norm_train_1333_fp16", "fp16", 4099, 1333, True, "weight"),
        # A wide model's norm, larger than the second-level cache.
        _norm("norm_train_32768_4096", "bf16", 32768, 4096, True),
        # Scoring one short sequence, token by token's loss, with the byte vocabulary.
        _loss("loss_score_197_fp32", "fp32", 197, 512, 256, False, "none"),
        # The byte language model's head, training.
        _loss("loss_train_bytes", "bf16", 16384, 512, 256, True),
        # A ragged batch whose prompts are not learnt (half of the targets), fp16 with a loss scale, odd vocabulary.
        _loss("loss_train_50021_fp16", "fp16", 4095, 1024, 50021, True, "sum", ignored=0.5),
        # A large vocabulary under a wide model.
        _loss("loss_train_131072", "bf16", 8192, 4096, 131072, True),
    ]


MOST_EMBED = (65536 + 131072) * 2048      # elements that the largest listed lookup's gradient reads and writes
MOST_NORM = 32768 * 4096
MOST_LOGITS = 8192 * 131072               # logits of the largest listed loss, and its multiply-adds per product
MOST_PRODUCT = MOST_LOGITS * 4096


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _dim(rng, low, high):
    """A model's width: mostly a multiple of 64 or of 8, now and then odd."""
    step = rng.choice([64, 64, 64, 8, 8, 1])
    return max(low, _log_uniform(rng, low, high) // step * step)


def draw(rng):
    kind = rng.choice(["embed", "embed_train", "embed_train", "norm", "norm_train", "norm_train", "loss", "loss_train", "loss_train"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    train = kind.endswith("train")
    tokens = _log_uniform(rng, 1, 65536)
    if kind.startswith("embed"):
        dim, vocab = _dim(rng, 64, 8192), _log_uniform(rng, 100, 200000)
        while (tokens + vocab) * dim * (2 if dtype == "fp32" else 1) > MOST_EMBED:
            tokens, vocab, dim = max(1, tokens * 3 // 4), max(100, vocab * 3 // 4), max(64, dim * 7 // 8)
        c = _embed(None, dtype, tokens, dim, vocab, train, rng.choice(["uniform", "zipf", "zipf"]), rng.choice([0.0, 0.0, 0.3]))
    elif kind.startswith("norm"):
        dim = _dim(rng, 64, 16384)
        while tokens * dim * (2 if dtype == "fp32" else 1) > MOST_NORM:
            tokens = max(1, tokens * 3 // 4)
        c = _norm(None, dtype, tokens, dim, train, rng.choice(["both", "both", "weight", "none"]))
    else:
        tokens, dim, vocab = _log_uniform(rng, 1, 16384), _dim(rng, 64, 8192), _log_uniform(rng, 100, 200000)
        cost = 6 if dtype == "fp32" else 1
        while tokens * vocab > MOST_LOGITS or tokens * vocab * dim * cost > MOST_PRODUCT:
            tokens, vocab = max(1, tokens * 3 // 4), max(100, vocab * 7 // 8)
        c = _loss(None, dtype, tokens, dim, vocab, train, rng.choice(["mean", "mean", "sum", "none"]), rng.choice([0.0, 0.0, 0.5]))
    del c["name"]
    return c


def _tokens(c, gen):
    """Token numbers: uniform ones as of random bytes, or with the frequencies of text, the rank's reciprocal (log-uniform
    ranks), where low numbers are frequent as tokenisers leave it."""
    u = torch.rand(c["tokens"], device="cuda", generator=gen, dtype=torch.float64)
    v = c["vocab"]
    if c.get("spread", "zipf") == "uniform":
        return (u * v).long().clamp_(max=v - 1)
    return (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)


def _randn(shape, dtype, gen, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def prepare(case, seed):
    c, dtype = case, DTYPES[case["dtype"]]
    n, d = c["tokens"], c["dim"]
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"].startswith("embed"):
        s["tokens"] = _tokens(c, gen)
        s["padding"] = None
        if c["padded"]:
            s["padding"] = c["vocab"] - 1
            s["tokens"][torch.rand(n, device="cuda", generator=gen) < c["padded"]] = s["padding"]
        s["weight"] = _randn((c["vocab"], d), dtype, gen, d ** -0.5)
        s["scale"] = d ** 0.5
        if c["kind"] == "embed_train":
            s["weight"].requires_grad_()
            s["grad"] = _randn((n, d), dtype, gen, 1e-2)
    elif c["kind"].startswith("norm"):
        # A residual stream: rows of different size and offset, a few channels much larger than the others.
        size = torch.empty((n, 1), device="cuda").uniform_(0.5, 4.0, generator=gen)
        x = _randn((n, d), torch.float32, gen).mul_(size).add_(_randn((n, 1), torch.float32, gen, 0.5))
        x[:, torch.randint(0, d, (1 + d // 500,), device="cuda", generator=gen)] *= 12.0
        s["x"] = x.to(dtype)
        s["weight"] = (1 + 0.1 * _randn((d,), torch.float32, gen)).to(dtype) if c["affine"] != "none" else None
        s["bias"] = _randn((d,), dtype, gen, 0.1) if c["affine"] == "both" else None
        s["eps"] = 1e-5
        if c["kind"] == "norm_train":
            for t in (s["x"], s["weight"], s["bias"]):
                if t is not None:
                    t.requires_grad_()
            s["grad"] = _randn((n, d), dtype, gen, 1e-2)
    else:
        # Logits of a model that has learnt something: their spread is 2, and half of the targets stand out.
        v = c["vocab"]
        s["weight"] = _randn((v, d), dtype, gen, 2 * d ** -0.5)
        t = _tokens(c, gen)
        known = (torch.rand((n, 1), device="cuda", generator=gen) < 0.5).float()
        s["x"] = (_randn((n, d), torch.float32, gen) + 2 * known * s["weight"][t].float()).to(dtype)
        left_out = torch.rand(n, device="cuda", generator=gen) < c["ignored"]
        left_out[0] = False          # something is learnt in every call, or its mean has no value
        t[left_out] = IGNORED
        s["targets"] = t
        if c["kind"] == "loss_train":
            s["x"].requires_grad_()
            s["weight"].requires_grad_()
            # fp16 gradients want a loss scale: with it those of single tokens are numbers around one
            scale = (float(n) if c["reduction"] == "mean" else 1.0) if c["dtype"] == "fp16" else 1.0
            s["grad"] = torch.full((), scale, device="cuda")
            if c["reduction"] == "none":
                s["grad"] = torch.empty(n, device="cuda").uniform_(0.25, 1.0, generator=gen)
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import lookahead_keys_attention_b200 as castle
    kind = s["case"]["kind"]
    if kind.startswith("embed"):
        y = castle.castle_embedding(s["tokens"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
        if kind == "embed":
            return y
        return {"y": y.detach(), "dweight": torch.autograd.grad(y, [s["weight"]], s["grad"])[0]}
    if kind.startswith("norm"):
        y = castle.castle_layer_norm(s["x"], s["weight"], s["bias"], eps=s["eps"])
        if kind == "norm":
            return y
        leaves = [t for t in (s["x"], s["weight"], s["bias"]) if t is not None]
        return {"y": y.detach(), "grads": torch.autograd.grad(y, leaves, s["grad"])}
    loss = castle.castle_linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORED, reduction=s["case"]["reduction"])
    if kind == "loss":
        return loss
    return {"loss": loss.detach(), "grads": torch.autograd.grad(loss, [s["x"], s["weight"]], s["grad"])}


def _run_plain(s):
    kind = s["case"]["kind"]
    with torch.no_grad():
        if kind.startswith("embed"):
            w, t = s["weight"], s["tokens"]
            y = (w[t].float() * s["scale"]).to(w.dtype)
            if kind == "embed":
                return y
            g = s["grad"].float() * s["scale"]
            if s["padding"] is not None:
                g = g * (t != s["padding"])[:, None]
            dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, t, g)
            return {"y": y, "dweight": dw.to(w.dtype)}
        if kind.startswith("norm"):
            x = s["x"].float()
            centred = x - x.mean(1, keepdim=True)
            rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
            xh = centred * rstd
            y = xh
            if s["weight"] is not None:
                y = y * s["weight"].float()
            if s["bias"] is not None:
                y = y + s["bias"].float()
            y = y.to(s["x"].dtype)
            if kind == "norm":
                return y
            dy = s["grad"].float()
            g = dy if s["weight"] is None else dy * s["weight"].float()
            dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
            grads = [dx.to(s["x"].dtype)]
            if s["weight"] is not None:
                grads.append((dy * xh).sum(0).to(s["weight"].dtype))
            if s["bias"] is not None:
                grads.append(dy.sum(0).to(s["bias"].dtype))
            return {"y": y, "grads": tuple(grads)}
        x, w, t, reduction = s["x"].float(), s["weight"].float(), s["targets"], s["case"]["reduction"]
        learnt = t != IGNORED
        at = torch.where(learnt, t, 0)[:, None]
        z = x @ w.t()
        zt = z.gather(1, at)[:, 0]
        m = z.amax(1, keepdim=True)
        e = torch.exp(z - m)
        total = e.sum(1, keepdim=True)
        loss = torch.where(learnt, (m + torch.log(total))[:, 0] - zt, 0.0)
        count = learnt.sum()
        if reduction == "sum":
            loss = loss.sum()
        elif reduction == "mean":
            loss = loss.sum() / count
        if kind == "loss":
            return loss
        c = s["grad"] / count if reduction == "mean" else s["grad"]
        c = torch.where(learnt, c, 0.0)[:, None]
        e *= c / total
        e.scatter_add_(1, at, -c)
        return {"loss": loss, "grads": ((e @ w).to(s["x"].dtype), (e.t() @ x).to(s["weight"].dtype))}


def exact(case, seed):
    """The definitions in 64 bits."""
    s, kind = prepare(case, seed), case["kind"]
    with torch.no_grad():
        if kind.startswith("embed"):
            w = s["weight"].double()
            y = torch.nn.functional.embedding(s["tokens"], w) * s["scale"]
            if kind == "embed":
                return y
            keep = torch.ones_like(s["tokens"], dtype=torch.bool) if s["padding"] is None else s["tokens"] != s["padding"]
            dw = torch.zeros_like(w)
            dw.index_put_((s["tokens"][keep],), s["grad"].double()[keep] * s["scale"], accumulate=True)
            return {"y": y, "dweight": dw}
        if kind.startswith("norm"):
            x = s["x"].double()
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            sd = torch.sqrt(var + s["eps"])
            w = torch.ones_like(x[0]) if s["weight"] is None else s["weight"].double()
            b = torch.zeros_like(x[0]) if s["bias"] is None else s["bias"].double()
            y = (x - mean) / sd * w + b
            if kind == "norm":
                return y
            dy, d = s["grad"].double(), x.shape[1]
            g = dy * w / sd
            dx = g - (g.sum(1, keepdim=True) + (x - mean) * ((x - mean) * g).sum(1, keepdim=True) / (sd * sd)) / d
            grads = [dx]
            if s["weight"] is not None:
                grads.append((dy * ((x - mean) / sd)).sum(0))
            if s["bias"] is not None:
                grads.append(dy.sum(0))
            return {"y": y, "grads": tuple(grads)}
        x, w, t = s["x"].double(), s["weight"].double(), s["targets"]
        rows = (t != IGNORED).nonzero()[:, 0]
        log_p = torch.log_softmax(x[rows] @ w.t(), 1)
        each = torch.zeros(len(t), dtype=torch.float64, device=x.device)
        each[rows] = -log_p[torch.arange(len(rows), device=x.device), t[rows]]
        loss = {"none": each, "sum": each.sum(), "mean": each.sum() / len(rows)}[case["reduction"]]
        if kind == "loss":
            return loss
        c = s["grad"].double().expand(len(t))[rows] / (len(rows) if case["reduction"] == "mean" else 1)
        g = log_p.exp_()
        g[torch.arange(len(rows), device=x.device), t[rows]] -= 1
        g *= c[:, None]
        dx = torch.zeros_like(x)
        dx[rows] = g @ w
        return {"loss": loss, "grads": (dx, g.t() @ x[rows])}


def work(case):
    """Bytes with every input read and every output written once, and the flops that the definitions take.  A lookup reads as
    many different rows of its table as its tokens can name; rows whose gradient is not wanted (padding) need not be read, rows
    that are not learnt have a gradient of zero and no logits; logits that a backward pass forms again count nothing."""
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    n, d = c["tokens"], c["dim"]
    train = c["kind"].endswith("train")
    if c["kind"].startswith("embed"):
        elements = (n + min(n, c["vocab"])) * d
        if train:
            elements += int(n * (1 - c["padded"])) * d + c["vocab"] * d
        return {"bytes": size * elements + 8 * n, "flops": n * d * (2 if train else 1)}
    if c["kind"].startswith("norm"):
        params = {"both": 2, "weight": 1, "none": 0}[c["affine"]] * d
        return {"bytes": size * (n * d * (5 if train else 2) + params * (2 if train else 1)), "flops": n * d * (20 if train else 7)}
    v = c["vocab"]
    learnt = max(1, int(n * (1 - c["ignored"])))
    product = 2 * learnt * v * d
    elements = (learnt + v) * d + ((n + v) * d if train else 0)
    return {"bytes": size * elements + 8 * n + 4 * (n if c["reduction"] == "none" else 1), "flops": product * (3 if train else 1) + 5 * learnt * v}
