"""Operator layer: the CASTLE attention core as torch-facing functions.  The work between a call and
the C-ABI library's launches (descriptors, scratch, the passes around the kernels, the autograd node)
is native, in csrc/host.cpp; this file holds the operators' contracts and limits.

`castle_attention` mirrors the reference operator
`castle_attention_triton(qc, kc, vc, qu, ku, vu, scale, return_U_for_cache)`
(lookahead_keys_attention/lookahead_keys_attention_triton.py:416-605): same
argument order (causal triple first), unscaled inputs, returns `out` or
`(out, U)`, six input gradients, no gradient through U.
`castle_decode_step` replaces the single-token branch of the reference module
(lookahead_keys_attention/lookahead_keys_attention.py:166-203).
"""
from __future__ import annotations

from array import array

import torch

from . import _lib
from ._lib import CastleTensor


def _device_index(device) -> int:
    device = torch.device(device)
    return torch.cuda.current_device() if device.index is None else device.index


def status_word(device) -> torch.Tensor:
    """Per-device int32 the kernels OR error bits into (0 = fine)."""
    return _lib.host().status_word(_device_index(device))


def check_status(device=None):
    """Synchronising check of the device status word; raises on a kernel-side failure."""
    devs = [_device_index(device)] if device is not None else _lib.host().status_devices()
    for d in devs:
        w = status_word(torch.device("cuda", d))
        v = int(w.item())
        if v != 0:
            w.zero_()
            raise RuntimeError(f"castle kernels reported status {v} on cuda:{d} (1 = a bounded wait ran out, "
                               "4 = a token or target outside the vocabulary, or a length or page outside its table or pool)")


def release_workspaces():
    """Free every cached scratch buffer (one per device and stream, grown on demand and kept between
    calls; they are re-created on the next call)."""
    _lib.host().release_workspaces()


def _desc(t: torch.Tensor) -> CastleTensor:
    """(B, H, N, d) tensor or view with a contiguous last dim -> castle_tensor_t, for callers of the C ABI."""
    assert t.dim() == 4 and (t.stride(3) == 1 or t.shape[3] == 1)
    return CastleTensor(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


# Bound on the forward's scratch per launch.  The soft-max partials take N^2/128 * (8 + 2*d) bytes
# per (batch, head) pair (O(N^2), where the reference kernel needs O(N*d)), so a call is cut into
# launches over whole batch rows, or over head ranges of one batch row, that each stay below it.
MAX_WORKSPACE_BYTES = 16 << 30


def forward_chunks(B: int, H: int, per_pair: int, limit: int | None = None):
    """Rectangles (b0, b1, h0, h1) of the (batch, head) grid that a forward is launched over, each needing at most
    `limit` bytes of scratch at `per_pair` bytes per pair.  A rectangle spans several batch rows only with all heads,
    so that the per-pair fp32 buffers (lse, state) of a rectangle stay contiguous.  (csrc/host.cpp, for_chunks.)"""
    return _lib.host().forward_chunks(B, H, per_pair, MAX_WORKSPACE_BYTES if limit is None else limit)


# From this sequence length on, bf16 callers are computed with fp16 operands.  The lookahead state W grows
# like sqrt(N) (|W| ~ 100 at N = 8192) and the gate's and the state's 16-bit copies are what the long-range
# gradients are made of: with 8 significant bits dqc misses |a-b| <= 2e-2 + 1e-2|b| from N ~ 8192 on, with
# fp16's 11 bits it holds at N = 16384.  (The tensor cores cannot mix an fp16 operand with a bf16 one in a
# single product, so the inputs are converted once instead; at these lengths that pass is < 1 % of the work.)
# fp32 callers run with fp16 operands at every length (as the reference operator does,
# lookahead_keys_attention_triton.py:437-442).
# Costs: values beyond +-65504 in q/k/v saturate, and the upstream gradient is rescaled by a power of two
# (exactly) so that small gradients do not underflow.
LONG_SEQ_FP16 = 6144


class _Traced(torch.autograd.Function):
    """An operator while torch.jit.trace is recording: a Python autograd function becomes a node of the traced graph,
    which calls it again when the graph runs; of the native operator the tracer would only see the allocations."""

    @staticmethod
    def forward(ctx, packed_op, scale, return_U, *inputs):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_(t.requires_grad) for t in inputs]
            limits = (scale, return_U, None, MAX_WORKSPACE_BYTES, LONG_SEQ_FP16)
            host = _lib.host()
            result = host.attention_packed(*leaves, *limits, None, True) if packed_op else host.attention(*leaves, *limits)
            ctx.anchors = _anchors(inputs)
        out, *U = result if return_U else (result,)
        ctx.graph = leaves, out
        if return_U:
            ctx.mark_non_differentiable(*U)
        return (out.detach(), *U) if return_U else out.detach()

    @staticmethod
    def backward(ctx, grad, *_):
        leaves, out = ctx.graph
        wanted = [t for t in leaves if t.requires_grad]
        grads = iter(_refuse_second(torch.autograd.grad(out, wanted, grad, retain_graph=True), (grad, *ctx.anchors)))
        return (None, None, None, *(next(grads) if t.requires_grad else None for t in leaves))


class _TracedCall(torch.autograd.Function):
    """The same for an operator with one result: `call(*inputs)`."""

    @staticmethod
    def forward(ctx, call, *inputs):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_(t.requires_grad) if isinstance(t, torch.Tensor) else t for t in inputs]
            out = call(*leaves)
            ctx.anchors = _anchors(inputs)
        ctx.graph = leaves, out
        return out.detach()

    @staticmethod
    def backward(ctx, grad):
        leaves, out = ctx.graph
        wanted = [t for t in leaves if isinstance(t, torch.Tensor) and t.requires_grad]
        grads = iter(_refuse_second(torch.autograd.grad(out, wanted, grad, retain_graph=True), (grad, *ctx.anchors)))
        return (None, *(next(grads) if isinstance(t, torch.Tensor) and t.requires_grad else None for t in leaves))


def _anchors(inputs):
    """Nothing of each differentiable input, by which its place in the graph can be kept."""
    return [t.narrow(0, 0, 0) for t in inputs if isinstance(t, torch.Tensor) and t.requires_grad]


def _refuse_second(grads, inputs):
    """The gradients that a traced operator's own graph gave, under create_graph behind a node that refuses second derivatives
    (what `refuse_second` of csrc/host.cpp does for the native nodes)."""
    inputs = [t for t in inputs if t.requires_grad]
    if not torch.is_grad_enabled() or not inputs:
        return grads
    refuse = torch._C._functions.DelayedError("castle: second derivatives are not implemented", len(grads) + len(inputs))
    return refuse(*(g.detach() for g in grads), *inputs)[:len(grads)]


def castle_attention_packed(packed, scale, return_U_for_cache=False, cache_out=None):
    """Parallel CASTLE attention on the packed projection output (B, N, 6, H, d), order
    qu,ku,vu,qc,kc,vc (the layout `to_all_qkv` produces).  Returns out (B, H, N, d) [, U].
    With `cache_out` = four (B, H, N, d) views (U, qu, kc, vc) of decode-cache buffers, the
    kernels write the cache rows themselves and the returned U is cache_out[0].
    Its gradient is the packed buffer the backward kernels write, so autograd has nothing to
    scatter or sum (six separate view-gradients cost ~10 extra passes)."""
    if torch._C._is_tracing() and cache_out is None:
        return _Traced.apply(True, float(scale), bool(return_U_for_cache), packed)
    return _lib.host().attention_packed(packed, scale, return_U_for_cache, cache_out, MAX_WORKSPACE_BYTES, LONG_SEQ_FP16,
                                        None, True)


def castle_attention(qc, kc, vc, qu, ku, vu, scale, return_U_for_cache=False, cache_out=None):
    """Parallel CASTLE attention on (B, H, N, d) tensors (views are fine).
    Returns `out`, or `(out, U)` when `return_U_for_cache`; `cache_out` as in `castle_attention_packed`."""
    if torch._C._is_tracing() and cache_out is None:
        return _Traced.apply(False, float(scale), bool(return_U_for_cache), qc, kc, vc, qu, ku, vu)
    return _lib.host().attention(qc, kc, vc, qu, ku, vu, scale, return_U_for_cache, cache_out, MAX_WORKSPACE_BYTES,
                                 LONG_SEQ_FP16)


def castle_decode_step(qc, kc, vc, qu, ku, vu, U, qu_cache, kc_cache, vc_cache, cache_len: int, scale: float):
    """One cached token.  The four caches are (B, H, capacity, d) buffers with `cache_len`
    valid rows; they are updated IN PLACE (row `cache_len` appended, U[0:cache_len] rewritten).
    The six new-token tensors are (B, H, 1, d).  Returns out (B, H, 1, d)."""
    return _lib.host().decode_step(qc, kc, vc, qu, ku, vu, U, qu_cache, kc_cache, vc_cache, cache_len, scale)


def castle_embedding(tokens, weight, scale: float = 1.0, padding_idx: int | None = None):
    """Rows of `weight` (vocabulary, dim) at `tokens` (any shape, int64 or int32), times `scale` (rounded once): the input of a
    language model around these layers (the reference's training script embeds its bytes, train_triton.py:73-175).
    The gradient of `weight` is dense and the same from call to call: every row's gradients are summed in the order of
    their positions, in fp32.  Tokens equal to `padding_idx` are looked up like others and contribute no gradient.  A token
    outside the vocabulary gives a row of NaN and no gradient, and `check_status()` raises."""
    if padding_idx is not None:
        vocab = weight.shape[0]
        if not -vocab <= padding_idx < vocab:
            raise ValueError("castle_embedding: padding_idx out of range")
        padding_idx %= vocab
    padding = -1 if padding_idx is None else padding_idx
    if torch._C._is_tracing():
        return _TracedCall.apply(lambda t, w: _lib.host().embedding(t, w, scale, padding), tokens, weight)
    return _lib.host().embedding(tokens, weight, scale, padding)


def castle_layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Layer norm over the last dimension of `x` (any size), with an optional weight and bias of its type: mean, variance and
    all sums in fp32, one rounding.  Under autocast weight and bias may have another type than `x` and are cast to its.
    `Castle(..., prenorm="layer")` has it in front of the layer."""
    if torch._C._is_tracing():
        return _TracedCall.apply(lambda *t: _lib.host().layer_norm(*t, eps), x, weight, bias)
    return _lib.host().layer_norm(x, weight, bias, eps)


_REDUCTIONS = {"mean": 0, "sum": 1, "none": 2}   # CASTLE_REDUCE_* of the C ABI


def castle_linear_cross_entropy(x, weight, targets, ignore_index: int = -100, reduction: str = "mean"):
    """Cross entropy of the logits `x @ weight.T` against `targets`, without the logits in memory: the head and the loss of a
    language model around these layers (the reference's training script, train_triton.py:73-175).  x (..., dim) and weight
    (vocabulary, dim) of one type (under autocast weight is cast to x's), targets (...) int64 or int32; the loss is fp32, logits and sums are, too.  Rows whose target is
    `ignore_index` take no part, whatever x holds there, and cost nothing; `reduction`: the mean of the others (NaN if there are
    none, with gradients of zero), their "sum", or "none" for each row's loss (0 where ignored).  The gradients of x and weight are formed in the backward
    pass, from logits formed again, and are the same from call to call.  A target outside the vocabulary gives NaN, and `check_status()` raises."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"castle_linear_cross_entropy: reduction {reduction!r} is not one of {', '.join(_REDUCTIONS)}")
    code = _REDUCTIONS[reduction]
    if torch._C._is_tracing():
        return _TracedCall.apply(lambda x, w, t: _lib.host().linear_cross_entropy(x, w, t, ignore_index, code), x, weight, targets)
    return _lib.host().linear_cross_entropy(x, weight, targets, ignore_index, code)


def _not_traced(who):
    """Operators that write their caller's tensors: of the call a tracer would record nothing."""
    if torch._C._is_tracing():
        raise RuntimeError(f"{who}: cannot be traced")


def castle_paged_decode_step(qc, kc, vc, qu, ku, vu, U_pages, qu_pages, kc_pages, vc_pages, U_table, table, lengths, scale: float):
    """`castle_decode_step` for sequences of different lengths whose caches lie in pages.  The six new-token tensors are
    (B, H, 1, d); the four pools (pages, H, page size, d), a head's rows of a page adjacent, page size a power of two from 16 to
    1024 (U's pool may have another number of pages than the others).  `lengths` (B) int32: the positions of each sequence, of which
    position k is row k % page size of page `table[b, k // page size]` (int32), for U of page `U_table[b, k // page size]`.  All
    of them are read on the device: a captured step can be replayed as they change.

    The pools are updated IN PLACE: U of every position rewritten, a row appended at position `lengths[b]`, whose page must be in the
    tables (`lengths` stay as they are).  So a page of U, and the page that gets the new row, must belong to one sequence of the
    batch; other pages of qu, kc and vc may be shared.  A negative length means no sequence: nothing is read or written for it, and its
    row of the result is zero.  A length that the tables have no place for, or a page outside its pool, gives NaN, and `check_status()`
    raises.  Returns out (B, H, 1, d)."""
    _not_traced("castle_paged_decode_step")
    return _lib.host().paged_decode_step(qc, kc, vc, qu, ku, vu, U_pages, qu_pages, kc_pages, vc_pages, U_table, table, lengths, scale)


def castle_write_pages(U, qu, kc, vc, U_pages, qu_pages, kc_pages, vc_pages, U_table, table, lengths):
    """A prompt's caches (B, H, N, d), as `Castle(..., return_next_cache=True)` returns them, into pages: the first `lengths[b]`
    (int32, at most N; none where negative) rows of each sequence, pools and tables as in `castle_paged_decode_step`."""
    _not_traced("castle_write_pages")
    _lib.host().write_pages(U, qu, kc, vc, U_pages, qu_pages, kc_pages, vc_pages, U_table, table, lengths)


def _page_numbers(pages):
    if isinstance(pages, torch.Tensor):
        return pages
    numbers = array("q", pages)   # (torch.tensor takes 43 us for a list of 900, this 14)
    return torch.frombuffer(numbers, dtype=torch.int64) if numbers else torch.empty(0, dtype=torch.int64, device="cpu")


def castle_copy_pages(pools, source, target):
    """Pages `source[i]` to `target[i]` of a (pages, ...) pool, or of each of a list of pools of one shape, type and device, in place: what a
    fork of a sequence or a compaction of its pages moves.  A page is a multiple of 16 bytes.  `source` and `target` are lists, or
    int64 or int32 tensors on the host (a CUDA graph keeps the pages it was captured with); a target that is a source too, or a target twice, is refused."""
    _not_traced("castle_copy_pages")
    pools = [pools] if isinstance(pools, torch.Tensor) else list(pools)
    _lib.host().copy_pages(pools, _page_numbers(source), _page_numbers(target))


def castle_pack_4bit(codes):
    """(out, in) codes of 0 to 15, of any integer type and on any device, as `castle_linear_4bit` takes them: eight to an int32 (their order: the C
    ABI's header), (ceil(out / 16), ceil(in / 256) * 512).  Other codes are refused (to signed ones, -8 to 7, add 8)."""
    if codes.dim() != 2 or codes.is_floating_point() or codes.is_complex() or codes.dtype == torch.bool:
        raise ValueError("castle_pack_4bit: (out, in) integer codes expected")
    if codes.numel():
        low, high = (int(v) for v in codes.aminmax())
        if low < 0 or high > 15:
            raise ValueError(f"castle_pack_4bit: codes from {low} to {high}, where 0 to 15 are expected")
    n, k = codes.shape
    tiles, blocks = (n + 15) // 16, (k + 255) // 256 * 2                               # (of 128 k)
    padded = torch.full((tiles * 16, blocks * 128), 8, dtype=torch.int32, device=codes.device)
    padded[:n, :k] = codes
    padded = padded.view(tiles, 2, 8, blocks, 4, 4, 8)                              # half, row; block, 32 k, 8 k of these, k
    word = torch.zeros((tiles, 2, 8, blocks, 4, 4), dtype=torch.int32, device=codes.device)
    for i in range(8):
        word |= padded[..., i] << (4 * (i // 2) + 16 * (i % 2))
    return word.permute(0, 3, 1, 2, 5, 4).reshape(tiles, blocks * 256)


def castle_quantize_4bit(weight, group_size: int = 64, zeros: bool = False):
    """(out, in) weights to the nearest of 16 values for each group of `group_size` (a power of two from 32 up) weights of a row: (codes, scales, zero points)
    for `castle_linear_4bit`.  Without zero points the values are scale * {-8 .. 7}, with them scale * ({0 .. 15} - zero), the least to the
    largest weight of the group.  Scales and zero points have the weights' type."""
    if weight.dim() != 2 or weight.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("castle_quantize_4bit: (out, in) weights in bf16, fp16 or fp32 expected")
    if group_size < 32 or group_size & (group_size - 1):
        raise ValueError(f"castle_quantize_4bit: group_size {group_size} is not a power of two from 32 up")
    with torch.no_grad():
        n, k = weight.shape
        groups = (k + group_size - 1) // group_size
        w = weight.float()
        if not bool(w.isfinite().all()):
            raise ValueError("castle_quantize_4bit: a weight is not finite")
        padded = torch.nn.functional.pad(w, (0, groups * group_size - k))             # (a value of zero is among the others' range below)
        inside = (torch.arange(groups * group_size, device=w.device) < k).view(groups, group_size)
        grouped = padded.view(n, groups, group_size)
        high = torch.where(inside, grouped, -torch.inf).amax(-1)
        low = torch.where(inside, grouped, torch.inf).amin(-1)
        scale = high / 15 - low / 15 if zeros else torch.maximum(high / 7, -low / 8)
        scale = scale.to(weight.dtype)
        scale = torch.where(scale > 0, scale, torch.ones_like(scale))                 # (all of a group alike, or too small for the type)
        zero = (-low / scale.float()).to(weight.dtype) if zeros else None
        codes = grouped / scale.float()[..., None] + (zero.float()[..., None] if zeros else 8.0)
        codes = codes.round().clamp(0, 15).to(torch.uint8).view(n, groups * group_size)[:, :k]
    return castle_pack_4bit(codes), scale, zero


def castle_linear_4bit(x, codes, scales, zeros=None, group_size: int = 64):
    """`x @ W.T` for weights of 4 bits: W[n, k] = scales[n, k // group_size] * (code[n, k] - zeros[n, k // group_size]), with zero points of 8 where there are
    none.  x (..., in); `codes` of `castle_pack_4bit` or `castle_quantize_4bit`; scales and zero points (out, ceil(in / group_size)) of x's type (under autocast they
    are cast to it), group_size a power of two from 32 up.  For a few rows (up to 8, and up to 32, of 32 bits any number, where that is faster) the codes are read as they are, the weights are not rounded, and sums
    are fp32; many rows are products with the weights rounded to x's type (and code - zero before that, where it is no whole number).  The gradient of x
    is a product with the weights at full width; the weights are frozen.  An infinity in x may give NaN in place of
    an infinity (for 16-bit rows, and with zero points)."""
    if torch._C._is_tracing():
        return _TracedCall.apply(lambda *t: _lib.host().linear_4bit(*t, group_size), x, codes, scales, zeros)
    return _lib.host().linear_4bit(x, codes, scales, zeros, group_size)
