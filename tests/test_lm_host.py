"""CPU: arguments that the entry points of the operators around the layers refuse on the host, before anything is launched."""
import pytest
import torch


def _lib():
    from lookahead_keys_attention_b200 import _lib
    _lib.build()
    return _lib, _lib.load()


def test_layernorm_arguments():
    L, lib = _lib()
    def fwd(dtype=L.BF16, rows=4, dim=16, x=32, stride=16, w=32, b=32, y=32, stats=32):
        return lib.castle_layernorm_fwd(dtype, rows, dim, x, stride, w, b, 1e-5, y, stats, None)
    for bad in [dict(dtype=3), dict(rows=0), dict(rows=2 ** 31), dict(dim=0), dict(dim=2 ** 25), dict(x=None), dict(y=None), dict(stride=-1), dict(x=33),
                dict(w=33), dict(b=1), dict(stats=4)]:
        assert fwd(**bad) < 0 and "castle_layernorm_fwd" in L.last_error(), bad
    size = lib.castle_layernorm_bwd_workspace_bytes(4, 16)
    assert size == 1 * 2 * 16 * 4 and lib.castle_layernorm_bwd_workspace_bytes(0, 16) == 0
    def bwd(dtype=L.F32, rows=4, dim=16, dy=32, x=32, w=32, stats=32, dx=32, dw=32, db=32, ws=32, n=size):
        return lib.castle_layernorm_bwd(dtype, rows, dim, dy, 16, x, 16, w, stats, dx, dw, db, ws, n, None)
    for bad in [dict(dtype=-1), dict(rows=-1), dict(dy=None), dict(x=None), dict(stats=None), dict(dx=2), dict(ws=None), dict(n=size - 1), dict(stats=36)]:
        assert bwd(**bad) < 0 and "castle_layernorm_bwd" in L.last_error(), bad


def test_embedding_arguments():
    L, lib = _lib()
    def fwd(dtype=L.BF16, ib=8, n=4, vocab=10, dim=16, t=32, w=32, stride=16, y=32, status=32):
        return lib.castle_embedding_fwd(dtype, ib, n, vocab, dim, t, w, stride, 1.0, y, status, None)
    for bad in [dict(dtype=7), dict(ib=2), dict(n=0), dict(n=2 ** 31), dict(vocab=0), dict(vocab=2 ** 31), dict(dim=0), dict(t=None), dict(t=36), dict(w=None),
                dict(w=33), dict(stride=-2), dict(y=None), dict(status=None)]:
        assert fwd(**bad) < 0 and "castle_embedding_fwd" in L.last_error(), bad
    size = lib.castle_embedding_bwd_workspace_bytes(4, 10, 16)
    assert size > 0 and lib.castle_embedding_bwd_workspace_bytes(4, 0, 16) == 0
    def bwd(dtype=L.BF16, ib=4, n=4, vocab=10, dim=16, t=32, dy=32, stride=16, dw=32, ws=32, size=size, status=32):
        return lib.castle_embedding_bwd(dtype, ib, n, vocab, dim, t, -1, dy, stride, 1.0, dw, ws, size, status, None)
    for bad in [dict(dtype=-1), dict(ib=16), dict(n=-5), dict(dy=None), dict(dy=33), dict(dw=None), dict(ws=None), dict(ws=40), dict(size=size - 1), dict(status=None)]:
        assert bwd(**bad) < 0 and "castle_embedding_bwd" in L.last_error(), bad


@pytest.mark.parametrize("padding", [-2, 10, 2 ** 32 - 1, 2 ** 32 + 5, -2 ** 32 + 5, 2 ** 63 - 1, -2 ** 63])
def test_padding_outside_the_table_is_refused(padding):
    """Cut to 32 bits, 2^32 + 5 would be row 5, whose gradient would be left out."""
    L, lib = _lib()
    size = lib.castle_embedding_bwd_workspace_bytes(4, 10, 16)
    assert lib.castle_embedding_bwd(L.BF16, 8, 4, 10, 16, 32, padding, 32, 16, 1.0, 32, 32, size, 32, None) < 0
    assert f"padding_idx {padding}" in L.last_error()


def test_embedding_limits():
    """Places in the sorted list are 32 bits: 2^30 tokens at most, and no scratch is named for what would be refused."""
    L, lib = _lib()
    size = lib.castle_embedding_bwd_workspace_bytes
    assert size(2 ** 30, 1536 * 2048, 1) > 2 ** 32
    assert size(2 ** 30 + 1, 10, 1) == size(2 ** 31 - 1, 10, 1) == size(4, 1536 * 2048 + 1, 1) == size(4, 2 ** 62, 1) == 0
    for n in (2 ** 30 + 1, 2 ** 31 - 1):
        assert lib.castle_embedding_fwd(L.BF16, 8, n, 10, 1, 32, 32, 1, 1.0, 32, 32, None) < 0
        assert lib.castle_embedding_bwd(L.BF16, 8, n, 10, 1, 32, -1, 32, 1, 1.0, 32, 32, 2 ** 40, 32, None) < 0
        assert "castle_embedding_bwd" in L.last_error()


def test_cpu_tensors_are_refused():
    from lookahead_keys_attention_b200 import castle_embedding, castle_layer_norm
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_layer_norm(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(4, 8))


def test_linear_ce_arguments():
    L, lib = _lib()
    size = [lib.castle_linear_ce_workspace_bytes(L.BF16, 4, 16, 10, b) for b in (0, 1)]
    assert min(size) > 0
    for bad in [(5, 4, 16, 10), (0, 0, 16, 10), (0, 4, 0, 10), (0, 4, 16, 0), (0, 2 ** 31, 16, 10), (0, 4, 2 ** 21, 10), (0, 4, 16, 2 ** 31)]:
        assert lib.castle_linear_ce_workspace_bytes(*bad, 1) == 0
    def fwd(dtype=L.BF16, n=4, dim=16, vocab=10, x=256, xs=16, w=256, ws=16, t=256, red=0, loss=256, lse=256, work=256, size=size[0], status=256):
        return lib.castle_linear_ce_fwd(dtype, n, dim, vocab, x, xs, w, ws, t, -100, red, loss, lse, work, size, status, None)
    for bad in [dict(dtype=3), dict(n=0), dict(dim=0), dict(vocab=-1), dict(x=None), dict(x=257), dict(xs=-1), dict(w=None), dict(ws=-1), dict(t=None), dict(t=260),
                dict(red=3), dict(red=-1), dict(loss=None), dict(lse=None), dict(lse=2), dict(work=None), dict(work=128), dict(size=size[0] - 1), dict(status=None)]:
        assert fwd(**bad) < 0 and "castle_linear_ce_fwd" in L.last_error(), bad
    def bwd(dtype=L.BF16, n=4, dim=16, vocab=10, lse=256, dloss=256, dx=256, dw=256, work=256, size=size[1]):
        return lib.castle_linear_ce_bwd(dtype, n, dim, vocab, 256, 16, 256, 16, 256, -100, 0, lse, dloss, dx, dw, work, size, 256, None)
    for bad in [dict(dtype=-1), dict(n=-1), dict(lse=None), dict(dloss=None), dict(dloss=6), dict(dx=1), dict(dw=3), dict(work=None), dict(size=size[1] - 1)]:
        assert bwd(**bad) < 0 and "castle_linear_ce_bwd" in L.last_error(), bad
    assert bwd(dx=None, dw=None) == 0          # nothing wanted, nothing launched


def test_the_losses_scratch_is_bounded():
    """About 1 GiB for a piece of the vocabulary beside what goes with the rows, whatever the vocabulary."""
    L, lib = _lib()
    for dtype, planes in ((L.BF16, 1), (L.F32, 3)):
        for n, dim, vocab in [(8192, 4096, 1 << 20), (65536, 512, 300000), (16384, 8192, 200000)]:
            for backward in (0, 1):
                rows = planes * (n + 64) * dim * 2 + n * 64
                slabs = n * dim * 4 * 32 * backward
                assert lib.castle_linear_ce_workspace_bytes(dtype, n, dim, vocab, backward) <= (1 << 30) * 1.1 + rows + slabs


def test_reduction_names():
    from lookahead_keys_attention_b200 import castle_linear_cross_entropy
    with pytest.raises(ValueError, match="reduction"):
        castle_linear_cross_entropy(torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(2, dtype=torch.int64), reduction="avg")
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_linear_cross_entropy(torch.zeros(2, 8), torch.zeros(3, 8), torch.zeros(2, dtype=torch.int64))


def test_prenorm_names():
    from lookahead_keys_attention_b200 import Castle
    for name in ("layernorm", "Layer", "rms", ""):          # not an RMSNorm, as any true value would give
        with pytest.raises(ValueError, match="prenorm"):
            Castle(16, heads=1, dim_head=16, prenorm=name)
    for value, norm in ((False, torch.nn.Identity), (None, torch.nn.Identity), (0, torch.nn.Identity), (True, torch.nn.RMSNorm), (1, torch.nn.RMSNorm),
                        ("layer", torch.nn.LayerNorm)):
        assert type(Castle(16, heads=1, dim_head=16, prenorm=value).norm) is norm
