"""CPU: the codes' layout, the quantisation, and the arguments that products with weights of 4 bits refuse on the host."""
import pytest
import torch


def _lib():
    from lookahead_keys_attention_b200 import _lib
    _lib.build()
    return _lib, _lib.load()


def _unpack(packed, n, k):
    """By the layout's description in the C ABI's header, a code at a time."""
    out = torch.empty(n, k, dtype=torch.int64)
    for r in range(n):
        tile, half, g = r // 16, r % 16 // 8, r % 8
        for i in range(k):
            block, rest = divmod(i, 128)
            j, t, o = rest // 32, rest % 32 // 8, rest % 8
            word = int(packed[tile, block * 256 + half * 128 + (g * 4 + t) * 4 + j]) & 0xffffffff
            out[r, i] = word >> (4 * (o // 2) + 16 * (o % 2)) & 15
    return out


@pytest.mark.parametrize("n,k,dtype", [(3, 128, torch.uint8), (5, 1, torch.int64), (33, 300, torch.int32), (1, 127, torch.uint8)])
def test_layout(n, k, dtype):
    from lookahead_keys_attention_b200 import castle_pack_4bit
    codes = torch.randint(0, 16, (n, k), generator=torch.Generator().manual_seed(k)).to(dtype)
    packed = castle_pack_4bit(codes)
    assert packed.dtype == torch.int32 and packed.shape == ((n + 15) // 16, (k + 255) // 256 * 512) and packed.is_contiguous()
    assert torch.equal(_unpack(packed, n, k), codes.long())


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_weights(zeros, dtype):
    """Every weight is at most half a step (and the rounding of scale and zero point: 16 steps times their half units) from its value."""
    from lookahead_keys_attention_b200 import castle_quantize_4bit
    gen = torch.Generator().manual_seed(1)
    w = (torch.randn(20, 200, generator=gen) * torch.rand(20, 1, generator=gen)).to(dtype)
    w[0], w[1, :64], w[2, 64:] = 0, 0.5, -w[2, 64:].abs()
    codes, scales, zp = castle_quantize_4bit(w, 64, zeros)
    assert scales.shape == (20, 4) and scales.dtype == dtype and (zp is None) == (not zeros)
    at = torch.arange(200) // 64
    back = (_unpack(codes, 20, 200).double() - (zp.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    unit = torch.finfo(dtype).eps / 2
    size = (15 + (zp.double().abs()[:, at] if zeros else 0)) * unit
    assert bool(((back - w.double()).abs() <= scales.double()[:, at] * (0.5 + 2 * size)).all())


@pytest.mark.parametrize("zeros", [False, True])
def test_weights_at_the_types_ends(zeros):
    """The largest weights have finite scales; weights that are not finite are refused."""
    from lookahead_keys_attention_b200 import castle_quantize_4bit
    top = torch.finfo(torch.float32).max
    w = torch.linspace(-1, 1, 64).repeat(2, 1) * top
    codes, scales, zp = castle_quantize_4bit(w, 64, zeros)
    assert bool(scales.isfinite().all())
    back = (_unpack(codes, 2, 64).double() - (zp.double() if zeros else 8.0)) * scales.double()
    # (half a step, and the roundings of 15 steps)
    assert bool(((back - w.double()).abs() <= scales.double() * (0.5 + 1e-4)).all())
    for bad in (float("nan"), float("inf"), -float("inf")):
        w = torch.zeros(2, 64)
        w[1, 5] = bad
        with pytest.raises(ValueError, match="finite"):
            castle_quantize_4bit(w, 64, zeros)


def test_arguments():
    L, lib = _lib()
    good = dict(dtype=L.BF16, rows=2, k=200, n=10, group=64, x=256, stride=200, codes=256, scales=256, zeros=256, y=256, status=256)
    def call(**kw):
        a = {**good, **kw}
        return lib.castle_linear_4bit(*a.values(), None)
    for bad in [dict(dtype=3), dict(rows=0), dict(rows=33), dict(k=0), dict(k=(1 << 24) + 1), dict(n=0), dict(n=2 ** 31), dict(group=16), dict(group=48), dict(group=0), dict(x=None),
                dict(x=257), dict(stride=-1), dict(codes=None), dict(codes=264), dict(scales=None), dict(scales=1), dict(zeros=3), dict(y=None), dict(y=255), dict(status=None), dict(status=2), dict(dtype=L.F32, rows=11)]:
        assert call(**bad) < 0 and "castle_linear_4bit" in L.last_error(), bad
    tile = dict(dtype=L.BF16, rows=100, k=200, n=10, group=64, x=256, stride=200, codes=256, scales=256, zeros=None, y=256, status=256)
    for bad in [dict(dtype=L.F32), dict(rows=0), dict(rows=2 ** 31), dict(k=0), dict(n=0), dict(group=24), dict(x=None), dict(x=264), dict(stride=196), dict(stride=192), dict(codes=8),
                dict(scales=None), dict(scales=1), dict(zeros=3), dict(y=None), dict(y=1), dict(status=None)]:
        a = {**tile, **bad}
        assert lib.castle_linear_4bit_tile(*a.values(), None) < 0 and "castle_linear_4bit_tile" in L.last_error(), bad
    wide = dict(dtype=L.BF16, k=200, n=10, group=64, codes=256, scales=256, zeros=None, w=256, stride=200)
    for bad in [dict(dtype=-1), dict(k=0), dict(n=-1), dict(group=33), dict(codes=8), dict(w=None), dict(w=264), dict(stride=192), dict(stride=204)]:
        a = {**wide, **bad}
        assert lib.castle_expand_4bit(*a.values(), None) < 0 and "castle_expand_4bit" in L.last_error(), bad


def test_what_fits():
    L, lib = _lib()
    assert all(lib.castle_linear_4bit_fits(L.BF16, r, 4096) == 1 for r in (1, 8, 32)) and lib.castle_linear_4bit_fits(L.F32, 10, 4096) == 1
    assert lib.castle_linear_4bit_fits(L.BF16, 32, 1 << 20) == 0 and lib.castle_linear_4bit_fits(L.F32, 11, 64) == 0 and lib.castle_linear_4bit_fits(7, 1, 64) == 0


def test_refusals_of_the_host():
    from lookahead_keys_attention_b200 import castle_linear_4bit, castle_pack_4bit, castle_quantize_4bit
    codes, scales, _ = castle_quantize_4bit(torch.randn(4, 64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_linear_4bit(torch.zeros(1, 64), codes, scales)
    for bad in (lambda: castle_pack_4bit(torch.zeros(4)), lambda: castle_pack_4bit(torch.zeros(4, 4)), lambda: castle_quantize_4bit(torch.zeros(4, 4, dtype=torch.int32)),
                lambda: castle_quantize_4bit(torch.zeros(4, 4), 40)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64])
def test_codes_of_more_or_other_bits_are_refused(dtype):
    """Signed codes, or ones of five bits, are not wrapped into others; the ends of 0 to 15 are taken."""
    from lookahead_keys_attention_b200 import castle_pack_4bit
    codes = torch.tensor([[0, 15], [15, 0], [7, 8]], dtype=dtype)
    assert torch.equal(_unpack(castle_pack_4bit(codes), 3, 2), codes.long())
    for bad in ([16, 255, 31] if dtype == torch.uint8 else [16, -1, -8, 127]):
        wrong = codes.clone()
        wrong[1, 1] = bad
        with pytest.raises(ValueError, match="0 to 15"):
            castle_pack_4bit(wrong)
    assert castle_pack_4bit(codes[:0]).shape == (0, 512) and castle_pack_4bit(codes[:, :0]).shape == (1, 0)
    with pytest.raises(ValueError):
        castle_pack_4bit(codes.to(torch.complex64))
