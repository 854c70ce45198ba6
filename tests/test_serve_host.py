"""CPU: arguments that the entry points of serving from a paged cache refuse on the host, before anything is launched."""
import ctypes

import pytest
import torch


def _lib():
    from lookahead_keys_attention_b200 import _lib
    _lib.build()
    return _lib, _lib.load()


def _problem(L, **kw):
    a = dict(batch=2, heads=4, seq_len=20, dim_head=64, dtype=L.BF16, scale=0.125)
    a.update({k: v for k, v in kw.items() if k in a})
    return L.CastleProblem(*a.values())


def _paged(L, lib, name, **kw):
    """The call with addresses that are never followed, and what differs from a good one."""
    a = dict(page_size=16, u_pages=10, pages=10, width=4, u_table=256, table=256, u_stride=4, stride=4, lengths=256, status=256, counters=256, ws=256, size=None,
             row=256, row_stride=64, pool=256, page_stride=4096, head_stride=1024, freqs=0, freqs_type=L.F32)
    p = _problem(L, **kw)
    a.update({k: v for k, v in kw.items() if k in a})
    rows = ctypes.byref(L.CastleTensor(a["row"], a["row_stride"], 64, 64))
    pool = ctypes.byref(L.CastlePages(a["pool"], a["page_stride"], a["head_stride"]))
    tables = (a["u_table"], a["u_stride"], a["table"], a["stride"], a["width"], a["lengths"])
    if name == "castle_write_pages":
        return lib.castle_write_pages(ctypes.byref(p), a["page_size"], a["u_pages"], a["pages"], *[rows] * 4, *[pool] * 4, *tables, a["status"], None)
    size = lib.castle_paged_decode_workspace_bytes(ctypes.byref(p), a["page_size"], a["width"]) if a["size"] is None else a["size"]
    rotary = ctypes.byref(L.CastleRotary(a["freqs"], a["freqs_type"], 0, 0))
    return lib.castle_paged_decode_step(ctypes.byref(p), a["page_size"], a["u_pages"], a["pages"], *[rows] * 6, *[pool] * 4, *tables, rows, rotary, a["counters"],
                                        a["ws"], size, a["status"], None)


COMMON = [dict(batch=0), dict(heads=0), dict(dtype=3), dict(dtype=-1), dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(u_pages=0), dict(pages=-1), dict(width=0),
          dict(u_table=None), dict(table=None), dict(table=258), dict(lengths=None), dict(lengths=257), dict(status=None), dict(u_stride=-1), dict(stride=-1),
          dict(row=None), dict(row=264), dict(row_stride=63), dict(pool=None), dict(pool=8), dict(page_stride=4095), dict(head_stride=4), dict(width=2 ** 30)]


@pytest.mark.parametrize("bad", COMMON + [dict(batch=4097), dict(dim_head=48), dict(dim_head=256), dict(counters=None), dict(counters=2), dict(ws=None), dict(ws=2), dict(size=1),
                                          dict(freqs=256, freqs_type=5), dict(batch=4096, heads=1 << 20, width=1 << 20)], ids=str)
def test_step_arguments(bad):
    L, lib = _lib()
    assert _paged(L, lib, "castle_paged_decode_step", **bad) < 0 and L.last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(seq_len=0), dict(dim_head=4), dict(dim_head=1 << 14), dict(batch=1 << 20, heads=1 << 20)], ids=str)
def test_write_arguments(bad):
    L, lib = _lib()
    assert _paged(L, lib, "castle_write_pages", **bad) < 0 and L.last_error()


def test_write_of_positions_at_the_end_of_32_bits():
    L, lib = _lib()
    assert _paged(L, lib, "castle_write_pages", batch=1, heads=1, seq_len=2 ** 31 - 1000) < 0 and "too many" in L.last_error()


def test_workspace_grows_with_what_a_call_may_hold():
    L, lib = _lib()
    size = lambda width, **kw: lib.castle_paged_decode_workspace_bytes(ctypes.byref(_problem(L, **kw)), 64, width)  # noqa: E731
    sizes = [size(w) for w in (1, 2, 10, 100, 1000, 10000, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert size(1 << 20, batch=64, heads=16) <= 592 * 2 * 68 * 4      # bounded, however wide the tables are
    assert size(0) == 0 and size(4, dim_head=80) == 0 and size(4, batch=5000) == 0


def _copy(lib, pools=1, ptr=(256,), page=(64,), block=(0,), blocks=1, block_bytes=64, pages=10, source=(1,), target=(2,), count=None):
    i64, i32 = (lambda v: (ctypes.c_int64 * len(v))(*v)), (lambda v: (ctypes.c_int32 * len(v))(*v))
    return lib.castle_copy_pages(pools, (ctypes.c_void_p * len(ptr))(*ptr), i64(page), i64(block), blocks, block_bytes, pages, i32(source), i32(target),
                                 len(source) if count is None else count, None)


@pytest.mark.parametrize("bad", [dict(pools=-1), dict(count=-1), dict(blocks=0), dict(block_bytes=0), dict(block_bytes=24), dict(ptr=(0,)), dict(ptr=(264,)), dict(page=(72,)),
                                 dict(block=(8,)), dict(source=(10,)), dict(source=(-1,)), dict(target=(10,)), dict(source=(1, 2), target=(3, 3)),
                                 dict(source=(1, 2), target=(3, 1)), dict(source=(1,), target=(1,)), dict(blocks=1 << 40),
                                 dict(pools=2, ptr=(256, 256), page=(64, 64), block=(0, 0))], ids=str)
def test_copy_arguments(bad):
    L, lib = _lib()
    assert _copy(lib, **bad) < 0 and "castle_copy_pages" in L.last_error()


def test_copies_of_many_pages():
    """A target twice and a target that is a source are found among any number of pairs, and named."""
    import random
    L, lib = _lib()
    for seed, count in enumerate((1, 2, 3, 17, 64, 65, 1000, 5000)):
        rng = random.Random(seed)
        pages = rng.sample(range(2 ** 31 - 1 if seed % 2 else 3 * count), 2 * count)
        source, target = [rng.choice(pages[:count]) for _ in range(count)], pages[count:]
        at, both = rng.randrange(count), rng.choice(source)
        assert _copy(lib, pages=2 ** 31 - 1, source=source, target=target[:at] + [both] + target[at + 1:]) < 0 and f"page {both} is a target and a source" in L.last_error()
        if count > 1:
            twice = rng.choice(target[:-1])
            assert _copy(lib, pages=2 ** 31 - 1, source=source, target=target[:-1] + [twice]) < 0 and f"page {twice} is a target twice" in L.last_error()


def test_page_numbers():
    from lookahead_keys_attention_b200.ops import _page_numbers
    for pages in ([3, 1, 2 ** 31], (5,), range(4), [True], [torch.tensor(7)], []):
        t = _page_numbers(pages)
        assert t.dtype == torch.int64 and t.device.type == "cpu" and t.tolist() == [int(p) for p in pages]
    with pytest.raises(TypeError):
        _page_numbers([1.5])


def test_nothing_to_copy_is_fine():
    L, lib = _lib()
    assert _copy(lib, source=(), target=()) == 0 and _copy(lib, pools=0) == 0


def test_cpu_tensors_are_refused():
    from lookahead_keys_attention_b200 import castle_copy_pages, castle_paged_decode_step, castle_write_pages
    rows, pool, table = torch.zeros(1, 2, 1, 64), torch.zeros(4, 2, 16, 64), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_paged_decode_step(*[rows] * 6, *[pool] * 4, table, table, table[:, 0], 0.125)
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_write_pages(*[rows] * 4, *[pool] * 4, table, table, table[:, 0])
    with pytest.raises(RuntimeError, match="no CPU path"):
        castle_copy_pages(pool, [0], [1])


def test_polls_of_the_self_test():
    L, lib = _lib()
    for bad in (-2, 65537):
        assert lib.castle_selftest_paged_polls(bad) < 0 and "castle_selftest_paged_polls" in L.last_error()
    assert lib.castle_selftest_paged_polls(0) == 0 and lib.castle_selftest_paged_polls(-1) == 0
