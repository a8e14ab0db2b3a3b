"""The paged 4-bit K/V cache without a GPU: the oracle's format, struct layouts, refusals."""
import ctypes
import subprocess

import pytest
import torch

from oracle import kv4
from physisserve_b200 import _lib, ops
from physisserve_b200.build import INCLUDE, build

BASE = 1 << 40


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


# ---------------------------------------------------------------------------------------
# The oracle's format
# ---------------------------------------------------------------------------------------
def test_scale_values_are_e4m3():
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(kv4.E4M3, want)


@pytest.mark.parametrize("x,code", [(0.25, 0), (0.2500001, 1), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6),
                                    (5.0, 6), (5.1, 7), (6.0, 7), (9.0, 7), (0.0, 0)])
def test_codes_round_to_nearest_even(x, code):
    assert int(kv4.nearest(torch.tensor([x], dtype=torch.float64), kv4.E2M1)) == code


def test_quantisation_error_is_within_half_a_step():
    """|x - value| <= half the widest step of its code (1 in code units, up to the scale's own rounding of at
    most 1/16 below max/6) times the scale: |x| <= 6.4 steps after the scale was rounded, so at most 1 step."""
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)).bfloat16()
    codes, scales = kv4.quantise(x, 1.0)
    back = kv4.dequantise(codes, scales, 1.0)
    step = kv4.E4M3[scales.long()].repeat_interleave(16, -1)
    assert bool(((x.double() - back).abs() <= step).all())
    again = kv4.quantise(back.float(), 1.0)
    assert torch.equal(kv4.dequantise(*again, 1.0), back)   # what the cache stands for is stored unchanged


# ---------------------------------------------------------------------------------------
# Layouts
# ---------------------------------------------------------------------------------------
STRUCTS = {"ps_kv4_cache": _lib.PsKv4Cache, "ps_kv4_prep_args": _lib.PsKv4PrepArgs, "ps_kv4_read_args": _lib.PsKv4ReadArgs,
           "ps_kv4_attn_args": _lib.PsKv4AttnArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = []
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {field}));' for field, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "physis_b200_kv4.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(INCLUDE), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, field).offset for field, _ in cls._fields_]
    assert got == want


def test_packed_arguments_match_the_layouts():
    assert ops._PREP4.size == ctypes.sizeof(_lib.PsKv4PrepArgs)
    assert ops._READ4.size == ctypes.sizeof(_lib.PsKv4ReadArgs)
    assert ops._ATTN4.size == ctypes.sizeof(_lib.PsKv4AttnArgs)
    assert ops._ATTN4_WORKSPACE == _lib.PsKv4AttnArgs.workspace.offset
    for name, offset in ops._PREP4_OFFSETS.items():
        assert offset == getattr(_lib.PsKv4PrepArgs, name).offset


# ---------------------------------------------------------------------------------------
# Refusals (fake addresses, never followed: validation makes no CUDA call)
# ---------------------------------------------------------------------------------------
def cache(**change):
    c = dict(pages=BASE, table=BASE, num_pages=40, members=2, table_pages=10, kv_heads=4, page_rows=16, k_scale=1.0,
             v_scale=1.0)
    c.update(change)
    return _lib.PsKv4Cache(**c)


CACHE_FAULTS = [
    (dict(pages=None), "NULL"), (dict(table=None), "NULL"), (dict(pages=BASE + 8), "ALIGN"),
    (dict(table=BASE + 2), "ALIGN"), (dict(page_rows=48), "SHAPE"), (dict(page_rows=256), "SHAPE"),
    (dict(page_rows=0), "SHAPE"), (dict(kv_heads=0), "SHAPE"), (dict(num_pages=0), "SHAPE"),
    (dict(num_pages=1 << 31), "SHAPE"), (dict(members=0), "SHAPE"), (dict(table_pages=0), "SHAPE"),
    (dict(k_scale=0.0), "SHAPE"), (dict(v_scale=-1.0), "SHAPE"), (dict(v_scale=float("nan")), "SHAPE"),
    (dict(k_scale=float("inf")), "SHAPE"),
]


def prep(cache_=None, seq=None, **change):
    seqs = (_lib.PsSeq * 1)(_lib.PsSeq(*(seq or (0, 12, 2, 3, 0, 0, 0, 4, 0, 0, 0))))
    a = dict(dtype=_lib.BF16, heads=4, head_dim=128, table_mode=_lib.TABLE_AXES, t_dim=44, h_dim=42, w_dim=42, n_seqs=1,
             eps=1e-6, launch=_lib.LAUNCH_PDL, in_rows=12, q=BASE, q_stride=512, k=BASE, k_stride=512, v=BASE,
             v_stride=512, q_weight=BASE, k_weight=BASE, cos=BASE, sin=BASE, table_rows=64, q_out=BASE, q_out_stride=512,
             cache=cache_ or cache(), seqs=ctypes.cast(seqs, ctypes.c_void_p))
    a.update(change)
    args = _lib.PsKv4PrepArgs(**a)
    args._keep = seqs
    return args


def read(cache_=None, **change):
    a = dict(dtype=_lib.BF16, row0=3, rows=100, k_out=BASE, k_member_stride=51200, k_row_stride=512, v_out=BASE,
             v_member_stride=51200, v_row_stride=512, cache=cache_ or cache())
    a.update(change)
    return _lib.PsKv4ReadArgs(**a)


def attn(cache_=None, **change):
    a = dict(heads=8, q_tokens=5, kv_tokens=160, q=BASE, q_member_stride=5120, q_row_stride=1024, out=BASE,
             out_member_stride=5120, out_row_stride=1024, cache=cache_ or cache())
    a.update(change)
    return _lib.PsKv4AttnArgs(**a)


def refused(lib, fn, args, status):
    rc = getattr(lib, fn)(ctypes.byref(args))
    assert _lib.STATUS_NAMES[rc] == f"PS_ERR_{status}", lib.ps_error_message()
    assert lib.ps_error_message()


@pytest.mark.parametrize("make,fn", [(prep, "ps_kv4_prep_validate"), (read, "ps_kv4_read_validate"),
                                     (attn, "ps_kv4_attention_validate")])
def test_bad_caches_are_refused(lib, make, fn):
    assert getattr(lib, fn)(ctypes.byref(make())) == _lib.OK, lib.ps_error_message()
    assert getattr(lib, fn)(None) == _lib.ERR_NULL
    for change, status in CACHE_FAULTS:
        refused(lib, fn, make(cache(**change)), status)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), "DTYPE"), (dict(weight_f32=2), "DTYPE"), (dict(head_dim=64), "UNSUPPORTED"), (dict(heads=0), "UNSUPPORTED"),
    (dict(heads=121, q_stride=121 * 128, q_out_stride=121 * 128), "UNSUPPORTED"),
    (dict(dtype=_lib.F32, heads=81, q_stride=81 * 128, q_out_stride=81 * 128), "UNSUPPORTED"),
    (dict(n_seqs=0), "SHAPE"), (dict(n_seqs=65), "TOO_MANY_SEQS"), (dict(seqs=None), "NULL"), (dict(launch=3), "SHAPE"),
    (dict(q=None, k=None, v=None, q_weight=None, k_weight=None), "NULL"), (dict(q=None), "SHAPE"), (dict(k=None), "SHAPE"),
    (dict(q=BASE + 4), "ALIGN"), (dict(q_stride=504), "SHAPE"), (dict(k_stride=516), "ALIGN"), (dict(v_stride=100), "SHAPE"),
    (dict(q_out=None), "NULL"), (dict(k_pre=BASE, k_pre_stride=8), "SHAPE"), (dict(cos=None), "NULL"), (dict(sin=BASE + 4), "ALIGN"),
    (dict(table_rows=0), "SHAPE"), (dict(table_mode=2), "SHAPE"), (dict(t_dim=43, h_dim=43), "SHAPE"), (dict(w_dim=40), "SHAPE"),
    (dict(in_rows=11), "BOUNDS"), (dict(table_rows=1), "BOUNDS"), (dict(eps=-1.0), "SHAPE"),
    (dict(q_weight=BASE + 8), "ALIGN"), (dict(in_rows=-1), "SHAPE"),
])
def test_prep_refusals(lib, change, status):
    refused(lib, "ps_kv4_prep_validate", prep(**change), status)


@pytest.mark.parametrize("seq,status", [
    ((0, 13, 2, 3, 0, 0, 0, 4, 0, 0, 0), "SHAPE"),       # not whole frames
    ((0, 12, 0, 3, 0, 0, 0, 4, 0, 0, 0), "SHAPE"),
    ((-1, 12, 2, 3, 0, 0, 0, 4, 0, 0, 0), "BOUNDS"),
    ((1, 12, 2, 3, 0, 0, 0, 4, 0, 0, 0), "BOUNDS"),
    ((0, 12, 2, 3, 63, 0, 0, 4, 0, 0, 0), "BOUNDS"),     # frame 64 of a 64-row table
    ((0, 12, 2, 3, 0, 0, 0, 0, 0, 0, 0), "BOUNDS"),      # no ring
    ((0, 12, 2, 3, 0, 0, 0, 4, 4, 0, 0), "BOUNDS"),      # slot outside the ring
    ((0, 12, 2, 3, 0, 0, 0, 1, 0, 0, 0), "BOUNDS"),      # two frames in a ring of one
    ((0, 12, 2, 3, 0, 0, 297, 4, 0, 0, 0), "BOUNDS"),    # rows 297 .. 320 of 320: one row too far
    ((0, 12, 2, 3, 0, 0, -1, 4, 0, 0, 0), "BOUNDS"),
    ((0, 12, 2, 3, 0, 0, 1 << 62, 4, 0, 0, 0), "BOUNDS"),
    ((0, 12, 2, 3, 0, 0, 0, 4, 0, 5, 0), "SHAPE"),       # unknown kind
    ((0, 12, 2, 3, 0, 0, 0, 4, 0, 1, 0), "NULL"),        # a sink without k_sink
])
def test_prep_sequence_refusals(lib, seq, status):
    refused(lib, "ps_kv4_prep_validate", prep(seq=seq), status)


def test_prep_accepts_the_last_ring_rows(lib):
    assert lib.ps_kv4_prep_validate(ctypes.byref(prep(seq=(0, 12, 2, 3, 62, 0, 296, 4, 3, 0, 0)))) == _lib.OK


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), "DTYPE"), (dict(row0=-1), "BOUNDS"), (dict(rows=-1), "BOUNDS"), (dict(row0=61), "BOUNDS"),
    (dict(row0=1 << 62), "BOUNDS"), (dict(k_out=None, v_out=None), "NULL"), (dict(k_out=BASE + 8), "ALIGN"),
    (dict(k_row_stride=500), "SHAPE"), (dict(v_row_stride=516, v_member_stride=51600), "ALIGN"), (dict(k_member_stride=51199), "SHAPE"),
    (dict(k_member_stride=51204), "ALIGN"),
])
def test_read_refusals(lib, change, status):
    refused(lib, "ps_kv4_read_validate", read(**change), status)


@pytest.mark.parametrize("change,status", [
    (dict(heads=6), "SHAPE"), (dict(heads=0), "SHAPE"), (dict(q_tokens=-1), "SHAPE"), (dict(kv_tokens=-1), "SHAPE"),
    (dict(kv_tokens=161), "BOUNDS"), (dict(causal_block=-1), "SHAPE"), (dict(kernel=3), "SHAPE"), (dict(key_chunks=65), "SHAPE"),
    (dict(q=None), "NULL"), (dict(q=BASE + 2), "ALIGN"), (dict(q_row_stride=1016), "SHAPE"), (dict(q_member_stride=5000), "SHAPE"),
    (dict(out_row_stride=1028, out_member_stride=8000), "ALIGN"), (dict(kv_lens=BASE + 1), "ALIGN"),
])
def test_attention_refusals(lib, change, status):
    refused(lib, "ps_kv4_attention_validate", attn(**change), status)


def test_attention_refuses_more_work_than_a_grid_holds(lib):
    big = attn(q_tokens=1 << 29)
    big.cache.members = 1 << 24
    big.cache.kv_heads, big.heads = 1024, 1024
    big.q_row_stride = big.out_row_stride = 1024 * 128
    big.q_member_stride = big.out_member_stride = (1 << 29) * 1024 * 128
    assert lib.ps_kv4_attention_validate(ctypes.byref(big)) == _lib.ERR_UNSUPPORTED


def test_attention_without_its_workspace_is_refused_before_any_launch(lib):
    """ps_attention_kv4 itself checks the workspace on the host; the size is what the query reports."""
    big = cache(table_pages=1000, num_pages=5000)
    args = attn(big, kv_tokens=16000, key_chunks=4)
    need = ctypes.c_int64(0)
    assert lib.ps_kv4_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == _lib.OK
    assert need.value > 0
    args.workspace, args.workspace_bytes = BASE, need.value - 1
    assert lib.ps_attention_kv4(ctypes.byref(args), None) == _lib.ERR_NULL
    args.workspace, args.workspace_bytes = BASE + 8, need.value
    assert lib.ps_attention_kv4(ctypes.byref(args), None) == _lib.ERR_ALIGN


def test_empty_calls_return_before_any_launch(lib):
    seq = (0, 0, 2, 3, 0, 0, 0, 4, 0, 0, 0)
    assert lib.ps_qk_norm_rope_kv4(ctypes.byref(prep(seq=seq)), None) == _lib.OK
    assert lib.ps_kv4_read(ctypes.byref(read(rows=0)), None) == _lib.OK
    assert lib.ps_attention_kv4(ctypes.byref(attn(q_tokens=0)), None) == _lib.OK


def test_wrappers_refuse_cpu_tensors_and_bad_pools():
    pages, table = ops.kv4_pages(3, 2, 16), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ops.PrepError, match="CUDA"):
        ops.read_kv4(pages, table, 4)
    with pytest.raises(ops.PrepError, match="page_rows"):
        ops.kv4_pages(3, 2, 48)
    with pytest.raises(ops.PrepError, match="int32"):
        ops.read_kv4(pages, table.long(), 4)
    with pytest.raises(ops.PrepError, match="uint8"):
        ops.read_kv4(pages.int(), table, 4)
    with pytest.raises(ops.PrepError, match="bytes a head"):
        ops.read_kv4(pages[..., :100].contiguous(), table, 4)


# ---------------------------------------------------------------------------------------
# The pool of the Wan ring caches
# ---------------------------------------------------------------------------------------
def test_pool_hands_out_every_page_once_and_takes_them_back():
    from physisserve_b200.wan import Kv4Pool, RingCache4

    pool = Kv4Pool(7, 2, page_rows=16)
    a, b = (RingCache4(heads=2, grid_h=2, grid_w=5, capacity=4, sink_frames=2, batch=n, pool=pool) for n in (1, 2))
    assert a.rows == 64 and b.rows == 64 and a.window_rows(0) == 20 and a.window_rows(9) == 60
    a.reserve([20])
    b.reserve([16, 33])
    assert pool.free_pages == 1
    held = [int(p) for cache in (a, b) for p in cache.table.flatten() if p >= 0]
    assert len(held) == len(set(held)) == 6
    a.reserve([20])                      # nothing more is needed
    assert pool.free_pages == 1
    with pytest.raises(ops.PrepError, match="free pages"):
        b.reserve([64, 64])
    assert pool.free_pages == 1          # a refused reservation takes nothing
    b.release()
    assert pool.free_pages == 5 and bool((b.table == -1).all())
    a.reserve([60])
    assert pool.free_pages == 3 and [int(p) for p in a.table[0, :2]] == held[:2]


def test_pool_takes_back_only_what_it_gave():
    from physisserve_b200.wan import Kv4Pool

    pool = Kv4Pool(4, 1, page_rows=16)
    held = pool.take(2)
    for bad in ([held[0], held[0]], [3 if 3 not in held else 0], [7]):
        with pytest.raises(ops.PrepError, match="held"):
            pool.give(bad)
    pool.give(held)
    with pytest.raises(ops.PrepError, match="held"):
        pool.give(held[:1])
    assert sorted(pool.take(4)) == [0, 1, 2, 3]


def test_ring_cache_refuses_other_heads():
    from physisserve_b200.wan import Kv4Pool, RingCache4

    with pytest.raises(ops.PrepError, match="128"):
        RingCache4(heads=2, head_dim=64, grid_h=2, grid_w=5)
    with pytest.raises(ops.PrepError, match="heads"):
        RingCache4(heads=2, grid_h=2, grid_w=5, pool=Kv4Pool(4, 3))


# ---------------------------------------------------------------------------------------
# The workspace of the tiles kernel
# ---------------------------------------------------------------------------------------
def test_tiles_workspace_has_room_from_any_16_byte_boundary(lib):
    """A query row's partial results (128 sums, a reference and a sum of weights) for 256 rows of the first and
    the last unit of each CTA, 16 bytes for each unit, all behind the first 32-byte boundary: the kernel stores 32
    bytes at a time.  1,000 steps are more than the grid of 148 CTAs needs."""
    args = attn(cache(table_pages=1000, num_pages=5000), kv_tokens=16000, kernel=_lib.KV4_TILES)
    need = ctypes.c_int64(0)
    assert lib.ps_kv4_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == _lib.OK
    assert need.value == 2 * 148 * 256 * (128 * 4 + 8) + 2 * 4 * 16 + 16
    for offset in (0, 16):
        args.workspace, args.workspace_bytes = BASE + offset, need.value - 1
        assert lib.ps_attention_kv4(ctypes.byref(args), None) == _lib.ERR_NULL
    args.workspace, args.workspace_bytes = BASE + 8, need.value
    assert lib.ps_attention_kv4(ctypes.byref(args), None) == _lib.ERR_ALIGN


def test_attention_refuses_columns_beyond_32_bits(lib):
    for heads, want in (((1 << 24) - 4, _lib.OK), (1 << 24, _lib.ERR_UNSUPPORTED)):
        wide = attn(heads=heads, q_tokens=1, q_row_stride=heads * 128, q_member_stride=heads * 128, out_row_stride=heads * 128,
                    out_member_stride=heads * 128)
        assert lib.ps_kv4_attention_validate(ctypes.byref(wide)) == want, lib.ps_error_message()


def test_prep_ring_refuses_a_split_that_the_4_bit_cache_does_not_have():
    from physisserve_b200.wan import RingCache4, prep_ring, wan_rope_tables, window_layout

    cache = RingCache4(heads=1, grid_h=2, grid_w=2, capacity=2, sink_frames=1)
    x, w = torch.zeros(1, 4, 128, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    pos = [window_layout(0, first_frames=1)]
    free = cache.pool.free_pages
    with pytest.raises(ops.PrepError, match="heads_per_thread"):
        prep_ring(x, x, x, w, w, 1e-6, *wan_rope_tables(128, 8), cache, pos, heads_per_thread=2)
    assert cache.pool.free_pages == free


def test_pool_gives_two_threads_different_pages():
    """A thread asks for pages while another is in the middle of taking its own."""
    import threading

    from physisserve_b200.wan import Kv4Pool

    pool, other = Kv4Pool(8, 1, page_rows=16), []
    thread = threading.Thread(target=lambda: other.extend(pool.take(3)))

    class Interrupted(list):
        def __getitem__(self, at):
            if not thread.ident:
                thread.start()
                thread.join(0.3)
            return list.__getitem__(self, at)

        def __delitem__(self, at):
            if not thread.ident:
                thread.start()
                thread.join(0.3)
            list.__delitem__(self, at)

    pool._free = Interrupted(pool._free)
    mine = pool.take(3)
    thread.join()
    assert len(set(mine) | set(other)) == 6 and sorted(mine + other + pool.take(2)) == list(range(8))


def test_a_reservation_is_taken_whole_or_not_at_all():
    """Pages that another thread takes between a cache's look at the pool and its taking."""
    from physisserve_b200.wan import Kv4Pool, RingCache4

    class Raced(Kv4Pool):
        def take(self, count):
            if not self._taken:
                Kv4Pool.take(self, 5)
            return Kv4Pool.take(self, count)

    pool = Raced(8, 1, page_rows=16)
    cell = RingCache4(heads=1, grid_h=2, grid_w=4, capacity=4, sink_frames=2, batch=2, pool=pool)
    with pytest.raises(ops.PrepError, match="free pages"):
        cell.reserve([40, 17])
    assert pool.free_pages == 3 and bool((cell.table == -1).all()) and cell._held == [[], []]


def test_a_cache_is_copied_with_its_pool():
    import copy

    from physisserve_b200.wan import RingCache4

    cell = RingCache4(heads=1, grid_h=2, grid_w=4, capacity=4, sink_frames=2, batch=1, page_rows=16)
    cell.reserve([20])
    other = copy.deepcopy(cell)
    other.reserve([40])
    assert cell.pool.free_pages == other.pool.free_pages + 1
    assert torch.equal(cell.table[0, :2], other.table[0, :2]) and cell._held != other._held
