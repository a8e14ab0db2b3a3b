"""GPU tests of the paged 4-bit K/V cache (include/physis_b200_kv4.h) against the 64-bit restatement in
oracle/kv4.py.

Append: everything that is quantised is reproduced bit for bit (the sum of squares is accumulated in 64
bits, every later step is an IEEE fp32 operation), so codes and scales have to be equal.  Q is rounded from
an fp32 sum of another order: within one bf16 ulp, as in the ring's tests.

Read: code * scale has 6 significant bits and is exact; times the tensor scale it is rounded once: within half
a step of the output type (bf16 2^-8, fp32 2^-24 relative).

Attention, per output element, with p the probabilities and A = sum p |v| (sum p = 1): the output's rounding to
bf16, 2^-8 |out|; each p's rounding to fp16, 2^-11 relative and so 2^-11 A; each score's fp32 accumulation over
128 products (128 * 2^-24 * sum |q k| / sqrt(128), below 2^-14 for |q k| sums up to 2^8 * sqrt(128)) and the
approximate 2^x (2^-22), together below 2^-13 A; a p below fp16's normal range loses at most 2^-25 absolutely
against a largest p of at least 1, N keys together 2^-25 N max|v|.  Tolerance: 2^-8 |out| + 2^-10 A + 2^-24 N max|v|.
"""
import ctypes

import pytest
import torch

from oracle import kv4, wan_prep
from physisserve_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make_table(members, table_pages, spare, seed):
    """(number of pages, table): distinct pages in random order, `spare` pages that nobody owns."""
    n = members * table_pages + spare
    return n, torch.randperm(n, generator=gen(seed))[:members * table_pages].view(members, table_pages).int()


def fill(members, rows, heads, page_rows, seed, k_scale=1.0, v_scale=1.0, extra_pages=1, k_size=1.0):
    """(pages, table, k fp64, v fp64): a cache filled by the oracle, unowned and unwritten rows full of 0xff
    (scale bytes that would read as NaN)."""
    table_pages = -(-rows // page_rows) + extra_pages
    n, table = make_table(members, table_pages, 2, seed)
    pages = torch.full((n, heads, 2, page_rows * 72), 0xff, dtype=torch.uint8)
    g = gen(seed + 1)
    back = []
    for which, scale in ((0, k_scale), (1, v_scale)):
        x = torch.randn(members * rows, heads, 128, generator=g) * (k_size if which == 0 else 1.0)
        flat = (torch.arange(members)[:, None] * table_pages * page_rows + torch.arange(rows)).flatten()
        kv4.store(pages, table, flat, x, which, scale)
        back.append(kv4.load(pages, table, flat, which, scale).view(members, rows, heads, 128))
    return pages, table, back[0], back[1]


# ---------------------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------------------
def append_case(streams, gh, gw, frames, heads, hk, page_rows, dtype, ring, seed, k_scale=1.0, v_scale=0.375,
                fused=False, w32=False, size=1.0, mode="axes"):
    hw, C, Ck = gh * gw, heads * 128, hk * 128
    n = hw * frames
    T = streams * n
    g = gen(seed)
    qkv = (torch.randn(T, C + 2 * Ck, generator=g) * size).to(dtype)
    wdt = torch.float32 if w32 else dtype
    wq, wk = ((torch.rand(c, generator=g) + 0.5).to(wdt) for c in (C, Ck))
    cos, sin = wan_prep.rope_tables(128, 256)
    table_pages = -(-ring * hw // page_rows)
    pages_n, table = make_table(streams, table_pages, 2, seed)
    pages = torch.randint(0, 256, (pages_n, hk, 2, page_rows * 72), generator=g, dtype=torch.uint8)
    offsets = torch.randint(0, 100, (streams,), generator=g).tolist()
    slots = torch.randint(0, ring, (streams,), generator=g).tolist()
    seqs, flat, cos_t, sin_t = [], [], [], []
    for b in range(streams):
        base = b * table_pages * page_rows
        seqs.append(ops.Seq(b * n, n, gh, gw, offsets[b], b * n, base, ring, slots[b]))
        f = torch.arange(n) // hw
        flat.append(base + ((slots[b] + f) % ring) * hw + torch.arange(n) % hw)
        c, s = wan_prep.frames_table(cos, sin, wan_prep.axis_dims(128), offsets[b], offsets[b] + frames, gh, gw)
        cos_t.append(c[0, :, 0])
        sin_t.append(s[0, :, 0])
    cos_t, sin_t, flat = torch.cat(cos_t), torch.cat(sin_t), torch.cat(flat)

    dev = qkv.to(DEV)
    q, k, v = dev.split((C, Ck, Ck), 1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    tables = (cos, sin) if mode == "axes" else (cos_t.contiguous(), sin_t.contiguous())
    got_pages, q_out = pages.to(DEV), torch.empty(T, C, dtype=dtype, device=DEV)
    kwargs = dict(heads=heads, kv_heads=hk, seqs=seqs, cos=tables[0].to(DEV), sin=tables[1].to(DEV), q=q, k=k, v=v,
                  q_weight=wq.to(DEV), k_weight=wk.to(DEV), eps=1e-6, q_out=q_out, pages=got_pages, table=table.to(DEV),
                  k_scale=k_scale, v_scale=v_scale, table_mode=mode)

    want = pages.clone()
    qn, kn = kv4.rms_norm(qkv[:, :C], wq, 1e-6), kv4.rms_norm(qkv[:, C:C + Ck], wk, 1e-6)
    q_ref = wan_prep.rope(qn.view(1, T, heads, 128), cos_t[None, :, None], sin_t[None, :, None])[0].flatten(1)
    k_rot = wan_prep.rope(kn.view(1, T, hk, 128), cos_t[None, :, None], sin_t[None, :, None])[0]
    kv4.store(want, table, flat, k_rot, 0, k_scale)
    kv4.store(want, table, flat, qkv[:, C + Ck:].view(T, hk, 128), 1, v_scale)
    return kwargs, want, q_ref, kn


def check_q(got, want, dtype):
    if dtype == torch.bfloat16:
        ulps = wan_prep.bf16_ulp_distance(got.cpu(), want)
        assert int(ulps.max()) <= 1 or float((ulps > 1).float().mean()) < 1e-3
        assert float((ulps > 0).float().mean()) <= 1e-3
    else:  # the fp32 sum's order: a few 2^-24 of the row's size
        err = (got.cpu().double() - want.double()).abs().max()
        assert float(err) <= 2 ** -20 * float(want.double().abs().max())


APPENDS = [
    # streams, grid, frames, heads, kv_heads, page_rows, dtype, ring frames
    (1, 1, 1, 1, 1, 1, 16, torch.bfloat16, 1),          # one token, one head
    (3, 1, 1, 1, 12, 12, 128, torch.bfloat16, 5),       # a decoding step
    (2, 5, 7, 2, 12, 12, 16, torch.bfloat16, 3),        # ring wraps; frames end inside a page
    (2, 5, 7, 2, 12, 4, 32, torch.bfloat16, 2),         # shared K/V heads
    (1, 6, 8, 1, 40, 40, 64, torch.bfloat16, 2),        # several warps a token
    (2, 3, 5, 1, 7, 7, 16, torch.bfloat16, 2),          # an odd number of heads
    (1, 3, 5, 1, 5, 1, 16, torch.bfloat16, 2),
    (1, 2, 3, 1, 120, 120, 16, torch.bfloat16, 2),      # the most heads
    (1, 2, 3, 1, 3, 9, 16, torch.bfloat16, 2),          # more K/V heads than query heads
    (2, 5, 7, 1, 12, 12, 16, torch.float32, 2),
    (1, 3, 5, 1, 20, 5, 128, torch.float32, 2),
    (1, 1, 3, 1, 80, 80, 16, torch.float32, 2),
]


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("fused", [False, True])
def test_append_matches_the_definition_bit_for_bit(case, fused):
    streams, gh, gw, frames, heads, hk, page_rows, dtype, ring = case
    kwargs, want, q_ref, _ = append_case(*case, seed=heads * 100 + gh, fused=fused)
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)     # rows of other slots and spare pages untouched too
    check_q(kwargs["q_out"], q_ref, dtype)
    assert ops.kv4_counters() == (0, 0, 0)


@pytest.mark.parametrize("case", [
    (1, 34, 42, 1, 12, 12, 128, torch.bfloat16, 1),     # more tokens than are resident: three blocks a thread
    (1, 34, 80, 1, 16, 4, 64, torch.bfloat16, 1),       # four
    (2, 34, 42, 1, 20, 3, 32, torch.bfloat16, 1),       # five, one warp a token
    (1, 23, 41, 1, 33, 33, 16, torch.bfloat16, 1),      # several warps, the last one with heads missing
    (1, 34, 42, 1, 12, 12, 128, torch.float32, 1),
    (1, 52, 52, 1, 7, 2, 16, torch.float32, 1),
])
def test_append_of_many_tokens(case):
    kwargs, want, q_ref, _ = append_case(*case, seed=case[4])
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)
    check_q(kwargs["q_out"], q_ref, case[7])


@pytest.mark.parametrize("k_scale,v_scale,size", [(0.37, 1.7, 1.0), (1e-3, 2.0 ** -20, 30.0), (1e4, 1e6, 1.0),
                                                  (1e-20, 1e20, 1.0)])
def test_append_tensor_scales(k_scale, v_scale, size):
    """Scales that leave blocks saturated, subnormal or zero."""
    kwargs, want, _, _ = append_case(2, 3, 5, 1, 4, 4, 16, torch.bfloat16, 2, seed=5, k_scale=k_scale, v_scale=v_scale,
                                     size=size)
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)


def test_append_unaligned_rows_fp32_weights_and_token_tables():
    """Rows on 16-byte but not 32-byte boundaries take the narrow loads; weights in fp32; explicit tables."""
    kwargs, want, q_ref, _ = append_case(2, 3, 5, 1, 12, 12, 16, torch.bfloat16, 2, seed=9, w32=True, mode="tokens")
    T, C = kwargs["q"].shape
    for name in ("q", "k", "v", "q_out"):
        wide = torch.empty(T, C + 8, dtype=torch.bfloat16, device=DEV)
        view = wide[:, 8:]
        assert view.data_ptr() % 32 == 16
        view.copy_(kwargs[name])
        kwargs[name] = view
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)
    check_q(kwargs["q_out"], q_ref, torch.bfloat16)


def test_append_more_sequences_than_one_launch():
    case = (70, 1, 3, 1, 2, 2, 16, torch.bfloat16, 2)
    kwargs, want, q_ref, _ = append_case(*case, seed=3)
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)
    check_q(kwargs["q_out"], q_ref, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_non_finite_and_zero_inputs(dtype):
    """V with NaN (stored as zero), infinities (saturate) and zero blocks; each block with one counts."""
    kwargs, want, _, _ = append_case(1, 4, 4, 1, 2, 2, 16, dtype, 1, seed=8)
    v = kwargs["v"].cpu()
    v[0, :16] = 0.0
    v[1, 3] = float("nan")
    v[2, 20], v[2, 21] = float("inf"), -float("inf")
    v[3, 40], v[3, 41] = float("nan"), float("-inf")
    kwargs["v"] = v.to(DEV)
    flat = torch.arange(16)
    table = kwargs["table"].cpu()
    kv4.store(want, table, flat, v.view(16, 2, 128), 1, kwargs["v_scale"])
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(**kwargs)
    assert torch.equal(kwargs["pages"].cpu(), want)
    assert ops.kv4_counters().nonfinite == 3
    back = ops.read_kv4(kwargs["pages"], kwargs["table"], 16, v_scale=kwargs["v_scale"])[1].cpu()
    assert bool(torch.isfinite(back).all()) and not back[0, 0, :16].any() and back[0, 1, 3] == 0


def test_append_nan_in_k_normalises_to_nan_as_the_ring_does():
    """A NaN in a K row makes RMSNorm's whole row NaN: stored as zeros, k_pre holds the NaN."""
    kwargs, want, _, kn = append_case(1, 2, 2, 1, 12, 12, 16, torch.bfloat16, 1, seed=8)
    kwargs["k"][1, 5] = float("nan")
    kwargs["k_pre"] = torch.empty_like(kwargs["k"])
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(**kwargs)
    assert ops.kv4_counters().nonfinite == 12 * 8
    assert bool(kwargs["k_pre"][1].isnan().all()) and torch.equal(kwargs["k_pre"][[0, 2, 3]].cpu(), kn[[0, 2, 3]])
    k, _ = ops.read_kv4(kwargs["pages"], kwargs["table"], 4)
    assert not k[0, 1].any() and bool(k[0, [0, 2, 3]].any(-1).all())


def test_append_roles_and_sinks():
    """V alone, K alone without a norm, Q alone, and sink rows beside a chunk in one launch."""
    kwargs, want, q_ref, kn = append_case(1, 3, 4, 1, 4, 4, 16, torch.bfloat16, 3, seed=21)
    base = {x: kwargs[x] for x in ("heads", "seqs", "cos", "sin", "table", "k_scale", "v_scale")}
    start = want.clone().zero_()
    pages = start.to(DEV)
    ops.qk_norm_rope_kv4(**base, pages=pages, v=kwargs["v"])
    assert torch.equal(kv4.split(pages.cpu())[0][:, :, 0], kv4.split(start)[0][:, :, 0])
    ops.qk_norm_rope_kv4(**base, pages=pages, k=kwargs["k"], k_weight=kwargs["k_weight"])
    rows = kv4.place(kwargs["table"].cpu(), torch.arange(12) + kwargs["seqs"][0].ring_slot0 * 12, 16)
    for got, ref in zip(kv4.split(pages.cpu()), kv4.split(want)):
        assert torch.equal(got[rows[0], :, :, rows[1]], ref[rows[0], :, :, rows[1]])
    q_out = torch.empty_like(kwargs["q"])
    ops.qk_norm_rope_kv4(**base, pages=pages, q=kwargs["q"], q_weight=kwargs["q_weight"], q_out=q_out)
    check_q(q_out, q_ref, torch.bfloat16)

    # A sink beside the chunk: its pre-RoPE rows, rotated at frame 9, into the ring's other slot.
    slot = (kwargs["seqs"][0].ring_slot0 + 1) % 3
    both = ops.kv4_pages(want.shape[0], 4, 16, DEV)
    sink = ops.Seq(0, 12, 3, 4, 9, 0, 0, 3, slot, ops.SEQ_SINK)
    args = {**kwargs, "pages": both, "seqs": [kwargs["seqs"][0], sink], "k_sink": kn.to(DEV)}
    ops.qk_norm_rope_kv4(**args)
    c, s = (t for t in wan_prep.frames_table(kwargs["cos"].cpu(), kwargs["sin"].cpu(), wan_prep.axis_dims(128), 9, 10, 3, 4))
    rot = wan_prep.rope(kn.view(1, 12, 4, 128), c, s)[0]
    ref = torch.zeros_like(want)
    kv4.store(ref, kwargs["table"].cpu(), torch.arange(12) + slot * 12, rot, 0, 1.0)
    place = kv4.place(kwargs["table"].cpu(), torch.arange(12) + slot * 12, 16)
    for got, r in zip(kv4.split(both.cpu()), kv4.split(ref)):
        assert torch.equal(got[place[0], :, 0, place[1]], r[place[0], :, 0, place[1]])
        assert not got[place[0], :, 1, place[1]].any()     # a sink writes no V


def test_append_bad_pages_are_skipped_and_counted():
    kwargs, want, _, _ = append_case(1, 4, 8, 1, 3, 3, 16, torch.bfloat16, 1, seed=30)
    before = kwargs["pages"].cpu()
    table = kwargs["table"].cpu()
    lost = int(table[0, 0])
    table[0, 0] = want.shape[0]
    kwargs["table"] = table.to(DEV)
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(**kwargs)
    got = kwargs["pages"].cpu()
    assert torch.equal(got[lost], before[lost])
    keep = [p for p in range(want.shape[0]) if p != lost]
    assert torch.equal(got[keep], want[keep])
    assert ops.kv4_counters().bad_pages > 0
    table[0, 0] = -1
    k, v = ops.read_kv4(kwargs["pages"], table.to(DEV), 32, v_scale=kwargs["v_scale"])
    assert not k[0, :16].any() and not v[0, :16].any() and bool(k[0, 16:].any())
    assert ops.kv4_counters().bad_pages > 0


@pytest.mark.parametrize("launch", ["stream", "pdl", "pdl_early_inputs"])
def test_append_launch_modes_store_the_same(launch):
    """A chain of appends of independent inputs, each read back by the next kernel on the stream."""
    cases = [append_case(2, 5, 7, 2, 12, 4, 32, torch.bfloat16, 2, seed=s) for s in range(4)]
    torch.cuda.synchronize()             # the inputs are there before the first launch
    back = []
    for kwargs, _, _, _ in cases:
        ops.qk_norm_rope_kv4(**kwargs, launch=launch)
        back.append(ops.read_kv4(kwargs["pages"], kwargs["table"], 70, v_scale=0.375))
    for (kwargs, want, q_ref, _), (k, v) in zip(cases, back):
        assert torch.equal(kwargs["pages"].cpu(), want)
        check_q(kwargs["q_out"], q_ref, torch.bfloat16)
        flat = torch.arange(70)
        for which, x, scale in ((0, k, 1.0), (1, v, 0.375)):
            for b in range(2):
                ref = kv4.load(want, kwargs["table"].cpu()[b:b + 1], flat, which, scale)
                assert bool(((x[b].cpu().double().view(ref.shape) - ref).abs() <= 2 ** -8 * ref.abs()).all())


def test_append_on_another_stream_than_the_current_one_before():
    kwargs, want, q_ref, _ = append_case(2, 3, 5, 1, 4, 4, 16, torch.bfloat16, 2, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.qk_norm_rope_kv4(**kwargs)
        k, _ = ops.read_kv4(kwargs["pages"], kwargs["table"], 30)
    side.synchronize()
    assert torch.equal(kwargs["pages"].cpu(), want) and bool(k.any())
    check_q(kwargs["q_out"], q_ref, torch.bfloat16)


def test_append_plan_swaps_tensors():
    case = (2, 3, 5, 1, 4, 4, 16, torch.bfloat16, 2)
    kwargs, _, _, _ = append_case(*case, seed=1)
    other, want, q_ref, _ = append_case(*case, seed=1, size=2.0)
    kwargs["pages"].copy_(other["pages"])
    plan = ops.Prep4Plan(**kwargs)
    plan.launch(q=other["q"], k=other["k"], v=other["v"], q_weight=other["q_weight"], k_weight=other["k_weight"])
    assert torch.equal(kwargs["pages"].cpu(), want)
    check_q(kwargs["q_out"], q_ref, torch.bfloat16)
    with pytest.raises(ops.PrepError, match="swapped"):
        plan.launch(pages=kwargs["pages"])
    with pytest.raises(ops.PrepError, match="match"):
        plan.launch(q=kwargs["q"].float())


# ---------------------------------------------------------------------------------------
# Read
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("members,rows,heads,page_rows,row0,tokens", [
    (1, 1, 1, 16, 0, 1), (2, 300, 3, 16, 0, 300), (3, 200, 5, 32, 41, 159), (2, 257, 2, 64, 63, 2), (1, 700, 12, 128, 127, 573),
    (2, 40, 2, 128, 7, 0),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_read_returns_what_the_cache_stands_for(members, rows, heads, page_rows, row0, tokens, dtype):
    k_scale, v_scale = 0.37, 1.0
    pages, table, k, v = fill(members, rows, heads, page_rows, rows, k_scale, v_scale)
    got = ops.read_kv4(pages.to(DEV), table.to(DEV), tokens, row0=row0, k_scale=k_scale, v_scale=v_scale, dtype=dtype)
    half = 2.0 ** (-8 if dtype == torch.bfloat16 else -24)
    for x, want in zip(got, (k, v)):
        assert x.shape == (members, tokens, heads * 128) and x.dtype == dtype
        want = want[:, row0:row0 + tokens].flatten(2)
        assert bool(((x.cpu().double() - want).abs() <= half * want.abs()).all())
    if not tokens:
        return
    # Into the caller's strided rows, on 16-byte boundaries only.
    wide = torch.full((members, tokens + 1, heads * 128 + 8), 7.0, dtype=dtype, device=DEV)
    out = wide[:, :tokens, 8:]
    ops.read_kv4(pages.to(DEV), table.to(DEV), tokens, row0=row0, k_scale=k_scale, v_scale=v_scale, k_out=out)
    assert torch.equal(out, got[0])
    assert bool((wide[:, tokens] == 7).all()) and bool((wide[..., :8] == 7).all())


def test_read_refuses_rows_behind_the_table():
    pages, table, _, _ = fill(1, 20, 1, 16, 1, extra_pages=0)
    with pytest.raises(ops.PrepError, match="BOUNDS"):
        ops.read_kv4(pages.to(DEV), table.to(DEV), 33)


# ---------------------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------------------
def check_attention(got, q, k, v, lens, heads, causal_block=0, scale=None, absent=None):
    want, size = kv4.attention(q, k, v, lens, heads, causal_block, scale, absent)
    got = got.cpu().double().view(want.shape)
    top = v.abs().amax(dim=(1, 2, 3))[:, None, None, None] if v.shape[1] else torch.zeros(v.shape[0], 1, 1, 1)
    bound = 2 ** -8 * want.abs() + 2 ** -10 * size + 2 ** -24 * k.shape[1] * top
    err = (got - want).abs()
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert bool(torch.isfinite(got).all())
    assert bool((err <= bound).all()), f"{worst:.2f} x the bound, error {float(err.max()):.3e}"


ATTENDS = [
    # members, Lq, heads, kv_heads, page_rows, rows, causal block
    (1, 1, 1, 1, 16, 1, 0),
    (1, 1, 12, 12, 128, 257, 0),
    (3, 1, 4, 4, 16, 100, 0),
    (2, 3, 8, 2, 16, 300, 1),         # shared heads, causal
    (2, 5, 4, 2, 32, 129, 0),
    (1, 8, 2, 2, 64, 128, 0),         # the eight rows of one block
    (1, 9, 2, 2, 64, 640, 1),
    (2, 17, 4, 1, 128, 1000, 4),      # several row blocks, blocks of four tokens
    (1, 40, 3, 3, 32, 33, 1),         # more query rows than window rows: rows that see nothing
    (2, 130, 2, 1, 16, 390, 30),      # frames of 30, the first query frame sees the past only
    (1, 300, 2, 2, 128, 1200, 0),
    (1, 257, 1, 1, 16, 1, 0),
    (1, 600, 2, 1, 64, 600, 100),
]


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("chunks", [0, 1, 3])
@pytest.mark.parametrize("case", ATTENDS)
def test_attention_matches_64_bits(case, chunks, kernel):
    members, Lq, heads, hk, page_rows, rows, cb = case
    pages, table, k, v = fill(members, rows, hk, page_rows, Lq + rows, 0.7, 0.375)
    q = (torch.randn(members, Lq, heads * 128, generator=gen(rows)) * 1.5).bfloat16()
    ops.kv4_counters()
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=heads, k_scale=0.7, v_scale=0.375,
                            causal_block=cb, key_chunks=chunks, kernel=kernel)
    assert got.shape == q.shape and got.dtype == torch.bfloat16
    check_attention(got, q, k, v, [rows] * members, heads, cb)
    assert ops.kv4_counters() == (0, 0, 0)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq,cb,chunks", [(1, 0, 0), (3, 1, 4), (200, 0, 2), (200, 60, 0)])
def test_attention_ragged_lengths(Lq, cb, chunks, kernel):
    """Lengths on the device: zero, one, inside a page, inside a tile, the whole table, beyond it (clamped)."""
    lens = [0, 1, 37, 130, 256, 500, 9999, -5]
    pages, table, k, v = fill(len(lens), 512, 2, 32, 77, extra_pages=0)
    q = torch.randn(len(lens), Lq, 4 * 128, generator=gen(1)).bfloat16()
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), heads=4,
                            causal_block=cb, key_chunks=chunks, kernel=kernel)
    check_attention(got, q, k, v, [min(max(n, 0), 512) for n in lens], 4, cb)
    assert not got[0].any() and not got[7].any()
    short = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), heads=4,
                              causal_block=cb, key_chunks=chunks, kernel=kernel, max_kv_tokens=300)
    check_attention(short, q, k, v, [min(max(n, 0), 300) for n in lens], 4, cb)


@pytest.mark.parametrize("members,Lq,heads,hk,cb,rows", [
    (5, 3, 4, 2, 1, 6000),      # two row blocks, long and short windows
    (40, 1, 2, 2, 0, 1500),     # more members than a warp has lanes
    (1, 1, 3, 3, 0, 8191),
    (2, 20, 2, 1, 7, 3000),
])
@pytest.mark.parametrize("lens", ["spread", "equal", "one", "none"])
def test_attention_splits_the_keys_by_the_lengths(members, Lq, heads, hk, cb, rows, lens):
    """Few units of work whose lengths only the device knows: chunks of like length, whatever the lengths are."""
    pages, table, k, v = fill(members, rows, hk, 64, 31)
    q = torch.randn(members, Lq, heads * 128, generator=gen(32)).bfloat16()
    ns = {"spread": torch.randint(0, rows + 1, (members,), generator=gen(33)), "equal": torch.full((members,), rows),
          "one": torch.where(torch.arange(members) == members - 1, rows, 1), "none": torch.zeros(members)}[lens].int()
    dev = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), ns.to(DEV), heads=heads, causal_block=cb, kernel="rows",
                            max_kv_tokens=rows)
    check_attention(dev, q, k, v, ns.tolist(), heads, cb)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [1, 200])
def test_attention_never_reads_behind_the_window(Lq, kernel):
    """Table entries behind the window name no page, unwritten rows hold 0xff: neither shows, none is counted."""
    rows = 70
    pages, table, k, v = fill(2, rows, 2, 16, 5, extra_pages=4)
    table[:, 5:] = 1 << 30
    q = torch.randn(2, Lq, 2 * 128, generator=gen(2)).bfloat16()
    ops.kv4_counters()
    for cb in (0, 1):
        got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=2, causal_block=cb, kernel=kernel)
        check_attention(got, q, k, v, [rows] * 2, 2, cb)
    assert ops.kv4_counters() == (0, 0, 0)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq,page_rows", [(1, 16), (2, 128), (150, 32), (150, 128)])
def test_attention_leaves_bad_pages_out(Lq, page_rows, kernel):
    rows = 500
    pages, table, k, v = fill(2, rows, 2, page_rows, 6)
    table[0, 1], table[1, 2] = -1, pages.shape[0]
    absent = torch.zeros(2, rows, dtype=torch.bool)
    absent[0, page_rows:2 * page_rows] = True
    absent[1, 2 * page_rows:3 * page_rows] = True
    q = torch.randn(2, Lq, 4 * 128, generator=gen(3)).bfloat16()
    ops.kv4_counters()
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=4, kernel=kernel)
    check_attention(got, q, k, v, [rows] * 2, 4, absent=absent)
    assert ops.kv4_counters().bad_pages > 0
    table[:] = -7
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=4, kernel=kernel)
    assert not got.any()
    ops.kv4_counters()


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [1, 300])
def test_attention_scores_that_grow_along_the_window(Lq, kernel):
    """The running reference has to move many times, by far more than 2^8."""
    rows = 1500
    pages, table, k, v = fill(1, rows, 2, 64, 9)
    flat = torch.arange(rows)
    x = k[0] * torch.linspace(0.1, 8.0, rows, dtype=torch.float64)[:, None, None]
    kv4.store(pages, table, flat, x.float(), 0, 1.0)
    k = kv4.load(pages, table, flat, 0, 1.0)[None]
    q = (torch.randn(1, Lq, 2 * 128, generator=gen(4)) * 4).bfloat16()
    for chunks in (1, 3):
        got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=2, key_chunks=chunks, kernel=kernel)
        check_attention(got, q, k, v, [rows], 2)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [2, 140])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -14, 1e4, 2.0 ** 80, 0.0])
def test_attention_query_rows_of_any_size(size, Lq, kernel):
    """Rows far outside fp16's range, with the scale that brings the scores back."""
    pages, table, k, v = fill(1, 200, 2, 16, 10)
    q = (torch.randn(1, Lq, 2 * 128, generator=gen(5)) * size).bfloat16()
    scale = 0.1 / size if size else None
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), 200, heads=2, scale=scale, kernel=kernel)
    check_attention(got, q, k, v, [200], 2, scale=scale)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [3, 140])
def test_attention_non_finite_queries_stay_in_their_rows(Lq, kernel):
    pages, table, k, v = fill(1, 300, 2, 128, 12)
    q = torch.randn(1, Lq, 2 * 128, generator=gen(6)).bfloat16()
    clean = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), 300, heads=2, kernel=kernel)
    q[0, 1, 7] = float("nan")          # head 0
    q[0, 2, 128 + 9] = float("inf")    # head 1
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), 300, heads=2, kernel=kernel)
    assert bool(got[0, 1, :128].isnan().all()) and bool(got[0, 2, 128:].isnan().all())
    got[0, 1, :128], got[0, 2, 128:] = clean[0, 1, :128], clean[0, 2, 128:]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [2, 150])
def test_attention_strides_and_outputs_in_place(Lq, kernel):
    """Q as [B, L, H, D] out of a wider buffer, the output into a wider one; nothing beside it is written."""
    pages, table, k, v = fill(2, 300, 2, 32, 13)
    buf = torch.randn(2, Lq + 3, 4 * 128 + 64, generator=gen(7)).bfloat16()
    q = buf[:, 1:Lq + 1, 32:32 + 512]
    wide = torch.full((2, Lq + 2, 640), 5.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, :Lq, 64:576]
    dev = buf.to(DEV)[:, 1:Lq + 1, 32:32 + 512].unflatten(2, (4, 128))
    got = ops.attention_kv4(dev, pages.to(DEV), table.to(DEV), 300, heads=4, out=out, kernel=kernel)
    assert got is out
    check_attention(out, q, k, v, [300] * 2, 4)
    assert bool((wide[:, Lq:] == 5).all()) and bool((wide[..., :64] == 5).all()) and bool((wide[..., 576:] == 5).all())


@pytest.mark.parametrize("Lq", [1, 200])
def test_attention_replays_from_a_graph_with_new_lengths(Lq):
    """One captured call: the lengths, pages and queries are read at replay."""
    pages, table, k, v = fill(2, 700, 2, 16, 14)
    q = torch.randn(2, Lq, 4 * 128, generator=gen(8)).bfloat16()
    dq, dp, dt = q.to(DEV), pages.to(DEV), table.to(DEV)
    lens = torch.tensor([700, 700], dtype=torch.int32, device=DEV)
    ops.attention_kv4(dq, dp, dt, lens, heads=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attention_kv4(dq, dp, dt, lens, heads=4)
    for ns in ([5, 640], [0, 129], [700, 1]):
        lens.copy_(torch.tensor(ns, dtype=torch.int32))
        graph.replay()
        check_attention(out, q, k, v, ns, 4)


def test_two_graphs_and_an_eager_call_do_not_share_partial_results():
    """Calls on two streams at once: each has its own workspace."""
    pages, table, k, v = fill(1, 3000, 2, 128, 15)
    dp, dt = pages.to(DEV), table.to(DEV)
    qs = [torch.randn(1, 2, 2 * 128, generator=gen(20 + i)).bfloat16() for i in range(3)]
    dq = [q.to(DEV) for q in qs]
    graphs, outs = [], []
    for i in range(2):
        ops.attention_kv4(dq[i], dp, dt, 3000, heads=2, key_chunks=8)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(ops.attention_kv4(dq[i], dp, dt, 3000, heads=2, key_chunks=8))
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.attention_kv4(dq[2], dp, dt, 3000, heads=2, key_chunks=8)
    torch.cuda.synchronize()
    for out, q in zip((*outs, eager), qs):
        check_attention(out, q, k, v, [3000], 2)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [1, 200])
def test_members_that_share_pages(Lq, kernel):
    """A page may stand in the table more than once: a prefix that two members share, a page twice in one."""
    pages, table, k, v = fill(1, 320, 2, 64, 23, extra_pages=0)
    first = table[0]
    shared = torch.stack([first, torch.stack([first[0], first[1], first[1], first[4], first[0]])])
    at = torch.cat([torch.arange(64) + 64 * i for i in (0, 1, 1, 4, 0)])
    k, v = torch.stack([k[0], k[0, at]]), torch.stack([v[0], v[0, at]])
    q = torch.randn(2, Lq, 2 * 128, generator=gen(24)).bfloat16()
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), shared.to(DEV), 320, heads=2, kernel=kernel)
    check_attention(got, q, k, v, [320] * 2, 2)


def test_a_captured_decoding_step_appends_and_attends():
    """One graph of append and attention, replayed for token after token: the lengths, the page table and the
    inputs change in place between replays; the same steps without a graph give the same bytes."""
    heads, hk, members, page_rows, steps = 8, 2, 2, 16, 20
    n_pages, table = make_table(members, 2, 3, 5)
    cos, sin = (t.to(DEV) for t in wan_prep.rope_tables(128, 256))
    x = torch.randn(steps, members, (heads + 2 * hk) * 128, generator=gen(6)).bfloat16().to(DEV)

    def run(captured):
        pages = ops.kv4_pages(n_pages, hk, page_rows, DEV)
        dt, lens = table.to(DEV), torch.zeros(members, dtype=torch.int32, device=DEV)
        row = torch.zeros(members, heads * 128 + 2 * hk * 128, dtype=torch.bfloat16, device=DEV)
        q, k, v = row.split((heads * 128, hk * 128, hk * 128), 1)
        # The ring of a step is one row, the first of the member's table: the table entry of that row moves on.
        step_table, q_out = dt.clone(), torch.empty(members, heads * 128, dtype=torch.bfloat16, device=DEV)
        plans = [ops.Prep4Plan(heads=heads, seqs=[ops.Seq(b, 1, 1, 1, 0, 0, b * 2 * page_rows + r, 1, 0)
                                                  for b in range(members)], cos=cos, sin=sin, q=q, k=k, v=v,
                               q_out=q_out, pages=pages, table=step_table) for r in range(page_rows)]
        out = torch.empty(members, 1, heads * 128, dtype=torch.bfloat16, device=DEV)

        def step(r):
            plans[r].launch()
            ops.attention_kv4(q_out.view(members, 1, -1), pages, dt, lens, heads=heads, out=out)

        graphs = {}
        if captured:
            step(0)
            pages.zero_()
            torch.cuda.synchronize()
            for r in range(page_rows):
                graphs[r] = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graphs[r]):
                    step(r)
        outs = []
        for t in range(steps):
            row.copy_(x[t])
            lens.fill_(t + 1)
            step_table[:, 0] = dt[:, t // page_rows]
            graphs[t % page_rows].replay() if captured else step(t % page_rows)
            outs.append(out.clone())
        return torch.stack(outs), pages

    outs, pages = run(False)
    outs2, pages2 = run(True)
    assert torch.equal(outs, outs2) and torch.equal(pages, pages2)
    flat = torch.arange(members)[:, None] * 2 * page_rows + torch.arange(steps)
    k, v = (kv4.load(pages.cpu(), table, flat.flatten(), w, 1.0).view(members, steps, hk, 128) for w in (0, 1))
    c, s = (t[:1, None].cpu() for t in (cos, sin))
    for t in (0, 15, 16, 19):
        q = wan_prep.rope(x[t, :, :heads * 128].cpu().view(1, members, heads, 128), c[None], s[None])[0].flatten(1)
        check_attention(outs[t], q.view(members, 1, -1), k[:, :t + 1], v[:, :t + 1], [t + 1] * members, heads)


def test_one_workspace_for_calls_of_unlike_shapes():
    """The caller's scratch, full of ones, for calls of both kernels one after another: nothing of it is taken for
    the call's own."""
    workspace = torch.full((1 << 27,), 0xff, dtype=torch.uint8, device=DEV)
    calls = []
    for members, Lq, heads, hk, rows, kernel in ((3, 2, 4, 2, 2500, "rows"), (2, 300, 2, 2, 900, "tiles"), (1, 1, 2, 1, 4000, "rows"),
                                                 (5, 130, 4, 4, 260, "tiles"), (6, 1, 2, 2, 1200, "rows")):
        pages, table, k, v = fill(members, rows, hk, 32, rows)
        q = torch.randn(members, Lq, heads * 128, generator=gen(Lq)).bfloat16()
        lens = torch.randint(0, rows + 1, (members,), generator=gen(rows)).int()
        calls.append((q, k, v, lens, heads, dict(q=q.to(DEV), pages=pages.to(DEV), table=table.to(DEV), heads=heads,
                                                 max_kv_tokens=rows, kernel=kernel, workspace=workspace)))
    lens_dev = [c[3].to(DEV) for c in calls]
    for _ in range(2):
        outs = [ops.attention_kv4(kv_tokens=n, **c[5]) for n, c in zip(lens_dev, calls)]
    for out, (q, k, v, lens, heads, _) in zip(outs, calls):
        check_attention(out, q, k, v, lens.tolist(), heads)


def test_results_do_not_depend_on_the_run():
    pages, table, _, _ = fill(2, 2000, 2, 64, 16)
    for Lq in (1, 300):
        q = torch.randn(2, Lq, 4 * 128, generator=gen(9)).bfloat16().to(DEV)
        runs = [ops.attention_kv4(q, pages.to(DEV), table.to(DEV), 2000, heads=4) for _ in range(3)]
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_attention_refusals():
    pages, table, _, _ = fill(2, 50, 2, 16, 17)
    dp, dt = pages.to(DEV), table.to(DEV)
    q = torch.zeros(2, 3, 512, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ops.PrepError, match="bfloat16"):
        ops.attention_kv4(q.float(), dp, dt, 50, heads=4)
    with pytest.raises(ops.PrepError):
        ops.attention_kv4(q, dp, dt, 50, heads=3)
    with pytest.raises(ops.PrepError):
        ops.attention_kv4(q[:1], dp, dt, 50, heads=4)
    with pytest.raises(ops.PrepError, match="outside"):
        ops.attention_kv4(q, dp, dt, 81, heads=4)
    with pytest.raises(ops.PrepError, match="int32"):
        ops.attention_kv4(q, dp, dt, torch.zeros(2, device=DEV), heads=4)
    with pytest.raises(ops.PrepError, match="out"):
        ops.attention_kv4(q, dp, dt, 50, heads=4, out=torch.empty(2, 4, 512, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ops.PrepError, match="kernel"):
        ops.attention_kv4(q, dp, dt, 50, heads=4, kernel="fast")
    for bad in (0.0, -1.0, 1e300, float("nan")):
        with pytest.raises(ops.PrepError, match="tensor scales"):
            ops.attention_kv4(q, dp, dt, 50, heads=4, k_scale=bad)
    with pytest.raises(ops.PrepError, match="workspace"):
        ops.attention_kv4(q, dp, dt, 50, heads=4, kernel="tiles",
                          workspace=torch.empty(1 << 22, dtype=torch.uint8, device=DEV)[1:])
    assert ops.attention_kv4(q[:, :0], dp, dt, 50, heads=4).shape == (2, 0, 512)


def test_offsets_beyond_32_bits():
    """A pool of over 4 GiB: the last pages are written and read where they are."""
    heads, page_rows = 40, 128
    page_bytes = heads * 2 * page_rows * 72
    n = (1 << 32) // page_bytes + 5
    pages = torch.zeros(n, heads, 2, page_rows * 72, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[n - 1, 3, n - 2]], dtype=torch.int32)
    g = gen(1)
    x = torch.randn(300, heads * 128, generator=g).bfloat16()
    seqs = [ops.Seq(0, 300, 1, 300, 0, 0, 0, 1, 0)]
    ops.qk_norm_rope_kv4(heads=heads, seqs=seqs, v=x.to(DEV), pages=pages, table=table.to(DEV))
    _, v = ops.read_kv4(pages, table.to(DEV), 300)
    ref = torch.zeros(3, heads, 2, page_rows * 72, dtype=torch.uint8)
    small = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    kv4.store(ref, small, torch.arange(300), x.view(300, heads, 128), 1, 1.0)
    want = kv4.load(ref, small, torch.arange(300), 1, 1.0)
    assert torch.equal(v.cpu().double().view(300, heads, 128), want)
    q = torch.randn(1, 1, heads * 128, generator=g).bfloat16()
    k = torch.zeros(1, 300, heads, 128, dtype=torch.float64)
    check_attention(ops.attention_kv4(q.to(DEV), pages, table.to(DEV), 300, heads=heads), q, k, want[None], [300], heads)


# ---------------------------------------------------------------------------------------
# Together: the Wan ring processor over a 4-bit cache
# ---------------------------------------------------------------------------------------
class FakeAttn(torch.nn.Module):
    def __init__(self, heads, C):
        super().__init__()
        self.heads = heads
        self.to_q, self.to_k, self.to_v = (torch.nn.Linear(C, C, bias=False) for _ in range(3))
        self.norm_q, self.norm_k = torch.nn.RMSNorm(C, eps=1e-6), torch.nn.RMSNorm(C, eps=1e-6)
        self.to_out = torch.nn.ModuleList([torch.nn.Identity(), torch.nn.Identity()])


@pytest.mark.parametrize("page_rows", [16, 128])
def test_ring_processor_over_a_4_bit_cache(page_rows):
    """A stream's chunks until its ring has wrapped and its sink has moved, beside the bf16 ring: the cache
    stands for the quantised rows of the ring, and every output is the exact attention over what it holds."""
    from physisserve_b200.wan import Kv4Pool, RingAttention, RingCache, RingCache4, wan_rope_tables, window_layout

    torch.manual_seed(0)
    heads, gh, gw, batch = 3, 3, 5, 2
    C, hw = heads * 128, gh * gw
    attn = FakeAttn(heads, C).to(DEV, torch.bfloat16)
    cos, sin = wan_rope_tables(128, 64, device=DEV)
    pool = Kv4Pool(200, heads, page_rows, device=DEV)
    other = RingCache4(heads=heads, grid_h=gh, grid_w=gw, pool=pool)
    other.reserve([40])                  # another cell's pages lie between
    ring = RingCache(heads=heads, head_dim=128, grid_h=gh, grid_w=gw, batch=batch, device=DEV)
    small = RingCache4(heads=heads, grid_h=gh, grid_w=gw, batch=batch, pool=pool, k_scale=0.9, v_scale=0.5)
    kernel, plain = RingAttention(), RingAttention()
    sdpa = RingAttention(attention_kernel=False)
    ops.kv4_counters()
    for chunk in range(24):
        pos = [window_layout(chunk)] * batch
        x = torch.randn(batch, pos[0].frames * hw, C, device=DEV).bfloat16()
        kernel.cache, plain.cache, sdpa.cache = small, ring, small
        with torch.no_grad():
            got = kernel(attn, x, rotary_emb=(cos, sin, pos))
            plain(attn, x, rotary_emb=(cos, sin, pos))
            q = attn.to_q(x)
        n = small.window_rows(chunk)
        k4, v4 = ops.read_kv4(small.pages, small.table, n, k_scale=0.9, v_scale=0.5, dtype=torch.float32)
        for have, held, which, scale in ((k4, ring.k, 0, 0.9), (v4, ring.v, 1, 0.5)):
            rows = held[:, :n].cpu().view(batch * n, heads, 128)
            want = kv4.dequantise(*kv4.quantise(rows, scale), scale).view(batch, n, C)
            # K's sum of squares has another order in the ring: a bf16 rounding in 10^4 may differ.
            differ = (have.cpu().double() - want).abs() > 2 ** -20 * want.abs()
            assert float(differ.float().mean()) <= (1e-3 if which == 0 else 0.0)
        q_rot = _rotated_q(attn, q, cos, sin, pos[0], heads, gh, gw)
        check_attention(got, q_rot, k4.cpu().double().view(batch, n, heads, 128), v4.cpu().double().view(batch, n, heads, 128),
                        [n] * batch, heads)
        if chunk in (0, 5, 23):          # SDPA over the window read back: the same to bf16 probabilities
            with torch.no_grad():
                again = sdpa(attn, x, rotary_emb=(cos, sin, pos))
            assert float((again.float() - got.float()).abs().max()) <= 2 ** -5 * float(got.float().abs().max())
    assert ops.kv4_counters() == (0, 0, 0)
    used = pool.free_pages
    small.release()
    assert pool.free_pages > used


def _rotated_q(attn, q, cos, sin, pos, heads, gh, gw):
    """Q as the prep kernel leaves it, from the library itself (tested bit for bit above)."""
    B, L, C = q.shape
    out = torch.empty_like(q)
    seqs = [ops.Seq(b * L, L, gh, gw, pos.frame_offset) for b in range(B)]
    pages = ops.kv4_pages(1, heads, 16, DEV)
    ops.qk_norm_rope_kv4(heads=heads, seqs=seqs, cos=cos, sin=sin, q=q, q_weight=attn.norm_q.weight.detach(), q_out=out,
                         pages=pages, table=torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    return out.cpu()


def test_ring_processor_members_at_different_chunks():
    """Members whose windows differ: one call with the lengths on the device."""
    from physisserve_b200.wan import RingAttention, RingCache4, wan_rope_tables, window_layout

    torch.manual_seed(1)
    heads, gh, gw = 2, 2, 4
    C, hw = heads * 128, gh * gw
    attn = FakeAttn(heads, C).to(DEV, torch.bfloat16)
    cos, sin = wan_rope_tables(128, 64, device=DEV)
    cache = RingCache4(heads=heads, grid_h=gh, grid_w=gw, batch=2, page_rows=16, device=DEV)
    proc = RingAttention()
    proc.cache = cache
    with torch.no_grad():
        proc(attn, torch.randn(2, 3 * hw, C, device=DEV).bfloat16(), rotary_emb=(cos, sin, [window_layout(0)] * 2))
        for chunks in ((1, 1), (2, 1), (3, 2), (3, 4)):
            pos = [window_layout(c) for c in chunks]
            x = torch.randn(2, hw, C, device=DEV).bfloat16()
            got = proc(attn, x, rotary_emb=(cos, sin, pos))
            lens = [cache.window_rows(c) for c in chunks]
            n = max(lens)
            k, v = ops.read_kv4(cache.pages, cache.table, n, dtype=torch.float32)
            q = attn.to_q(x)
            q_rot = torch.cat([_rotated_q(attn, q[b:b + 1], cos, sin, pos[b], heads, gh, gw) for b in range(2)])
            check_attention(got, q_rot, k.cpu().double().view(2, n, heads, 128), v.cpu().double().view(2, n, heads, 128), lens,
                            heads)
    ops.kv4_counters()


def test_unlike_windows_read_back_touch_their_own_pages():
    """SDPA over windows of unlike length: a member's read asks for the pages that it holds, no others."""
    from physisserve_b200.wan import RingAttention, RingCache4, wan_rope_tables, window_layout

    torch.manual_seed(2)
    heads, gh, gw = 2, 2, 4
    C, hw = heads * 128, gh * gw
    attn = FakeAttn(heads, C).to(DEV, torch.bfloat16)
    cos, sin = wan_rope_tables(128, 64, device=DEV)
    cache = RingCache4(heads=heads, grid_h=gh, grid_w=gw, batch=2, page_rows=16, device=DEV)
    proc, sdpa = RingAttention(), RingAttention(attention_kernel=False)
    proc.cache = sdpa.cache = cache
    ops.kv4_counters()
    with torch.no_grad():
        proc(attn, torch.randn(2, 3 * hw, C, device=DEV).bfloat16(), rotary_emb=(cos, sin, [window_layout(0)] * 2))
        for chunks in ((1, 1), (2, 1), (3, 1), (4, 1)):
            rotary = (cos, sin, [window_layout(c) for c in chunks])
            x = torch.randn(2, hw, C, device=DEV).bfloat16()
            got, again = proc(attn, x, rotary_emb=rotary), sdpa(attn, x, rotary_emb=rotary)
            assert float((again.float() - got.float()).abs().max()) <= 2 ** -5 * float(got.float().abs().max())
    assert ops.kv4_counters().bad_pages == 0
    k, _ = cache.window(4, 0)
    assert k.shape == (1, heads, cache.window_rows(4), 128)


# ---------------------------------------------------------------------------------------
# The caller's workspace
# ---------------------------------------------------------------------------------------
def workspace_bytes(q, pages, table, rows, heads, kernel, lens=0):
    """What ps_kv4_attention_workspace reports for a call of contiguous tensors."""
    args = _lib.PsKv4AttnArgs(heads=heads, q_tokens=q.shape[1], kv_tokens=rows, kernel=kernel, q=q.data_ptr(),
                              q_member_stride=q.stride(0), q_row_stride=q.stride(1), out=q.data_ptr(),
                              out_member_stride=q.stride(0), out_row_stride=q.stride(1), kv_lens=lens,
                              cache=_lib.PsKv4Cache(*ops._kv4_cache(pages, table, 1.0, 1.0)[3]))
    need = ctypes.c_int64(0)
    assert _lib.load().ps_kv4_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == _lib.OK
    return need.value


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("offset", [0, 16, 32, 48])
def test_attention_workspace_on_any_16_byte_boundary(kernel, offset):
    """The scratch cut out of a larger buffer: no byte outside of it is written."""
    rows, Lq = 2500, 3 if kernel == "rows" else 300
    pages, table, k, v = fill(1, rows, 2, 128, 61)
    q = torch.randn(1, Lq, 256, generator=gen(62)).bfloat16()
    dev = q.to(DEV), pages.to(DEV), table.to(DEV)
    need = workspace_bytes(*dev, rows, 2, {"rows": _lib.KV4_ROWS, "tiles": _lib.KV4_TILES}[kernel])
    assert need > 0
    arena = torch.full((offset + need + 64,), 0x5a, dtype=torch.uint8, device=DEV)
    workspace = arena[offset:offset + need]
    assert workspace.data_ptr() % 64 == offset
    got = ops.attention_kv4(*dev, rows, heads=2, kernel=kernel, workspace=workspace)
    check_attention(got, q, k, v, [rows], 2)
    assert bool((arena[:offset] == 0x5a).all()) and bool((arena[offset + need:] == 0x5a).all())
    assert not bool((workspace == 0x5a).all())


@pytest.mark.parametrize("members,Lq,heads,rows,cb,lens", [
    (1, 3, 1, 1, 0, None),                              # one unit, one step
    (1, 300, 2, 2500, 0, None),                         # units shared by several CTAs
    (3, 700, 4, 900, 70, [900, 0, 333]),                # unlike units, more of them than CTAs have segments
    (2, 5000, 40, 130, 1, [130, 64]),                   # many units a CTA
])
def test_the_tiles_kernel_leaves_every_unit_its_ctas(members, Lq, heads, rows, cb, lens):
    """The merge takes indices from the units' table, so every entry has to be there: the first CTA, the last one
    and the first one's slot of each (member, head, 256 query rows), by the same cut of all steps into ranges."""
    pages, table, k, v = fill(members, rows, heads, 64, 63)
    q = torch.randn(members, Lq, heads * 128, generator=gen(64)).bfloat16()
    dev = q.to(DEV), pages.to(DEV), table.to(DEV)
    n = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    need = workspace_bytes(*dev, rows, heads, _lib.KV4_TILES, 0 if n is None else n.data_ptr())
    workspace = torch.full((need,), 0xff, dtype=torch.uint8, device=DEV)
    assert workspace.data_ptr() % 32 == 0
    ops.attention_kv4(*dev, rows if n is None else n, heads=heads, causal_block=cb, max_kv_tokens=rows, kernel="tiles",
                      workspace=workspace)
    steps = []
    for b in range(members):
        limits = kv4.limits(rows if lens is None else lens[b], Lq, cb)
        last = [min(Lq, 256 * (i + 1)) - 1 for i in range(-(-Lq // 256))]
        steps += [max(1, -(-int(limits[i]) // 128)) for i in last] * heads
    steps = torch.tensor(steps)
    before = steps.cumsum(0) - steps
    most = len(steps) * max(1, -(-rows // 128))
    grid = min(torch.cuda.get_device_properties(0).multi_processor_count, -(-most // 2))
    per = max(-(-int(steps.sum()) // grid), 2)
    want = torch.stack([before // per, (before + steps - 1) // per, (before % per != 0).long(), torch.zeros_like(steps)], 1)
    at = 2 * grid * 256 * (128 * 4 + 8)
    got = workspace[at:at + 16 * len(steps)].view(torch.int32).view(-1, 4).cpu()
    assert torch.equal(got.long(), want)


@pytest.mark.parametrize("page_rows", [16, 128])
@pytest.mark.parametrize("rows", [131, 200])
def test_attention_limits_of_rows_whose_first_pages_are_missing(rows, page_rows):
    """Eight rows of unlike limits over a window whose first tile has no page: nothing but the limits themselves
    tells the warps what each row sees."""
    pages, table, k, v = fill(3, rows, 2, page_rows, 66)
    table[:, :128 // page_rows] = -1
    absent = torch.zeros(3, rows, dtype=torch.bool)
    absent[:, :128] = True
    q = torch.randn(3, 8, 2 * 128, generator=gen(67)).bfloat16()
    ops.kv4_counters()
    for _ in range(5):
        got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=2, causal_block=1, kernel="rows")
        check_attention(got, q, k, v, [rows] * 3, 2, 1, absent=absent)
    assert ops.kv4_counters().bad_pages > 0


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [2, 140])
@pytest.mark.parametrize("exponent", [124, 125, 126, 127])
def test_attention_query_rows_up_to_the_largest_numbers(exponent, Lq, kernel):
    """Largest elements in [2^exponent, 2^(exponent + 1)): finite in bf16, so the rows' outputs are."""
    pages, table, k, v = fill(1, 200, 2, 16, 40, k_scale=0.02, k_size=0.02)
    q = (torch.rand(1, Lq, 2 * 128, generator=gen(41)) * 2 - 1).bfloat16() * 1.5 * 2.0 ** exponent
    q[..., ::128] = 1.75 * 2.0 ** exponent
    assert q.dtype == torch.bfloat16 and bool(torch.isfinite(q).all())
    scale = 2.0 ** (3 - exponent)
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), 200, heads=2, scale=scale, k_scale=0.02, kernel=kernel)
    check_attention(got, q, k, v, [200], 2, scale=scale)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [4, 200])
def test_attention_small_probabilities_count(Lq, kernel):
    """Every 32nd key takes nearly all of the probability and has a V of zero: what the output holds comes from
    keys of 2^-21.6 to 2^-26 of it.  Bound: the output's rounding 2^-8 |out|, the probabilities' 2^-11 and the
    scores' and exponentials' 2^-13 of A = out, and for probabilities below fp16's normal range half of its last
    step, 2^-25, 2^7 times smaller against the largest: N 2^-32 max|v| / sum."""
    rows = 1000
    n, table = make_table(1, -(-rows // 32), 2, 50)
    pages = torch.full((n, 1, 2, 32 * 72), 0xff, dtype=torch.uint8)
    top = torch.arange(rows) % 32 == 0
    x = torch.zeros(rows, 1, 128)
    x[top, 0, 0] = 6.0
    y = torch.rand(rows, 1, 128, generator=gen(51)) + 0.5
    y[top] = 0.0
    for which, t in ((0, x), (1, y)):
        kv4.store(pages, table, torch.arange(rows), t, which, 1.0)
    k, v = (kv4.load(pages, table, torch.arange(rows), w, 1.0)[None] for w in (0, 1))
    assert torch.equal(k[0].float(), x)
    q = torch.zeros(1, Lq, 128, dtype=torch.bfloat16)
    q[0, :, 0] = torch.tensor([2.5, 2.75, 2.84375, 3.0]).repeat(-(-Lq // 4))[:Lq]    # times 6 / ln 2: 21.6, 23.8, 24.6, 26.0
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=1, scale=1.0, key_chunks=1, kernel=kernel)
    want, size = kv4.attention(q, k, v, [rows], 1, scale=1.0)
    bound = 2 ** -8 * want + 2 ** -10 * size + 2 ** -32 * rows * float(v.max()) / int(top.sum())
    assert float(want.min()) > 2 ** -24
    err = (got.cpu().double().view(want.shape) - want).abs()
    assert bool((err <= bound).all()), f"{float((err / bound).max()):.2f} x the bound"


def test_looking_for_timeouts_keeps_the_other_counts():
    kwargs, _, _, _ = append_case(1, 4, 4, 1, 2, 2, 16, torch.bfloat16, 1, seed=8)
    kwargs["v"][3, 5] = float("nan")
    table = kwargs["table"].clone()
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(**kwargs)
    kwargs["table"][0, 0] = -1
    ops.read_kv4(kwargs["pages"], kwargs["table"], 16)
    q = torch.randn(1, 1, 256, generator=gen(60)).bfloat16().to(DEV)
    ops.attention_kv4(q, kwargs["pages"], table, 16, heads=2, check_timeouts=True)
    counts = ops.kv4_counters(reset=False)
    assert counts.nonfinite == 1 and counts.bad_pages > 0 and counts.timeouts == 0
    assert ops.kv4_counters() == counts and ops.kv4_counters() == (0, 0, 0)


def test_append_to_a_ring_of_nearly_two_to_the_31_frames():
    """One-token frames around the end of the largest ring: the slot of the frame behind the last one is 0, by
    arithmetic that passes 2^31."""
    frames, page_rows, heads = (1 << 31) - 1, 128, 2
    table = torch.full((1, (1 << 31) // page_rows), -1, dtype=torch.int32, device=DEV)
    table[0, 0], table[0, -1] = 2, 1
    pages = ops.kv4_pages(3, heads, page_rows, DEV)
    x = torch.randn(5, heads * 128, generator=gen(70)).bfloat16()
    ops.kv4_counters()
    ops.qk_norm_rope_kv4(heads=heads, seqs=[ops.Seq(0, 5, 1, 1, 0, 0, 0, frames, frames - 2)], v=x.to(DEV), pages=pages, table=table)
    assert ops.kv4_counters() == (0, 0, 0)
    want = torch.zeros_like(pages, device="cpu")
    at = torch.cat([torch.tensor([1, 1]) * page_rows + torch.tensor([125, 126]), 2 * page_rows + torch.arange(3)])
    kv4.store(want, torch.arange(3)[None], at, x.view(5, heads, 128), 1, 1.0)
    assert torch.equal(pages.cpu(), want)


def test_read_refuses_outputs_of_other_shapes():
    pages, table, _, _ = fill(2, 20, 1, 16, 71)
    dev = pages.to(DEV), table.to(DEV)
    for shape in ((2,), (), (2, 19, 128), (1, 20, 128), (2, 20, 64), (2, 20)):
        for name in ("k_out", "v_out"):
            with pytest.raises(ops.PrepError, match=name):
                ops.read_kv4(*dev, 20, **{name: torch.empty(shape, dtype=torch.bfloat16, device=DEV)})


def test_tiles_offsets_beyond_32_bits():
    """Many query rows over the last pages of a pool of over 4 GiB."""
    heads, page_rows = 40, 128
    n = (1 << 32) // (heads * 2 * page_rows * 72) + 5
    pages = torch.zeros(n, heads, 2, page_rows * 72, dtype=torch.uint8, device=DEV)
    _, _, k, v = fill(1, 300, heads, page_rows, 72, extra_pages=0)
    at = torch.tensor([n - 1, 3, n - 2])
    table = torch.arange(3, dtype=torch.int32)[None]
    own = torch.full((3, heads, 2, page_rows * 72), 0xff, dtype=torch.uint8)
    for which, x in ((0, k), (1, v)):
        kv4.store(own, table, torch.arange(300), x[0].float(), which, 1.0)
    pages[at.to(DEV)] = own.to(DEV)
    k, v = (kv4.load(own, table, torch.arange(300), w, 1.0)[None] for w in (0, 1))
    q = torch.randn(1, 130, heads * 128, generator=gen(73)).bfloat16()
    got = ops.attention_kv4(q.to(DEV), pages, at[None].int().to(DEV), 300, heads=heads, kernel="tiles")
    check_attention(got, q, k, v, [300], heads)


# ---------------------------------------------------------------------------------------
# Scores far beyond the range of the exponentials
# ---------------------------------------------------------------------------------------
def one_element_cache(rows, elements, seed):
    """A cache of one head whose keys are zero but for the given {element: e2m1 numbers}, under scales of 1."""
    n, table = make_table(1, -(-rows // 128), 1, seed)
    pages = torch.full((n, 1, 2, 128 * 72), 0xff, dtype=torch.uint8)
    kv4.store(pages, table, torch.arange(rows), torch.rand(rows, 1, 128, generator=gen(seed)) + 0.5, 1, 1.0)
    nibbles, x = torch.zeros(rows, 128, dtype=torch.uint8), torch.zeros(rows, 128)
    for e, numbers in elements.items():
        x[:, e] = numbers
        nibbles[:, e] = torch.searchsorted(kv4.E2M1, numbers.abs().double()).byte() | (torch.signbit(numbers).byte() << 3)
    codes, scales = kv4.split(pages)
    page, row = kv4.place(table, torch.arange(rows), 128)
    codes[page, 0, 0, row], scales[page, 0, 0, row] = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4), 0x38
    k, v = (kv4.load(pages, table, torch.arange(rows), w, 1.0)[None] for w in (0, 1))
    assert torch.equal(k[0, :, 0].float(), x)
    return pages, table, k, v


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("exponent", [10, 20, 24, 25])
@pytest.mark.parametrize("step", [1, 2, 4, 8])
def test_attention_of_scores_a_few_steps_apart(step, exponent, kernel):
    """Scores in log2 units of 2^exponent and a little more, exact in fp32 (up to 2^25 in steps of 4): the
    reference lags behind them, and its distance is rounded like they are."""
    if exponent == 25 and step < 4 or exponent == 24 and step < 2:
        step *= 4
    rows, Lq = 600, 4
    more = torch.zeros(rows)
    more[[130, 260]] = 1.0                # behind the first tile
    more[[391, 500]] = 2.0
    pages, table, k, v = one_element_cache(rows, {0: torch.full((rows,), 4.0), 64: more}, 82)
    q = torch.zeros(1, Lq, 128, dtype=torch.bfloat16)
    q[0, :, 0], q[0, :, 64] = 2.0 ** (exponent - 2), float(step)
    q[0, 1::2, 0] *= -1.0
    scale = 0.6931471805599453            # times log2(e): 1
    got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=1, scale=scale, key_chunks=1, kernel=kernel)
    check_attention(got, q, k, v, [rows], 1, scale=scale)


@pytest.mark.parametrize("kernel", ["rows", "tiles"])
@pytest.mark.parametrize("Lq", [3, 200])
@pytest.mark.parametrize("exponent", [10, 21, 24, 25, 26, 28, 34, 60, 100])
def test_attention_of_scores_of_any_size(exponent, Lq, kernel):
    """Scores of about 2^exponent, of either sign, a few keys sharing the largest: their V's mean."""
    rows = 700
    numbers = torch.tensor([0.5, 1.0, 2.0, 3.0])[torch.randint(0, 4, (rows,), generator=gen(80))]
    numbers[::90] = 4.0
    numbers[::70] = -4.0
    pages, table, k, v = one_element_cache(rows, {0: numbers}, 81)
    q = torch.zeros(1, Lq, 128, dtype=torch.bfloat16)
    q[0, :, 0] = torch.tensor([1.0, -1.25, 1.40625, 1.9921875]).repeat(-(-Lq // 4))[:Lq] * 2.0 ** exponent
    for chunks in (1, 0):
        got = ops.attention_kv4(q.to(DEV), pages.to(DEV), table.to(DEV), rows, heads=1, key_chunks=chunks, kernel=kernel)
        check_attention(got, q, k, v, [rows], 1)
