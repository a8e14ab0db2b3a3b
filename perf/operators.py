"""The 4-bit K/V cache measured: appending to it, reading it back, and attention over it.

Every case is one pass of one operator (``run``) on inputs made from a seed (``prepare``).  With
``own`` false a pass is the operator's plain form in elementary torch operations; with ``own`` true it
is the call of this package.  ``exact`` evaluates the definitions in 64 bits.

The cache.  A pool of pages, ``uint8 [pages, kv_heads, 2, page_rows * 72]``: for each head K (index 0)
and V (index 1), first ``page_rows`` rows of 64 code bytes, then ``page_rows`` rows of 8 scale bytes.
A row is one token's 128 numbers of one head.  Code byte j holds elements 2j (low four bits) and
2j + 1 (high four bits) as e2m1 (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6);
scale byte i is the e4m3 scale of elements 16i .. 16i + 15.  A number is code * scale * tensor scale.
``table[b, i]`` is the page of rows ``[i * page_rows, (i + 1) * page_rows)`` of member b.

Quantising a block of 16 numbers x: scale = e4m3(max|x| / (6 * tensor scale)), codes = e2m1(x / (scale *
tensor scale)), both to nearest with ties to even and saturating.  What is quantised is the rotated K
(and V) in the type of the activations, the rows that a cache of that type would hold, so the roundings
of the RMSNorm's and the rotation's results to that type belong to the definition.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128                 # head dimension
BLOCK = 16              # elements per scale
ROW = 72                # bytes of a row: 64 of codes, 8 of scales
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
TABLE_LEN = 1024        # positions in the rotation tables
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ----------------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------------
def _append(name, streams, grid_h, grid_w, frames, heads, kv_heads, page_rows, dtype="bf16", fused=False,
            ring_frames=2):
    return {"name": name, "op": "append", "streams": streams, "grid_h": grid_h, "grid_w": grid_w, "frames": frames,
            "heads": heads, "kv_heads": kv_heads, "page_rows": page_rows, "dtype": dtype, "fused": fused,
            "ring_frames": ring_frames}


def _read(name, members, tokens, kv_heads, page_rows, row0=0):
    return {"name": name, "op": "read", "members": members, "tokens": tokens, "kv_heads": kv_heads,
            "page_rows": page_rows, "row0": row0}


def _attend(name, members, q_tokens, kv_tokens, heads, kv_heads, page_rows, causal_block=0, ragged=False):
    return {"name": name, "op": "attend", "members": members, "q_tokens": q_tokens, "kv_tokens": kv_tokens,
            "heads": heads, "kv_heads": kv_heads, "page_rows": page_rows, "causal_block": causal_block,
            "ragged": ragged}


def listed():
    return [
        # One new token for each of eight sequences: the append of a decoding step.
        _append("append 8 tokens", 8, 1, 1, 1, 12, 12, 128, ring_frames=300),
        # One latent frame of one 1.3B stream (a 30 x 52 grid, 12 heads), q, k and v in one fused buffer.
        _append("append frame 12 heads", 1, 30, 52, 1, 12, 12, 128, fused=True),
        # One frame of each of eight 14B streams (40 heads).
        _append("append 8 frames 40 heads", 8, 30, 52, 1, 40, 40, 128),
        # Odd frames, fp32 activations, shared K/V heads, small pages.
        _append("append odd frames f32", 3, 27, 41, 2, 20, 5, 16, dtype="f32"),
        # The whole window of a 1.3B stream as bf16 rows, for an attention that reads bf16.
        _read("read window", 1, 34320, 12, 128),
        # Parts of three short sequences in small pages, from the middle of a page.
        _read("read short", 3, 777, 5, 16, row0=41),
        # One query row over a short window: the latency of a call.
        _attend("attend 1 row 257 keys", 1, 1, 257, 12, 12, 128),
        # One query row of each of sixteen sequences over full windows: bound by reading the cache.
        _attend("attend 16 x 1 row", 16, 1, 34320, 12, 12, 128),
        # Three drafted tokens of seven sequences of unlike lengths, causal, four query heads per K/V head.
        _attend("attend 7 x 3 rows shared", 7, 3, 8191, 32, 8, 16, causal_block=1, ragged=True),
        # The block call of a 1.3B stream: a frame's queries over the 22-frame window.
        _attend("attend frame 12 heads", 1, 1560, 34320, 12, 12, 128),
        # The block call of a 14B stream.
        _attend("attend frame 40 heads", 1, 1560, 34320, 40, 40, 128),
        # Seven given frames at once, each seeing itself and the frames before it.
        _attend("attend 7 frames causal", 1, 10920, 10920, 12, 12, 64, causal_block=1560),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    group = rng.choice((1, 1, 1, 2, 4, 5, 8))
    kv = max(1, _log(rng, 1, 40) // group)
    return kv * group, kv


def draw(rng):
    op = rng.choice(("append", "append", "read", "attend", "attend", "attend"))
    page_rows = rng.choice((16, 32, 64, 128, 128))
    if op == "append":
        heads, kv = _heads(rng)
        streams, gh, gw, frames = rng.randint(1, 12), _log(rng, 1, 40), _log(rng, 1, 60), rng.randint(1, 3)
        while streams * gh * gw * frames * heads > 12480 * 40:
            streams, gh = max(1, streams // 2), max(1, gh // 2)
        return {k: v for k, v in _append("", streams, gh, gw, frames, heads, kv, page_rows,
                                         rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.5,
                                         frames + rng.randint(0, 3)).items() if k != "name"}
    if op == "read":
        members, tokens, kv = rng.randint(1, 6), _log(rng, 1, 34320), rng.randint(1, 16)
        while members * tokens * kv > 34320 * 12:
            tokens = max(1, tokens // 2)
        return {k: v for k, v in _read("", members, tokens, kv, page_rows, rng.choice((0, rng.randint(0, 500)))).items()
                if k != "name"}
    heads, kv = _heads(rng)
    members = rng.randint(1, 16)
    if rng.random() < 0.5:
        q_tokens, kv_tokens = _log(rng, 1, 20), _log(rng, 1, 34320)
    else:
        q_tokens, kv_tokens = _log(rng, 20, 4000), _log(rng, 1, 34320)
    causal = rng.choice((0, 0, 1, _log(rng, 2, 1560)))
    # As much as the largest listed case at most: the products, and the plain form's score matrix.
    while members * heads * q_tokens * kv_tokens > 40 * 1560 * 34320 or members * kv * kv_tokens > 16 * 12 * 34320:
        members, kv_tokens = max(1, members // 2), max(1, kv_tokens // 2)
    return {k: v for k, v in _attend("", members, q_tokens, kv_tokens, heads, kv, page_rows, causal,
                                     rng.random() < 0.4).items() if k != "name"}


# ----------------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------------
def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _rope_tables():
    """cos and sin [TABLE_LEN, D]: the frame, row and column angles in columns 44 | 42 | 42, each twice."""
    h = 2 * (D // 6)
    parts = []
    for d in (D - 2 * h, h, h):
        freq = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
        parts.append(torch.outer(torch.arange(TABLE_LEN, dtype=torch.float64, device=DEV), freq).repeat_interleave(2, 1))
    angles = torch.cat(parts, 1)
    return angles.cos().float(), angles.sin().float()


def _new_pages(members, rows, kv_heads, page_rows, gen):
    """An empty pool with a few pages that nobody owns, and a table of pages in random order."""
    per = -(-rows // page_rows)
    count = members * per + 3
    pages = torch.zeros(count, kv_heads, 2, page_rows * ROW, dtype=torch.uint8, device=DEV)
    table = torch.randperm(count, generator=gen, device=DEV)[:members * per].view(members, per).int()
    return pages, table


def _prepare_append(case, gen):
    hw = case["grid_h"] * case["grid_w"]
    n, dtype = hw * case["frames"], DTYPES[case["dtype"]]
    T, C, Ck = case["streams"] * n, case["heads"] * D, case["kv_heads"] * D
    # Projection outputs: channels of unlike size, a few of them large.
    size = torch.exp(_randn((C + 2 * Ck,), gen) * 0.5)
    qkv = (_randn((T, C + 2 * Ck), gen) * size).to(dtype)
    q, k, v = qkv.split((C, Ck, Ck), 1)
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    pages, table = _new_pages(case["streams"], case["ring_frames"] * hw, case["kv_heads"], case["page_rows"], gen)
    cos, sin = _rope_tables()
    slot0 = int(torch.randint(0, case["ring_frames"] - case["frames"] + 1, (1,), generator=gen, device=DEV))
    offsets = torch.randint(0, 500, (case["streams"],), generator=gen, device=DEV).tolist()
    return {"q": q, "k": k, "v": v, "q_weight": (1 + 0.2 * _randn((C,), gen)).to(dtype),
            "k_weight": (1 + 0.2 * _randn((Ck,), gen)).to(dtype), "cos": cos, "sin": sin, "pages": pages,
            "table": table, "slot0": slot0, "offsets": offsets, "n": n, "hw": hw, "k_scale": 1.0, "v_scale": 0.375}


def _fill(pages, table, rows, kv_heads, page_rows, gen, k_scale, v_scale):
    """Fills every member's rows with quantised keys and values."""
    at = torch.arange(rows, device=DEV)
    for b in range(table.shape[0]):
        for which, scale in ((0, k_scale), (1, v_scale)):
            x = _randn((rows, kv_heads, D), gen)
            if which:
                x += 0.3 * _randn((1, kv_heads, D), gen)     # channels of V that do not average to zero
            _store(pages, page_rows, table[b, at // page_rows].long(), at % page_rows, which, *_quantise(x, scale))


def _prepare_read(case, gen):
    rows = case["row0"] + case["tokens"]
    pages, table = _new_pages(case["members"], rows, case["kv_heads"], case["page_rows"], gen)
    state = {"pages": pages, "table": table, "k_scale": 1.0, "v_scale": 0.375}
    _fill(pages, table, rows, case["kv_heads"], case["page_rows"], gen, 1.0, 0.375)
    return state


def _prepare_attend(case, gen):
    pages, table = _new_pages(case["members"], case["kv_tokens"], case["kv_heads"], case["page_rows"], gen)
    _fill(pages, table, case["kv_tokens"], case["kv_heads"], case["page_rows"], gen, 1.0, 0.375)
    # Heads of unlike sharpness.
    sharp = torch.empty(1, 1, case["heads"], 1, device=DEV).uniform_(0.5, 2.5, generator=gen)
    q = (_randn((case["members"], case["q_tokens"], case["heads"], D), gen) * sharp).bfloat16()
    lens = case["kv_tokens"]
    if case["ragged"]:
        low = 0 if case["kv_tokens"] < 64 else case["kv_tokens"] // 8
        lens = torch.randint(low, case["kv_tokens"] + 1, (case["members"],), generator=gen, device=DEV).int()
    return {"q": q.flatten(2), "pages": pages, "table": table, "lens": lens, "k_scale": 1.0, "v_scale": 0.375}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    state = {"append": _prepare_append, "read": _prepare_read, "attend": _prepare_attend}[case["op"]](case, gen)
    state["case"] = dict(case)
    return state


# ----------------------------------------------------------------------------------------
# Plain forms
# ----------------------------------------------------------------------------------------
def _quantise(x, tensor_scale):
    """(codes uint8 [..., D/2], scales uint8 [..., D/16]) of x [..., D].  The two quotients are taken in 64
    bits and rounded to 32: both formats have few bits, so numbers do lie midway between two of theirs."""
    blocks = x.double().unflatten(-1, (D // BLOCK, BLOCK))
    six = torch.tensor(6.0 * tensor_scale, dtype=torch.float32, device=x.device).double()
    scales = (blocks.abs().amax(-1) / six).float().clamp(max=448.0).to(torch.float8_e4m3fn)
    step = (scales.float() * tensor_scale).double()[..., None]
    y = torch.where(step > 0, blocks / step, 0.0).float()
    m = y.abs()
    code = ((m > 0.25).byte() + (m >= 0.75).byte() + (m > 1.25).byte() + (m >= 1.75).byte() + (m > 2.5).byte()
            + (m >= 3.5).byte() + (m > 5.0).byte()) | (torch.signbit(y).byte() << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales.view(torch.uint8)


def _split(pages, page_rows):
    """Views of a pool: codes [pages, heads, 2, page_rows, 64] and scales [pages, heads, 2, page_rows, 8]."""
    codes = pages[..., :page_rows * 64].unflatten(-1, (page_rows, 64))
    return codes, pages[..., page_rows * 64:].unflatten(-1, (page_rows, 8))


def _store(pages, page_rows, page, row, which, codes, scales):
    code_rows, scale_rows = _split(pages, page_rows)
    code_rows[page, :, which, row] = codes
    scale_rows[page, :, which, row] = scales


def _load(pages, table, page_rows, row0, tokens, which, tensor_scale):
    """Rows [row0, row0 + tokens) of every member, fp32 [members, tokens, heads, D]."""
    at = torch.arange(row0, row0 + tokens, device=pages.device)
    page, row = table[:, at // page_rows].long(), (at % page_rows).expand(table.shape[0], -1)
    codes, scales = (t[page, :, which, row] for t in _split(pages, page_rows))
    values = torch.tensor(VALUES + tuple(-x for x in VALUES), device=pages.device)
    x = values[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()]
    s = scales.view(torch.float8_e4m3fn).float() * tensor_scale
    return (x.unflatten(-1, (D // BLOCK, BLOCK)) * s[..., None]).flatten(-2)


def _rms_norm(x, weight):
    """The row's sum of squares in 64 bits, the rest in 32 with IEEE steps, rounded to x's type."""
    mean = x.double().square().sum(-1, keepdim=True).float().double().div(x.shape[-1]).float() + EPS
    rstd = mean.double().sqrt().float().double().reciprocal().float()
    return (x.float() * rstd * weight.float()).to(x.dtype)


def _token_tables(cos, sin, case, offsets):
    l = torch.arange(case["grid_h"] * case["grid_w"] * case["frames"], device=cos.device)
    hw, gw = case["grid_h"] * case["grid_w"], case["grid_w"]
    frame = torch.tensor(offsets, device=cos.device)[:, None] + l // hw
    row, col = ((l // gw) % case["grid_h"]).expand_as(frame), (l % gw).expand_as(frame)
    h = 2 * (D // 6)
    t = D - 2 * h
    return tuple(torch.cat((x[frame, :t], x[row, t:t + h], x[col, t + h:]), -1).flatten(0, 1)[:, None]
                 for x in (cos, sin))


def _rotate(x, cos, sin, heads):
    x = x.unflatten(-1, (heads, D))
    pairs = x.float()
    e, o = pairs[..., 0::2], pairs[..., 1::2]
    out = torch.stack((e * cos[..., 0::2] - o * sin[..., 1::2], e * sin[..., 0::2] + o * cos[..., 1::2]), -1)
    return out.flatten(-2).to(x.dtype)


def _plain_append(s):
    case = s["case"]
    pr, first = case["page_rows"], s["slot0"] * s["hw"]
    cos, sin = _token_tables(s["cos"], s["sin"], case, s["offsets"])
    q = _rotate(_rms_norm(s["q"], s["q_weight"]), cos, sin, case["heads"]).flatten(1)
    k = _rotate(_rms_norm(s["k"], s["k_weight"]), cos, sin, case["kv_heads"])
    v = s["v"].unflatten(-1, (case["kv_heads"], D))
    at = torch.arange(first, first + s["n"], device=DEV)
    page, row = s["table"][:, at // pr].long().flatten(), (at % pr).repeat(case["streams"])
    _store(s["pages"], pr, page, row, 0, *_quantise(k, s["k_scale"]))
    _store(s["pages"], pr, page, row, 1, *_quantise(v, s["v_scale"]))
    return {"q": q, "k": _load(s["pages"], s["table"], pr, first, s["n"], 0, s["k_scale"]).flatten(2).bfloat16(),
            "v": _load(s["pages"], s["table"], pr, first, s["n"], 1, s["v_scale"]).flatten(2).bfloat16()}


def _plain_read(s):
    case = s["case"]
    at = (s["pages"], s["table"], case["page_rows"], case["row0"], case["tokens"])
    return {"k": _load(*at, 0, s["k_scale"]).flatten(2).bfloat16(),
            "v": _load(*at, 1, s["v_scale"]).flatten(2).bfloat16()}


def _limits(case, lens):
    """Keys that each query row sees, [members, q_tokens]."""
    i = torch.arange(case["q_tokens"], device=DEV)
    lens = lens.long()[:, None] if torch.is_tensor(lens) else torch.full((case["members"], 1), lens, device=DEV)
    if not case["causal_block"]:
        return lens.expand(-1, case["q_tokens"])
    return torch.minimum(lens, lens - case["q_tokens"] + (i // case["causal_block"] + 1) * case["causal_block"])


def _plain_attend(s):
    case = s["case"]
    n, kv, group = case["kv_tokens"], case["kv_heads"], case["heads"] // case["kv_heads"]
    k = _load(s["pages"], s["table"], case["page_rows"], 0, n, 0, s["k_scale"]).permute(0, 2, 3, 1)
    q = s["q"].float().unflatten(-1, (kv, group, D)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ k).mul_(D ** -0.5).unflatten(2, (group, case["q_tokens"]))
    del k
    limits = _limits(case, s["lens"])
    hidden = torch.arange(n, device=DEV) >= limits[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = _load(s["pages"], s["table"], case["page_rows"], 0, n, 1, s["v_scale"]).permute(0, 2, 1, 3)
    out = (scores.flatten(2, 3) @ v).unflatten(2, (group, case["q_tokens"]))
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).flatten(2).bfloat16()


# ----------------------------------------------------------------------------------------
# The calls of this package
# ----------------------------------------------------------------------------------------
def _own_append(s):
    from physisserve_b200 import ops
    case = s["case"]
    first = s["slot0"] * s["hw"]
    if "plan" not in s:     # kept over the steps and layers of a program, as the sequences stay the same
        rows = s["table"].shape[1] * case["page_rows"]
        seqs = [ops.Seq(b * s["n"], s["n"], case["grid_h"], case["grid_w"], frame_offset=s["offsets"][b],
                        ring_row=b * rows, ring_frames=case["ring_frames"], ring_slot0=s["slot0"])
                for b in range(case["streams"])]
        s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
        s["plan"] = ops.Prep4Plan(heads=case["heads"], kv_heads=case["kv_heads"], head_dim=D, seqs=seqs, cos=s["cos"],
                                  sin=s["sin"], q=s["q"], k=s["k"], v=s["v"], q_weight=s["q_weight"],
                                  k_weight=s["k_weight"], eps=EPS, q_out=s["q_out"], pages=s["pages"],
                                  table=s["table"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    s["plan"].launch(q=s["q"], k=s["k"], v=s["v"])
    k, v = ops.read_kv4(s["pages"], s["table"], s["n"], row0=first, k_scale=s["k_scale"], v_scale=s["v_scale"])
    return {"q": s["q_out"], "k": k, "v": v}


def _own_read(s):
    from physisserve_b200 import ops
    case = s["case"]
    k, v = ops.read_kv4(s["pages"], s["table"], case["tokens"], row0=case["row0"], k_scale=s["k_scale"],
                        v_scale=s["v_scale"])
    return {"k": k, "v": v}


def _own_attend(s):
    from physisserve_b200 import ops
    case = s["case"]
    return ops.attention_kv4(s["q"], s["pages"], s["table"], s["lens"], heads=case["heads"], k_scale=s["k_scale"],
                             v_scale=s["v_scale"], causal_block=case["causal_block"])


def run(state):
    plain, mine = {"append": (_plain_append, _own_append), "read": (_plain_read, _own_read),
                   "attend": (_plain_attend, _own_attend)}[state["case"]["op"]]
    return mine(state) if own else plain(state)


# ----------------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "append":
        tokens = case["streams"] * case["frames"] * case["grid_h"] * case["grid_w"]
        C, Ck, size = case["heads"] * D, case["kv_heads"] * D, 2 if case["dtype"] == "bf16" else 4
        # q, k, v in; rotated q and the cache rows out; the rows' values in bf16.
        per = 2 * C * size + 2 * Ck * size + 2 * case["kv_heads"] * ROW + 2 * Ck * 2
        return {"bytes": tokens * per, "flops": tokens * (C * 8 + Ck * 16)}
    if case["op"] == "read":
        rows = case["members"] * case["tokens"] * case["kv_heads"] * 2
        return {"bytes": rows * (ROW + 2 * D), "flops": rows * D}
    members, n, lq = case["members"], case["kv_tokens"], case["q_tokens"]
    share = 0.5625 if case["ragged"] and n >= 64 else 1.0   # the mean of the lengths that are drawn
    pairs = members * lq * n * share
    if case["causal_block"]:
        b, low = case["causal_block"], n * share - lq
        pairs = members * sum(b * max(0.0, min(n * share, low + (j + 1) * b)) for j in range(lq // b))
        pairs += members * (lq % b) * n * share
    bytes_ = members * (2 * lq * case["heads"] * D * 2 + 2 * n * share * case["kv_heads"] * ROW)
    return {"bytes": int(bytes_), "flops": int(max(1, 4 * D * case["heads"] * pairs))}


# ----------------------------------------------------------------------------------------
# The definitions in 64 bits
# ----------------------------------------------------------------------------------------
def _exact_decode(codes, scales, tensor_scale):
    """Numbers of code bytes [..., 64] and scale bytes [..., 8] by the bits of the two formats, in 64 bits."""
    nibbles = torch.empty(*codes.shape, 2, dtype=torch.int32, device=codes.device)
    nibbles[..., 0], nibbles[..., 1] = codes.int() % 16, codes.int() // 16
    nibbles = nibbles.flatten(-2)
    e, m = (nibbles // 2) % 4, nibbles % 2
    x = torch.where(e > 0, (2.0 + m.double()) * torch.exp2(e.double() - 2.0), 0.5 * m.double())
    x = torch.where(nibbles >= 8, -x, x)
    b = scales.int()
    e, m = b // 8, b % 8
    s = torch.where(e > 0, (8.0 + m.double()) * torch.exp2(e.double() - 10.0), m.double() * 2.0 ** -9)
    return (x.unflatten(-1, (D // BLOCK, BLOCK)) * (s * tensor_scale)[..., None]).flatten(-2)


def _exact_rows(state, member, head, row0, tokens, which, tensor_scale):
    """fp64 [tokens, D] of one member and head."""
    pr = state["case"]["page_rows"]
    count = (row0 + tokens - 1) // pr + 1
    raw = state["pages"][state["table"][member, :count].long(), head, which]
    codes = raw[:, :pr * 64].reshape(count * pr, 64)[row0:row0 + tokens]
    return _exact_decode(codes, raw[:, pr * 64:].reshape(count * pr, 8)[row0:row0 + tokens], tensor_scale)


def _nearest(x, grid):
    """The nearest value of a sorted grid, of two equally near ones that with the even index; saturating."""
    x = x.clamp(max=float(grid[-1]))
    i = torch.searchsorted(grid, x.contiguous()).clamp(1, len(grid) - 1)
    low, high = grid[i - 1], grid[i]
    up = (high - x < x - low) | ((high - x == x - low) & (i % 2 == 0))
    return torch.where(up, high, low)


def _exact_quantised(x, tensor_scale):
    """fp64 numbers that the cache stands for after x [..., D] was stored."""
    e4m3 = torch.tensor([(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device=x.device)
    e2m1 = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    blocks = x.double().unflatten(-1, (D // BLOCK, BLOCK))
    s = _nearest(blocks.abs().amax(-1, keepdim=True) / (6.0 * tensor_scale), e4m3) * tensor_scale
    codes = _nearest(torch.where(s > 0, blocks.abs() / s, 0.0), e2m1)
    return (codes * s * blocks.sign()).flatten(-2)


def _exact_rotated(x, weight, angles, heads):
    """RMSNorm and rotation of x [T, heads * D] by fp64 tables, rounded to x's type after each."""
    cos, sin = angles
    n = x.double() / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    n = n.to(x.dtype).double().unflatten(-1, (heads, D // 2, 2))
    c, s = cos.double().unflatten(-1, (D // 2, 2)), sin.double().unflatten(-1, (D // 2, 2))
    out = torch.empty_like(n)
    out[..., 0] = n[..., 0] * c[..., 0] - n[..., 1] * s[..., 1]
    out[..., 1] = n[..., 0] * s[..., 0] + n[..., 1] * c[..., 1]
    return out.flatten(-2).to(x.dtype)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        out = {"q": [], "k": [], "v": []}
        for b in range(case["streams"]):        # a member at a time, for the memory
            rows = slice(b * s["n"], (b + 1) * s["n"])
            angles = _token_tables(s["cos"], s["sin"], case, [s["offsets"][b]])
            out["q"].append(_exact_rotated(s["q"][rows], s["q_weight"], angles, case["heads"]).double().flatten(1))
            k = _exact_rotated(s["k"][rows], s["k_weight"], angles, case["kv_heads"])
            out["k"].append(_exact_quantised(k, s["k_scale"]).flatten(1))
            out["v"].append(_exact_quantised(s["v"][rows].unflatten(-1, (case["kv_heads"], D)), s["v_scale"]).flatten(1))
        return {"q": torch.cat(out["q"]), "k": torch.stack(out["k"]), "v": torch.stack(out["v"])}
    if case["op"] == "read":
        def rows(which, scale):
            return torch.stack([torch.cat([_exact_rows(s, b, h, case["row0"], case["tokens"], which, scale)
                                           for h in range(case["kv_heads"])], 1) for b in range(case["members"])])
        return {"k": rows(0, s["k_scale"]), "v": rows(1, s["v_scale"])}
    group, n = case["heads"] // case["kv_heads"], case["kv_tokens"]
    out = torch.zeros(case["members"], case["q_tokens"], case["heads"], D, dtype=torch.float64, device=DEV)
    limits = _limits(case, s["lens"])
    q = s["q"].unflatten(-1, (case["heads"], D))
    for b in range(case["members"]):
        seen = torch.arange(n, device=DEV) < limits[b][:, None]
        some = seen.any(-1)
        for h in range(case["kv_heads"]):
            k, v = (_exact_rows(s, b, h, 0, n, w, t) for w, t in ((0, s["k_scale"]), (1, s["v_scale"])))
            for g in range(h * group, (h + 1) * group):
                scores = (q[b, :, g].double() @ k.T / math.sqrt(D)).masked_fill(~seen, -math.inf)
                out[b, some, g] = torch.softmax(scores[some], -1) @ v
    return out.flatten(2)
