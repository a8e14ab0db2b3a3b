"""CPU restatement of the paged 4-bit K/V cache (include/physis_b200_kv4.h): the format by its bits, the
quantisation with correctly rounded quotients, paging by a page table, and attention in 64 bits."""
from __future__ import annotations

import torch

D, BLOCK, ROW_BYTES = 128, 16, 72
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# e4m3 without its sign: 127 finite values, exponent bias 7, subnormals of 2^-9.
E4M3 = torch.tensor([(m if e == 0 else 8 + m) * 2.0 ** (max(e, 1) - 10) for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def nearest(x: torch.Tensor, grid: torch.Tensor) -> torch.Tensor:
    """Index of the nearest value of an increasing grid from 0; midway goes to the even index; saturates."""
    mid = (grid[1:] + grid[:-1]) / 2
    low, high = torch.searchsorted(mid, x.contiguous()), torch.searchsorted(mid, x.contiguous(), right=True)
    return torch.where(high > low, low + low % 2, low)   # exactly on a midpoint: low or low + 1, whichever is even


def quantise(x: torch.Tensor, tensor_scale: float):
    """x [..., 128] (bf16 or fp32) -> (code bytes uint8 [..., 64], scale bytes uint8 [..., 8])."""
    most = 448.0 * float(torch.tensor(6.0 * tensor_scale, dtype=torch.float32))
    v = x.double().unflatten(-1, (D // BLOCK, BLOCK))
    v = torch.where(v.isnan(), 0.0, v.clamp(-most, most))
    six = float(torch.tensor(6.0, dtype=torch.float32) * torch.tensor(tensor_scale, dtype=torch.float32))
    scale = nearest((v.abs().amax(-1) / six).float().double(), E4M3)
    step = (E4M3[scale].float() * torch.tensor(tensor_scale, dtype=torch.float32)).double()[..., None]
    y = torch.where(step > 0, v / step, 0.0).float().double()
    code = nearest(y.abs(), E2M1) + 8 * torch.signbit(v)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.to(torch.uint8)


def dequantise(codes: torch.Tensor, scales: torch.Tensor, tensor_scale: float) -> torch.Tensor:
    """fp64 numbers [..., 128]."""
    nibbles = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    x = torch.where(nibbles >= 8, -E2M1[nibbles % 8], E2M1[nibbles % 8])
    s = E4M3[scales.long().clamp(max=126)] * float(torch.tensor(tensor_scale, dtype=torch.float32))
    return (x.unflatten(-1, (D // BLOCK, BLOCK)) * s[..., None]).flatten(-2)


def split(pages: torch.Tensor):
    """Views (codes [pages, heads, 2, page_rows, 64], scales [pages, heads, 2, page_rows, 8]) of a pool."""
    rows = pages.shape[-1] // ROW_BYTES
    return pages[..., :rows * 64].unflatten(-1, (rows, 64)), pages[..., rows * 64:].unflatten(-1, (rows, 8))


def place(table: torch.Tensor, rows: torch.Tensor, page_rows: int):
    """(page, row in it) of flat logical rows."""
    return table.flatten().long()[rows // page_rows], rows % page_rows


def store(pages: torch.Tensor, table: torch.Tensor, rows: torch.Tensor, x: torch.Tensor, which: int, tensor_scale: float):
    """Quantises x [n, heads, 128] into the flat logical rows; which: 0 = K, 1 = V."""
    codes, scales = split(pages)
    page, row = place(table, rows, codes.shape[3])
    codes[page, :, which, row], scales[page, :, which, row] = quantise(x, tensor_scale)


def load(pages: torch.Tensor, table: torch.Tensor, rows: torch.Tensor, which: int, tensor_scale: float) -> torch.Tensor:
    """fp64 [n, heads, 128] of the flat logical rows."""
    codes, scales = split(pages)
    page, row = place(table, rows, codes.shape[3])
    return dequantise(codes[page, :, which, row], scales[page, :, which, row], tensor_scale)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """RMSNorm over the last dimension: the sum of squares in 64 bits, every later step in IEEE fp32, one
    rounding to x's type (fp64 quotients and roots rounded once to fp32 are the IEEE ones)."""
    mean = (x.double().square().sum(-1, keepdim=True).float().double() / x.shape[-1]).float()
    mean = mean + torch.tensor(eps, dtype=torch.float32)
    rstd = (1.0 / mean.double().sqrt().float().double()).float()
    return (x.float() * rstd * weight.float()).to(x.dtype)


def limits(n: int, q_tokens: int, causal_block: int) -> torch.Tensor:
    """Keys that each query row of a member with n window rows sees."""
    t = torch.arange(q_tokens)
    if causal_block == 0:
        return torch.full((q_tokens,), n)
    return (n - q_tokens + (t // causal_block + 1) * causal_block).clamp(0, n)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens, heads: int, causal_block: int = 0,
              scale: float | None = None, absent: torch.Tensor | None = None):
    """q [B, Lq, heads*128], k/v fp64 [B, rows, kv_heads, 128] -> (out, mean of |v| under the probabilities,
    largest |v|), each fp64 [B, Lq, heads, 128] (the last [B]).  absent [B, rows]: keys that nothing sees."""
    B, Lq = q.shape[:2]
    group = heads // k.shape[2]
    qd = q.double().view(B, Lq, heads, D)
    out = torch.zeros(B, Lq, heads, D, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b in range(B):
        seen = torch.arange(k.shape[1]) < limits(int(lens[b]), Lq, causal_block)[:, None]
        if absent is not None:
            seen &= ~absent[b]
        some = seen.any(-1)
        if not some.any():
            continue
        for h in range(heads):
            s = qd[b, :, h] @ k[b, :, h // group].T * (scale if scale else D ** -0.5)
            p = s.masked_fill(~seen, -torch.inf)[some].softmax(-1)
            # What is not seen does not enter, whatever it holds.
            vh = torch.where(seen.any(0)[:, None], v[b, :, h // group], 0.0)
            out[b, some, h], size[b, some, h] = p @ vh, p @ vh.abs()
    return out, size
