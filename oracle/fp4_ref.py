"""The 4-bit pools and the operators around them, from their definitions in 64 bits.  TEST INFRASTRUCTURE ONLY (see
`oracle/__init__.py`); the reference has no 4-bit cache, so the definitions in include/mlb_paged_kv.h are the pin.

Pool: uint8 [num_blocks, Hkv, 17, Dh / 2]; rows 0..15 e2m1 codes (dim 2i in the low nibble), row 16 the scale bytes at
[run of 32 dims][2 * (token % 8) + token // 8].
"""

from __future__ import annotations

import math

import numpy as np
import torch

RUN, BLOCK = 32, 16
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SCALES = np.array([(b % 8) / 8 * 2.0**-14 if b < 8 else (1 + (b % 8) / 8) * 2.0 ** (b // 8 - 15) for b in range(227)])


def _nearest(x: np.ndarray, table: np.ndarray) -> np.ndarray:
    """Index of the nearest entry of an ascending table, the even index of two equally near ones."""
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    up, down = table[hi] - x, x - table[hi - 1]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def quantise(x: torch.Tensor) -> tuple[np.ndarray, np.ndarray]:
    """(codes [..., Dh] with the sign in bit 3, scale bytes [..., Dh / 32]) of rows of any float type."""
    v = x.double().numpy()
    v = np.clip(np.where(np.isnan(v), 0.0, v), -61440.0, 61440.0)
    runs = v.reshape(*v.shape[:-1], -1, RUN)
    byte = _nearest(np.abs(runs).max(-1) / 6.0, SCALES)
    s = SCALES[byte][..., None]
    ratio = np.divide(np.abs(runs), s, out=np.zeros_like(runs), where=s > 0)
    code = _nearest(np.minimum(ratio, 6.0), LEVELS) | (np.signbit(runs).astype(np.int64) << 3)
    return code.reshape(v.shape).astype(np.uint8), byte.astype(np.uint8)


def append(pool: torch.Tensor, slots: list[int], x: torch.Tensor) -> None:
    """Rows x [N, Hkv, Dh] into the pool (CPU) at their slots; slots out of range are skipped."""
    code, byte = quantise(x)
    p = pool.numpy()
    for i, s in enumerate(slots):
        if not 0 <= s < p.shape[0] * BLOCK:
            continue
        b, t = divmod(s, BLOCK)
        p[b, :, t] = code[i, :, 0::2] | (code[i, :, 1::2] << 4)
        for r in range(byte.shape[-1]):
            p[b, :, BLOCK, r * BLOCK + 2 * (t % 8) + t // 8] = byte[i, :, r]


def values(pool: torch.Tensor) -> torch.Tensor:
    """Every stored value in 64 bits: [num_blocks, 16, Hkv, Dh] (the 16-bit pools' layout).  Scale bytes that no
    append makes (above 226) give NaN."""
    p = pool.cpu().numpy()
    nb, hkv, _, half = p.shape
    code = np.empty((nb, hkv, BLOCK, 2 * half), dtype=np.int64)
    code[..., 0::2], code[..., 1::2] = p[:, :, :BLOCK] & 15, p[:, :, :BLOCK] >> 4
    order = np.array([2 * (t % 8) + t // 8 for t in range(BLOCK)])
    byte = p[:, :, BLOCK].reshape(nb, hkv, half // BLOCK, BLOCK)[..., order].swapaxes(2, 3)
    scale = np.append(SCALES, [np.nan] * 29)[byte]
    v = np.where(code >= 8, -1.0, 1.0) * LEVELS[code % 8] * np.repeat(scale, RUN, axis=-1)
    return torch.from_numpy(v).transpose(1, 2).contiguous()


def norm_rope(x: torch.Tensor, weight: torch.Tensor | None, positions: torch.Tensor, cos_sin: torch.Tensor,
              eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(the rotated rows, |a| + |b| of each element's rotation pair: what its rounding errors scale with)."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    r = cos_sin.shape[1]
    a, b = y[..., :r // 2], y[..., r // 2:r]
    c, s = cos_sin.double()[positions][:, None].split(r // 2, dim=-1) if r else (a, b)
    mag = a.abs() + b.abs()
    out = torch.cat([a * c - b * s, b * c + a * s, y[..., r:]], dim=-1)
    return out, torch.cat([mag, mag, y[..., r:].abs()], dim=-1)


def attention(q: torch.Tensor, k_values: torch.Tensor, v_values: torch.Tensor, seqs, scale: float | None = None):
    """Causal paged attention of q [N, H, Dh] over `values` pools, and how far a kernel may be from it before its
    output rounding.  seqs: (num_cached, num_new, block_ids) of each row.

    The bound, per element, with A = sum p |v| / sum p (L keys, Dh products a score):
    - P rounded to fp16: half a step, 2^-11 of each term -> A 2^-11; weights below 2^-14 of a unit lose at most 2^-25
      each -> L 2^-25 max|v|;
    - a score's fp32 sum of Dh exact products, 2^-23 of sum |q k| for each of Dh / 16 + 4 additions (an MMA adds 16
      products at once, truncating), and three roundings more on the way into the exponent; an error e in the exponent
      moves numerator and denominator by a factor 1 + e each -> 2 e A;
    - exp2: 2^-22 relative -> 2 * 2^-22 A;
    - fp32 sums over L / 16 pages, the merge of warps and pieces: 2^-23 A for each of L / 16 + 64 additions, twice."""
    n, h, dh = q.shape
    hkv = k_values.shape[2]
    g = h // hkv
    scale = 1.0 / math.sqrt(dh) if scale is None else scale
    out, bound = torch.zeros(n, h, dh, dtype=torch.float64), torch.zeros(n, h, dh, dtype=torch.float64)
    at = 0
    for cached, new, ids in seqs:
        length = cached + new
        pages = torch.tensor(ids[:-(-length // BLOCK)], dtype=torch.long)
        k = k_values[pages].reshape(-1, hkv, dh)[:length].repeat_interleave(g, dim=1)  # [L, H, Dh]
        v = v_values[pages].reshape(-1, hkv, dh)[:length].repeat_interleave(g, dim=1)
        x = q[at:at + new].double()
        s = torch.einsum("nhd,lhd->hnl", x, k) * scale
        mag = torch.einsum("nhd,lhd->hnl", x.abs(), k.abs()) * scale
        hidden = torch.arange(length)[None, :] > cached + torch.arange(new)[:, None]
        p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
        a = torch.einsum("hnl,lhd->nhd", p, v.abs())
        e = ((dh / 16 + 4 + 3) * 2.0**-23 * mag.masked_fill(hidden, 0.0).amax(-1)).transpose(0, 1)[..., None]
        out[at:at + new] = torch.einsum("hnl,lhd->nhd", p, v)
        bound[at:at + new] = (a * (2.0**-11 + 2 * e + 2 * 2.0**-22 + 2 * (length / 16 + 64) * 2.0**-23)
                              + length * 2.0**-25 * v.abs().amax(0))
        at += new
    return out, bound
