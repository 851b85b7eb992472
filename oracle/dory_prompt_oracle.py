"""CPU restatement, in FP64, of the prompt side's operators: rotary positions, the rotated
and normalised append, chunk attention over the paged cache.

The reference has no kernels of these (its prompts run on vLLM), so the formulas themselves
are the oracle.  Everything returns FP64 values before the final rounding, and where a
tolerance needs it the size of the terms that were added up.
"""

from __future__ import annotations

import torch

E4M3_MAX = 448.0


def rotary(x: torch.Tensor, positions, cos_sin: torch.Tensor, interleaved: bool = False,
           inverse: bool = False):
    """x [T, H, D] -> (rotated FP64, |a c| + |b s| of each element, FP64).  A position outside
    the table gives zeros."""
    x = x.double()
    T, _, D = x.shape
    R = cos_sin.shape[1]
    table = cos_sin.double()
    y, size = x.clone(), x.abs()
    for t in range(T):
        p = int(positions[t])
        if not 0 <= p < table.shape[0]:
            y[t], size[t] = 0.0, 0.0
            continue
        c, s = table[p, :R // 2], table[p, R // 2:]
        if inverse:
            s = -s
        first = torch.arange(R // 2) * (2 if interleaved else 1)
        second = first + (1 if interleaved else R // 2)
        a, b = x[t][:, first], x[t][:, second]
        y[t][:, first], y[t][:, second] = a * c - b * s, b * c + a * s
        size[t][:, first] = (a * c).abs() + (b * s).abs()
        size[t][:, second] = (b * c).abs() + (a * s).abs()
    return y, size


def normalised(y: torch.Tensor, eps: float, weight: torch.Tensor | None = None,
               factor: float = 1.0):
    """(y / sqrt(sum y^2 + eps) [* (weight * factor)^2], the factor of each element)."""
    f = 1.0 / torch.sqrt((y * y).sum(-1, keepdim=True) + eps)
    f = f.expand_as(y).clone()
    if weight is not None:
        w = weight.double() * factor
        f *= (w * w).view(1, *y.shape[1:])
    return y * f, f


def chunk_attention(q: torch.Tensor, key: torch.Tensor, value: torch.Tensor, tables: torch.Tensor,
                    query_start, seq_lens, window: int, scale: float, gate=None):
    """q [T, NH, D]; key / value [blocks, B, NKV, D] (already dequantised); tables [S, width];
    any device.  -> (out FP64 [T, NH * D], softmax-weighted mean of |v|, FP64, same shape).
    Rows no sequence owns are NaN; a token that sees nothing gives zero; positions whose block
    id is outside the cache (or beyond the table) are left out.  Hidden positions take no part
    at all, whatever they hold."""
    T, NH, D = q.shape
    blocks, B, NKV, _ = key.shape
    G, dev = NH // NKV, q.device
    out = torch.full((T, NH, D), float("nan"), dtype=torch.float64, device=dev)
    size = torch.zeros_like(out)
    for i, length in enumerate(int(n) for n in seq_lens):
        t0, t1 = int(query_start[i]), int(query_start[i + 1])
        if t1 <= t0:
            continue
        out[t0:t1], size[t0:t1] = 0.0, 0.0
        p = length - (t1 - t0) + torch.arange(t1 - t0, device=dev)[:, None]
        pos = torch.arange(max(0, min(length, tables.shape[1] * B)), device=dev)
        ids = tables[i].to(dev)[pos // B].long()
        ok = (ids >= 0) & (ids < blocks)
        pos, ids = pos[ok], ids[ok]
        seen = pos[None] <= p
        if window:
            seen &= pos[None] > p - window
        some = seen.any(0)
        pos, ids, seen = pos[some], ids[some], seen[:, some]
        if not len(pos):
            continue
        rows = seen.any(1)
        for g in range(NKV):
            k, v = key[ids, pos % B, g].double(), value[ids, pos % B, g].double()
            finite = torch.isfinite(v).all()
            for h in range(g * G, (g + 1) * G):
                s = (q[t0:t1, h].double() @ k.T * scale).masked_fill(~seen, -torch.inf)
                w = torch.where(rows[:, None], torch.softmax(s, dim=-1), 0.0)
                if finite:
                    out[t0:t1, h], size[t0:t1, h] = w @ v, w @ v.abs()
                else:  # a hidden Inf or NaN must not reach a row
                    for j in range(t1 - t0):
                        see = seen[j]
                        out[t0 + j, h] = w[j, see] @ v[see]
                        size[t0 + j, h] = w[j, see] @ v[see].abs()
    out, size = out.reshape(T, NH * D), size.reshape(T, NH * D)
    if gate is not None:
        out, size = out * gate.double(), size * gate.double().abs()
    return out, size
