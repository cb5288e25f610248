"""Shared by the tests of 8-bit caches and of attention in its other forms: the definitions in 64 bits."""
from __future__ import annotations

import math

import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, head_map, randn

LOWEST, HIGHEST = -117, 119  # exponents of a row's scale


def e4m3_values(x):
    """The values that rows x [..., D] stand as in an 8-bit cache, in 64 bits: c 2^e with e the smallest exponent that
    keeps the largest finite |x| at or below 448 2^e, c the nearest number of 3 bits behind its first (even on a tie)."""
    x = x.double()
    finite = torch.where(x.abs() < math.inf, x, 0.0)
    units = torch.tensor([2.0**k for k in range(LOWEST, HIGHEST + 1)], dtype=torch.float64).to(x.device)
    top = finite.abs().amax(-1, keepdim=True)
    unit = units[torch.searchsorted(448 * units, top).clamp(max=units.numel() - 1)]
    y = (x / unit).clamp(-448, 448)
    grid = torch.tensor([0.0] + [m * 2.0**-9 for m in range(1, 8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                        dtype=torch.float64).to(x.device)  # every number of the type, its code the index
    a = y.abs().nan_to_num(0.0)
    hi = torch.searchsorted(grid, a).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.where(y.isnan(), math.nan, torch.copysign(grid[code], y) * unit)


def filled_as(heads, kv_heads, D, dtype, lengths, seed=1, max_seq=None, layers=1, layer=0, edit=None):
    """A cache of any type whose sequence i holds lengths[i] seeded positions, and the values it holds: [(K, V)] of [length,
    kv_heads, D] (64 bits for an 8-bit cache, whose rows were bf16).  edit(i, k, v) may change a sequence's rows first."""
    max_seq = max_seq or max(max(lengths), 1)
    kv = qr.PagedKvCache(layers, heads, kv_heads, D, max_seq, dtype, len(lengths))
    rows = []
    for i, n in enumerate(lengths):
        k, v = (randn(seed + 100 * i + j, n, kv_heads, D, dtype="bf16" if dtype == "e4m3" else dtype) for j in (0, 1))
        if edit:
            edit(i, k, v)
        if n:
            kv.AppendNormRopeDev(layer, [i], [0], [n], None, k.view(n, -1), v.view(n, -1), None, None, None, 1e-6, 1e4, rotary_dim=0)
        rows.append((e4m3_values(k), e4m3_values(v)) if dtype == "e4m3" else (k, v))
    return kv, rows


def forms64(q, k, v, pos, scale, heads, kv_heads, cap=0.0, slopes=None, window=0, first=0, full=0):
    """out [rows, heads, D] and its size [rows, heads] in 64 bits: row j of q [rows, heads, D] stands at position pos + j of
    the keys k / v [positions, kv_heads, D]; a row that sees nothing is zeros."""
    n, L, dev = q.shape[0], k.shape[0], q.device
    p, t = (pos + torch.arange(n, device=dev))[:, None], torch.arange(L, device=dev)[None]
    seen = (t >= first) & ((t <= p) | (t < full))
    if window:
        seen &= t > p - window
    out = torch.zeros(n, heads, q.shape[2], dtype=torch.float64, device=dev)
    size = torch.zeros(n, heads, dtype=torch.float64, device=dev)
    for h, g in enumerate(head_map(heads, kv_heads)):
        kh, vh = k[:, g].double(), v[:, g].double()
        z = (q[:, h].double().contiguous() @ torch.where(seen.any(0)[:, None], kh, 0.0).t().contiguous()) * scale
        if cap:
            z = cap * torch.tanh(z / cap)
        if slopes is not None:
            z = z - slopes[h].double() * (p - t).abs()
        w = torch.softmax(z.masked_fill(~seen, -math.inf), 1).nan_to_num(0.0) if L else z
        vh = torch.where(seen.any(0)[:, None], vh, 0.0)
        out[:, h] = w @ vh.contiguous()
        size[:, h] = (w.square() @ vh.square().sum(1)).sqrt()
    return out, size
