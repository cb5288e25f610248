"""Shared by the tests of the calls over chunks of several sequences: caches filled from seeded rows, and the
operators from their definitions in 64 bits."""
from __future__ import annotations

import math

import torch

import qauntrunner_amd as qr

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def randn(seed, *shape, dtype="f32", scale=1.0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(TORCH[dtype]).cuda()


def filled(heads, kv_heads, D, dtype, lengths, seed=1, max_seq=None, layers=1, layer=0):
    """A cache whose sequence i holds lengths[i] seeded positions, and their rows: [(K, V)] of [length, kv_heads, D]."""
    max_seq = max_seq or max(max(lengths), 1)
    kv = qr.PagedKvCache(layers, heads, kv_heads, D, max_seq, dtype, len(lengths))
    rows = []
    for i, n in enumerate(lengths):
        k, v = (randn(seed + 100 * i + j, n, kv_heads, D, dtype=dtype) for j in (0, 1))
        if n:
            kv.AppendRangeDev(layer, 0, k.view(n, -1), v.view(n, -1), dtype, seq_id=i)
        rows.append((k, v))
    return kv, rows


def head_map(heads, kv_heads):
    return [h * kv_heads // heads for h in range(heads)]


def attend64(q, k, v, pos0, scale, heads, kv_heads):
    """out [rows, heads, D], its size [rows, heads] and weights [kv_heads, pos0 + rows] in 64 bits; q [rows, heads, D],
    k / v [>= pos0 + rows, kv_heads, D].

    Weights p_t that are each off by e p_t, independently, move a row by the 2-norm sqrt(sum (e p_t |v_t|)^2): e times
    its size sqrt(sum (p_t |v_t|)^2), however far the row's own terms cancel (with one value per head to nothing)."""
    n = q.shape[0]
    end = pos0 + n
    late = torch.arange(end, device=q.device)[None] > pos0 + torch.arange(n, device=q.device)[:, None]
    out = torch.empty(n, heads, q.shape[2], dtype=torch.float64, device=q.device)
    size = torch.empty(n, heads, dtype=torch.float64, device=q.device)
    w = torch.zeros(kv_heads, end, dtype=torch.float64, device=q.device)
    for h, g in enumerate(head_map(heads, kv_heads)):
        kh, vh = k[:end, g].double(), v[:end, g].double()
        s = (q[:, h].double().contiguous() @ kh.t().contiguous()) * scale
        p = torch.softmax(s.masked_fill(late, -math.inf), 1)
        out[:, h] = p @ vh.contiguous()
        size[:, h] = (p.square() @ vh.square().sum(1)).sqrt()
        w[g] += p.sum(0)
    return out, size, w


def row_errors(got, want, size=None):
    """Largest 2-norm error of a row, relative to its norm (or its size, where that is more)."""
    got, want = got.double(), want.double()
    by = want.norm(dim=-1) if size is None else torch.maximum(want.norm(dim=-1), size)
    return float(((got - want).norm(dim=-1) / by.clamp_min(1e-30)).max()) if got.numel() else 0.0
