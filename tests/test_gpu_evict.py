"""GPU tests of eviction by accumulated attention weight (qr_kv_evict_dev), against its definition on the CPU: what is
kept, the rows that move and the weights are copies, so every comparison is exact."""
import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import attend64, filled, randn, row_errors

pytestmark = pytest.mark.gpu


def kept_of(w, n, first, heavy, recent):
    """Positions that one kv head keeps, from its n weights (a Python list)."""
    if n <= first + heavy + recent:
        return list(range(n))
    mid = range(first, n - recent)
    # NaN below every number, then the value, then the lower position
    best = sorted(mid, key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))[:heavy]
    return list(range(first)) + sorted(best) + list(range(n - recent, n))


def check(kv, rows, ids, lengths, first, heavy, recent, w, in_place=False):
    """Evicts and compares everything; returns kept."""
    n, kvh, keep = len(ids), kv.KvHeads, first + heavy + recent
    before = w.clone()
    out = w if in_place else randn(99, *w.shape)
    out0 = out.clone()
    kept = torch.full((n, kvh, keep), -7, dtype=torch.int32, device="cuda")
    kv.EvictDev(0, ids, lengths, first, heavy, recent, w, kept, kept_weights=None if in_place else out)
    got = kept.cpu().tolist()
    want_w = out0.cpu()
    for e, (s, m) in enumerate(zip(ids, lengths)):
        k, v = rows[s]
        k, v = k.clone(), v.clone()
        for g in range(kvh):
            wl = before[s, g].cpu().tolist()
            want = kept_of(wl, m, first, heavy, recent)
            assert got[e][g] == want + [-1] * (keep - len(want)), f"sequence {s}, head {g}"
            idx = torch.tensor(want, dtype=torch.long)
            k[:len(want), g], v[:len(want), g] = rows[s][0][idx.cuda(), g], rows[s][1][idx.cuda(), g]
            want_w[s, g, :m] = 0
            want_w[s, g, :len(want)] = before[s, g].cpu()[idx]
        if m:
            held = k.shape[0]
            ko, vo = (torch.empty(held, kvh * kv.HeadDim, dtype=k.dtype, device="cuda") for _ in range(2))
            kv.ReadDev(0, [s], [0], [held], ko, vo)
            # slots behind the kept ones, and behind the length, keep what they held
            assert torch.equal(ko.view_as(k), k) and torch.equal(vo.view_as(v), v), f"sequence {s}"
            rows[s] = (k, v)
    assert torch.equal(out.cpu().view(torch.int32), want_w.view(torch.int32))
    if not in_place:
        assert torch.equal(w.view(torch.int32), before.view(torch.int32))
    return kept


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("first,heavy,recent", [(4, 60, 100), (0, 1, 0), (0, 0, 30), (7, 0, 0), (0, 500, 1), (3, 296, 1)])
@pytest.mark.parametrize("dtype,kv_heads,D", [("f32", 2, 64), ("bf16", 2, 128), ("f16", 4, 64), ("bf16", 1, 96), ("f32", 1, 7), ("f16", 2, 20)])
def test_shapes(gpu, dtype, kv_heads, D, first, heavy, recent, in_place):
    lengths = [300, 0, 1029, 301, 37, 1]
    kv, rows = filled(kv_heads, kv_heads, D, dtype, lengths, max_seq=1100)
    with kv:
        w = randn(5, 6, kv_heads, 1100).exp()
        check(kv, rows, [2, 0, 1, 3, 5, 4], [1029, 300, 0, 299, 1, 37], first, heavy, recent, w, in_place)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("kind", ["equal", "few values", "negative", "special", "zeros"])
def test_ties_and_special_weights(gpu, kind, dtype, D):
    n = 2500
    kv, rows = filled(2, 2, D, dtype, [n])
    with kv:
        w = randn(4, 1, 2, n)
        if kind == "equal":
            w.fill_(0.5)
        elif kind == "few values":
            w = (w * 2).round() / 2
        elif kind == "zeros":
            w = torch.where(w > 0, 0.0, -0.0)
        elif kind == "special":
            w[0, 0, ::5] = float("nan")
            w[0, 0, 1::7] = float("inf")
            w[0, 0, 2::7] = -float("inf")
            w[0, 1] = float("nan")
        check(kv, rows, [0], [n], 3, 1700, 100, w)


@pytest.mark.parametrize("dtype,D", [("f16", 128), ("f32", 128)])
def test_long(gpu, dtype, D):
    n = 20011
    kv, rows = filled(2, 2, D, dtype, [n, 9000])
    with kv:
        check(kv, rows, [1, 0], [9000, n], 4, 5000, 1000, randn(4, 2, 2, n).exp())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", ["plain", "equal", "special"])
@pytest.mark.parametrize("first,heavy,recent", [(4, 9000, 1000), (0, 20000, 0), (9000, 0, 100), (0, 1, 9000), (1, 1, 20000)])
def test_rows_of_several_workgroups(gpu, kind, first, heavy, recent, in_place):
    n = 40007
    kv, rows = filled(3, 2, 8, "f32", [n, 17000, 900])
    with kv:
        w = randn(4, 3, 2, n).exp()
        if kind == "equal":
            w = (w * 0).add_(0.25)
            w[0, 0, 30000:] = 0.5
        elif kind == "special":
            w[0, 0, ::2] = float("nan")
            w[0, 0, 1::7] = float("inf")
            w[0, 1] = float("nan")
            w[1, 0, ::3] *= -1
        check(kv, rows, [1, 2, 0], [17000, 900, n], first, heavy, recent, w, in_place)


@pytest.mark.parametrize("first,heavy,recent", [(4, 9000, 1000), (0, 69998, 1)])
def test_captured_first(gpu, first, heavy, recent):
    """Captured with no call before: no workspace to share rows with."""
    n = 70001
    kv, rows = filled(1, 1, 8, "f32", [n])
    with kv:
        w, out, w0 = randn(4, 1, 1, n).exp(), randn(5, 1, 1, n), randn(6, 1, 1, n)
        keep = first + heavy + recent
        kept = torch.zeros(1, 1, keep, dtype=torch.int32, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            kv.EvictDev(0, [0], [n], first, heavy, recent, w0, kept, kept_weights=out)
        w0.copy_(w)
        g.replay()
        want = kept_of(w[0, 0].tolist(), n, first, heavy, recent)
        assert kept[0, 0].tolist() == want
        idx = torch.tensor(want, device="cuda")
        assert torch.equal(out[0, 0, :keep], w[0, 0, idx]) and not out[0, 0, keep:].any()
        ko, vo = (torch.empty(keep, 8, device="cuda") for _ in range(2))
        kv.ReadDev(0, [0], [0], [keep], ko, vo)
        assert torch.equal(ko, rows[0][0][idx, 0]) and torch.equal(vo, rows[0][1][idx, 0])


def test_more_sequences_than_one_launch_takes(gpu):
    n = 70
    lengths = [20 + (i * 13) % 90 for i in range(n)]
    kv, rows = filled(1, 1, 64, "bf16", lengths, max_seq=128)
    with kv:
        check(kv, rows, list(range(n)), lengths, 2, 30, 16, randn(4, n, 1, 128).exp())


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 64), ("f16", 48)])
def test_a_serving_loop(gpu, dtype, D):
    """Prompt, tokens one by one, eviction at the budget, more tokens: the cache then attends as one that holds only
    the kept rows, at rotation positions of its own."""
    heads, kvh, act = 8, 2, "f32"
    first, heavy, recent, budget = 2, 60, 64, 126
    with qr.PagedKvCache(1, heads, kvh, D, 512, dtype, 2) as kv:
        w = torch.zeros(2, kvh, 512, device="cuda")
        norm = 1 + 0.2 * randn(1, D)
        kept = torch.empty(2, kvh, budget, dtype=torch.int32, device="cuda")
        scale = D ** -0.5
        held, seen, sums = [0, 0], [0, 0], torch.zeros(2, kvh, 512, dtype=torch.float64, device="cuda")
        model = [None, None]  # the rows that the cache should hold
        for step, new in enumerate([(100, 37), (1, 1), (40, 1), (1, 120), (9, 9), (1, 1)]):
            total = sum(new)
            qkv = randn(40 + step, total, (heads + 2 * kvh) * D)
            q, k, v = qkv.split([heads * D, kvh * D, kvh * D], 1)
            qo, out = torch.empty(total, heads * D, device="cuda"), torch.empty(total, heads * D, device="cuda")
            kv.AppendNormRopeDev(0, [0, 1], held, list(new), q, k, v, qo, norm, norm, 1e-6, 10000.0, rope_pos0=seen)
            ko, vo = (torch.empty(total, kvh * D, dtype={"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype], device="cuda") for _ in range(2))
            kv.ReadDev(0, [0, 1], held, list(new), ko, vo)
            kv.AttentionChunksDev(0, [0, 1], held, list(new), qo, out, scale, weights=w)
            at = 0
            for s, m in enumerate(new):
                rows = (ko[at:at + m].view(m, kvh, D), vo[at:at + m].view(m, kvh, D))
                model[s] = rows if model[s] is None else tuple(torch.cat(x) for x in zip(model[s], rows))
                o, size, x = attend64(qo[at:at + m].view(m, heads, D), *model[s], held[s], scale, heads, kvh)
                assert row_errors(out[at:at + m].view(m, heads, D), o, size) <= 2.0 ** -15
                sums[s, :, :held[s] + m] += x
                held[s] += m
                seen[s] += m
                at += m
            assert row_errors(w, sums) <= 2.0 ** -14  # several steps' errors
            kv.EvictDev(0, [0, 1], held, first, heavy, recent, w, kept)
            sums.copy_(w)
            for s in (0, 1):
                if held[s] > budget:
                    idx = kept[s].long()
                    model[s] = tuple(torch.stack([x[idx[g], g] for g in range(kvh)], 1) for x in model[s])
                    held[s] = budget
                    kv.Truncate(budget, s)
                    assert kv.seq_len(s) == budget


def test_captured_and_replayed(gpu):
    kv, rows = filled(2, 2, 64, "bf16", [400, 90], max_seq=512)
    with kv:
        w, out = randn(5, 2, 2, 512).exp(), torch.zeros(2, 2, 512, device="cuda")
        kept = torch.zeros(2, 2, 100, dtype=torch.int32, device="cuda")
        args = (0, [0, 1], [400, 90], 4, 60, 36)

        def fill():
            for s, n in ((0, 400), (1, 90)):
                kv.AppendRangeDev(0, 0, rows[s][0].reshape(n, -1), rows[s][1].reshape(n, -1), "bf16", seq_id=s)

        def state():
            ko, vo = (torch.empty(490, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv.ReadDev(0, [0, 1], [0, 0], [400, 90], ko, vo)
            torch.cuda.synchronize()
            return [x.clone() for x in (kept, out, ko, vo)]

        kv.EvictDev(*args, w, kept, kept_weights=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.EvictDev(*args, w, kept, kept_weights=out)
        for j in range(3):
            w.copy_(randn(60 + j, 2, 2, 512).exp())
            fill()
            g.replay()
            got = state()
            fill()
            kept.zero_()
            out.zero_()
            kv.EvictDev(*args, w, kept, kept_weights=out)
            assert all(torch.equal(a, b) for a, b in zip(got, state()))


def test_refusals(gpu):
    kv, _ = filled(2, 2, 64, "f32", [300, 20], max_seq=512)
    with kv:
        w = torch.zeros(2, 2, 512, device="cuda")

        def go(ids=(0,), ln=(300,), first=1, heavy=2, recent=3, w=w, kept=None, layer=0, **kw):
            n = torch.empty(len(ids), 2, max(first + heavy + recent, 0), dtype=torch.int32, device="cuda") if kept is None else kept
            kv.EvictDev(layer, list(ids), list(ln), first, heavy, recent, w, n, **kw)

        for kw in (dict(ids=(0, 0), ln=(300, 300)), dict(ids=(2,)), dict(layer=1), dict(ln=(-1,)), dict(first=0, heavy=0, recent=0), dict(heavy=600)):
            with pytest.raises(qr.QrInvalidArgument):
                go(**kw)
        with pytest.raises(qr.QrNotResident):
            go(ids=(1,), ln=(257,))
        with pytest.raises(qr.QrOutOfRange):
            go(ln=(513,))
        for kw in (dict(first=-1), dict(w=w.cpu()), dict(w=w[:, :, :300]), dict(w=w.double()), dict(ln=(300, 20)),
                   dict(kept=torch.empty(1, 2, 6, device="cuda")), dict(kept=torch.empty(1, 2, 5, dtype=torch.int32, device="cuda")),
                   dict(kept_weights=w[:1])):
            with pytest.raises(ValueError):
                go(**kw)
