"""GPU tests of 8-bit caches: what the append writes and what comes back (qr_kv_append_norm_rope_dev, qr_kv_read_as_dev),
against the definition in 64 bits.  Codes and scales have one right answer: the values that come back are equal.  (K is
rounded from its value in 64 bits; that a sum of D products in another order lies on the other side of a border between two
codes has a chance of about D 2^-53 / 2^-4 for each value.)
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, randn
from tests.formutil import HIGHEST, LOWEST, e4m3_values
from tests.test_gpu_norm_rope import CHUNKS, EPS, THETA, close, want64

pytestmark = pytest.mark.gpu


def read_as(kv, ids, pos, n, dtype="f32", layer=0):
    k, v = (torch.full((sum(n), kv.KvDim), 7.0, dtype=TORCH[dtype], device="cuda") for _ in range(2))
    kv.ReadAsDev(layer, ids, pos, n, k, v)
    return (x.view(-1, kv.KvHeads, kv.HeadDim) for x in (k, v))


def same(got, want):
    assert torch.equal(got.isnan(), want.isnan())
    bad = (got.double() != want) & ~want.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} differ, first at {bad.nonzero()[0].tolist()}"


def put(kv, ids, pos, n, k, v, layer=0):
    kv.AppendNormRopeDev(layer, ids, pos, n, None, k.reshape(sum(n), -1), v.reshape(sum(n), -1), None, None, None, EPS, THETA, rotary_dim=0)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 96, 40, 1, 512])
@pytest.mark.parametrize("name", list(CHUNKS))
def test_append_and_read_back(gpu, name, D, act):
    """Norms, rotation and rounding of k, rounding of v; the queries as for the other caches."""
    heads, kv_heads, chunks = 4, 2, CHUNKS[name]
    rot = D // 2 * 2
    total, qw, kw = sum(c[2] for c in chunks), heads * D, kv_heads * D
    q, k, v = randn(3, total, qw + 2 * kw, dtype=act).split([qw, kw, kw], 1)
    qn, kn = (1 + 0.2 * randn(8 + i, D) for i in (0, 1))
    ids, p, n = ([c[i] for c in chunks] for i in range(3))
    q_out = torch.empty(total, qw, dtype=TORCH[act], device="cuda")
    with qr.PagedKvCache(1, heads, kv_heads, D, 600, "e4m3", 4) as kv:
        kv.AppendNormRopeDev(0, ids, p, n, q, k, v, q_out, qn, kn, EPS, THETA, rotary_dim=rot)
        pos = torch.tensor([x for a, m in zip(p, n) for x in range(a, a + m)], device="cuda")
        close(q_out.view(total, heads, D), want64(q.reshape(total, heads, D), qn, pos, rot, THETA), act)
        ko, vo = read_as(kv, ids, p, n)
        same(ko, e4m3_values(want64(k.reshape(total, kv_heads, D), kn, pos, rot, THETA, eps=float(torch.tensor(EPS)))))
        same(vo, e4m3_values(v.reshape(total, kv_heads, D)))
        for i, m in zip(ids, n):
            assert kv.seq_len(i) >= m


@pytest.mark.parametrize("rot,norms,rope", [(0, True, None), (20, True, None), (8, True, [2**20, 100000, 2**30]), (64, False, None), (32, True, [1000, 5, 77])])
def test_partial_rotation(gpu, rot, norms, rope):
    kv_heads, D, n = 3, 64, [5, 1, 40]
    total = sum(n)
    k, v = (randn(i, total, kv_heads * D, dtype="bf16") for i in (1, 2))
    kn = 1 + 0.2 * randn(9, D) if norms else None
    with qr.PagedKvCache(1, 6, kv_heads, D, 300, "e4m3", 3) as kv:
        kv.AppendNormRopeDev(0, [0, 1, 2], [7, 0, 250], n, None, k, v, None, None, kn, EPS, THETA, rotary_dim=rot, rope_pos0=rope)
        at = [x for a, m in zip(rope or [7, 0, 250], n) for x in range(a, a + m)]
        ko, vo = read_as(kv, [0, 1, 2], [7, 0, 250], n)
        same(ko, e4m3_values(want64(k.view(total, kv_heads, D), kn, torch.tensor(at, device="cuda"), rot, THETA, eps=float(torch.tensor(EPS)))))
        same(vo, e4m3_values(v.view(total, kv_heads, D)))


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 24])
@pytest.mark.parametrize("rows", [1, 37])
def test_every_magnitude(gpu, rows, D, act):
    """Ties between codes, values below a row's normal codes, rows of zeros, rows of the type's smallest and largest numbers,
    infinities and NaN."""
    kv_heads = 8
    x = randn(5, rows, kv_heads, D, dtype="f32")
    x[:, 0] = 0
    x[:, 1] *= torch.finfo(TORCH[act]).tiny
    x[:, 2] = torch.sign(x[:, 2]) * torch.finfo(TORCH[act]).max
    x[:, 3, ::3] = math.inf
    x[:, 3, 1::3] = -math.inf
    x[:, 4, D // 2] = math.nan
    # halves between two codes: 8.5, 9.5, ... sixteenths of a power of two, beside a row's largest 448
    ties = (torch.arange(D) % 16 + 16.5) * 2.0 ** (torch.arange(D) % 18 - 14.0)
    x[:, 5] = torch.where(ties > 448, 448.0, ties).cuda()
    x[:, 5, 0] = 448
    x[:, 6] = x[:, 5] * 2.0**-6
    x[:, 6, 0] = 448 * (1 + 2.0**-7)  # one step of bf16 above 448: the next exponent
    x[:, 7, :] = torch.logspace(-6, 0, D, base=10).cuda()
    x = x.to(TORCH[act])
    with qr.PagedKvCache(1, 8, kv_heads, D, 64, "e4m3") as kv:
        put(kv, [0], [3], [rows], x, -x)
        want = e4m3_values(x)
        for got, w in zip(read_as(kv, [0], [3], [rows]), (want, -want)):
            same(got, w)


def test_values_of_each_type(gpu):
    """bf16 and fp32 hold every value; fp16 rounds to nearest even."""
    x = randn(5, 50, 2 * 64) * torch.logspace(-9, 4, 50, base=10).cuda()[:, None]
    with qr.PagedKvCache(1, 2, 2, 64, 64, "e4m3") as kv:
        put(kv, [0], [0], [50], x, x)
        want = e4m3_values(x.view(50, 2, 64))
        for act in ("f32", "bf16", "f16"):
            for got in read_as(kv, [0], [0], [50], act):
                assert torch.equal(got, want.to(torch.float32).to(TORCH[act]))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [64, 72])
def test_read_as_of_the_other_caches(gpu, dtype, act, D):
    n = 300
    k, v = (randn(i, n, 2 * D, dtype=dtype) for i in (1, 2))
    with qr.PagedKvCache(1, 2, 2, D, 512, dtype) as kv:
        kv.AppendRangeDev(0, 0, k, v, dtype)
        for got, x in zip(read_as(kv, [0], [3], [290], act), (k, v)):
            assert torch.equal(got, x.view(n, 2, D)[3:293].to(TORCH[act]))


@pytest.mark.parametrize("D", [64, 128, 24])
def test_rows_beside_the_chunk_stay(gpu, D):
    """Appends of one row, of runs that end inside a page's steps and over what stood there leave the other slots alone."""
    kv_heads, n = 2, 520
    x = randn(1, n, kv_heads, D, dtype="bf16")
    with qr.PagedKvCache(1, 2, kv_heads, D, 600, "e4m3", 2) as kv:
        put(kv, [0], [0], [n], x, -x)
        want = x.clone()
        for i, (p, m) in enumerate([(0, 1), (255, 2), (17, 30), (500, 20), (33, 1), (16, 16), (100, 201)]):
            y = randn(50 + i, m, kv_heads, D, dtype="bf16", scale=10.0)
            put(kv, [0], [p], [m], y, -y)
            want[p:p + m] = y
            ko, vo = read_as(kv, [0], [0], [n])
            same(ko, e4m3_values(want))
            same(vo, -e4m3_values(want))
        assert kv.seq_len(0) == n and kv.seq_len(1) == 0
        # a page holds its slots' codes and scales
        assert kv.BytesUsed == 3 * 256 * kv_heads * (D + 1) * 2 and kv.BytesPerToken == kv_heads * (D + 1) * 2


def test_slots_never_written_read_as_zeros(gpu):
    x = randn(1, 1, 128, dtype="bf16")
    with qr.PagedKvCache(1, 2, 2, 64, 256, "e4m3") as kv:
        put(kv, [0], [9], [1], x, x)
        ko, vo = read_as(kv, [0], [0], [256])
        keep = torch.arange(256, device="cuda") != 9
        assert not ko[keep].any() and not vo[keep].any()


def test_layers_and_many_chunks(gpu):
    """More chunks than one launch takes, on a layer of several."""
    seqs, D = 150, 64
    n = [1 + i % 5 for i in range(seqs)]
    pos = [(37 * i) % 400 for i in range(seqs)]
    k, v = (randn(i, sum(n), 2, D, dtype="f16") for i in (1, 2))
    with qr.PagedKvCache(3, 2, 2, D, 512, "e4m3", seqs) as kv:
        put(kv, list(range(seqs)), pos, n, k, v, layer=1)
        ko, vo = read_as(kv, list(range(seqs)), pos, n, layer=1)
        same(ko, e4m3_values(k))
        same(vo, e4m3_values(v))


def test_a_captured_append_and_read(gpu):
    """Replays repeat the captured positions on new rows, beside eager work."""
    D, n = 128, 33
    k, v = (randn(i, n, 2 * D, dtype="bf16") for i in (1, 2))
    ko, vo = (torch.empty(n, 2 * D, device="cuda") for _ in range(2))
    with qr.PagedKvCache(1, 4, 2, D, 256, "e4m3", 2) as kv:
        kv.Reserve(4)
        put(kv, [0], [5], [n], k, v)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                put(kv, [0], [5], [n], k, v)
                kv.ReadAsDev(0, [0], [5], [n], ko, vo)
        torch.cuda.synchronize()
        for i in range(4):
            k.copy_(randn(10 + i, n, 2 * D, dtype="bf16"))
            v.copy_(randn(20 + i, n, 2 * D, dtype="bf16"))
            g.replay()
            torch.cuda.synchronize()
            same(ko.view(n, 2, D), e4m3_values(k.view(n, 2, D)))
            same(vo.view(n, 2, D), e4m3_values(v.view(n, 2, D)))
            put(kv, [1], [0], [n], v, k)  # eager work between
            for got, x in zip(read_as(kv, [1], [0], [n]), (v, k)):
                same(got, e4m3_values(x.view(n, 2, D)))


def test_another_stream(gpu):
    D, n = 64, 100
    s = torch.cuda.Stream()
    with qr.PagedKvCache(1, 2, 2, D, 256, "e4m3") as kv:
        k, v = (randn(i, n, 2 * D) for i in (1, 2))
        ko, vo = (torch.empty(n, 2 * D, device="cuda") for _ in range(2))
        s.wait_stream(torch.cuda.current_stream())
        kv.AppendNormRopeDev(0, [0], [0], [n], None, k, v, None, None, None, EPS, THETA, rotary_dim=0, stream=s)
        kv.ReadAsDev(0, [0], [0], [n], ko, vo, stream=s)
        s.synchronize()
        same(ko.view(n, 2, D), e4m3_values(k.view(n, 2, D)))
        same(vo.view(n, 2, D), e4m3_values(v.view(n, 2, D)))


def test_refusals(gpu):
    D = 64
    q, w, kept = torch.zeros(1, 2 * D, device="cuda"), torch.zeros(1, 2, 256, device="cuda"), torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")
    row = torch.zeros(1, 2 * D, device="cuda")
    with qr.PagedKvCache(1, 2, 2, D, 256, "e4m3") as kv:
        put(kv, [0], [0], [1], row, row)
        out = torch.empty_like(q)
        for call in (lambda: kv.Append(0, 0, [0.0], [0.0]), lambda: kv.AppendRangeDev(0, 0, row, row), lambda: kv.Read(0, 0, 1),
                     lambda: kv.AppendRopeDev(0, 0, q, row, row, 1e4), lambda: kv.Attention(0, 0, [0.0] * 2 * D, 1.0),
                     lambda: kv.AttentionDev(0, [0], [0], q, out, 1.0), lambda: kv.AttentionDevNoAlloc(0, [0], [0], q, out, 1.0),
                     lambda: kv.AttentionChunkDev(0, 0, q, out, 1.0), lambda: kv.DecodePlan(0, [0], [0]),
                     lambda: kv.AppendRopeStepDev(0, torch.zeros(1, dtype=torch.int32, device="cuda"), q, row, row, 1e4),
                     lambda: kv.AttentionStepDev(0, [0], torch.zeros(1, dtype=torch.int32, device="cuda"), q, out, 1.0),
                     lambda: kv.AttentionChunksDev(0, [0], [0], [1], q, out, 1.0, weights=w),
                     lambda: kv.EvictDev(0, [0], [1], 1, 1, 1, w, kept)):
            with pytest.raises(qr.QrInvalidArgument, match="8-bit"):
                call()
        with pytest.raises(ValueError, match="ReadAsDev"):
            kv.ReadDev(0, [0], [0], [1], row, out)
        with pytest.raises(qr.QrNotResident):
            kv2 = qr.PagedKvCache(1, 2, 2, D, 512, "e4m3")
            with kv2:
                kv2.ReadAsDev(0, [0], [0], [1], row, out)
        with pytest.raises(ValueError):
            kv.ReadAsDev(0, [0], [0], [1], row.half(), out)
        kv.AttentionChunksDev(0, [0], [0], [1], q, out, 1.0)
        assert not out.any()
