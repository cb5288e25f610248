"""GPU tests of the append with query / key norms and rotation over chunks of several sequences
(qr_kv_append_norm_rope_dev) and of reading rows back (qr_kv_read_dev), against the definition in 64 bits.

Tolerances, per element relative to its head's largest value: a norm's sum and the products round a few times at
2^-24, the angle's fraction of a turn is exact to 2^-25 turns = 2^-22.3 rad: 2^-20 in fp32; a value stored in 16 bits
adds half a step of its own, eps / 2.
"""
import math

import pytest
import torch

import qauntrunner_amd as qr
from tests.chunkutil import TORCH, randn

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 500000.0


def want64(x, w, pos, rot, theta, eps=EPS):
    """x [rows, heads, D] -> normed (w None: not) and rotated, in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = rot // 2
    a = pos.double()[:, None] * theta ** (-2.0 * torch.arange(half, dtype=torch.float64, device=x.device) / max(rot, 1))
    c, s = a.cos()[:, None], a.sin()[:, None]
    lo, hi = x[..., :half], x[..., half:rot]
    return torch.cat([lo * c - hi * s, lo * s + hi * c, x[..., rot:]], -1)


def close(got, want, kind):
    """Within 2^-20 of the head's largest value, and half a step of the stored type."""
    scale = want.abs().amax(-1, keepdim=True)
    bound = 2.0 ** -20 * scale
    if kind != "f32":
        fi = torch.finfo(TORCH[kind])
        bound = bound + want.abs() * (fi.eps / 2) * (1 + 2.0 ** -9) + fi.smallest_normal * fi.eps
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, the worst by {float(((got.double() - want).abs() / bound).max()):.3g} bounds"


CHUNKS = {
    "decode": [(0, 0, 1), (1, 300, 1), (2, 255, 1), (3, 256, 1)],
    "ragged": [(3, 250, 70), (0, 0, 1), (1, 31, 2), (2, 7, 0)],
    "prompts": [(0, 5, 517), (2, 256, 256), (1, 0, 8)],
}


def call(kv, chunks, heads, kv_heads, D, dtype, act, rot=None, norms=True, fused=True, rope=None, theta=THETA, seed=3, in_place=False, queries=True):
    total = sum(c[2] for c in chunks)
    rot = D if rot is None else rot
    qw, kw = heads * D, kv_heads * D
    if fused:
        q, k, v = randn(seed, total, qw + 2 * kw, dtype=act).split([qw, kw, kw], 1)
    else:
        q, k, v = (randn(seed + i, total, n, dtype=act) for i, n in enumerate((qw, kw, kw)))
    qn, kn = (1 + 0.2 * randn(seed + 5 + i, D) for i in (0, 1)) if norms else (None, None)
    q_in = q.clone()
    q_out = (q if in_place else torch.empty(total, qw, dtype=TORCH[act], device="cuda")) if queries else None
    ids, p, n = ([c[i] for c in chunks] for i in range(3))
    kv.AppendNormRopeDev(0, ids, p, n, q if queries else None, k, v, q_out, qn, kn, EPS, theta, rotary_dim=rot, rope_pos0=rope)
    at = [x for c, r in zip(chunks, rope or p) for x in range(r, r + c[2])]
    pos = torch.tensor(at, device="cuda", dtype=torch.int64)
    if queries:
        close(q_out.view(total, heads, D), want64(q_in.reshape(total, heads, D), qn, pos, rot, theta), act)
    ko, vo = (torch.empty(total, kw, dtype=TORCH[dtype], device="cuda") for _ in range(2))
    kv.ReadDev(0, ids, p, n, ko, vo)
    close(ko.view(total, kv_heads, D), want64(k.reshape(total, kv_heads, D), kn, pos, rot, theta), dtype)
    close(vo.view(total, kv_heads, D), v.reshape(total, kv_heads, D).double(), dtype)
    return q_out, ko, vo


SHAPES = [(8, 2, 64, None), (32, 8, 128, None), (28, 4, 128, 64), (6, 2, 96, None), (4, 2, 96, 32), (5, 5, 40, 16), (3, 1, 20, 6), (2, 1, 512, None),
          (4, 1, 256, 64), (2, 2, 1, 0), (4, 2, 7, 2), (8, 2, 64, 0)]


@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("heads,kv_heads,D,rot", SHAPES)
@pytest.mark.parametrize("dtype,act", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("f32", "bf16")])
def test_shapes(gpu, dtype, act, heads, kv_heads, D, rot, name):
    with qr.PagedKvCache(1, heads, kv_heads, D, 600, dtype, 4) as kv:
        call(kv, CHUNKS[name], heads, kv_heads, D, dtype, act, rot)
        for s, p, n in CHUNKS[name]:
            assert kv.seq_len(s) == (p + n if n else 0)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_norms_strides_and_no_queries(gpu, act, norms, fused):
    with qr.PagedKvCache(1, 8, 2, 128, 600, "bf16", 4) as kv:
        for queries in (True, False):
            call(kv, CHUNKS["ragged"], 8, 2, 128, "bf16", act, norms=norms, fused=fused, queries=queries)


@pytest.mark.parametrize("D", [128, 24])
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_queries_in_place(gpu, act, D):
    with qr.PagedKvCache(1, 8, 2, D, 600, "f16", 4) as kv:
        call(kv, CHUNKS["prompts"], 8, 2, D, "f16", act, fused=False, in_place=True)


@pytest.mark.parametrize("offset", [1, 2, 4])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_rows_off_vector_alignment(gpu, act, offset):
    """Rows whose addresses are aligned to their element only."""
    heads, kv_heads, D, n = 4, 2, 64, 37
    with qr.PagedKvCache(1, heads, kv_heads, D, 64, "bf16", 1) as kv:
        width = (heads + 2 * kv_heads) * D + 2 * offset + 1
        big = randn(1, n, width, dtype=act)
        q, k, v = big[:, offset:offset + 256], big[:, offset + 256:offset + 384], big[:, offset + 384:offset + 512]
        flat = torch.empty(n * 256 + offset, dtype=TORCH[act], device="cuda")
        q_out = flat[offset:].view(n, 256)
        w = (1 + 0.2 * randn(2, D + 1))[1:]
        kv.AppendNormRopeDev(0, [0], [3], [n], q, k, v, q_out, w, w, EPS, THETA)
        pos = torch.arange(3, 3 + n, device="cuda")
        close(q_out.reshape(n, heads, D), want64(q.reshape(n, heads, D), w, pos, D, THETA), act)
        ko, vo = (torch.empty(n, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kv.ReadDev(0, [0], [3], [n], ko, vo)
        close(ko.view(n, 2, D), want64(k.reshape(n, 2, D), w, pos, D, THETA), "bf16")
        close(vo.view(n, 2, D), v.reshape(n, 2, D).double(), "bf16")


def test_far_rotation_positions(gpu):
    """Angles in 64 bits: positions to 2^31, apart from the slots."""
    with qr.PagedKvCache(1, 4, 2, 128, 300, "f32", 3) as kv:
        for theta in (10000.0, 500000.0, 1.0):
            call(kv, [(0, 0, 5), (1, 255, 3), (2, 17, 2)], 4, 2, 128, "f32", "f32", rope=[131072, 1000003, 2 ** 31 - 4], theta=theta)


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 64), ("f32", 64), ("bf16", 96)])
def test_neighbours_keep_their_rows(gpu, dtype, D):
    """Chunks that start and end inside a run of 8 slots leave the slots beside them."""
    kvh, n = 2, 300
    with qr.PagedKvCache(1, 4, kvh, D, n, dtype, 2) as kv:
        k0, v0 = (randn(50 + i, n, kvh * D, dtype=dtype) for i in (0, 1))
        for s in (0, 1):
            kv.AppendRangeDev(0, 0, k0, v0, dtype, seq_id=s)
        for p, m in ((3, 1), (5, 9), (8, 8), (250, 13), (17, 30), (299, 1)):
            call(kv, [(1, p, m)], 4, kvh, D, dtype, "f32", seed=p)
            ko, vo = torch.empty_like(k0), torch.empty_like(v0)
            kv.ReadDev(0, [1], [0], [n], ko, vo)
            keep = torch.ones(n, dtype=torch.bool, device="cuda")
            keep[p:p + m] = False
            assert torch.equal(ko[keep], k0[keep]) and torch.equal(vo[keep], v0[keep])
            kv.AppendRangeDev(0, 0, k0, v0, dtype, seq_id=1)
        ko, vo = torch.empty_like(k0), torch.empty_like(v0)
        kv.ReadDev(0, [0], [0], [n], ko, vo)
        assert torch.equal(ko, k0) and torch.equal(vo, v0)


def test_read_equals_the_host_copy(gpu):
    for dtype, D in (("f32", 64), ("bf16", 128), ("f16", 64), ("bf16", 24)):
        with qr.PagedKvCache(2, 4, 2, D, 700, dtype, 2) as kv:
            k, v = (randn(i, 600, 2 * D, dtype=dtype) for i in (0, 1))
            kv.AppendRangeDev(1, 0, k, v, dtype, seq_id=1)
            ko, vo = (torch.empty(404, 2 * D, dtype=TORCH[dtype], device="cuda") for _ in range(2))
            kv.ReadDev(1, [1, 1, 1], [200, 0, 597], [400, 1, 3], ko, vo)
            want = torch.cat([torch.arange(200, 600), torch.arange(0, 1), torch.arange(597, 600)]).cuda()
            assert torch.equal(ko, k[want]) and torch.equal(vo, v[want])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_every_rounding(gpu, dtype):
    """Every upper half of an fp32 value with lower halves at, below and above the places where it rounds: the bits that
    the append without norms and rotation stores, and NaN for NaN."""
    hi = torch.arange(65536, dtype=torch.int32, device="cuda") << 16
    low = torch.tensor([0, 1, 0x0FFF, 0x1000, 0x1001, 0x7FFF, 0x8000, 0x8001, 0xFFFF], dtype=torch.int32, device="cuda")
    x = (hi[:, None] | low).view(torch.float32).reshape(-1, 256).contiguous()
    n = x.shape[0]
    with qr.PagedKvCache(1, 2, 2, 128, n, dtype, 1) as kv:
        def rows():
            out = [torch.empty(n, 256, dtype=TORCH[dtype], device="cuda") for _ in range(2)]
            kv.ReadDev(0, [0], [0], [n], *out)
            return out
        kv.AppendRangeDev(0, 0, x, x, "f32")
        want = rows()
        kv.AppendNormRopeDev(0, [0], [0], [n], None, x, x, None, None, None, EPS, THETA, rotary_dim=0)
        for got, ref in zip(rows(), want):
            assert torch.equal(got.isnan(), x.isnan())
            assert torch.equal(got.view(torch.int16)[~x.isnan()], ref.view(torch.int16)[~x.isnan()])


def test_zero_rows_and_infinities(gpu):
    """A row of zeros stays zero (eps > 0); an infinite value makes its own head NaN, not its neighbours."""
    with qr.PagedKvCache(1, 2, 2, 64, 16, "f32", 1) as kv:
        q, k, v = (randn(i, 2, 128) for i in range(3))
        q[0] = 0
        k[1, 3] = float("inf")
        w = torch.ones(64, device="cuda")
        out = torch.empty_like(q)
        kv.AppendNormRopeDev(0, [0], [2], [2], q, k, v, out, w, w, EPS, THETA)
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        kv.ReadDev(0, [0], [2], [2], ko, vo)
        assert not out[0].any() and torch.isfinite(out[1]).all()
        assert torch.isnan(ko[1, 3]) and torch.isfinite(ko[1, 64:]).all() and torch.isfinite(ko[0]).all()
        assert torch.equal(vo, v)


def test_more_chunks_than_one_launch_takes(gpu):
    n = 150
    with qr.PagedKvCache(1, 4, 2, 64, 64, "bf16", n) as kv:
        call(kv, [(i, i % 40, (i * 7) % 5) for i in range(n)], 4, 2, 64, "bf16", "bf16")


def test_captured_and_replayed(gpu):
    with qr.PagedKvCache(1, 8, 2, 128, 600, "bf16", 3) as kv:
        kv.Reserve(12)
        q, k, v = (randn(i, 30, w, dtype="bf16") for i, w in enumerate((1024, 256, 256)))
        wn = 1 + 0.2 * randn(9, 128)
        args = (0, [2, 0], [250, 3], [20, 10])
        out = torch.empty_like(q)
        kv.AppendNormRopeDev(*args, q, k, v, out, wn, wn, EPS, THETA)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv.AppendNormRopeDev(*args, q, k, v, out, wn, wn, EPS, THETA)
        read = lambda: [kv.ReadDev(*args, *r) or r for r in [(torch.empty_like(k), torch.empty_like(v))]][0]  # noqa: E731
        for j in range(3):
            for i, x in enumerate((q, k, v)):
                x.copy_(randn(30 + 3 * j + i, *x.shape, dtype="bf16"))
            g.replay()
            torch.cuda.synchronize()
            got = (out.clone(), *read())
            out.zero_()
            kv.AppendNormRopeDev(*args, q, k, v, out, wn, wn, EPS, THETA)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (out, *read())))


def test_refusals(gpu):
    with qr.PagedKvCache(1, 4, 2, 64, 300, "bf16", 2) as kv:
        q, k, v = (torch.zeros(3, w, device="cuda") for w in (256, 128, 128))
        out, w = torch.empty_like(q), torch.ones(64, device="cuda")

        def go(ids=(0,), pos=(0,), n=(3,), q=q, k=k, v=v, out=out, qn=w, kn=w, eps=EPS, theta=THETA, **kw):
            kv.AppendNormRopeDev(kw.pop("layer", 0), list(ids), list(pos), list(n), q, k, v, out, qn, kn, eps, theta, **kw)

        with pytest.raises(qr.QrInvalidArgument, match="two entries"):
            go((0, 0), (0, 5), (1, 2))
        with pytest.raises(qr.QrOutOfRange):
            go(pos=(298,))
        with pytest.raises(qr.QrInvalidArgument):
            go(ids=(2,))
        with pytest.raises(qr.QrInvalidArgument):
            go(layer=1)
        for kw in (dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=-2), dict(theta=0.0), dict(theta=float("inf")), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(rope_pos0=[-1]), dict(rope_pos0=[2 ** 31 - 2])):
            with pytest.raises(qr.QrInvalidArgument):
                go(**kw)
        for kw in (dict(q=None), dict(out=None), dict(k=k.half()), dict(v=v[:2]), dict(q=q.cpu()), dict(out=out.t()), dict(qn=w.half()),
                   dict(kn=w[:32]), dict(rope_pos0=[0, 1]), dict(out=q.expand(3, 256)[:, :128]), dict(q=q[:1].expand(3, 256)),
                   dict(q=torch.zeros(3, 512, device="cuda")[:, ::2])):
            with pytest.raises(ValueError):
                go(**kw)
        both = torch.zeros(4, 256, device="cuda")
        with pytest.raises(ValueError, match="overlaps"):
            go(q=both[:3], out=both[1:])
        assert kv.SeqLen == 0 and kv.BytesUsed == 0  # nothing of a refused call was done
