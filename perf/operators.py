"""Timing cases of the operators of a serving step over several sequences: the append of chunks with
query / key norms and rotation, causal attention of those chunks over the paged cache (with the
attention weight that each cached position received, where asked for), and eviction from the cache
by that weight.

Every case is one call for one layer.  Sizes are those of the tests and of the other timing cases
(a tiny GQA shape, the 8B and 70B GQA shapes, 28 heads over 4, 24 over 8) and generic ones between.

    own                 False: plain torch in 32 bits; True: this library's entry points
    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs and the cache of one pass, on the GPU
    run(state)          one pass; returns its outputs
    work(case)          bytes and flops a pass cannot do without
    exact(case, seed)   the outputs from the definitions in 64 bits
"""
import math

import torch

own = False

PAGE = 256
EPS = 1e-6
THETA = 500000.0
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token of each of 16 running sequences enters the cache: the launch counts
        dict(name="append-decode-bf16", kind="append", heads=32, kv=8, D=128, rot=128, dtype="bf16", act="bf16",
             seqs=16, ctx_lo=130, ctx_hi=16000, new_lo=1, new_hi=1),
        # prompt chunks of four sequences from a fused QKV product
        dict(name="append-prompts-bf16", kind="append", heads=32, kv=8, D=128, rot=128, dtype="bf16", act="bf16",
             seqs=4, ctx_lo=1, ctx_hi=6144, new_lo=500, new_hi=2500),
        # an odd chunk in the default cache type, half of each head rotated
        dict(name="append-prompt-f32", kind="append", heads=28, kv=4, D=128, rot=64, dtype="f32", act="f32",
             seqs=1, ctx_lo=777, ctx_hi=777, new_lo=1001, new_hi=1001),
        # the smallest attention call: a tiny model's layer, two sequences, one token each
        dict(name="attend-tiny-f32", kind="attend", heads=8, kv=2, D=64, dtype="f32", act="f32", seqs=2, ctx_lo=400,
             ctx_hi=512, new_lo=1, new_hi=1, weights=True),
        # a decode batch of very different lengths that keeps the weights for eviction
        dict(name="attend-decode-f16-weights", kind="attend", heads=32, kv=8, D=128, dtype="f16", act="f16", seqs=16,
             ctx_lo=130, ctx_hi=16000, new_lo=1, new_hi=1, weights=True),
        # speculative verify of a batch, 70B shape, queries in 32 bits
        dict(name="attend-verify-bf16", kind="attend", heads=64, kv=8, D=128, dtype="bf16", act="f32", seqs=8,
             ctx_lo=2000, ctx_hi=32000, new_lo=5, new_hi=9, weights=False),
        # a chunk of one long prompt
        dict(name="attend-prompt-bf16", kind="attend", heads=32, kv=8, D=128, dtype="bf16", act="bf16", seqs=1,
             ctx_lo=6144, ctx_hi=6144, new_lo=2048, new_hi=2048, weights=False),
        # prompt chunks of several sequences, odd lengths, with weights
        dict(name="attend-prompts-bf16-weights", kind="attend", heads=32, kv=8, D=128, dtype="bf16", act="bf16",
             seqs=6, ctx_lo=1, ctx_hi=3001, new_lo=101, new_hi=1501, weights=True),
        # the default cache type, an odd group of heads, with weights
        dict(name="attend-prompts-f32-weights", kind="attend", heads=28, kv=4, D=128, dtype="f32", act="f32", seqs=3,
             ctx_lo=11, ctx_hi=1501, new_lo=61, new_hi=501, weights=True),
        # one sequence that runs against its budget: 256 of 2304 positions leave
        dict(name="evict-step-f16", kind="evict", kv=8, D=128, dtype="f16", seqs=1, len_lo=2304, len_hi=2304, first=4,
             heavy=1020, recent=1024),
        # after the prompts of a batch: long caches cut down to the budget, short ones left
        dict(name="evict-batch-bf16", kind="evict", kv=8, D=128, dtype="bf16", seqs=16, len_lo=3000, len_hi=17001,
             first=4, heavy=2044, recent=2048),
        # a very long prompt in the default cache type
        dict(name="evict-long-f32", kind="evict", kv=8, D=128, dtype="f32", seqs=1, len_lo=65536, len_hi=65536,
             first=0, heavy=6144, recent=2048),
    ]


# ------------------------------------------------------------------ drawn cases
GQA = [(8, 2), (16, 16), (24, 8), (28, 4), (32, 8), (64, 8)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges of listed(); none costs more than the largest listed one of its kind."""
    kind = rng.choice(["append", "attend", "attend", "evict"])
    while True:
        heads, kv = rng.choice(GQA)
        D = rng.choice([64, 128, 128, 128, 96])
        dtype = rng.choice(["f32", "f16", "bf16"])
        act = rng.choice(["f32", dtype])
        seqs = _log(rng, 1, 16)
        ctx_hi = _log(rng, 20, 32000)
        ctx_lo = max(1, ctx_hi // rng.choice([1, 3, 30]))
        new_hi = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 2500)])
        new_lo = max(1, new_hi // rng.choice([1, 4]))
        if kind == "append":
            c = dict(kind=kind, heads=heads, kv=kv, D=D, rot=rng.choice([D, D, D // 2]), dtype=dtype, act=act,
                     seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new_lo=new_lo, new_hi=new_hi)
        elif kind == "attend":
            c = dict(kind=kind, heads=heads, kv=kv, D=D, dtype=dtype, act=act, seqs=seqs, ctx_lo=ctx_lo,
                     ctx_hi=ctx_hi, new_lo=new_lo, new_hi=new_hi, weights=rng.random() < 0.5)
        else:
            keep = _log(rng, 64, 8192)
            len_hi = keep + _log(rng, 1, 57000)
            recent, first = keep // rng.choice([2, 4]), rng.choice([0, 4])
            c = dict(kind=kind, kv=kv, D=D, dtype=dtype, seqs=seqs, len_lo=max(1, len_hi // rng.choice([1, 2, 6])),
                     len_hi=len_hi, first=first, heavy=keep - first - recent, recent=recent)
        if _cost(c) <= max(_cost(x) for x in listed() if x["kind"] == kind):
            return c


def _cost(c):
    """Rough units of work for bounding a drawn case: 32-bit arithmetic costs more per flop, the caches and the
    padded scores of the plain form have to fit."""
    w = work(c)
    if c["kind"] == "attend":
        pad = c["seqs"] * c["heads"] * c["new_hi"] * (c["ctx_hi"] + c["new_hi"])
        slow = c["dtype"] == "f32" or c["D"] == 96
        return max(w["flops"] * (4 if slow else 1), 50 * w["bytes"], 400 * pad)
    return w["bytes"]


# ------------------------------------------------------------------ sizes
def _spread(lo, hi, n):
    """n lengths from hi down to lo, evenly over their logarithm."""
    if n == 1:
        return [hi]
    return [int(round(hi * (lo / hi) ** (i / (n - 1)))) for i in range(n)]


def _ctx(c):
    return _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])


def _new(c):
    return _spread(c["new_lo"], c["new_hi"], c["seqs"])[::-1]


def _lens(c):
    return _spread(c["len_lo"], c["len_hi"], c["seqs"])


def _keep(c):
    return c["first"] + c["heavy"] + c["recent"]


def work(c):
    kvD, es = c["kv"] * c["D"], SIZE[c["dtype"]]
    if c["kind"] == "append":
        rows, qD, a = sum(_new(c)), c["heads"] * c["D"], SIZE[c["act"]]
        return {"bytes": rows * ((2 * qD + 2 * kvD) * a + 2 * kvD * es), "flops": rows * (qD + kvD) * 8}
    if c["kind"] == "attend":
        rows, qD, a = sum(_new(c)), c["heads"] * c["D"], SIZE[c["act"]]
        keys = sum(x + y for x, y in zip(_ctx(c), _new(c)))
        pairs = sum(y * x + y * (y + 1) // 2 for x, y in zip(_ctx(c), _new(c)))
        return {"bytes": keys * 2 * kvD * es + 2 * rows * qD * a + (8 * c["kv"] * keys if c["weights"] else 0),
                "flops": 4 * c["heads"] * c["D"] * pairs}
    keep = _keep(c)
    over = [n for n in _lens(c) if n > keep]
    return {"bytes": sum(4 * c["kv"] * n for n in _lens(c)) + len(over) * keep * (4 * kvD * es + 8 * c["kv"]),
            "flops": sum(4 * c["kv"] * n for n in _lens(c))}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _inputs(c, seed):
    """The tensors of a case, the same for both sides: cached rows [sum of lengths][kv D] of the sequences one after
    another, and what the call takes."""
    g, dt = _gen(seed), TORCH[c["dtype"]]
    kvD = c["kv"] * c["D"]
    s = {}
    if c["kind"] == "evict":
        rows = sum(_lens(c))
        # positions receive very different weight: a few most of it
        s["weights"] = torch.exp(2.0 * _randn(g, c["seqs"], c["kv"], max(_lens(c))))
    else:
        rows, act = sum(_ctx(c)), TORCH[c["act"]]
        new = sum(_new(c))
        if c["kind"] == "append":
            s["qkv"] = _randn(g, new, c["heads"] * c["D"] + 2 * kvD, dtype=act)
            s["q_norm"] = 1 + 0.2 * _randn(g, c["D"])
            s["k_norm"] = 1 + 0.2 * _randn(g, c["D"])
        else:
            rows += new  # the chunk's own rows are in the cache when it attends
            s["q"] = (1.5 * _randn(g, new, c["heads"] * c["D"])).to(act)
            if c["weights"]:
                # what earlier steps left: of the size of one step's, so that neither hides the other
                s["weights"] = 1e-3 * torch.rand(c["seqs"], c["kv"], _max_seq(c), device="cuda", generator=g)
    s["k"] = _randn(g, rows, kvD, dtype=dt)
    s["v"] = _randn(g, rows, kvD, dtype=dt)
    return s


def _max_seq(c):
    n = max(_lens(c)) if c["kind"] == "evict" else max(x + y for x, y in zip(_ctx(c), _new(c)))
    return -(-n // PAGE) * PAGE


def _cached(c):
    if c["kind"] == "evict":
        return _lens(c)
    return _ctx(c) if c["kind"] == "append" else [x + y for x, y in zip(_ctx(c), _new(c))]


def prepare(c, seed):
    s = _inputs(c, seed)
    s["case"] = c
    new = _lens(c) if c["kind"] == "evict" else _new(c)
    s["ids"], s["new"] = list(range(c["seqs"])), new
    cached, max_seq = _cached(c), _max_seq(c)
    pages = c["seqs"] * (max_seq // PAGE)
    at = _offsets(cached)
    dt = TORCH[c["dtype"]]
    kvD = c["kv"] * c["D"]
    if c["kind"] == "evict":
        out_rows = sum(min(n, _keep(c)) for n in new)
        s["pos0"] = [0] * c["seqs"]
        s["out_lens"] = [min(n, _keep(c)) for n in new]
    else:
        out_rows = sum(new)
        s["pos0"] = _ctx(c)
    if own:
        import qauntrunner_amd as qr

        kv = qr.PagedKvCache(1, c.get("heads", c["kv"]), c["kv"], c["D"], max_seq, c["dtype"], c["seqs"])
        kv.Reserve(pages)
        for i, n in enumerate(cached):
            if n:
                kv.AppendRangeDev(0, 0, s["k"][at[i]:at[i + 1]], s["v"][at[i]:at[i + 1]], c["dtype"], seq_id=i)
        s["kv"] = kv
        if c["kind"] != "attend":
            s["k_out"] = torch.empty(out_rows, kvD, dtype=dt, device="cuda")
            s["v_out"] = torch.empty_like(s["k_out"])
        if c["kind"] == "append":
            s["q_out"] = torch.empty(out_rows, c["heads"] * c["D"], dtype=TORCH[c["act"]], device="cuda")
        elif c["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
        else:
            full = torch.zeros(c["seqs"], c["kv"], max_seq, device="cuda")
            full[:, :, :s["weights"].shape[2]] = s["weights"]
            s["weights"], s["kept_weights"] = full, torch.zeros_like(full)
            s["kept"] = torch.empty(c["seqs"], c["kv"], _keep(c), dtype=torch.int32, device="cuda")
    else:
        # pages in no order, as a cache that has run for a while holds them
        g = _gen(seed + 1)
        table = torch.randperm(pages, device="cuda", generator=g).view(c["seqs"], -1)
        s["table"] = table
        s["pool_k"] = torch.zeros(pages, c["kv"], PAGE, c["D"], dtype=dt, device="cuda")
        s["pool_v"] = torch.zeros_like(s["pool_k"])
        seq = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(cached)).cuda()
        pos = torch.cat([torch.arange(n) for n in cached]).cuda()
        s["pool_k"][table[seq, pos // PAGE], :, pos % PAGE] = s["k"].view(-1, c["kv"], c["D"])
        s["pool_v"][table[seq, pos // PAGE], :, pos % PAGE] = s["v"].view(-1, c["kv"], c["D"])
        # which sequence and which of its rows each new row is
        s["seq"] = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(new)).cuda()
        s["off"] = torch.cat([torch.arange(n) for n in new]).cuda()
        s["pos0_t"] = torch.tensor(s["pos0"]).cuda()
        s["len_t"] = torch.tensor(new).cuda()
        if c["kind"] == "evict":
            out = s["out_lens"]
            s["out_seq"] = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(out)).cuda()
            s["out_off"] = torch.cat([torch.arange(n) for n in out]).cuda()
            s["kept_weights"] = torch.zeros(c["seqs"], c["kv"], max_seq, device="cuda")
    del s["k"], s["v"]
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own_append(s) if kind == "append" else _own_attend(s) if kind == "attend" else _own_evict(s)
    return _plain_append(s) if kind == "append" else _plain_attend(s) if kind == "attend" else _plain_evict(s)


def _own_append(s):
    c, kv = s["case"], s["kv"]
    qD, kvD = c["heads"] * c["D"], c["kv"] * c["D"]
    q, k, v = s["qkv"].split([qD, kvD, kvD], dim=1)
    kv.AppendNormRopeDev(0, s["ids"], s["pos0"], s["new"], q, k, v, s["q_out"], s["q_norm"], s["k_norm"], EPS, THETA,
                         rotary_dim=c["rot"])
    kv.ReadDev(0, s["ids"], s["pos0"], s["new"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attend(s):
    c = s["case"]
    s["kv"].AttentionChunksDev(0, s["ids"], s["pos0"], s["new"], s["q"], s["out"], 1 / math.sqrt(c["D"]),
                               weights=s.get("weights"))
    return (s["out"], s["weights"]) if c["weights"] else s["out"]


def _own_evict(s):
    c, kv = s["case"], s["kv"]
    kv.EvictDev(0, s["ids"], s["new"], c["first"], c["heavy"], c["recent"], s["weights"], s["kept"],
                kept_weights=s["kept_weights"])
    kv.ReadDev(0, s["ids"], s["pos0"], s["out_lens"], s["k_out"], s["v_out"])
    return s["kept"], s["kept_weights"], s["k_out"], s["v_out"]


def _norm_rope(x, w, pos, rot):
    """x [rows][heads][D] in 32 bits: each head's row normed and rotated (angles in 64 bits)."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    half = rot // 2
    inv = THETA ** (torch.arange(half, device=x.device, dtype=torch.float64) * (-2.0 / rot))
    ang = pos.double()[:, None] * inv
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    heads, kv, D = c["heads"], c["kv"], c["D"]
    rows = s["qkv"].shape[0]
    q, k, v = s["qkv"].float().split([heads * D, kv * D, kv * D], dim=1)
    pos = s["pos0_t"][s["seq"]] + s["off"]
    q = _norm_rope(q.reshape(rows, heads, D), s["q_norm"], pos, c["rot"])
    k = _norm_rope(k.reshape(rows, kv, D), s["k_norm"], pos, c["rot"])
    page, slot = s["table"][s["seq"], pos // PAGE], pos % PAGE
    dt = s["pool_k"].dtype
    s["pool_k"][page, :, slot] = k.to(dt)
    s["pool_v"][page, :, slot] = v.reshape(rows, kv, D).to(dt)
    return (q.reshape(rows, -1).to(s["qkv"].dtype), s["pool_k"][page, :, slot].reshape(rows, -1),
            s["pool_v"][page, :, slot].reshape(rows, -1))


def _plain_attend(s):
    c = s["case"]
    n, heads, kv, D = c["seqs"], c["heads"], c["kv"], c["D"]
    G, nq = heads // kv, max(s["new"])
    k = s["pool_k"][s["table"]].permute(0, 2, 1, 3, 4).reshape(n * kv, -1, D).float()
    v = s["pool_v"][s["table"]].permute(0, 2, 1, 3, 4).reshape(n * kv, -1, D).float()
    L = k.shape[1]
    q = torch.zeros(n, nq, heads, D, device=k.device)
    q[s["seq"], s["off"]] = s["q"].float().view(-1, heads, D)
    q = q.view(n, nq, kv, G, D).permute(0, 2, 3, 1, 4).reshape(n * kv, G * nq, D)
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1 / math.sqrt(D))
    row = torch.arange(nq, device=k.device)
    last = s["pos0_t"][:, None] + row  # the last position that each row sees
    seen = torch.arange(L, device=k.device) <= last[..., None]  # [n][nq][L]
    x = x.view(n, kv, G, nq, L).masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n * kv, G * nq, L), v).view(n, kv, G, nq, D).permute(0, 3, 1, 2, 4).reshape(n, nq, -1)
    o = o[s["seq"], s["off"]].to(s["q"].dtype)
    if not c["weights"]:
        return o
    x *= (row < s["len_t"][:, None])[:, None, None, :, None]
    s["weights"] += x.sum((2, 3), dtype=torch.float64).float()
    return o, s["weights"]


def _plain_evict(s):
    c = s["case"]
    n, kv, D, keep = c["seqs"], c["kv"], c["D"], _keep(c)
    w = s["weights"]
    L = w.shape[2]
    at, length = torch.arange(L, device=w.device), s["len_t"][:, None]
    held = at < length
    safe = held & ((at < c["first"]) | (at >= length - c["recent"]))
    key = torch.where(safe[:, None], math.inf, torch.where(held[:, None], w, -1.0))
    best = torch.sort(key, dim=2, descending=True, stable=True)[1][:, :, :keep]
    best = torch.where(best < length[:, None], best, L)
    kept = torch.sort(best, dim=2)[0]
    if kept.shape[2] < keep:
        kept = torch.cat([kept, kept.new_full((n, kv, keep - kept.shape[2]), L)], 2)
    count = torch.minimum(length, length.new_tensor(keep))[:, None]  # [n][1][1]
    src = torch.where(kept < L, kept, 0)
    whole = s["kept_weights"]
    new = torch.zeros_like(whole)
    new[:, :, :keep] = torch.where(kept < L, w.gather(2, src), 0.0)[:, :, :new.shape[2]]
    held = torch.arange(whole.shape[2], device=w.device) < length
    whole.copy_(torch.where(held[:, None], new, whole))
    head = torch.arange(kv, device=w.device)[None, :, None]
    page = torch.gather(s["table"][:, None].expand(n, kv, -1), 2, src // PAGE)
    rows_k, rows_v = s["pool_k"][page, head, src % PAGE], s["pool_v"][page, head, src % PAGE]  # [n][kv][keep][D]
    ok = (torch.arange(keep, device=w.device) < count).expand(n, kv, keep)
    to = torch.where(ok, torch.arange(keep, device=w.device), 0)
    page = torch.gather(s["table"][:, None].expand(n, kv, -1), 2, to // PAGE)
    head = head.expand(n, kv, keep)
    s["pool_k"][page[ok], head[ok], to[ok] % PAGE] = rows_k[ok]
    s["pool_v"][page[ok], head[ok], to[ok] % PAGE] = rows_v[ok]
    rows_k = rows_k.permute(0, 2, 1, 3)[s["out_seq"], s["out_off"]].reshape(-1, kv * D)
    rows_v = rows_v.permute(0, 2, 1, 3)[s["out_seq"], s["out_off"]].reshape(-1, kv * D)
    return torch.where(kept < L, kept, -1).int(), whole, rows_k, rows_v


# ------------------------------------------------------------------ 64 bits
def exact(c, seed):
    s = _inputs(c, seed)
    kv, D = c["kv"], c["D"]
    at = _offsets(_cached(c))
    if c["kind"] == "append":
        heads = c["heads"]
        x = s["qkv"].double()
        pos = torch.cat([torch.arange(p, p + m, device="cuda") for p, m in zip(_ctx(c), _new(c))]).double()
        half = c["rot"] // 2
        turn = torch.outer(pos, torch.exp(torch.arange(half, device="cuda").double() * (-2 * math.log(THETA) / c["rot"])))
        unit = torch.polar(torch.ones_like(turn), turn)[:, None]  # rotation as a complex product

        def heads_of(y, w):
            y = y.reshape(y.shape[0], -1, D)
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * unit
            return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1).flatten(1)

        return (heads_of(x[:, :heads * D], s["q_norm"]), heads_of(x[:, heads * D:(heads + kv) * D], s["k_norm"]),
                x[:, (heads + kv) * D:])
    if c["kind"] == "attend":
        G = c["heads"] // kv
        outs, first = [], 0
        w = s["weights"].double() if c["weights"] else None
        for i, (p, m) in enumerate(zip(_ctx(c), _new(c))):
            k = s["k"][at[i]:at[i + 1]].double().view(-1, kv, D)
            v = s["v"][at[i]:at[i + 1]].double().view(-1, kv, D)
            q = s["q"][first:first + m].double().view(m, kv, G, D)
            first += m
            late = torch.arange(p + m, device="cuda")[None] > p + torch.arange(m, device="cuda")[:, None]
            o = torch.empty(m, kv, G, D, dtype=torch.float64, device="cuda")
            for h in range(kv):
                for j in range(G):
                    a = q[:, h, j].contiguous() @ k[:, h].t().contiguous() / math.sqrt(D)
                    a = torch.softmax(a.masked_fill(late, -math.inf), 1)
                    o[:, h, j] = a @ v[:, h].contiguous()
                    if w is not None:
                        w[i, h, :p + m] += a.sum(0)
            outs.append(o.view(m, -1))
        return (torch.cat(outs), w) if c["weights"] else torch.cat(outs)
    keep, ks, vs = _keep(c), [], []
    kept = torch.full((c["seqs"], kv, keep), -1, dtype=torch.int32, device="cuda")
    left = torch.zeros(c["seqs"], kv, _max_seq(c), dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lens(c)):
        k, v = (t[at[i]:at[i + 1]].double().view(n, kv, D) for t in (s["k"], s["v"]))
        idx = torch.arange(n, device="cuda").expand(kv, n)
        if n > keep:
            mid = s["weights"][i, :, c["first"]:n - c["recent"]]
            order = torch.argsort(mid, dim=1, descending=True, stable=True)[:, :c["heavy"]] + c["first"]
            idx = torch.cat([idx[:, :c["first"]], order.sort(1)[0], idx[:, n - c["recent"]:]], 1)
        m = idx.shape[1]
        kept[i, :, :m] = idx.int()
        left[i, :, :m] = s["weights"][i].double().gather(1, idx)
        pick = idx.t()[..., None].expand(m, kv, D)
        ks.append(k.gather(0, pick).reshape(m, -1))
        vs.append(v.gather(0, pick).reshape(m, -1))
    return kept, left, torch.cat(ks), torch.cat(vs)
