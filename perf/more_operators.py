"""Timing cases of serving operators over a cache of 8 bits and of attention in its other forms: the append that
quantises as it writes, reading such a cache back, attention whose scores are capped or fall with distance, under
windows, document and prefix masks, and attention of a batch that shares a long prefix.

Every case is one pass for one layer.  Sizes are those of the tests and of the other timing cases (a tiny GQA shape, the
8B and 70B GQA shapes, 28 heads over 4, 24 over 8) and generic ones between.

    own                 False: plain torch; True: this library's entry points
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
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def listed():
    base = dict(prefix=0, groups=1, cap=0.0, slopes=False, window=0, docs=False, full=False)
    return [
        # one token of each of 16 running sequences enters an 8-bit cache: the launch counts
        dict(name="quant-decode-bf16", kind="quant", heads=32, kv=8, D=128, rot=128, act="bf16", seqs=16, ctx_lo=130,
             ctx_hi=16000, new_lo=1, new_hi=1),
        # prompt chunks of four sequences from a fused QKV product
        dict(name="quant-prompts-bf16", kind="quant", heads=32, kv=8, D=128, rot=128, act="bf16", seqs=4, ctx_lo=1,
             ctx_hi=6144, new_lo=500, new_hi=2500),
        # an odd chunk in 32 bits, half of each head rotated
        dict(name="quant-prompt-f32", kind="quant", heads=28, kv=4, D=128, rot=64, act="f32", seqs=1, ctx_lo=777,
             ctx_hi=777, new_lo=1001, new_hi=1001),
        # the cached rows of a batch back as 16-bit values, as a sequence that moves elsewhere takes them
        dict(name="read-batch-bf16", kind="read", heads=32, kv=8, D=128, act="bf16", seqs=16, ctx_lo=3000, ctx_hi=17001),
        # a decode batch of very different lengths over the 8-bit cache
        dict(base, name="attend-decode-e4m3", kind="attend", heads=32, kv=8, D=128, dtype="e4m3", act="bf16", seqs=16,
             ctx_lo=130, ctx_hi=16000, new_lo=1, new_hi=1),
        # a chunk of one long prompt over the 8-bit cache
        dict(base, name="attend-prompt-e4m3", kind="attend", heads=32, kv=8, D=128, dtype="e4m3", act="bf16", seqs=1,
             ctx_lo=6144, ctx_hi=6144, new_lo=2048, new_hi=2048),
        # the smallest attention call: a tiny model's layer, capped scores, one token of two sequences
        dict(base, name="forms-tiny-f32", kind="attend", heads=8, kv=2, D=64, dtype="f32", act="f32", seqs=2, ctx_lo=400,
             ctx_hi=512, new_lo=1, new_hi=1, cap=30.0, window=300),
        # a decode batch of a model with capped scores, a layer with a window
        dict(base, name="forms-decode-f16", kind="attend", heads=32, kv=8, D=128, dtype="f16", act="f16", seqs=16,
             ctx_lo=130, ctx_hi=16000, new_lo=1, new_hi=1, cap=50.0, window=4096),
        # prompt chunks of several documents packed behind each other, capped scores
        dict(base, name="forms-prompts-bf16", kind="attend", heads=32, kv=8, D=128, dtype="bf16", act="bf16", seqs=6,
             ctx_lo=1, ctx_hi=3001, new_lo=101, new_hi=1501, cap=50.0, docs=True),
        # scores that fall with distance, a prefix that every row sees, an odd group of heads, the default cache type
        dict(base, name="forms-prompts-f32", kind="attend", heads=28, kv=4, D=128, dtype="f32", act="f32", seqs=3,
             ctx_lo=11, ctx_hi=1501, new_lo=61, new_hi=501, slopes=True, full=True),
        # one token of 64 sequences behind one long system prompt
        dict(base, name="shared-decode-bf16", kind="attend", heads=32, kv=8, D=128, dtype="bf16", act="bf16", seqs=64,
             ctx_lo=10, ctx_hi=1000, new_lo=1, new_hi=1, prefix=8192),
        # speculative verify of sequences behind two prompts, 70B shape, 8-bit cache
        dict(base, name="shared-verify-e4m3", kind="attend", heads=64, kv=8, D=128, dtype="e4m3", act="bf16", seqs=16,
             ctx_lo=100, ctx_hi=4001, new_lo=5, new_hi=9, prefix=16001, groups=2),
    ]


# ------------------------------------------------------------------ drawn cases
GQA = [(8, 2), (16, 16), (24, 8), (28, 4), (32, 8), (64, 8)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the ranges of listed(); none costs more than the largest listed one of its kind."""
    kind = rng.choice(["quant", "read", "attend", "attend", "attend"])
    while True:
        heads, kv = rng.choice(GQA)
        D = rng.choice([64, 128, 128])
        seqs = _log(rng, 1, 64)
        ctx_hi = _log(rng, 20, 32000)
        ctx_lo = max(1, ctx_hi // rng.choice([1, 3, 30]))
        new_hi = rng.choice([1, _log(rng, 2, 16), _log(rng, 17, 2500)])
        new_lo = max(1, new_hi // rng.choice([1, 4]))
        c = dict(kind=kind, heads=heads, kv=kv, D=D, act=rng.choice(["f32", "f16", "bf16", "bf16"]), seqs=seqs,
                 ctx_lo=ctx_lo, ctx_hi=ctx_hi)
        if kind != "read":
            c.update(new_lo=new_lo, new_hi=new_hi)
        if kind == "quant":
            c["rot"] = rng.choice([D, D, D // 2])
        if kind == "attend":
            c["dtype"] = rng.choice(["f32", "f16", "bf16", "e4m3", "e4m3"])
            c["act"] = rng.choice([c["act"], "bf16" if c["dtype"] == "e4m3" else c["dtype"]])
            shared = rng.random() < 0.35
            c.update(prefix=_log(rng, 100, 16000) if shared else 0, groups=rng.choice([1, 1, 2]) if shared else 1,
                     cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.25,
                     window=rng.choice([0, 0, _log(rng, 10, 8192)]), docs=rng.random() < 0.2, full=rng.random() < 0.2)
        most = [_cost(x) for x in listed() if x["kind"] == kind]
        if all(cost <= max(of) for cost, of in zip(_cost(c), zip(*most))):
            return c


def _cost(c):
    """Units of work for bounding a drawn case: time (32-bit arithmetic costs more per flop), and the padded scores and
    keys of the plain form, which have to fit."""
    w = work(c)
    if c["kind"] != "attend":
        return w["bytes"], 0
    pad = c["seqs"] * c["heads"] * c["new_hi"] * (c["prefix"] + c["ctx_hi"] + c["new_hi"])
    keys = c["seqs"] * c["kv"] * c["D"] * (c["ctx_hi"] + c["new_hi"])
    return max(w["flops"] * (8 if "f32" in (c["dtype"], c["act"]) else 1), 200 * w["bytes"]), max(pad, keys / 4)


# ------------------------------------------------------------------ sizes
def _spread(lo, hi, n):
    """n lengths from hi down to lo, evenly over their logarithm."""
    if n == 1:
        return [hi]
    return [int(round(hi * (lo / hi) ** (i / (n - 1)))) for i in range(n)]


def _ctx(c):
    return _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])


def _new(c):
    return [0] * c["seqs"] if c["kind"] == "read" else _spread(c["new_lo"], c["new_hi"], c["seqs"])[::-1]


def _cached(c):
    """Slots that a sequence holds before the pass (attention: its own rows are in the cache)."""
    return [x + y for x, y in zip(_ctx(c), _new(c))] if c["kind"] == "attend" else _ctx(c)


def _groups(c):
    """The runs of sequences [a, b) that share a prefix."""
    n, g = c["seqs"], min(c["groups"], c["seqs"])
    return [(n * i // g, n * (i + 1) // g) for i in range(g)]


def _first(c):
    """First position that each chunk's rows see: a document that starts a third into the context."""
    return [(c["prefix"] + x) // 3 if c["docs"] else 0 for x in _ctx(c)]


def _full(c):
    """Positions below it are seen by every row of the chunk: half of its own rows too."""
    return [c["prefix"] + x + y // 2 if c["full"] else 0 for x, y in zip(_ctx(c), _new(c))]


def _slopes(c):
    return [2.0 ** (-8.0 * (h + 1) / c["heads"]) for h in range(c["heads"])]


def _seen(c):
    """Of each sequence: (query, position) pairs, positions of the prefix and of its own that some row sees."""
    out = []
    for x, y, first, full in zip(_ctx(c), _new(c), _first(c), _full(c)):
        pairs, lo, p0 = 0, None, c["prefix"] + x
        if not c["window"]:
            both = max(0, min(y, full - p0))  # rows that see up to `full`, the others up to themselves
            pairs = both * (full - first) + sum(range(p0 + both + 1 - first, p0 + y + 1 - first))
            lo = first
        else:
            for j in range(y):
                a = max(first, p0 + j - c["window"] + 1)
                pairs += max(p0 + j + 1, full) - a
                lo = a if lo is None else min(lo, a)
        hi = max(p0 + y, full)
        out.append((pairs, min(lo, c["prefix"]), hi - max(lo, c["prefix"])))
    return out


def work(c):
    kvD, qD, a = c["kv"] * c["D"], c["heads"] * c["D"], SIZE[c["act"]]
    if c["kind"] == "quant":  # the rows in, the queries out, codes and scales in the cache and back as values
        rows = sum(_new(c))
        return {"bytes": rows * ((2 * qD + 2 * kvD) * a + 2 * kvD + 2 * c["kv"]), "flops": rows * (qD + kvD) * 8}
    if c["kind"] == "read":
        rows = sum(_ctx(c))
        return {"bytes": rows * (2 * kvD * (1 + a) + 2 * c["kv"]), "flops": rows * 2 * kvD}
    rows, seen = sum(_new(c)), _seen(c)
    keys = sum(k for _, _, k in seen)
    for x, y in _groups(c):
        keys += c["prefix"] - min(lo for _, lo, _ in seen[x:y])
    per = 2 * kvD * SIZE[c["dtype"]] + (2 * c["kv"] if c["dtype"] == "e4m3" else 0)
    return {"bytes": keys * per + 2 * rows * qD * a, "flops": 4 * qD * sum(p for p, _, _ in seen)}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 31)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _rows_type(c):
    """Type of the rows that fill the cache: its own, 16 bits for the 8-bit one."""
    return TORCH["bf16" if c.get("dtype", "e4m3") == "e4m3" else c["dtype"]]


def _inputs(c, seed):
    """The tensors of a case, the same for both sides: cached rows of the sequences one after another (the prefixes
    last), and what the call takes."""
    g, s = _gen(seed), {}
    kvD, rows = c["kv"] * c["D"], sum(_cached(c))
    if c["kind"] == "quant":
        s["qkv"] = _randn(g, sum(_new(c)), c["heads"] * c["D"] + 2 * kvD, dtype=TORCH[c["act"]])
        s["q_norm"] = 1 + 0.2 * _randn(g, c["D"])
        s["k_norm"] = 1 + 0.2 * _randn(g, c["D"])
        return s
    if c["kind"] == "attend":
        rows += c["prefix"] * len(_groups(c))
        s["q"] = (1.5 * _randn(g, sum(_new(c)), c["heads"] * c["D"])).to(TORCH[c["act"]])
    s["k"] = _randn(g, rows, kvD, dtype=_rows_type(c))
    s["v"] = _randn(g, rows, kvD, dtype=_rows_type(c))
    return s


def _max_seq(c):
    n = max([x + y for x, y in zip(_ctx(c), _new(c))] + [c.get("prefix", 0)])
    return -(-n // PAGE) * PAGE


def prepare(c, seed):
    s = _inputs(c, seed)
    s["case"] = c
    shared = c["kind"] == "attend" and c["prefix"] > 0
    cached = _cached(c) + ([c["prefix"]] * len(_groups(c)) if shared else [])
    n, max_seq, at = len(cached), _max_seq(c), _offsets(cached)
    s["ids"], s["new"], s["ctx"] = list(range(c["seqs"])), _new(c), _ctx(c)
    kvD = c["kv"] * c["D"]
    if c["kind"] == "attend":
        s["first"], s["full"] = (_first(c) if c["docs"] else None), (_full(c) if c["full"] else None)
        s["slopes"] = torch.tensor(_slopes(c), device="cuda") if c["slopes"] else None
    if own:
        import qauntrunner_amd as qr

        kv = qr.PagedKvCache(1, c["heads"], c["kv"], c["D"], max_seq, c.get("dtype", "e4m3"), n)
        kv.Reserve(n * (max_seq // PAGE))
        if c["kind"] != "quant":
            kv.AppendNormRopeDev(0, list(range(n)), [0] * n, cached, None, s["k"], s["v"], None, None, None, EPS, THETA,
                                 rotary_dim=0)
        s["kv"] = kv
        if c["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            if shared:
                s["prefix_ids"] = [c["seqs"] + i for i, (a, b) in enumerate(_groups(c)) for _ in range(a, b)]
                s["prefix_len"] = [c["prefix"]] * c["seqs"]
        else:
            rows = sum(s["new"] if c["kind"] == "quant" else s["ctx"])
            s["k_out"] = torch.empty(rows, kvD, dtype=TORCH[c["act"]], device="cuda")
            s["v_out"] = torch.empty_like(s["k_out"])
            if c["kind"] == "quant":
                s["q_out"] = torch.empty(rows, c["heads"] * c["D"], dtype=TORCH[c["act"]], device="cuda")
    else:
        # pages in no order, as a cache that has run for a while holds them
        pages, g = n * (max_seq // PAGE), _gen(seed + 1)
        table = torch.randperm(pages, device="cuda", generator=g).view(n, -1)
        s["table"] = table
        code = torch.uint8 if c.get("dtype", "e4m3") == "e4m3" else TORCH[c["dtype"]]
        for p in "kv":
            s["pool_" + p] = torch.zeros(pages, c["kv"], PAGE, c["D"], dtype=code, device="cuda")
            s["exp_" + p] = torch.zeros(pages, c["kv"], PAGE, dtype=torch.int8, device="cuda")
        if c["kind"] != "quant":
            seq = torch.repeat_interleave(torch.arange(n), torch.tensor(cached)).cuda()
            pos = torch.cat([torch.arange(x) for x in cached]).cuda()
            for p in "kv":
                _put(s, p, table[seq, pos // PAGE], pos % PAGE, s[p].view(-1, c["kv"], c["D"]))
        # which sequence and which of its rows each row is
        rows = s["ctx"] if c["kind"] == "read" else s["new"]
        s["seq"] = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(rows)).cuda()
        s["off"] = torch.cat([torch.arange(x) for x in rows]).cuda()
        s["ctx_t"] = torch.tensor(s["ctx"]).cuda()
        if c["kind"] == "attend":
            s["first_t"] = torch.tensor(_first(c)).cuda()
            s["full_t"] = torch.tensor(_full(c)).cuda()
    s.pop("k", None), s.pop("v", None)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own_quant(s) if kind == "quant" else _own_read(s) if kind == "read" else _own_attend(s)
    return _plain_quant(s) if kind == "quant" else _plain_read(s) if kind == "read" else _plain_attend(s)


def _own_quant(s):
    c, kv = s["case"], s["kv"]
    qD, kvD = c["heads"] * c["D"], c["kv"] * c["D"]
    q, k, v = s["qkv"].split([qD, kvD, kvD], dim=1)
    kv.AppendNormRopeDev(0, s["ids"], s["ctx"], s["new"], q, k, v, s["q_out"], s["q_norm"], s["k_norm"], EPS, THETA,
                         rotary_dim=c["rot"])
    kv.ReadAsDev(0, s["ids"], s["ctx"], s["new"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_read(s):
    s["kv"].ReadAsDev(0, s["ids"], [0] * len(s["ids"]), s["ctx"], s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _own_attend(s):
    c = s["case"]
    s["kv"].AttentionFormsDev(0, s["ids"], s["ctx"], s["new"], s["q"], s["out"], 1 / math.sqrt(c["D"]), cap=c["cap"],
                              slopes=s["slopes"], window=c["window"], first=s["first"], full=s["full"],
                              prefix_ids=s.get("prefix_ids"), prefix_len=s.get("prefix_len"))
    return s["out"]


def _powers(x, lo, hi, at):
    """2^at for at in lo..hi (from a table: a device's pow may be off by a step)."""
    table = torch.tensor([2.0**i for i in range(lo, hi + 1)], dtype=x.dtype).to(x.device)
    return table[(at - lo).long()]


def _quantise(x):
    """Codes of 8 bits and exponents of rows x [..., D]: the smallest e with max |x| <= 448 2^e."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # the largest is m 2^e, m in [1/2, 1)
    e = torch.clamp(e - 9 + (m > 448 / 512).int(), -117, 119)
    # nearest even by an addition that leaves the steps' bits: steps of 2^-3 of a value's power of two, 2^-9 at least
    y = x.double()
    y = y * _powers(y, -119, 117, -e)
    step = _powers(y, -9, 5, torch.clamp(torch.frexp(y)[1] - 4, min=-9))
    y = (y + step * (1.5 * 2.0**52)) - step * (1.5 * 2.0**52)
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8), e[..., 0].to(torch.int8)


def _put(s, p, page, slot, x):
    """Rows x [rows][kv][D] into the cache's slots."""
    if s["pool_" + p].dtype == torch.uint8:
        codes, e = _quantise(x)
        s["pool_" + p][page, :, slot] = codes
        s["exp_" + p][page, :, slot] = e
    else:
        s["pool_" + p][page, :, slot] = x.to(s["pool_" + p].dtype)


def _values(codes, e):
    """Cached values in 32 bits."""
    if codes.dtype != torch.uint8:
        return codes.float()
    y = codes.view(torch.float8_e4m3fn).float()
    return y * _powers(y, -117, 119, e[..., None])


def _norm_rope(x, w, pos, rot):
    """x [rows][heads][D]: each head's row normed and rotated (angles in 64 bits)."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    half = rot // 2
    inv = THETA ** (torch.arange(half, device=x.device, dtype=torch.float64) * (-2.0 / rot))
    ang = pos.double()[:, None] * inv
    cos, sin = torch.cos(ang).to(x.dtype)[:, None], torch.sin(ang).to(x.dtype)[:, None]
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)


def _plain_quant(s):
    c = s["case"]
    heads, kv, D = c["heads"], c["kv"], c["D"]
    rows = s["qkv"].shape[0]
    q, k, v = s["qkv"].float().split([heads * D, kv * D, kv * D], dim=1)
    pos = s["ctx_t"][s["seq"]] + s["off"]
    q = _norm_rope(q.reshape(rows, heads, D), s["q_norm"], pos, c["rot"])
    # in 64 bits: the codes of values next to a border between two
    k = _norm_rope(k.double().reshape(rows, kv, D), s["k_norm"].double(), pos, c["rot"])
    page, slot = s["table"][s["seq"], pos // PAGE], pos % PAGE
    _put(s, "k", page, slot, k)
    _put(s, "v", page, slot, v.reshape(rows, kv, D))
    back = [_values(s["pool_" + p][page, :, slot], s["exp_" + p][page, :, slot]) for p in "kv"]
    dt = s["qkv"].dtype
    return q.reshape(rows, -1).to(dt), back[0].reshape(rows, -1).to(dt), back[1].reshape(rows, -1).to(dt)


def _plain_read(s):
    c = s["case"]
    page, slot = s["table"][s["seq"], s["off"] // PAGE], s["off"] % PAGE
    return tuple(_values(s["pool_" + p][page, :, slot], s["exp_" + p][page, :, slot]).flatten(1).to(TORCH[c["act"]])
                 for p in "kv")


def _plain_attend(s):
    c = s["case"]
    n, heads, kv, D, plen = c["seqs"], c["heads"], c["kv"], c["D"], c["prefix"]
    G, nq = heads // kv, max(s["new"])

    def cached(p, seqs):  # [sequences][kv][slots][D]
        t = s["table"][seqs]
        x = _values(s["pool_" + p][t], s["exp_" + p][t])
        return x.permute(0, 2, 1, 3, 4).flatten(2, 3)

    k, v = cached("k", slice(0, n)), cached("v", slice(0, n))
    L, dev = k.shape[2], k.device
    q = torch.zeros(n, nq, heads, D, device=dev)
    q[s["seq"], s["off"]] = s["q"].float().view(-1, heads, D)
    q = q.view(n, nq, kv, G, D).permute(0, 2, 3, 1, 4).reshape(n, kv, G * nq, D)
    x = torch.matmul(q.flatten(0, 1), k.flatten(0, 1).transpose(1, 2).contiguous()).view(n, kv, G, nq, L)
    at = plen + torch.arange(L, device=dev)
    if plen:
        # the prefix's scores by one product for all sequences that share it
        shared = []
        for i, (a, b) in enumerate(_groups(c)):
            kp = cached("k", slice(n + i, n + i + 1))[0, :, :plen]
            rows = q[a:b].transpose(0, 1).reshape(kv, (b - a) * G * nq, D)
            y = torch.matmul(rows, kp.transpose(1, 2).contiguous())
            shared.append(y.view(kv, b - a, G, nq, plen).transpose(0, 1))
        x = torch.cat([torch.cat(shared), x], -1)
        at = torch.cat([torch.arange(plen, device=dev), at])
    x *= 1 / math.sqrt(D)
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    pos = plen + s["ctx_t"][:, None] + torch.arange(nq, device=dev)  # [n][nq]
    away = pos[..., None] - at  # [n][nq][positions]
    if c["slopes"]:
        x = x - s["slopes"].view(1, kv, G, 1, 1) * away.abs()[:, None, None]
    seen = ((away >= 0) | (at < s["full_t"][:, None, None])) & (at >= s["first_t"][:, None, None])
    if c["window"]:
        seen &= away < c["window"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    size = x.sum(-1, keepdim=True)
    x /= torch.where(size == 0, 1.0, size)
    own_part = x[..., plen:].reshape(n * kv, G * nq, L).contiguous()
    o = torch.matmul(own_part, v.flatten(0, 1)).view(n, kv, G, nq, D)
    if plen:
        for i, (a, b) in enumerate(_groups(c)):
            vp = cached("v", slice(n + i, n + i + 1))[0, :, :plen].contiguous()
            rows = x[a:b, ..., :plen].transpose(0, 1).reshape(kv, (b - a) * G * nq, plen)
            o[a:b] += torch.matmul(rows, vp).view(kv, b - a, G, nq, D).transpose(0, 1)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, nq, -1)
    return o[s["seq"], s["off"]].to(s["q"].dtype)


# ------------------------------------------------------------------ 64 bits
def _exact_e4m3(x):
    """The values of 8 bits that rows x [..., D] stand as: of the two steps around x / 2^e the nearer, of two as near the
    even one."""
    x = x.double()
    units = torch.tensor([2.0**k for k in range(-117, 120)], dtype=torch.float64).to(x.device)
    top = x.abs().max(-1, keepdim=True)[0]
    unit = units[torch.searchsorted(448 * units, top).clamp(max=units.numel() - 1)]  # the first with top <= 448 of it
    y = x.abs() / unit
    step = torch.full_like(y, 2.0**-9)
    for k in range(-5, 9):  # y in [2^k, 2^(k + 1)): steps of 2^(k - 3)
        step = torch.where(y >= 2.0**k, 2.0 ** (k - 3), step)
    low = torch.floor(y / step)
    rest = y / step - low
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.sign(x) * (low + up.double()) * step * unit


def exact(c, seed):
    s = _inputs(c, seed)
    kv, D = c["kv"], c["D"]
    if c["kind"] == "quant":
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
            return torch.cat([z.real, z.imag, y[..., 2 * half:]], -1)

        k = heads_of(x[:, heads * D:(heads + kv) * D], s["k_norm"])
        v = x[:, (heads + kv) * D:].reshape(-1, kv, D)
        return heads_of(x[:, :heads * D], s["q_norm"]).flatten(1), _exact_e4m3(k).flatten(1), _exact_e4m3(v).flatten(1)
    if c["kind"] == "read":
        return tuple(_exact_e4m3(s[p].view(-1, kv, D)).flatten(1) for p in "kv")
    G, plen = c["heads"] // kv, c["prefix"]
    lens = _cached(c) + [plen] * (len(_groups(c)) if plen else 0)
    at = _offsets(lens)
    group = [i for i, (a, b) in enumerate(_groups(c)) for _ in range(a, b)]
    slope = _slopes(c)

    def rows_of(p, i):
        x = s[p][at[i]:at[i + 1]].view(-1, kv, D)
        return _exact_e4m3(x) if c["dtype"] == "e4m3" else x.double()

    prefixes = [(rows_of("k", c["seqs"] + i), rows_of("v", c["seqs"] + i)) for i in range(len(_groups(c)) if plen else 0)]
    outs, begin = [], 0
    for i, (ctx, m) in enumerate(zip(_ctx(c), _new(c))):
        k, v = rows_of("k", i), rows_of("v", i)
        if plen:
            k, v = torch.cat([prefixes[group[i]][0], k]), torch.cat([prefixes[group[i]][1], v])
        q = s["q"][begin:begin + m].double().view(m, kv, G, D)
        begin += m
        row = (plen + ctx + torch.arange(m, device="cuda"))[:, None]
        t = torch.arange(k.shape[0], device="cuda")[None]
        hidden = (t < _first(c)[i]) | (t > torch.clamp(row, min=_full(c)[i] - 1))
        if c["window"]:
            hidden |= t <= row - c["window"]
        far = (row - t).abs().double()
        o = torch.empty(m, kv, G, D, dtype=torch.float64, device="cuda")
        for h in range(kv):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for j in range(G):
                a = q[:, h, j].contiguous() @ kt / math.sqrt(D)
                if c["cap"]:
                    a = torch.tanh(a / c["cap"]) * c["cap"]
                if c["slopes"]:
                    a -= far * slope[h * G + j]
                a = a.masked_fill(hidden, -math.inf)
                o[:, h, j] = torch.nan_to_num(torch.softmax(a, 1)) @ vh
        outs.append(o.view(m, -1))
    return torch.cat(outs)
