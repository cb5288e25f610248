// qr_chunks.hip -- plan, launches, split merge and the last step of the weights of the attention of
// chunks of several sequences.
#include "qr_chunks.hpp"

namespace qr {
namespace {

// The weight of a partial or of a sum in a merge.  A weight may round to zero where the formula has none that is: an infinity
// stays one.
__device__ __forceinline__ float merge_weight(float x, float w) { return fabsf(x) == INFINITY ? 1.f : w; }

// Merge of the splits, any head size: one wave per (row, head).  A split without keys for the row
// holds m = -inf, l = 0.
__global__ void __launch_bounds__(64) chunks_merge_any_kernel(const ChunksK p) {
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const long long r = blockIdx.x - it.unit0, rh = static_cast<long long>(it.row0) * p.heads + r;
    const int D = p.geom.head_dim, lane = threadIdx.x;
    const long long base = it.slot0 + r * it.splits;
    float m = -INFINITY;
    for (int s = 0; s < it.splits; ++s) m = fmaxf(m, p.part_ml[base + s].x);
    float l = 0.f, o[kGenericMaxDim / 64];
#pragma unroll
    for (int i = 0; i < kGenericMaxDim / 64; ++i) o[i] = 0.f;
    for (int s = 0; s < it.splits; ++s) {
        const float2 ml = p.part_ml[base + s];
        const float c = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m);
        l = fmaf(ml.y, c, l);
#pragma unroll
        for (int i = 0; i < kGenericMaxDim / 64; ++i)
            if (lane + 64 * i < D) {
                const float x = p.part_acc[(base + s) * D + lane + 64 * i];
                o[i] = fmaf(x, merge_weight(x, c), o[i]);
            }
    }
#pragma unroll
    for (int i = 0; i < kGenericMaxDim / 64; ++i)
        if (lane + 64 * i < D) store_out(p.out, p.act, rh * D + lane + 64 * i, o[i] / l);
    if (p.row_ml && lane == 0) p.row_ml[rh] = make_float2(m, l);
}

// Weights from the stored scores of a chunk's rows (up to 32 of a kv head): one thread per position.  The rows' maxima and sums
// come from the partials, eight threads a row, so that the merge can run beside it.
__device__ __forceinline__ void add_scores(const ChunksK& p, const ChunkItem& it, int u) {
    __shared__ float2 row[32];
    const int t = u % it.blocks * 256 + threadIdx.x, kvh = u / it.blocks;
    const int g = p.heads / p.geom.kv_heads, stride = chunk_score_len(it);
    const bool on = t < it.pos0 + it.rows;
    float* const w = p.weights + (static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t;
    const float before = on ? *w : 0.f;
    const int r = threadIdx.x >> 3;
    float m = -INFINITY, l = 0.f;
    if (r < it.rows * g) {
        const long long rh = static_cast<long long>(r / g) * p.heads + kvh * g + r % g;
        if (it.splits == 1) {
            const float2 ml = p.row_ml[static_cast<long long>(it.row0) * p.heads + rh];
            m = ml.x;
            l = threadIdx.x & 7 ? 0.f : ml.y;
        } else {
            const float2* ml = p.part_ml + it.slot0 + rh * it.splits;
            for (int s = threadIdx.x & 7; s < it.splits; s += 8) m = fmaxf(m, ml[s].x);
            for (int x = 1; x < 8; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
            for (int s = threadIdx.x & 7; s < it.splits; s += 8) l = fmaf(ml[s].y, ml[s].x == -INFINITY ? 0.f : fast_exp2(ml[s].x - m), l);
        }
    }
    for (int x = 1; x < 8; x <<= 1) l += __shfl_xor(l, x);
    if ((threadIdx.x & 7) == 0) row[r] = make_float2(m, l);
    __syncthreads();
    const float* s = p.scores + it.score0 + static_cast<long long>(kvh) * g * stride + (on ? t : 0);
    float sum = 0.f;
    for (int j = 0; j < it.rows; ++j, s += static_cast<long long>(p.heads) * stride) {
        const bool see = t <= it.pos0 + j;
#pragma unroll 4
        for (int h = 0; h < g; ++h) {
            const float2 ml = row[j * g + h];
            const float x = fast_exp2(s[static_cast<long long>(h) * stride] - ml.x) / ml.y;
            if (see) sum += x;
        }
    }
    if (on) *w = before + sum;
}

// The merge for the tiles' head sizes: D / 4 threads per (row, head), 4 dims each, the partials of 8
// splits requested at once (16 rows of 32 heads over 17 splits: 7.6 -> 4 us against one wave per row).  Behind a chunk's
// merge units stand those that add its weights from stored scores: one launch for both (16 decode rows of 130 to
// 16000 positions with weights 56.7 -> 55.4 us, two of a tiny model 15 -> 12).
constexpr int merge_rows(int D) { return 256 / (D / 4); }
__host__ __device__ inline int merge_units(const ChunkItem& it, int heads, int rows) {
    return it.splits > 1 ? static_cast<int>((static_cast<long long>(it.rows) * heads + rows - 1) / rows) : 0;
}
template <int D>
__global__ void __launch_bounds__(256) chunks_merge_kernel(const ChunksK p) {
    constexpr int TPR = D / 4, RPB = merge_rows(D), kB = 8;
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int merges = merge_units(it, p.heads, RPB);
    if (static_cast<int>(blockIdx.x) - it.unit0 >= merges) {
        add_scores(p, it, blockIdx.x - it.unit0 - merges);
        return;
    }
    const int rr = threadIdx.x / TPR, c = threadIdx.x - rr * TPR;
    const long long r = static_cast<long long>(blockIdx.x - it.unit0) * RPB + rr;
    if (rr >= RPB || r >= static_cast<long long>(it.rows) * p.heads) return;
    const long long base = it.slot0 + r * it.splits;
    int parts = it.splits;
    if (it.per) {
        const KeyTiles t = p.geom.mfma_layout ? kKeyTiles16 : key_tiles32(p.heads / p.geom.kv_heads);
        const int g = p.heads / p.geom.kv_heads, q = static_cast<int>(r / p.heads), h = static_cast<int>(r - static_cast<long long>(q) * p.heads);
        parts = t.parts(it, g, (q * g + h % g) / t.rows, it.per);
        if (parts == 1) return;  // written by its unit
    }
    const float4* part = reinterpret_cast<const float4*>(p.part_acc) + base * TPR + c;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += kB) {
        float4 a[kB];
        float2 ml[kB];
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int s = min(s0 + i, parts - 1);
            a[i] = part[static_cast<long long>(s) * TPR];
            ml[i] = p.part_ml[base + s];
        }
        float mb = m;
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            if (s0 + i >= parts) ml[i].x = -INFINITY;  // a repeated split
            mb = fmaxf(mb, ml[i].x);
        }
        const float cm = m == -INFINITY ? 0.f : fast_exp2(m - mb);
        l *= cm;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] *= merge_weight(o[x], cm);
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            if (s0 + i >= parts) continue;
            const float w = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - mb);
            l = fmaf(ml[i].y, w, l);
            o[0] = fmaf(a[i].x, merge_weight(a[i].x, w), o[0]);
            o[1] = fmaf(a[i].y, merge_weight(a[i].y, w), o[1]);
            o[2] = fmaf(a[i].z, merge_weight(a[i].z, w), o[2]);
            o[3] = fmaf(a[i].w, merge_weight(a[i].w, w), o[3]);
        }
        m = mb;
    }
    const long long rh = static_cast<long long>(it.row0) * p.heads + r;
    const float inv = 1.f / l;
    if (p.act == QR_DTYPE_F32) {
        float* out = static_cast<float*>(p.out) + rh * D + 4 * c;
#pragma unroll
        for (int x = 0; x < 4; ++x) out[x] = o[x] * inv;
    } else {
        uint16_t b[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) b[x] = f32_to_out16(o[x] * inv, p.act);
        __builtin_memcpy(static_cast<uint16_t*>(p.out) + rh * D + 4 * c, b, 8);
    }
    if (p.row_ml && c == 0) p.row_ml[rh] = make_float2(m, l);
}

// Parts of the weights' sums: one thread per position.
__global__ void __launch_bounds__(256) chunks_wmerge_kernel(const ChunksK p) {
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0, len = it.pos0 + it.rows;
    const int t = u % it.blocks * 256 + threadIdx.x, kvh = u / it.blocks;
    if (t >= len) return;
    const WeightTiles w = p.geom.mfma_layout ? kWeightTiles16 : kWeightTiles32;
    const int parts = w.parts(it, p.heads / p.geom.kv_heads, t / w.positions, it.per);
    if (parts == 1) return;  // added by its unit
    const float* const from = p.wpart + it.slot0 + static_cast<long long>(kvh) * len + t;
    const long long stride = static_cast<long long>(p.geom.kv_heads) * len;
    float sum = 0.f;
    for (int s0 = 0; s0 < parts; s0 += 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = from[min(s0 + i, parts - 1) * stride];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += s0 + i < parts ? x[i] : 0.f;
    }
    p.weights[(static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t] += sum;
}

struct KindGeom {
    int rows, tile;   // of a workgroup
    long long want;   // units that fill the GPU
};
constexpr KindGeom kGeom[kChunkKinds] = {{kChunkAnyRows, kChunkAnyTile, 1024}, {32, 128, 256}, {128, 64, 512}, {256, 64, 256}, {32, 32, 256}, {64, 32, 256}};

// Scores that a launch keeps for its weights: 256 MB, a token of 32 heads over 32768 positions for each of its 64 chunks.
constexpr long long kMaxScores = 64LL * 32 * 32768;

int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

}  // namespace

ChunksPlan plan_chunks(const ChunksArgs& a) {
    ChunksPlan pl{};
    const int kv = a.geom.kv_heads, gmax = cdiv(a.heads, kv);
    const bool tiles = a.geom.mfma_layout && a.heads % kv == 0;
    const bool f32 = !tiles && chunks_f32_takes(a.dtype, a.geom.head_dim, a.heads, kv);
    // Three parts of bf16 need more registers than the kernel of many rows has (fp32 rows over a bf16 cache, 2048 after 6144: 645
    // us here, 414 there with two, whose error is 4e-6 where three have 4e-7).
    const bool parts3 = chunk_parts(a.dtype, a.act != a.dtype) == 3;
    for (int i = 0; i < a.n; ++i) {
        const long long rows = static_cast<long long>(a.it[i].rows) * gmax;
        if (f32) {
            // whole queries per block
            pl.it[i].kind = rows <= 32 ? kChunkF32Half : kChunkF32;
            pl.it[i].blocks = cdiv(a.it[i].rows, kGeom[pl.it[i].kind].rows / gmax);
            continue;
        }
        pl.it[i].kind = !tiles ? kChunkAny : rows <= 32 ? kChunkStream32 : rows <= 128 || parts3 ? kChunkStream : kChunkTile;
        pl.it[i].blocks = cdiv(rows, kGeom[pl.it[i].kind].rows);
    }
    // The keys of a kind's blocks are split while its units do not fill the GPU: as many tiles per unit as leave
    // no more units than that, or one.  (Every tile of a kind takes about the same time: kChunkStream's are of 32 positions
    // for more than 64 rows, else of 64.)
    auto tiles_of = [&](int i) {
        int tile = kGeom[pl.it[i].kind].tile;
        if (pl.it[i].kind == kChunkStream && static_cast<long long>(a.it[i].rows) * gmax > 64) tile = 32;
        return cdiv(a.it[i].pos0 + a.it[i].rows, tile);
    };
    long long slots = 0;
    for (int kind = 0; kind < kChunkKinds; ++kind) {
        KindGeom g = kGeom[kind];
        if (kind == kChunkF32Half || kind == kChunkF32) g.want *= chunks_f32_per_cu(a.dtype, a.geom.head_dim, kind == kChunkF32Half);
        const bool by_block = kind == kChunkTile || kind == kChunkF32;
        const KeyTiles kt = kind == kChunkTile ? kKeyTiles16 : key_tiles32(std::min(gmax, 64));
        long long base = 0, work = 0;
        for (int i = 0; i < a.n; ++i)
            if (pl.it[i].kind == kind) {
                base += static_cast<long long>(pl.it[i].blocks) * kv;
                work += kv * (by_block ? kt.units(a.it[i], gmax, 1) : static_cast<long long>(pl.it[i].blocks) * tiles_of(i));
            }
        if (!base) continue;
        // tiles of a unit.  Enough units already: those with much more than a CU's share are split all the same (six bf16
        // prompts of 101 to 1501 rows after 3001 to 1 positions, with weights: 119 us, 130 without, 127 where fewer tiles than
        // a quarter more than the share are split too)
        long long per = base >= g.want ? std::max<long long>(8, work * 5 / (g.want * 4)) : std::max<long long>(1, work / g.want);
        auto units = [&](long long per_) {
            long long u = 0;
            for (int i = 0; i < a.n; ++i)
                if (pl.it[i].kind == kind)
                    u += kv * (by_block ? kt.units(a.it[i], gmax, static_cast<int>(per_)) : static_cast<long long>(pl.it[i].blocks) * cdiv(tiles_of(i), per_));
            return u;
        };
        if (base < g.want)
            while (units(per) > g.want && per < (1 << 24)) per += std::max<long long>(1, per / 64);
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            if (it.kind != kind) continue;
            it.splits = std::min(cdiv(tiles_of(i), per), 256);
            it.slot0 = slots;
            if (by_block) {
                it.per = std::max(static_cast<int>(per), cdiv(tiles_of(i), 256));
                it.blocks = static_cast<int>(kt.units(a.it[i], gmax, it.per));
                it.splits = cdiv(tiles_of(i), it.per);
            }
            if (it.splits > 1) slots += static_cast<long long>(a.it[i].rows) * a.heads * it.splits;
        }
    }
    long long wslots = 0, scores = 0;
    if (a.weights) {
        const WeightTiles wt = tiles ? kWeightTiles16 : kWeightTiles32;
        long long rounds = 0;
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            it.wkind = it.kind == kChunkAny ? kWeightsAny : it.kind == kChunkStream32 || it.kind == kChunkF32Half ? kWeightsScores
                     : it.kind == kChunkF32 ? kWeightsF32 : kWeightsTile;
            it.score0 = -1;
            if (it.wkind == kWeightsScores) {
                // up to a bound, the others compute theirs again: the workspace stays with the handle
                const long long n = static_cast<long long>(a.it[i].rows) * a.heads * chunk_score_len(a.it[i]);
                if (scores + n <= kMaxScores) {
                    it.score0 = scores;
                    scores += n;
                } else {
                    it.wkind = tiles ? kWeightsTile : kWeightsF32;
                }
            }
            it.wblocks = cdiv(a.it[i].pos0 + a.it[i].rows, it.wkind == kWeightsAny ? kChunkAnyTile : 256);
            if (it.wkind >= kWeightsTile) rounds += kv * wt.units(a.it[i], gmax, 1);
        }
        // units of an equal share of the rounds
        const long long want = tiles ? 1024 : 512;
        const int per = static_cast<int>(std::max<long long>(tiles ? 1 : 4, (rounds + want - 1) / want));
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            if (it.wkind < kWeightsTile) continue;
            it.wper = per;
            it.wblocks = static_cast<int>(wt.units(a.it[i], gmax, per));
            it.wparts = wt.parts(a.it[i], gmax, 0, per);
            it.wslot0 = wslots;
            if (it.wparts > 1) {
                wslots += static_cast<long long>(it.wparts) * kv * (a.it[i].pos0 + a.it[i].rows);
                pl.wmerge = true;
            }
        }
    }
    auto next = [](size_t& at, size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) & ~size_t(255);
        return r;
    };
    size_t at = 0;
    const size_t rh = static_cast<size_t>(a.rows) * a.heads;
    next(at, static_cast<size_t>(slots) * a.geom.head_dim * sizeof(float));
    pl.part_ml = next(at, static_cast<size_t>(slots) * sizeof(float2));
    pl.row_ml = next(at, a.weights ? rh * sizeof(float2) : 0);
    pl.row_scale = next(at, a.weights ? rh * sizeof(float) : 0);
    pl.scores = next(at, static_cast<size_t>(scores) * sizeof(float));
    pl.wpart = next(at, static_cast<size_t>(wslots) * sizeof(float));
    pl.workspace_bytes = at;
    return pl;
}

hipError_t launch_chunks(const ChunksArgs& a, const ChunksPlan& plan, void* workspace, hipStream_t stream) {
    ChunksK k{};
    k.pool = static_cast<const char*>(a.pool);
    k.page_table = a.page_table;
    k.geom = a.geom;
    k.dtype = a.dtype;
    k.act = a.act;
    k.heads = a.heads;
    k.q = a.q;
    k.out = a.out;
    k.weights = a.weights;
    k.max_seq = a.max_seq;
    k.qscale = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
    char* w = static_cast<char*>(workspace);
    k.part_acc = reinterpret_cast<float*>(w);
    k.part_ml = reinterpret_cast<float2*>(w + plan.part_ml);
    if (a.weights) {
        k.row_ml = reinterpret_cast<float2*>(w + plan.row_ml);
        if (a.dtype == QR_DTYPE_F16 && a.act != QR_DTYPE_F16) k.row_scale = reinterpret_cast<float*>(w + plan.row_scale);
        k.wpart = reinterpret_cast<float*>(w + plan.wpart);
    }
    const int kv = a.geom.kv_heads;
    // the chunks that `in` takes, with a launch's blocks and splits
    // (tile kernels: per kv head, the chunks with the longest units first)
    int order[kBatch];
    for (int i = 0; i < a.n; ++i) order[i] = i;
    std::stable_sort(order, order + a.n, [&](int x, int y) {
        return static_cast<long long>(a.it[x].pos0 + a.it[x].rows) * plan.it[y].splits > static_cast<long long>(a.it[y].pos0 + a.it[y].rows) * plan.it[x].splits;
    });
    auto gather = [&](auto in, bool weights, bool per_head = false) {
        k.n = k.units = 0;
        for (int o = 0; o < a.n; ++o) {
            const int i = per_head ? order[o] : o;
            const ChunkPlanItem& pi = plan.it[i];
            if (!in(pi)) continue;
            ChunkItem& it = k.it[k.n++];
            it = a.it[i];
            it.unit0 = k.units;
            it.blocks = weights ? pi.wblocks : pi.blocks;
            it.splits = weights ? 1 : pi.splits;
            it.parts = it.splits;
            it.per = weights ? pi.wper : pi.per;
            it.slot0 = static_cast<int>(weights ? pi.wslot0 : pi.slot0);
            it.score0 = pi.score0;
            k.units += it.blocks * (it.per ? 1 : it.splits) * (per_head ? 1 : kv);
        }
        return k.n > 0;
    };
    hipError_t e = hipSuccess;
    for (int kind = 0; kind < kChunkKinds && e == hipSuccess; ++kind) {
        if (!gather([&](const ChunkPlanItem& p) { return p.kind == kind; }, false, kind >= kChunkTile)) continue;
        k.paired = kind >= kChunkF32Half && static_cast<long long>(k.units) * kv <= 256LL * chunks_f32_per_cu(a.dtype, a.geom.head_dim, kind == kChunkF32Half);
        k.scores = a.weights && (kind == kChunkStream32 || kind == kChunkF32Half) ? reinterpret_cast<float*>(w + plan.scores) : nullptr;
        e = kind == kChunkAny ? launch_chunks_any(k, stream) : kind >= kChunkF32Half ? launch_chunks_f32(k, kind, stream)
          : launch_chunks_tile(k, kind, stream);
    }
    auto scored = [&](const ChunkPlanItem& p) { return a.weights && p.wkind == kWeightsScores; };
    if (e == hipSuccess && gather([&](const ChunkPlanItem& p) { return p.splits > 1 || scored(p); }, false)) {
        const int D = a.geom.head_dim;
        const bool vec = D == 64 || D == 96 || D == 128 || D == 256;
        k.scores = reinterpret_cast<float*>(w + plan.scores);
        k.units = 0;
        for (int i = 0; i < k.n; ++i) {
            ChunkItem& it = k.it[i];
            it.unit0 = k.units;
            k.units += merge_units(it, a.heads, vec ? merge_rows(D) : 1);
            if (!a.weights || it.score0 < 0) continue;
            it.blocks = cdiv(it.pos0 + it.rows, 256);
            k.units += it.blocks * kv;
        }
        if (D == 64) hipLaunchKernelGGL(chunks_merge_kernel<64>, dim3(k.units), dim3(256), 0, stream, k);
        else if (D == 96) hipLaunchKernelGGL(chunks_merge_kernel<96>, dim3(k.units), dim3(256), 0, stream, k);
        else if (D == 128) hipLaunchKernelGGL(chunks_merge_kernel<128>, dim3(k.units), dim3(256), 0, stream, k);
        else if (D == 256) hipLaunchKernelGGL(chunks_merge_kernel<256>, dim3(k.units), dim3(256), 0, stream, k);
        else hipLaunchKernelGGL(chunks_merge_any_kernel, dim3(k.units), dim3(64), 0, stream, k);
        e = hipGetLastError();
    }
    if (!a.weights) return e;
    for (int kind = 0; kind < kWeightsKinds && e == hipSuccess; ++kind) {
        if (kind == kWeightsScores || !gather([&](const ChunkPlanItem& p) { return p.wkind == kind; }, true)) continue;
        e = kind == kWeightsAny ? launch_chunks_any_weights(k, stream) : kind == kWeightsF32 ? launch_chunks_f32(k, kChunkKinds, stream)
          : launch_chunks_tile(k, kChunkKinds, stream);
    }
    if (e == hipSuccess && plan.wmerge) {
        gather([](const ChunkPlanItem& p) { return p.wkind >= kWeightsTile && p.wparts > 1; }, true);
        k.units = 0;  // one unit per 256 positions and kv head
        for (int i = 0; i < k.n; ++i) {
            k.it[i].unit0 = k.units;
            k.it[i].blocks = cdiv(k.it[i].pos0 + k.it[i].rows, 256);
            k.units += k.it[i].blocks * kv;
        }
        hipLaunchKernelGGL(chunks_wmerge_kernel, dim3(k.units), dim3(256), 0, stream, k);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace qr
