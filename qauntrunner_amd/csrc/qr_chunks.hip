// qr_chunks.hip -- plan, launches, split merge and the last step of the weights of the attention of
// chunks of several sequences.
#include "qr_chunks.hpp"

namespace qr {
namespace {

// Merge of the splits: one wave per (row, head).  A split without keys for the row holds
// m = -inf, l = 0.
__global__ void __launch_bounds__(64) chunks_combine_kernel(const ChunksK p) {
    const int row = blockIdx.x / p.heads, h = blockIdx.x - row * p.heads;
    const int e = batch_find(p.n, row, [&](int i) { return p.it[i].row0; });
    const int splits = p.it[e].splits;
    if (splits == 1) return;
    const int D = p.geom.head_dim, lane = threadIdx.x;
    const long long base = p.it[e].slot0 + (static_cast<long long>(row - p.it[e].row0) * p.heads + h) * splits;
    float m = -INFINITY;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, p.part_ml[base + s].x);
    float l = 0.f, o[kGenericMaxDim / 64];
#pragma unroll
    for (int i = 0; i < kGenericMaxDim / 64; ++i) o[i] = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float2 ml = p.part_ml[base + s];
        const float c = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m);
        l = fmaf(ml.y, c, l);
#pragma unroll
        for (int i = 0; i < kGenericMaxDim / 64; ++i)
            if (lane + 64 * i < D) o[i] = fmaf(p.part_acc[(base + s) * D + lane + 64 * i], c, o[i]);
    }
    const long long rh = blockIdx.x;
#pragma unroll
    for (int i = 0; i < kGenericMaxDim / 64; ++i)
        if (lane + 64 * i < D) store_out(p.out, p.act, rh * D + lane + 64 * i, o[i] / l);
    if (p.row_ml && lane == 0) p.row_ml[rh] = make_float2(m, l);
}

// Weights from the stored scores of a chunk's rows: one thread per position.
__global__ void __launch_bounds__(256) chunks_scores_kernel(const ChunksK p) {
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0;
    const int t = u % it.blocks * 256 + threadIdx.x, kvh = u / it.blocks;
    if (t >= it.pos0 + it.rows) return;
    const int g = p.heads / p.geom.kv_heads, stride = chunk_score_len(it);
    float sum = 0.f;
    for (int j = max(0, t - it.pos0); j < it.rows; ++j)
        for (int h = kvh * g; h < kvh * g + g; ++h) {
            const float2 ml = p.row_ml[static_cast<long long>(it.row0 + j) * p.heads + h];
            sum += fast_exp2(p.scores[it.score0 + (static_cast<long long>(j) * p.heads + h) * stride + t] - ml.x) / ml.y;
        }
    p.weights[(static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t] += sum;
}

// Parts of the weights' sums: one thread per position.
__global__ void __launch_bounds__(256) chunks_wmerge_kernel(const ChunksK p) {
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0, len = it.pos0 + it.rows;
    const int t = u % it.blocks * 256 + threadIdx.x, kvh = u / it.blocks;
    if (t >= len) return;
    float sum = 0.f;
    for (int s = 0; s < it.splits; ++s) sum += p.wpart[it.slot0 + (static_cast<long long>(s) * p.geom.kv_heads + kvh) * len + t];
    p.weights[(static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t] += sum;
}

struct KindGeom {
    int rows, tile;   // of a workgroup
    long long want;   // units that fill the GPU
};
constexpr KindGeom kGeom[kChunkKinds] = {{kChunkAnyRows, kChunkAnyTile, 1024}, {32, 128, 256}, {64, 128, 256}, {128, 64, 256}, {256, 64, 256}, {32, 32, 256}, {64, 32, 256}};

int cdiv(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

}  // namespace

ChunksPlan plan_chunks(const ChunksArgs& a) {
    ChunksPlan pl{};
    const int kv = a.geom.kv_heads, gmax = cdiv(a.heads, kv);
    const bool tiles = a.geom.mfma_layout && a.heads % kv == 0;
    const bool f32 = !tiles && chunks_f32_takes(a.dtype, a.geom.head_dim, a.heads, kv);
    for (int i = 0; i < a.n; ++i) {
        const long long rows = static_cast<long long>(a.it[i].rows) * gmax;
        if (f32) {
            // whole queries per block
            pl.it[i].kind = rows <= 32 ? kChunkF32Half : kChunkF32;
            pl.it[i].blocks = cdiv(a.it[i].rows, kGeom[pl.it[i].kind].rows / gmax);
            continue;
        }
        pl.it[i].kind = !tiles ? kChunkAny : rows <= 32 ? kChunkStream32 : rows <= 64 ? kChunkStream64 : rows <= 128 ? kChunkStream128 : kChunkTile;
        pl.it[i].blocks = cdiv(rows, kGeom[pl.it[i].kind].rows);
    }
    // The keys of a kind's blocks are split while its units do not fill the GPU: as many positions
    // per unit as leave no more units than that, or one tile.
    long long slots = 0;
    for (int kind = 0; kind < kChunkKinds; ++kind) {
        KindGeom g = kGeom[kind];
        if (kind == kChunkF32Half || kind == kChunkF32) g.want *= chunks_f32_per_cu(a.dtype, a.geom.head_dim, kind == kChunkF32Half);
        long long base = 0, work = 0;
        for (int i = 0; i < a.n; ++i)
            if (pl.it[i].kind == kind) {
                base += static_cast<long long>(pl.it[i].blocks) * kv;
                work += static_cast<long long>(pl.it[i].blocks) * kv * cdiv(a.it[i].pos0 + a.it[i].rows, g.tile);
            }
        if (!base) continue;
        long long per = base >= g.want ? 1LL << 40 : std::max<long long>(1, work / g.want);  // tiles of a unit
        auto units = [&](long long per_) {
            long long u = 0;
            for (int i = 0; i < a.n; ++i)
                if (pl.it[i].kind == kind)
                    u += static_cast<long long>(pl.it[i].blocks) * kv * cdiv(cdiv(a.it[i].pos0 + a.it[i].rows, g.tile), per_);
            return u;
        };
        if (base < g.want)
            while (units(per) > g.want && per < (1 << 24)) per += std::max<long long>(1, per / 16);
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            if (it.kind != kind) continue;
            it.splits = std::min(cdiv(cdiv(a.it[i].pos0 + a.it[i].rows, g.tile), per), 256);
            it.slot0 = slots;
            if (it.splits > 1) {
                slots += static_cast<long long>(a.it[i].rows) * a.heads * it.splits;
                pl.merge = true;
            }
        }
    }
    long long wslots = 0, scores = 0;
    if (a.weights) {
        long long units = 0;
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            it.wkind = it.kind == kChunkAny ? kWeightsAny : it.kind == kChunkStream32 || it.kind == kChunkF32Half ? kWeightsScores
                     : it.kind == kChunkF32 ? kWeightsF32 : kWeightsTile;
            it.wblocks = cdiv(a.it[i].pos0 + a.it[i].rows, it.wkind == kWeightsAny ? kChunkAnyTile : it.wkind == kWeightsF32 ? 128 : 256);
            it.wsplits = 1;
            if (it.wkind >= kWeightsTile) units += static_cast<long long>(it.wblocks) * kv;
            if (it.wkind == kWeightsScores) {
                it.score0 = scores;
                scores += static_cast<long long>(a.it[i].rows) * a.heads * chunk_score_len(a.it[i]);
            }
        }
        // few position blocks: their rows are split too, 64 rows or more a part
        for (int i = 0; i < a.n; ++i) {
            ChunkPlanItem& it = pl.it[i];
            if (it.wkind < kWeightsTile || units >= 1024) continue;
            it.wsplits = std::max(1, std::min(cdiv(1024, units), cdiv(static_cast<long long>(a.it[i].rows) * gmax, 64)));
            it.wslot0 = wslots;
            if (it.wsplits > 1) {
                wslots += static_cast<long long>(it.wsplits) * kv * (a.it[i].pos0 + a.it[i].rows);
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
    auto gather = [&](auto in, bool weights) {
        k.n = k.units = 0;
        for (int i = 0; i < a.n; ++i) {
            const ChunkPlanItem& pi = plan.it[i];
            if (!in(pi)) continue;
            ChunkItem& it = k.it[k.n++];
            it = a.it[i];
            it.unit0 = k.units;
            it.blocks = weights ? pi.wblocks : pi.blocks;
            it.splits = weights ? pi.wsplits : pi.splits;
            it.slot0 = static_cast<int>(weights ? pi.wslot0 : pi.slot0);
            it.score0 = pi.score0;
            k.units += it.blocks * it.splits * kv;
        }
        return k.n > 0;
    };
    hipError_t e = hipSuccess;
    for (int kind = 0; kind < kChunkKinds && e == hipSuccess; ++kind) {
        if (!gather([&](const ChunkPlanItem& p) { return p.kind == kind; }, false)) continue;
        k.scores = a.weights && (kind == kChunkStream32 || kind == kChunkF32Half) ? reinterpret_cast<float*>(w + plan.scores) : nullptr;
        e = kind == kChunkAny ? launch_chunks_any(k, stream) : kind >= kChunkF32Half ? launch_chunks_f32(k, kind, stream)
          : launch_chunks_tile(k, kind, stream);
    }
    if (e == hipSuccess && plan.merge) {
        gather([](const ChunkPlanItem&) { return true; }, false);
        hipLaunchKernelGGL(chunks_combine_kernel, dim3(a.rows * a.heads), dim3(64), 0, stream, k);
        e = hipGetLastError();
    }
    if (!a.weights) return e;
    k.scores = reinterpret_cast<float*>(w + plan.scores);
    for (int kind = 0; kind < kWeightsKinds && e == hipSuccess; ++kind) {
        if (!gather([&](const ChunkPlanItem& p) { return p.wkind == kind; }, true)) continue;
        if (kind == kWeightsScores) {
            hipLaunchKernelGGL(chunks_scores_kernel, dim3(k.units), dim3(256), 0, stream, k);
            e = hipGetLastError();
        } else {
            e = kind == kWeightsAny ? launch_chunks_any_weights(k, stream) : kind == kWeightsF32 ? launch_chunks_f32(k, kChunkKinds, stream)
              : launch_chunks_tile(k, kChunkKinds, stream);
        }
    }
    if (e == hipSuccess && plan.wmerge) {
        gather([](const ChunkPlanItem& p) { return p.wkind >= kWeightsTile && p.wsplits > 1; }, true);
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
