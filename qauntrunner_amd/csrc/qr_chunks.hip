// qr_chunks.hip -- plan, launch and split merge of the attention of chunks of several sequences.
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
        if (lane + 64 * i < D) store_elem(p.out, p.act, rh * D + lane + 64 * i, o[i] / l);
    if (p.row_ml && lane == 0) p.row_ml[rh] = make_float2(m, l);
}

}  // namespace

ChunksPlan plan_chunks(ChunksArgs& a) {
    ChunksPlan pl{};
    const int kv = a.geom.kv_heads, gmax = (a.heads + kv - 1) / kv;
    const int R = chunks_any_rows(), T = chunks_any_tile();
    // units without splits, and the (block, position) pairs that they read
    long long base = 0, work = 0;
    for (int i = 0; i < a.n; ++i) {
        const long long b = (static_cast<long long>(a.it[i].rows) * gmax + R - 1) / R;
        base += b * kv;
        work += b * kv * (a.it[i].pos0 + a.it[i].rows);
    }
    const long long want = 1024;
    const long long per = base >= want ? (1LL << 40) : std::max<long long>(2 * T, work / want);
    for (int i = 0; i < a.n; ++i) {
        ChunkItem& it = a.it[i];
        const int len = it.pos0 + it.rows;
        it.blocks = static_cast<int>((static_cast<long long>(it.rows) * gmax + R - 1) / R);
        it.splits = static_cast<int>(std::min<long long>((len + per - 1) / per, 256));
        it.unit0 = pl.units;
        pl.units += it.blocks * it.splits * kv;
        it.slot0 = static_cast<int>(pl.slots);
        if (it.splits > 1) pl.slots += static_cast<long long>(it.rows) * a.heads * it.splits;
        it.wunit0 = pl.wunits;
        pl.wunits += (len + T - 1) / T * kv;
    }
    pl.part_ml_off = static_cast<size_t>(pl.slots) * a.geom.head_dim * sizeof(float);
    pl.part_ml_off = (pl.part_ml_off + 255) & ~size_t(255);
    pl.row_ml_off = pl.part_ml_off + ((static_cast<size_t>(pl.slots) * sizeof(float2) + 255) & ~size_t(255));
    pl.workspace_bytes = pl.row_ml_off + (a.weights ? static_cast<size_t>(a.rows) * a.heads * sizeof(float2) : 0);
    return pl;
}

hipError_t launch_chunks(const ChunksArgs& a, const ChunksPlan& plan, void* workspace, hipStream_t stream) {
    ChunksK k{};
    std::copy(a.it, a.it + a.n, k.it);
    k.n = a.n;
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
    k.part_ml = reinterpret_cast<float2*>(w + plan.part_ml_off);
    k.row_ml = a.weights ? reinterpret_cast<float2*>(w + plan.row_ml_off) : nullptr;
    hipError_t e = launch_chunks_any(k, plan, stream);
    if (e == hipSuccess && plan.slots) {
        hipLaunchKernelGGL(chunks_combine_kernel, dim3(a.rows * a.heads), dim3(64), 0, stream, k);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.weights) e = launch_chunks_any_weights(k, plan, stream);
    return e;
}

}  // namespace qr
