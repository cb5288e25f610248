// qr_chunks_any.hip -- causal attention of chunks of several sequences over the paged cache, and
// the weight that each cached position received: any cache type, head size and head count, gfx950.
//
// Row (j, h) of a chunk -- query j, query head h -- attends positions 0..pos0 + j of its sequence:
// s_t = scale q.k_t, out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m), m the largest s_t so far.
// One pass over K and V; a block's keys may be split over workgroups, whose (m, l, o) are merged.
// The weights need every row's final m and l, so they take a second pass over the K rows:
// weights[t] += sum over rows of e^(s_t - m) / l, each position added up by one workgroup.
//
// Products and sums are fp32.  A row never touches a position that it does not see, so that what
// such a slot holds (NaN too) does not matter.
#include "qr_chunks.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = kChunkAnyRows;
constexpr int kTile = kChunkAnyTile;

// Positions t0 .. t0 + 31 (below `end`, one page) of one plane and kv head into LDS as fp32, rows
// of D + 1 values: a column's 32 reads hit 32 banks.
__device__ __forceinline__ void load_tile(const ChunksK& p, int pt_off, int plane, int kvh, int t0, int end, float* tile) {
    const int D = p.geom.head_dim;
    const long long phys = p.page_table[pt_off + (t0 >> kPageShift)];
    const int n = min(kTile, end - t0) * D;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int t = i / D, d = i - t * D;
        tile[t * (D + 1) + d] = load_elem(p.pool, p.dtype, p.geom.offset(phys, plane, kvh, (t0 & (kPageTokens - 1)) + t, d));
    }
}

// q rows rho0 .. rho0 + 7 of a kv head's rows (query rho / g, head rho % g) as fp32, scaled
__device__ __forceinline__ void load_rows(const ChunksK& p, const ChunkItem& it, int rho0, int h0, int g, float* q) {
    const int D = p.geom.head_dim;
    for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        const int rho = min(rho0 + r, it.rows * g - 1);
        const long long row = it.row0 + rho / g;
        q[r * D + d] = load_elem(p.q, p.act, (row * p.heads + h0 + rho % g) * D + d) * p.qscale;
    }
}

__device__ __forceinline__ float dot(const float* q, const float* k, int D) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int d = 0;
    for (; d + 4 <= D; d += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(q[d + i], k[d + i], s[i]);
    for (; d < D; ++d) s[0] = fmaf(q[d], k[d], s[0]);
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ void __launch_bounds__(kThreads) chunks_any_kernel(const ChunksK p) {
    extern __shared__ float lds[];
    const int D = p.geom.head_dim;
    float* const q = lds;                   // [8][D]
    float* const tile = q + kRows * D;      // [32][D + 1]
    float* const prob = tile + kTile * (D + 1);  // [8][32]
    float* const corr = prob + kRows * kTile;    // [8]
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0;
    const int split = u % it.splits, block = u / it.splits % it.blocks, kvh = u / (it.splits * it.blocks);
    int h0, g;
    chunk_heads(p, kvh, &h0, &g);
    const int rho0 = block * kRows;
    if (rho0 >= it.rows * g) return;
    const int rho1 = min(rho0 + kRows, it.rows * g);
    load_rows(p, it, rho0, h0, g, q);
    int t0, t1;
    chunk_keys(it, it.pos0 + (rho1 - 1) / g + 1, split, kTile, &t0, &t1);

    const int r = threadIdx.x >> 5, tl = threadIdx.x & 31;  // this thread's score
    const int seen = it.pos0 + min(rho0 + r, rho1 - 1) / g;  // the last position of row r
    float m = -INFINITY, l = 0.f;                            // of row r, the same in its 32 lanes
    constexpr int NC = kGenericMaxDim / kThreads;
    float acc[kRows][NC];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = 0.f;
    for (int t = t0; t < t1; t += kTile) {
        __syncthreads();
        load_tile(p, it.pt_off, 0, kvh, t, t1, tile);
        __syncthreads();
        const bool on = t + tl <= seen && t + tl < t1;
        const float s = on ? dot(q + r * D, tile + tl * (D + 1), D) : -INFINITY;
        float tm = s;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) tm = fmaxf(tm, __shfl_xor(tm, x));
        const float mn = fmaxf(m, tm), ref = mn == -INFINITY ? 0.f : mn;
        const float w = on ? fast_exp2(s - ref) : 0.f;
        float ws = w;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) ws += __shfl_xor(ws, x);
        const float c = m == -INFINITY ? 0.f : fast_exp2(m - ref);
        l = fmaf(l, c, ws);
        m = mn;
        prob[threadIdx.x] = w;
        if (tl == 0) corr[r] = c;
        __syncthreads();
        load_tile(p, it.pt_off, 1, kvh, t, t1, tile);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int cnt = min(min(kTile, t1 - t), it.pos0 + min(rho0 + i, rho1 - 1) / g + 1 - t);
#pragma unroll
            for (int c2 = 0; c2 < NC; ++c2) {
                const int d = threadIdx.x + kThreads * c2;
                if (d >= D) continue;
                float o = 0.f;
                for (int k = 0; k < cnt; ++k) o = fmaf(prob[i * kTile + k], tile[k * (D + 1) + d], o);
                acc[i][c2] = fmaf(acc[i][c2], corr[i], o);
            }
        }
    }
    // (m, l) of the rows to every thread
    __syncthreads();
    if (tl == 0) {
        prob[r] = m;
        prob[kRows + r] = l;
    }
    __syncthreads();
    // A sum that is no number though the weights are: an infinite V of a weight that rounds to zero.  It is that infinity,
    // unless the row sees a NaN or both.
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = threadIdx.x + kThreads * c;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kRows; ++i) bad |= rho0 + i < rho1 && acc[i][c] != acc[i][c] && prob[kRows + i] == prob[kRows + i];
        if (d >= D || !bad) continue;
        const NotFinite f = find_not_finite(p.pool, p.page_table + it.pt_off, p.geom, p.dtype, kvh, d, t0, t1);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (acc[i][c] != acc[i][c] && prob[kRows + i] == prob[kRows + i])
                acc[i][c] = f.settle(it.pos0 + min(rho0 + i, rho1 - 1) / g + 1, acc[i][c]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int rho = rho0 + i;
        if (rho >= rho1) break;
        const long long rh = static_cast<long long>(it.row0 + rho / g) * p.heads + h0 + rho % g;
        const float mi = prob[i], li = prob[kRows + i];
        const long long slot = it.slot0 + (static_cast<long long>(rho / g) * p.heads + h0 + rho % g) * it.splits + split;
        for (int c = 0; c < NC; ++c) {
            const int d = threadIdx.x + kThreads * c;
            if (d >= D) continue;
            if (it.splits == 1) store_out(p.out, p.act, rh * D + d, acc[i][c] / li);
            else p.part_acc[slot * D + d] = acc[i][c];
        }
        if (threadIdx.x == 0) {
            if (it.splits > 1) p.part_ml[slot] = make_float2(mi, li);
            else if (p.row_ml) p.row_ml[rh] = make_float2(mi, li);
        }
    }
}

// Weights of 32 positions of one kv head: a thread keeps the sum of one position over every
// eighth row, the eight sums are added at the end.
__global__ void __launch_bounds__(kThreads) chunks_any_weights_kernel(const ChunksK p) {
    extern __shared__ float lds[];
    const int D = p.geom.head_dim;
    float* const q = lds;               // [8][D]
    float* const tile = q + kRows * D;  // [32][D + 1]
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int len = it.pos0 + it.rows;
    const int u = blockIdx.x - it.unit0;
    const int t0 = u % it.blocks * kTile, kvh = u / it.blocks;
    int h0, g;
    chunk_heads(p, kvh, &h0, &g);
    load_tile(p, it.pt_off, 0, kvh, t0, len, tile);
    const int r = threadIdx.x >> 5, tl = threadIdx.x & 31, t = t0 + tl;
    float sum = 0.f;
    const int first = max(0, t0 - it.pos0) * g;  // rows before it see none of the tile
    for (int rho0 = first / kRows * kRows; rho0 < it.rows * g; rho0 += kRows) {
        __syncthreads();
        load_rows(p, it, rho0, h0, g, q);
        __syncthreads();
        const int rho = rho0 + r;
        if (rho < it.rows * g && t <= it.pos0 + rho / g) {
            const float2 ml = p.row_ml[static_cast<long long>(it.row0 + rho / g) * p.heads + h0 + rho % g];
            sum += fast_exp2(dot(q + r * D, tile + tl * (D + 1), D) - ml.x) / ml.y;
        }
    }
    __syncthreads();
    q[threadIdx.x] = sum;
    __syncthreads();
    if (r == 0 && t < len) {
        float s[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) s[i] = q[32 * i + tl];
        float* w = p.weights + (static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t;
        *w += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }
}

size_t any_lds(int D) { return (kRows * std::max(D, 32) + kTile * (D + 1) + kRows * kTile + kRows) * sizeof(float); }

}  // namespace

hipError_t launch_chunks_any(const ChunksK& k, hipStream_t s) {
    hipLaunchKernelGGL(chunks_any_kernel, dim3(k.units), dim3(kThreads), any_lds(k.geom.head_dim), s, k);
    return hipGetLastError();
}
hipError_t launch_chunks_any_weights(const ChunksK& k, hipStream_t s) {
    hipLaunchKernelGGL(chunks_any_weights_kernel, dim3(k.units), dim3(kThreads), any_lds(k.geom.head_dim), s, k);
    return hipGetLastError();
}

}  // namespace qr
