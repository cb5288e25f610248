// qr_forms_any.hip -- attention in its other forms and behind shared prefixes: any cache type, head size and head count (what
// the MFMA kernels do not take: other head sizes, head counts that do not divide), gfx950.  A workgroup takes 8 rows (query, query
// head pairs of a kv head) against a part of an item's keys, 32 at a time through LDS in 32 bits; a thread has one score, then
// some dims of every row.
//
// Bound by LDS reads, one for each product: with 32 heads of 96 over 8 kv heads, 16 bf16 sequences of 4096 positions took 412 us and
// 512 rows after 3584 4650 us, where fp32 MFMAs take 59 and 266 (qr_forms_f32.hip).
//
// A row never touches a position that it does not see, so that what such a slot holds (NaN too) does not matter.
#include "qr_forms.hpp"
#include "qr_quant.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = kFormAnyRows;
constexpr int kTile = kFormAnyTile;

__device__ __forceinline__ float load_cached(const FormsK& p, long long phys, int plane, int kvh, int slot, int d) {
    const long long at = p.geom.offset(phys, plane, kvh, slot, d);
    if (!p.geom.scaled()) return load_elem(p.pool, p.dtype, at);
    const uint8_t* b = reinterpret_cast<const uint8_t*>(p.pool);
    return quant_value<0>(b[at]) * scale_of(b[p.geom.scale_offset(phys, plane, kvh, slot)]);
}

// Slots t0 .. t0 + 31 (up to `last`, one page) of one plane and kv head into LDS as fp32, rows of D + 1 values: a column's
// 32 reads hit 32 banks.
__device__ __forceinline__ void load_tile(const FormsK& p, int pt_off, int plane, int kvh, int t0, int last, float* tile) {
    const int D = p.geom.head_dim;
    const long long phys = p.page_table[pt_off + (t0 >> kPageShift)];
    const int n = min(kTile, last + 1 - t0) * D;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int t = i / D, d = i - t * D;
        tile[t * (D + 1) + d] = load_cached(p, phys, plane, kvh, (t0 & (kPageTokens - 1)) + t, d);
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

__global__ void __launch_bounds__(kThreads) forms_any_kernel(const FormsK p) {
    extern __shared__ float lds[];
    __shared__ int lo[kRows], hi[kRows], pos[kRows], chunk[kRows];
    const int D = p.geom.head_dim;
    float* const q = lds;                        // [8][D]
    float* const tile = q + kRows * D;           // [32][D + 1]
    float* const prob = tile + kTile * (D + 1);  // [8][32]
    float* const corr = prob + kRows * kTile;    // [8]
    const FormItem it = p.it[form_find(p, blockIdx.x)];
    const int u = blockIdx.x - it.unit0;
    const FormUnit un = form_unit(p, it, (p.heads + p.geom.kv_heads - 1) / p.geom.kv_heads, kRows, kTile, u);
    const int split = un.part, kvh = un.kvh;
    int h0, g;
    form_heads(p, kvh, &h0, &g);
    const int rho0 = un.block * kRows;
    if (rho0 >= it.rows * g) return;
    const int rho1 = min(rho0 + kRows, it.rows * g);
    if (threadIdx.x < kRows) {
        const FormSpan s = form_row(p, it, min(rho0 + static_cast<int>(threadIdx.x), rho1 - 1) / g);
        lo[threadIdx.x] = s.lo;
        hi[threadIdx.x] = s.hi;
        pos[threadIdx.x] = s.pos - it.base;
        chunk[threadIdx.x] = s.chunk;
    }
    for (int i = threadIdx.x; i < kRows * D; i += kThreads) {
        const int r = i / D, d = i - r * D;
        const int rho = min(rho0 + r, rho1 - 1);
        q[i] = load_elem(p.q, p.act, ((it.row0 + rho / g) * static_cast<long long>(p.heads) + h0 + rho % g) * D + d) * p.qscale;
    }
    __syncthreads();
    int first = it.keys, last = -1;  // slots that some row sees
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        if (lo[i] <= hi[i]) {
            first = min(first, lo[i]);
            last = max(last, hi[i]);
        }
    const int tile0 = first / kTile, tiles = last < first ? 0 : last / kTile - tile0 + 1;
    const int t0 = (tile0 + static_cast<int>(static_cast<long long>(tiles) * split / un.parts)) * kTile;
    const int t1 = (tile0 + static_cast<int>(static_cast<long long>(tiles) * (split + 1) / un.parts)) * kTile;

    const int r = threadIdx.x >> 5, tl = threadIdx.x & 31;  // this thread's score
    const float slope = p.slopes ? p.slopes[h0 + min(rho0 + r, rho1 - 1) % g] * kLog2e : 0.f;
    float m = -INFINITY, l = 0.f;  // of row r, the same in its 32 lanes
    constexpr int NC = kGenericMaxDim / kThreads;
    float acc[kRows][NC];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = 0.f;
    for (int t = t0; t < t1; t += kTile) {
        __syncthreads();
        load_tile(p, it.pt_off, 0, kvh, t, last, tile);
        __syncthreads();
        const bool on = t + tl >= lo[r] && t + tl <= hi[r];
        const float s = on ? form_score(dot(q + r * D, tile + tl * (D + 1), D), p.cap, slope, static_cast<float>(t + tl - pos[r])) : -INFINITY;
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
        load_tile(p, it.pt_off, 1, kvh, t, last, tile);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int k0 = max(lo[i] - t, 0), k1 = min(hi[i] + 1 - t, kTile);
#pragma unroll
            for (int c2 = 0; c2 < NC; ++c2) {
                const int d = threadIdx.x + kThreads * c2;
                if (d >= D) continue;
                float o = 0.f;
                for (int k = k0; k < k1; ++k) o = fmaf(prob[i * kTile + k], tile[k * (D + 1) + d], o);
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
    // A sum that is no number while that of its weights is: an infinite V whose weight is zero in 32 bits, but none in the
    // formula.  The row shows the sum of these elements, found in one pass over the dim.
#pragma unroll
    for (int c2 = 0; c2 < NC; ++c2) {
        const int d = threadIdx.x + kThreads * c2;
        bool lost = false;
#pragma unroll
        for (int i = 0; i < kRows; ++i) lost |= acc[i][c2] != acc[i][c2] && prob[kRows + i] == prob[kRows + i];
        if (d >= D || !lost || p.geom.scaled()) continue;
        float shown[kRows] = {};
        for (int t = t0; t < min(t1, last + 1); ++t) {
            const float x = load_cached(p, p.page_table[it.pt_off + (t >> kPageShift)], 1, kvh, t & (kPageTokens - 1), d);
            if (fabsf(x) < INFINITY) continue;
#pragma unroll
            for (int i = 0; i < kRows; ++i)
                if (t >= lo[i] && t <= hi[i]) shown[i] += x;
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (acc[i][c2] != acc[i][c2]) acc[i][c2] = shown[i];
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int rho = rho0 + i;
        if (rho >= rho1) break;
        const FormRows& c = p.c[chunk[i]];
        const int row = it.row0 + rho / g;
        const float mi = prob[i], li = prob[kRows + i];
        const long long slot = c.slot0 + (static_cast<long long>(row - c.row0) * p.heads + h0 + rho % g) * c.parts + it.part0 + split;
#pragma unroll
        for (int c2 = 0; c2 < NC; ++c2) {
            const int d = threadIdx.x + kThreads * c2;
            if (d >= D) continue;
            if (form_whole(c, it, un.parts)) store_out(p.out, p.act, (static_cast<long long>(row) * p.heads + h0 + rho % g) * D + d, li == 0.f ? 0.f : acc[i][c2] / li);
            else p.part_acc[slot * D + d] = acc[i][c2];
        }
        if (threadIdx.x == 0) form_store_ml(p, c, it, slot, un, mi, li);
    }
}

size_t any_lds(int D) { return (kRows * std::max(D, 32) + kTile * (D + 1) + kRows * kTile + kRows) * sizeof(float); }

}  // namespace

hipError_t launch_forms_any(const FormsK& k, int units, hipStream_t s) {
    hipLaunchKernelGGL(forms_any_kernel, dim3(units), dim3(kThreads), any_lds(k.geom.head_dim), s, k);
    return hipGetLastError();
}

}  // namespace qr
