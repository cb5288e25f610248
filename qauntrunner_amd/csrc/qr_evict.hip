// qr_evict.hip -- eviction from the paged cache by accumulated attention weight, gfx950.
//
// Of a sequence's `len` positions each kv head keeps the first `first`, the last `recent` and the
// `heavy` positions between them that have the largest weight (ties: the lower position; NaN counts
// below every number), in their order: slot j takes what slot kept[j] held, kept[j] >= j.
#include "qr_batch.hpp"

namespace qr {
namespace {

constexpr int kSelThreads = 1024;

// Ascending with the value; -0 and 0 are equal, NaN lowest.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per (entry, kv head): the key of the last position taken, digit by digit from the
// top (8 bits a pass), then the kept positions in order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    constexpr int kWaves = kSelThreads / 64;
    __shared__ int hist[256];
    __shared__ int wsum[2][kWaves];
    __shared__ uint32_t sh_prefix;
    __shared__ int sh_need;
    const int kvh = blockIdx.x % a.geom.kv_heads;
    const EvictItem it = a.it[blockIdx.x / a.geom.kv_heads];
    const long long wrow = (static_cast<long long>(it.seq) * a.geom.kv_heads + kvh) * a.max_seq;
    const float* const w = a.weights + wrow;
    float* const ow = a.kept_weights + wrow;
    const int keep = a.first + a.heavy + a.recent;
    int* const kept = a.kept + (static_cast<long long>(it.entry) * a.geom.kv_heads + kvh) * keep;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (it.len <= keep) {  // nothing leaves
        for (int i = tid; i < keep; i += kSelThreads) kept[i] = i < it.len ? i : -1;
        if (ow != w)
            for (int i = tid; i < it.len; i += kSelThreads) ow[i] = w[i];
        return;
    }
    const int lo = a.first, hi = it.len - a.recent;  // candidates
    uint32_t prefix = 0, mask = 0;
    int need = a.heavy;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kSelThreads) {
                const uint32_t k = weight_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {  // from the largest digit down, until `need` are passed
                int left = need, d = 255;
                while (d > 0 && hist[d] < left) left -= hist[d--];
                sh_need = left;
                sh_prefix = prefix | static_cast<uint32_t>(d) << shift;
            }
            __syncthreads();
            prefix = sh_prefix;
            need = sh_need;
            mask |= 255u << shift;
            __syncthreads();
        }
    }
    // in order: every position above the key, and the first `need` of those that equal it
    int eq_before = 0, out_before = 0;
    for (int i0 = 0; i0 < it.len; i0 += kSelThreads) {
        const int i = i0 + tid;
        const bool held = i < it.len, cand = i >= lo && i < hi;
        const float x = held ? w[i] : 0.f;
        const uint32_t k = weight_key(x);
        const bool eq = cand && a.heavy > 0 && k == prefix;
        const uint64_t be = __builtin_amdgcn_ballot_w64(eq);
        if (lane == 0) wsum[0][wave] = __popcll(be);
        __syncthreads();  // every weight of the tile is read
        int eq_at = eq_before + __popcll(be & ((1ull << lane) - 1)), eq_all = 0;
        for (int j = 0; j < kWaves; ++j) {
            if (j < wave) eq_at += wsum[0][j];
            eq_all += wsum[0][j];
        }
        const bool take = held && (!cand || (a.heavy > 0 && (k > prefix || (eq && eq_at < need))));
        const uint64_t bt = __builtin_amdgcn_ballot_w64(take);
        if (lane == 0) wsum[1][wave] = __popcll(bt);
        __syncthreads();
        int at = out_before + __popcll(bt & ((1ull << lane) - 1)), all = 0;
        for (int j = 0; j < kWaves; ++j) {
            if (j < wave) at += wsum[1][j];
            all += wsum[1][j];
        }
        if (take) {
            kept[at] = i;
            ow[at] = x;  // at <= i: its own weight is read, in this tile or an earlier one
        }
        eq_before += eq_all;
        out_before += all;
    }
    __syncthreads();
    for (int i = keep + tid; i < it.len; i += kSelThreads) ow[i] = 0.f;
}

constexpr int kMoveThreads = 256;

// K or V rows of one kv head, up to 8 dims of them: slots in ascending order, each tile read whole
// before it is written (a slot's source lies at or behind it, so a later tile's sources are not
// written yet).
__global__ void __launch_bounds__(kMoveThreads) evict_move_any_kernel(const EvictArgs a) {
    const int D = a.geom.head_dim, slices = (D + 7) / 8;
    int u = blockIdx.x;
    const int slice = u % slices;
    u /= slices;
    const int plane = u & 1;
    u >>= 1;
    const int kvh = u % a.geom.kv_heads;
    const EvictItem it = a.it[u / a.geom.kv_heads];
    const int keep = a.first + a.heavy + a.recent;
    if (it.len <= keep) return;
    const int* const kept = a.kept + (static_cast<long long>(it.entry) * a.geom.kv_heads + kvh) * keep;
    const int d0 = 8 * slice, nd = min(8, D - d0);
    for (int j0 = 0; j0 < keep; j0 += kMoveThreads) {
        const int j = j0 + threadIdx.x;
        const int src = j < keep ? kept[j] : j;
        uint32_t x[8];
        if (src != j) {
            const long long phys = a.page_table[it.pt_off + (src >> kPageShift)];
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                if (d >= nd) continue;
                const long long at = a.geom.offset(phys, plane, kvh, src & (kPageTokens - 1), d0 + d);
                x[d] = a.dtype == QR_DTYPE_F32 ? static_cast<const uint32_t*>(a.pool)[at] : static_cast<const uint16_t*>(a.pool)[at];
            }
        }
        __syncthreads();
        if (src != j) {
            const long long phys = a.page_table[it.pt_off + (j >> kPageShift)];
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                if (d >= nd) continue;
                const long long at = a.geom.offset(phys, plane, kvh, j & (kPageTokens - 1), d0 + d);
                if (a.dtype == QR_DTYPE_F32) static_cast<uint32_t*>(a.pool)[at] = x[d];
                else static_cast<uint16_t*>(a.pool)[at] = static_cast<uint16_t>(x[d]);
            }
        }
        __syncthreads();
    }
}

}  // namespace

hipError_t launch_evict(const EvictArgs& a, hipStream_t stream) {
    if (!a.n) return hipSuccess;
    const int rows = a.n * a.geom.kv_heads;
    hipLaunchKernelGGL(evict_select_kernel, dim3(rows), dim3(kSelThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(evict_move_any_kernel, dim3(rows * 2 * ((a.geom.head_dim + 7) / 8)), dim3(kMoveThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qr
