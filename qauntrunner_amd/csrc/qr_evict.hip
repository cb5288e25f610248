// qr_evict.hip -- eviction from the paged cache by accumulated attention weight, gfx950.
//
// Of a sequence's `len` positions each kv head keeps the first `first`, the last `recent` and the
// `heavy` positions between them that have the largest weight (ties: the lower position; NaN counts
// below every number), in their order: slot j takes what slot kept[j] held, kept[j] >= j.
#include "qr_batch.hpp"

#include <algorithm>

namespace qr {
namespace {

constexpr int kSelThreads = 1024;

// Ascending with the value; -0 and 0 are equal, NaN lowest.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (x != x) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Inclusive sum over a workgroup of 1024 threads; `wsum` holds a value per wave.
__device__ __forceinline__ int block_scan(int x, int* wsum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) wsum[wave] = x;
    __syncthreads();
    for (int w = 0; w < wave; ++w) x += wsum[w];
    __syncthreads();
    return x;
}

// The weight of a key (any NaN for 0).
__device__ __forceinline__ float key_weight(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// One workgroup per (entry, kv head): the key of the last position taken, digit by digit from the
// top (11, 11 and 10 bits: counts in LDS, then a scan from the largest digit down), then the kept positions in order.
// The weights stay in registers, C per thread; C = 0: longer rows, read from L2 in every pass.  Bound by the instructions
// of its one CU.
template <int C>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    constexpr int kWaves = kSelThreads / 64, kBins = 2048;
    __shared__ int hist[kBins];
    __shared__ int wsum[kWaves];
    __shared__ int before[2][C > 0 ? C * kWaves : 1];
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
    const int chunks = C > 0 ? C : (it.len + kSelThreads - 1) / kSelThreads;
    float x[C > 0 ? C : 1];
    if (C > 0)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = c * kSelThreads + tid;
            x[c] = i < it.len ? w[i] : 0.f;
        }
    auto value = [&](int c, int i) { return C > 0 ? x[C > 0 ? c : 0] : i < it.len ? w[i] : 0.f; };
    uint32_t prefix = 0, mask = 0;
    int need = a.heavy;
    if (need > 0) {
        constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            auto count = [&](int c) __attribute__((always_inline)) {
                if (c * kSelThreads >= hi) return;
                const int i = c * kSelThreads + tid;
                const uint32_t k = weight_key(value(c, i));
                if (static_cast<uint32_t>(i - lo) < static_cast<uint32_t>(hi - lo) && (k & mask) == prefix)
                    atomicAdd(&hist[(k >> kShift[pass]) & ((1 << kBits[pass]) - 1)], 1);
            };
            if (C > 0) {
#pragma unroll
                for (int c = 0; c < C; ++c) count(c);
            } else {
                for (int c = 0; c < chunks; ++c) count(c);
            }
            __syncthreads();
            // thread t: the digits kBins - 1 - 2t and the one below; the one where the counts from above reach `need`
            const int top = kBins - 1 - 2 * tid, h1 = hist[top], h0 = hist[top - 1];
            const int upto = block_scan(h1 + h0, wsum), above = upto - h1 - h0;
            if (above < need && need <= upto) {
                const bool first = need <= above + h1;
                sh_need = need - above - (first ? 0 : h1);
                sh_prefix = prefix | static_cast<uint32_t>(first ? top : top - 1) << kShift[pass];
            }
            __syncthreads();
            prefix = sh_prefix;
            need = sh_need;
            mask |= ((1u << kBits[pass]) - 1) << kShift[pass];
        }
    }
    // in order: the positions outside the candidates, those above the key, and the first `need` of those that equal it.
    // With A the former two and E the last before a position, it goes to slot A + min(E, need).
    const float T = a.heavy > 0 ? key_weight(prefix) : INFINITY;
    const bool nan = a.heavy > 0 && prefix == 0;  // even some NaN stay: the numbers do before them
    auto flags = [&](int c, int i, bool* sure, bool* eq) __attribute__((always_inline)) {
        const float v = value(c, i);
        const bool cand = static_cast<uint32_t>(i - lo) < static_cast<uint32_t>(hi - lo);
        *sure = cand ? (nan ? v == v : v > T) : i < it.len;
        *eq = a.heavy > 0 && cand && (nan ? v != v : v == T);
    };
    const uint64_t below = (1ull << lane) - 1;
    if (C > 0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            bool sure, eq;
            flags(c, c * kSelThreads + tid, &sure, &eq);
            const uint64_t bs = __builtin_amdgcn_ballot_w64(sure), be = __builtin_amdgcn_ballot_w64(eq);
            if (lane == 0) {
                before[0][C > 0 ? c * kWaves + wave : 0] = __popcll(bs);
                before[1][C > 0 ? c * kWaves + wave : 0] = __popcll(be);
            }
        }
        __syncthreads();  // every weight is read
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int v = tid < C * kWaves ? before[q][C > 0 ? tid : 0] : 0;
            const int s = block_scan(v, wsum) - v;
            if (tid < C * kWaves) before[q][C > 0 ? tid : 0] = s;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c * kSelThreads >= it.len) break;
            const int i = c * kSelThreads + tid;
            bool sure, eq;
            flags(c, i, &sure, &eq);
            const uint64_t bs = __builtin_amdgcn_ballot_w64(sure), be = __builtin_amdgcn_ballot_w64(eq);
            const int e = before[1][C > 0 ? c * kWaves + wave : 0] + __popcll(be & below);
            const int at = before[0][C > 0 ? c * kWaves + wave : 0] + __popcll(bs & below) + min(e, need);
            if (sure || (eq && e < need)) {
                kept[at] = i;
                ow[at] = value(c, i);
            }
        }
    } else {
        __shared__ int cnt[2][kWaves];
        int sure_before = 0, eq_before = 0;
        for (int c = 0; c < chunks; ++c) {
            const int i = c * kSelThreads + tid;
            const float v = value(c, i);
            bool sure, eq;
            flags(c, i, &sure, &eq);
            const uint64_t bs = __builtin_amdgcn_ballot_w64(sure), be = __builtin_amdgcn_ballot_w64(eq);
            if (lane == 0) {
                cnt[0][wave] = __popcll(bs);
                cnt[1][wave] = __popcll(be);
            }
            __syncthreads();  // every weight of the chunk is read: slot at <= i, in this chunk or an earlier one
            int s = sure_before + __popcll(bs & below), e = eq_before + __popcll(be & below);
            for (int q = 0; q < kWaves; ++q) {
                if (q < wave) {
                    s += cnt[0][q];
                    e += cnt[1][q];
                }
                sure_before += cnt[0][q];
                eq_before += cnt[1][q];
            }
            __syncthreads();
            if (sure || (eq && e < need)) {
                kept[s + min(e, need)] = i;
                ow[s + min(e, need)] = v;
            }
        }
        __syncthreads();
    }
    for (int i = keep + tid; i < it.len; i += kSelThreads) ow[i] = 0.f;
}

constexpr int kMoveThreads = 256;

// The same for head sizes whose rows are whole 16-byte pieces, P of a row (or what is left of it) per workgroup, 2048 / P
// slots at a time; the next ones are read before these are written.  V of the MFMA page layout: 16 dims per workgroup, a thread
// gathers 8 slots of a dim (16 bytes of the page; reading ahead here costs registers and 10 us of 38).  Bound by HBM for
// many workgroups, else by the latency of a tile.
template <int ES, bool MFMA, int P>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
    constexpr int N = 16 / ES, TILE = MFMA ? 512 : 2048 / P;
    const int D = a.geom.head_dim, pieces = D / N;
    const int ks = (pieces + P - 1) / P, vs = MFMA ? D / 16 : ks;  // workgroups of the K and the V rows of a kv head
    int u = blockIdx.x;
    const int part = u % (ks + vs);
    u /= ks + vs;
    const int kvh = u % a.geom.kv_heads;
    const EvictItem it = a.it[u / a.geom.kv_heads];
    const int keep = a.first + a.heavy + a.recent;
    if (it.len <= keep) return;
    const int* const kept = a.kept + (static_cast<long long>(it.entry) * a.geom.kv_heads + kvh) * keep;
    const int* const pages = a.page_table + it.pt_off;
    auto page = [&](int j) { return static_cast<long long>(pages[j >> kPageShift]); };
    const int plane = part >= ks, s = part - plane * ks;
    auto moved = [&](int j0) { return kept[min(j0 + TILE, keep) - 1] != min(j0 + TILE, keep) - 1; };
    int j0 = 0;
    while (j0 < keep && !moved(j0)) j0 += TILE;  // slots that keep what they hold
    if (j0 >= keep) return;
    if (MFMA && plane) {
        constexpr int IT = 16 * TILE / 8 / kMoveThreads;
        const int d = 16 * s + (threadIdx.x & 15);
        for (; j0 < keep; j0 += TILE) {
            uint16_t x[IT][8];
#pragma unroll
            for (int c = 0; c < IT; ++c) {
                const int j = j0 + 8 * ((threadIdx.x >> 4) + kMoveThreads / 16 * c);
                int src[8];
                long long phys[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) src[k] = kept[min(j + k, keep - 1)];
#pragma unroll
                for (int k = 0; k < 8; ++k) phys[k] = page(src[k]);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    x[c][k] = static_cast<const uint16_t*>(a.pool)[a.geom.offset(phys[k], 1, kvh, src[k] & (kPageTokens - 1), d)];
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < IT; ++c) {
                const int j = j0 + 8 * ((threadIdx.x >> 4) + kMoveThreads / 16 * c);
                if (j >= keep) continue;
                uint16_t* o = static_cast<uint16_t*>(a.pool) + a.geom.offset(pages[j >> kPageShift], 1, kvh, j & (kPageTokens - 1), d);
                if (j + 8 <= keep) {
                    uint4 v;
                    __builtin_memcpy(&v, x[c], 16);
                    *reinterpret_cast<uint4*>(o) = v;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (j + k < keep) o[k] = x[c][k];
                }
            }
        }
        return;
    }
    constexpr int IT = 8, STEP = kMoveThreads / P;
    static_assert(IT * STEP == TILE, "whole tiles");
    // MFMA layout: consecutive lanes take consecutive slots (their pieces lie side by side), else the pieces of a slot
    const int pc = P * s + static_cast<int>(MFMA ? threadIdx.x / STEP : threadIdx.x % P);
    const int q0 = MFMA ? threadIdx.x % STEP : threadIdx.x / P;
    const bool in = pc < pieces;
    const int piece = in ? pc : pieces - 1;  // (an idle thread reads a piece that it does not write)
    int src[IT];
    U32x4 x[IT], y[IT];
    char* const pool = static_cast<char*>(a.pool);
    auto look = [&](int j1) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < IT; ++c) src[c] = kept[min(j1 + q0 + STEP * c, keep - 1)];
    };
    auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < IT; ++c)
            y[c] = load16(pool + ES * a.geom.offset(page(src[c]), plane, kvh, src[c] & (kPageTokens - 1), N * piece));
    };
    look(j0);
    load();
    look(j0 + TILE);
    for (; j0 < keep; j0 += TILE) {
#pragma unroll
        for (int c = 0; c < IT; ++c) x[c] = y[c];
        if (j0 + TILE < keep) {
            load();
            look(j0 + 2 * TILE);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < IT; ++c) {
            const int j = j0 + q0 + STEP * c;
            if (in && j < keep)
                *reinterpret_cast<U32x4*>(pool + ES * a.geom.offset(page(j), plane, kvh, j & (kPageTokens - 1), N * pc)) = x[c];
        }
    }
}

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
    const int rows = a.n * a.geom.kv_heads, keep = a.first + a.heavy + a.recent;
    int longest = 0;
    for (int i = 0; i < a.n; ++i)
        if (a.it[i].len > keep) longest = std::max(longest, a.it[i].len);
    const dim3 grid(rows), block(kSelThreads);
    if (longest <= 4 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<4>, grid, block, 0, stream, a);
    else if (longest <= 16 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<16>, grid, block, 0, stream, a);
    else if (longest <= 32 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<32>, grid, block, 0, stream, a);
    else if (longest <= 64 * kSelThreads) hipLaunchKernelGGL(evict_select_kernel<64>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !longest) return e;
    // four pieces of a row per workgroup, two where that leaves CUs idle (8192 of 65536 fp32 positions
    // kept: 74 us, 103 with four)
    const int D = a.geom.head_dim, n = 16 / dtype_size(a.dtype), ks4 = (D / n + 3) / 4, ks2 = (D / n + 1) / 2;
    const dim3 mblock(kMoveThreads);
    const bool two = rows * 2 * ks4 < 512;
    if (D % n) hipLaunchKernelGGL(evict_move_any_kernel, dim3(rows * 2 * ((D + 7) / 8)), mblock, 0, stream, a);
    else if (a.geom.mfma_layout) hipLaunchKernelGGL((evict_move_kernel<2, true, 4>), dim3(rows * (ks4 + D / 16)), mblock, 0, stream, a);
    else if (a.dtype == QR_DTYPE_F32 && two) hipLaunchKernelGGL((evict_move_kernel<4, false, 2>), dim3(rows * 2 * ks2), mblock, 0, stream, a);
    else if (a.dtype == QR_DTYPE_F32) hipLaunchKernelGGL((evict_move_kernel<4, false, 4>), dim3(rows * 2 * ks4), mblock, 0, stream, a);
    else if (two) hipLaunchKernelGGL((evict_move_kernel<2, false, 2>), dim3(rows * 2 * ks2), mblock, 0, stream, a);
    else hipLaunchKernelGGL((evict_move_kernel<2, false, 4>), dim3(rows * 2 * ks4), mblock, 0, stream, a);
    return hipGetLastError();
}

}  // namespace qr
