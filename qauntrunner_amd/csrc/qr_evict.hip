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
#pragma unroll
    for (int w = 0; w < kSelThreads / 64; ++w) x += w < wave ? wsum[w] : 0;
    __syncthreads();
    return x;
}

// The weight of a key (any NaN for 0).
__device__ __forceinline__ float key_weight(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// The digits of a key, from the top.
constexpr int kBins = 2048;
__device__ constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
__device__ __forceinline__ uint32_t digits_above(int pass) { return pass ? ~0u << kShift[pass - 1] : 0u; }

// Which positions stay: `sure` those outside the candidates and those above the key, and the first `need` of `eq`, that
// equal it.  With A of the former and E of the latter before a position, it goes to slot A + min(E, need).
struct Stay {
    int lo, hi, len, heavy;
    uint32_t key;
    __device__ __forceinline__ bool candidate(int i) const { return static_cast<uint32_t>(i - lo) < static_cast<uint32_t>(hi - lo); }
    __device__ __forceinline__ void operator()(int i, float v, bool* sure, bool* eq) const {
        const float T = heavy > 0 ? key_weight(key) : INFINITY;
        const bool nan = heavy > 0 && key == 0;  // even some NaN stay: the numbers do before them
        const bool cand = candidate(i);
        *sure = cand ? (nan ? v == v : v > T) : i < len;
        *eq = heavy > 0 && cand && (nan ? v != v : v == T);
    }
};

// In order: x holds the weights of positions c * 1024 + thread + p0, A and E stand before p0.  out may hold the weights read.
template <int C>
__device__ __forceinline__ void place(const Stay& stay, const float (&x)[C], int p0, int A, int E, int need, int (&before)[2][C * kSelThreads / 64],
                                      int* wsum, int* kept, float* out) {
    constexpr int kWaves = kSelThreads / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        bool sure, eq;
        stay(p0 + c * kSelThreads + tid, x[c], &sure, &eq);
        const uint64_t bs = __builtin_amdgcn_ballot_w64(sure), be = __builtin_amdgcn_ballot_w64(eq);
        if (lane == 0) {
            before[0][c * kWaves + wave] = __popcll(bs);
            before[1][c * kWaves + wave] = __popcll(be);
        }
    }
    __syncthreads();  // every weight is read
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int v = tid < C * kWaves ? before[q][tid] : 0;
        const int s = block_scan(v, wsum) - v;
        if (tid < C * kWaves) before[q][tid] = s;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = p0 + c * kSelThreads + tid;
        if (p0 + c * kSelThreads >= stay.len) break;
        bool sure, eq;
        stay(i, x[c], &sure, &eq);
        const uint64_t bs = __builtin_amdgcn_ballot_w64(sure), be = __builtin_amdgcn_ballot_w64(eq);
        const int e = E + before[1][c * kWaves + wave] + __popcll(be & below);
        const int at = A + before[0][c * kWaves + wave] + __popcll(bs & below) + min(e, need);
        if (sure || (eq && e < need)) {
            kept[at] = i;
            out[at] = x[c];
        }
    }
}

// One workgroup per (entry, kv head): the key of the last position taken, digit by digit from the
// top (11, 11 and 10 bits: counts in LDS, then a scan from the largest digit down), then the kept positions in order.
// The weights stay in registers, C per thread; C = 0: longer rows, read from L2 in every pass.  Bound by the instructions
// of its one CU.
template <int C>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    constexpr int kWaves = kSelThreads / 64;
    __shared__ int hist[kBins];
    __shared__ int wsum[kWaves];
    __shared__ int before[2][(C > 0 ? C : 1) * kWaves];
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
    uint32_t prefix = 0;
    int need = a.heavy;
    if (need > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            auto count = [&](int c) __attribute__((always_inline)) {
                if (c * kSelThreads >= hi) return;
                const int i = c * kSelThreads + tid;
                const uint32_t k = weight_key(value(c, i));
                if (static_cast<uint32_t>(i - lo) < static_cast<uint32_t>(hi - lo) && (k & digits_above(pass)) == prefix)
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
        }
    }
    const Stay stay{lo, hi, it.len, a.heavy, prefix};
    if (C > 0) {
        place(stay, x, 0, 0, 0, need, before, wsum, kept, ow);
    } else {
        __shared__ int cnt[2][kWaves];
        const uint64_t below = (1ull << lane) - 1;
        int sure_before = 0, eq_before = 0;
        for (int c = 0; c < chunks; ++c) {
            const int i = c * kSelThreads + tid;
            const float v = value(c, i);
            bool sure, eq;
            stay(i, v, &sure, &eq);
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

// ---- long rows: one workgroup per kPart positions of a row, the digits counted by a launch each
constexpr int kPartC = 8, kPart = kPartC * kSelThreads;

// The workspace: digit counts of [row][digit][part], per (row, digit) the key's digits up to there and what is
// still to be taken, per (row, digit, part) the candidates before the part that lie above it, and the kept weights.
struct Parts {
    int n;  // of the longest row
    int* counts;
    int2* state;
    int* above;
    float* staged;
    __device__ __forceinline__ int* at(int row, int pass, int part) const { return counts + ((static_cast<long long>(row) * 3 + pass) * n + part) * kBins; }
};

// From the counts of all parts: the digit of `pass`, what is still to be taken, the candidates in the parts before this
// one that lie above the digit, and (`equal`) those that have it.
struct Digit {
    uint32_t prefix;
    int need, above, equal;
};
__device__ __forceinline__ Digit find_digit(const Parts& w, int row, int parts, int part, int pass, uint32_t prefix, int need, int* wsum) {
    __shared__ Digit found;
    const int tid = threadIdx.x, top = kBins - 1 - 2 * tid;
    int h1 = 0, h0 = 0, b1 = 0, b0 = 0;
#pragma unroll 8
    for (int g = 0; g < parts; ++g) {
        const int2 h = *reinterpret_cast<const int2*>(w.at(row, pass, g) + top - 1);
        h0 += h.x;
        h1 += h.y;
        if (g < part) {
            b0 += h.x;
            b1 += h.y;
        }
    }
    const int upto = block_scan(h1 + h0, wsum), above = upto - h1 - h0;
    const int bupto = block_scan(b1 + b0, wsum);
    if (above < need && need <= upto) {
        const bool first = need <= above + h1;
        found = {prefix | static_cast<uint32_t>(first ? top : top - 1) << kShift[pass], need - above - (first ? 0 : h1),
                 bupto - b0 - (first ? b1 : 0), first ? b1 : b0};
    }
    __syncthreads();
    return found;
}

template <int PASS>
__global__ void __launch_bounds__(kSelThreads) evict_count_kernel(const EvictArgs a, const Parts w) {
    __shared__ int hist[kBins];
    __shared__ int wsum[kSelThreads / 64];
    const int part = blockIdx.x % w.n, row = blockIdx.x / w.n, kvh = row % a.geom.kv_heads;
    const EvictItem it = a.it[row / a.geom.kv_heads];
    const int keep = a.first + a.heavy + a.recent, parts = (it.len + kPart - 1) / kPart;
    if (it.len <= keep || part >= parts) return;
    const float* const wt = a.weights + (static_cast<long long>(it.seq) * a.geom.kv_heads + kvh) * a.max_seq;
    const int tid = threadIdx.x, lo = a.first, hi = it.len - a.recent;
    float x[kPartC];
#pragma unroll
    for (int c = 0; c < kPartC; ++c) {
        const int i = part * kPart + c * kSelThreads + tid;
        x[c] = i < it.len ? wt[i] : 0.f;
    }
    uint32_t prefix = 0;
    if (PASS > 0) {
        const int2 s = PASS > 1 ? w.state[row * 2] : make_int2(0, a.heavy);
        const Digit d = find_digit(w, row, parts, part, PASS - 1, static_cast<uint32_t>(s.x), s.y, wsum);
        prefix = d.prefix;
        if (tid == 0) {
            if (part == 0) w.state[row * 2 + PASS - 1] = make_int2(static_cast<int>(d.prefix), d.need);
            w.above[(row * 2 + PASS - 1) * w.n + part] = d.above;
        }
    }
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kPartC; ++c) {
        const int i = part * kPart + c * kSelThreads + tid;
        const uint32_t k = weight_key(x[c]);
        if (static_cast<uint32_t>(i - lo) < static_cast<uint32_t>(hi - lo) && (k & digits_above(PASS)) == prefix)
            atomicAdd(&hist[(k >> kShift[PASS]) & ((1 << kBits[PASS]) - 1)], 1);
    }
    __syncthreads();
    for (int i = tid; i < kBins; i += kSelThreads) w.at(row, PASS, part)[i] = hist[i];
}

__global__ void __launch_bounds__(kSelThreads) evict_place_kernel(const EvictArgs a, const Parts w) {
    __shared__ int wsum[kSelThreads / 64];
    __shared__ int before[2][kPartC * kSelThreads / 64];
    const int part = blockIdx.x % w.n, row = blockIdx.x / w.n, kvh = row % a.geom.kv_heads;
    const EvictItem it = a.it[row / a.geom.kv_heads];
    const int keep = a.first + a.heavy + a.recent, parts = (it.len + kPart - 1) / kPart;
    int* const kept = a.kept + (static_cast<long long>(it.entry) * a.geom.kv_heads + kvh) * keep;
    const int tid = threadIdx.x, p0 = part * kPart;
    if (it.len <= keep) {  // nothing leaves
        if (part == 0)
            for (int i = tid; i < keep; i += kSelThreads) kept[i] = i < it.len ? i : -1;
        return;
    }
    if (part >= parts) return;
    const float* const wt = a.weights + (static_cast<long long>(it.seq) * a.geom.kv_heads + kvh) * a.max_seq;
    const int lo = a.first, hi = it.len - a.recent;
    float x[kPartC];
#pragma unroll
    for (int c = 0; c < kPartC; ++c) {
        const int i = p0 + c * kSelThreads + tid;
        x[c] = i < it.len ? wt[i] : 0.f;
    }
    Digit d{0, 0, 0, 0};
    if (a.heavy > 0) {
        const int2 s = w.state[row * 2 + 1];
        d = find_digit(w, row, parts, part, 2, static_cast<uint32_t>(s.x), s.y, wsum);
        d.above += w.above[row * 2 * w.n + part] + w.above[(row * 2 + 1) * w.n + part];
    }
    place(Stay{lo, hi, it.len, a.heavy, d.prefix}, x, p0, min(p0, lo) + max(p0 - hi, 0) + d.above, d.equal, d.need, before, wsum, kept,
          w.staged + static_cast<long long>(row) * keep);
}

// kept_weights may be weights: written once all are read
__global__ void __launch_bounds__(256) evict_weights_kernel(const EvictArgs a, const Parts w) {
    const int blocks = kPart / 256 * w.n, row = blockIdx.x / blocks, kvh = row % a.geom.kv_heads;
    const EvictItem it = a.it[row / a.geom.kv_heads];
    const int keep = a.first + a.heavy + a.recent, i = blockIdx.x % blocks * 256 + threadIdx.x;
    if (i >= it.len) return;
    const long long at = (static_cast<long long>(it.seq) * a.geom.kv_heads + kvh) * a.max_seq + i;
    if (it.len > keep) a.kept_weights[at] = i < keep ? w.staged[static_cast<long long>(row) * keep + i] : 0.f;
    else if (a.kept_weights != a.weights) a.kept_weights[at] = a.weights[at];
}

constexpr int kMoveThreads = 1024;

// K and V rows to the slots that keep them, head sizes whose rows are whole 16-byte pieces: P pieces of a row (or what is left
// of it) per workgroup, 8192 / P slots at a time, since a tile is read before it is written; the next ones are read
// before these are written.  V of the MFMA page layout: 16 dims per workgroup, a thread gathers 8 slots of a dim (16 bytes
// of the page; reading ahead here costs registers and a third of the time).  Bound by HBM for many workgroups (16
// sequences of 3000 to 17000 bf16 positions, whose gaps share lines with what stays: 167 us), else by the latency of a tile:
// 1024 threads 14 us for one sequence of 2304, 256 threads with tiles of a quarter 22.
template <int ES, bool MFMA, int P>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a) {
    constexpr int N = 16 / ES, TILE = MFMA ? 2 * kMoveThreads : 8 * kMoveThreads / P;
    const int D = a.geom.head_dim, pieces = D / N;
    const int ks = (pieces + P - 1) / P, vs = MFMA ? D / 16 : ks;  // workgroups of the K and the V rows of a kv head
    // plain pages: the parts of a row run on one XCD where the rows are whole eights, whose L2 joins their pieces to lines
    const int rows = gridDim.x / (ks + vs);
    const int part = MFMA ? blockIdx.x % (ks + vs) : blockIdx.x / rows, u = MFMA ? blockIdx.x / (ks + vs) : blockIdx.x % rows;
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

namespace {
struct EvictShape {
    int rows, keep, longest;  // of the entries that give positions up
    int parts;                // workgroups per row, 0: one
};
// Rows of more than 32768 positions are shared by workgroups while the counts stay in L2 (8 rows of 65536: 32 us, one
// workgroup each 93; 128 rows of up to 17000: 40 us, 27)
EvictShape evict_shape(const EvictArgs& a) {
    EvictShape s{a.n * a.geom.kv_heads, a.first + a.heavy + a.recent, 0, 0};
    for (int i = 0; i < a.n; ++i)
        if (a.it[i].len > s.keep) s.longest = std::max(s.longest, a.it[i].len);
    const long long parts = (s.longest + kPart - 1) / kPart;
    if (parts > 4 && s.rows * parts <= 512) s.parts = static_cast<int>(parts);
    return s;
}
}  // namespace

size_t evict_workspace_bytes(const EvictArgs& a) {
    const EvictShape s = evict_shape(a);
    return 4 * static_cast<size_t>(s.rows) * (s.parts ? static_cast<size_t>(s.parts) * (3 * kBins + 2) + 4 + s.keep : 0);
}

hipError_t launch_evict(const EvictArgs& a, void* workspace, hipStream_t stream) {
    if (!a.n) return hipSuccess;
    const EvictShape sh = evict_shape(a);
    const int rows = sh.rows, longest = sh.longest;
    const dim3 grid(rows), block(kSelThreads);
    if (sh.parts && workspace) {
        Parts w{sh.parts, static_cast<int*>(workspace), nullptr, nullptr, nullptr};
        w.state = reinterpret_cast<int2*>(w.counts + static_cast<size_t>(rows) * 3 * w.n * kBins);
        w.above = reinterpret_cast<int*>(w.state + 2 * rows);
        w.staged = reinterpret_cast<float*>(w.above + 2 * rows * w.n);
        const dim3 pgrid(rows * w.n);
        if (a.heavy > 0) {
            hipLaunchKernelGGL(evict_count_kernel<0>, pgrid, block, 0, stream, a, w);
            hipLaunchKernelGGL(evict_count_kernel<1>, pgrid, block, 0, stream, a, w);
            hipLaunchKernelGGL(evict_count_kernel<2>, pgrid, block, 0, stream, a, w);
        }
        hipLaunchKernelGGL(evict_place_kernel, pgrid, block, 0, stream, a, w);
        hipLaunchKernelGGL(evict_weights_kernel, dim3(rows * w.n * (kPart / 256)), dim3(256), 0, stream, a, w);
    } else if (longest <= 4 * kSelThreads) {
        hipLaunchKernelGGL(evict_select_kernel<4>, grid, block, 0, stream, a);
    } else if (longest <= 16 * kSelThreads) {
        hipLaunchKernelGGL(evict_select_kernel<16>, grid, block, 0, stream, a);
    } else if (longest <= 32 * kSelThreads) {
        hipLaunchKernelGGL(evict_select_kernel<32>, grid, block, 0, stream, a);
    } else if (longest <= 64 * kSelThreads) {
        hipLaunchKernelGGL(evict_select_kernel<64>, grid, block, 0, stream, a);
    } else {
        hipLaunchKernelGGL(evict_select_kernel<0>, grid, block, 0, stream, a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !longest) return e;
    // four pieces of a row per workgroup, two where that leaves CUs idle (8192 of 65536 fp32 positions
    // kept: 43 us, 49 with four, 60 with one)
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
