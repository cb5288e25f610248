// qr_chunk_f32.hpp -- causal multi-query attention in fp32 arithmetic on fp32 MFMA tiles, gfx950: the
// workgroup's part, shared by the calls over one sequence's chunk (qr_chunk_f32.hip, where the
// layouts and measurements stand) and over chunks of several sequences (qr_chunks_f32.hip).
#pragma once

#include "qr_batch.hpp"
#include "qr_mfma.hpp"

namespace qr {
namespace {

constexpr int kTP = 32;               // positions per tile

struct ChunkF32K {
    const char* pool;
    const int* page_table;   // row of (sequence, layer)
    long long page_elems;
    long long plane_elems;
    int heads;
    int group;
    int pos0;
    int nq;
    int q_dtype;
    const void* q;           // [nq][heads][D]
    float* out;              // [nq][heads][D]
    float* part_acc;         // [nq*heads][splits][D]
    float2* part_ml;         // [nq*heads][splits]
    float qscale;            // scale * log2(e)
    int queries_per_block;
    int splits;
    int qblocks;
    int units;               // splits x qblocks x kv_heads
    int per_xcd;             // launch slots per XCD: ceil(units / 8)
    // chunks of several sequences:
    int out_dtype;           // of out, which is then no float array unless F32
    float2* row_ml;          // [nq*heads] (maximum, sum), may be null
    float* scores;           // [nq*heads][score_len] scaled scores, may be null
    int score_len;
    int stride;              // partials of a row, splits or more
    PageGeom geom;
    int dtype;               // cache
};

template <typename ST, int D>
struct F32Geom {
    static constexpr int EPC = Chunk<ST>::kElems;        // cache elements per 16-byte chunk
    static constexpr int ESZ = 16 / EPC;
    static constexpr int RB = D * ESZ;                   // bytes of a row
    static constexpr int NCH = RB / 16;                  // chunks of a row
    static constexpr int SW = NCH % 8 == 0 ? 7 : 3;      // swizzle mask (a row is whole groups of SW + 1)
    static constexpr int NJ = NCH / 4;                   // QK steps (4 chunks)
    static constexpr int KB = kTP * RB;                  // bytes of a K (or V) tile
    static constexpr int NI = KB / 1024;                 // DMA loads of a K (or V) tile
    static constexpr int NIW = (NI + 3) / 4;             // of one wave
    static constexpr int PE = D % 64 == 0 ? 4 : 2;       // dims per lane and PV read
    static constexpr int NG = D / (16 * PE);             // PV reads of a row
    static_assert(NCH % 4 == 0 && KB % 1024 == 0 && D % (16 * PE) == 0, "whole steps");
    // resident workgroups per CU (one wave per SIMD each): the LDS of two stages of K and V, and
    // about 60 + D registers a lane
    // (head_dim 256: more than 256 with two M tiles, so 16-bit pages prefer position halves)
    static constexpr int kByLds = 160 * 1024 / (4 * KB);
    static constexpr int by_regs(int pg) { return D <= 64 ? 4 : D <= 128 ? 3 : pg; }
    static constexpr int wg_per_cu(int pg) { return kByLds < by_regs(pg) ? kByLds : by_regs(pg); }
};

// q elements 4 EPC j + EPC q4 + e of the row at `row`, scaled.  Element loads: the caller's q
// needs only element alignment; the dtype branch sits outside the loads.
template <int NJ, int EPC>
__device__ __forceinline__ void load_q(const void* q, int dtype, size_t row, int q4, float scale, float (&x)[NJ][EPC]) {
    if (dtype == QR_DTYPE_F32) {
        const float* f = static_cast<const float*>(q) + row;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < EPC; ++e) x[j][e] = f[4 * EPC * j + EPC * q4 + e];
    } else {
        const uint16_t* h = static_cast<const uint16_t*>(q) + row;
        const bool bf = dtype == QR_DTYPE_BF16;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int e = 0; e < EPC; ++e) {
                const uint16_t u = h[4 * EPC * j + EPC * q4 + e];
                x[j][e] = bf ? bf16_bits_to_f32(u) : f16_bits_to_f32(u);
            }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < EPC; ++e) x[j][e] *= scale;
}

// N = 2 or 4 cache elements at p (LDS): the raw words, and widened to fp32
template <typename ST, int N> struct Elems {
    static constexpr int kWords = std::is_same<ST, float>::value ? N : N / 2;
    typedef uint32_t type __attribute__((ext_vector_type(kWords)));
    __device__ static __forceinline__ type read(const char* p) { return *reinterpret_cast<const type*>(p); }
    // a pair with the elements that are not kept cleared
    __device__ static __forceinline__ type keep(type w, bool k0, bool k1) {
        if constexpr (std::is_same<ST, float>::value) {
            if (!k0) w[0] = 0;
            if (!k1) w[1] = 0;
        } else {
            w[0] &= (k0 ? 0xFFFFu : 0u) | (k1 ? 0xFFFF0000u : 0u);
        }
        return w;
    }
    __device__ static __forceinline__ void widen(const type w, float (&o)[N]) {
        if constexpr (std::is_same<ST, float>::value) {
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const uint32_t u = w[i];
                if constexpr (std::is_same<ST, BF16Tag>::value) {
                    o[2 * i] = __uint_as_float(u << 16);
                    o[2 * i + 1] = __uint_as_float(u & 0xFFFF0000u);
                } else {
                    o[2 * i] = f16_bits_to_f32(static_cast<uint16_t>(u & 0xFFFFu));
                    o[2 * i + 1] = f16_bits_to_f32(static_cast<uint16_t>(u >> 16));
                }
            }
        }
    }
};

// Sum of 1, 2 or 4 chains, pairwise.
template <int N> __device__ __forceinline__ f32x4_t chain_sum(const f32x4_t (&c)[N]) {
    if constexpr (N == 1) return c[0];
    else if constexpr (N == 2) return c[0] + c[1];
    else return (c[0] + c[1]) + (c[2] + c[3]);
}

// One split of one query block of one kv head, by a workgroup of four waves.  BATCH: a chunk of a
// call over several sequences, which has more outputs (ChunkF32K's last members).
template <typename ST, int D, int PG, bool BATCH>
__device__ __forceinline__ void chunk_f32_tiles(const ChunkF32K& p, int split, int qblk, int kvh,
                                                char (&lds)[2][2 * F32Geom<ST, D>::KB]) {
    using Gm = F32Geom<ST, D>;
    using El = Elems<ST, Gm::PE>;
    constexpr int EPC = Gm::EPC, RB = Gm::RB, NCH = Gm::NCH, SW = Gm::SW, NJ = Gm::NJ, KB = Gm::KB;
    constexpr int PE = Gm::PE, NG = Gm::NG;
    constexpr int NMT = kTP / 16 / PG;       // 16-position M tiles per wave and tile
    constexpr int RG = 4 / PG;               // row groups of 16 rows
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int rw = wave % RG;
    const int ph = wave / RG;                // position half (PG = 2)
    const int q4 = lane >> 4;
    const int l16 = lane & 15;

    const int q_first = qblk * p.queries_per_block;
    const int q_last = min(p.nq, q_first + p.queries_per_block) - 1;
    const int rho = rw * 16 + l16;
    const int row_q = q_first + rho / p.group;
    const int row_h = kvh * p.group + rho % p.group;
    const bool row_on = row_q <= q_last;
    // the block's own keys spread evenly over the splits, in whole tiles
    const int keys = p.pos0 + q_last + 1;
    const int tiles = (keys + kTP - 1) / kTP;
    const int tile0 = static_cast<int>(static_cast<long long>(tiles) * split / p.splits);
    const int ntiles = static_cast<int>(static_cast<long long>(tiles) * (split + 1) / p.splits) - tile0;
    const int unmasked_end = p.pos0 + q_first + 1;  // positions below it are seen by every row

    // ---- DMA of a tile: rows past the last key lie outside the buffer range and read as zeros
    const long long kblk = static_cast<long long>(kvh) * kPageTokens * D;
    uint32_t voff[Gm::NIW];
#pragma unroll
    for (int i = 0; i < Gm::NIW; ++i) {
        const int n = 64 * (wave + 4 * i) + lane;  // LDS chunk of the tile
        const int r = n / NCH, c = n - r * NCH;
        voff[i] = static_cast<uint32_t>(r * RB + 16 * (c ^ (r & SW)));
    }
    auto page_entry = [&](int it) {  // a scalar load: no kernel writes the table while this one runs
        return reinterpret_cast<const __attribute__((address_space(4))) int*>(
            reinterpret_cast<uintptr_t>(p.page_table))[((tile0 + it) * kTP) >> kPageShift];
    };
    auto dma = [&](int it, int phys_entry) {
        const int t0 = (tile0 + it) * kTP;
        const long long phys = phys_entry;
        char* dst = lds[it & 1];
        const char* kbase =
            p.pool + (phys * p.page_elems + kblk + static_cast<long long>(t0 & (kPageTokens - 1)) * D) * Gm::ESZ;
        const int bytes = min(kTP, keys - t0) * RB;
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kbase), 0, bytes, kBufferFlags);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<char*>(kbase + p.plane_elems * Gm::ESZ), 0, bytes, kBufferFlags);
#pragma unroll
        for (int i = 0; i < Gm::NIW; ++i)
            if (Gm::NI % 4 == 0 || wave + 4 * i < Gm::NI) {
                buffer_load_lds16(rk, dst + 1024 * (wave + 4 * i), voff[i], 0);
                buffer_load_lds16(rv, dst + KB + 1024 * (wave + 4 * i), voff[i], 0);
            }
    };
    if (ntiles > 0) dma(0, page_entry(0));
    int phys_pf = ntiles > 1 ? page_entry(1) : 0;

    float qv[NJ][EPC];
    load_q<NJ, EPC>(p.q, p.q_dtype, (static_cast<size_t>(row_on ? row_q : q_first) * p.heads + row_h) * D, q4, p.qscale, qv);

    f32x4_t acc[NG][PE];
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < PE; ++e) acc[g][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int row_lim = p.pos0 + min(row_q, q_last);  // last position the row sees
    // QK reads: chunk 4j + q4 of row l16 of an M tile at kx[j & 1] + 128 (j >> 1)
    const int half0 = ph * NMT * 16;  // first position of this wave in a tile
    int kx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) kx[i] = (half0 + l16) * RB + 16 * ((4 * i + q4) ^ (l16 & SW));
    // PV reads: PE dims from 16 PE g + PE l16 of row 4q4 + r at vx[r] + 16 PE ESZ g
    int vx[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = half0 + 4 * q4 + r, b = l16 * PE * Gm::ESZ;
        vx[r] = KB + row * RB + 16 * ((b >> 4) ^ (row & SW)) + (b & 15);
    }

    for (int it = 0; it < ntiles; ++it) {
        const int t0 = (tile0 + it) * kTP;
        wait_dma();     // this wave's part of tile `it` has landed
        lds_barrier();  // everyone's has, and the stage refilled next was consumed
        if (it + 1 < ntiles) {
            dma(it + 1, phys_pf);
            if (it + 2 < ntiles) phys_pf = page_entry(it + 2);
        }
        const char* const base = lds[it & 1];

        // ---- scores: the K chunks of step jj + 1 are read before the MFMAs of step jj, whose
        // partial sums are added during step jj + 1
        f32x4_t sc[NMT];
        {
            constexpr int NC = EPC / 2;  // chains of two MFMAs
            U32x4 raw[2][NMT];
            f32x4_t part[2][NMT][NC], sum[2][NMT];
            auto add = [&](int jj) __attribute__((always_inline)) {  // step jj's chains to the sum of its parity
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt) {
                    const f32x4_t s = chain_sum<NC>(part[jj & 1][mt]);
                    sum[jj & 1][mt] = jj < 2 ? s : sum[jj & 1][mt] + s;
                }
            };
            auto kread = [&](int jj) __attribute__((always_inline)) {
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt) raw[jj & 1][mt] = load16(base + kx[jj & 1] + 128 * (jj >> 1) + 16 * mt * RB);
            };
            kread(0);
#pragma unroll
            for (int jj = 0; jj < NJ; ++jj) {
                if (jj + 1 < NJ) kread(jj + 1);
                __builtin_amdgcn_sched_barrier(0);
                float kv[NMT][EPC];
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt) {
                    Chunk<ST>::widen(raw[jj & 1][mt], kv[mt]);
#pragma unroll
                    for (int c = 0; c < NC; ++c) part[jj & 1][mt][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int e = 0; e < EPC; ++e) {
                    if (jj > 0 && e == EPC / 2) {
                        __builtin_amdgcn_sched_barrier(0);
                        add(jj - 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int mt = 0; mt < NMT; ++mt)
                        part[jj & 1][mt][e % NC] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(kv[mt][e], qv[jj][e], part[jj & 1][mt][e % NC], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            add(NJ - 1);
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt) sc[mt] = sum[0][mt] + sum[1][mt];
        }

        // ---- causal mask, only on tiles that reach past the block's first query (the keys'
        // end lies past every row's own limit)
        const bool edge = t0 + kTP > unmasked_end;
        bool bad = false;  // a V element of an edge tile is not finite
        if (edge) {
#pragma unroll
            for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    sc[mt][r] = t0 + half0 + 16 * mt + 4 * q4 + r <= row_lim ? sc[mt][r] : -INFINITY;
            // the whole tile, so that every wave finds the same; V times zero is zero or NaN
            float z = 0.f;
#pragma unroll 4
            for (int i = 0; i < kTP * NCH / 64; ++i) {
                float v[EPC];
                Chunk<ST>::widen(load16(base + KB + 16 * (lane + 64 * i)), v);
#pragma unroll
                for (int e = 0; e < EPC; ++e) z = fmaf(v[e], 0.f, z);
            }
            bad = __builtin_amdgcn_ballot_w64(!(z == 0.f)) != 0;
        }

        if constexpr (BATCH) {
            if (p.scores && row_on) {  // for the weights; a row of scores is whole runs of 8
                float* const s = p.scores + (static_cast<long long>(row_q) * p.heads + row_h) * p.score_len + t0 + half0 + 4 * q4;
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt)
                    if (t0 + half0 + 16 * mt + 4 * q4 < keys) *reinterpret_cast<f32x4_t*>(s + 16 * mt) = sc[mt];
            }
        }

        // ---- online softmax.  The maximum does not lag, so that P <= 1 as in the decode kernels: a V
        // of more than 2^120 would overflow under P <= 256.
        float tm = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) tm = fmaxf(tm, sc[mt][r]);
        tm = max_xor32(max_xor16(tm));
        const bool grow = tm > m;
        const bool rescale = grow && m != -INFINITY;
        if (__builtin_amdgcn_ballot_w64(rescale)) {
            const float corr = rescale ? fast_exp2(m - tm) : 1.f;
            l *= corr;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < PE; ++e) acc[g][e] *= corr;
        }
        if (grow) m = tm;
        const float mref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[mt][r] = fast_exp2(sc[mt][r] - mref);
        f32x4_t ls = sc[0];
#pragma unroll
        for (int mt = 1; mt < NMT; ++mt) ls += sc[mt];
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);

        if (bad) {
            // A row must not meet the V of a position that it does not see: 0 x inf is NaN.  The
            // elements that are not finite are added here, only where the row sees their position
            // (rare), and cleared for the products below.
#pragma unroll 1
            for (int k = 0; k < NMT * 16; ++k) {  // position 16 (k / 16) + 4 ((k / 4) % 4) + k % 4
                const int pos = half0 + k;
                float own = 0.f;
#pragma unroll
                for (int mt = 0; mt < NMT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) own = (k >> 4) == mt && (k & 3) == r ? sc[mt][r] : own;
                const float w = __shfl(own, 16 * ((k >> 2) & 3) + l16, 64);
                const bool see = t0 + pos <= row_lim;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr) {
                        const int b = (16 * g + 4 * q4 + rr) * PE * Gm::ESZ;
                        float v[PE];
                        El::widen(El::read(base + KB + pos * RB + 16 * ((b >> 4) ^ (pos & SW)) + (b & 15)), v);
#pragma unroll
                        for (int e = 0; e < PE; ++e)
                            if (see && !(fabsf(v[e]) < INFINITY)) acc[g][e][rr] = fmaf(w, v[e], acc[g][e][rr]);
                        asm volatile("" ::: "memory");  // no registers for all reads at once
                    }
                }
            }
            lds_barrier();  // every wave has read them
            for (int c = threadIdx.x; c < kTP * NCH; c += 256) {
                typedef typename Elems<ST, 2>::type Pair;
#pragma unroll
                for (int i = 0; i < EPC / 2; ++i) {
                    Pair* const w = reinterpret_cast<Pair*>(const_cast<char*>(base) + KB + 16 * c) + i;
                    float v[2];
                    Elems<ST, 2>::widen(*w, v);
                    const bool b0 = !(fabsf(v[0]) < INFINITY), b1 = !(fabsf(v[1]) < INFINITY);
                    if (b0 || b1) *w = Elems<ST, 2>::keep(*w, !b0, !b1);
                }
            }
            lds_barrier();
        }

        // ---- weighted sum of V (step st = 4 mt + r of dim group g; V read two steps ahead)
        constexpr int CL = D == 256 && EPC == 8 ? 4 : 2;  // steps of a chain
        constexpr int NS = 4 * NMT, NC = NS / CL, NO = NC + 1;
        typename El::type vb[3];
        auto vread = [&](int i) __attribute__((always_inline)) {
            const int g = i / NS, st = i % NS;
            vb[i % 3] = El::read(base + vx[st & 3] + 16 * (st >> 2) * RB + 16 * PE * Gm::ESZ * g);
        };
        vread(0);
        vread(1);
        f32x4_t o[NO][PE];  // chain c of group g in o[(NC g + c) % NO]: the next group's first chain leaves g's alone
        auto add = [&](int g) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < PE; ++e) {
                f32x4_t s[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) s[c] = o[(NC * g + c) % NO][e];
                acc[g][e] += chain_sum<NC>(s);
            }
        };
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                const int i = NS * g + st, c = i / CL % NO;
                if (st % CL == 0) {
#pragma unroll
                    for (int e = 0; e < PE; ++e) o[c][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                }
                if (i + 2 < NS * NG) vread(i + 2);
                __builtin_amdgcn_sched_barrier(0);
                float v[PE];
                El::widen(vb[i % 3], v);
#pragma unroll
                for (int e = 0; e < PE; ++e)
                    o[c][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], sc[st >> 2][st & 3], o[c][e], 0, 0, 0);
                if (g > 0 && st == 1) add(g - 1);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        add(NG - 1);
    }
    l = sum_xor32(sum_xor16(l));

    if constexpr (PG == 2) {
        // the upper halves hand (m, l, o) to the lower ones through LDS
        constexpr int NA = NG * PE;
        static_assert(RG * 64 * (NA * 16 + 8) <= 4 * KB, "the handed-over rows fit the tile buffers");
        f32x4_t* xo = reinterpret_cast<f32x4_t*>(lds[0]) + rw * NA * 64 + lane;
        float2* xm = reinterpret_cast<float2*>(lds[0] + RG * NA * 64 * 16) + rw * 64 + lane;
        __syncthreads();
        if (ph == 1) {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < PE; ++e) xo[(g * PE + e) * 64] = acc[g][e];
            *xm = make_float2(m, l);
        }
        __syncthreads();
        if (ph == 1) return;
        const float2 o = *xm;
        const float M = fmaxf(m, o.x);
        const float c0 = m == -INFINITY ? 0.f : fast_exp2(m - M);
        const float c1 = o.x == -INFINITY ? 0.f : fast_exp2(o.x - M);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < PE; ++e) acc[g][e] = acc[g][e] * c0 + xo[(g * PE + e) * 64] * c1;
        l = l * c0 + o.y * c1;
        m = M;
    }

    // lane (q4, l16) holds dims 16 PE g + PE (4q4 + r) + e of row l16 in acc[g][e][r]
    if constexpr (BATCH) {
        // A sum that is no number though the weights are: an infinite V of a weight that rounds to zero.  It is that
        // infinity, unless the row sees a NaN or both; one pass over the unit's values, a dim per lane.
        bool bad = false;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < PE; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) bad |= !(acc[g][e][r] == acc[g][e][r]);
        bad = bad && row_on && l == l;
        if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll 1
            for (int k = 0; k < (D + 63) / 64; ++k) {
                const NotFinite f = find_not_finite(p.pool, p.page_table, p.geom, p.dtype, kvh, min(64 * k + lane, D - 1), tile0 * kTP,
                                                    min((tile0 + ntiles) * kTP, keys));
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (16 * PE * g / 64 != k) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int e = 0; e < PE; ++e) {
                            const NotFinite o = f.of_lane(16 * PE * g % 64 + PE * (4 * q4 + r) + e);
                            const float x = acc[g][e][r];
                            acc[g][e][r] = bad && !(x == x) ? o.settle(row_lim + 1, x) : x;
                        }
                }
            }
        }
    }
    if (!row_on) return;
    const size_t r0 = static_cast<size_t>(row_q) * p.heads + row_h;
    const size_t slot = r0 * (BATCH ? p.stride : p.splits) + split;
    if constexpr (BATCH) {
        if (p.row_ml && p.splits == 1 && q4 == 0) p.row_ml[r0] = make_float2(m, l);
        if (p.splits == 1 && p.out_dtype != QR_DTYPE_F32) {
            uint16_t* o = reinterpret_cast<uint16_t*>(p.out) + r0 * D + 4 * PE * q4;
            const float inv = 1.f / l;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    uint16_t b[PE];
#pragma unroll
                    for (int e = 0; e < PE; ++e) b[e] = f32_to_out16(acc[g][e][r] * inv, p.out_dtype);
                    __builtin_memcpy(o + 16 * PE * g + PE * r, b, sizeof b);
                }
            return;
        }
    }
    const float by = p.splits == 1 ? 1.f / l : 1.f;
    float* o = (p.splits == 1 ? p.out + r0 * D : p.part_acc + slot * D) + 4 * PE * q4;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < PE; ++e) {
                const float a = acc[g][e][r];
                float x = a * by;
                if (p.splits == 1 && fabsf(x) < INFINITY) x = fmaf(fmaf(-x, l, a), by, x);  // a / l to the last bit or so
                o[16 * PE * g + PE * r + e] = x;
            }
    if (p.splits > 1 && q4 == 0) p.part_ml[slot] = make_float2(m, l);
}

}  // namespace
}  // namespace qr
