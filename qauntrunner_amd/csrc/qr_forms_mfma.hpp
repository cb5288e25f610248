// qr_forms_mfma.hpp -- attention in its other forms and behind shared prefixes on 32x32x16 MFMA tiles: caches of 16 and 8
// bits, head sizes 64 and 128 (operand page layouts, qr_kernels.hpp), whole groups of query heads, gfx950.
//
// A row is one (query, query head) pair of a kv head; a wave owns 32 rows:
//   QK  S^T[position][row] = K . q^T    (A = K, B = q)
//   PV  O^T[dim][row]     += V^T . P^T  (A = V, B = P)
// v_mfma_f32_32x32x16: A[m = lane % 32][k = 8 (lane / 32) + i], B[k = 8 (lane / 32) + i][n = lane % 32],
// D[m = 8 (r / 4) + 4 (lane / 32) + r % 4][n = lane % 32].  A row's scores lie in two lanes, l and l ^ 32.  Which position of a
// step of 32 an A row m stands for is chosen so that a lane's scores r are its k-slots of the PV steps, in order:
//   16 bits: m = 16 s + 8 a + 4 h + b is position 16 s + 8 h + 4 a + b, score r = 8 s + i position 16 s + 8 (lane / 32) + i;
//   8 bits:  m = 16 s + 8 a + 4 h + b is position 16 h + 8 s + 4 a + b, score r position 16 (lane / 32) + r, so that a lane's
//            operands of both PV steps are 16 bytes of the page.
//
// 8 bits: codes become bf16 exactly.  K's scale is one number per lane there (a lane holds dims of one position), a factor
// of the conversion; V's scale differs between a lane's positions and goes into the weights, after their sum.
//
// Scores in log2 units: z = s sscale, capped, less the slope; weights 2^(z - m) of at most 2^kTop, m moved (and the
// accumulators rescaled) only when a score passes m + kTop, and then to leave kHead log2 units to the next move.  bf16
// weights stay at or below 1; fp16, with few exponents below 1, takes them up to 2^15.  Sums are of the fp32 weights.
// Queries and weights of a type with more bits than the tile's enter as PARTS of it: bf16 three (24 bits), fp16 two (22).
#pragma once

#include <cmath>

#include "qr_forms.hpp"
#include "qr_mfma.hpp"
#include "qr_quant.hpp"

namespace qr {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16_t mfma32(f16x8_t a, f16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// (fmaxf's quieting of NaNs, one more v_max each, is not needed: a NaN score reaches its row through its weight.  The
// compiler does not count the wait states between an MFMA and an asm that reads its result: mfma_done stands between.)
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ float max3abs(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, |%1|, |%2|, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ void mfma_done(f32x16_t (&s)[1]) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s[0])); }
__device__ __forceinline__ void mfma_done(f32x16_t (&s)[2]) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s[0]), "+v"(s[1])); }

template <int CT> struct FormElem {
    static constexpr bool BF16 = CT != QR_DTYPE_F16;
    using T = typename std::conditional<BF16, __bf16, _Float16>::type;
    typedef T vec8 __attribute__((ext_vector_type(8)));
};

// 8 codes times `scale`.
__device__ __forceinline__ bf16x8_t widen8(uint32_t lo, uint32_t hi, float scale) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Copies into LDS by buffer loads, 16 bytes per lane to `to` + 16 lane; past the source's bytes zeros.  As asm: behind a
// load that the compiler knows to write LDS it waits for memory before the next read of LDS, whichever bytes that reads, and
// the tiles ahead would be awaited in every turn (three quarters of the time of a tile).  Nothing is written to registers;
// wait_vmcnt and a barrier stand between a copy and the reads of its bytes.  (s_nop: a scalar that a vector instruction wrote is
// read by a buffer load five wait states later at the earliest.)
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4_t dma_source(const char* base, int bytes) {
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    return u32x4_t{static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32) & 0xFFFFu, static_cast<uint32_t>(bytes), kBufferFlags};
}
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p)));
}
__device__ __forceinline__ void dma16(u32x4_t source, const char* to, uint32_t at, uint32_t from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 : : "s"(lds_address(to)), "v"(at), "s"(source), "s"(from) : "memory", "m0");
}
// One wave's 32 rows.
template <int CT, int D, int PARTS, int SCORES>
struct FormTile {
    static constexpr bool BF16 = FormElem<CT>::BF16, E8 = CT == QR_DTYPE_E4M3, SPLIT = PARTS > 1;
    using T = typename FormElem<CT>::T;
    using vec8 = typename FormElem<CT>::vec8;
    static constexpr int NK = D / 16;   // QK k-steps
    static constexpr int ND = D / 32;   // PV dim tiles
    static constexpr float kTop = BF16 ? 0.f : 15.f, kHead = SPLIT ? 0.f : 4.f;

    int lane, half;
    int row, head, chunk;  // of row lane % 32
    bool on;
    int lo, hi;            // slots that the row sees (none past the item's rows)
    int away;              // position less the item's base
    float slope;           // in log2 units
    vec8 q[PARTS][NK];
    float sscale;          // log2 units per score
    float m, l;            // l: this lane's half of the positions
    float cap[5], by[5];   // the capped score of a small s: s (cap[0] + cap[1] s^2 + ... + cap[4] s^8); what the tile takes
    float small;           // |s| up to which it is
    bool wide;             // the tile's scores are capped already
    f32x16_t acc[ND];

    __device__ __forceinline__ void init(const FormsK& p, const FormItem& it, int kvh, int g, int rho) {
        lane = threadIdx.x & 63;
        half = lane >> 5;
        const int r = rho + (lane & 31);
        on = r < it.rows * g;
        const int rr = on ? r : it.rows * g - 1;
        const int j = rr / g;
        head = kvh * g + rr - j * g;
        row = it.row0 + j;
        const FormSpan s = form_row(p, it, j);
        chunk = s.chunk;
        lo = s.lo;
        hi = on ? s.hi : -1;
        away = s.pos - it.base;
        slope = (SCORES == kScoresSlope || SCORES == kScoresBoth) && p.slopes ? p.slopes[head] * kLog2e : 0.f;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    }
    __device__ __forceinline__ FormRange range() const {
        const bool sees = lo <= hi;
        return {wave_min(sees ? lo : 0x7FFFFFFF), wave_max(sees ? hi : -1), wave_max(on ? lo : -1), wave_min(on ? hi : 0x7FFFFFFF)};
    }

    // Dims of this lane's part of k-step kk.  The sign of the scale goes into q: the maximum is taken before the scores are
    // scaled.
    __device__ __forceinline__ int dim0(int kk) const { return E8 ? 32 * (kk >> 1) + 16 * half + 8 * (kk & 1) : 16 * kk + 8 * half; }
    __device__ __forceinline__ void load_q(const FormsK& p) {
        const long long at = (static_cast<long long>(row) * p.heads + head) * D;
        const float sign = p.qscale == 0.f ? 0.f : p.qscale < 0.f ? -1.f : 1.f;
        sscale = p.qscale == 0.f ? 1.f : fabsf(p.qscale);
        float x[NK][8];
        if (p.act == QR_DTYPE_F32) {
            const float* f = static_cast<const float*>(p.q) + at;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) __builtin_memcpy(x[kk], f + dim0(kk), 32);
        } else {
            const uint16_t* h = static_cast<const uint16_t*>(p.q) + at;
            uint16_t u[NK][8];
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) __builtin_memcpy(u[kk], h + dim0(kk), 16);
            const bool bf = p.act == QR_DTYPE_BF16;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[kk][i] = bf ? bf16_bits_to_f32(u[kk][i]) : f16_bits_to_f32(u[kk][i]);
        }
        float by = sign;
        if (SPLIT && !BF16) {
            // fp16 parts: the row's largest value to 2^13 .. 2^14, a power of two that the score scale takes back
            float a = 0.f;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x[kk][i]));
            a = max_xor32(a);
            if (a > 1e-30f && a < 3e38f) {
                const int ex = ilogbf(a) - 13;
                by = ldexpf(sign, -ex);
                sscale = ldexpf(sscale, ex);
            }
        }
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = x[kk][i] * by;
#pragma unroll
                for (int c = 0; c < PARTS; ++c) {
                    q[c][kk][i] = static_cast<T>(v);
                    v -= static_cast<float>(q[c][kk][i]);
                }
            }
        init_cap(p);
    }

    // Position of score r within its step of 32.
    __device__ __forceinline__ int at(int r) const { return E8 ? 16 * half + r : 16 * (r >> 3) + 8 * half + (r & 7); }

    // Capped scores without slopes ascend with the products, so that the maximum is taken of these, and a product becomes its
    // capped score where it becomes a weight (PER_WEIGHT): 1 - 2 / (e^2x + 1) would be two more operations of a quarter of the rate
    // for each, but scores are mostly far below the cap, and tanh x / x on |x| <= 1/2 is a polynomial of x^2 (least squares at
    // Chebyshev's points, off by 3e-8; its last coefficient is positive).  Tiles with larger ones, at positions that a row does not
    // see and in other rows too, are capped in front, and the coefficients become those of s.  That quotient is off by up to 2^-22 of the
    // cap for small scores, so that larger caps take kScoresBoth, as where the coefficients would leave fp32's range (per_weight).
    static constexpr float kTanh[5] = {0.99999999f, -0.33333071f, 0.1332483f, -0.05298926f, 0.01714132f};
    static constexpr bool PER_WEIGHT = SCORES == kScoresCap && !SPLIT;
    // What stands for a score that the row does not see; a polynomial of it is a large negative number or -infinity.
    static constexpr float kHidden = PER_WEIGHT ? -1e18f : -INFINITY;
    __device__ __forceinline__ void init_cap(const FormsK& p) {
        if (!PER_WEIGHT) return;
        const float in = sscale / p.cap, i2 = in * in;
        cap[0] = p.cap * in * kTanh[0];
        cap[1] = p.cap * in * i2 * kTanh[1];
        cap[2] = p.cap * in * i2 * i2 * kTanh[2];
        cap[3] = p.cap * in * i2 * i2 * i2 * kTanh[3];
        cap[4] = p.cap * in * i2 * i2 * i2 * i2 * kTanh[4];
        small = 0.5f / in;
    }
    __device__ __forceinline__ float capped(float s, float add) const {
        const float x = s * s;
        return fmaf(s, fmaf(fmaf(fmaf(fmaf(by[4], x, by[3]), x, by[2]), x, by[1]), x, by[0]), add);
    }
    // NS steps' products, from step t0 on, as `form` leaves them.
    template <int NS>
    __device__ __forceinline__ void prepare(const FormsK& p, f32x16_t (&s)[NS], int t0, bool edge) {
        if (PER_WEIGHT) {
            mfma_done(s);
            float most = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; r += 2) most = max3abs(s[n][r], s[n][r + 1], most);
            wide = __builtin_amdgcn_ballot_w64(!(most <= small)) != 0;
#pragma unroll
            for (int i = 0; i < 5; ++i) by[i] = wide ? (i == 0 ? 1.f : 0.f) : cap[i];
            if (wide) {
                const float in = 2.f * kLog2e * sscale / p.cap;
#pragma unroll
                for (int n = 0; n < NS; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[n][r] = fmaf(-2.f * p.cap, __builtin_amdgcn_rcpf(fast_exp2(s[n][r] * in) + 1.f), p.cap);
            }
        }
#pragma unroll
        for (int n = 0; n < NS; ++n) form(p, s[n], t0 + 32 * n, edge);
    }

    // Scores of step t0 in log2 units (plain ones are scaled as they become weights, those PER_WEIGHT capped too), masked where
    // some row does not see the whole step: `edge`.
    __device__ __forceinline__ void form(const FormsK& p, f32x16_t& s, int t0, bool edge) const {
        if ((SCORES == kScoresCap && !PER_WEIGHT) || SCORES == kScoresBoth) {
            const float in = sscale / p.cap;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float t = s[r] * in, x = t * t;
                if (SPLIT) {
                    s[r] = p.cap * tanhf(t);
                } else {
                    // (the quotient loses a small tanh's bits: 2^-24 of the cap)
                    const float a = t * fmaf(fmaf(fmaf(fmaf(kTanh[4], x, kTanh[3]), x, kTanh[2]), x, kTanh[1]), x, kTanh[0]);
                    const float b = fmaf(-2.f, __builtin_amdgcn_rcpf(fast_exp2(t * (2.f * kLog2e)) + 1.f), 1.f);
                    s[r] = p.cap * (fabsf(t) <= 0.5f ? a : b);
                }
            }
        }
        if (SCORES == kScoresSlope || SCORES == kScoresBoth) {
            const float first = static_cast<float>(t0 + (E8 ? 16 : 8) * half - away);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float d = fabsf(first + static_cast<float>(E8 ? r : 16 * (r >> 3) + (r & 7)));
                s[r] = SCORES == kScoresBoth ? fmaf(-slope, d, s[r]) : fmaf(s[r], sscale, -slope * d);
            }
        }
        if (edge) {
            const int a = lo - t0 - (E8 ? 16 : 8) * half, b = hi - t0 - (E8 ? 16 : 8) * half;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int x = E8 ? r : 16 * (r >> 3) + (r & 7);
                if (x < a || x > b) s[r] = kHidden;
            }
        }
    }

    // The row's maximum with NS steps' scores; what was summed so far has to be weighed by the result.
    template <int NS>
    __device__ __forceinline__ float raise(f32x16_t (&s)[NS]) {
        mfma_done(s);
        float mx[2 * NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const float a = max3f(s[n][0], s[n][1], s[n][2]), b = max3f(s[n][3], s[n][4], s[n][5]);
            const float c = max3f(s[n][6], s[n][7], s[n][8]), d = max3f(s[n][9], s[n][10], s[n][11]);
            mx[2 * n] = max3f(s[n][12], s[n][13], s[n][14]);
            mx[2 * n] = max3f(mx[2 * n], s[n][15], a);
            mx[2 * n + 1] = max3f(b, c, d);
        }
        float t = mx[0];
#pragma unroll
        for (int n = 1; n < 2 * NS; ++n) t = fmaxf(t, mx[n]);
        t = max_xor32(t);
        if (PER_WEIGHT) t = t > 0.1f * kHidden ? capped(t, 0.f) : -INFINITY;
        const float by = SCORES == kScoresPlain ? sscale : 1.f;
        if (!(fmaf(t, by, -m) > kTop)) return 1.f;
        float mn = fmaf(t, by, kHead - kTop);
        if (fmaf(t, by, -mn) > kTop) {  // rounded down, where a step of m is that large
            const int b = __float_as_int(mn);
            mn = __int_as_float(b < 0 ? b - 1 : b + 1);
        }
        const float c = m == -INFINITY ? 1.f : fast_exp2(m - mn);  // (nothing was summed yet)
        m = mn;
        return c;
    }
    __device__ __forceinline__ void rescale(float c) {
        if (__builtin_amdgcn_ballot_w64(c != 1.f)) {
            l *= c;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= c;
        }
    }
    // What a weight is a power of 2 of.
    __device__ __forceinline__ float logit(float s, float ref) const {
        return SCORES == kScoresPlain ? fmaf(s, sscale, ref) : PER_WEIGHT ? capped(s, ref) : s + ref;
    }
    // Weights of NS steps' scores, as PV operands (8 bits: times V's scales); their sum.
    template <int NS, class F>
    __device__ __forceinline__ float weigh(const f32x16_t (&s)[NS], vec8 (&w)[PARTS][NS][2], F vscale) const {
        const float ref = m == -INFINITY ? 0.f : -m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = fast_exp2(logit(s[n][r], ref));
                sum[r & 3] += e;
                float v = E8 ? e * vscale(n, r) : e;
#pragma unroll
                for (int c = 0; c < PARTS; ++c) {
                    w[c][n][r >> 3][r & 7] = static_cast<T>(v);
                    v -= static_cast<float>(w[c][n][r >> 3][r & 7]);
                }
            }
        return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    template <int NS, class F>
    __device__ __forceinline__ void softmax(f32x16_t (&s)[NS], vec8 (&w)[PARTS][NS][2], F vscale) {
        rescale(raise(s));
        l += weigh(s, w, vscale);
    }

    // V's element of slot t and dim d of a step of the page (8 bits: without its scale).
    __device__ __forceinline__ static float v_value(const char* step, int t, int d) {
        if (E8) return quant_value<0>(static_cast<uint8_t>(step[1024 * (d >> 5) + 16 * (32 * (t >> 4) + (d & 31)) + (t & 15)]));
        return static_cast<float>(*reinterpret_cast<const T*>(step + 1024 * (d >> 4) + 16 * (16 * (t >> 3) + (d & 15)) + 2 * (t & 7)));
    }
    // A step that not every row sees whole may hold V elements that are not finite at slots some rows do not see, where 0 x inf
    // would reach them.  Adds them to the rows that see them as they are (no finite weight changes them); the caller clears
    // them in its operands.
    __device__ __forceinline__ void add_bad(const FormsK& p, const FormItem& it, int kvh, int t0) {
        constexpr int ES = E8 ? 1 : 2;
        const char* const step = p.pool + (static_cast<long long>(form_page(p, it.pt_off, t0)) * p.geom.page_elems() + p.geom.plane_elems() +
                                           static_cast<long long>(kvh) * kPageTokens * D + (t0 & (kPageTokens - 1)) * D) * ES;
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
            const bool sees = t0 + k >= lo && t0 + k <= hi;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float x = v_value(step, k, 32 * d + 8 * (r >> 2) + 4 * half + (r & 3));
                    if (!(fabsf(x) < INFINITY) && sees) acc[d][r] += x;
                    if ((r & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // no registers for all reads at once
                }
        }
    }

    // A sum that is no number while that of its weights is: an infinite V of little weight (0 x inf), or one between the parts of a
    // weight (inf - inf).  No weight of the formula is zero, so the row shows the sum of these elements.  Steps step0, step0 +
    // stride, ... below step1 were the wave's.  (8 bits hold no infinity.)
    __device__ __forceinline__ void settle(const FormsK& p, const FormItem& it, int kvh, int step0, int step1, int stride) {
        if (E8) return;
        f32x16_t all = acc[0];
#pragma unroll
        for (int d = 1; d < ND; ++d) all += acc[d];
        float sum[4] = {all[0], all[1], all[2], all[3]};
#pragma unroll
        for (int r = 4; r < 16; ++r) sum[r & 3] += all[r];
        const float s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (__builtin_expect(!__builtin_amdgcn_ballot_w64(s != s && l == l), 1)) return;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = acc[d][r] != acc[d][r] ? 0.f : acc[d][r];
#pragma unroll 1
        for (int st = step0; st < step1; st += stride) {
            const char* const step = p.pool + (static_cast<long long>(form_page(p, it.pt_off, 32 * st)) * p.geom.page_elems() + p.geom.plane_elems() +
                                               static_cast<long long>(kvh) * kPageTokens * D + (32 * st & (kPageTokens - 1)) * D) * 2;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const vec8 x = *reinterpret_cast<const vec8*>(step + 16 * (lane + 64 * i));
#pragma unroll
                for (int j = 0; j < 8; ++j) bad |= !(fabsf(static_cast<float>(x[j])) < INFINITY);
            }
            if (__builtin_amdgcn_ballot_w64(bad)) add_bad(p, it, kvh, 32 * st);
        }
    }

    // The row's output or partial: N groups of 4 dims from group g0 on, of the weighed sums a.  Group g holds dims 32 (g / 4) +
    // 8 (g % 4) + 4 half .. + 3.
    __device__ __forceinline__ long long slot(const FormsK& p, const FormItem& it, int split) const {
        const FormRows& c = p.c[chunk];
        return c.slot0 + (static_cast<long long>(row - c.row0) * p.heads + head) * c.parts + it.part0 + split;
    }
    template <int N>
    __device__ __forceinline__ void store(const FormsK& p, const FormItem& it, const FormUnit& u, int g0, float lsum, const f32x4_t (&a)[N]) const {
        if (!on) return;
        auto dim = [&](int i) { return 32 * ((g0 + i) >> 2) + 8 * ((g0 + i) & 3) + 4 * half; };
        if (!form_whole(p.c[chunk], it, u.parts)) {
            float* o = p.part_acc + slot(p, it, u.part) * D;
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<f32x4_t*>(o + dim(i)) = a[i];
            return;
        }
        const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
        const long long at = (static_cast<long long>(row) * p.heads + head) * D;
        if (p.act == QR_DTYPE_BF16) store16<__bf16>(static_cast<uint16_t*>(p.out) + at, inv, a, dim);
        else if (p.act == QR_DTYPE_F16) store16<_Float16>(static_cast<uint16_t*>(p.out) + at, inv, a, dim);
        else {
            float* o = static_cast<float*>(p.out) + at;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const f32x4_t x = a[i] * inv;
                __builtin_memcpy(o + dim(i), &x, 16);
            }
        }
    }
    // one store per group, element-aligned
    template <class O, int N, class G>
    __device__ static __forceinline__ void store16(uint16_t* o, float inv, const f32x4_t (&a)[N], G dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const f32x4_t x = a[i] * inv;
            O b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = static_cast<O>(x[j]);
            __builtin_memcpy(o + dim(i), b, 8);
        }
    }
    __device__ __forceinline__ void store_ml(const FormsK& p, const FormItem& it, const FormUnit& u, float mm, float lsum) const {
        if (on && !half) form_store_ml(p, p.c[chunk], it, slot(p, it, u.part), u, mm, lsum);
    }
};

// The PW waves of a row group merge: each adds up its share of the dim groups.  (Afterwards lds and rest may be used again only behind
// a barrier.)
template <class F, int RW, int PW>
__device__ __forceinline__ void merge_waves(const FormsK& p, const FormItem& it, const FormUnit& un, F& w, int rw, int pw, char* lds, char* rest) {
    constexpr int NG = 4 * F::ND, NP = NG / PW;  // f32x4 groups of a row in a lane; of them a wave's
    f32x4_t out[NP];
    float M = w.m, L = w.l;
    if constexpr (PW == 1) {
#pragma unroll
        for (int i = 0; i < NG; ++i) out[i] = f32x4_t{w.acc[i >> 2][4 * (i & 3)], w.acc[i >> 2][4 * (i & 3) + 1], w.acc[i >> 2][4 * (i & 3) + 2], w.acc[i >> 2][4 * (i & 3) + 3]};
    } else {
        f32x4_t* const xa = reinterpret_cast<f32x4_t*>(lds);  // [row group][wave][NG][64]
        float2* const xm = reinterpret_cast<float2*>(rest);   // [row group][wave][64]
        wait_dma();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NG; ++i)
            xa[((rw * PW + pw) * NG + i) * 64 + w.lane] = f32x4_t{w.acc[i >> 2][4 * (i & 3)], w.acc[i >> 2][4 * (i & 3) + 1], w.acc[i >> 2][4 * (i & 3) + 2], w.acc[i >> 2][4 * (i & 3) + 3]};
        xm[(rw * PW + pw) * 64 + w.lane] = make_float2(w.m, w.l);
        __syncthreads();
        float c[PW];
        M = -INFINITY;
        L = 0.f;
#pragma unroll
        for (int x = 0; x < PW; ++x) M = fmaxf(M, xm[(rw * PW + x) * 64 + w.lane].x);
#pragma unroll
        for (int x = 0; x < PW; ++x) {
            const float2 ml = xm[(rw * PW + x) * 64 + w.lane];
            c[x] = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - M);
            L = fmaf(ml.y, c[x], L);
        }
        f32x4_t all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            out[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < PW; ++x) out[i] += xa[((rw * PW + x) * NG + pw * NP + i) * 64 + w.lane] * c[x];
            all += out[i];
        }
        const float sum = (all[0] + all[1]) + (all[2] + all[3]);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum != sum && L == L) != 0, 0)) {  // (form_weighed throughout: 2 us of 33)
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                out[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < PW; ++x) out[i] += form_weighed(xa[((rw * PW + x) * NG + pw * NP + i) * 64 + w.lane], c[x]);
            }
        }
    }
    w.store(p, it, un, pw * NP, L, out);
    if (pw == 0) w.store_ml(p, it, un, M, L);
}

// ------------------------------------------------------------------ few rows: HBM-bound
// Up to 32 rows; four waves take every fourth step of 32 slots, their operands straight from the page into registers (K of the
// next step while this one's softmax runs, V while the next one's scores are computed), and merge at the end.  No wave waits
// for another before that.  Bound by HBM: 16 sequences of 130 to 16000 positions, 8 kv heads of 128: 8 bits 25 to 27 us for 120 MB, 4.4
// to 4.8 TB/s; fp16 with capped scores and a window of 4096 24 to 27 us for 131 MB (a large copy: 4.8 to 5.1 TB/s).
template <int CT, int D> struct FormStep {  // one step's operands
    using E = FormElem<CT>;
    static constexpr bool E8 = CT == QR_DTYPE_E4M3;
    static constexpr int N = E8 ? D / 32 : D / 16;  // 16-byte loads of K and of V
    uint4 k[N], v[N];
    uint4 vs;            // 8 bits: scale bytes of V at the lane's 16 positions
    uint32_t ks;         // and of K at its own
};

template <int CT, int D, int PARTS, int SCORES>
__device__ __forceinline__ void forms_stream(const FormsK& p, const FormItem& it, int u, char* lds, char* rest) {
    using F = FormTile<CT, D, PARTS, SCORES>;
    using vec8 = typename F::vec8;
    constexpr bool E8 = F::E8;
    constexpr int ROWS = form_rows(kFormStream), TILE = form_tile(kFormStream);
    static_assert(ROWS == 32 && TILE == 32, "a wave's rows and steps");
    constexpr int ES = E8 ? 1 : 2;
    const int kv = p.geom.kv_heads, g = p.heads / kv;
    const FormUnit un = form_unit(p, it, g, ROWS, TILE, u);
    const int kvh = un.kvh, split = un.part, block = un.block;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    F w;
    w.init(p, it, kvh, g, 32 * block);
    const FormRange range = w.range();
    const int step0 = range.lo >> 5, steps = range.lo > range.hi ? 0 : (range.hi >> 5) - step0 + 1;
    const int s0 = __builtin_amdgcn_readfirstlane(step0 + static_cast<int>(static_cast<long long>(steps) * split / un.parts));
    const int s1 = __builtin_amdgcn_readfirstlane(step0 + static_cast<int>(static_cast<long long>(steps) * (split + 1) / un.parts));

    const long long page_bytes = p.geom.page_elems() * ES, plane_bytes = p.geom.plane_elems() * ES;
    const long long head_bytes = static_cast<long long>(kvh) * kPageTokens * D * ES;
    const int m_ = w.lane & 31, sx = m_ >> 4, ax = (m_ >> 3) & 1, hx = (m_ >> 2) & 1, bx = m_ & 3;
    // this lane's part of the operands of a step
    const int ko = E8 ? 16 * w.lane : 1024 * ax * (D / 32) + 16 * (16 * w.half + 4 * (2 * sx + hx) + bx);
    const int vo = E8 ? 16 * w.lane : 1024 * (m_ >> 4) + 16 * (16 * w.half + (w.lane & 15));
    FormStep<CT, D> o;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    auto get = [](const char* a) __attribute__((always_inline)) {
        const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a));
        return make_uint4(x[0], x[1], x[2], x[3]);
    };
    auto load_k = [&](int st, int phys) __attribute__((always_inline)) {
        const char* page = p.pool + static_cast<long long>(phys) * page_bytes;
        const char* k = page + head_bytes + static_cast<long long>(st & 7) * 32 * D * ES;
#pragma unroll
        for (int i = 0; i < FormStep<CT, D>::N; ++i) o.k[i] = get(k + ko + (E8 ? 1024 : 512) * i);
        if (E8) o.ks = static_cast<uint8_t>(page[2 * plane_bytes + kvh * kPageTokens + 32 * (st & 7) + 16 * hx + 8 * sx + 4 * ax + bx]);
    };
    auto load_v = [&](int st, int phys) __attribute__((always_inline)) {
        const char* page = p.pool + static_cast<long long>(phys) * page_bytes;
        const char* v = page + plane_bytes + head_bytes + static_cast<long long>(st & 7) * 32 * D * ES;
#pragma unroll
        for (int i = 0; i < FormStep<CT, D>::N; ++i) o.v[i] = get(v + vo + (E8 ? 1024 * i : 2048 * (i % F::ND) + 512 * (i / F::ND)));
        if (E8) o.vs = *reinterpret_cast<const uint4*>(page + 2 * plane_bytes + (kv + kvh) * kPageTokens + 32 * (st & 7) + 16 * w.half);
    };
    auto page = [&](int st) __attribute__((always_inline)) { return st < s1 ? form_page(p, it.pt_off, 32 * st) : 0; };
    auto as8 = [](uint4 x) __attribute__((always_inline)) {
        vec8 r;
        __builtin_memcpy(&r, &x, 16);
        return r;
    };
    int st = s0 + wave;
    int phys = page(st);
    if (st < s1) {
        load_k(st, phys);
        load_v(st, phys);
    }
    w.load_q(p);
    for (; st < s1; st += 4) {
        phys = page(st + 4);
        f32x16_t s[1];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
        const float ks = E8 ? scale_of(o.ks) : 1.f;
#pragma unroll
        for (int kk = 0; kk < F::NK; ++kk) {
            vec8 a;
            if constexpr (E8) {
                const uint4 x = o.k[kk >> 1];
                a = kk & 1 ? widen8(x.z, x.w, ks) : widen8(x.x, x.y, ks);
            } else {
                a = as8(o.k[kk]);
            }
#pragma unroll
            for (int c = 0; c < PARTS; ++c) s[0] = mfma32(a, w.q[c][kk], s[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (st + 4 < s1) load_k(st + 4, phys);
        const bool edge = !range.all(32 * st, 32);
        w.prepare(p, s, 32 * st, edge);
        if (edge) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < FormStep<CT, D>::N; ++i) {
                uint32_t x[4] = {o.v[i].x, o.v[i].y, o.v[i].z, o.v[i].w};
                constexpr uint32_t exps = E8 ? 0x7F7F7F7Fu : F::BF16 ? 0x7F807F80u : 0x7C007C00u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t y = ~x[j] & exps;  // an element of zeros: not a number or infinite
                    bad |= E8 ? ((y - 0x01010101u) & ~y & 0x80808080u) != 0 : (y & 0xFFFFu) == 0 || (y >> 16) == 0;
                }
            }
            if (__builtin_amdgcn_ballot_w64(bad)) {
                w.add_bad(p, it, kvh, 32 * st);
#pragma unroll
                for (int i = 0; i < FormStep<CT, D>::N; ++i) {
                    uint32_t x[4] = {o.v[i].x, o.v[i].y, o.v[i].z, o.v[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int b = 0; b < 32; b += 8 * ES) {
                            constexpr uint32_t exps = E8 ? 0x7Fu : F::BF16 ? 0x7F80u : 0x7C00u;
                            if ((x[j] >> b & exps) == exps) x[j] &= ~((E8 ? 0xFFu : 0xFFFFu) << b);
                        }
                    o.v[i] = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
        }
        vec8 wt[PARTS][1][2];
        const uint32_t vs[4] = {o.vs.x, o.vs.y, o.vs.z, o.vs.w};
        w.template softmax<1>(s, wt, [&](int, int r) __attribute__((always_inline)) { return scale_of(vs[r >> 2] >> (8 * (r & 3)) & 0xFF); });
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int d = 0; d < F::ND; ++d) {
                vec8 a;
                if constexpr (E8) a = x ? widen8(o.v[d].z, o.v[d].w, 1.f) : widen8(o.v[d].x, o.v[d].y, 1.f);
                else a = as8(o.v[x * F::ND + d]);
#pragma unroll
                for (int c = 0; c < PARTS; ++c) w.acc[d] = mfma32(a, wt[c][0][x], w.acc[d]);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (st + 4 < s1) load_v(st + 4, phys);
    }
    w.l = sum_xor32(w.l);
    w.settle(p, it, kvh, s0 + wave, s1, 4);
    merge_waves<F, 1, 4>(p, it, un, w, 0, wave, lds, rest);
}

// ------------------------------------------------------------------ many rows: bound by MFMAs and the softmax
// Four waves, RW of them of 32 rows each; with RW = 4 a wave takes whole tiles of 64 slots, with RW = 2 two waves share a row group, a
// step of 32 of every tile each.  K and V of a tile are shared through LDS, two tiles of each, and two workgroups on a CU fill
// each other's barriers, starts and ends (one of eight waves and 256 rows: six prompts of 101 to 1501 rows with capped scores 118 us).
// 16 bits: tiles are copied by buffer-load DMA as they lie in the page.  8 bits: a thread takes 16 bytes of K and V through
// registers and writes them as bf16 operands, once for all waves.
// Bound by MFMAs beside the exponentials, at the clock that the power limit leaves (1.7 to 2.1 of 2.4 GHz; a large product reaches
// 1.2 to 1.27 PFLOP/s): 2048 rows after 6144, 32 heads of 128 over 8 kv heads, 240 GFLOP, on four cards: bf16 236 to 248 us (970 to
// 1020 TFLOP/s), fp16 247 to 258, 8 bits 265 to 275, bf16 with slopes 279 to 289, with scores below a cap of 50 293 to 313 and
// about it 360 to 372, with caps beyond 64 399 to 407, fp32 queries in three parts 577 to 606 (three times the MFMAs; they, and those
// over 8 bits, spill 80 to 152 bytes of a lane at head size 128).
template <int D> struct FormRings {
    static constexpr int KB = 128 * D;                       // bytes of a tile's operands of K (or V)
    static constexpr int NST = 2;                            // tiles of each
    static constexpr int LDS = 2 * NST * KB;                 // (four waves' sums, at the end, are as many)
    static constexpr int REST = 4 * 64 * 8 + 4 * 64 * 4 + 64;  // (maximum, sum) of the waves; scales of V; spans
};

template <int CT, int D, int PARTS, int SCORES, int RW>
__device__ __forceinline__ void forms_tile(const FormsK& p, const FormItem& it, int u, char* lds, char* rest) {
    using F = FormTile<CT, D, PARTS, SCORES>;
    using L = FormRings<D>;
    using vec8 = typename F::vec8;
    using T = typename F::T;
    constexpr bool E8 = F::E8;
    constexpr int ES = E8 ? 1 : 2, STEPS = RW / 2, NS = PARTS == 1 ? STEPS : 1;  // steps of a tile that are a wave's; of them at a time
    constexpr int ROWS = 32 * RW, TILE = form_tile(kFormTiles);
    static_assert(TILE == 64 && form_tile(kFormTilesHalf) == 64 && form_rows(kFormTiles) == 128 && form_rows(kFormTilesHalf) == 64, "two steps, four or two waves of rows");
    constexpr int SB = 64 * D, KB = L::KB;         // bytes of a step's and of a tile's operands
    constexpr int PER = KB / 1024 / 4;             // DMA loads per wave for a tile of K (or V)
    constexpr int NP = 64 * D / 16 / 256;          // 8 bits: 16-byte pieces of K (or V) per thread
    float(*const vscale)[64] = reinterpret_cast<float(*)[64]>(rest + 4 * 64 * 8);             // [4][64]
    int(*const spans)[4] = reinterpret_cast<int(*)[4]>(rest + 4 * 64 * 8 + 4 * 64 * 4);       // [4][4]
    const int kv = p.geom.kv_heads, g = p.heads / kv;
    const FormUnit un = form_unit(p, it, g, ROWS, TILE, u);
    const int kvh = un.kvh, split = un.part, block = un.block;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rw = wave % RW;
    int st0 = wave / RW;  // its first step
    F w;
    w.init(p, it, kvh, g, ROWS * block + 32 * rw);
    FormRange range = w.range();
    if (w.lane == 0) {
        spans[wave][0] = range.lo;
        spans[wave][1] = range.hi;
        spans[wave][2] = range.all_lo;
        spans[wave][3] = range.all_hi;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        range.lo = min(range.lo, spans[i][0]);
        range.hi = max(range.hi, spans[i][1]);
        range.all_lo = max(range.all_lo, spans[i][2]);
        range.all_hi = min(range.all_hi, spans[i][3]);
    }
    range.lo = __builtin_amdgcn_readfirstlane(range.lo);
    range.hi = __builtin_amdgcn_readfirstlane(range.hi);
    range.all_lo = __builtin_amdgcn_readfirstlane(range.all_lo);
    range.all_hi = __builtin_amdgcn_readfirstlane(range.all_hi);
    const int tile0 = range.lo / TILE, tiles = range.lo > range.hi ? 0 : range.hi / TILE - tile0 + 1;
    // (the same in every lane: buffer resources and page lookups are scalar)
    const int i0 = __builtin_amdgcn_readfirstlane(tile0 + static_cast<int>(static_cast<long long>(tiles) * split / un.parts));
    const int i1 = __builtin_amdgcn_readfirstlane(tile0 + static_cast<int>(static_cast<long long>(tiles) * (split + 1) / un.parts));

    const long long page_bytes = p.geom.page_elems() * ES, plane_bytes = p.geom.plane_elems() * ES;
    const long long head_bytes = static_cast<long long>(kvh) * kPageTokens * D * ES;
    auto page = [&](int i) { return i < i1 ? form_page(p, it.pt_off, TILE * i) : 0; };
    // (tile numbers are not negative)
    auto k_at = [&](int i) { return lds + (static_cast<unsigned>(i) % L::NST) * KB; };
    auto v_at = [&](int i) { return lds + (L::NST + static_cast<unsigned>(i) % L::NST) * KB; };
    // 16 bits: request K or V of tile i, a load at a time
    auto source = [&](int i, int phys, bool v) __attribute__((always_inline)) {
        const char* base = p.pool + static_cast<long long>(phys) * page_bytes + head_bytes + (v ? plane_bytes : 0) + static_cast<long long>(TILE * i & (kPageTokens - 1)) * D * ES;
        return dma_source(base, i < i1 ? KB : 0);  // past the last tile: no records, no memory is read
    };
    auto load = [&](u32x4_t r, int i, bool v, int c) __attribute__((always_inline)) {
        dma16(r, (v ? v_at(i) : k_at(i)) + 1024 * (wave + 4 * c), 16 * w.lane, 1024 * (wave + 4 * c));
    };
    auto request = [&](int i, int phys, bool v) __attribute__((always_inline)) {
        const u32x4_t r = source(i, phys, v);
#pragma unroll
        for (int c = 0; c < PER; ++c) load(r, i, v, c);
    };
    constexpr int LOADS = E8 ? 0 : 2 * PER;  // per wave of K and V of a tile
    // 8 bits: pieces of K or V of tile i into registers (the scales of V with K), and from there as operands into LDS
    uint4 pk[E8 ? NP : 1], pv_[E8 ? NP : 1];
    uint32_t ps[E8 ? NP : 1], pvs = 0;
    auto fetch = [&](int i, int phys, bool v) __attribute__((always_inline)) {
        if (i >= i1) return;
        const char* pg = p.pool + static_cast<long long>(phys) * page_bytes;
        const char* base = pg + head_bytes + static_cast<long long>(TILE * i & (kPageTokens - 1)) * D;
        if (v) {
#pragma unroll
            for (int c = 0; c < NP; ++c) pv_[c] = *reinterpret_cast<const uint4*>(base + plane_bytes + 16 * (threadIdx.x + 256 * c));
            return;
        }
        const char* sc = pg + 2 * plane_bytes + kvh * kPageTokens + (TILE * i & (kPageTokens - 1));
#pragma unroll
        for (int c = 0; c < NP; ++c) {
            const int x = threadIdx.x + 256 * c, m = x & 31;  // piece x: step x / (2 D), lane x % 64
            pk[c] = *reinterpret_cast<const uint4*>(base + 16 * x);
            ps[c] = static_cast<uint8_t>(sc[32 * (x / (2 * D)) + 16 * (m >> 2 & 1) + 8 * (m >> 4) + 4 * (m >> 3 & 1) + (m & 3)]);
        }
        if (threadIdx.x < 64) pvs = static_cast<uint8_t>(sc[kv * kPageTokens + threadIdx.x]);
    };
    auto put = [&](int i, bool v) __attribute__((always_inline)) {
        if constexpr (E8) {
#pragma unroll
            for (int c = 0; c < NP; ++c) {
                const int x = threadIdx.x + 256 * c, st = x / (2 * D), j = x / 64 % (D / 32), l = x & 63;
                const float by = v ? 1.f : scale_of(ps[c]);
                const uint4 y = v ? pv_[c] : pk[c];
                bf16x8_t* to = reinterpret_cast<bf16x8_t*>(v ? v_at(i) + SB * st + 1024 * j + 16 * l : k_at(i) + SB * st + 2048 * j + 16 * l);
                to[0] = widen8(y.x, y.y, by);
                to[v ? 64 * F::ND : 64] = widen8(y.z, y.w, by);
            }
            if (!v && threadIdx.x < 64) vscale[i & 3][threadIdx.x] = scale_of(pvs);
        }
    };
    // what was requested (or put) in the last turn is there for every wave, what it read is free
    auto turn = [&]() __attribute__((always_inline)) {
        if (!E8) wait_dma();
        lds_barrier_dma_in_flight();
    };
    // this lane's part of the operands: K of step st, k-step kk; V of step st, PV step x, dim tile d
    const int m_ = w.lane & 31, sx = m_ >> 4, ax = (m_ >> 3) & 1, hx = (m_ >> 2) & 1, bx = m_ & 3;
    const int ko = E8 ? 16 * w.lane : 1024 * ax * (D / 32) + 16 * (16 * w.half + 4 * (2 * sx + hx) + bx);
    const int vo = E8 ? 16 * w.lane : 1024 * (m_ >> 4) + 16 * (16 * w.half + (w.lane & 15));
    auto k_op = [&](const char* k, int st, int kk) __attribute__((always_inline)) {
        return *reinterpret_cast<const vec8*>(k + SB * (st0 + st) + ko + (E8 ? 1024 : 512) * kk);
    };
    auto v_op = [&](const char* v, int st, int x, int d) __attribute__((always_inline)) {
        return *reinterpret_cast<const vec8*>(v + SB * (st0 + st) + vo + (E8 ? 1024 * (x * F::ND + d) : 2048 * d + 512 * x));
    };
    auto qk = [&](f32x16_t (&s)[NS], int i) __attribute__((always_inline)) {
        const char* const k = k_at(i);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[st][r] = 0.f;
#pragma unroll
            for (int kk = 0; kk < F::NK; ++kk) {
                const vec8 a = k_op(k, st, kk);
#pragma unroll
                for (int c = 0; c < PARTS; ++c) s[st] = mfma32(a, w.q[c][kk], s[st]);
            }
        }
    };
    auto pv = [&](const vec8 (&wt)[PARTS][NS][2], int i) __attribute__((always_inline)) {
        const char* const v = v_at(i);
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int d = 0; d < F::ND; ++d) {
                    const vec8 a = v_op(v, st, x, d);
#pragma unroll
                    for (int c = 0; c < PARTS; ++c) w.acc[d] = mfma32(a, wt[c][st][x], w.acc[d]);
                }
    };
    auto edge = [&](int i) __attribute__((always_inline)) { return !range.all(TILE * i, TILE); };
    // V elements that are not finite, of a tile that not every row sees whole: a product of all of them with zeros shows them (the
    // same in every wave).
    auto check_v = [&](int i) __attribute__((always_inline)) {
        char* const v = v_at(i);
        vec8 zero;
#pragma unroll
        for (int j = 0; j < 8; ++j) zero[j] = static_cast<T>(0.f);
        f32x16_t z;
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] = 0.f;
#pragma unroll
        for (int c = 0; c < KB / 1024; ++c) z = mfma32(*reinterpret_cast<const vec8*>(v + 1024 * c + 16 * w.lane), zero, z);
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) t += z[j];
        if (__builtin_amdgcn_ballot_w64(!(t == 0.f))) {
#pragma unroll 1
            for (int st = 0; st < STEPS; ++st) w.add_bad(p, it, kvh, TILE * i + 32 * (wave / RW + st));
            lds_barrier_dma_in_flight();
            for (int c = threadIdx.x; c < KB / 2; c += 256) {
                T* x = reinterpret_cast<T*>(v) + c;
                if (!(fabsf(static_cast<float>(*x)) < INFINITY)) *x = static_cast<T>(0.f);
            }
            lds_barrier_dma_in_flight();
        }
    };
    auto v_scale = [&](int i) {
        return [&, i](int n, int r) __attribute__((always_inline)) { return vscale[i & 3][32 * (st0 + n) + 16 * w.half + r]; };
    };
    auto form = [&](f32x16_t (&s)[NS], int i) __attribute__((always_inline)) { w.prepare(p, s, TILE * i + 32 * st0, edge(i)); };
    if (i0 < i1) {
        if constexpr (PARTS == 1) {
            // Tile i's softmax runs between the MFMAs of the scores of tile i + 1 and of V of tile i - 1: none of the three needs
            // another.  At the turn in front of it K of tile i + 1 and V of tile i - 1 are there; K of tile i + 2 and V of tile i come over
            // what the last turn read.
            f32x16_t s[2][NS];
            uint32_t wt[NS][2][4];  // a tile's weights, as operands
            int phys[3];            // of tiles i .. i + 2
#pragma unroll
            for (int x = 0; x < 3; ++x) phys[x] = page(i0 + x);
            if (E8) {
                fetch(i0, phys[0], false);
                w.load_q(p);
                put(i0, false);
                fetch(i0 + 1, phys[1], false);
                put(i0 + 1, false);
                fetch(i0 + 2, phys[2], false);
                fetch(i0, phys[0], true);
            } else {
                request(i0, phys[0], false);
                request(i0 + 1, phys[1], false);
                w.load_q(p);
                wait_vmcnt<PER>();
            }
            lds_barrier_dma_in_flight();
            qk(s[0], i0);
            auto weights8 = [](const uint32_t (&x)[4]) __attribute__((always_inline)) {
                vec8 r;
                __builtin_memcpy(&r, x, 16);
                return r;
            };
            // V of tile i - 1, then the scores of tile i + 1, an operand read kAhead MFMAs in front of its use, and beside them tile i's
            // weights, two at a time (left to itself, the compiler computes all weights, then has each MFMA wait for its operand).  The
            // weights follow the MFMAs that take the last tile's by ND, into their registers.  A load takes its wave some hundred cycles to
            // issue when eight waves issue at once (four in front of the MFMAs: 1470 cycles of 5260 a tile), so the requests stand
            // between them too, and with 8 bits what becomes operands.
            constexpr int kAhead = 4, EXTRAS = E8 ? 4 : LOADS;
            auto between = [&](int i, const f32x16_t (&s)[NS], f32x16_t (&next)[NS], uint32_t (&wt)[NS][2][4], auto first, auto extra) __attribute__((always_inline)) {
                constexpr bool PV = !decltype(first)::value;
                constexpr int NQ = NS * F::NK, OPS = PV ? 2 * NQ : NQ, PAIRS = 8 * NS;
                static_assert(NS * 2 * F::ND == NQ && F::NK % 4 == 0, "as many of each");
                const char *const k = k_at(i + 1), *const v = v_at(PV ? i - 1 : i);
                vec8 ring[kAhead];
                auto read = [&](int x) __attribute__((always_inline)) -> vec8 {
                    if (PV && x < NQ) return v_op(v, x / (2 * F::ND), x / F::ND % 2, x % F::ND);
                    const int j = PV ? x - NQ : x;
                    return k_op(k, j % NS, j / NS);
                };
#pragma unroll
                for (int x = 0; x < kAhead; ++x) ring[x] = read(x);
                const float ref = w.m == -INFINITY ? 0.f : -w.m;
                float sum[2] = {0.f, 0.f}, e[2];
                float2 vs[2];
                auto scales = [&](int y) __attribute__((always_inline)) {
                    return *reinterpret_cast<const float2*>(&vscale[i & 3][32 * (st0 + (y >> 3)) + 16 * w.half + 2 * (y & 7)]);
                };
                if (E8) vs[0] = scales(0);
                auto begin = [&](int y) __attribute__((always_inline)) {
                    const int n = y >> 3, r = 2 * (y & 7);
                    if (E8 && y + 1 < PAIRS) vs[(y & 1) ^ 1] = scales(y + 1);
                    e[0] = s[n][r];
                    e[1] = s[n][r + 1];
                    asm volatile("" : "+v"(e[0]), "+v"(e[1]));  // not before the MFMA in front
                    e[0] = fast_exp2(w.logit(e[0], ref));
                    e[1] = fast_exp2(w.logit(e[1], ref));
                };
                auto end = [&](int y) __attribute__((always_inline)) {
                    const int n = y >> 3, r = 2 * (y & 7);
                    sum[0] += e[0];
                    sum[1] += e[1];
                    if (E8) {
                        e[0] *= vs[y & 1].x;
                        e[1] *= vs[y & 1].y;
                    }
                    typedef float f32x2 __attribute__((ext_vector_type(2)));
                    typedef T T2 __attribute__((ext_vector_type(2)));
                    const T2 pair = __builtin_convertvector((f32x2{e[0], e[1]}), T2);
                    uint32_t b;
                    __builtin_memcpy(&b, &pair, 4);
                    asm volatile("" : "+v"(b), "+v"(sum[0]), "+v"(sum[1]));  // nor after the next
                    wt[n][r >> 3][(r & 7) >> 1] = b;
                };
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int x = 0; x < OPS + (PV ? F::ND : 0); ++x) {
                    if (x < OPS) {
                        if (PV && x < NQ) {
                            w.acc[x % F::ND] = mfma32(ring[x % kAhead], weights8(wt[x / (2 * F::ND)][x / F::ND % 2]), w.acc[x % F::ND]);
                        } else {
                            const int j = PV ? x - NQ : x, st = j % NS, kk = j / NS;
                            if (kk == 0)
#pragma unroll
                                for (int r = 0; r < 16; ++r) next[st][r] = 0.f;
                            next[st] = mfma32(ring[x % kAhead], w.q[0][kk], next[st]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                        constexpr int EACH = (EXTRAS + OPS - 1) / OPS;
#pragma unroll
                        for (int k = EACH * x; k < EACH * (x + 1); ++k)
                            if (k < EXTRAS) extra(k);
                    }
                    if constexpr (PV) {
                        constexpr int SP = OPS / PAIRS;  // MFMAs to a pair
                        const int t = x - F::ND;
                        if (t >= 0 && t % SP == 0) begin(t / SP);
                        if (SP > 1 && t >= 0 && t % SP == 0) asm volatile("" : "+v"(e[0]), "+v"(e[1]));
                        if (t >= 0 && t % SP == SP - 1) end(t / SP);
                    } else {
#pragma unroll
                        for (int y = x * PAIRS / OPS; y < (x + 1) * PAIRS / OPS; ++y) {
                            begin(y);
                            end(y);
                        }
                    }
                    if (x + kAhead < OPS) ring[x % kAhead] = read(x + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
                return sum[0] + sum[1];
            };
            auto tile = [&](int i, f32x16_t (&s)[NS], f32x16_t (&next)[NS], auto first) __attribute__((always_inline)) {
                turn();
                const int p0 = phys[0], p1 = phys[1], p2 = phys[2], p3 = page(i + 3);
                const u32x4_t rk = source(i + 2, p2, false), rv = source(i, p0, true);
                phys[0] = p1;
                phys[1] = p2;
                phys[2] = p3;
                auto extra = [&](int k) __attribute__((always_inline)) {
                    if (!E8) {
                        if (k < PER) load(rk, i + 2, false, k);
                        else load(rv, i, true, k - PER);
                        return;
                    }
                    if (k == 0) put(i + 2, false);
                    if (k == 1) fetch(i + 3, p3, false);
                    if (k == 2) put(i, true);
                    if (k == 3) fetch(i + 1, p1, true);
                };
                if (!first.value && edge(i - 1)) check_v(i - 1);
                form(s, i);
                const float c = w.raise(s);
                const float sum = between(i, s, next, wt, first, extra);
                w.rescale(c);
                w.l += sum;
            };
            tile(i0, s[0], s[1], std::true_type{});
            int i = i0 + 1;
            for (; i + 1 < i1; i += 2) {
                tile(i, s[1], s[0], std::false_type{});
                tile(i + 1, s[0], s[1], std::false_type{});
            }
            if (i < i1) tile(i, s[1], s[0], std::false_type{});
            turn();
            if (edge(i1 - 1)) check_v(i1 - 1);
            vec8 last[PARTS][NS][2];
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                last[0][n][0] = weights8(wt[n][0]);
                last[0][n][1] = weights8(wt[n][1]);
            }
            pv(last, i1 - 1);
        } else {
            // Parts take the registers: one step after another.
            int phys = page(i0 + 1);
            const int p0 = page(i0);
            if (E8) {
                fetch(i0, p0, false);
                fetch(i0, p0, true);
                w.load_q(p);
                put(i0, false);
                put(i0, true);
                fetch(i0 + 1, phys, false);
                fetch(i0 + 1, phys, true);
                phys = page(i0 + 2);
            } else {
                request(i0, p0, false);
                request(i0, p0, true);
                w.load_q(p);
            }
            for (int i = i0; i < i1; ++i) {
                turn();
                if (E8) {
                    put(i + 1, false);
                    put(i + 1, true);
                    fetch(i + 2, phys, false);
                    fetch(i + 2, phys, true);
                    phys = page(i + 3);
                } else {
                    request(i + 1, phys, false);
                    request(i + 1, phys, true);
                    phys = page(i + 2);
                }
                if (edge(i)) check_v(i);
#pragma unroll 1
                for (st0 = wave / RW; st0 < wave / RW + STEPS; ++st0) {
                    f32x16_t s[NS];
                    qk(s, i);
                    form(s, i);
                    vec8 wt[PARTS][NS][2];
                    w.softmax(s, wt, v_scale(i));
                    pv(wt, i);
                }
            }
            wait_dma();  // (of the tile behind the last: nothing is read, but zeros are written)
        }
    }
    w.l = sum_xor32(w.l);
    w.settle(p, it, kvh, 2 * i0 + wave / RW, 2 * i1, RW == 4 ? 1 : 2);
    merge_waves<F, RW, 4 / RW>(p, it, un, w, rw, wave / RW, lds, rest);
}

// Items of both sorts in one launch: what one leaves of HBM or the MFMAs the other takes (64 rows behind 8192 shared positions
// and their own keys: 50 us in two launches, 40 in one).
template <int CT, int D, int PARTS, int SCORES>
__global__ void __launch_bounds__(256, 2) forms_mfma_kernel(const FormsK p) {
    using L = FormRings<D>;
    __shared__ __attribute__((aligned(1024))) char lds[L::LDS];
    __shared__ __attribute__((aligned(16))) char rest[L::REST];
    const FormItem it = p.it[form_find(p, blockIdx.x)];
    const int u = blockIdx.x - it.unit0;
    if (it.kind == kFormStream) forms_stream<CT, D, PARTS, SCORES>(p, it, u, lds, rest);
    else if (it.kind == kFormTilesHalf) forms_tile<CT, D, PARTS, SCORES, 2>(p, it, u, lds, rest);
    else forms_tile<CT, D, PARTS, SCORES, 4>(p, it, u, lds, rest);
}
template <int CT, int D, int PARTS> hipError_t form_launch_scores(const FormsK& k, int units, hipStream_t s) {
    const double in = std::fabs(k.qscale) / static_cast<double>(k.cap), last = k.cap * std::pow(in, 9.0) * 0.017;  // the last coefficient
    // Caps beyond 64 take the arithmetic that tells small scores from large ones: 2^-22 of a cap of 64 is 2^-16 of a weight, a 32nd of
    // what fp16 rounds off; of a million it would be a quarter.  (2048 bf16 rows after 6144, 32 heads of 128 over 8 kv heads: 293 us
    // with scores far below the cap and 362 about it per weight, 399 whatever the scores by kScoresBoth.)  Queries in
    // parts are capped score by score in either; kScoresCap takes no slope off.
    const bool per_weight = PARTS > 1 || (k.cap <= 64.f * kLog2e && in < 1e3 && last > 1e-36 && last < 1e30);
    if (k.cap > 0.f && (k.slopes || !per_weight)) hipLaunchKernelGGL((forms_mfma_kernel<CT, D, PARTS, kScoresBoth>), dim3(units), dim3(256), 0, s, k);
    else if (k.cap > 0.f) hipLaunchKernelGGL((forms_mfma_kernel<CT, D, PARTS, kScoresCap>), dim3(units), dim3(256), 0, s, k);
    else if (k.slopes) hipLaunchKernelGGL((forms_mfma_kernel<CT, D, PARTS, kScoresSlope>), dim3(units), dim3(256), 0, s, k);
    else hipLaunchKernelGGL((forms_mfma_kernel<CT, D, PARTS, kScoresPlain>), dim3(units), dim3(256), 0, s, k);
    return hipGetLastError();
}
// Queries that the tile's type holds enter as one part, others as two of fp16 or three of bf16.
template <int CT> hipError_t form_launch_type(const FormsK& k, int units, hipStream_t s) {
    constexpr int OWN = CT == QR_DTYPE_F16 ? QR_DTYPE_F16 : QR_DTYPE_BF16, PARTS = CT == QR_DTYPE_F16 ? 2 : 3;
    if (k.geom.head_dim == 128) return k.act == OWN ? form_launch_scores<CT, 128, 1>(k, units, s) : form_launch_scores<CT, 128, PARTS>(k, units, s);
    return k.act == OWN ? form_launch_scores<CT, 64, 1>(k, units, s) : form_launch_scores<CT, 64, PARTS>(k, units, s);
}

}  // namespace qr
