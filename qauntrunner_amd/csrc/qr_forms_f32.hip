// qr_forms_f32.hip -- attention in its other forms and behind shared prefixes on fp32 MFMA tiles: fp32 caches of head size 64,
// 96, 128 or 256, caches of 16 and 8 bits of head size 96 or 256 (rows in order in the page), whole groups of query heads, gfx950.
//
// A wave owns RT tiles of 16 rows (query, query head pairs of a kv head) and takes steps of 16 positions:
//   QK  S^T[position][row] = K . q^T,  PV  O^T[dim][row] += V^T . P^T
// v_mfma_f32_16x16x4_f32: A[m = lane % 16][k = lane / 16], B[k = lane / 16][n = lane % 16], D[m = 4 (lane / 16) + r][n = lane % 16].
// With Q = lane / 16: an A operand of QK is K of position lane % 16, dim 16 j + 4 Q + c for MFMA (j, c), so that a lane's
// operands are 4 consecutive values of a row; a lane's scores r are positions 4 Q + r, its k-slots of MFMA r of PV; and V's operand of
// dim tile (j, c), c < PE, is V of position 4 Q + r, dim 16 PE j + PE (lane % 16) + c, again PE consecutive values, so that acc[j][c][i]
// is dim 16 PE j + PE (4 Q + i) + c.  Operands come straight from the page, narrower ones become fp32 where an MFMA takes them;
// products and sums are fp32 throughout.
//
// Four waves of a workgroup take every fourth step of a block's keys and merge at the end.  32 rows are bound by their MFMAs (an eighth
// of the 16-bit rate: 157 TFLOP/s), 16 by HBM.  Three prompts of 61 to 501 rows, 28 heads of 128 with slopes: 77 us for 4.3 GFLOP of
// which a product would take 28; the rest is blocks that see part of their steps, the longest unit's end, and the operands
// that come from L2 once for every 32 rows (64 rows per wave: registers).  With 32 heads of 96 over 8 kv heads, bf16: 16 sequences of 4096
// positions 54 to 59 us (3.4 to 3.7 TB/s), 512 rows after 3584 251 to 266 us (91 to 97 TFLOP/s); with heads of 256 149 us (3.6 TB/s)
// and 1260 (51 TFLOP/s), 8 bits 140 and 833.
#include "qr_forms.hpp"
#include "qr_mfma.hpp"
#include "qr_quant.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ f32x4_t mfma4(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// N consecutive values of a row of a cache of type CT (8 bits: without their scale).
template <int CT, int N> struct Few {
    typedef typename std::conditional<CT == QR_DTYPE_F32, float, typename std::conditional<CT == QR_DTYPE_E4M3, uint8_t, uint16_t>::type>::type E;
    E v[N];
    __device__ __forceinline__ void load(const E* p) { __builtin_memcpy(v, __builtin_assume_aligned(p, sizeof(v)), sizeof(v)); }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (CT == QR_DTYPE_F32) return v[i];
        else if constexpr (CT == QR_DTYPE_BF16) return bf16_bits_to_f32(v[i]);
        else if constexpr (CT == QR_DTYPE_F16) return f16_bits_to_f32(v[i]);
        else {
            uint32_t w = 0;
            __builtin_memcpy(&w, v, N);
            return i == 0 ? quant_value<0>(w) : i == 1 ? quant_value<1>(w) : i == 2 ? quant_value<2>(w) : quant_value<3>(w);
        }
    }
};

template <int CT, int D, int RT, int SCORES>
__device__ __forceinline__ void forms_f32(const FormsK& p, const FormItem& it, int u, char* lds, float2* xm) {
    constexpr bool E8 = CT == QR_DTYPE_E4M3;
    constexpr int PE = D % 64 ? 2 : 4, NK = D / 16, NJ = D / (16 * PE), NG = 4 * NJ;  // NG: groups of PE dims of a row tile in a lane
    static_assert(D % (16 * PE) == 0 && NG % 4 == 0, "whole groups, a wave's share of them");
    typedef float few __attribute__((ext_vector_type(PE)));
    typedef typename Few<CT, 4>::E E;
    few* const xa = reinterpret_cast<few*>(lds);  // [4][RT][NG][64]
    // xm: [4][RT][64]
    const int kv = p.geom.kv_heads, g = p.heads / kv;
    const FormUnit un = form_unit(p, it, g, 16 * RT, form_tile(kFormF32), u);
    static_assert(form_tile(kFormF32) == 16 && form_rows(kFormF32) == 32 && form_rows(kFormF32Half) == 16, "steps and row tiles");
    const int kvh = un.kvh, split = un.part, block = un.block;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, Q = lane >> 4;
    int row[RT], head[RT], lo[RT], hi[RT], chunk[RT];
    bool on[RT];
    int away[RT];
    float slope[RT];
    f32x4_t q[RT][NK];
    FormRange range{0x7FFFFFFF, -1, -1, 0x7FFFFFFF};
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = 16 * (RT * block + t) + n;
        on[t] = r < it.rows * g;
        const int rr = on[t] ? r : it.rows * g - 1, j = rr / g;
        head[t] = kvh * g + rr - j * g;
        row[t] = it.row0 + j;
        const FormSpan s = form_row(p, it, j);
        chunk[t] = s.chunk;
        lo[t] = s.lo;
        hi[t] = on[t] ? s.hi : -1;
        away[t] = s.pos - it.base;
        slope[t] = SCORES == kScoresSlope || SCORES == kScoresBoth ? p.slopes[head[t]] * kLog2e : 0.f;
        if (lo[t] <= hi[t]) {
            range.lo = min(range.lo, lo[t]);
            range.hi = max(range.hi, hi[t]);
        }
        if (on[t]) {
            range.all_lo = max(range.all_lo, lo[t]);
            range.all_hi = min(range.all_hi, hi[t]);
        }
    }
    range = {__builtin_amdgcn_readfirstlane(wave_min(range.lo)), __builtin_amdgcn_readfirstlane(wave_max(range.hi)),
             __builtin_amdgcn_readfirstlane(wave_max(range.all_lo)), __builtin_amdgcn_readfirstlane(wave_min(range.all_hi))};
    const int step0 = range.lo >> 4, steps = range.lo > range.hi ? 0 : (range.hi >> 4) - step0 + 1;
    const int s0 = __builtin_amdgcn_readfirstlane(step0 + static_cast<int>(static_cast<long long>(steps) * split / un.parts));
    const int s1 = __builtin_amdgcn_readfirstlane(step0 + static_cast<int>(static_cast<long long>(steps) * (split + 1) / un.parts));

    const long long page_elems = p.geom.page_elems(), plane = p.geom.plane_elems();
    const char* const scales = p.pool + 2 * plane + kvh * kPageTokens;  // (8 bits: elements are bytes)
    const E* const pool = reinterpret_cast<const E*>(p.pool) + static_cast<long long>(kvh) * kPageTokens * D;
    Few<CT, 4> k[NK];
    Few<CT, PE> v[4][NJ];
    uint32_t ks = 0, vs = 0;  // 8 bits: scale bytes of K at the lane's position and of V at its four
    auto load_k = [&](int st, int phys) __attribute__((always_inline)) {
        const E* b = pool + phys * page_elems + static_cast<long long>(16 * (st & 15) + n) * D + 4 * Q;
#pragma unroll
        for (int j = 0; j < NK; ++j) k[j].load(b + 16 * j);
        if (E8) ks = static_cast<uint8_t>(scales[phys * page_elems + 16 * (st & 15) + n]);
    };
    auto load_v = [&](int st, int phys) __attribute__((always_inline)) {
        const E* b = pool + phys * page_elems + plane + static_cast<long long>(16 * (st & 15) + 4 * Q) * D + PE * n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[r][j].load(b + r * D + 16 * PE * j);
        if (E8) vs = *reinterpret_cast<const uint32_t*>(scales + phys * page_elems + kv * kPageTokens + 16 * (st & 15) + 4 * Q);
    };
    auto page = [&](int st) __attribute__((always_inline)) { return st < s1 ? form_page(p, it.pt_off, 16 * st) : 0; };
    int st = s0 + wave;
    int phys = page(st);
    if (st < s1) {
        load_k(st, phys);
        load_v(st, phys);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const long long at = (static_cast<long long>(row[t]) * p.heads + head[t]) * D + 4 * Q;
        if (p.act == QR_DTYPE_F32) {
#pragma unroll
            for (int j = 0; j < NK; ++j) __builtin_memcpy(&q[t][j], static_cast<const float*>(p.q) + at + 16 * j, 16);
        } else {
            uint16_t x[NK][4];
#pragma unroll
            for (int j = 0; j < NK; ++j) __builtin_memcpy(x[j], static_cast<const uint16_t*>(p.q) + at + 16 * j, 8);
            const bool bf = p.act == QR_DTYPE_BF16;
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) q[t][j][c] = bf ? bf16_bits_to_f32(x[j][c]) : f16_bits_to_f32(x[j][c]);
        }
#pragma unroll
        for (int j = 0; j < NK; ++j) q[t][j] *= p.qscale;
    }
    float m[RT], l[RT];
    f32x4_t acc[RT][NJ][PE];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < PE; ++c) acc[t][j][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // V elements of the loaded step that are not finite; they as they are to the rows that see them.
    auto bad_v = [&]() __attribute__((always_inline)) {
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < PE; ++c) bad |= !(fabsf(v[r][j][c]) < INFINITY);
        return __builtin_amdgcn_ballot_w64(bad) != 0;
    };
    auto add_bad = [&](int st, int phys) __attribute__((always_inline)) {
        const E* b = pool + phys * page_elems + plane + static_cast<long long>(16 * (st & 15)) * D;
#pragma unroll 1
        for (int x = 0; x < 16; ++x)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    Few<CT, PE> y;
                    y.load(b + x * D + 16 * PE * j + PE * (4 * Q + i));
#pragma unroll
                    for (int c = 0; c < PE; ++c)
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            if (!(fabsf(y[c]) < INFINITY) && 16 * st + x >= lo[t] && 16 * st + x <= hi[t]) acc[t][j][c][i] += y[c];
                }
    };
    for (; st < s1; st += 4) {
        const int now = phys, t0 = 16 * st;
        phys = page(st + 4);
        f32x4_t s[RT][2];  // (two chains of products)
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][0] = s[t][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        const float by = E8 ? scale_of(ks) : 1.f;
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float x = E8 ? k[j][c] * by : k[j][c];
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][c & 1] = mfma4(x, q[t][j][c], s[t][c & 1]);
            }
        __builtin_amdgcn_sched_barrier(0);
        if (st + 4 < s1) load_k(st + 4, phys);
        const bool edge = !range.all(t0, 16);
        f32x4_t w[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            f32x4_t z = s[t][0] + s[t][1];
            const int t1 = t0 + 4 * Q;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (SCORES == kScoresCap || SCORES == kScoresBoth) z[r] = p.cap * tanhf(z[r] / p.cap);
                if (SCORES == kScoresSlope || SCORES == kScoresBoth) z[r] = fmaf(-slope[t], fabsf(static_cast<float>(t1 + r - away[t])), z[r]);
                if (edge && (t1 + r < lo[t] || t1 + r > hi[t])) z[r] = -INFINITY;
            }
            const float top = max_xor32(max_xor16(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]))));
            const float mn = fmaxf(m[t], top);
            if (__builtin_amdgcn_ballot_w64(mn > m[t])) {
                const float c = m[t] == -INFINITY ? 0.f : fast_exp2(m[t] - mn);
                m[t] = mn;
                l[t] *= c;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int x = 0; x < PE; ++x) acc[t][j][x] *= c;
            }
            const float ref = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[t][r] = fast_exp2(z[r] - ref);
            l[t] += (w[t][0] + w[t][1]) + (w[t][2] + w[t][3]);
            if (E8)
#pragma unroll
                for (int r = 0; r < 4; ++r) w[t][r] *= scale_of(vs >> (8 * r) & 0xFF);
        }
        // Elements of V that are not finite would reach rows that do not see them as 0 x inf: they are added to the rows that see
        // them as they are (no finite weight changes them), and count as zeros.
        const bool odd = edge && bad_v();
        if (odd) add_bad(st, now);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < PE; ++c) {
                    float x = v[r][j][c];
                    if (odd) x = fabsf(x) < INFINITY ? x : 0.f;
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[t][j][c] = mfma4(x, w[t][r], acc[t][j][c]);
                }
        __builtin_amdgcn_sched_barrier(0);
        if (st + 4 < s1) load_v(st + 4, phys);
    }

    // A sum that is no number while that of its weights is: an infinite V whose weight is zero in 32 bits, but none in the
    // formula.  The row shows the sum of these elements.
    bool lost = false;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] = sum_xor32(sum_xor16(l[t]));
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < PE; ++c) sum += acc[t][j][c];
        const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        lost |= all != all && l[t] == l[t];
    }
    if (__builtin_amdgcn_ballot_w64(lost)) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < PE; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][j][c][i] = acc[t][j][c][i] != acc[t][j][c][i] ? 0.f : acc[t][j][c][i];
#pragma unroll 1
        for (st = s0 + wave; st < s1; st += 4) {
            phys = page(st);
            load_v(st, phys);
            if (bad_v()) add_bad(st, phys);
        }
    }

    // the waves merge: each adds up a quarter of the groups (j, i) of PE dims
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                few x;
#pragma unroll
                for (int c = 0; c < PE; ++c) x[c] = acc[t][j][c][i];
                xa[((wave * RT + t) * NG + 4 * j + i) * 64 + lane] = x;
            }
        xm[(wave * RT + t) * 64 + lane] = make_float2(m[t], l[t]);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float M = -INFINITY, L = 0.f, c[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) M = fmaxf(M, xm[(x * RT + t) * 64 + lane].x);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float2 ml = xm[(x * RT + t) * 64 + lane];
            c[x] = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - M);
            L = fmaf(ml.y, c[x], L);
        }
        if (!on[t]) continue;
        const FormRows& ch = p.c[chunk[t]];
        const bool whole = form_whole(ch, it, un.parts);
        const long long slot = ch.slot0 + (static_cast<long long>(row[t] - ch.row0) * p.heads + head[t]) * ch.parts + it.part0 + split;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const long long at = (static_cast<long long>(row[t]) * p.heads + head[t]) * D;
#pragma unroll
        for (int x = 0; x < NG / 4; ++x) {
            const int i = wave * (NG / 4) + x, d = 16 * PE * (i >> 2) + PE * (4 * Q + (i & 3));
            few o{};
            float sum = 0.f;
#pragma unroll
            for (int y = 0; y < 4; ++y) o += xa[((y * RT + t) * NG + i) * 64 + lane] * c[y];
#pragma unroll
            for (int z = 0; z < PE; ++z) sum += o[z];
            if (__builtin_expect(sum != sum && L == L, 0)) {
                o = few{};
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int z = 0; z < PE; ++z) o[z] += form_weighed(xa[((y * RT + t) * NG + i) * 64 + lane][z], c[y]);
            }
            if (!whole) {
                *reinterpret_cast<few*>(p.part_acc + slot * D + d) = o;
            } else {
                o *= inv;
                if (p.act == QR_DTYPE_F32) {
                    __builtin_memcpy(static_cast<float*>(p.out) + at + d, &o, sizeof(o));
                } else {
                    uint16_t b[PE];
#pragma unroll
                    for (int y = 0; y < PE; ++y) b[y] = f32_to_out16(o[y], p.act);
                    __builtin_memcpy(static_cast<uint16_t*>(p.out) + at + d, b, sizeof(b));
                }
            }
        }
        if (wave == 0 && Q == 0) form_store_ml(p, ch, it, slot, un, M, L);
    }
}

// (Head size 256: a row tile's queries, sums, K and V are 300 to 400 registers of a lane and 128 KB of LDS at the end: one workgroup
// on a CU, 64 to 320 bytes of a lane spilled but for 8 bits.)
template <int CT, int D, int SCORES>
__global__ void __launch_bounds__(kThreads, D > 128 ? 1 : 2) forms_f32_kernel(const FormsK p) {
    __shared__ __attribute__((aligned(16))) char lds[4 * 2 * (D / 4) * 4 * 64];
    __shared__ float2 xm[4 * 2 * 64];
    const FormItem it = p.it[form_find(p, blockIdx.x)];
    const int u = blockIdx.x - it.unit0;
    if (it.kind == kFormF32Half) forms_f32<CT, D, 1, SCORES>(p, it, u, lds, xm);
    else forms_f32<CT, D, 2, SCORES>(p, it, u, lds, xm);
}
template <int CT, int D> hipError_t launch_scores(const FormsK& k, int units, hipStream_t s) {
    if (k.cap > 0.f && k.slopes) hipLaunchKernelGGL((forms_f32_kernel<CT, D, kScoresBoth>), dim3(units), dim3(kThreads), 0, s, k);
    else if (k.cap > 0.f) hipLaunchKernelGGL((forms_f32_kernel<CT, D, kScoresCap>), dim3(units), dim3(kThreads), 0, s, k);
    else if (k.slopes) hipLaunchKernelGGL((forms_f32_kernel<CT, D, kScoresSlope>), dim3(units), dim3(kThreads), 0, s, k);
    else hipLaunchKernelGGL((forms_f32_kernel<CT, D, kScoresPlain>), dim3(units), dim3(kThreads), 0, s, k);
    return hipGetLastError();
}
template <int CT> hipError_t launch_wide(const FormsK& k, int units, hipStream_t s) {
    return k.geom.head_dim == 96 ? launch_scores<CT, 96>(k, units, s) : launch_scores<CT, 256>(k, units, s);
}

}  // namespace

hipError_t launch_forms_f32(const FormsK& k, int units, hipStream_t s) {
    switch (k.dtype) {
        case QR_DTYPE_F16: return launch_wide<QR_DTYPE_F16>(k, units, s);
        case QR_DTYPE_BF16: return launch_wide<QR_DTYPE_BF16>(k, units, s);
        case QR_DTYPE_E4M3: return launch_wide<QR_DTYPE_E4M3>(k, units, s);
        default: break;
    }
    if (k.geom.head_dim == 64) return launch_scores<QR_DTYPE_F32, 64>(k, units, s);
    if (k.geom.head_dim == 128) return launch_scores<QR_DTYPE_F32, 128>(k, units, s);
    return launch_wide<QR_DTYPE_F32>(k, units, s);
}

}  // namespace qr
