// qr_forms_f32.hip -- attention in its other forms and behind shared prefixes on fp32 MFMA tiles: fp32 caches of head size 64
// or 128, whole groups of query heads, gfx950.
//
// A wave owns RT tiles of 16 rows (query, query head pairs of a kv head) and takes steps of 16 positions:
//   QK  S^T[position][row] = K . q^T,  PV  O^T[dim][row] += V^T . P^T
// v_mfma_f32_16x16x4_f32: A[m = lane % 16][k = lane / 16], B[k = lane / 16][n = lane % 16], D[m = 4 (lane / 16) + r][n = lane % 16].
// With Q = lane / 16: an A operand of QK is K of position lane % 16, dim 16 j + 4 Q + c for MFMA (j, c), so that a lane's
// operands are 16 bytes of a row; a lane's scores r are positions 4 Q + r, its k-slots of MFMA r of PV; and V's operand of dim tile
// (j, c) is V of position 4 Q + r, dim 64 j + 4 (lane % 16) + c, again 16 bytes of a row, so that acc[j][c][i] is dim 64 j + 16 Q +
// 4 i + c.  Operands come straight from the page; products and sums are fp32 throughout.
//
// Four waves of a workgroup take every fourth step of a block's keys and merge at the end.
#include "qr_forms.hpp"
#include "qr_mfma.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ f32x4_t mfma4(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

template <int D, int RT, int SCORES>
__device__ __forceinline__ void forms_f32(const FormsK& p, const FormItem& it, int u, f32x4_t* xa, float2* xm) {
    constexpr int NK = D / 16, NJ = D / 64, NG = D / 16;  // NG: f32x4 groups of a row tile in a lane
    // xa: [4][RT][NG][64], xm: [4][RT][64]
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
    const float* const pool = reinterpret_cast<const float*>(p.pool) + static_cast<long long>(kvh) * kPageTokens * D;
    f32x4_t k[NK], v[4][NJ];
    auto load_k = [&](int st, int phys) __attribute__((always_inline)) {
        const float* b = pool + phys * page_elems + static_cast<long long>(16 * (st & 15) + n) * D + 4 * Q;
#pragma unroll
        for (int j = 0; j < NK; ++j) k[j] = *reinterpret_cast<const f32x4_t*>(b + 16 * j);
    };
    auto load_v = [&](int st, int phys) __attribute__((always_inline)) {
        const float* b = pool + phys * page_elems + plane + static_cast<long long>(16 * (st & 15) + 4 * Q) * D + 4 * n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j) v[r][j] = *reinterpret_cast<const f32x4_t*>(b + r * D + 64 * j);
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
    f32x4_t acc[RT][NJ][4];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[t][j][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    // V elements of the loaded step that are not finite; they as they are to the rows that see them.
    auto bad_v = [&]() __attribute__((always_inline)) {
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) bad |= !(fabsf(v[r][j][c]) < INFINITY);
        return __builtin_amdgcn_ballot_w64(bad) != 0;
    };
    auto add_bad = [&](int st, int phys) __attribute__((always_inline)) {
        const float* b = pool + phys * page_elems + plane + static_cast<long long>(16 * (st & 15)) * D;
#pragma unroll 1
        for (int x = 0; x < 16; ++x)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(b + x * D + 64 * j + 16 * Q + 4 * i);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
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
#pragma unroll
        for (int j = 0; j < NK; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int t = 0; t < RT; ++t) s[t][c & 1] = mfma4(k[j][c], q[t][j][c], s[t][c & 1]);
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
                    for (int x = 0; x < 4; ++x) acc[t][j][x] *= c;
            }
            const float ref = m[t] == -INFINITY ? 0.f : m[t];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[t][r] = fast_exp2(z[r] - ref);
            l[t] += (w[t][0] + w[t][1]) + (w[t][2] + w[t][3]);
        }
        if (edge) {
            // Elements of V that are not finite would reach rows that do not see them as 0 x inf: they are added to the rows that see
            // them as they are (no finite weight changes them), and cleared.
            if (bad_v()) {
                add_bad(st, now);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[r][j][c] = fabsf(v[r][j][c]) < INFINITY ? v[r][j][c] : 0.f;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int t = 0; t < RT; ++t) acc[t][j][c] = mfma4(v[r][j][c], w[t][r], acc[t][j][c]);
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
            for (int c = 0; c < 4; ++c) sum += acc[t][j][c];
        const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        lost |= all != all && l[t] == l[t];
    }
    if (__builtin_amdgcn_ballot_w64(lost)) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][j][c][i] = acc[t][j][c][i] != acc[t][j][c][i] ? 0.f : acc[t][j][c][i];
#pragma unroll 1
        for (st = s0 + wave; st < s1; st += 4) {
            phys = page(st);
            load_v(st, phys);
            if (bad_v()) add_bad(st, phys);
        }
    }

    // the waves merge: wave w adds up row groups w, w + 4, ... of (tile, j, i), 4 dims each
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                xa[((wave * RT + t) * NG + 4 * j + i) * 64 + lane] = f32x4_t{acc[t][j][0][i], acc[t][j][1][i], acc[t][j][2][i], acc[t][j][3][i]};
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
            const int i = wave * (NG / 4) + x, d = 64 * (i >> 2) + 16 * Q + 4 * (i & 3);
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y < 4; ++y) o += form_weighed(xa[((y * RT + t) * NG + i) * 64 + lane], c[y]);
            if (!whole) {
                *reinterpret_cast<f32x4_t*>(p.part_acc + slot * D + d) = o;
            } else {
                o *= inv;
                if (p.act == QR_DTYPE_F32) {
                    __builtin_memcpy(static_cast<float*>(p.out) + at + d, &o, 16);
                } else {
                    uint16_t b[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) b[y] = f32_to_out16(o[y], p.act);
                    __builtin_memcpy(static_cast<uint16_t*>(p.out) + at + d, b, 8);
                }
            }
        }
        if (wave == 0 && Q == 0) form_store_ml(p, ch, it, slot, un, M, L);
    }
}

template <int D, int SCORES>
__global__ void __launch_bounds__(kThreads, 2) forms_f32_kernel(const FormsK p) {
    __shared__ f32x4_t xa[4 * 2 * (D / 16) * 64];
    __shared__ float2 xm[4 * 2 * 64];
    const FormItem it = p.it[form_find(p, blockIdx.x)];
    const int u = blockIdx.x - it.unit0;
    if (it.kind == kFormF32Half) forms_f32<D, 1, SCORES>(p, it, u, xa, xm);
    else forms_f32<D, 2, SCORES>(p, it, u, xa, xm);
}
template <int D> hipError_t launch_scores(const FormsK& k, int units, hipStream_t s) {
    if (k.cap > 0.f && k.slopes) hipLaunchKernelGGL((forms_f32_kernel<D, kScoresBoth>), dim3(units), dim3(kThreads), 0, s, k);
    else if (k.cap > 0.f) hipLaunchKernelGGL((forms_f32_kernel<D, kScoresCap>), dim3(units), dim3(kThreads), 0, s, k);
    else if (k.slopes) hipLaunchKernelGGL((forms_f32_kernel<D, kScoresSlope>), dim3(units), dim3(kThreads), 0, s, k);
    else hipLaunchKernelGGL((forms_f32_kernel<D, kScoresPlain>), dim3(units), dim3(kThreads), 0, s, k);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_forms_f32(const FormsK& k, int units, hipStream_t s) {
    return k.geom.head_dim == 128 ? launch_scores<128>(k, units, s) : launch_scores<64>(k, units, s);
}

}  // namespace qr
