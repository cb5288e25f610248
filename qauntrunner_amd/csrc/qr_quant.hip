// qr_quant.hip -- append of chunks of several sequences to an 8-bit cache (query / key norms and rotation in the same
// pass, rows quantised as they are written) and reading rows back as values of 16 or 32 bits, gfx950.
//
// q is normed and rotated in 32 bits, as for the other caches.  k is rounded to 3 bits behind its first, and a value that
// 32 bits move across a border between two codes would be off by a whole code: its norm, angles and rotation are in 64
// bits.  v needs no arithmetic but the division by a power of two, which is exact.
#include "qr_quant.hpp"

#include <algorithm>
#include <type_traits>

#include "qr_batch.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
    return x;
}
__device__ __forceinline__ float wave_sum(float x) { return sum_xor32(sum_xor16(group_sum(x, 16))); }
template <class T> __device__ __forceinline__ T wave_max(T x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const T o = __shfl_xor(x, i);
        x = o > x ? o : x;
    }
    return x;
}

// A head's values, lane + 64 c in y[c] (zeros past D), normed and rotated in T.
template <class T, int NC>
__device__ __forceinline__ void norm_rotate(T (&y)[NC], int lane, int D, const float* w, float eps, int rot, const T* cs, const T* sn, T* line) {
    if (w) {
        T ss = 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) ss += y[c] * y[c];
        const T r = T(1) / sqrt(wave_sum(ss) / static_cast<T>(D) + static_cast<T>(eps));
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (lane + 64 * c < D) y[c] = y[c] * r * static_cast<T>(w[lane + 64 * c]);
    }
    const int half = rot >> 1;
#pragma unroll
    for (int c = 0; c < NC; ++c) line[lane + 64 * c] = y[c];
    __builtin_amdgcn_wave_barrier();  // (one wave's line: its LDS accesses are in order)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = lane + 64 * c;
        if (i >= rot) continue;
        const T o = line[i < half ? i + half : i - half];  // the pair's other value
        y[c] = i < half ? y[c] * cs[i] - o * sn[i] : o * sn[i - half] + y[c] * cs[i - half];
    }
    __builtin_amdgcn_wave_barrier();
}

// Any head size: one workgroup per row, one wave per head, a lane every 64th value.  (The simple form, for caches without an operand
// layout and rotations that split a run of 4: 512 rows of 32 + 8 + 8 heads of 96 take 21 to 26 us.)
__global__ void __launch_bounds__(kThreads) quant_any_kernel(const NormRopeArgs a) {
    __shared__ double csd[kMaxRopeHalf], snd[kMaxRopeHalf];
    __shared__ float cs[kMaxRopeHalf], sn[kMaxRopeHalf];
    __shared__ double lines[kThreads / 64][kGenericMaxDim];
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int j = row - a.it[e].row0;
    for (int i = threadIdx.x; i < a.rot / 2; i += kThreads) {
        const double t = (a.it[e].rope0 + j) * a.turn[i];
        sincospif(2.f * static_cast<float>(t - rint(t)), &sn[i], &cs[i]);
        sincospi(2.0 * (t - rint(t)), &snd[i], &csd[i]);
    }
    __syncthreads();
    const int D = a.geom.head_dim, kvh = a.geom.kv_heads;
    const int pos = a.it[e].pos0 + j, slot = pos & (kPageTokens - 1);
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    uint8_t* const pool = static_cast<uint8_t*>(a.pool);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int NC = kGenericMaxDim / 64;
    for (int h = wave; h < a.heads + 2 * kvh; h += kThreads / 64) {
        const bool is_q = h < a.heads, is_v = h >= a.heads + kvh;
        if (is_q) {
            if (!a.q) continue;
            float y[NC];
            const long long at = static_cast<long long>(row) * a.q_stride + h * D;
#pragma unroll
            for (int c = 0; c < NC; ++c) y[c] = lane + 64 * c < D ? load_elem(a.q, a.act, at + lane + 64 * c) : 0.f;
            norm_rotate(y, lane, D, a.q_norm, a.eps, a.rot, cs, sn, reinterpret_cast<float*>(lines[wave]));
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (lane + 64 * c < D) store_elem(a.q_out, a.act, (static_cast<long long>(row) * a.heads + h) * D + lane + 64 * c, y[c]);
            continue;
        }
        const int hh = is_v ? h - a.heads - kvh : h - a.heads;
        const long long at = static_cast<long long>(row) * (is_v ? a.v_stride : a.k_stride) + hh * D;
        double y[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) y[c] = lane + 64 * c < D ? load_elem(is_v ? a.v : a.k, a.act, at + lane + 64 * c) : 0.f;
        if (!is_v) norm_rotate(y, lane, D, a.k_norm, a.eps, a.rot, csd, snd, lines[wave]);
        double top = 0.;
#pragma unroll
        for (int c = 0; c < NC; ++c) top = fabs(y[c]) < INFINITY ? fmax(top, fabs(y[c])) : top;
        const int ex = quant_exp(wave_max(top));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float x = quant_round(ldexp(y[c], -ex));
            if (lane + 64 * c < D) pool[a.geom.offset(phys, is_v, hh, slot, lane + 64 * c)] = quant4(x, 0.f, 0.f, 0.f) & 0xFF;
        }
        if (lane == 0) pool[a.geom.scale_offset(phys, is_v, hh, slot)] = ex + 127;
    }
}

// Rows back as values of a.act, any cache: a workgroup per row.  (Single elements: 16 sequences of 4096 rows of 8 heads, 8-bit heads of 96
// as bf16 302 MB in 182 to 194 us, bf16 heads of 128 as fp32 805 MB in 347, fp32 as bf16 in 329: 1.6 to 2.4 TB/s where the operand
// layout's kernel below reaches 4.5.  The cache's own type goes by pieces of 16 bytes.)
__global__ void __launch_bounds__(kThreads) read_as_any_kernel(const ReadArgs a) {
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int pos = a.it[e].pos0 + row - a.it[e].row0, slot = pos & (kPageTokens - 1);
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    const int D = a.geom.head_dim, width = a.geom.kv_heads * D;
    const uint8_t* const bytes = static_cast<const uint8_t*>(a.pool);
    for (int i = threadIdx.x; i < 2 * width; i += kThreads) {
        const int plane = i >= width, c = i - plane * width;
        const long long from = a.geom.offset(phys, plane, c / D, slot, c % D);
        const float x = a.geom.scaled() ? quant_value<0>(bytes[from]) * scale_of(bytes[a.geom.scale_offset(phys, plane, c / D, slot)])
                                      : load_elem(a.pool, a.dtype, from);
        store_out(plane ? a.v : a.k, a.act, static_cast<long long>(row) * width + c, x);
    }
}

// ---- head sizes 64 and 128 (the operand layout), rotations of whole runs of 8 values
// An item is 8 values of a head, two runs of 4: item j < rot / 8 holds the pairs 4 j .. 4 j + 3 (and rot / 2 further), the others 8
// values behind the rotated ones.  The items of a head are D / 8 lanes, so that its sum and its largest value are lane exchanges.
template <int T> struct Four {  // 4 consecutive values of dtype T, element-aligned
    typedef typename std::conditional<T == QR_DTYPE_F32, float, uint16_t>::type E;
    E v[4];
    __device__ __forceinline__ void load(const void* p, long long at) { __builtin_memcpy(v, static_cast<const E*>(p) + at, sizeof(v)); }
    __device__ __forceinline__ float operator[](int i) const {
        return T == QR_DTYPE_F32 ? v[i] : T == QR_DTYPE_BF16 ? bf16_bits_to_f32(v[i]) : f16_bits_to_f32(v[i]);
    }
};
template <int T> __device__ __forceinline__ void store_four(void* p, long long at, const float* x) {
    if (T == QR_DTYPE_F32) {
        __builtin_memcpy(static_cast<float*>(p) + at, x, 16);
    } else {
        uint16_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = f32_to_bits16(x[i], T);
        __builtin_memcpy(static_cast<uint16_t*>(p) + at, b, 8);
    }
}
// Over the LPH (8 or 16) lanes of a head.
template <int LPH> __device__ __forceinline__ double head_sum(double x) {
#pragma unroll
    for (int i = 1; i < LPH; i <<= 1) x += __shfl_xor(x, i);
    return x;
}
template <int LPH> __device__ __forceinline__ float head_max(float x) {
    x = fmaxf(x, dpp_xor1(x));
    x = fmaxf(x, dpp_xor2(x));
    x = fmaxf(x, dpp_half_mirror(x));
    return LPH == 16 ? fmaxf(x, dpp_mirror(x)) : x;
}
// The exponent of a head's values in 64 bits: the exponents of its lanes' largest, the largest of them (quant_exp ascends).
template <int LPH> __device__ __forceinline__ int head_exp(double top) {
    return __float_as_int(head_max<LPH>(__int_as_float(quant_exp(top) + 127))) - 127;  // (positive whole numbers order as floats do)
}
// A head's 8 values rotated; w: the norm's weights, or no norm.
template <class T, int LPH> __device__ __forceinline__ void norm_rotate8(T (&x)[8], bool norm, const float* w, int D, float eps, bool pair, const double* cs, const double* sn) {
    if (norm) {
        T ss = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
        if constexpr (sizeof(T) == 8) ss = head_sum<LPH>(ss);
        else ss = group_sum(ss, LPH);
        const T r = T(1) / sqrt(ss / static_cast<T>(D) + static_cast<T>(eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * static_cast<T>(w[i]);
    }
    if (pair) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const T lo = x[i], hi = x[i + 4], c = static_cast<T>(cs[i]), s = static_cast<T>(sn[i]);
            x[i] = lo * c - hi * s;
            x[i + 4] = lo * s + hi * c;
        }
    }
}
__device__ __forceinline__ float quant_unit(int ex) { return pow2f(-ex); }

// One workgroup per row and gridDim.y-th part of its heads (K, then q, then V unless it goes by runs), all loads of its items first.
// Bound by HBM, less what 64 bits cost: 5317 bf16 rows of 32 + 8 heads take 31 to 33 us for 104 MB, 3.2 TB/s where a copy reaches
// 4.8 (angles and rotation of K in 64 bits are 6 of them; sine and cosine by a table product in 64 bits were no faster).  Words of
// K at two places of the row cost a line of the page each, which the row's other heads fill.
template <int ACT, int D, int IPT>
__global__ void __launch_bounds__(kThreads) quant_kernel(const NormRopeArgs a, int v_heads) {
    constexpr int LPH = D / 8;
    __shared__ __attribute__((aligned(16))) double cs[D / 2], sn[D / 2];
    const int kv = a.geom.kv_heads;
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int j = row - a.it[e].row0, pos = a.it[e].pos0 + j, slot = pos & (kPageTokens - 1);
    const int qh = a.q ? a.heads : 0, heads = kv + qh + v_heads;
    const int li = threadIdx.x & (LPH - 1);
    const bool pair = 8 * li < a.rot;
    const int at_a = pair ? 4 * li : 8 * li, at_b = pair ? at_a + a.rot / 2 : at_a + 4;
    const int h0 = blockIdx.y * (kThreads / LPH * IPT) + threadIdx.x / LPH;
    constexpr int es = ACT == QR_DTYPE_F32 ? 4 : 2;
    const char* const rows[3] = {static_cast<const char*>(a.k) + row * a.k_stride * es, static_cast<const char*>(a.q) + row * a.q_stride * es,
                                 static_cast<const char*>(a.v) + row * a.v_stride * es};
    Four<ACT> ra[IPT], rb[IPT];
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
        const int h = min(h0 + kThreads / LPH * k, heads - 1);
        const bool is_k = h < kv, is_q = !is_k && h < kv + qh;
        const long long at = static_cast<long long>(is_k ? h : is_q ? h - kv : h - kv - qh) * D;
        const char* src = is_k ? rows[0] : is_q ? rows[1] : rows[2];
        ra[k].load(src, at + at_a);
        rb[k].load(src, at + at_b);
    }
    for (int i = threadIdx.x; i < a.rot / 2; i += kThreads) {
        const double t = (a.it[e].rope0 + j) * a.turn[i];
        sincospi(2.0 * (t - rint(t)), &sn[i], &cs[i]);
    }
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    float w[2][8];  // of K heads, of q heads
    const bool kn = a.k_norm, qn = a.q_norm;
    if (kn) {
        __builtin_memcpy(w[0], a.k_norm + at_a, 16);
        __builtin_memcpy(w[0] + 4, a.k_norm + at_b, 16);
    }
    if (qn) {
        __builtin_memcpy(w[1], a.q_norm + at_a, 16);
        __builtin_memcpy(w[1] + 4, a.q_norm + at_b, 16);
    }
    __syncthreads();
    uint8_t* const pool = static_cast<uint8_t*>(a.pool);
    const int ci = pair ? at_a : 0;
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
        const int h = h0 + kThreads / LPH * k;
        const bool is_k = h < kv, is_q = !is_k && h < kv + qh;
        if (is_q) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = ra[k][i];
                x[i + 4] = rb[k][i];
            }
            norm_rotate8<float, LPH>(x, qn, w[1], D, a.eps, pair, cs + ci, sn + ci);
            // (q_out may be q: the loads of every item that a workgroup stores stand before the barrier)
            const long long at = (static_cast<long long>(row) * a.heads + h - kv) * D;
            store_four<ACT>(a.q_out, at + at_a, x);
            store_four<ACT>(a.q_out, at + at_b, x + 4);
            continue;
        }
        if (h >= heads) continue;
        const int hh = is_k ? h : h - kv - qh;
        double x[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = ra[k][i];
            x[i + 4] = rb[k][i];
        }
        if (is_k) norm_rotate8<double, LPH>(x, kn, w[0], D, a.eps, pair, cs + ci, sn + ci);
        double top = 0.;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fabs(x[i]) < INFINITY ? fmax(top, fabs(x[i])) : top;
        const int ex = head_exp<LPH>(top);
        const double unit = quant_unit(ex);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = quant_round(x[i] * unit);
        const uint32_t c[2] = {quant4(y[0], y[1], y[2], y[3]), quant4(y[4], y[5], y[6], y[7])};
        if (is_k) {
            *reinterpret_cast<uint32_t*>(pool + a.geom.offset(phys, 0, hh, slot, at_a)) = c[0];
            *reinterpret_cast<uint32_t*>(pool + a.geom.offset(phys, 0, hh, slot, at_b)) = c[1];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                pool[a.geom.offset(phys, 1, hh, slot, (i < 4 ? at_a : at_b - 4) + i)] = static_cast<uint8_t>(c[i >> 2] >> (8 * (i & 3)));
        }
        if (li == 0) pool[a.geom.scale_offset(phys, !is_k, hh, slot)] = ex + 127;
    }
}

// Bytes of four words as four words of their i-th bytes.
__device__ __forceinline__ void transpose4(const uint32_t (&x)[4], uint32_t (&y)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602);
    const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
    y[0] = __builtin_amdgcn_perm(c, a, 0x05040100);
    y[1] = __builtin_amdgcn_perm(c, a, 0x07060302);
    y[2] = __builtin_amdgcn_perm(d, b, 0x05040100);
    y[3] = __builtin_amdgcn_perm(d, b, 0x07060302);
}

// V by runs of 16 slots, which are 16 bytes of a dim in the page: a workgroup takes a run of 256 / (D / 8) heads' rows, 8 values
// per thread, and hands the codes through LDS to threads of 4 dims each.  Slots outside the chunk are left alone.  As part of
// quant_kernel it wrote single bytes: a line of the page for each (16 sequences of one row: 7 us, where a second launch would be 4 more;
// 5317 rows: these 16 MB take 9 us).
template <int ACT, int D>
__global__ void __launch_bounds__(kThreads) quant_v_kernel(const NormRopeArgs a) {
    constexpr int LPH = D / 8, GROUPS = kThreads / LPH / 16;  // (run, head) pairs of a workgroup
    __shared__ uint32_t codes[GROUPS][16][D / 4 + 1];
    const int e = batch_find(a.n, blockIdx.x, [&](int i) { return a.it[i].unit0; });
    const NormRopeItem it = a.it[e];
    const int kv = a.geom.kv_heads, runs = ((it.pos0 + it.rows - 1) >> 4) - (it.pos0 >> 4) + 1;
    const int u0 = (static_cast<int>(blockIdx.x) - it.unit0) * GROUPS;
    uint8_t* const pool = static_cast<uint8_t*>(a.pool);
    {
        const int gr = threadIdx.x / (16 * LPH), t = threadIdx.x / LPH & 15, li = threadIdx.x & (LPH - 1);
        const int u = min(u0 + gr, runs * kv - 1), kvh = u % kv, p = (((it.pos0 >> 4) + u / kv) << 4) + t, j = p - it.pos0;
        const long long at = static_cast<long long>(it.row0 + min(max(j, 0), it.rows - 1)) * a.v_stride + kvh * D + 8 * li;
        Four<ACT> ra, rb;
        ra.load(a.v, at);
        rb.load(a.v, at + 4);
        float x[8], top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = ra[i];
            x[i + 4] = rb[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fabsf(x[i]) < INFINITY ? fmaxf(top, fabsf(x[i])) : top;
        const int ex = quant_exp(head_max<LPH>(top));
        const float unit = quant_unit(ex);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = quant_clamp(x[i] * unit);
        codes[gr][t][2 * li] = quant4(x[0], x[1], x[2], x[3]);
        codes[gr][t][2 * li + 1] = quant4(x[4], x[5], x[6], x[7]);
        if (li == 0 && j >= 0 && j < it.rows && u0 + gr < runs * kv) {
            const long long phys = a.page_table[it.pt_off + (p >> kPageShift)];
            pool[a.geom.scale_offset(phys, 1, kvh, p & (kPageTokens - 1))] = ex + 127;
        }
    }
    __syncthreads();
    const int gr = threadIdx.x / (D / 4), n = threadIdx.x % (D / 4), u = u0 + gr;  // dims 4 n .. 4 n + 3
    if (gr >= GROUPS || u >= runs * kv) return;
    const int kvh = u % kv, p0 = ((it.pos0 >> 4) + u / kv) << 4;
    const long long phys = a.page_table[it.pt_off + (p0 >> kPageShift)];
    uint8_t* const o = pool + a.geom.offset(phys, 1, kvh, p0 & (kPageTokens - 1), 4 * n);  // (dims are 16 bytes apart)
    uint32_t y[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t x[4], z[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) x[t] = codes[gr][4 * i + t][n];
        transpose4(x, z);
#pragma unroll
        for (int d = 0; d < 4; ++d) y[d][i] = z[d];
    }
    if (p0 >= it.pos0 && p0 + 16 <= it.pos0 + it.rows) {
#pragma unroll
        for (int d = 0; d < 4; ++d) *reinterpret_cast<uint4*>(o + 16 * d) = make_uint4(y[d][0], y[d][1], y[d][2], y[d][3]);
    } else {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int t = 0; t < 16; ++t)
                if (p0 + t >= it.pos0 && p0 + t < it.pos0 + it.rows) o[16 * d + t] = static_cast<uint8_t>(y[d][t >> 2] >> (8 * (t & 3)));
    }
}

// 8 codes of a scale as 8 values of dtype T at o (element-aligned).
template <int T> __device__ __forceinline__ void widen8(uint32_t lo, uint32_t hi, float scale, void* o) {
    if constexpr (T == QR_DTYPE_BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 y[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
                             __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)};
        __builtin_memcpy(o, y, 16);
    } else {
        const float x[8] = {quant_value<0>(lo) * scale, quant_value<1>(lo) * scale, quant_value<2>(lo) * scale, quant_value<3>(lo) * scale,
                            quant_value<0>(hi) * scale, quant_value<1>(hi) * scale, quant_value<2>(hi) * scale, quant_value<3>(hi) * scale};
        if constexpr (T == QR_DTYPE_F32) {
            __builtin_memcpy(o, x, 32);
        } else {
            uint16_t b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = f32_to_out16(x[i], T);
            __builtin_memcpy(o, b, 16);
        }
    }
}

// Rows of the 8-bit operand layout back as values: a workgroup takes 128 slots of a kv head, K by 16 dims of a slot per thread (the
// D / 16 threads of a slot beside each other: whole lines of the page, whole rows of the output), V by 8 dims of 8 slots, whose
// codes are transposed in registers.  Bound by HBM, two thirds of it writes: 808 MB in 165 to 178 us, 4.5 to 4.9
// TB/s (a copy: 4.8); with 8-byte stores 221.
constexpr int kReadRun = 128;
template <int T, int D>
__global__ void __launch_bounds__(kThreads) read_as_kernel(const ReadArgs a) {
    typedef typename std::conditional<T == QR_DTYPE_F32, float, uint16_t>::type E;
    constexpr int P = D / 16, KP = kReadRun * P / kThreads;  // pieces of a slot; of K per thread
    static_assert(kReadRun / 8 * (D / 8) <= kThreads, "threads that take V");
    const int e = batch_find(a.n, blockIdx.x, [&](int i) { return a.it[i].unit0; });
    const ReadItem it = a.it[e];
    const int kv = a.geom.kv_heads, u = blockIdx.x - it.unit0, kvh = u % kv;
    const int p0 = ((it.pos0 >> 7) + u / kv) << 7, s0 = p0 & (kPageTokens - 1);
    const long long phys = a.page_table[it.pt_off + (p0 >> kPageShift)];
    const uint8_t* const page = static_cast<const uint8_t*>(a.pool) + phys * a.geom.page_elems();
    const uint8_t* const k = page + (static_cast<long long>(kvh) * kPageTokens + s0) * D;
    const uint8_t* const v = k + a.geom.plane_elems();
    const uint8_t* const scales = page + 2 * a.geom.plane_elems() + kvh * kPageTokens + s0;
    const int end = it.pos0 + it.rows;
    auto row = [&](void* to, int t) __attribute__((always_inline)) {
        return static_cast<E*>(to) + (static_cast<long long>(it.row0 + p0 + t - it.pos0) * kv + kvh) * D;
    };
    uint4 kc[KP];
    uint32_t ks[KP];
    int kt[KP];
    const int piece = threadIdx.x % P;  // dims 16 piece ..
#pragma unroll
    for (int c = 0; c < KP; ++c) {
        const int x = threadIdx.x / P + kThreads / P * c, m = x & 31;  // step x / 32, row m of it
        kt[c] = 32 * (x >> 5) + 16 * (m >> 2 & 1) + 8 * (m >> 4) + 4 * (m >> 3 & 1) + (m & 3);
        if (p0 + kt[c] >= it.pos0 && p0 + kt[c] < end) {
            kc[c] = *reinterpret_cast<const uint4*>(k + (x >> 5) * 32 * D + 1024 * (piece >> 1) + 16 * (32 * (piece & 1) + m));
            ks[c] = scales[kt[c]];
        }
    }
    const int run = threadIdx.x / (D / 8), n = threadIdx.x % (D / 8);  // slots 8 run .., dims 8 n ..
    const bool takes = run < kReadRun / 8 && p0 + 8 * run < end && p0 + 8 * run + 8 > it.pos0;
    uint2 vc[8], vs;
    if (takes) {
        const uint8_t* b = v + (run >> 2) * 32 * D + 1024 * (n >> 2) + 16 * (32 * (run >> 1 & 1) + 8 * (n & 3)) + 8 * (run & 1);
#pragma unroll
        for (int d = 0; d < 8; ++d) vc[d] = *reinterpret_cast<const uint2*>(b + 16 * d);
        vs = *reinterpret_cast<const uint2*>(scales + kv * kPageTokens + 8 * run);
    }
#pragma unroll
    for (int c = 0; c < KP; ++c) {
        if (p0 + kt[c] < it.pos0 || p0 + kt[c] >= end) continue;
        E* o = row(a.k, kt[c]) + 16 * piece;
        const float scale = scale_of(ks[c]);
        widen8<T>(kc[c].x, kc[c].y, scale, o);
        widen8<T>(kc[c].z, kc[c].w, scale, o + 8);
    }
    if (!takes) return;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t lo[4] = {i ? vc[0].y : vc[0].x, i ? vc[1].y : vc[1].x, i ? vc[2].y : vc[2].x, i ? vc[3].y : vc[3].x};
        const uint32_t hi[4] = {i ? vc[4].y : vc[4].x, i ? vc[5].y : vc[5].x, i ? vc[6].y : vc[6].x, i ? vc[7].y : vc[7].x};
        uint32_t y[4], z[4];
        transpose4(lo, y);
        transpose4(hi, z);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int p = p0 + 8 * run + 4 * i + t;
            const float scale = scale_of((i ? vs.y : vs.x) >> (8 * t) & 0xFF);
            if (p >= it.pos0 && p < end) widen8<T>(y[t], z[t], scale, row(a.v, 8 * run + 4 * i + t) + 8 * n);
        }
    }
}

template <int ACT, int D> void launch_rows(NormRopeArgs& a, hipStream_t s) {
    constexpr int LPH = D / 8, GROUPS = kThreads / LPH / 16;
    // V goes by runs of 16 slots unless the chunks have few rows: single bytes otherwise, but one launch
    const bool runs = a.rows >= 4 * a.n;
    if (runs) {
        int groups = 0;
        for (int i = 0; i < a.n; ++i) {
            const int n = ((a.it[i].pos0 + a.it[i].rows - 1) >> 4) - (a.it[i].pos0 >> 4) + 1;
            a.it[i].unit0 = groups;
            groups += (n * a.geom.kv_heads + GROUPS - 1) / GROUPS;
        }
        hipLaunchKernelGGL((quant_v_kernel<ACT, D>), dim3(groups), dim3(kThreads), 0, s, a);
    }
    const int v_heads = runs ? 0 : a.geom.kv_heads, heads = a.geom.kv_heads + (a.q ? a.heads : 0) + v_heads;
    const int turns = (heads * LPH + kThreads - 1) / kThreads, ipt = std::min(turns, 4);
    const dim3 grid(a.rows, (turns + ipt - 1) / ipt);
    if (ipt == 1) hipLaunchKernelGGL((quant_kernel<ACT, D, 1>), grid, dim3(kThreads), 0, s, a, v_heads);
    else if (ipt == 2) hipLaunchKernelGGL((quant_kernel<ACT, D, 2>), grid, dim3(kThreads), 0, s, a, v_heads);
    else if (ipt == 3) hipLaunchKernelGGL((quant_kernel<ACT, D, 3>), grid, dim3(kThreads), 0, s, a, v_heads);
    else hipLaunchKernelGGL((quant_kernel<ACT, D, 4>), grid, dim3(kThreads), 0, s, a, v_heads);
}
template <int ACT> void launch_act(NormRopeArgs& a, hipStream_t s) {
    if (a.geom.head_dim == 128) launch_rows<ACT, 128>(a, s);
    else launch_rows<ACT, 64>(a, s);
}
template <int T> void launch_read_type(const ReadArgs& a, int groups, hipStream_t s) {
    if (a.geom.head_dim == 128) hipLaunchKernelGGL((read_as_kernel<T, 128>), dim3(groups), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((read_as_kernel<T, 64>), dim3(groups), dim3(kThreads), 0, s, a);
}

}  // namespace

hipError_t launch_quant(NormRopeArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (!(a.geom.mfma_layout & 1) || a.rot % 8) hipLaunchKernelGGL(quant_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
    else if (a.act == QR_DTYPE_F32) launch_act<QR_DTYPE_F32>(a, stream);
    else if (a.act == QR_DTYPE_F16) launch_act<QR_DTYPE_F16>(a, stream);
    else launch_act<QR_DTYPE_BF16>(a, stream);
    return hipGetLastError();
}

hipError_t launch_read_as(ReadArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    if (a.geom.mfma_layout != 3) {
        hipLaunchKernelGGL(read_as_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    int groups = 0;
    for (int i = 0; i < a.n; ++i) {
        a.it[i].unit0 = groups;
        groups += (((a.it[i].pos0 + a.it[i].rows - 1) >> 7) - (a.it[i].pos0 >> 7) + 1) * a.geom.kv_heads;
    }
    if (a.act == QR_DTYPE_F32) launch_read_type<QR_DTYPE_F32>(a, groups, stream);
    else if (a.act == QR_DTYPE_F16) launch_read_type<QR_DTYPE_F16>(a, groups, stream);
    else launch_read_type<QR_DTYPE_BF16>(a, groups, stream);
    return hipGetLastError();
}

}  // namespace qr
