// qr_quant.hip -- append of chunks of several sequences to an 8-bit cache (query / key norms and rotation in the same
// pass, rows quantised as they are written) and reading rows back as values of 16 or 32 bits, gfx950.
//
// q is normed and rotated in 32 bits, as for the other caches.  k is rounded to 3 bits behind its first, and a value that
// 32 bits move across a border between two codes would be off by a whole code: its norm, angles and rotation are in 64
// bits.  v needs no arithmetic but the division by a power of two, which is exact.
#include "qr_quant.hpp"

#include <algorithm>

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

// Any head size: one workgroup per row, one wave per head, a lane every 64th value.
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

// Rows back as values of a.act, any cache: a workgroup per row.
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

}  // namespace

hipError_t launch_quant(NormRopeArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    hipLaunchKernelGGL(quant_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_read_as(ReadArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    hipLaunchKernelGGL(read_as_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qr
