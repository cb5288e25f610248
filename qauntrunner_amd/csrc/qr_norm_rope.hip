// qr_norm_rope.hip -- append of chunks of several sequences with a norm over each query and key
// head and the rotation in the same pass, and reading cache rows back, gfx950.
//
// A row x of D values (one head of q or k): y = x w / sqrt(mean(x^2) + eps), then the pairs
// (i, i + R/2), i < R/2, of its first R values turn by the angle p theta^(-2i/R).  K and V go to
// the row's page slot, q to q_out.
//
// Norm sums and products are fp32, one rounding when a value is stored.  The angle is a product in
// 64 bits, reduced to a fraction of a turn before it becomes fp32: at position 131072 an fp32
// product is off by 2^-8 of a radian.
#include "qr_batch.hpp"

namespace qr {
namespace {

constexpr int kThreads = 256;

// cos and sin of the row's angles, computed once per workgroup
__device__ __forceinline__ void angles(const NormRopeArgs& a, int pos, float* cs, float* sn) {
    for (int i = threadIdx.x; i < a.rot / 2; i += kThreads) {
        const double t = pos * a.turn[i];
        sincospif(2.f * static_cast<float>(t - rint(t)), &sn[i], &cs[i]);
    }
}

// Any head size: one workgroup per row, one wave per head, a lane every 64th value.
__global__ void __launch_bounds__(kThreads) norm_rope_any_kernel(const NormRopeArgs a) {
    __shared__ float cs[kMaxRopeHalf], sn[kMaxRopeHalf];
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int j = row - a.it[e].row0;
    angles(a, a.it[e].rope0 + j, cs, sn);
    __syncthreads();
    const int D = a.geom.head_dim, half = a.rot >> 1, kvh = a.geom.kv_heads;
    const int pos = a.it[e].pos0 + j, slot = pos & (kPageTokens - 1);
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    const int lane = threadIdx.x & 63;
    for (int h = threadIdx.x >> 6; h < a.heads + 2 * kvh; h += kThreads / 64) {
        const bool is_q = h < a.heads, is_v = h >= a.heads + kvh;
        if (is_q && !a.q) continue;
        const void* src = is_q ? a.q : is_v ? a.v : a.k;
        const int hh = is_q ? h : is_v ? h - a.heads - kvh : h - a.heads;
        const long long at = static_cast<long long>(row) * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + hh * D;
        const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        float y[kGenericMaxDim / 64];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < kGenericMaxDim / 64; ++c) {
            const int i = lane + 64 * c;
            y[c] = i < D ? load_elem(src, a.act, at + i) : 0.f;
            ss = fmaf(y[c], y[c], ss);
        }
        float r = 1.f;
        if (w) {
            ss = sum_xor32(sum_xor16(group_sum(ss, 16)));
            r = 1.f / sqrtf(ss / static_cast<float>(D) + a.eps);
        }
#pragma unroll
        for (int c = 0; c < kGenericMaxDim / 64; ++c) {
            const int i = lane + 64 * c;
            if (i >= D) continue;
            if (w) y[c] = y[c] * r * w[i];
            if (i < a.rot && !is_v) {
                const int o = i < half ? i + half : i - half;  // the pair's other value
                float x = load_elem(src, a.act, at + o);
                if (w) x = x * r * w[o];
                y[c] = i < half ? y[c] * cs[i] - x * sn[i] : x * sn[o] + y[c] * cs[o];
            }
        }
        // every load of the head stands before its stores: q_out may be q
#pragma unroll
        for (int c = 0; c < kGenericMaxDim / 64; ++c) {
            const int i = lane + 64 * c;
            if (i >= D) continue;
            if (is_q) store_elem(a.q_out, a.act, (static_cast<long long>(row) * a.heads + hh) * D + i, y[c]);
            else store_elem(a.pool, a.dtype, a.geom.offset(phys, is_v, hh, slot, i), y[c]);
        }
    }
}

__global__ void __launch_bounds__(kThreads) read_any_kernel(const ReadArgs a) {
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int pos = a.it[e].pos0 + row - a.it[e].row0;
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    const int D = a.geom.head_dim, width = a.geom.kv_heads * D;
    for (int i = threadIdx.x; i < 2 * width; i += kThreads) {
        const int plane = i >= width, c = i - plane * width;
        const long long from = a.geom.offset(phys, plane, c / D, pos & (kPageTokens - 1), c % D);
        const long long to = static_cast<long long>(row) * width + c;
        void* out = plane ? a.v : a.k;
        if (a.dtype == QR_DTYPE_F32) static_cast<float*>(out)[to] = static_cast<const float*>(a.pool)[from];
        else static_cast<uint16_t*>(out)[to] = static_cast<const uint16_t*>(a.pool)[from];
    }
}

}  // namespace

hipError_t launch_norm_rope(const NormRopeArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    hipLaunchKernelGGL(norm_rope_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_read(const ReadArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    hipLaunchKernelGGL(read_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace qr
