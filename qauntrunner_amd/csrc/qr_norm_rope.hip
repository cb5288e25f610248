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

#include <algorithm>
#include <type_traits>

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

// ---- head sizes of whole runs of 8 values (and rotations of as many)
// An item is 8 values of a head, two runs of 4: item j < R/8 holds the pairs 4j .. 4j + 3 (and R/2 further), the others 8
// values behind the rotated ones.  The items of a head lie in LPH = 2^n lanes, so that its sum is a lane exchange; a
// thread's items are the same values of several heads, which share the norm's weights.
struct Item {
    int a, b;  // first values of its two runs
    bool pair;
};
__device__ __forceinline__ Item item_of(int j, int rot) {
    if (8 * j < rot) return {4 * j, 4 * j + rot / 2, true};
    return {8 * j, 8 * j + 4, false};
}
template <int T> struct Run {  // 4 consecutive values of dtype T, element-aligned
    typedef typename std::conditional<T == QR_DTYPE_F32, float, uint16_t>::type E;
    E v[4];
    __device__ __forceinline__ void load(const void* p, long long at) { __builtin_memcpy(v, static_cast<const E*>(p) + at, sizeof(v)); }
    __device__ __forceinline__ void widen(float (&x)[8], int o) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[o + i] = T == QR_DTYPE_F32 ? v[i] : T == QR_DTYPE_BF16 ? bf16_bits_to_f32(v[i]) : f16_bits_to_f32(v[i]);
    }
};
// 4 values to p[at .. at + 3], element-aligned
template <int T> __device__ __forceinline__ void store_run(void* p, long long at, const float* x) {
    if (T == QR_DTYPE_F32) {
        __builtin_memcpy(static_cast<float*>(p) + at, x, 16);
    } else {
        uint16_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = f32_to_bits16(x[i], T);
        __builtin_memcpy(static_cast<uint16_t*>(p) + at, b, 8);
    }
}

// V rows of the MFMA page layout, where 8 aligned slots of a dim are 16 bytes: a thread takes 8 dims of such a run, 8 loads
// of 8 values and 8 stores of 16 bytes, 128 bytes in a row of the page.  Slots outside the chunk are left alone.  5317 rows
// of 8 heads of 128: 11 us for 21.8 MB read and written, 1.9 TB/s: one round of 332 workgroups, each its loads and
// then its stores.
template <int ACT, int DT>
__global__ void __launch_bounds__(kThreads) v_runs_kernel(const NormRopeArgs a) {
    const int e = batch_find(a.n, blockIdx.x, [&](int i) { return a.it[i].unit0; });
    const NormRopeItem it = a.it[e];
    const int per = a.geom.head_dim / 8, slices = a.geom.kv_heads * per;
    const int runs = ((it.pos0 + it.rows - 1) >> 3) - (it.pos0 >> 3) + 1;
    const int u = (static_cast<int>(blockIdx.x) - it.unit0) * kThreads + threadIdx.x;
    if (u >= runs * slices) return;
    const int slice = u % slices, kvh = slice / per, d0 = 8 * (slice - kvh * per);
    const int p0 = ((it.pos0 >> 3) + u / slices) << 3;  // position of the run's first slot
    Run<ACT> x[8][2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int j = min(max(p0 + k - it.pos0, 0), it.rows - 1);
        const long long at = static_cast<long long>(it.row0 + j) * a.v_stride + slice * 8;
        x[k][0].load(a.v, at);
        x[k][1].load(a.v, at + 4);
    }
    const long long phys = a.page_table[it.pt_off + (p0 >> kPageShift)];
    float y[8][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        x[k][0].widen(y[k], 0);
        x[k][1].widen(y[k], 4);
    }
    const bool whole = p0 >= it.pos0 && p0 + 8 <= it.pos0 + it.rows;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        uint16_t b[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) b[k] = f32_to_bits16(y[k][d], DT);
        uint16_t* o = static_cast<uint16_t*>(a.pool) + a.geom.offset(phys, 1, kvh, p0 & (kPageTokens - 1), d0 + d);
        if (whole) {
            uint4 w;
            __builtin_memcpy(&w, b, 16);
            *reinterpret_cast<uint4*>(o) = w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (p0 + k >= it.pos0 && p0 + k < it.pos0 + it.rows) o[k] = b[k];
        }
    }
}

// One workgroup per row and gridDim.y-th part of its heads (K, then q, then V unless it goes by runs).  The loads of all of
// a thread's items are issued before the angles are computed.  Bound by HBM, for few rows by the launch: four bf16 prompts
// of 32 / 8 heads (q and K: 109 MB read and written) 31 us, 3.5 TB/s, of which the norms take 2 and the 16-byte pieces of K 6; runs of 8
// values or workgroups of several rows are no faster, 16-bit types that the kernel is not compiled for cost 8.
template <int ACT, int DT, int IPT>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRopeArgs a, int lph, int v_heads) {
    __shared__ __attribute__((aligned(16))) float cs[kMaxRopeHalf], sn[kMaxRopeHalf];
    const int D = a.geom.head_dim, kv = a.geom.kv_heads, per = D / 8;
    const int row = blockIdx.x;
    const int e = batch_find(a.n, row, [&](int i) { return a.it[i].row0; });
    const int j = row - a.it[e].row0, pos = a.it[e].pos0 + j, slot = pos & (kPageTokens - 1);
    const int qh = a.q ? a.heads : 0, heads = kv + qh + v_heads;
    const int li = threadIdx.x & (lph - 1);  // item within its head
    const bool in = li < per;
    const Item im = item_of(in ? li : 0, a.rot);
    const int h0 = blockIdx.y * (kThreads / lph * IPT) + threadIdx.x / lph;
    constexpr int es = ACT == QR_DTYPE_F32 ? 4 : 2;
    const char* const rows[3] = {static_cast<const char*>(a.k) + row * a.k_stride * es, static_cast<const char*>(a.q) + row * a.q_stride * es,
                                 static_cast<const char*>(a.v) + row * a.v_stride * es};
    Run<ACT> ra[IPT], rb[IPT];
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
        const int h = min(h0 + kThreads / lph * k, heads - 1);
        const bool is_k = h < kv, is_q = !is_k && h < kv + qh;
        const long long at = static_cast<long long>(is_k ? h : is_q ? h - kv : h - kv - qh) * D;
        const char* src = is_k ? rows[0] : is_q ? rows[1] : rows[2];
        ra[k].load(src, at + im.a);
        rb[k].load(src, at + im.b);
    }
    angles(a, a.it[e].rope0 + j, cs, sn);
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    float w[2][8];  // of K heads, of q heads
    const bool kn = a.k_norm, qn = a.q_norm;
    if (kn) {
        __builtin_memcpy(w[0], a.k_norm + im.a, 16);
        __builtin_memcpy(w[0] + 4, a.k_norm + im.b, 16);
    }
    if (qn) {
        __builtin_memcpy(w[1], a.q_norm + im.a, 16);
        __builtin_memcpy(w[1] + 4, a.q_norm + im.b, 16);
    }
    __syncthreads();
    float c4[4] = {1.f, 1.f, 1.f, 1.f}, s4[4] = {0.f, 0.f, 0.f, 0.f};
    if (im.pair) {
        __builtin_memcpy(c4, cs + im.a, 16);
        __builtin_memcpy(s4, sn + im.a, 16);
    }
#pragma unroll
    for (int k = 0; k < IPT; ++k) {
        const int h = h0 + kThreads / lph * k;
        const bool is_k = h < kv, is_q = !is_k && h < kv + qh;
        float x[8];
        ra[k].widen(x, 0);
        rb[k].widen(x, 4);
        if (is_k || is_q) {
            if (is_k ? kn : qn) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
                ss = group_sum(in ? ss : 0.f, lph);
                if (lph == 64) ss = sum_xor32(ss);
                const float r = 1.f / sqrtf(ss / static_cast<float>(D) + a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (is_k ? w[0][i] : w[1][i]);
            }
            if (im.pair) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float lo = x[i], hi = x[i + 4];
                    x[i] = lo * c4[i] - hi * s4[i];
                    x[i + 4] = lo * s4[i] + hi * c4[i];
                }
            }
        }
        if (!in || h >= heads) continue;
        // (q_out may be q: the loads of every item that a workgroup stores stand before the barrier)
        if (is_q) {
            const long long at = (static_cast<long long>(row) * a.heads + h - kv) * D;
            store_run<ACT>(a.q_out, at + im.a, x);
            store_run<ACT>(a.q_out, at + im.b, x + 4);
        } else if (is_k || !a.geom.mfma_layout) {
            const int hh = is_k ? h : h - kv - qh;
            store_run<DT>(a.pool, a.geom.offset(phys, !is_k, hh, slot, im.a), x);
            store_run<DT>(a.pool, a.geom.offset(phys, !is_k, hh, slot, im.b), x + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                store_elem(a.pool, DT, a.geom.offset(phys, 1, h - kv - qh, slot, (i < 4 ? im.a : im.b - 4) + i), x[i]);
        }
    }
}

// Rows back, head sizes whose rows are whole 16-byte pieces: a thread per piece; V of the MFMA page layout a thread per 8
// dims of a run of 8 slots (128 bytes of the page), the first v_groups workgroups.  Bound by HBM: 519 MB read and written
// in 125 us.
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a, int v_groups) {
    const int D = a.geom.head_dim, kv = a.geom.kv_heads;
    if (static_cast<int>(blockIdx.x) < v_groups) {
        const int e = batch_find(a.n, blockIdx.x, [&](int i) { return a.it[i].unit0; });
        const ReadItem it = a.it[e];
        const int per = D / 8, slices = kv * per, runs = ((it.pos0 + it.rows - 1) >> 3) - (it.pos0 >> 3) + 1;
        const int u = (static_cast<int>(blockIdx.x) - it.unit0) * kThreads + threadIdx.x;
        if (u >= runs * slices) return;
        const int run = u / slices, slice = u % slices;
        const int p0 = ((it.pos0 >> 3) + run) << 3;
        const long long phys = a.page_table[it.pt_off + (p0 >> kPageShift)];
        const uint16_t* src = static_cast<const uint16_t*>(a.pool) + a.geom.offset(phys, 1, slice / per, p0 & (kPageTokens - 1), 8 * (slice % per));
        uint16_t x[8][8];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + 8 * d);
            __builtin_memcpy(x[d], &w, 16);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (p0 + k < it.pos0 || p0 + k >= it.pos0 + it.rows) continue;
            uint16_t y[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) y[d] = x[d][k];
            __builtin_memcpy(static_cast<uint16_t*>(a.v) + static_cast<long long>(it.row0 + p0 + k - it.pos0) * kv * D + 8 * slice, y, 16);
        }
        return;
    }
    const int es = dtype_size(a.dtype), n = 16 / es, per = D / n, pieces = kv * per;  // of a row
    const int planes = v_groups ? 1 : 2;
    const long long u = (static_cast<long long>(blockIdx.x) - v_groups) * kThreads + threadIdx.x;
    const int row = min(static_cast<int>(u / (planes * pieces)), a.rows - 1);
    // the rows of a wave lie in one chunk or a few: each thread looks its own up
    int e = 0;
    for (int i = 1; i < a.n; ++i) e += a.it[i].row0 <= row;
    if (u >= static_cast<long long>(a.rows) * planes * pieces) return;
    const int c = static_cast<int>(u - static_cast<long long>(row) * planes * pieces), plane = c >= pieces, x = c - plane * pieces;
    const int pos = a.it[e].pos0 + row - a.it[e].row0;
    const long long phys = a.page_table[a.it[e].pt_off + (pos >> kPageShift)];
    const long long from = a.geom.offset(phys, plane, x / per, pos & (kPageTokens - 1), n * (x % per));
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.pool) + from * es);
    __builtin_memcpy(static_cast<char*>(plane ? a.v : a.k) + (static_cast<long long>(row) * pieces + x) * 16, &w, 16);
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


// V of the MFMA layout goes by runs of 8 slots unless the chunks have few rows: 2 bytes per store otherwise, but one
// launch of one workgroup per row.
template <class Args> int v_run_groups(Args& a) {
    if (!a.geom.mfma_layout || a.rows < 4 * a.n) return 0;
    int groups = 0;
    for (int i = 0; i < a.n; ++i) {
        const long long runs = ((a.it[i].pos0 + a.it[i].rows - 1) >> 3) - (a.it[i].pos0 >> 3) + 1;
        a.it[i].unit0 = groups;
        groups += static_cast<int>((runs * a.geom.kv_heads * (a.geom.head_dim / 8) + kThreads - 1) / kThreads);
    }
    return groups;
}

template <int ACT, int DT> void launch_runs(const NormRopeArgs& a, int v_groups, int lph, hipStream_t s) {
    if (DT != QR_DTYPE_F32 && v_groups) hipLaunchKernelGGL((v_runs_kernel<ACT, DT == QR_DTYPE_F32 ? QR_DTYPE_F16 : DT>), dim3(v_groups), dim3(kThreads), 0, s, a);
    const int v_heads = v_groups ? 0 : a.geom.kv_heads, heads = a.geom.kv_heads + (a.q ? a.heads : 0) + v_heads;
    const int slots = (heads * lph + kThreads - 1) / kThreads, ipt = std::min(slots, 4);
    const dim3 grid(a.rows, (slots + ipt - 1) / ipt);
    if (ipt == 1) hipLaunchKernelGGL((norm_rope_kernel<ACT, DT, 1>), grid, dim3(kThreads), 0, s, a, lph, v_heads);
    else if (ipt == 2) hipLaunchKernelGGL((norm_rope_kernel<ACT, DT, 2>), grid, dim3(kThreads), 0, s, a, lph, v_heads);
    else if (ipt == 3) hipLaunchKernelGGL((norm_rope_kernel<ACT, DT, 3>), grid, dim3(kThreads), 0, s, a, lph, v_heads);
    else hipLaunchKernelGGL((norm_rope_kernel<ACT, DT, 4>), grid, dim3(kThreads), 0, s, a, lph, v_heads);
}
template <int ACT> void launch_dtype(const NormRopeArgs& a, int v_groups, int lph, hipStream_t s) {
    if (a.dtype == QR_DTYPE_F32) launch_runs<ACT, QR_DTYPE_F32>(a, v_groups, lph, s);
    else if (a.dtype == QR_DTYPE_F16) launch_runs<ACT, QR_DTYPE_F16>(a, v_groups, lph, s);
    else launch_runs<ACT, QR_DTYPE_BF16>(a, v_groups, lph, s);
}

}  // namespace

hipError_t launch_norm_rope(NormRopeArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    const int D = a.geom.head_dim;
    if (D % 8 || a.rot % 8) {
        hipLaunchKernelGGL(norm_rope_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    int lph = 1;
    while (lph < D / 8) lph *= 2;
    const int v_groups = v_run_groups(a);
    if (a.act == QR_DTYPE_F32) launch_dtype<QR_DTYPE_F32>(a, v_groups, lph, stream);
    else if (a.act == QR_DTYPE_F16) launch_dtype<QR_DTYPE_F16>(a, v_groups, lph, stream);
    else launch_dtype<QR_DTYPE_BF16>(a, v_groups, lph, stream);
    return hipGetLastError();
}

hipError_t launch_read(ReadArgs& a, hipStream_t stream) {
    if (!a.rows) return hipSuccess;
    const int n = 16 / dtype_size(a.dtype);
    if (a.geom.head_dim % n) {
        hipLaunchKernelGGL(read_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    const int v_groups = v_run_groups(a);
    if (a.geom.mfma_layout && !v_groups) {
        hipLaunchKernelGGL(read_any_kernel, dim3(a.rows), dim3(kThreads), 0, stream, a);
        return hipGetLastError();
    }
    const long long pieces = static_cast<long long>(a.rows) * (v_groups ? 1 : 2) * a.geom.kv_heads * (a.geom.head_dim / n);
    hipLaunchKernelGGL(read_kernel, dim3(v_groups + static_cast<unsigned>((pieces + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, a, v_groups);
    return hipGetLastError();
}

}  // namespace qr
