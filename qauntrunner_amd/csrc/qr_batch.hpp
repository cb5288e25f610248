// qr_batch.hpp -- launch interfaces of the calls over chunks of several sequences: append with
// query / key norms and rotation, causal attention with the weight that each cached position
// received, eviction by that weight, and reading rows back.
//
// A call's chunks are described by value (no copy to the device, so a call can be captured), up to
// kBatch of them per launch; the host drops chunks without rows.  Work is counted in units, the
// chunks' one after another: unit0 is a chunk's first.
#pragma once

#include "qr_kernels.hpp"

namespace qr {

constexpr int kBatch = 64;  // one lane each: a unit's chunk is found by one ballot

// Chunk of a unit: the last one whose first unit is not past it.  `first(i)` of i < n ascends.
template <class F> __device__ __forceinline__ int batch_find(int n, int unit, F first) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < n && first(lane < n ? lane : 0) <= unit;
    return __builtin_amdgcn_readfirstlane(static_cast<int>(__popcll(__builtin_amdgcn_ballot_w64(at))) - 1);
}

// One element of a dtype at p[i], widened; NaN stays NaN when one is stored.
__device__ __forceinline__ float load_elem(const void* p, int dtype, long long i) {
    if (dtype == QR_DTYPE_F32) return static_cast<const float*>(p)[i];
    const uint16_t u = static_cast<const uint16_t*>(p)[i];
    return dtype == QR_DTYPE_F16 ? f16_bits_to_f32(u) : bf16_bits_to_f32(u);
}
// (fp16: f32_to_f16_bits_ref without its branches; below 2^-14 both round to nearest even)
__device__ __forceinline__ uint16_t f32_to_bits16(float x, int dtype) {
    if (dtype == QR_DTYPE_F16) {
        const uint32_t b = __float_as_uint(x), a = b & 0x7FFFFFFFu;
        const uint32_t normal = min((a - 0x37FFF000u) >> 13, 0x7C00u), small = __half_as_ushort(__float2half(__uint_as_float(a)));
        return static_cast<uint16_t>((b >> 16 & 0x8000u) | (a > 0x7F800000u ? 0x7E00u : a < 0x38800000u ? small : normal));
    }
    uint16_t u;
    const __bf16 y = static_cast<__bf16>(x);  // (nearest even)
    __builtin_memcpy(&u, &y, 2);
    return u;
}
__device__ __forceinline__ void store_elem(void* p, int dtype, long long i, float x) {
    if (dtype == QR_DTYPE_F32) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = f32_to_bits16(x, dtype);
}

// An output of attention: rounded to nearest even, NaN stays NaN.
__device__ __forceinline__ uint16_t f32_to_out16(float x, int dtype) {
    return dtype == QR_DTYPE_F16 ? __half_as_ushort(__float2half(x)) : f32_to_bits16(x, dtype);
}
__device__ __forceinline__ void store_out(void* p, int dtype, long long i, float x) {
    if (dtype == QR_DTYPE_F32) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = f32_to_out16(x, dtype);
}

// Values of V at dim d that are not finite: the first positions in [t0, t1) of each sort, INT_MAX where there is none.  Whole
// runs of 8 slots are read (16 bytes in the MFMA layout), which lie in held pages where t0 and t1 do.
struct NotFinite {
    int plus, minus, nan;
    // what a sum over positions below `end` is that meets them with weights above zero; `sum` without any
    __device__ __forceinline__ float settle(int end, float sum) const {
        const bool p = plus < end, m = minus < end;
        return nan < end || (p && m) ? NAN : p ? INFINITY : m ? -INFINITY : sum;
    }
    __device__ __forceinline__ NotFinite of_lane(int lane) const { return {__shfl(plus, lane), __shfl(minus, lane), __shfl(nan, lane)}; }
};
__device__ __forceinline__ NotFinite find_not_finite(const void* pool, const int* pages, const PageGeom& geom, int dtype, int kvh, int d, int t0, int t1) {
    NotFinite f{0x7FFFFFFF, 0x7FFFFFFF, 0x7FFFFFFF};
    for (int t = t0 & ~7; t < t1; t += 8) {
        const long long at = geom.offset(pages[t >> kPageShift], 1, kvh, t & (kPageTokens - 1), d);
        float v[8];
        if (geom.mfma_layout) {
            uint16_t u[8];
            __builtin_memcpy(u, static_cast<const uint16_t*>(pool) + at, 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = dtype == QR_DTYPE_F16 ? f16_bits_to_f32(u[i]) : bf16_bits_to_f32(u[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = load_elem(pool, dtype, at + i * geom.head_dim);
        }
#pragma unroll
        for (int i = 7; i >= 0; --i) {
            if (fabsf(v[i]) < INFINITY || t + i < t0 || t + i >= t1) continue;
            if (v[i] != v[i]) f.nan = min(f.nan, t + i);
            else if (v[i] > 0.f) f.plus = min(f.plus, t + i);
            else f.minus = min(f.minus, t + i);
        }
    }
    return f;
}

// ------------------------------------------------------------------ append
struct NormRopeItem {
    int pt_off;  // page-table row of (sequence, layer)
    int pos0;    // slot of the first row
    int rows;
    int row0;    // first row in q / k / v
    int rope0;   // position that the first row is rotated by
    int unit0;
};
struct NormRopeArgs {
    NormRopeItem it[kBatch];
    int n;
    int rows;                // rows of all chunks
    void* pool;
    const int* page_table;
    PageGeom geom;
    int dtype;               // cache
    int act;                 // q / k / v
    int heads;
    const void *q, *k, *v;   // q may be null
    long long q_stride, k_stride, v_stride;  // elements between rows
    void* q_out;             // [rows][heads * head_dim]
    const float *q_norm, *k_norm;            // [head_dim]; null: no norm
    float eps;
    int rot;                 // rotated dims, even
    double turn[kMaxRopeHalf];               // revolutions per position of pair i
};
hipError_t launch_norm_rope(NormRopeArgs& a, hipStream_t stream);  // sets unit0
hipError_t launch_quant(NormRopeArgs& a, hipStream_t stream);      // the same on an 8-bit cache

// ------------------------------------------------------------------ rows back
struct ReadItem {
    int pt_off, pos0, rows, row0;
    int unit0;
};
struct ReadArgs {
    ReadItem it[kBatch];
    int n;
    int rows;
    const void* pool;
    const int* page_table;
    PageGeom geom;
    int dtype;
    int act;                 // of k and v where they are values of another type (launch_read_as)
    void *k, *v;             // [rows][kv_heads * head_dim] in the cache's type
};
hipError_t launch_read(ReadArgs& a, hipStream_t stream);     // sets unit0
hipError_t launch_read_as(ReadArgs& a, hipStream_t stream);  // any cache, values of a.act

// ------------------------------------------------------------------ attention
struct ChunkItem {
    int pt_off;
    int seq;                 // row of the weights
    int pos0;
    int rows;
    int row0;                // first row in q / out
    // of a launch:
    int unit0;
    int blocks;              // row blocks per kv head (weights: position blocks); of the tile kernels units
    int splits;              // parts of a block's keys, of the tile kernels of the block that has the most
    int slot0;               // first split partial: (row * heads + head) * splits + split from here
    int per;                 // tile kernels: tiles of keys (weights: rounds of rows) of a unit, up to; else 0
    int parts;               // (within a kernel) of this block's keys; splits where all blocks have as many
    long long score0;        // first score: (row * heads + head) * chunk_score_len from here; -1: none are kept
};
struct ChunksArgs {
    ChunkItem it[kBatch];
    int n;
    int rows;                // rows of all chunks
    const void* pool;
    const int* page_table;
    PageGeom geom;
    int dtype;               // cache
    int act;                 // q and out
    int heads;
    const void* q;           // [rows][heads][head_dim]
    void* out;
    float* weights;          // [sequences][kv_heads][max_seq], may be null
    int max_seq;
    float scale;
};
// Which kernel takes a chunk, and how its work is cut.
struct ChunkPlanItem {
    int kind, blocks, splits, per;
    long long slot0;
    int wkind, wblocks, wper, wparts;
    long long wslot0, score0;
};
struct ChunksPlan {
    ChunkPlanItem it[kBatch];
    bool wmerge;             // some chunk's weights are summed in parts
    size_t part_ml, row_ml, row_scale, scores, wpart;  // offsets in the workspace; the partials' sums come first
    size_t workspace_bytes;
};
ChunksPlan plan_chunks(const ChunksArgs& a);
hipError_t launch_chunks(const ChunksArgs& a, const ChunksPlan& plan, void* workspace, hipStream_t stream);

// ------------------------------------------------------------------ eviction
struct EvictItem {
    int pt_off;
    int seq;
    int len;                 // positions held
    int entry;               // row of kept
};
struct EvictArgs {
    EvictItem it[kBatch];
    int n;
    void* pool;
    const int* page_table;
    PageGeom geom;
    int dtype;
    int first, heavy, recent;
    const float* weights;    // [sequences][kv_heads][max_seq]
    float* kept_weights;     // the same layout; may be weights
    int max_seq;
    int* kept;               // [entries][kv_heads][first + heavy + recent]
};
size_t evict_workspace_bytes(const EvictArgs& a);  // 0: it takes none
// workspace null: each row by one workgroup
hipError_t launch_evict(const EvictArgs& a, void* workspace, hipStream_t stream);

}  // namespace qr
