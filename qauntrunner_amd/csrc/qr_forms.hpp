// qr_forms.hpp -- attention of chunks of several sequences in the forms of qr_attn_form (capped scores, a slope over the
// distance, windows, document and prefix masks) and behind prefixes that several chunks share.
//
// A chunk's rows attend one or two lists of keys: its own sequence's and its prefix's.  A list and the rows that read it
// are an item: all rows of a run of chunks with one prefix against the prefix, or one chunk's rows against its own keys.
// An item's rows are cut into blocks, a block's keys into parts; a part leaves (m, l, o) of each row -- the largest score,
// the sum of e^(z - m) and the values weighed by it -- unless it is the row's only one, and a last kernel joins a row's
// parts over both lists: out = sum o e^(m - M) / sum l e^(m - M), M the largest m.
#pragma once

#include "qr_batch.hpp"

namespace qr {

// Kernels of a launch.
enum FormKind { kFormAny, kFormStream, kFormTiles, kFormF32Half, kFormF32, kFormKinds };
constexpr int kFormAnyRows = 8, kFormAnyTile = 32;

// What the host knows of a chunk.
struct FormChunk {
    int pt_off;              // page-table row of (sequence, layer)
    int pre_off;             // of its prefix
    int pre_len;             // 0: none
    int pos0, rows, row0;    // first slot; rows; first row in q / out
    int first, full;
};
struct FormsArgs {
    FormChunk c[kBatch];
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
    float scale, cap;
    const float* slopes;     // [heads], may be null
    int window;
};

// A chunk as the kernels see it.
struct FormRows {
    int row0, rows;
    int p0;                  // position of its first row
    int first, full;
    int parts;               // of a row, over both lists; 1: no partials
    long long slot0;         // first partial: (row * heads + head) * parts + part from here
};
// A list of keys and the rows that read it.
struct FormItem {
    int pt_off;
    int c0, nc;              // chunks
    int row0, rows;
    int base;                // position of slot 0
    int keys;                // slots
    int unit0, blocks, splits;
    int part0;               // part of a row that split 0 is
    int kind;
};
constexpr int kFormItems = 2 * kBatch;  // of a launch: a prefix and the own keys for each chunk
struct FormsK {
    FormItem it[kFormItems];
    FormRows c[kBatch];
    int n;                   // items of this launch
    int chunks;
    const char* pool;
    const int* page_table;
    PageGeom geom;
    int dtype, act, heads;
    const void* q;
    void* out;
    float qscale;            // scale log2(e): scores are in log2 units
    float cap;               // in log2 units; 0: none
    const float* slopes;
    int window;
    float* part_acc;         // [partials][head_dim]
    float2* part_ml;         // [partials] (maximum, sum)
};

// How a call's work is cut.
struct FormsPlan {
    FormItem it[kFormItems];
    int n;
    FormRows c[kBatch];
    size_t part_ml;          // offset in the workspace; the partials' sums come first
    size_t workspace_bytes;
    bool merge;
};
FormsPlan plan_forms(const FormsArgs& a);
hipError_t launch_forms(const FormsArgs& a, const FormsPlan& plan, void* workspace, hipStream_t stream);

hipError_t launch_forms_any(const FormsK& k, int units, hipStream_t s);
// MFMA tiles (kinds kFormStream, kFormTiles): operand page layouts, whole groups.
// fp32 tiles (kinds kFormF32Half, kFormF32): fp32 caches of head size 64 or 128, whole groups.
hipError_t launch_forms_f32(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_f16(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_bf16(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_e4m3(const FormsK& k, int units, hipStream_t s);

// Item of a unit.
__device__ __forceinline__ int form_find(const FormsK& p, int unit) {
    static_assert(kFormItems == 128, "two ballots");
    const int lane = threadIdx.x & 63;
    const bool a = lane < p.n && p.it[lane].unit0 <= unit, b = lane + 64 < p.n && p.it[lane + 64].unit0 <= unit;
    return __builtin_amdgcn_readfirstlane(static_cast<int>(__popcll(__builtin_amdgcn_ballot_w64(a)) + __popcll(__builtin_amdgcn_ballot_w64(b))) - 1);
}

// Query heads h0 .. h0 + g - 1 read kv head kvh (head h reads h * kv_heads / heads).
__device__ __forceinline__ void form_heads(const FormsK& p, int kvh, int* h0, int* g) {
    const int kv = p.geom.kv_heads;
    *h0 = (kvh * p.heads + kv - 1) / kv;
    *g = ((kvh + 1) * p.heads + kv - 1) / kv - *h0;
}

// Row j of an item: its position, and the slots lo .. hi of the item's keys that it sees (lo > hi: none).
struct FormSpan {
    int chunk;
    int pos;
    int lo, hi;
};
__host__ __device__ inline FormSpan form_span(const FormRows& r, int row, int window, int base, int keys) {
    const int pos = r.p0 + row - r.row0;
    const int from = window ? (pos - window + 1 > r.first ? pos - window + 1 : r.first) : r.first;
    const int to = pos > r.full - 1 ? pos : r.full - 1;
    const int lo = from > base ? from - base : 0, hi = to - base < keys - 1 ? to - base : keys - 1;
    return {0, pos, lo, hi};
}
__device__ __forceinline__ FormSpan form_row(const FormsK& p, const FormItem& it, int j) {
    const int row = it.row0 + j;
    int c = it.c0;
    for (int i = 1; i < it.nc; ++i) c += p.c[it.c0 + i].row0 <= row;
    FormSpan s = form_span(p.c[c], row, p.window, it.base, it.keys);
    s.chunk = c;
    return s;
}

// A score in log2 units capped and less its slope: cap tanh(z / cap) = cap (1 - 2 / (e^(2 z / cap) + 1)).
__device__ __forceinline__ float form_score(float z, float cap, float slope, float away) {
    if (cap > 0.f) z = cap * tanhf(z / cap);
    return slope != 0.f ? fmaf(-slope, fabsf(away), z) : z;
}
constexpr float kLog2e = 1.4426950408889634f;

enum FormScores { kScoresPlain, kScoresSlope, kScoresCap };  // (capped scores may have a slope too)

// Page of a slot, by a scalar load (no kernel writes the table while this one runs).
__device__ __forceinline__ int form_page(const FormsK& p, int pt_off, int t) {
    return reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p.page_table))[pt_off + (t >> kPageShift)];
}

// Slots that the rows of a block see: some row [lo, hi], every row [all_lo, all_hi].
struct FormRange {
    int lo, hi, all_lo, all_hi;
    __device__ __forceinline__ bool all(int t, int n) const { return t >= all_lo && t + n - 1 <= all_hi; }
};
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x = min(x, __shfl_xor(x, i));
    return x;
}
__device__ __forceinline__ int wave_max(int x) { return ~wave_min(~x); }

}  // namespace qr
