// qr_forms.hpp -- attention of chunks of several sequences in the forms of qr_attn_form (capped scores, a slope over the
// distance, windows, document and prefix masks) and behind prefixes that several chunks share.
//
// A chunk's rows attend one or two lists of keys: its own sequence's and its prefix's.  A list and the rows that read it
// are an item: all rows of a run of chunks with one prefix against the prefix, or one chunk's rows against its own keys.
// An item's rows are cut into blocks, a block's keys into parts; a part leaves (m, l, o) of each row -- the largest score,
// the sum of e^(z - m) and the values weighed by it -- unless it is the row's only one, and a last kernel joins a row's
// parts over both lists: out = sum o e^(m - M) / sum l e^(m - M), M the largest m.
#pragma once

#include <algorithm>

#include "qr_batch.hpp"

namespace qr {

// Kernels of a launch.
enum FormKind { kFormAny, kFormStream, kFormTilesHalf, kFormTiles, kFormF32Half, kFormF32, kFormKinds };
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

// Partials of a launch, at most (64 bf16 sequences of 8 rows behind 65536 positions would have more); a row alone may have more yet.
constexpr long long kFormPartialBytes = 256LL << 20;
__host__ __device__ constexpr long long form_partial_bytes(int head_dim) { return 4LL * head_dim + 8; }
// Rows behind prefixes that a launch takes: one part of either list for each takes half of these bytes.
constexpr int form_rows_behind(int heads, int head_dim) {
    const long long n = kFormPartialBytes / 2 / (2 * form_partial_bytes(head_dim) * heads);
    return n < 1 ? 1 : static_cast<int>(n);
}

// Whether some row of a chunk sees its prefix: its first, at position p0, sees the most of it.
inline bool form_sees_prefix(int pre_len, int p0, int first, int window) {
    return pre_len > std::max(first, window ? p0 - window + 1 : 0);
}

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
    int unit0, blocks;
    int splits;              // parts of the block that has the most
    int per;                 // tiles of a part, up to; 0: every block has `splits` parts
    int part0;               // part of a row that a block's first one is
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
    float us[kFormItems];    // of an item's longest unit, by the plan
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
// fp32 tiles (kinds kFormF32Half, kFormF32): head sizes 64, 96, 128 and 256 of rows in order in the page, whole groups.
hipError_t launch_forms_f32(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_f16(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_bf16(const FormsK& k, int units, hipStream_t s);
hipError_t launch_forms_e4m3(const FormsK& k, int units, hipStream_t s);

// (query, head) rows of a block and slots of a tile of each kernel.
__host__ __device__ constexpr int form_rows(int kind) {
    return kind == kFormAny ? kFormAnyRows : kind == kFormTiles ? 128 : kind == kFormTilesHalf ? 64 : kind == kFormF32Half ? 16 : 32;
}
__host__ __device__ constexpr int form_tile(int kind) {
    return kind == kFormTiles || kind == kFormTilesHalf ? 64 : kind == kFormF32Half || kind == kFormF32 ? 16 : 32;
}

// Row `row` of a chunk: its position, and the slots lo .. hi of `keys` slots from position `base` on that it sees (lo > hi: none).
struct FormSpan {
    int chunk;
    int pos;
    int lo, hi;
};
__host__ __device__ inline FormSpan form_span(const FormRows& r, int row, int window, int base, int keys) {
    const int pos = r.p0 + row - r.row0;
    const int from = window && pos - window + 1 > r.first ? pos - window + 1 : r.first;
    const int to = pos > r.full - 1 ? pos : r.full - 1;
    const int lo = from > base ? from - base : 0, hi = to - base < keys - 1 ? to - base : keys - 1;
    return {0, pos, lo, hi};
}
// Parts of a block's keys (of an item of one chunk, g query heads per kv head): what the last and first of its rows see, a rule that
// the host's count of units and the kernels share.
__host__ __device__ inline int form_parts(const FormItem& it, const FormRows& r, int window, int g, int rows, int tile, int block) {
    if (!it.per) return it.splits;
    const int end = (block + 1) * rows < it.rows * g ? (block + 1) * rows : it.rows * g;
    const FormSpan a = form_span(r, it.row0 + block * rows / g, window, it.base, it.keys);
    const FormSpan b = form_span(r, it.row0 + (end - 1) / g, window, it.base, it.keys);
    const int lo = a.lo < b.lo ? a.lo : b.lo, hi = a.hi > b.hi ? a.hi : b.hi;
    const int n = hi < lo ? 1 : (hi / tile - lo / tile + it.per) / it.per;
    return n < it.splits ? n : it.splits;
}

// A unit of an item: kv heads fastest (an XCD keeps few of them in its L2), from the last block, which sees the most keys, down.
struct FormUnit {
    int kvh, block, part, parts;
};
__device__ __forceinline__ FormUnit form_unit(const FormsK& p, const FormItem& it, int g, int rows, int tile, int unit) {
    const int kv = p.geom.kv_heads, kvh = unit % kv;
    int u = unit / kv;
    if (!it.per || it.splits == 1) {
        const int b = u / it.splits;
        return {kvh, it.blocks - 1 - b, u - b * it.splits, it.splits};
    }
    const FormRows r = p.c[it.c0];
    const int lane = threadIdx.x & 63;
    for (int b0 = it.blocks - 1;; b0 -= 64) {  // 64 blocks at a time, a running sum of their parts over the lanes
        const int n = b0 - lane >= 0 ? form_parts(it, r, p.window, g, rows, tile, b0 - lane) : 0;
        int sum = n;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
            const int o = __shfl_up(sum, x);
            sum += lane >= x ? o : 0;
        }
        const int all = __builtin_amdgcn_readfirstlane(__shfl(sum, 63));
        if (u < all || b0 < 64) {
            const int l = __builtin_amdgcn_readfirstlane(static_cast<int>(__popcll(__builtin_amdgcn_ballot_w64(sum <= u))));
            return {kvh, b0 - l, __builtin_amdgcn_readfirstlane(u - __shfl(sum - n, l)), __builtin_amdgcn_readfirstlane(__shfl(n, l))};
        }
        u -= all;
    }
}

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

// Row j of an item.
__device__ __forceinline__ FormSpan form_row(const FormsK& p, const FormItem& it, int j) {
    const int row = it.row0 + j;
    if (it.nc == 1) {  // (scalar loads)
        FormSpan s = form_span(p.c[it.c0], row, p.window, it.base, it.keys);
        s.chunk = it.c0;
        return s;
    }
    int c = it.c0;
    for (int i = 1; i < it.nc; ++i) c += p.c[it.c0 + i].row0 <= row;
    FormSpan s = form_span(p.c[c], row, p.window, it.base, it.keys);
    s.chunk = c;
    return s;
}

// A block of one part whose rows have no other list needs no partials: it writes the output, and marks the rows' first partial.
__device__ __forceinline__ bool form_whole(const FormRows& c, const FormItem& it, int parts) { return parts == 1 && c.parts == it.splits; }
constexpr float kFormDone = -1.f;  // a sum that no part has

// (m, l) of a row's part; the last of a block's parts fills those that its rows have and it has not.
__device__ __forceinline__ void form_store_ml(const FormsK& p, const FormRows& c, const FormItem& it, long long slot, const FormUnit& u, float m, float l) {
    if (c.parts == 1) return;
    p.part_ml[slot] = form_whole(c, it, u.parts) ? make_float2(0.f, kFormDone) : make_float2(m, l);
    if (u.part == u.parts - 1)
        for (int x = u.parts; x < it.splits; ++x) p.part_ml[slot + x - u.part] = make_float2(-INFINITY, 0.f);
}

// What a part's sums add to the whole: an infinite one shows however little the part weighs.
template <class V> __device__ __forceinline__ V form_weighed(V o, float w) {
    V x = o * w;
    if constexpr (std::is_same<V, float>::value) return x == x ? x : o;
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = x[i] == x[i] ? x[i] : o[i];
        return x;
    }
}

// A score in log2 units capped and less its slope: cap tanh(z / cap) = cap (1 - 2 / (e^(2 z / cap) + 1)).
__device__ __forceinline__ float form_score(float z, float cap, float slope, float away) {
    if (cap > 0.f) z = cap * tanhf(z / cap);
    return slope != 0.f ? fmaf(-slope, fabsf(away), z) : z;
}
constexpr float kLog2e = 1.4426950408889634f;

enum FormScores { kScoresPlain, kScoresSlope, kScoresCap, kScoresBoth };

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
