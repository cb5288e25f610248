// qr_chunks.hpp -- what the kernels of attention over chunks of several sequences share.
#pragma once

#include <algorithm>

#include "qr_batch.hpp"

namespace qr {

// Kernels of a launch; rows (query, query head pairs of a kv head) of a workgroup, positions of a tile.
enum ChunkKind { kChunkAny, kChunkStream32, kChunkStream, kChunkTile, kChunkF32Half, kChunkF32, kChunkKinds };
// The passes after the attention that add up the weights.
enum ChunkWeights { kWeightsAny, kWeightsScores, kWeightsTile, kWeightsF32, kWeightsKinds };

constexpr int kChunkAnyRows = 8, kChunkAnyTile = 32;
// Parts of the cache's 16-bit type that the streaming kernel takes a query value and a weight as: queries of another type
// keep 24 bits in three of bf16, 22 in two of fp16 (of values within 2^-16 of a row's largest; fp16 ends below).
constexpr int chunk_parts(int cache, bool other) { return !other ? 1 : cache == QR_DTYPE_BF16 ? 3 : 2; }
struct ChunksK {
    ChunkItem it[kBatch];
    int n;
    int units;
    bool paired;             // (tile kernels) fewer units than run at once
    const char* pool;
    const int* page_table;
    PageGeom geom;
    int dtype;               // cache
    int act;                 // q and out
    int heads;
    const void* q;           // [rows][heads][head_dim]
    void* out;
    float* weights;          // [sequences][kv_heads][max_seq]
    int max_seq;
    float qscale;            // scale log2(e): scores are in log2 units
    float* part_acc;         // [slots][head_dim]
    float2* part_ml;         // [slots] (maximum, sum)
    float2* row_ml;          // [rows * heads] (maximum, sum), null where no weights are wanted
    float* row_scale;        // [rows * heads] log2 units per score where q was scaled by a power of two, else null
    float* scores;           // scaled scores of the chunks whose weights pass reads them, else null
    float* wpart;            // partial sums of weights: [split][kv head][length] of a chunk from slot0 on
};

// Query heads h0 .. h0 + g - 1 read kv head kvh (head h reads h * kv_heads / heads).
__device__ __forceinline__ void chunk_heads(const ChunksK& p, int kvh, int* h0, int* g) {
    const int kv = p.geom.kv_heads;
    *h0 = (kvh * p.heads + kv - 1) / kv;
    *g = ((kvh + 1) * p.heads + kv - 1) / kv - *h0;
}

// Launch slot b of the tile kernels runs on XCD b % 8.  Where the kv heads divide among the XCDs, one takes all units of a
// kv head (or every 8 / kv_heads-th of them): its K/V stays in one L2 and every XCD has the same share of every chunk.
// p.units: units of one kv head, the largest chunks' first.
__device__ __forceinline__ bool chunk_unit(const ChunksK& p, int* kvh, int* unit) {
    const int kv = p.geom.kv_heads, b = blockIdx.x, x = b & 7, j = b >> 3;
    if (kv % 8 == 0) {
        *kvh = x + 8 * (j / p.units);
        *unit = j % p.units;
    } else if (8 % kv == 0) {
        *kvh = x % kv;
        *unit = j * (8 / kv) + x / kv;
    } else {
        *kvh = b % kv;
        *unit = b / kv;
    }
    if (*unit >= p.units || *kvh >= kv) return false;
    // all units run at once, several on a CU: the long ones share it with short ones (512 fp32 rows after 1536: 161 us, 166
    // from the longest down)
    const int h = (p.units + 1) >> 1;
    if (p.paired && *unit >= h) *unit = p.units - 1 - (*unit - h);
    return true;
}
inline int chunk_grid(const ChunksK& p) {
    const int kv = p.geom.kv_heads;
    return kv % 8 && 8 % kv == 0 ? 8 * ((p.units * kv + 7) / 8) : p.units * kv;
}

// The tile kernels' row blocks: a block's keys are split into parts of up to `per` tiles, so that late blocks, which see
// more keys, have more units.
struct KeyTiles {
    int rows, tile;  // (query, head) rows of a block, positions of a tile
    __host__ __device__ int blocks(const ChunkItem& it, int g) const { return (it.rows * g + rows - 1) / rows; }
    __host__ __device__ int tiles(const ChunkItem& it, int g, int block) const {
        const int r0 = block * rows, left = it.rows * g - r0, last = r0 + (left < rows ? left : rows) - 1;
        return (it.pos0 + last / g + tile) / tile;
    }
    __host__ __device__ int parts(const ChunkItem& it, int g, int block, int per) const { return (tiles(it, g, block) + per - 1) / per; }
    long long units(const ChunkItem& it, int g, int per) const {  // of a kv head
        long long u = 0;
        for (int b = 0; b < blocks(it, g); ++b) u += parts(it, g, b, per);
        return u;
    }
    // from the last block, which has the most keys, down; sets it.parts.  (Without divisions in the loop: 40 blocks
    // would cost a unit several microseconds.)
    __device__ __forceinline__ void find(ChunkItem& it, int g, int unit, int* block, int* part) const {
        int b = blocks(it, g) - 1, s = it.splits;
        if (s == 1) {
            b -= unit;
            unit = 0;
        } else if (unit >= s) {
            unit -= s;
            const int end = b * rows - 1, step = rows / g, over = rows - step * g;
            int query = end / g, head = end - query * g;  // of the last row of block b - 1
            for (--b;; --b) {
                const int n = (it.pos0 + query + tile) / tile;
                while ((s - 1) * it.per >= n) --s;
                if (unit < s) break;
                unit -= s;
                query -= step;
                head -= over;
                if (head < 0) {
                    head += g;
                    --query;
                }
            }
        }
        *block = b;
        *part = unit;
        it.parts = s;
    }
};
constexpr KeyTiles kKeyTiles16{256, 64};
__host__ __device__ constexpr KeyTiles key_tiles32(int g) { return {64 / g * g, 32}; }  // whole queries

// The weights passes by tiles: a unit takes the rows of a block of positions that see part of it, in rounds, up to `per`
// of them.  Rows before the block see none of it, so later blocks have fewer units.
struct WeightTiles {
    int positions, rows;  // of a block, of a round
    __host__ __device__ int first(const ChunkItem& it, int g, int block) const {
        const int b0 = block * positions;
        return b0 > it.pos0 ? (b0 - it.pos0) * g : 0;
    }
    __host__ __device__ int rounds(const ChunkItem& it, int g, int block) const { return (it.rows * g - first(it, g, block) + rows - 1) / rows; }
    __host__ __device__ int parts(const ChunkItem& it, int g, int block, int per) const { return (rounds(it, g, block) + per - 1) / per; }
    __host__ __device__ int blocks(const ChunkItem& it) const { return (it.pos0 + it.rows + positions - 1) / positions; }
    __host__ __device__ int whole(const ChunkItem& it) const {  // blocks that every row sees
        const int n = it.pos0 / positions + 1, m = blocks(it);
        return n < m ? n : m;
    }
    // units of a kv head
    long long units(const ChunkItem& it, int g, int per) const {
        long long u = static_cast<long long>(whole(it)) * parts(it, g, 0, per);
        for (int b = whole(it); b < blocks(it); ++b) u += parts(it, g, b, per);
        return u;
    }
    __device__ __forceinline__ void find(const ChunkItem& it, int g, int unit, int* block, int* part, int* n) const {
        const int s0 = parts(it, g, 0, it.per), n0 = whole(it);
        if (unit < n0 * s0) {
            *block = unit / s0;
            *part = unit - *block * s0;
            *n = s0;
            return;
        }
        unit -= n0 * s0;
        int b = n0, s = s0;
        for (;; ++b) {
            const int n = rounds(it, g, b);
            while ((s - 1) * it.per >= n) --s;
            if (unit < s) break;
            unit -= s;
        }
        *block = b;
        *part = unit;
        *n = s;
    }
};
constexpr WeightTiles kWeightTiles16{256, 128}, kWeightTiles32{128, 16};

// Part `split` of the positions [0, keys) in whole tiles.
__device__ __forceinline__ void chunk_keys(const ChunkItem& it, int keys, int split, int tile, int* t0, int* t1) {
    const int tiles = (keys + tile - 1) / tile;
    *t0 = static_cast<int>(static_cast<long long>(tiles) * split / it.parts) * tile;
    *t1 = std::min(static_cast<int>(static_cast<long long>(tiles) * (split + 1) / it.parts) * tile, keys);
}

// Entries of a row of scores: positions of the chunk's last row, whole runs of 8.
__host__ __device__ inline int chunk_score_len(const ChunkItem& it) { return (it.pos0 + it.rows + 7) & ~7; }

hipError_t launch_chunks_any(const ChunksK& k, hipStream_t s);
hipError_t launch_chunks_any_weights(const ChunksK& k, hipStream_t s);
// 16-bit caches in the MFMA page layout, whole groups: kinds kChunkStream32 (up to 32 rows), kChunkStream (up to 128), kChunkTile; kChunkKinds:
// the weights pass.
hipError_t launch_chunks_tile(const ChunksK& k, int kind, hipStream_t s);
// fp32 tiles: kinds kChunkF32Half (32 rows), kChunkF32 (64 rows); kChunkKinds: the weights pass.
bool chunks_f32_takes(int dtype, int head_dim, int heads, int kv_heads);
int chunks_f32_per_cu(int dtype, int head_dim, bool half);  // resident workgroups
hipError_t launch_chunks_f32(const ChunksK& k, int kind, hipStream_t s);

}  // namespace qr
