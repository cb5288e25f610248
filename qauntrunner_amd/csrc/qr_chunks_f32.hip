// qr_chunks_f32.hip -- causal attention of chunks of several sequences in fp32 arithmetic on fp32 MFMA
// tiles: fp32 caches (head size 64, 96, 128, 256) and 16-bit caches with token-major pages (96, 256),
// whole groups of up to 64 query heads, gfx950.  The tiles are those of one sequence's chunk
// (qr_chunk_f32.hpp, qr_chunk_f32.hip); here a workgroup finds its chunk first.  Bound by the fp32 MFMAs where
// the units are long (512 rows of 32 heads after 1536: 161 us, 93 TFLOP/s of the 154 that a large product reaches); three
// prompts of 61 to 501 rows, 3.8 GFLOP, take 64 us: a tile of a block takes 1.7 us and the longest unit has 14.
#include "qr_chunk_f32.hpp"
#include "qr_chunks.hpp"

namespace qr {
namespace {

template <typename ST, int D, int PG>
__global__ void __launch_bounds__(256, (F32Geom<ST, D>::wg_per_cu(PG))) chunks_f32_kernel(const ChunksK p) {
    __shared__ __attribute__((aligned(1024))) char lds[2][2 * F32Geom<ST, D>::KB];
    int kvh, unit;
    if (!chunk_unit(p, &kvh, &unit)) return;
    const int e = batch_find(p.n, unit, [&](int i) { return p.it[i].unit0; });
    ChunkItem it = p.it[e];
    const int g = p.heads / p.geom.kv_heads;
    int block, split;
    if (PG == 1) {
        key_tiles32(g).find(it, g, unit - it.unit0, &block, &split);
    } else {
        const int u = unit - it.unit0;
        split = u % it.splits;
        block = it.blocks - 1 - u / it.splits;
    }
    const long long row0 = static_cast<long long>(it.row0) * p.heads;
    ChunkF32K k{};
    k.pool = p.pool;
    k.page_table = p.page_table + it.pt_off;
    k.page_elems = p.geom.page_elems();
    k.plane_elems = p.geom.plane_elems();
    k.heads = p.heads;
    k.group = g;
    k.pos0 = it.pos0;
    k.nq = it.rows;
    k.q_dtype = k.out_dtype = p.act;
    k.q = static_cast<const char*>(p.q) + row0 * D * dtype_size(p.act);
    k.out = reinterpret_cast<float*>(static_cast<char*>(p.out) + row0 * D * dtype_size(p.act));
    k.part_acc = p.part_acc + static_cast<long long>(it.slot0) * D;
    k.part_ml = p.part_ml + it.slot0;
    k.qscale = p.qscale;
    k.queries_per_block = 64 / PG / k.group;
    k.splits = it.parts;
    k.stride = it.splits;
    k.row_ml = p.row_ml ? p.row_ml + row0 : nullptr;
    k.scores = p.scores && it.score0 >= 0 ? p.scores + it.score0 : nullptr;
    k.score_len = chunk_score_len(it);
    k.geom = p.geom;
    k.dtype = p.dtype;
    chunk_f32_tiles<ST, D, PG, true>(k, split, block, kvh, lds);
}

// Weights of 128 positions of one kv head over a part of its rows: a wave keeps the K rows of 32
// positions as operands (two M tiles) and takes the rows 16 at a time from LDS, where the workgroup
// puts them in operand order: chunk 4j + q4 of row l16 at 16 (64 j + lane).  Bound by the fp32
// MFMAs (2 D flop per score; the layouts of qr_chunk_f32.hpp): 34 us for three prompts' 1.9 GFLOP.
template <typename ST, int D>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) chunks_f32_weights_kernel(const ChunksK p) {
    using Gm = F32Geom<ST, D>;
    constexpr int EPC = Gm::EPC, NJ = Gm::NJ, NW = EPC / 4;  // fp32 16-byte chunks per cache chunk
    constexpr int QB = NJ * NW * 1024;                       // bytes of 16 rows
    __shared__ __attribute__((aligned(1024))) char lds[2][QB];
    __shared__ float4 info[2][16];                           // of the rows: maximum, 1 / sum, last position seen
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0;
    const int kvh = u / it.blocks, g = p.heads / p.geom.kv_heads, rows = it.rows * g;
    int split, block, splits;
    kWeightTiles32.find(it, g, u - kvh * it.blocks, &block, &split, &splits);
    const int lane = threadIdx.x & 63, q4 = lane >> 4, l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int len = it.pos0 + it.rows;
    const int b0 = block * kWeightTiles32.positions, t0 = b0 + 32 * wave;
    const int first = kWeightTiles32.first(it, g, block), rounds = kWeightTiles32.rounds(it, g, block);
    const int r0 = first + static_cast<int>(static_cast<long long>(rounds) * split / splits) * 16;
    const int r1 = min(rows, first + static_cast<int>(static_cast<long long>(rounds) * (split + 1) / splits) * 16);

    float kv[2][NJ][EPC];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        const int t = t0 + 16 * mt + l16;
        const long long phys = t0 < len ? p.page_table[it.pt_off + (t0 >> kPageShift)] : 0;  // 32 positions: one page
        const char* src = p.pool + (phys * p.geom.page_elems() + (static_cast<long long>(kvh) * kPageTokens + (t & (kPageTokens - 1))) * D) * Gm::ESZ;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            U32x4 c = {0, 0, 0, 0};
            if (t < len) c = load16(src + 16 * (4 * j + q4));
            Chunk<ST>::widen(c, kv[mt][j]);
        }
    }
    // a thread's share of 16 rows: fp32 chunks n = threadIdx.x + 256 c, of which lane n % 64's j = n / 64
    constexpr int CH = NJ * NW * 64, SHARE = (CH + 255) / 256;
    f32x4_t x[SHARE];
    float4 inf;
    auto fetch = [&](int r) __attribute__((always_inline)) {
        if (threadIdx.x < 16) {
            const int rho = r + static_cast<int>(threadIdx.x), rr = rho < r1 ? rho : rows - 1, query = rr / g;
            const float2 ml = p.row_ml[static_cast<long long>(it.row0 + query) * p.heads + kvh * g + rr - query * g];
            inf = make_float4(ml.x, 1.f / ml.y, __int_as_float(rho < r1 ? it.pos0 + query : -1), 0.f);
        }
#pragma unroll
        for (int c = 0; c < SHARE; ++c) {
            const int n = threadIdx.x + 256 * c, ln = n & 63, jw = n >> 6;
            if (n >= CH) break;
            const int rho = min(r + (ln & 15), rows - 1);
            const long long row = static_cast<long long>(it.row0 + rho / g) * p.heads + kvh * g + rho % g;
            const long long at = row * D + (4 * (jw / NW) + (ln >> 4)) * EPC + 4 * (jw % NW);
            if (p.act == QR_DTYPE_F32) {
                __builtin_memcpy(&x[c], static_cast<const float*>(p.q) + at, 16);
            } else {
                uint16_t h[4];
                __builtin_memcpy(h, static_cast<const uint16_t*>(p.q) + at, 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[c][i] = p.act == QR_DTYPE_BF16 ? bf16_bits_to_f32(h[i]) : f16_bits_to_f32(h[i]);
            }
        }
    };
    auto put = [&](int b) __attribute__((always_inline)) {
        char* const to = lds[b];
        if (threadIdx.x < 16) info[b][threadIdx.x] = inf;
#pragma unroll
        for (int c = 0; c < SHARE; ++c)
            if (CH % 256 == 0 || threadIdx.x + 256 * c < CH) *reinterpret_cast<f32x4_t*>(to + 16 * (threadIdx.x + 256 * c)) = x[c] * p.qscale;
    };
    float sum[2][4] = {};
    if (r0 < r1) {
        fetch(r0);
        put(0);
    }
    int at = 0;
    for (int r = r0; r < r1; r += 16, at ^= 1) {
        __syncthreads();
        const bool more = r + 16 < r1;
        if (more) fetch(r + 16);
        const float4 f = info[at][l16];
        f32x4_t s[2][2] = {};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            float q[EPC];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const f32x4_t v = *reinterpret_cast<const f32x4_t*>(lds[at] + 1024 * (j * NW + w) + 16 * lane);
#pragma unroll
                for (int i = 0; i < 4; ++i) q[4 * w + i] = v[i];
            }
#pragma unroll
            for (int i = 0; i < EPC; ++i)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
                    s[mt][j & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[mt][j][i], q[i], s[mt][j & 1], 0, 0, 0);
        }
        const int last = __float_as_int(f.z) - t0 - 4 * q4;  // of this lane's positions, the last the row sees
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (16 * mt + i <= last) sum[mt][i] = fmaf(fast_exp2(s[mt][0][i] + s[mt][1][i] - f.x), f.y, sum[mt][i]);
        if (more) put(at ^ 1);
    }
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float s = group_sum(sum[mt][i], 16);  // over the rows
            const int t = t0 + 16 * mt + 4 * q4 + i;
            if (l16 == 4 * mt + i && t < len) {
                if (splits == 1) p.weights[(static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t] += s;
                else p.wpart[it.slot0 + (static_cast<long long>(split) * p.geom.kv_heads + kvh) * len + t] = s;
            }
        }
}

template <typename ST, int D> hipError_t launch_st(const ChunksK& k, int kind, hipStream_t s) {
    const dim3 grid(chunk_grid(k));
    if (kind == kChunkF32Half) hipLaunchKernelGGL((chunks_f32_kernel<ST, D, 2>), grid, dim3(256), 0, s, k);
    else if (kind == kChunkF32) hipLaunchKernelGGL((chunks_f32_kernel<ST, D, 1>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((chunks_f32_weights_kernel<ST, D>), dim3(k.units), dim3(256), 0, s, k);
    return hipGetLastError();
}

}  // namespace

bool chunks_f32_takes(int dtype, int head_dim, int heads, int kv_heads) {
    if (heads % kv_heads || heads / kv_heads > 32) return false;
    return head_dim == 96 || head_dim == 256 || (dtype == QR_DTYPE_F32 && (head_dim == 64 || head_dim == 128));
}

int chunks_f32_per_cu(int dtype, int head_dim, bool half) {
    const int pg = half ? 2 : 1;
    if (dtype != QR_DTYPE_F32) return head_dim == 96 ? F32Geom<F16Tag, 96>::wg_per_cu(pg) : F32Geom<F16Tag, 256>::wg_per_cu(pg);
    return head_dim == 64 ? F32Geom<float, 64>::wg_per_cu(pg) : head_dim == 96 ? F32Geom<float, 96>::wg_per_cu(pg)
         : head_dim == 128 ? F32Geom<float, 128>::wg_per_cu(pg) : F32Geom<float, 256>::wg_per_cu(pg);
}

hipError_t launch_chunks_f32(const ChunksK& k, int kind, hipStream_t s) {
    const int D = k.geom.head_dim;
    if (k.dtype == QR_DTYPE_F32)
        return D == 64 ? launch_st<float, 64>(k, kind, s) : D == 96 ? launch_st<float, 96>(k, kind, s)
             : D == 128 ? launch_st<float, 128>(k, kind, s) : launch_st<float, 256>(k, kind, s);
    if (k.dtype == QR_DTYPE_BF16) return D == 96 ? launch_st<BF16Tag, 96>(k, kind, s) : launch_st<BF16Tag, 256>(k, kind, s);
    return D == 96 ? launch_st<F16Tag, 96>(k, kind, s) : launch_st<F16Tag, 256>(k, kind, s);
}

}  // namespace qr
