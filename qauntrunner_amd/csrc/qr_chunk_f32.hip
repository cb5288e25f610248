// qr_chunk_f32.hip -- causal multi-query attention in fp32 arithmetic on fp32 MFMA tiles,
// gfx950: fp32 caches (head_dim 64, 96, 128, 256) and 16-bit caches whose pages are
// token-major (head_dim 96, 256), any whole group of up to 64 heads per kv head.
//
// Semantics as qr_chunk.hip: query i of the chunk sits at position pos0 + i and attends
// positions 0..pos0 + i (StreamingEngine.cs:831-836).  K, V, q and P all enter in fp32 and
// every product and sum is fp32, as in the decode kernels.
//
// Bound by the fp32 MFMA rate (v_mfma_f32_16x16x4_f32: 256 flop per clk and CU, 153 TFLOP/s in
// a large product).  As one decode entry per query, the path before, every query read its own
// K/V: 512 queries after 1536 positions (32 heads over 8 kv heads, head_dim 128, 15 GFLOP: 98 us
// at that rate) took 8 launches of 61 us, 506 us per call with the append; in two splits here 158
// (traced, which slows each: kernel 162, merge 7.5, append 6.6).  The matrix units are busy 77% of
// the cycles in which waves are resident (1.0 LDS conflict cycle per MFMA); the rest is the sums,
// the softmax and the tile barriers.
// Error against 64-bit results there: 2.9e-7 (decode entries 3.15e-7).
//
// A row is one (query, query head) pair.  Workgroup = 4 waves; the K/V tile of 32 positions is
// copied into LDS by buffer-load DMA (two stages) and serves 64 / PG rows:
//   PG = 1  each wave scores all 32 positions for its own 16 rows;
//   PG = 2  (few rows) two waves per 16 rows, one 16-position half of the tile each, merged
//           through LDS at the end.
// Layouts (checked on gfx950): A[m = lane%16][k = lane/16], B[k = lane/16][n = lane%16],
// D[m = 4(lane/16) + r][n = lane%16].
//   QK  S^T[pos][row]: lane (q4, l16) holds chunk 4j + q4 of K row l16 (A) and of q row l16 (B):
//       k-slot q4 of MFMA e is element e of that 16-byte chunk.  q stays in registers, scaled
//       by scale log2 e.
//   PV  O^T[dim][row]: lane quarter q4 holds the scores of positions 4q4 + r; step r takes
//       those four positions as its k-slots, so P enters from the lane's own registers.  A is
//       V row 4q4 + r, PE consecutive dims per lane: one LDS read feeds PE MFMAs.
// Sums are blocked, because an fp32 MFMA chain rounds at the size of its running sum (one chain
// over 512 positions: 9.5e-7 from 64-bit results where the decode entries have 3.1e-7).  A score is
// chains of two MFMAs (8 dims), added in pairs and then to the sum of the even or the odd steps;
// an output adds chains of two MFMAs (8 positions; four for 16-bit head_dim 256) in pairs before
// they go to the accumulator.  Distance from 64-bit results, decode entries and here: 3.15e-7 and
// 2.92e-7 at the shape above, 1.85e-7 and 1.84e-7 for 1000 queries from scratch (chains of four
// and eight MFMAs: 3.34e-7 and 2.25e-7; chains of one and two 2.90e-7 and 1.83e-7, 7% slower).
// 16-byte chunk c of an LDS row r sits at c ^ (r & SW): the 16 rows that a QK read takes lie a
// multiple of 128 bytes apart.
#include "qr_chunk.hpp"
#include "qr_chunk_f32.hpp"

#include <algorithm>

namespace qr {
namespace {

template <typename ST, int D, int PG>
__global__ void __launch_bounds__(256, (F32Geom<ST, D>::wg_per_cu(PG))) chunk_f32_kernel(const ChunkF32K p) {
    __shared__ __attribute__((aligned(1024))) char lds[2][2 * F32Geom<ST, D>::KB];

    // Launch slot b runs on XCD b % 8; XCD x takes contiguous units, splits fastest, then query
    // blocks, then kv heads, so the blocks of one kv head share an L2; the first half of a kv
    // head's blocks runs from the last (most keys) down, the second from the first up, so that
    // the two workgroups of a CU sum to about the same keys (as qr_chunk.hip, measured there).
    const int unit = (blockIdx.x & 7) * p.per_xcd + (blockIdx.x >> 3);
    if (unit >= p.units) return;
    const int split = unit % p.splits;
    const int uq = (unit / p.splits) % p.qblocks;
    const int hq = (p.qblocks + 1) >> 1;
    const int qblk = uq < hq ? p.qblocks - 1 - uq : uq - hq;
    const int kvh = unit / (p.splits * p.qblocks);
    chunk_f32_tiles<ST, D, PG, false>(p, split, qblk, kvh, lds);
}

// Merge of the splits: D / 4 threads per (query, head) row, 4 dims each; the (max, sum) pairs
// of up to 8 splits and their partials are loaded at once.
template <int D>
__global__ void __launch_bounds__(256) chunk_f32_combine_kernel(const ChunkF32K p, long long rows) {
    constexpr int TPR = D / 4, RPB = 256 / TPR;
    const int rr = threadIdx.x / TPR;
    const long long r = static_cast<long long>(blockIdx.x) * RPB + rr;
    if (rr >= RPB || r >= rows) return;
    const int c = threadIdx.x - rr * TPR;
    const size_t base = static_cast<size_t>(r) * p.splits;
    const f32x4_t* part = reinterpret_cast<const f32x4_t*>(p.part_acc) + c;
    constexpr int kB = 8;
    float m = -INFINITY, l = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += kB) {
        f32x4_t a[kB];
        float2 ml[kB];
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int s = min(s0 + i, p.splits - 1);
            a[i] = part[(base + s) * TPR];
            ml[i] = p.part_ml[base + s];
        }
        float mb = m;
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            if (s0 + i >= p.splits) ml[i] = make_float2(-INFINITY, 0.f);  // a repeated split
            mb = fmaxf(mb, ml[i].x);
        }
        const float cm = m == -INFINITY ? 0.f : fast_exp2(m - mb);
        l *= cm;
        o *= cm;
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const float w = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - mb);
            l = fmaf(ml[i].y, w, l);
            if (s0 + i < p.splits) o += a[i] * w;
        }
        m = mb;
    }
    float* out = p.out + static_cast<size_t>(r) * D + 4 * c;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = o[e] / l;
}

int cu_count() {
    static int n = 0;
    if (n == 0) {
        int dev = 0;
        hipDeviceProp_t prop;
        if (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&prop, dev) == hipSuccess)
            n = prop.multiProcessorCount;
        if (n <= 0) n = 256;
    }
    return n;
}

int wgs_per_cu(int kv_dtype, int D, int pg) {
    if (kv_dtype != QR_DTYPE_F32) return D == 96 ? F32Geom<F16Tag, 96>::wg_per_cu(pg) : F32Geom<F16Tag, 256>::wg_per_cu(pg);
    switch (D) {
        case 64: return F32Geom<float, 64>::wg_per_cu(pg);
        case 96: return F32Geom<float, 96>::wg_per_cu(pg);
        case 128: return F32Geom<float, 128>::wg_per_cu(pg);
        default: return F32Geom<float, 256>::wg_per_cu(pg);
    }
}

template <typename ST, int D>
hipError_t launch_geom(const ChunkF32K& k, const ChunkPlan& pl, hipStream_t s, hipEvent_t after_split) {
    const dim3 grid(8 * k.per_xcd);
    if (pl.pg == 2) hipLaunchKernelGGL((chunk_f32_kernel<ST, D, 2>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((chunk_f32_kernel<ST, D, 1>), grid, dim3(256), 0, s, k);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (after_split && (e = hipEventRecord(after_split, s)) != hipSuccess) return e;
    if (pl.splits == 1) return hipSuccess;
    const long long rows = static_cast<long long>(k.nq) * k.heads;
    constexpr int RPB = 256 / (D / 4);
    hipLaunchKernelGGL((chunk_f32_combine_kernel<D>), dim3(static_cast<unsigned>((rows + RPB - 1) / RPB)), dim3(256), 0, s,
                       k, rows);
    return hipGetLastError();
}

}  // namespace

bool chunk_f32_eligible(int kv_dtype, int head_dim, int heads, int kv_heads, int pos0, int nq) {
    if (heads % kv_heads || heads / kv_heads > 64) return false;
    if (nq < 2 || static_cast<long long>(nq) * (heads / kv_heads) < kChunkF32MinRows) return false;
    const bool f32 = kv_dtype == QR_DTYPE_F32;
    if (head_dim != 96 && head_dim != 256 && !(f32 && (head_dim == 64 || head_dim == 128))) return false;
    // More than 64 queries took several decode launches (128 from scratch, 32 heads over 8: 21.4 us
    // against 16.0 here).  Few queries over few keys: one launch of up to 64 entries, merged in the
    // kernel, costs less than this kernel and its merge.  The lines are by the K/V bytes that the
    // entries would read themselves (us as entries and here, the append included):
    //   32 to 64 queries, two heads per kv head: 200 MB 16.0 and 19.4 (64 after 349, head_dim 128), 300
    //   MB 18.2 and 19.5 or ahead; three: 200 MB 21.8 and 25.1; four and more: 100 MB 16.4 and 19.2, 140
    //   ahead; head_dim 256, two heads: 200 MB 23.5 and 35.0, 300 MB 28.7 and 31.7 in fp32, 140 MB 29.0
    //   and 30.5 in 16 bits;
    //   fewer: 66 MB 18.7 and 19.8 (4 after 2000), 197 MB 29.6 and 26.9; very few rows leave CUs idle
    //   here (4 queries of 8 heads over 1 after 48826: 34.0 and 36.6, head_dim 64);
    //   one head per kv head, where the entries do a third of the work per byte: 64 after 400 (226 MB)
    //   17.2 and 20.7 (head_dim 128), 32 after 1000 (266 MB) 17.8 and 19.8 (64), 16 after 2000 (263 MB)
    //   21.7 and 20.2; at head_dim 256, where two launches are still ahead, 64 after 300 (174 MB in 16
    //   bits, 8 heads) 23.8 and 27.7, 32 after 500 (271 MB, 16 heads) 30.3 and 30.8, 65 after 100 (141
    //   MB in fp32) 27.9 and 32.9, 64 after 400 (453 MB in fp32) 28.9 and 31.8.
    // The entries of head_dim 96 are slower (4 queries after 500, 32 heads over 8: 25.8 and 18.8); with
    // one head per kv head they are ahead over few keys (32 after 300 16.3 and 18.4, 8 after 500 16.9
    // and 18.9, 8 after 2000 26.9 and 18.7).
    const int g = heads / kv_heads;
    if (head_dim == 96) return nq > 64 || g > 1 || pos0 + nq > 540;
    if (nq > (g == 1 && head_dim == 256 ? 128 : 64)) return true;
    if (head_dim < 256 && nq * heads < 64) return false;
    const bool wide32 = head_dim == 256 && f32;
    double line = 96e6;
    if (g == 1) line = wide32 ? 500e6 : 280e6;
    else if (nq >= 32) line = g == 2 ? (wide32 ? 350e6 : head_dim == 256 ? 200e6 : 300e6) : g == 3 ? 210e6 : 140e6;
    const double bytes = 2.0 * nq * (pos0 + 0.5 * nq) * kv_heads * head_dim * (f32 ? 4 : 2);
    return bytes >= line;
}

ChunkPlan plan_chunk_f32(const ChunkArgs& a) {
    const int g = a.heads / a.geom.kv_heads, D = a.geom.head_dim;
    const long long rows = static_cast<long long>(a.nq) * a.heads;
    const int tiles = (a.pos0 + a.nq + kTP - 1) / kTP;
    ChunkPlan best{};
    double best_cost = 0;
    // Position halves and splits of the keys by the time of the matrix work plus the partials'
    // traffic (written and read once, about 4 TB/s) and the merge's launch.  A tile of 64 rows and
    // 32 positions is 32 D cycles of a CU's matrix units; with w workgroups resident a tile of each
    // takes 0.8 (w + 1) of that (a workgroup alone leaves the units idle in its softmax and
    // barriers, several overlap), position halves 0.65 of it instead of a half (a barrier per half
    // the work).  Query blocks of like lengths (many keys before them) run in whole rounds of the
    // longest; blocks from scratch mix, so they take the mean length.  Over 163 shapes the choice
    // took 2.6% more than the fastest of up to ten (by whole occupancy rounds alone 7.9%).  At the
    // shape above 64 rows in 1, 2, 3 and 4 splits 193, 158, 195 and 164 us with the append, halves in
    // 1 and 2 163 and 177; 1059 queries from scratch at head_dim 64: 64 rows 91, halves 68; 512 after
    // 1536 at head_dim 256 in 16 bits: 64 rows 468, halves 346.
    // Splits are for units that leave CUs idle: no more of them than fill the CUs four times over,
    // which bounds the partials too (4 x 768 workgroups x 64 rows of head_dim 96: 77 MB).
    const int cus = cu_count();
    const double like = static_cast<double>(a.pos0) / (a.pos0 + a.nq);  // 0 from scratch
    auto tile_cost = [](double w) { return 0.8 * (w + 1.0); };
    for (int pg = 1; pg <= 2; ++pg) {
        const int per_cu = wgs_per_cu(a.kv_dtype, D, pg), slots = cus * per_cu;
        const int wg_rows = 64 / pg;
        if (wg_rows < g) continue;
        const int qpb = wg_rows / g, qblocks = (a.nq + qpb - 1) / qpb;
        const long long units = static_cast<long long>(qblocks) * a.geom.kv_heads;
        const double tile_us = 32.0 * D / 2400 * (pg == 2 ? 0.65 : 1.0);
        const int smax = std::min(64, std::max(1, tiles / 4));
        auto bytes = [&](int s) { return static_cast<size_t>(rows) * s * (static_cast<size_t>(D) * 4 + 8); };
        for (int s = 1; s <= smax && (s == 1 || (units * s <= 4LL * slots && bytes(s) <= a.room)); ++s) {
            const long long full = units * s / slots, rest = units * s % slots;
            const double longest = (tiles + s - 1) / s + 1.0;
            const double mean = (a.pos0 + 0.5 * a.nq) / kTP / s + 1.0;
            const double per = static_cast<double>(units) * s / cus, w = std::min<double>(per_cu, std::max(1.0, per));
            const double rounds = (full * tile_cost(per_cu) + (rest ? tile_cost((rest + cus - 1) / cus) : 0.0)) * longest;
            const double mixed = std::max(longest * tile_cost(1), per * mean * tile_cost(w) / w);
            const double traffic = s > 1 ? 5.0 + static_cast<double>(rows) * s * D * 8 / 4e6 : 0.0;
            const double cost = (like * rounds + (1.0 - like) * mixed) * tile_us + traffic;
            if (best.splits == 0 || cost < best_cost) {
                best_cost = cost;
                best.nt = 1;
                best.pg = pg;
                best.queries_per_block = qpb;
                best.qblocks = qblocks;
                best.splits = s;
            }
        }
    }
    best.workspace_bytes = best.splits > 1 ? static_cast<size_t>(rows) * best.splits * (static_cast<size_t>(D) * 4 + 8) : 0;
    return best;
}

hipError_t launch_chunk_f32(const ChunkArgs& a, const ChunkPlan& pl, void* workspace, hipStream_t stream,
                            hipEvent_t after_split) {
    ChunkF32K k{};
    k.pool = static_cast<const char*>(a.pool);
    k.page_table = a.page_table;
    k.page_elems = a.geom.page_elems();
    k.plane_elems = a.geom.plane_elems();
    k.heads = a.heads;
    k.group = a.heads / a.geom.kv_heads;
    k.pos0 = a.pos0;
    k.nq = a.nq;
    k.q_dtype = a.q_dtype;
    k.q = a.q;
    k.out = a.out;
    k.part_acc = static_cast<float*>(workspace);
    k.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) +
                                          static_cast<size_t>(a.nq) * a.heads * pl.splits * a.geom.head_dim * 4);
    k.qscale = static_cast<float>(static_cast<double>(a.scale) * 1.4426950408889634);
    k.queries_per_block = pl.queries_per_block;
    k.splits = pl.splits;
    k.qblocks = pl.qblocks;
    k.units = pl.splits * pl.qblocks * a.geom.kv_heads;
    k.per_xcd = (k.units + 7) / 8;
    if (a.kv_dtype == QR_DTYPE_F32) {
        switch (a.geom.head_dim) {
            case 64: return launch_geom<float, 64>(k, pl, stream, after_split);
            case 96: return launch_geom<float, 96>(k, pl, stream, after_split);
            case 128: return launch_geom<float, 128>(k, pl, stream, after_split);
            default: return launch_geom<float, 256>(k, pl, stream, after_split);
        }
    }
    if (a.kv_dtype == QR_DTYPE_BF16)
        return a.geom.head_dim == 96 ? launch_geom<BF16Tag, 96>(k, pl, stream, after_split)
                                     : launch_geom<BF16Tag, 256>(k, pl, stream, after_split);
    return a.geom.head_dim == 96 ? launch_geom<F16Tag, 96>(k, pl, stream, after_split)
                                 : launch_geom<F16Tag, 256>(k, pl, stream, after_split);
}

}  // namespace qr
