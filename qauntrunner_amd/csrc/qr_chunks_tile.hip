// qr_chunks_tile.hip -- causal attention of chunks of several sequences on 32x32x16 MFMA tiles:
// 16-bit caches of head size 64 or 128 (the MFMA page layout, qr_kernels.hpp), whole groups of
// query heads, gfx950.
//
// A row is one (query, query head) pair of a kv head; a wave owns 32 rows:
//   QK  S^T[position][row] = K . q^T    (A = K, B = q)
//   PV  O^T[dim][row]     += V^T . P^T  (A = V, B = P)
// v_mfma_f32_32x32x16: A[m = lane % 32][k = 8 (lane / 32) + i], B[k = 8 (lane / 32) + i][n = lane % 32],
// D[m = 8 (r / 4) + 4 (lane / 32) + r % 4][n = lane % 32].  A row's scores lie in two lanes, l and
// l ^ 32.  QK row m = 16 s + 8 a + 4 h + b stands for position 16 s + 8 h + 4 a + b of its step of 32, so that
// a lane's scores r = 8 s + i are positions 16 s + 8 (lane / 32) + i: its k-slots of PV step s, and
// V's operand is 8 consecutive positions of a dim, 16 bytes of the page.
//
// Softmax in log2 units: weights 2^(s - m) of at most 2^kTop, m moved (and the accumulators rescaled) only when a score
// passes m + kTop, and then to leave kHead log2 units to the next move.  bf16 weights stay at or below 1: a V near the type's
// largest value does not overflow.  fp16 has few exponents below 1 (subnormal from 2^-14, nothing below 2^-25), so its
// weights go up to 2^15: whole down to 2^-25 of a row's largest or less, and products of up to 2^31 leave the sums room for
// any number of keys.  Sums are of the fp32 weights.
// Queries that are not of the cache's type enter as parts of it, and so do the weights: two parts keep 16 (bf16) or 22
// (fp16) bits of both -- of a weight w of the row's largest in fp16 no less than 2^-40 / w -- three of bf16 24.  bf16 takes
// three (the error of eight verify chunks 4e-6 with two, 4e-7 with three, 87 and 102 us), fp16 two.  Otherwise the weights are
// rounded to the type once, as the output is (2048 bf16 rows after 6144: 2.3e-3 from 64 bits where fp32 weights have 1.7e-3; a
// second part would be half as many MFMAs again).
//
// Tiles are copied into LDS by buffer-load DMA as they lie in the page.
#include "qr_chunks.hpp"
#include "qr_mfma.hpp"

namespace qr {
namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16_t mfma32(f16x8_t a, f16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// (the scores come from MFMAs: fmaxf's quieting of NaNs, one more v_max each, is not needed; a NaN score reaches its
// row through its weight)
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <bool BF16> struct Elem {
    using T = typename std::conditional<BF16, __bf16, _Float16>::type;
    typedef T vec8 __attribute__((ext_vector_type(8)));
};

// One wave's 32 rows.  PARTS of the cache's type that a query value and a weight enter as.
template <bool BF16, int D, int PARTS>
struct Rows {
    static constexpr bool SPLIT = PARTS > 1;
    using T = typename Elem<BF16>::T;
    using vec8 = typename Elem<BF16>::vec8;
    static constexpr int NK = D / 16;   // QK k-steps
    static constexpr int ND = D / 32;   // PV dim tiles
    static constexpr float kTop = BF16 ? 0.f : 15.f, kHead = SPLIT ? 0.f : 4.f;

    int lane, half;
    int query, head;     // of row lane % 32
    bool on;
    int lim;             // last position the row sees
    vec8 q[PARTS][NK];
    float sscale;        // log2 units per score
    float m, l;          // l: this lane's half of the positions
    f32x16_t acc[ND];

    __device__ __forceinline__ void init(const ChunksK& p, const ChunkItem& it, int kvh, int g, int rho) {
        lane = threadIdx.x & 63;
        half = lane >> 5;
        const int r = rho + (lane & 31);
        on = r < it.rows * g;
        const int rr = on ? r : it.rows * g - 1;
        query = rr / g;
        head = kvh * g + rr - query * g;
        lim = it.pos0 + query;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    }

    // dims 16 kk + 8 half .. + 7 of the row.  The sign of the scale goes into q: the maximum is
    // taken before the scores are scaled.
    __device__ __forceinline__ void load_q(const ChunksK& p, const ChunkItem& it) {
        const long long at = (static_cast<long long>(it.row0 + query) * p.heads + head) * D + 8 * half;
        const float sign = p.qscale == 0.f ? 0.f : p.qscale < 0.f ? -1.f : 1.f;
        sscale = p.qscale == 0.f ? 1.f : fabsf(p.qscale);
        float x[NK][8];
        if (p.act == QR_DTYPE_F32) {
            const float* f = static_cast<const float*>(p.q) + at;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[kk][i] = f[16 * kk + i];
        } else {
            const uint16_t* h = static_cast<const uint16_t*>(p.q) + at;
            uint16_t u[NK][8];
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) u[kk][i] = h[16 * kk + i];
            const bool bf = p.act == QR_DTYPE_BF16;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[kk][i] = bf ? bf16_bits_to_f32(u[kk][i]) : f16_bits_to_f32(u[kk][i]);
        }
        float by = sign;
        if (SPLIT && !BF16) {
            // fp16 parts: the row's largest value to 2^13 .. 2^14, a power of two that the score scale takes back
            float a = 0.f;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(x[kk][i]));
            a = max_xor32(a);
            if (a > 1e-30f && a < 3e38f) {
                const int ex = ilogbf(a) - 13;
                by = ldexpf(sign, -ex);
                sscale = ldexpf(sscale, ex);
            }
        }
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float v = x[kk][i] * by;
#pragma unroll
                for (int c = 0; c < PARTS; ++c) {
                    q[c][kk][i] = static_cast<T>(v);
                    v -= static_cast<float>(q[c][kk][i]);
                }
            }
    }

    // LDS offset of this lane's part of the K operand of a step (k-step kk: + 512 kk) ...
    __device__ __forceinline__ int k_off() const {
        const int m_ = lane & 31, s = m_ >> 4, a = (m_ >> 3) & 1, h = (m_ >> 2) & 1, b = m_ & 3;
        return 1024 * a * (D / 32) + 16 * (16 * half + 4 * (2 * s + h) + b);
    }
    // ... and of the V operand (dim tile md, PV step s: + 2048 md + 512 s)
    __device__ __forceinline__ int v_off() const { return 1024 * ((lane & 31) >> 4) + 16 * (16 * half + (lane & 15)); }

    // positions t0 + 16 s + 8 half + i past the row's own, or past the end, get no weight
    __device__ __forceinline__ void mask(f32x16_t& s, int t0, int end) const {
        const int last = min(lim, end - 1) - t0 - 8 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (16 * (r >> 3) + (r & 7) > last) s[r] = -INFINITY;
    }

    // Weights of NS steps' scores, as PV operands; rescales what was summed when the maximum moves.  `step(k)` is
    // called after every eighth weight, k = 0 .. 2 NS - 1.
    template <int NS, class F>
    __device__ __forceinline__ void softmax(const f32x16_t (&s)[NS], vec8 (&w)[PARTS][NS][2], F step) {
        float mx[2 * NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const float a = max3f(s[n][0], s[n][1], s[n][2]), b = max3f(s[n][3], s[n][4], s[n][5]);
            const float c = max3f(s[n][6], s[n][7], s[n][8]), d = max3f(s[n][9], s[n][10], s[n][11]);
            mx[2 * n] = max3f(s[n][12], s[n][13], s[n][14]);
            mx[2 * n] = max3f(mx[2 * n], s[n][15], a);
            mx[2 * n + 1] = max3f(b, c, d);
        }
        float t = mx[0];
#pragma unroll
        for (int n = 1; n < 2 * NS; ++n) t = fmaxf(t, mx[n]);
        t = max_xor32(t);
        const bool grow = fmaf(t, sscale, -m) > kTop;
        if (__builtin_amdgcn_ballot_w64(grow)) {
            float mn = fmaf(t, sscale, kHead - kTop);
            if (fmaf(t, sscale, -mn) > kTop) {  // rounded down, where a step of m is that large
                const int b = __float_as_int(mn);
                mn = __int_as_float(b < 0 ? b - 1 : b + 1);
            }
            mn = grow ? mn : m;
            const float c = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            if (__builtin_amdgcn_ballot_w64(grow && m != -INFINITY)) {
                const float cc = grow && m != -INFINITY ? c : 1.f;
                l *= cc;
#pragma unroll
                for (int d = 0; d < ND; ++d) acc[d] *= cc;
            }
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.f : -m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float e = fast_exp2(fmaf(s[n][r], sscale, ref));
                sum[r & 3] += e;
                float v = e;
#pragma unroll
                for (int c = 0; c < PARTS; ++c) {
                    w[c][n][r >> 3][r & 7] = static_cast<T>(v);
                    v -= static_cast<float>(w[c][n][r >> 3][r & 7]);
                }
                if ((r & 7) == 7) step(2 * n + (r >> 3));
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // A tile that reaches past what every row sees may hold V elements that are not finite at
    // positions some rows do not see, where 0 x inf would reach them.  True if the step at `v` has such an element
    // (the same in every wave that looks).
    __device__ __forceinline__ bool v_bad(const char* v) const {
        vec8 zero;
#pragma unroll
        for (int i = 0; i < 8; ++i) zero[i] = static_cast<T>(0.f);
        f32x16_t z;
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * ND; ++c) z = mfma32(*reinterpret_cast<const vec8*>(v + 1024 * c + 16 * lane), zero, z);
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += z[i];
        return __builtin_amdgcn_ballot_w64(!(t == 0.f)) != 0;
    }
    // Adds the elements of the step at `v` (positions t0 .. t0 + 31) that are not finite to the rows that see them, as they
    // are: no finite weight changes them.
    __device__ __forceinline__ void add_bad(const char* v, int t0, int end) {
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int dim = 32 * d + 8 * (r >> 2) + 4 * half + (r & 3);
                    const float x = static_cast<float>(*reinterpret_cast<const T*>(
                        v + 1024 * (dim >> 4) + 16 * (16 * (k >> 3) + (dim & 15)) + 2 * (k & 7)));
                    if (!(fabsf(x) < INFINITY) && t0 + k <= min(lim, end - 1)) acc[d][r] += x;
                    if ((r & 3) == 3) asm volatile("" ::: "memory");  // no registers for all reads at once
                }
        }
    }

    // The row's output or split partial: N groups of 4 dims from group g0 on, of the weighted sums a.
    // Group g holds dims 32 (g / 4) + 8 (g % 4) + 4 half .. + 3.
    // A sum that is no number though the weights are comes from an infinite V: a part of a weight may be negative, or a weight
    // round to zero.  It is that infinity, unless the row sees a NaN or both: one pass over the unit's values, a dim per lane (70
    // bf16 queries in each of 64 sequences of 8192 positions: 1.0 ms, 2.0 with one value of NaNs).
    template <int N>
    __device__ __forceinline__ void settle(const ChunksK& p, const ChunkItem& it, int t0, int t1, int g0, float lsum, f32x4_t (&a)[N]) const {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 4 * N; ++i) bad |= !(a[i >> 2][i & 3] == a[i >> 2][i & 3]);
        bad = bad && on && lsum == lsum;
        if (!__builtin_amdgcn_ballot_w64(bad)) return;
        const int kvh = __builtin_amdgcn_readfirstlane(head / (p.heads / p.geom.kv_heads)), end = min(t1, lim + 1);
#pragma unroll 1
        for (int k = g0 >> 3; k <= (g0 + N - 1) >> 3; ++k) {  // dims 64 k .. 64 k + 63 are groups 8 k .. 8 k + 7
            const NotFinite f = find_not_finite(p.pool, p.page_table + it.pt_off, p.geom, p.dtype, kvh, 64 * k + lane, t0, t1);
#pragma unroll
            for (int i = 0; i < 4 * N; ++i) {
                const int d = 8 * (g0 + (i >> 2)) + 4 * half + (i & 3);
                const NotFinite o = f.of_lane(d & 63);
                const float x = a[i >> 2][i & 3];
                a[i >> 2][i & 3] = bad && d >> 6 == k && !(x == x) ? o.settle(end, x) : x;
                if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // no registers for all of them at once
            }
        }
    }
    template <int N>
    __device__ __forceinline__ void store(const ChunksK& p, const ChunkItem& it, int split, int g0, float lsum, const f32x4_t (&a)[N]) const {
        if (!on) return;
        const long long rh = static_cast<long long>(it.row0 + query) * p.heads + head;
        auto dim = [&](int i) { return 32 * ((g0 + i) >> 2) + 8 * ((g0 + i) & 3) + 4 * half; };
        if (it.parts > 1) {
            float* o = p.part_acc + (it.slot0 + (static_cast<long long>(query) * p.heads + head) * it.splits + split) * D;
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<f32x4_t*>(o + dim(i)) = a[i];
            return;
        }
        const float inv = 1.f / lsum;
        if (!SPLIT) store16<T>(static_cast<uint16_t*>(p.out) + rh * D, inv, a, dim);
        else if (p.act == QR_DTYPE_BF16) store16<__bf16>(static_cast<uint16_t*>(p.out) + rh * D, inv, a, dim);
        else if (p.act == QR_DTYPE_F16) store16<_Float16>(static_cast<uint16_t*>(p.out) + rh * D, inv, a, dim);
        else {
            float* o = static_cast<float*>(p.out) + rh * D;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const f32x4_t x = a[i] * inv;
                __builtin_memcpy(o + dim(i), &x, 16);
            }
        }
    }
    // one store per group, element-aligned
    template <class O, int N, class G>
    __device__ static __forceinline__ void store16(uint16_t* o, float inv, const f32x4_t (&a)[N], G dim) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const f32x4_t x = a[i] * inv;
            O b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = static_cast<O>(x[j]);
            __builtin_memcpy(o + dim(i), b, 8);
        }
    }
    __device__ __forceinline__ void store_ml(const ChunksK& p, const ChunkItem& it, int split, float mm, float lsum) const {
        if (!on || half) return;
        if (p.row_scale) p.row_scale[static_cast<long long>(it.row0 + query) * p.heads + head] = sscale;  // the same in every split
        if (it.parts > 1) p.part_ml[it.slot0 + (static_cast<long long>(query) * p.heads + head) * it.splits + split] = make_float2(mm, lsum);
        else if (p.row_ml) p.row_ml[static_cast<long long>(it.row0 + query) * p.heads + head] = make_float2(mm, lsum);
    }
};

// Clears the elements of `bytes` bytes of V that are not finite, by `threads` threads.
template <class T> __device__ __forceinline__ void clear_bad(char* v, int bytes, int thread, int threads) {
    for (int c = thread; c < bytes / 2; c += threads) {
        T* e = reinterpret_cast<T*>(v) + c;
        if (!(fabsf(static_cast<float>(*e)) < INFINITY)) *e = static_cast<T>(0.f);
    }
}

// Page of a position, by a scalar load (no kernel writes the table while this one runs).
__device__ __forceinline__ int page_of(const ChunksK& p, int pt_off, int t) {
    return reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p.page_table))[pt_off + (t >> kPageShift)];
}

// ------------------------------------------------------------------ few rows: HBM-bound
// RW waves of 32 rows each x PW waves that take one step of 32 positions of every tile.  K and V of a tile are
// units of a ring in LDS that fills it, most of them in flight while one is used.  With RW = 1 a wave copies its own steps
// and no wave waits for another before the end, where the PW (m, l, o) of a row merge.  16 decode rows of 32 heads over
// 130 to 16000 fp16 positions: 47 us for 241 MB, 5.1 TB/s; eight chunks of 5 to 9 rows of 64 heads, fp32 queries over 2000 to
// 32000 bf16 positions: 89 to 99 us for 388 MB, two thirds of it the MFMAs of the three parts, not wholly beside the loads.

template <bool BF16, int D, int PARTS, int RW, int PW, int LDS>
__device__ __forceinline__ void chunk_stream(const ChunksK& p, const ChunkItem& it, int u, char* lds) {
    using R = Rows<BF16, D, PARTS>;
    using T = typename R::T;
    using vec8 = typename R::vec8;
    constexpr int WAVES = RW * PW;
    constexpr int TILE = 32 * PW;
    constexpr int SB = 64 * D;                    // bytes of a step of K (or V)
    constexpr int UB = SB * PW;                   // of a unit
    constexpr int UL = UB / 1024 / WAVES;         // DMA loads per wave and unit
    constexpr int NU = LDS / UB < 10 ? LDS / UB : 10;
    constexpr int NG = D / 8;                     // f32x4 groups of a row in a lane
    static_assert(NG % PW == 0 && WAVES * 64 * (NG * 16 + 8) <= LDS, "the waves' (acc, m, l) fit");
    static_assert(UL >= 1 && NU >= 4 && (NU - 2) * UL < 64, "vmcnt");
    // (kv heads fastest, so that an XCD keeps few of them in its L2 where a chunk has many blocks; from the last block down)
    const int kvh = u % p.geom.kv_heads, split = u / p.geom.kv_heads % it.splits, block = it.blocks - 1 - u / p.geom.kv_heads / it.splits;
    const int g = p.heads / p.geom.kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RW, pw = wave / RW;
    const int rho0 = block * 32 * RW;
    const int last = min(rho0 + 32 * RW, it.rows * g) - 1;
    int t0, t1;
    chunk_keys(it, it.pos0 + last / g + 1, split, TILE, &t0, &t1);
    const int ntiles = t1 > t0 ? (t1 - t0 + TILE - 1) / TILE : 0;
    const int seen = it.pos0 + rho0 / g + 1;  // positions below it are seen by every row

    const long long page_bytes = p.geom.page_elems() * 2, plane_bytes = p.geom.plane_elems() * 2;
    const long long head_bytes = static_cast<long long>(kvh) * kPageTokens * D * 2;
    const uint32_t lane16 = 16 * (threadIdx.x & 63);
    // Unit n: K (n even) or V of tile n / 2, load c of this wave.  A step past the keys' end has no records: zeros are
    // written and no memory is read (it may lie past the held pages, its page is not looked up).
    // A tile lies in one page, whose entry is looked up a tile ahead (a lookup at its use held the wave for its latency, twice a
    // tile).
    auto page = [&](int n) __attribute__((always_inline)) {
        const int ts = t0 + (n >> 1) * TILE;
        return ts < t1 ? page_of(p, it.pt_off, ts) : 0;
    };
    auto load = [&](int n, int c, int phys) __attribute__((always_inline)) {
        const int x = RW == 1 ? pw * (SB / 1024) + c : wave + WAVES * c;  // RW = 1: the wave's own step
        const int ts = t0 + (n >> 1) * TILE + 32 * (x / (SB / 1024));
        const bool in = ts < t1;
        const char* base = p.pool + static_cast<long long>(phys) * page_bytes + head_bytes + (n & 1 ? plane_bytes : 0) +
                           static_cast<long long>(ts & (kPageTokens - 1)) * D * 2;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, in ? SB : 0, kBufferFlags);
        buffer_load_lds16<kCacheNt>(r, lds + n % NU * UB + 1024 * x, lane16, 1024 * (x % (SB / 1024)));
    };
    auto request = [&](int n, int phys) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < UL; ++c) load(n, c, phys);
    };
    // Unit n has landed in every wave, and the one before it was read by every wave.
    auto turn = [&]() __attribute__((always_inline)) {
        wait_vmcnt<(NU - 2) * UL>();
        if (RW > 1) lds_barrier_dma_in_flight();
    };
    int phys0 = 0, phys1 = 0;  // of the next request in each half of a tile
    if (ntiles > 0) {
        for (int n = 0; n < NU - 1; ++n) request(n, page(n));
        phys0 = page(NU - 1);
        phys1 = page(NU);
    }

    R w;
    w.init(p, it, kvh, g, rho0 + 32 * rw);
    w.load_q(p, it);
    const int ko = w.k_off(), vo = w.v_off();
    float* const scores = RW == 1 && p.scores && it.score0 >= 0 ? p.scores + it.score0 + (static_cast<long long>(w.query) * p.heads + w.head) * chunk_score_len(it) : nullptr;

    for (int i = 0; i < ntiles; ++i) {
        turn();
        request(2 * i + NU - 1, phys0);  // over V of tile i - 1
        phys0 = page(2 * i + NU + 1);
        const int ts = t0 + i * TILE + 32 * pw;
        const char* const kt = lds + 2 * i % NU * UB + SB * pw;
        const bool edge = t0 + (i + 1) * TILE > seen || t0 + (i + 1) * TILE > t1;
        f32x16_t s[1];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = 0.f;
        {
            vec8 a[R::NK];
#pragma unroll
            for (int kk = 0; kk < R::NK; ++kk) a[kk] = *reinterpret_cast<const vec8*>(kt + ko + 512 * kk);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < R::NK; ++kk)
#pragma unroll
                for (int c = 0; c < PARTS; ++c) s[0] = mfma32(a[kk], w.q[c][kk], s[0]);
        }
        if (edge) w.mask(s[0], ts, t1);
        if (scores && w.on) {
            // for the weights: a row's 8 positions are 32 bytes (whole: a row of scores is whole runs of 8)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                if (ts + 16 * x + 8 * w.half < t1) {
                    f32x4_t* o = reinterpret_cast<f32x4_t*>(scores + ts + 16 * x + 8 * w.half);
                    o[0] = f32x4_t{s[0][8 * x], s[0][8 * x + 1], s[0][8 * x + 2], s[0][8 * x + 3]} * w.sscale;
                    o[1] = f32x4_t{s[0][8 * x + 4], s[0][8 * x + 5], s[0][8 * x + 6], s[0][8 * x + 7]} * w.sscale;
                }
        }
        turn();
        char* const vu = lds + (2 * i + 1) % NU * UB;
        char* const vt = vu + SB * pw;
        if (edge) {
            if (RW > 1) {
                bool bad = false;
                for (int x = 0; x < PW; ++x) bad |= w.v_bad(vu + SB * x);
                if (bad) {  // the same in every wave
                    w.add_bad(vt, ts, t1);
                    lds_barrier_dma_in_flight();
                    clear_bad<T>(vu, UB, threadIdx.x, 64 * WAVES);
                    lds_barrier_dma_in_flight();
                }
            } else if (w.v_bad(vt)) {
                w.add_bad(vt, ts, t1);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                clear_bad<T>(vt, SB, w.lane, 64);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
        request(2 * i + NU, phys1);  // over K of this tile
        phys1 = page(2 * i + NU + 2);
        vec8 wt[PARTS][1][2];
        w.template softmax<1>(s, wt, [](int) {});
        {
            vec8 a[2][R::ND];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int d = 0; d < R::ND; ++d) a[x][d] = *reinterpret_cast<const vec8*>(vt + vo + 2048 * d + 512 * x);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int c = 0; c < PARTS; ++c)
#pragma unroll
                    for (int d = 0; d < R::ND; ++d) w.acc[d] = mfma32(a[x][d], wt[c][0][x], w.acc[d]);
        }
    }
    w.l = sum_xor32(w.l);

    // the PW waves of a row group merge: each adds up NG / PW of the dim groups
    wait_dma();
    __syncthreads();
    f32x4_t* const xa = reinterpret_cast<f32x4_t*>(lds);                        // [wave][group][64]
    float2* const xm = reinterpret_cast<float2*>(lds + WAVES * 64 * NG * 16);   // [wave][64]
#pragma unroll
    for (int d = 0; d < R::ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            xa[(wave * NG + 4 * d + q) * 64 + w.lane] = f32x4_t{w.acc[d][4 * q], w.acc[d][4 * q + 1], w.acc[d][4 * q + 2], w.acc[d][4 * q + 3]};
    xm[wave * 64 + w.lane] = make_float2(w.m, w.l);
    __syncthreads();
    float M = -INFINITY, L = 0.f, c[PW];
#pragma unroll
    for (int x = 0; x < PW; ++x) M = fmaxf(M, xm[(x * RW + rw) * 64 + w.lane].x);
#pragma unroll
    for (int x = 0; x < PW; ++x) {
        const float2 ml = xm[(x * RW + rw) * 64 + w.lane];
        c[x] = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
        L = fmaf(ml.y, c[x], L);
    }
    constexpr int NP = NG / PW;
    f32x4_t o[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        o[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < PW; ++x) o[q] += xa[((x * RW + rw) * NG + pw * NP + q) * 64 + w.lane] * c[x];
    }
    w.settle(p, it, t0, t1, pw * NP, L, o);
    w.store(p, it, split, pw * NP, L, o);
    if (pw == 0) w.store_ml(p, it, split, M, L);
}

// Chunks of up to 32 rows: one workgroup per CU, all its LDS.
template <bool BF16, int D, int PARTS>
__global__ void __launch_bounds__(256, 1) chunks_stream32_kernel(const ChunksK p) {
    constexpr int LDS = 160 * 1024;
    __shared__ __attribute__((aligned(1024))) char lds[LDS];
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    chunk_stream<BF16, D, PARTS, 1, 4, LDS>(p, it, blockIdx.x - it.unit0, lds);
}
// Chunks of up to 128 rows, each in its own shape: two workgroups per CU, so that one computes while the other stands
// at a barrier (one of eight waves: 111 us where this takes 102).
template <bool BF16, int D, int PARTS>
__global__ void __launch_bounds__(256, 2) chunks_stream_kernel(const ChunksK p) {
    constexpr int LDS = 80 * 1024;
    __shared__ __attribute__((aligned(1024))) char lds[LDS];
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0;
    if (it.rows * (p.heads / p.geom.kv_heads) <= 64) chunk_stream<BF16, D, PARTS, 2, 2, LDS>(p, it, u, lds);
    else chunk_stream<BF16, D, PARTS, 4, 1, LDS>(p, it, u, lds);
}

// ------------------------------------------------------------------ many rows: MFMA-bound
// Eight waves of 32 rows share every tile of 64 positions.  Waves 0-3 and 4-7 run half a tile apart: while
// one group's MFMAs run (scores of tile t, weighted V of tile t - 1), the other group computes its
// softmax on the same SIMDs; a barrier ends each half.  2048 bf16 rows of 32 heads after 6144: 230 to 240 us, 1.0 PFLOP/s of the
// 1.2 that a large product reaches; the MFMAs and LDS reads alone take 161, the softmax with the copies 117.  Short units
// pay about 6 us to start and end.
template <bool BF16, int D, bool SPLIT>
__global__ void __launch_bounds__(512, 1) chunks_tile_kernel(const ChunksK p) {
    constexpr int PARTS = SPLIT ? 2 : 1;
    using R = Rows<BF16, D, PARTS>;
    using vec8 = typename R::vec8;
    constexpr int TILE = kKeyTiles16.tile, NST = 3;
    constexpr int SB = 64 * D;           // bytes of a step of K (or V)
    constexpr int KB = 2 * SB;           // of a tile of K (or V)
    constexpr int PER = KB / 1024 / 8;   // DMA loads per wave for a tile of K (or V)
    __shared__ __attribute__((aligned(1024))) char lds[2 * NST * KB];  // K tiles, then V tiles

    int kvh, unit;
    if (!chunk_unit(p, &kvh, &unit)) return;
    const int e = batch_find(p.n, unit, [&](int i) { return p.it[i].unit0; });
    ChunkItem it = p.it[e];
    const int g = p.heads / p.geom.kv_heads;
    int block, split;
    kKeyTiles16.find(it, g, unit - it.unit0, &block, &split);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    static_assert(kKeyTiles16.rows == 256, "8 waves of 32 rows");
    const int rho0 = block * 256;
    const int last = min(rho0 + 256, it.rows * g) - 1;
    int t0, t1;
    chunk_keys(it, it.pos0 + last / g + 1, split, TILE, &t0, &t1);
    const int ntiles = t1 > t0 ? (t1 - t0 + TILE - 1) / TILE : 0;
    const int seen = it.pos0 + rho0 / g + 1;  // positions below it are seen by every row

    const long long page_bytes = p.geom.page_elems() * 2, plane_bytes = p.geom.plane_elems() * 2;
    const long long head_bytes = static_cast<long long>(kvh) * kPageTokens * D * 2;
    const uint32_t lane16 = 16 * (threadIdx.x & 63);
    auto page = [&](int i) { return page_of(p, it.pt_off, t0 + min(i, ntiles - 1) * TILE); };
    auto source = [&](int i, int plane, int phys) {
        const bool in = i < ntiles;  // past the last tile: no records, no memory is read
        const int t = t0 + min(i, ntiles - 1) * TILE;
        const char* base = p.pool + static_cast<long long>(phys) * page_bytes + head_bytes + plane * plane_bytes +
                           static_cast<long long>(t & (kPageTokens - 1)) * D * 2;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, in ? KB : 0, kBufferFlags);
    };
    auto load = [&](__amdgpu_buffer_rsrc_t r, int i, int plane, int c) {
        buffer_load_lds16(r, lds + plane * NST * KB + (i % NST) * KB + 1024 * (wave + 8 * c), lane16, 1024 * (wave + 8 * c));
    };
    auto dma = [&](int i, int plane) {
        const __amdgpu_buffer_rsrc_t r = source(i, plane, page(i));
#pragma unroll
        for (int c = 0; c < PER; ++c) load(r, i, plane, c);
    };
    R w;
    w.init(p, it, kvh, g, rho0 + 32 * wave);
    if (ntiles > 0) {
        dma(0, 0);
        dma(1, 0);
        dma(0, 1);
    }
    w.load_q(p, it);
    const int ko = w.k_off(), vo = w.v_off();
    vec8 pw[PARTS][2][2];
    f32x16_t s[2];

    auto barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier_dma_in_flight();
        __builtin_amdgcn_sched_barrier(0);
    };
    // operand reads run kAhead MFMAs in front of their use
    constexpr int kAhead = SPLIT ? 3 : 6;
    auto qk_pv = [&](const char* kt, const char* vt, bool qk, bool pv) __attribute__((always_inline)) {
        constexpr int NQ = 2 * R::NK, NP = 4 * R::ND;  // operands: K (step, kk), V (step, PV step, dim tile)
        static_assert(NQ == NP, "one of each in turn");
        vec8 ring[kAhead];
        auto read = [&](int i) __attribute__((always_inline)) -> vec8 {
            const int j = i >> 1;
            if (i & 1) return *reinterpret_cast<const vec8*>(vt + SB * (j / (2 * R::ND)) + vo + 2048 * (j % R::ND) + 512 * (j / R::ND % 2));
            return *reinterpret_cast<const vec8*>(kt + SB * (j & 1) + ko + 512 * (j >> 1));
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if ((i & 1) ? pv : qk) ring[i] = read(i);
#pragma unroll
        for (int i = 0; i < NQ + NP; ++i) {
            const int j = i >> 1;
            if (i & 1) {
                if (pv) {
                    const int st = j / (2 * R::ND), x = j / R::ND % 2, d = j % R::ND;
#pragma unroll
                    for (int c = 0; c < PARTS; ++c) w.acc[d] = mfma32(ring[i % kAhead], pw[c][st][x], w.acc[d]);
                }
            } else if (qk) {
                const int st = j & 1, kk = j >> 1;
                if (kk == 0)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[st][r] = 0.f;
#pragma unroll
                for (int c = 0; c < PARTS; ++c) s[st] = mfma32(ring[i % kAhead], w.q[c][kk], s[st]);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (i + kAhead < NQ + NP && ((i + kAhead) & 1 ? pv : qk)) ring[i % kAhead] = read(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    auto k_at = [&](int i) { return lds + (i % NST) * KB; };
    auto v_at = [&](int i) { return lds + NST * KB + (i % NST) * KB; };
    // K of tile i + 2 over K of tile i - 1, V of tile i + 1 over V of tile i - 2
    auto request = [&](int i) __attribute__((always_inline)) {
        dma(i + 2, 0);
        dma(i + 1, 1);
    };
    // Tiles that every row sees whole.  The early group (waves 0-3) computes scores of tile i and weighs V of tile
    // i - 1 in half 2i, its softmax of tile i in half 2i + 1; the late group each one half later.  Every wave
    // makes request(i) during its softmax, the early group in half 2i + 1, the late group in half 2i (it read what that
    // replaces for the last time in half 2i - 1), and awaits it before the barrier that ends half 2i + 3, when
    // the next request may be in flight.  The loads stand between the exponentials: a load takes its wave some
    // hundred cycles to issue when eight waves issue at once, which delayed the MFMAs (271 us a call against 214
    // without any; 2048 queries after 6144 positions).
    const int nfull = max(0, min(seen, t1) - t0) / TILE;
    if (nfull > 0) {
        const bool late = wave >= 4;
        int phys1 = page(late ? 2 : 1), phys2 = page(late ? 3 : 2);  // of tiles i + 1, i + 2 of the next request
        auto weigh = [&](int i) __attribute__((always_inline)) {  // with request(i)
            const __amdgpu_buffer_rsrc_t rk = source(i + 2, 0, phys2), rv = source(i + 1, 1, phys1);
            phys1 = phys2;
            phys2 = page(i + 3);  // looked up one tile before its use
            if (SPLIT) {  // (no registers for loads between)
#pragma unroll
                for (int c = 0; c < PER; ++c) load(rk, i + 2, 0, c);
#pragma unroll
                for (int c = 0; c < PER; ++c) load(rv, i + 1, 1, c);
                w.template softmax<2>(s, pw, [](int) {});
                return;
            }
            w.template softmax<2>(s, pw, [&](int c) __attribute__((always_inline)) {
                if (c < PER) load(rk, i + 2, 0, c);
                else if (c < 2 * PER) load(rv, i + 1, 1, c - PER);
            });
        };
        wait_vmcnt<2 * PER>();  // K of tile 0
        barrier();
        if (late) {
            request(0);
            barrier();
        }
        qk_pv(k_at(0), nullptr, true, false);
        if (late) wait_vmcnt<2 * PER>();
        barrier();
        for (int i = 0; i + 1 < nfull; ++i) {
            weigh(late ? i + 1 : i);
            if (!late) wait_vmcnt<2 * PER>();
            barrier();
            qk_pv(k_at(i + 1), v_at(i), true, true);
            if (late) wait_vmcnt<2 * PER>();
            barrier();
        }
        if (late) w.template softmax<2>(s, pw, [](int) {});
        else weigh(nfull - 1);
        if (!late) wait_vmcnt<2 * PER>();
        barrier();
        qk_pv(nullptr, v_at(nfull - 1), false, true);
        if (!late) barrier();
    }
    // The others, masked, all waves together.  K of tiles nfull and nfull + 1 and V of tile nfull are requested.
    for (int i = nfull; i < ntiles; ++i) {
        wait_dma();
        barrier();
        request(i);
        char* const v = v_at(i);
        const bool b0 = w.v_bad(v), b1 = w.v_bad(v + SB);
        if (b0 || b1) {  // the same in every wave
            w.add_bad(v, t0 + i * TILE, t1);
            w.add_bad(v + SB, t0 + i * TILE + 32, t1);
            barrier();
            clear_bad<typename R::T>(v, KB, threadIdx.x, 512);
            barrier();
        }
        qk_pv(k_at(i), nullptr, true, false);
        w.mask(s[0], t0 + i * TILE, t1);
        w.mask(s[1], t0 + i * TILE + 32, t1);
        w.template softmax<2>(s, pw, [](int) {});
        qk_pv(nullptr, v, false, true);
    }
    w.l = sum_xor32(w.l);
    f32x4_t o[4 * R::ND];
#pragma unroll
    for (int q = 0; q < 4 * R::ND; ++q)
        o[q] = f32x4_t{w.acc[q >> 2][4 * (q & 3)], w.acc[q >> 2][4 * (q & 3) + 1], w.acc[q >> 2][4 * (q & 3) + 2], w.acc[q >> 2][4 * (q & 3) + 3]};
    w.settle(p, it, t0, t1, 0, w.l, o);
    w.store(p, it, split, 0, w.l, o);
    w.store_ml(p, it, split, w.m, w.l);
}


// ------------------------------------------------------------------ weights
// Weights of 256 positions of one kv head over a part of its rows: a wave keeps the K rows of 32
// positions as operands; the workgroup puts 128 rows at a time into LDS as operands (each wave its share of the
// k-steps), with each row's maximum, 1 / sum, last position seen and score scale.  Six prompts of 101 to 1501 rows, 69
// million scores: 46 us, of which issue takes 18 (16 cycles per 64 exponentials, 8 for the multiply-adds around them, 16 for
// the MFMAs); the rest goes with the rows, which every unit takes from memory through registers into LDS (with 64 positions
// per wave, half the LDS reads, 11 us more).
template <bool BF16, int D, int PARTS>
__global__ void __launch_bounds__(512, PARTS > 1 && D == 128 ? 1 : 2) chunks_tile_weights_kernel(const ChunksK p) {
    using T = typename Elem<BF16>::T;
    using vec8 = typename Elem<BF16>::vec8;
    constexpr bool SPLIT = PARTS > 1;
    constexpr int NK = D / 16, RT = PARTS > 2 ? 2 : 4, ROWS = 32 * RT;
    constexpr int CN = NK * RT / 8;          // operands per wave of a round
    constexpr int QB = NK * RT * 1024;  // bytes of a part of the rows
    __shared__ __attribute__((aligned(1024))) char lds[2][PARTS * QB];
    __shared__ float4 info[2][ROWS];
    const int e = batch_find(p.n, blockIdx.x, [&](int i) { return p.it[i].unit0; });
    const ChunkItem it = p.it[e];
    const int u = blockIdx.x - it.unit0;
    const int kvh = u / it.blocks, g = p.heads / p.geom.kv_heads, rows = it.rows * g;
    static_assert(kWeightTiles16.rows % ROWS == 0, "rounds of whole turns");
    int split, block, splits;
    kWeightTiles16.find(it, g, u - kvh * it.blocks, &block, &split, &splits);
    const int lane = threadIdx.x & 63, half = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int len = it.pos0 + it.rows;
    const int b0 = block * kWeightTiles16.positions, t0 = b0 + 32 * wave;
    const int first = kWeightTiles16.first(it, g, block), rounds = kWeightTiles16.rounds(it, g, block);
    const int r0 = first + static_cast<int>(static_cast<long long>(rounds) * split / splits) * kWeightTiles16.rows;
    const int r1 = min(rows, first + static_cast<int>(static_cast<long long>(rounds) * (split + 1) / splits) * kWeightTiles16.rows);
    const float sign = p.qscale == 0.f ? 0.f : p.qscale < 0.f ? -1.f : 1.f;
    const float base = p.qscale == 0.f ? 1.f : fabsf(p.qscale);
    auto row_of = [&](int rho) { return static_cast<long long>(it.row0 + rho / g) * p.heads + kvh * g + rho % g; };

    // a round's share of this thread: operand wave + 8 c is k-step op % NK of row tile op / NK
    float x[SPLIT ? CN : 1][8];
    vec8 raw[SPLIT ? 1 : CN];
    float4 inf;
    // its row as (query, head), from one operand to the next and on to the next round without divisions
    constexpr int STEP = 32 * 8 / NK;
    static_assert(STEP * CN == ROWS, "a round");
    const int step_q = STEP / g, step_h = STEP % g;
    int fq = (r0 + 32 * (wave / NK) + n) / g, fh = (r0 + 32 * (wave / NK) + n) % g;
    auto fetch = [&](int r) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CN; ++c) {
            const int op = wave + 8 * c;
            const long long row = static_cast<long long>(it.row0 + min(fq, it.rows - 1)) * p.heads + kvh * g + fh;
            const long long at = row * D + 16 * (op % NK) + 8 * half;
            fq += step_q;
            fh += step_h;
            if (fh >= g) {
                fh -= g;
                ++fq;
            }
            if (!SPLIT) {
                __builtin_memcpy(&raw[SPLIT ? 0 : c], static_cast<const uint16_t*>(p.q) + at, 16);
            } else if (p.act == QR_DTYPE_F32) {
                __builtin_memcpy(x[SPLIT ? c : 0], static_cast<const float*>(p.q) + at, 32);
            } else {
                uint16_t h[8];
                __builtin_memcpy(h, static_cast<const uint16_t*>(p.q) + at, 16);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[SPLIT ? c : 0][i] = p.act == QR_DTYPE_BF16 ? bf16_bits_to_f32(h[i]) : f16_bits_to_f32(h[i]);
            }
            if (SPLIT && p.row_scale) {  // a power of two
                const float by = base / p.row_scale[row];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[SPLIT ? c : 0][i] *= by;
            }
        }
        if (threadIdx.x < ROWS) {
            const int rho = r + static_cast<int>(threadIdx.x);
            const bool on = rho < r1;
            const long long row = row_of(on ? rho : rows - 1);
            const float2 ml = p.row_ml[row];
            inf = make_float4(-ml.x, 1.f / ml.y, __int_as_float(on ? it.pos0 + rho / g : -1), p.row_scale ? p.row_scale[row] : base);
        }
    };
    auto put = [&](int to) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < CN; ++c) {
            char* o = lds[to] + 1024 * (wave + 8 * c) + 16 * lane;
            vec8 hi;
            if (!SPLIT) {
                hi = raw[SPLIT ? 0 : c];
                if (p.qscale <= 0.f)
#pragma unroll
                    for (int i = 0; i < 8; ++i) hi[i] = static_cast<T>(static_cast<float>(hi[i]) * sign);
            } else {
                vec8 part[PARTS];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float v = x[SPLIT ? c : 0][i] * sign;
#pragma unroll
                    for (int q = 0; q < PARTS; ++q) {
                        part[q][i] = static_cast<T>(v);
                        v -= static_cast<float>(part[q][i]);
                    }
                }
                hi = part[0];
#pragma unroll
                for (int q = 1; q < PARTS; ++q) *reinterpret_cast<vec8*>(o + q * QB) = part[q];
            }
            *reinterpret_cast<vec8*>(o) = hi;
        }
        if (threadIdx.x < ROWS) info[to][threadIdx.x] = inf;
    };
    if (r0 < r1) fetch(r0);
    vec8 k[NK];
    {
        const int s = n >> 4, a = (n >> 3) & 1, h = (n >> 2) & 1, b = n & 3;
        const int off = 1024 * a * (D / 32) + 16 * (16 * half + 4 * (2 * s + h) + b);
        const bool in = t0 < len;  // a block's steps past the end hold no page
        const long long phys = in ? page_of(p, it.pt_off, t0) : 0;
        const char* src = p.pool + (phys * p.geom.page_elems() + static_cast<long long>(kvh) * kPageTokens * D +
                                    static_cast<long long>(t0 & (kPageTokens - 1)) * D) * 2 + off;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
#pragma unroll
            for (int i = 0; i < 8; ++i) k[kk][i] = static_cast<T>(0.f);
            if (in) k[kk] = *reinterpret_cast<const vec8*>(src + 512 * kk);
        }
    }
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.f;
    if (r0 < r1) put(0);
    int at = 0;
    for (int r = r0; r < r1; r += ROWS, at ^= 1) {
        __syncthreads();
        const bool more = r + ROWS < r1;
        if (more) fetch(r + ROWS);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (r + 32 * rt >= r1) break;
            const float4 f = info[at][32 * rt + n];
            f32x16_t s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                const char* q = lds[at] + 1024 * (rt * NK + kk) + 16 * lane;
#pragma unroll
                for (int x = 0; x < PARTS; ++x) s = mfma32(k[kk], *reinterpret_cast<const vec8*>(q + x * QB), s);
            }
            // rows that do not see every position of the wave's, or stand past the end
            const int last = __float_as_int(f.z) - t0 - 8 * half;
            if (__builtin_amdgcn_ballot_w64(last < 24)) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (16 * (i >> 3) + (i & 7) <= last) sum[i] = fmaf(fast_exp2(fmaf(s[i], f.w, f.x)), f.y, sum[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[i] = fmaf(fast_exp2(fmaf(s[i], f.w, f.x)), f.y, sum[i]);
            }
        }
        if (more) put(at ^ 1);
    }
    // over the 32 lanes of a half
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[i] = sum_xor16(group_sum(sum[i], 16));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int t = t0 + 16 * (i >> 3) + 8 * half + (i & 7);
        if (n == i && t < len) {
            if (splits == 1) p.weights[(static_cast<long long>(it.seq) * p.geom.kv_heads + kvh) * p.max_seq + t] += sum[i];
            else p.wpart[it.slot0 + (static_cast<long long>(split) * p.geom.kv_heads + kvh) * len + t] = sum[i];
        }
    }
}

template <bool BF16, int D, bool SPLIT>
hipError_t launch_kind(const ChunksK& k, int kind, hipStream_t s) {
    constexpr int PARTS = chunk_parts(BF16 ? QR_DTYPE_BF16 : QR_DTYPE_F16, SPLIT);
    switch (kind) {
        case kChunkStream32: hipLaunchKernelGGL((chunks_stream32_kernel<BF16, D, PARTS>), dim3(k.units), dim3(256), 0, s, k); break;
        case kChunkStream: hipLaunchKernelGGL((chunks_stream_kernel<BF16, D, PARTS>), dim3(k.units), dim3(256), 0, s, k); break;
        case kChunkTile:
            if constexpr (PARTS < 3) hipLaunchKernelGGL((chunks_tile_kernel<BF16, D, SPLIT>), dim3(chunk_grid(k)), dim3(512), 0, s, k);
            break;
        default: hipLaunchKernelGGL((chunks_tile_weights_kernel<BF16, D, PARTS>), dim3(k.units), dim3(512), 0, s, k); break;
    }
    return hipGetLastError();
}
template <bool BF16> hipError_t launch_d(const ChunksK& k, int kind, hipStream_t s) {
    const bool split = k.act != k.dtype;
    if (k.geom.head_dim == 128) return split ? launch_kind<BF16, 128, true>(k, kind, s) : launch_kind<BF16, 128, false>(k, kind, s);
    return split ? launch_kind<BF16, 64, true>(k, kind, s) : launch_kind<BF16, 64, false>(k, kind, s);
}

}  // namespace

hipError_t launch_chunks_tile(const ChunksK& k, int kind, hipStream_t s) {
    return k.dtype == QR_DTYPE_BF16 ? launch_d<true>(k, kind, s) : launch_d<false>(k, kind, s);
}

}  // namespace qr
