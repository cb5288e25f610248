// qr_forms.hip -- plan, launch and the joining of parts of attention in its other forms and behind shared prefixes, gfx950.
#include "qr_forms.hpp"

#include <algorithm>
#include <cmath>

namespace qr {
namespace {

constexpr int kThreads = 256;

// out of a row's parts: a wave per (row, head), the parts' sums weighed by 2^(m - M).  A row that saw nothing is zeros.  A
// partial's sums are D / 4 lanes' float4, so that a wave reads several of them at once, and each lane four ahead (VEC; other
// head sizes: a lane every 64th value of one).
template <bool VEC>
__global__ void __launch_bounds__(kThreads) forms_merge_kernel(const FormsK p, int rows) {
    const long long at = static_cast<long long>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(at / p.heads)), h = __builtin_amdgcn_readfirstlane(static_cast<int>(at % p.heads));
    if (row >= rows) return;
    const int e = batch_find(p.chunks, row, [&](int i) { return p.c[i].row0; });
    const FormRows c = p.c[e];
    if (c.parts == 1) return;
    const int D = p.geom.head_dim, lane = threadIdx.x & 63;
    const long long slot = c.slot0 + (static_cast<long long>(row - c.row0) * p.heads + h) * c.parts;
    const long long to = (static_cast<long long>(row) * p.heads + h) * D;
    float M = -INFINITY;
    for (int x = lane; x < c.parts; x += 64) M = fmaxf(M, p.part_ml[slot + x].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    // weight of a part: nothing of one that saw nothing
    auto weight = [&](float2 ml) __attribute__((always_inline)) { return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - M); };
    float L = 0.f;
    if (VEC) {
        const int gl = D / 4, per = 64 / gl, sub = lane / gl, d = 4 * (lane % gl);  // gl: 16 or 32
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        for (int x0 = sub; x0 < c.parts; x0 += 4 * per) {
            float4 a[4];
            float2 ml[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = min(x0 + per * i, c.parts - 1);
                ml[i] = p.part_ml[slot + x];
                a[i] = *reinterpret_cast<const float4*>(p.part_acc + (slot + x) * D + d);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = x0 + per * i < c.parts ? weight(ml[i]) : 0.f;
                if (w == 0.f) continue;  // (its sums may not have been written)
                L = fmaf(ml[i].y, w, L);
                o[0] = fmaf(a[i].x, w, o[0]);
                o[1] = fmaf(a[i].y, w, o[1]);
                o[2] = fmaf(a[i].z, w, o[2]);
                o[3] = fmaf(a[i].w, w, o[3]);
            }
        }
        for (int x = gl; x < 64; x <<= 1) {
            L += __shfl_xor(L, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
        }
        if (sub) return;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (p.act == QR_DTYPE_F32) {
            const float4 y = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            __builtin_memcpy(static_cast<float*>(p.out) + to + d, &y, 16);
        } else {
            uint16_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = f32_to_out16(o[i] * inv, p.act);
            __builtin_memcpy(static_cast<uint16_t*>(p.out) + to + d, b, 8);
        }
        return;
    }
    constexpr int NC = kGenericMaxDim / 64;
    float o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = 0.f;
    for (int x = 0; x < c.parts; ++x) {
        const float2 ml = p.part_ml[slot + x];
        const float w = weight(ml);
        if (w == 0.f) continue;
        L = fmaf(ml.y, w, L);
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (lane + 64 * i < D) o[i] = fmaf(p.part_acc[(slot + x) * D + lane + 64 * i], w, o[i]);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (lane + 64 * i < D) store_out(p.out, p.act, to + lane + 64 * i, L == 0.f ? 0.f : o[i] / L);
}

struct Shape {
    int rows, tile;  // (query, head) rows of a block, slots of a tile
    int target;      // units that run at once
    int least;       // tiles of a part, at least
};
Shape shape_of(int kind) {
    switch (kind) {
        case kFormStream: return {32, 32, 512, 8};
        case kFormTiles: return {128, 64, 512, 8};
        case kFormF32Half: return {16, 16, 512, 8};
        case kFormF32: return {32, 16, 512, 8};
        default: return {kFormAnyRows, kFormAnyTile, 1024, 2};
    }
}
int kind_of(const FormsArgs& a, int rows) {
    const int D = a.geom.head_dim;
    if ((D != 64 && D != 128) || a.heads % a.geom.kv_heads) return kFormAny;
    const long long n = static_cast<long long>(rows) * (a.heads / a.geom.kv_heads);
    if (a.dtype == QR_DTYPE_F32) return n <= 16 ? kFormF32Half : kFormF32;
    return n <= 32 ? kFormStream : kFormTiles;
}
hipError_t launch(const FormsK& k, int units, hipStream_t s) {
    if (k.it[0].kind == kFormAny) return launch_forms_any(k, units, s);
    if (k.dtype == QR_DTYPE_F32) return launch_forms_f32(k, units, s);
    if (k.dtype == QR_DTYPE_F16) return launch_forms_f16(k, units, s);
    return k.dtype == QR_DTYPE_BF16 ? launch_forms_bf16(k, units, s) : launch_forms_e4m3(k, units, s);
}

// Tiles of the slots that row j of an item sees.
int tiles_of(const FormsPlan& p, const FormItem& it, int window, int j, int tile) {
    int c = it.c0;
    while (c + 1 < it.c0 + it.nc && p.c[c + 1].row0 <= it.row0 + j) ++c;
    const FormSpan s = form_span(p.c[c], it.row0 + j, window, it.base, it.keys);
    return s.lo > s.hi ? 0 : s.hi / tile - s.lo / tile + 1;
}

}  // namespace

FormsPlan plan_forms(const FormsArgs& a) {
    FormsPlan p{};
    const int kv = a.geom.kv_heads, g = (a.heads + kv - 1) / kv;
    auto add = [&](int pt_off, int c0, int nc, int rows, int base, int keys) {
        FormItem& it = p.it[p.n];
        it = {};
        it.pt_off = pt_off;
        it.c0 = c0;
        it.nc = nc;
        it.row0 = a.c[c0].row0;
        it.rows = rows;
        it.base = base;
        it.keys = keys;
        it.kind = kind_of(a, rows);
        ++p.n;
    };
    for (int i = 0; i < a.n; ++i) {
        const FormChunk& c = a.c[i];
        p.c[i] = {c.row0, c.rows, c.pre_len + c.pos0, c.first, c.full, 0, 0};
    }
    // the prefixes, then the chunks' own keys
    for (int i = 0; i < a.n;) {
        const FormChunk& c = a.c[i];
        if (!c.pre_len) {
            ++i;
            continue;
        }
        int j = i, rows = 0;
        for (; j < a.n && a.c[j].pre_len == c.pre_len && a.c[j].pre_off == c.pre_off; ++j) rows += a.c[j].rows;
        add(c.pre_off, i, j - i, rows, 0, c.pre_len);
        i = j;
    }
    for (int i = 0; i < a.n; ++i) {
        const FormChunk& c = a.c[i];
        add(c.pt_off, i, 1, c.rows, c.pre_len, std::max(c.pos0 + c.rows, c.full - c.pre_len));
    }
    // tiles of a part: the fewest with which the units still run at once, or the partials stay below 256 MB
    struct Cost {
        long long blocks;
        int avg, most;
    } cost[kFormItems];
    for (int i = 0; i < p.n; ++i) {
        FormItem& it = p.it[i];
        const Shape s = shape_of(p.it[i].kind);
        it.blocks = static_cast<int>((static_cast<long long>(it.rows) * g + s.rows - 1) / s.rows);
        const int x = tiles_of(p, it, a.window, 0, s.tile), y = tiles_of(p, it, a.window, it.rows - 1, s.tile);
        int most = std::max(x, y);
        for (int c = 1; c < it.nc; ++c) most = std::max(most, tiles_of(p, it, a.window, p.c[it.c0 + c].row0 - it.row0, s.tile));
        cost[i] = {static_cast<long long>(it.blocks) * kv, std::max(1, (x + y + 1) / 2), std::max(1, most)};
    }
    const long long partial = static_cast<long long>(a.geom.head_dim) * 4 + 8;
    for (int kind = 0; kind < kFormKinds; ++kind) {
        const Shape s = shape_of(kind);
        int lo = s.least, hi = s.least;
        for (int i = 0; i < p.n; ++i)
            if (p.it[i].kind == kind) hi = std::max(hi, cost[i].most);
        auto fits = [&](int per) {
            long long units = 0, bytes = 0;
            for (int i = 0; i < p.n; ++i)
                if (p.it[i].kind == kind) {
                    units += cost[i].blocks * ((cost[i].avg + per - 1) / per);
                    bytes += partial * p.it[i].rows * a.heads * ((cost[i].avg + per - 1) / per);
                }
            return units <= s.target && bytes <= (256LL << 20);
        };
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            if (fits(mid)) hi = mid;
            else lo = mid + 1;
        }
        for (int i = 0; i < p.n; ++i)
            if (p.it[i].kind == kind) p.it[i].splits = (cost[i].avg + lo - 1) / lo;
    }
    for (int i = 0; i < p.n; ++i) {
        FormItem& it = p.it[i];
        it.part0 = p.c[it.c0].parts;  // the chunks of an item have had the same lists before it
        for (int c = 0; c < it.nc; ++c) p.c[it.c0 + c].parts += it.splits;
    }
    long long slots = 0;
    for (int i = 0; i < a.n; ++i) {
        if (p.c[i].parts == 1) continue;
        p.merge = true;
        p.c[i].slot0 = slots;
        slots += static_cast<long long>(p.c[i].rows) * a.heads * p.c[i].parts;
    }
    p.part_ml = static_cast<size_t>(slots) * a.geom.head_dim * 4;
    p.workspace_bytes = p.part_ml + static_cast<size_t>(slots) * 8;
    return p;
}

hipError_t launch_forms(const FormsArgs& a, const FormsPlan& plan, void* workspace, hipStream_t stream) {
    FormsK k{};
    std::copy(plan.c, plan.c + a.n, k.c);
    k.chunks = a.n;
    k.pool = static_cast<const char*>(a.pool);
    k.page_table = a.page_table;
    k.geom = a.geom;
    k.dtype = a.dtype;
    k.act = a.act;
    k.heads = a.heads;
    k.q = a.q;
    k.out = a.out;
    k.qscale = a.scale * kLog2e;
    k.cap = a.cap * kLog2e;
    k.slopes = a.slopes;
    k.window = a.window;
    k.part_acc = static_cast<float*>(workspace);
    k.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + plan.part_ml);
    int units = 0;
    for (int pass = 0; pass < 2; ++pass)  // the items of many rows first: theirs are the longest units
        for (int i = 0; i < plan.n; ++i) {
            if ((plan.it[i].kind == kFormTiles || plan.it[i].kind == kFormF32) != (pass == 0)) continue;
            FormItem& it = k.it[k.n++] = plan.it[i];
            it.unit0 = units;
            units += it.blocks * it.splits * a.geom.kv_heads;
        }
    const hipError_t e = launch(k, units, stream);
    if (e != hipSuccess) return e;
    if (plan.merge) {
        const long long waves = static_cast<long long>(a.rows) * a.heads;
        const dim3 grid(static_cast<unsigned>((waves + 3) / 4));
        if (a.geom.head_dim == 64 || a.geom.head_dim == 128) hipLaunchKernelGGL(forms_merge_kernel<true>, grid, dim3(kThreads), 0, stream, k, a.rows);
        else hipLaunchKernelGGL(forms_merge_kernel<false>, grid, dim3(kThreads), 0, stream, k, a.rows);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace qr
