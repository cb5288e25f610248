// qr_forms.hip -- plan, launch and the joining of parts of attention in its other forms and behind shared prefixes, gfx950.
#include "qr_forms.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace qr {
namespace {

constexpr int kThreads = 256;

// out of a row's parts: a wave per (row, head), the parts' sums weighed by 2^(m - M).  A row that saw nothing is zeros.  A
// partial's sums are D / 4 lanes' float4, so that a wave reads several of them at once, and each lane four ahead (VEC; other
// head sizes: a lane every 64th value of one).  Bound by latency: 4 to 5 us for 16 to 1500 rows, 8 for 115 rows of 64 heads in some
// ten parts.
template <bool VEC>
__global__ void __launch_bounds__(kThreads) forms_merge_kernel(const FormsK p, int rows) {
    const long long at = static_cast<long long>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    const int of = __builtin_amdgcn_readfirstlane(static_cast<int>(at / p.heads)), h = __builtin_amdgcn_readfirstlane(static_cast<int>(at % p.heads));
    if (of >= rows) return;
    const int e = batch_find(p.chunks, of, [&](int i) { return p.c[i].full; });  // (here a chunk's first row of the merge)
    const FormRows c = p.c[e];
    const int row = c.row0 + of - c.full;
    const int D = p.geom.head_dim, lane = threadIdx.x & 63;
    const long long slot = c.slot0 + (static_cast<long long>(row - c.row0) * p.heads + h) * c.parts;
    const long long to = (static_cast<long long>(row) * p.heads + h) * D;
    if (p.part_ml[slot].y == kFormDone) return;  // one part wrote the output
    float M = -INFINITY;
    for (int x = lane; x < c.parts; x += 64) M = fmaxf(M, p.part_ml[slot + x].x);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    auto saw_nothing = [](float2 ml) __attribute__((always_inline)) { return ml.x == -INFINITY && ml.y == 0.f; };  // (its sums may not have been written)
    auto weight = [&](float2 ml) __attribute__((always_inline)) { return ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - M); };  // (1: a sum that is no number)
    float L = 0.f;
    if (VEC) {
        const int gl = D / 4, per = 64 / gl, sub = lane / gl, d = 4 * (lane % gl);  // gl: 16, 32 or 64
        float o[4];
        auto join = [&](auto shown) __attribute__((always_inline)) {
            L = o[0] = o[1] = o[2] = o[3] = 0.f;
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
                    if (x0 + per * i >= c.parts || saw_nothing(ml[i])) continue;
                    const float w = weight(ml[i]);
                    L = fmaf(ml[i].y, w, L);
                    auto add = [&](float& to, float of) __attribute__((always_inline)) { to = decltype(shown)::value ? to + form_weighed(of, w) : fmaf(of, w, to); };
                    add(o[0], a[i].x);
                    add(o[1], a[i].y);
                    add(o[2], a[i].z);
                    add(o[3], a[i].w);
                }
            }
            for (int x = gl; x < 64; x <<= 1) {
                L += __shfl_xor(L, x);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], x);
            }
        };
        join(std::false_type{});
        const float sum = (o[0] + o[1]) + (o[2] + o[3]);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(sum != sum && L == L) != 0, 0)) join(std::true_type{});
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
        if (saw_nothing(ml)) continue;
        const float w = weight(ml);
        L = fmaf(ml.y, w, L);
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (lane + 64 * i < D) o[i] += form_weighed(p.part_acc[(slot + x) * D + lane + 64 * i], w);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
        if (lane + 64 * i < D) store_out(p.out, p.act, to + lane + 64 * i, L == 0.f ? 0.f : o[i] / L);
}

// Queries that the MFMA tiles take in one part.
bool whole_queries(const FormsArgs& a) { return a.act == (a.dtype == QR_DTYPE_F16 ? QR_DTYPE_F16 : QR_DTYPE_BF16); }

// What a unit of a kernel takes, in microseconds: a tile of it, its start and end, and its share of what runs at once on a CU.
// Measured (D = 128): a tile of 64 slots 2.2 for 128 rows, 1.3 for 64 (8 bits, whose codes
// become operands whatever the rows: 3.0 and 2.5), 1.4 times as long with capped scores and 2.2 times in parts; a
// streamed step of 32 slots by its bytes, 5 TB/s over all CUs; fp32 MFMAs' steps of 16 slots by their bytes for 16 rows, by their
// MFMAs for 32.  (With 0.4 to 1.5 times the part that this gives, the cases it was tried on took 0 to 30% longer.  16 verify chunks of 64
// heads behind two prefixes of 16001 positions, 8 bits: 136 us with the tiles of 16 bits, 100 with these.)
struct Shape {
    float tile, start, share;
    int least;  // tiles that a part has at least
};
constexpr float kCus = 256.f;
Shape shape_of(const FormsArgs& a, int kind) {
    const float wide = a.geom.head_dim / 128.f;
    const float tile = wide * (whole_queries(a) ? 1.f : 2.2f) * (a.cap > 0.f ? 1.4f : a.slopes ? 1.2f : 1.f);
    // one workgroup on a CU at head size 256, which has it to itself
    auto alone = [&](Shape s) { return a.geom.head_dim == 256 ? Shape{0.5f * s.tile, s.start, 1.f, s.least} : s; };
    switch (kind) {
        case kFormStream: return {wide * (a.geom.scaled() ? 0.9f : 1.7f), 5.f, 0.5f, 8};
        case kFormTilesHalf: return {(a.geom.scaled() ? 2.5f : 1.3f) * tile, 6.f, 0.5f, 4};
        case kFormTiles: return {(a.geom.scaled() ? 3.f : 2.2f) * tile, 6.f, 0.5f, 4};
        case kFormF32Half: return alone({wide * (a.dtype == QR_DTYPE_F32 ? 1.7f : 1.f), 5.f, 0.5f, 8});
        case kFormF32: return alone({wide * 1.f, 5.f, 0.5f, 8});
        default: return {4.f, 5.f, 0.25f, 2};
    }
}
int kind_of(const FormsArgs& a, int rows) {
    const int D = a.geom.head_dim;
    if ((D != 64 && D != 96 && D != 128 && D != 256) || a.heads % a.geom.kv_heads) return kFormAny;
    const long long n = static_cast<long long>(rows) * (a.heads / a.geom.kv_heads);
    if (a.dtype == QR_DTYPE_F32 || !(a.geom.mfma_layout & 1)) return n <= 16 ? kFormF32Half : kFormF32;
    return n <= 32 ? kFormStream : n <= 64 ? kFormTilesHalf : kFormTiles;
}
hipError_t launch(const FormsK& k, int units, hipStream_t s) {
    if (k.it[0].kind == kFormAny) return launch_forms_any(k, units, s);
    if (k.it[0].kind == kFormF32Half || k.it[0].kind == kFormF32) return launch_forms_f32(k, units, s);
    if (k.dtype == QR_DTYPE_F16) return launch_forms_f16(k, units, s);
    return k.dtype == QR_DTYPE_BF16 ? launch_forms_bf16(k, units, s) : launch_forms_e4m3(k, units, s);
}

int per_of(const Shape& s, float part) { return std::max(s.least, static_cast<int>(std::min(1e9f, part / s.tile + 0.999f))); }

// Blocks of an item, of which some stand for the others: their tiles.
struct Sample {
    int item, tiles;
    float units;  // of this length, all kv heads
};
// The time of a part with which the units and the partials' way through memory take least: whole blocks, an even share of what
// the CUs run at once, or some between and beyond.
float best_part(const FormsArgs& a, const FormsPlan& p, const Sample* smp, int n) {
    const int kv = a.geom.kv_heads;
    const float partial = form_partial_bytes(a.geom.head_dim) * 0.5e-6f;  // written and read at 4 TB/s
    Shape shape[kFormKinds];
    for (int k = 0; k < kFormKinds; ++k) shape[k] = shape_of(a, k);
    float whole = 0.f, work = 0.f;
    for (int i = 0; i < n; ++i) {
        const Shape& s = shape[p.it[smp[i].item].kind];
        whole = std::max(whole, smp[i].tiles * s.tile);
        work += smp[i].units * smp[i].tiles * s.tile * s.share;
    }
    auto cost = [&](float part) {
        float busy = 0.f, used = 0.f, longest = 0.f, parts = 0.f;
        for (int i = 0; i < n; ++i) {
            const FormItem& it = p.it[smp[i].item];
            const Shape& s = shape[it.kind];
            const int per = per_of(s, part), c = (smp[i].tiles + per - 1) / per;
            const float t = s.start + s.tile * static_cast<float>((smp[i].tiles + c - 1) / c);
            busy += smp[i].units * c * t * s.share;
            used += smp[i].units * c * s.share;
            longest = std::max(longest, t);
            const long long rows = static_cast<long long>(it.rows) * (a.heads / kv);
            if (c > 1 || p.c[it.c0].parts) parts += smp[i].units * c * static_cast<float>(std::min<long long>(form_rows(it.kind), rows));
        }
        const float run = used <= kCus ? longest : std::max(longest, busy / kCus + 0.25f * longest);
        return run + parts * partial + (parts > 0.f ? 4.f : 0.f);
    };
    float best = whole, least = cost(whole);
    auto consider = [&](float part) {
        const float us = cost(part);
        if (us < least) {
            least = us;
            best = part;
        }
    };
    const float even = work / kCus;
    for (const float f : {0.35f, 0.5f, 0.7f, 0.85f, 1.f, 1.04f, 1.08f, 1.15f, 1.25f, 1.4f, 1.7f, 2.f, 3.f})
        if (even * f < whole) consider(even * f);
    // longer parts where the partials would pass their bytes
    for (;; best *= 1.25f) {
        int parts[kBatch] = {}, longest = 1;
        for (int i = 0; i < n;) {
            const FormItem& it = p.it[smp[i].item];
            const int per = per_of(shape[it.kind], best);
            int most = 1, j = i;
            for (; j < n && smp[j].item == smp[i].item; ++j) most = std::max(most, (smp[j].tiles + per - 1) / per);
            for (int c = 0; c < it.nc; ++c) parts[it.c0 + c] += most;
            longest = std::max(longest, most);
            i = j;
        }
        long long bytes = 0;
        for (int c = 0; c < a.n; ++c)
            if (parts[c] > 1) bytes += form_partial_bytes(a.geom.head_dim) * a.c[c].rows * a.heads * parts[c];
        if (longest == 1 || bytes <= kFormPartialBytes) return best;
    }
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
    // the prefixes that some row of a chunk sees, then the chunks' own keys
    auto sees = [&](int i) { return form_sees_prefix(a.c[i].pre_len, p.c[i].p0, a.c[i].first, a.window); };
    for (int i = 0; i < a.n;) {
        const FormChunk& c = a.c[i];
        if (!sees(i)) {
            ++i;
            continue;
        }
        int j = i, rows = 0;
        for (; j < a.n && a.c[j].pre_len == c.pre_len && a.c[j].pre_off == c.pre_off && sees(j); ++j) rows += a.c[j].rows;
        add(c.pre_off, i, j - i, rows, 0, c.pre_len);
        i = j;
    }
    for (int i = 0; i < a.n; ++i) {
        const FormChunk& c = a.c[i];
        add(c.pt_off, i, 1, c.rows, c.pre_len, std::max(c.pos0 + c.rows, c.full - c.pre_len));
    }
    for (int i = 0; i < p.n; ++i)  // lists of each row, for now
        for (int c = 0; c < p.it[i].nc; ++c) ++p.c[p.it[i].c0 + c].parts;
    for (int i = 0; i < a.n; ++i) --p.c[i].parts;
    constexpr int kSamples = 8;
    Sample smp[kFormItems * kSamples];
    int n = 0;
    for (int i = 0; i < p.n; ++i) {
        FormItem& it = p.it[i];
        const int rows = form_rows(it.kind), tile = form_tile(it.kind);
        it.blocks = static_cast<int>((static_cast<long long>(it.rows) * g + rows - 1) / rows);
        it.per = 1;
        it.splits = 0x7FFFFFFF;
        if (it.nc > 1) {  // (rows of many chunks: whatever one of them sees of the prefix)
            int tiles = 1;
            for (int c = 0; c < it.nc; ++c) {
                const FormRows& r = p.c[it.c0 + c];
                const FormSpan x = form_span(r, r.row0, a.window, it.base, it.keys);
                if (x.lo <= x.hi) tiles = std::max(tiles, x.hi / tile - x.lo / tile + 1);
            }
            smp[n++] = {i, tiles, static_cast<float>(it.blocks) * kv};
            continue;
        }
        const int m = std::min(it.blocks, kSamples);
        for (int x = 0; x < m; ++x) {
            const int b = m == 1 ? 0 : static_cast<int>(static_cast<long long>(it.blocks - 1) * x / (m - 1));
            smp[n++] = {i, form_parts(it, p.c[it.c0], a.window, g, rows, tile, b), static_cast<float>(it.blocks) * kv / m};
        }
    }
    const float part = best_part(a, p, smp, n);
    for (int x = 0; x < n; ++x) {
        FormItem& it = p.it[smp[x].item];
        const int per = per_of(shape_of(a, it.kind), part);
        if (x == 0 || smp[x - 1].item != smp[x].item) it.splits = 1;
        it.splits = std::max(it.splits, (smp[x].tiles + per - 1) / per);
        it.per = it.nc == 1 ? per : 0;
        p.us[smp[x].item] = std::max(p.us[smp[x].item], shape_of(a, it.kind).tile * static_cast<float>(std::min(per, smp[x].tiles)));
    }
    for (int i = 0; i < a.n; ++i) p.c[i].parts = 0;
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
    p.part_ml = (static_cast<size_t>(slots) * a.geom.head_dim * 4 + 15) & ~static_cast<size_t>(15);
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
    const int g = (a.heads + a.geom.kv_heads - 1) / a.geom.kv_heads;
    // the longest units first
    int order[kFormItems];
    float us[kFormItems];
    for (int i = 0; i < plan.n; ++i) {
        order[i] = i;
        us[i] = plan.us[i];
    }
    std::sort(order, order + plan.n, [&](int x, int y) { return us[x] != us[y] ? us[x] > us[y] : x < y; });
    int units = 0;
    for (int i = 0; i < plan.n; ++i) {
        FormItem& it = k.it[k.n++] = plan.it[order[i]];
        it.unit0 = units;
        int n = it.blocks * it.splits;
        if (it.per && it.splits > 1) {
            n = 0;
            for (int b = 0; b < it.blocks; ++b) n += form_parts(it, k.c[it.c0], a.window, g, form_rows(it.kind), form_tile(it.kind), b);
        }
        units += n * a.geom.kv_heads;
    }
    const hipError_t e = launch(k, units, stream);
    if (e != hipSuccess) return e;
    if (plan.merge) {
        // the chunks whose rows have several parts
        k.chunks = 0;
        int rows = 0;
        for (int i = 0; i < a.n; ++i) {
            if (plan.c[i].parts == 1) continue;
            FormRows& c = k.c[k.chunks++] = plan.c[i];
            c.full = rows;  // (its first row of the merge)
            rows += c.rows;
        }
        const long long waves = static_cast<long long>(rows) * a.heads;
        const dim3 grid(static_cast<unsigned>((waves + 3) / 4));
        if (a.geom.head_dim == 64 || a.geom.head_dim == 128 || a.geom.head_dim == 256) hipLaunchKernelGGL(forms_merge_kernel<true>, grid, dim3(kThreads), 0, stream, k, rows);
        else hipLaunchKernelGGL(forms_merge_kernel<false>, grid, dim3(kThreads), 0, stream, k, rows);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace qr
