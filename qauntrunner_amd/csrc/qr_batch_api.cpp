// qr_batch_api.cpp -- C ABI of the calls over chunks of several sequences (append with query / key
// norms and rotation, causal attention with weights, eviction, rows back).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

#include "qr_batch.hpp"
#include "qr_forms.hpp"
#include "qr_kv.hpp"

using namespace qr;

namespace {

// No C++ exception leaves a C entry.
template <class F> int guarded(F f) {
    clear_error();
    try {
        return f();
    } catch (const std::bad_alloc&) {
        set_error("host allocation failed");
        return QR_ERR_OUT_OF_MEMORY;
    }
}

constexpr long long kMaxRows = 1 << 24;  // (row, query head) pairs of a launch stay below 2^31

// Checks the chunks' arrays and returns their rows.  Chunks without rows take no part (their
// sequence is checked all the same).
int check_chunks(const qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows, long long* total) {
    QR_CHECK_ARG(n >= 0, "negative number of chunks %d", n);
    QR_CHECK_ARG(n == 0 || (seq_ids && pos0 && rows), "null seq_ids/pos0/rows array");
    QR_CHECK_ARG(layer >= 0 && layer < kv->layers, "layer %d outside [0, %d)", layer, kv->layers);
    *total = 0;
    for (int i = 0; i < n; ++i) {
        QR_TRY(check_seq_layer(kv, seq_ids[i], layer));
        QR_CHECK_ARG(rows[i] >= 0, "chunk %d: negative row count %d", i, rows[i]);
        if (rows[i] == 0) continue;
        QR_TRY(check_pos(kv, pos0[i]));
        if (rows[i] > kv->max_seq - pos0[i]) {
            set_error("chunk %d: positions %d..%lld reach past max_seq=%d", i, pos0[i],
                      static_cast<long long>(pos0[i]) + rows[i] - 1, kv->max_seq);
            return QR_ERR_OUT_OF_RANGE;
        }
        *total += rows[i];
    }
    QR_CHECK_ARG(*total * std::max(kv->heads, 2 * kv->kv_heads) < (1LL << 31) && *total < kMaxRows,
                 "%lld rows are too many for one call", *total);
    return QR_OK;
}

// No sequence twice among the chunks that have rows.
int check_distinct(const qr_kv* kv, int n, const int* seq_ids, const int* rows, const char* why) {
    std::vector<bool> seen(kv->max_batch, false);
    for (int i = 0; i < n; ++i) {
        if (rows && rows[i] == 0) continue;
        QR_CHECK_ARG(!seen[seq_ids[i]], "sequence %d stands in two entries: %s", seq_ids[i], why);
        seen[seq_ids[i]] = true;
    }
    return QR_OK;
}

int check_aligned(const void* p, size_t to, const char* what) {
    QR_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0, "%s must be aligned to its element size", what);
    return QR_OK;
}

// The kernels of attend_forms count slots in 32 bits up to the tile behind a list's last.
int check_near(int chunk, int prefix, int pos0, int rows) {
    if (static_cast<long long>(prefix) + pos0 + rows <= 1 << 30) return QR_OK;
    set_error("chunk %d: positions past 2^30", chunk);
    return QR_ERR_OUT_OF_RANGE;
}

const char* offset_bytes(const void* p, long long bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; }

// Attention of checked chunks (rows in all) in the forms of `f`.
int attend_forms(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows, const void* q_dev, int dtype,
                 void* attn_dev, float scale, const qr_attn_form& f, hipStream_t st) {
    FormsArgs a{};
    a.pool = kv->store.pool();
    a.page_table = kv->store.page_table_dev();
    a.geom = kv->store.geom();
    a.dtype = kv->dtype;
    a.act = dtype;
    a.heads = kv->heads;
    a.scale = scale;
    a.cap = f.cap;
    a.slopes = f.slopes_dev;
    a.window = f.window;
    // rows behind prefixes that they see of a launch, even shares of them all
    auto sees = [&](int i, int row) {
        const int len = f.prefix_len ? f.prefix_len[i] : 0;
        return form_sees_prefix(len, len + pos0[i] + row, f.first ? f.first[i] : 0, f.window);
    };
    long long all = 0;
    for (int i = 0; i < n; ++i)
        if (rows[i] && sees(i, 0)) all += rows[i];
    const long long fit = form_rows_behind(kv->heads, kv->head_dim), launches = std::max(1LL, (all + fit - 1) / fit);
    const int most = static_cast<int>((all + launches - 1) / launches);
    long long done = 0;
    int taken = 0;  // rows of chunk i that earlier launches took
    for (int i = 0; i < n;) {
        a.n = a.rows = 0;
        const long long at = done * kv->heads * kv->head_dim * dtype_size(dtype);
        a.q = offset_bytes(q_dev, at);
        a.out = const_cast<char*>(offset_bytes(attn_dev, at));
        for (int behind = 0; i < n && a.n < kBatch;) {
            const bool shares = rows[i] && sees(i, taken);
            const int take = shares ? std::min(rows[i] - taken, most - behind) : rows[i] - taken;
            if (take) {
                FormChunk& c = a.c[a.n++];
                c = {};
                c.pt_off = kv->store.pt_offset(seq_ids[i], layer);
                c.pos0 = pos0[i] + taken;
                c.rows = take;
                c.row0 = a.rows;
                c.first = f.first ? f.first[i] : 0;
                c.full = f.full ? f.full[i] : 0;
                c.pre_len = f.prefix_len ? f.prefix_len[i] : 0;
                if (c.pre_len) c.pre_off = kv->store.pt_offset(f.prefix_ids[i], layer);
                if (shares) behind += take;
                a.rows += take;
                taken += take;
            }
            if (taken < rows[i]) break;  // the rest is the next launch's
            taken = 0;
            ++i;
        }
        done += a.rows;
        if (!a.n) break;
        const FormsPlan plan = plan_forms(a);
        QR_TRY(grow_workspace(kv, plan.workspace_bytes, st));
        QR_HIP(launch_forms(a, plan, kv->workspace.get(), st));
    }
    return QR_OK;
}

// The chunks' rows in the cache's own type, or as values of another.
int read_rows(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows, int dtype, void* k_out_dev,
              void* v_out_dev, hipStream_t st) {
    QR_TRY(sync_host(kv, st, true));
    long long total = 0;
    QR_TRY(check_chunks(kv, n, seq_ids, layer, pos0, rows, &total));
    for (int i = 0; i < n; ++i)
        if (rows[i]) QR_TRY(check_resident(kv, seq_ids[i], layer, pos0[i] + rows[i] - 1));
    if (total == 0) return QR_OK;
    QR_CHECK_ARG(k_out_dev && v_out_dev, "null output rows");
    const int es = dtype_size(dtype);
    QR_TRY(check_aligned(k_out_dev, es, "k_out"));
    QR_TRY(check_aligned(v_out_dev, es, "v_out"));
    DeviceGuard dg(kv->device);
    note_capture(kv, st);
    ReadArgs a{};
    a.pool = kv->store.pool();
    a.page_table = kv->store.page_table_dev();
    a.geom = kv->store.geom();
    a.dtype = kv->dtype;
    a.act = dtype;
    long long done = 0;
    for (int i = 0; i < n;) {
        a.n = a.rows = 0;
        a.k = const_cast<char*>(offset_bytes(k_out_dev, done * kv->kv_dim * es));
        a.v = const_cast<char*>(offset_bytes(v_out_dev, done * kv->kv_dim * es));
        for (; i < n && a.n < kBatch; ++i) {
            if (!rows[i]) continue;
            a.it[a.n++] = {kv->store.pt_offset(seq_ids[i], layer), pos0[i], rows[i], a.rows, 0};
            a.rows += rows[i];
        }
        done += a.rows;
        QR_HIP(dtype == kv->dtype ? launch_read(a, st) : launch_read_as(a, st));
    }
    return QR_OK;
}

}  // namespace

extern "C" {

int qr_kv_device(const qr_kv* kv, int* out) {
    clear_error();
    QR_TRY(check_handle(kv));
    QR_CHECK_ARG(out, "null output pointer");
    *out = kv->device;
    return QR_OK;
}

int qr_kv_append_norm_rope_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows,
                               const int* rope_pos0, const void* q_dev, long long q_stride, const void* k_dev,
                               long long k_stride, const void* v_dev, long long v_stride, int dtype, void* q_out_dev,
                               const float* q_norm_dev, const float* k_norm_dev, float eps, float theta, int rotary_dim,
                               void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        const hipStream_t st = as_stream(stream);
        QR_TRY(sync_host(kv, st, true));
        long long total = 0;
        QR_TRY(check_chunks(kv, n, seq_ids, layer, pos0, rows, &total));
        QR_TRY(check_distinct(kv, n, seq_ids, rows, "its rows would race"));
        QR_CHECK_ARG(dtype_valid(dtype), "unknown row dtype %d", dtype);
        const int D = kv->head_dim;
        QR_CHECK_ARG(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 2 == 0,
                     "rotary_dim %d: an even number from 0 to head_dim %d", rotary_dim, D);
        QR_CHECK_ARG(std::isfinite(theta) && theta > 0.f, "theta must be a positive number");
        QR_CHECK_ARG(std::isfinite(eps) && eps >= 0.f, "eps must be a number of at least 0");
        if (total == 0) return QR_OK;
        QR_CHECK_ARG(k_dev && v_dev, "null k/v rows");
        QR_CHECK_ARG((q_dev == nullptr) == (q_out_dev == nullptr), "q and q_out come together");
        const long long qw = static_cast<long long>(kv->heads) * D;
        QR_CHECK_ARG((!q_dev || q_stride >= qw) && k_stride >= kv->kv_dim && v_stride >= kv->kv_dim,
                     "row strides of at least the rows' width are needed (got %lld/%lld/%lld for %lld/%d/%d)", q_stride,
                     k_stride, v_stride, qw, kv->kv_dim, kv->kv_dim);
        const int es = dtype_size(dtype);
        QR_TRY(check_aligned(q_dev, es, "q"));
        QR_TRY(check_aligned(k_dev, es, "k"));
        QR_TRY(check_aligned(v_dev, es, "v"));
        QR_TRY(check_aligned(q_out_dev, es, "q_out"));
        QR_TRY(check_aligned(q_norm_dev, 4, "q_norm"));
        QR_TRY(check_aligned(k_norm_dev, 4, "k_norm"));
        for (int i = 0; i < n; ++i) {
            if (!rows[i] || !rope_pos0) continue;
            QR_CHECK_ARG(rope_pos0[i] >= 0 && rope_pos0[i] <= 0x7FFFFFFF - rows[i], "chunk %d: rotation position %d", i, rope_pos0[i]);
        }
        DeviceGuard dg(kv->device);
        note_capture(kv, st);
        // the pool's growth for all chunks at once: it fails before any chunk's pages are taken
        long long pages = kv->store.pages_used();
        for (int i = 0; i < n; ++i)
            if (rows[i])
                pages += std::max(0, pages_of(pos0[i] + rows[i]) - kv->store.pages_held(seq_ids[i], layer));
        if (pages > kv->store.capacity()) {
            QR_CHECK_ARG(pages < (1LL << 31), "%lld pages are too many", pages);
            QR_TRY(kv->store.reserve(static_cast<int>(pages)));  // (to twice the pool where that fits)
        }
        for (int i = 0; i < n; ++i)
            if (rows[i]) QR_TRY(kv->store.ensure(seq_ids[i], layer, pos0[i] + rows[i], st));
        NormRopeArgs a{};
        a.pool = kv->store.pool();
        a.page_table = kv->store.page_table_dev();
        a.geom = kv->store.geom();
        a.dtype = kv->dtype;
        a.act = dtype;
        a.heads = kv->heads;
        a.q_stride = q_stride;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.q_norm = q_norm_dev;
        a.k_norm = k_norm_dev;
        a.eps = eps;
        a.rot = rotary_dim;
        if (kv->turn_theta != theta || kv->turn_dim != rotary_dim) {
            kv->turn.resize(rotary_dim / 2);
            for (int i = 0; i < rotary_dim / 2; ++i)
                kv->turn[i] = std::pow(static_cast<double>(theta), -2.0 * i / rotary_dim) / (2.0 * 3.14159265358979323846);
            kv->turn_theta = theta;
            kv->turn_dim = rotary_dim;
        }
        std::copy(kv->turn.begin(), kv->turn.end(), a.turn);
        long long done = 0;
        for (int i = 0; i < n;) {
            a.n = a.rows = 0;
            a.q = offset_bytes(q_dev, done * q_stride * es);
            a.k = offset_bytes(k_dev, done * k_stride * es);
            a.v = offset_bytes(v_dev, done * v_stride * es);
            a.q_out = const_cast<char*>(offset_bytes(q_out_dev, done * qw * es));
            for (; i < n && a.n < kBatch; ++i) {
                if (!rows[i]) continue;
                a.it[a.n++] = {kv->store.pt_offset(seq_ids[i], layer), pos0[i], rows[i], a.rows, (rope_pos0 ? rope_pos0 : pos0)[i], 0};
                a.rows += rows[i];
            }
            done += a.rows;
            QR_HIP(kv->dtype == QR_DTYPE_E4M3 ? launch_quant(a, st) : launch_norm_rope(a, st));
        }
        for (int i = 0; i < n; ++i)
            if (rows[i]) kv->seq_len[seq_ids[i]] = std::max(kv->seq_len[seq_ids[i]], pos0[i] + rows[i]);
        return sync_device(kv, st);
    });
}

int qr_kv_attention_chunks_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows,
                               const void* q_dev, int dtype, void* attn_dev, float* weights_dev, float scale, void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        const hipStream_t st = as_stream(stream);
        QR_TRY(sync_host(kv, st, true));
        long long total = 0;
        QR_TRY(check_chunks(kv, n, seq_ids, layer, pos0, rows, &total));
        if (weights_dev) QR_TRY(check_wide(kv));
        if (weights_dev) QR_TRY(check_distinct(kv, n, seq_ids, rows, "its weights would race"));
        QR_CHECK_ARG(dtype_valid(dtype), "unknown q dtype %d", dtype);
        QR_CHECK_ARG(std::isfinite(scale), "scale must be a number");
        for (int i = 0; i < n; ++i)
            if (rows[i] && kv->dtype == QR_DTYPE_E4M3) QR_TRY(check_near(i, 0, pos0[i], rows[i]));
        for (int i = 0; i < n; ++i)
            if (rows[i]) QR_TRY(check_resident(kv, seq_ids[i], layer, pos0[i] + rows[i] - 1));
        if (total == 0) return QR_OK;
        QR_CHECK_ARG(q_dev && attn_dev, "null q/attn pointer");
        const int es = dtype_size(dtype);
        QR_TRY(check_aligned(q_dev, es, "q"));
        QR_TRY(check_aligned(attn_dev, es, "attn"));
        QR_TRY(check_aligned(weights_dev, 4, "weights"));
        DeviceGuard dg(kv->device);
        note_capture(kv, st);
        if (kv->dtype == QR_DTYPE_E4M3) return attend_forms(kv, n, seq_ids, layer, pos0, rows, q_dev, dtype, attn_dev, scale, {}, st);
        ChunksArgs a{};
        a.pool = kv->store.pool();
        a.page_table = kv->store.page_table_dev();
        a.geom = kv->store.geom();
        a.dtype = kv->dtype;
        a.act = dtype;
        a.heads = kv->heads;
        a.weights = weights_dev;
        a.max_seq = kv->max_seq;
        a.scale = scale;
        long long done = 0;
        for (int i = 0; i < n;) {
            a.n = a.rows = 0;
            const long long at = done * kv->heads * kv->head_dim * es;
            a.q = offset_bytes(q_dev, at);
            a.out = const_cast<char*>(offset_bytes(attn_dev, at));
            for (; i < n && a.n < kBatch; ++i) {
                if (!rows[i]) continue;
                ChunkItem& it = a.it[a.n++];
                it = {};
                it.pt_off = kv->store.pt_offset(seq_ids[i], layer);
                it.seq = seq_ids[i];
                it.pos0 = pos0[i];
                it.rows = rows[i];
                it.row0 = a.rows;
                a.rows += rows[i];
            }
            done += a.rows;
            if (!a.n) break;
            const ChunksPlan plan = plan_chunks(a);
            QR_TRY(grow_workspace(kv, plan.workspace_bytes, st));
            QR_HIP(launch_chunks(a, plan, kv->workspace.get(), st));
        }
        return QR_OK;
    });
}

int qr_kv_evict_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* len, int first, int heavy, int recent,
                    const float* weights_dev, float* kept_weights_dev, int* kept_dev, void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        QR_TRY(check_wide(kv));
        const hipStream_t st = as_stream(stream);
        QR_TRY(sync_host(kv, st, true));
        QR_CHECK_ARG(n >= 0, "negative number of sequences %d", n);
        QR_CHECK_ARG(n == 0 || (seq_ids && len), "null seq_ids/len array");
        QR_CHECK_ARG(layer >= 0 && layer < kv->layers, "layer %d outside [0, %d)", layer, kv->layers);
        QR_CHECK_ARG(first >= 0 && heavy >= 0 && recent >= 0, "negative budget (first %d, heavy %d, recent %d)", first, heavy, recent);
        const long long keep = static_cast<long long>(first) + heavy + recent;
        QR_CHECK_ARG(keep >= 1 && keep <= kv->max_seq, "a budget of %lld positions outside [1, max_seq=%d]", keep, kv->max_seq);
        for (int i = 0; i < n; ++i) {
            QR_TRY(check_seq_layer(kv, seq_ids[i], layer));
            QR_CHECK_ARG(len[i] >= 0, "entry %d: negative length %d", i, len[i]);
            if (len[i] == 0) continue;
            QR_TRY(check_pos(kv, len[i] - 1));
            QR_TRY(check_resident(kv, seq_ids[i], layer, len[i] - 1));
        }
        QR_TRY(check_distinct(kv, n, seq_ids, nullptr, "its positions would race"));
        if (n == 0) return QR_OK;
        QR_CHECK_ARG(weights_dev && kept_weights_dev && kept_dev, "null weights/kept_weights/kept pointer");
        QR_TRY(check_aligned(weights_dev, 4, "weights"));
        QR_TRY(check_aligned(kept_weights_dev, 4, "kept_weights"));
        QR_TRY(check_aligned(kept_dev, 4, "kept"));
        DeviceGuard dg(kv->device);
        note_capture(kv, st);
        EvictArgs a{};
        a.pool = kv->store.pool();
        a.page_table = kv->store.page_table_dev();
        a.geom = kv->store.geom();
        a.dtype = kv->dtype;
        a.first = first;
        a.heavy = heavy;
        a.recent = recent;
        a.weights = weights_dev;
        a.kept_weights = kept_weights_dev;
        a.max_seq = kv->max_seq;
        a.kept = kept_dev;
        for (int i = 0; i < n;) {
            for (a.n = 0; i < n && a.n < kBatch; ++i) a.it[a.n++] = {kv->store.pt_offset(seq_ids[i], layer), seq_ids[i], len[i], i};
            // a captured call cannot grow the workspace: without room for it, each row is selected by one workgroup
            const size_t bytes = evict_workspace_bytes(a);
            const bool room = !capturing(st) || kv->workspace.size() >= bytes;
            if (room && bytes) QR_TRY(grow_workspace(kv, bytes, st));
            QR_HIP(launch_evict(a, room && bytes ? kv->workspace.get() : nullptr, st));
        }
        return QR_OK;
    });
}

int qr_kv_attention_forms_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows,
                              const void* q_dev, int dtype, void* attn_dev, float scale, const qr_attn_form* form,
                              void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        const hipStream_t st = as_stream(stream);
        QR_TRY(sync_host(kv, st, true));
        long long total = 0;
        QR_TRY(check_chunks(kv, n, seq_ids, layer, pos0, rows, &total));
        QR_CHECK_ARG(dtype_valid(dtype), "unknown q dtype %d", dtype);
        QR_CHECK_ARG(std::isfinite(scale), "scale must be a number");
        const qr_attn_form f = form ? *form : qr_attn_form{};
        QR_CHECK_ARG(f.cap == 0.f || (f.cap >= 1e-3f && f.cap <= 1e6f), "cap must be 0 or a number from 0.001 to 1000000");
        QR_CHECK_ARG(f.window >= 0, "negative window %d", f.window);
        QR_CHECK_ARG((f.prefix_ids == nullptr) == (f.prefix_len == nullptr), "prefix_ids and prefix_len come together");
        for (int i = 0; i < n; ++i) {
            if (!rows[i]) continue;
            const int len = f.prefix_len ? f.prefix_len[i] : 0;
            QR_CHECK_ARG(len >= 0, "chunk %d: negative prefix length %d", i, len);
            if (len) {
                QR_TRY(check_seq_layer(kv, f.prefix_ids[i], layer));
                QR_TRY(check_pos(kv, len - 1));
                QR_TRY(check_resident(kv, f.prefix_ids[i], layer, len - 1));
            }
            QR_TRY(check_near(i, len, pos0[i], rows[i]));
            const int first = f.first ? f.first[i] : 0, full = f.full ? f.full[i] : 0;
            QR_CHECK_ARG(first >= 0 && full >= 0, "chunk %d: negative first %d or full %d", i, first, full);
            QR_TRY(check_near(i, 0, full, 0));
            const int last = std::max(pos0[i] + rows[i], full - len) - 1;  // of its own slots
            QR_TRY(check_pos(kv, last));
            QR_TRY(check_resident(kv, seq_ids[i], layer, last));
        }
        if (total == 0) return QR_OK;
        QR_CHECK_ARG(q_dev && attn_dev, "null q/attn pointer");
        const int es = dtype_size(dtype);
        QR_TRY(check_aligned(q_dev, es, "q"));
        QR_TRY(check_aligned(attn_dev, es, "attn"));
        QR_TRY(check_aligned(f.slopes_dev, 4, "slopes"));
        DeviceGuard dg(kv->device);
        note_capture(kv, st);
        return attend_forms(kv, n, seq_ids, layer, pos0, rows, q_dev, dtype, attn_dev, scale, f, st);
    });
}

int qr_kv_read_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows, void* k_out_dev,
                   void* v_out_dev, void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        QR_TRY(check_wide(kv));
        return read_rows(kv, n, seq_ids, layer, pos0, rows, kv->dtype, k_out_dev, v_out_dev, as_stream(stream));
    });
}

int qr_kv_read_as_dev(qr_kv* kv, int n, const int* seq_ids, int layer, const int* pos0, const int* rows, int dtype,
                      void* k_out_dev, void* v_out_dev, void* stream) {
    return guarded([&]() -> int {
        QR_TRY(check_handle(kv));
        QR_CHECK_ARG(dtype_valid(dtype), "unknown row dtype %d", dtype);
        return read_rows(kv, n, seq_ids, layer, pos0, rows, dtype, k_out_dev, v_out_dev, as_stream(stream));
    });
}

}  // extern "C"
