// qr_kv.hpp -- the PagedKvCache handle and the checks its entry points share.
#pragma once

#include <algorithm>
#include <vector>

#include "qr_store.hpp"

struct qr_kv {
    int device = 0;
    int layers = 0, heads = 0, kv_heads = 0, head_dim = 0, max_seq = 0, dtype = 0, max_batch = 0;
    int kv_dim = 0;
    qr::PagedStore store;
    std::vector<int> seq_len;
    hipStream_t stream = nullptr;
    qr::DevBuf stage;      // host <-> device staging of rows, queries and outputs
    qr::DevBuf workspace;  // split-K partials
    qr::DevBuf steppos;    // device positions of the queries of a device-position chunk (kMaxDecodeBatch ints)
    qr::DevBuf counters;   // arrival counters of the in-kernel split merge (kDecodeCounters, zero between calls)
    hipEvent_t split_event = nullptr;  // benchmark instrumentation (qr_kv_set_split_event)
    void* scratch = nullptr;           // this device's decode scratch array (no-allocation calls)
    bool device_steps = false;         // the device copy of the page accounting is in use
    std::vector<double> turn;          // turns per position of the pairs of a rotation of turn_dim values, base turn_theta
    float turn_theta = 0.f;            // (64 powers take 1.5 us; the last call's stay)
    int turn_dim = 0;
};

namespace qr {

inline int check_handle(const qr_kv* kv) {
    if (!kv) {
        set_error("null qr_kv handle");
        return QR_ERR_INVALID_ARGUMENT;
    }
    return QR_OK;
}

// The calls that know no 8-bit cache.
inline int check_wide(const qr_kv* kv) {
    QR_CHECK_ARG(kv->dtype != QR_DTYPE_E4M3,
                 "this call takes caches of 16 and 32 bits (an 8-bit cache: append_norm_rope_dev, attention_chunks_dev without "
                 "weights, attention_forms_dev, read_as_dev)");
    return QR_OK;
}

inline int check_seq_layer(const qr_kv* kv, int seq_id, int layer) {
    QR_CHECK_ARG(seq_id >= 0 && seq_id < kv->max_batch, "seq_id %d outside [0, %d)", seq_id, kv->max_batch);
    QR_CHECK_ARG(layer >= 0 && layer < kv->layers, "layer %d outside [0, %d)", layer, kv->layers);
    return QR_OK;
}

inline int check_pos(const qr_kv* kv, int pos) {
    if (pos < 0 || pos >= kv->max_seq) {
        set_error("position %d outside [0, max_seq=%d)", pos, kv->max_seq);
        return QR_ERR_OUT_OF_RANGE;
    }
    return QR_OK;
}

inline int check_resident(const qr_kv* kv, int seq_id, int layer, int pos) {
    if (!kv->store.resident(seq_id, layer, pos)) {
        set_error("position %d of sequence %d layer %d was never appended (%d pages resident)", pos,
                  seq_id, layer, kv->store.pages_held(seq_id, layer));
        return QR_ERR_NOT_RESIDENT;
    }
    return QR_OK;
}

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

inline bool capturing(hipStream_t stream) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(stream, &st) == hipSuccess && st != hipStreamCaptureStatusNone;
}

// Host view of the page accounting and SeqLen, read back from the device after
// device-side appends (a no-op otherwise).  A device-pointer call enqueued under stream
// capture skips the read-back (it would wait for the device): its checks then use the
// host accounting, which never runs ahead of the device's (pages and SeqLen only grow
// on the device), so they can reject a position the device already holds but never
// accept one it does not.
inline int sync_host(const qr_kv* ckv, hipStream_t stream = nullptr, bool device_call = false) {
    qr_kv* kv = const_cast<qr_kv*>(ckv);
    if (!kv->store.device_ahead()) return QR_OK;
    if (device_call && capturing(stream)) return QR_OK;
    DeviceGuard dg(kv->device);
    return kv->store.pull(kv->seq_len);
}

// A call enqueued under stream capture leaves the addresses of the pool, the split
// workspace and the position buffer in the graph: from then on the pool never moves
// (growing it is an error) and a workspace that grows keeps its old allocation alive
// for the graph's replays until the handle is destroyed.
inline void note_capture(qr_kv* kv, hipStream_t stream) {
    if (!capturing(stream)) return;
    kv->store.freeze();
    kv->workspace.keep_retired();
    kv->steppos.keep_retired();
}

// Device copy of the accounting after host-side changes (once device-side appends are in use).
inline int sync_device(qr_kv* kv, hipStream_t stream) {
    if (!kv->device_steps) return QR_OK;
    return kv->store.push(kv->seq_len, stream);
}

// The split workspace may only grow outside stream capture.
inline int grow_workspace(qr_kv* kv, size_t bytes, hipStream_t st) {
    const size_t ws = std::max<size_t>(bytes, 256);
    if (ws > kv->workspace.size()) {
        QR_CHECK_ARG(!capturing(st), "the split workspace must grow to %zu bytes: make one call outside capture first", ws);
        QR_TRY(kv->workspace.ensure(ws));
    }
    return QR_OK;
}

}  // namespace qr
