// vk_bkv_capi.hip — the block-scaled KV cache behind include/vokra_hip.h:
// checks, buffers, and the host-array forms of the calls.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <new>

#include "../../include/vokra_hip.h"
#include "vk_bkv.h"
#include "vk_launch.h"

struct vokra_hip_bkv {
    vokra_hip_ctx* ctx = nullptr;
    BkvView v = {};
    size_t max_rows = 0;
    float* part = nullptr;  // the context's partial results of split attention
    // host-array calls: item ids (4 x kBkvMaxItems ints) and, for write, attn
    // and read, rows in and out (grown by those calls only)
    int* items = nullptr;
    float* rows = nullptr;
    size_t rows_cap = 0;
    // what the host knows of the current step
    size_t step_n = 0, step_rows = 0, step_count = 0, step_len = 0;
};

namespace {

using vk::ctx_fail;
constexpr int BAD = VOKRA_HIP_ERROR_INVALID_ARGUMENT;

#define BK_TRY(call, what)                                                                                       \
    do {                                                                                                         \
        hipError_t _e = (call);                                                                                  \
        if (_e != hipSuccess)                                                                                    \
            return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "%s: %s", (what), hipGetErrorString(_e));       \
    } while (0)
#define BK_ST(x)             \
    do {                     \
        int _st = (x);       \
        if (_st) return _st; \
    } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check(const vokra_hip_ctx* c, const vokra_hip_bkv* kv, const char* what) {
    if (!c || !kv || kv->ctx != c) return ctx_fail(BAD, "%s: bad context or cache", what);
    BK_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    return VOKRA_HIP_OK;
}

int check_items(size_t n, const char* what) {
    if (n > (size_t)kBkvMaxItems) return ctx_fail(BAD, "%s: at most %d items per call, got %zu", what, kBkvMaxItems, n);
    return VOKRA_HIP_OK;
}

int check_layer(const vokra_hip_bkv* kv, size_t layer) {
    if (layer >= (size_t)kv->v.n_layer) return ctx_fail(BAD, "layer %zu >= n_layer %d", layer, kv->v.n_layer);
    return VOKRA_HIP_OK;
}

// Host ids into the cache's staging: array k of the call.
int stage_ids(vokra_hip_bkv* kv, int k, const int32_t* ids, size_t n, const int** d) {
    int* p = kv->items + (size_t)k * kBkvMaxItems;
    BK_TRY(hipMemcpyAsync(p, ids, n * sizeof(int32_t), hipMemcpyHostToDevice, vk::ctx_stream(kv->ctx)),
           "hipMemcpyAsync");
    *d = p;
    return VOKRA_HIP_OK;
}

// At least n floats of row staging.
int stage_rows(vokra_hip_bkv* kv, size_t n) {
    if (n <= kv->rows_cap) return VOKRA_HIP_OK;
    if (kv->rows) BK_TRY(hipFree(kv->rows), "hipFree");
    kv->rows = nullptr;
    kv->rows_cap = 0;
    BK_TRY(hipMalloc((void**)&kv->rows, n * sizeof(float)), "hipMalloc(cache rows)");
    kv->rows_cap = n;
    return VOKRA_HIP_OK;
}

int read_meta(vokra_hip_bkv* kv, int* m) {
    BK_TRY(hipMemcpyAsync(m, kv->v.meta, BKV_META_INTS * sizeof(int), hipMemcpyDeviceToHost, vk::ctx_stream(kv->ctx)),
           "hipMemcpyAsync");
    BK_TRY(hipStreamSynchronize(vk::ctx_stream(kv->ctx)), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

int status_of(vokra_hip_bkv* kv, const char* what, size_t* n_done) {
    int m[BKV_META_INTS];
    BK_ST(read_meta(kv, m));
    if (n_done) *n_done = (size_t)m[BKV_DONE];
    if (m[BKV_STATUS] == VOKRA_HIP_ERROR_KV_CACHE_EXHAUSTED)
        return ctx_fail(m[BKV_STATUS], "%s: item %d finds no free page (%d of %d free)", what, m[BKV_DONE], m[BKV_FREE],
                        kv->v.n_page);
    if (m[BKV_STATUS] != VOKRA_HIP_OK)
        return ctx_fail(m[BKV_STATUS], "%s: item %d is not valid for this cache's state", what, m[BKV_DONE]);
    return VOKRA_HIP_OK;
}

void release(vokra_hip_bkv* kv) {
    BkvView& v = kv->v;
    for (void* p : {(void*)v.pool, (void*)v.scales, (void*)v.ring, (void*)v.table, (void*)v.len, (void*)v.floor_,
                    (void*)v.refs, (void*)v.used, (void*)v.fresh, (void*)v.moves, (void*)v.remap,
                    (void*)v.meta, (void*)v.step, (void*)v.plan, (void*)v.work, (void*)kv->items,
                    (void*)kv->rows})
        if (p) (void)hipFree(p);
    delete kv;
}

template <class T>
void reserve(hipError_t* e, T** p, size_t n) {
    if (*e == hipSuccess) *e = hipMalloc((void**)p, (n * sizeof(T) + 31) / 16 * 16);
}

// The blocks that a step of n items and n_rows rows can reach.
size_t work_bound(const vokra_hip_bkv* kv, size_t n, size_t n_rows) {
    const size_t bs = (size_t)kv->v.bs;
    return std::min(n_rows, n + (n_rows + n * (bs - 2)) / bs);
}

int step_launch(vokra_hip_bkv* kv, size_t n, size_t n_rows, size_t max_count, size_t max_len, const int* seqs,
                const int* starts, const int* counts) {
    BK_TRY(vk::launch_bkv_step(vk::ctx_stream(kv->ctx), kv->v, (int)n, (int)n_rows, (int)max_count, seqs, starts,
                               counts),
           "launch(vk_bkv_step)");
    kv->step_n = n;
    kv->step_rows = n_rows;
    kv->step_count = max_count;
    kv->step_len = std::min(max_len, (size_t)kv->v.max_time);
    return VOKRA_HIP_OK;
}

int check_hq(const vokra_hip_bkv* kv, size_t n_head_q) {
    if (n_head_q == 0 || n_head_q % (size_t)kv->v.n_head != 0 || n_head_q > 65535)
        return ctx_fail(BAD, "bkv_attn: n_head_q %zu is not a multiple of n_head %d up to 65535", n_head_q,
                        kv->v.n_head);
    return VOKRA_HIP_OK;
}

int attn_launch(vokra_hip_bkv* kv, size_t layer, size_t n_head_q, const float* q, float scale, float* out) {
    BK_TRY(vk::launch_bkv_attn(vk::ctx_stream(kv->ctx), kv->v, (int)layer, (int)kv->step_n, (int)kv->step_rows,
                               (int)kv->step_count, (int)kv->step_len, (int)n_head_q, q, scale, out, kv->part),
           "launch(vk_bkv_attn)");
    return VOKRA_HIP_OK;
}

int check_copy(const vokra_hip_bkv* d, const vokra_hip_bkv* s) {
    const BkvView &a = d->v, &b = s->v;
    if (a.n_layer != b.n_layer || a.n_head != b.n_head || a.hd != b.hd || a.bs != b.bs || a.codec != b.codec)
        return ctx_fail(BAD, "bkv_copy: the caches differ in layers, heads, d_head, block_size or codec");
    return VOKRA_HIP_OK;
}

}  // namespace

extern "C" {

int vokra_hip_bkv_create(vokra_hip_ctx_t* c, size_t n_layer, size_t n_head, size_t d_head, size_t n_seq,
                         size_t max_time, size_t block_size, size_t n_page, size_t max_rows, int codec,
                         vokra_hip_bkv_t** out) {
    if (!c || !out) return ctx_fail(BAD, "bkv_create: NULL argument");
    *out = nullptr;
    if (!n_layer || !n_head || !d_head || !n_seq || !max_time || !block_size || !n_page || !max_rows)
        return ctx_fail(BAD, "bkv_create: every size must be > 0");
    if (codec != VOKRA_HIP_BKV_INT8 && codec != VOKRA_HIP_BKV_E4M3)
        return ctx_fail(VOKRA_HIP_ERROR_UNSUPPORTED_OP, "bkv_create: unknown codec %d", codec);
    if (d_head != 64 && d_head != 128)
        return ctx_fail(VOKRA_HIP_ERROR_UNSUPPORTED_OP, "bkv_create: d_head %zu is not wired (64 or 128)", d_head);
    if (block_size != 16 && block_size != 32 && block_size != 64)
        return ctx_fail(VOKRA_HIP_ERROR_UNSUPPORTED_OP, "bkv_create: block_size %zu is not wired (16, 32 or 64)",
                        block_size);
    // int32 ids and counters, also summed over the items of a call
    if (n_layer > 4096 || n_head > 1024 || n_seq > 65535 || max_time > (1u << 24) || n_page > (1u << 26) ||
        max_rows > (1u << 20))
        return ctx_fail(BAD, "bkv_create: a size is too large (n_layer <= 4096, n_head <= 1024, n_seq <= 65535, "
                             "max_time <= 2^24, n_page <= 2^26, max_rows <= 2^20)");
    BK_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    void* part = nullptr;
    BK_ST(vk::ctx_bkv_part(c, &part));
    auto* kv = new (std::nothrow) vokra_hip_bkv();
    if (!kv) return ctx_fail(VOKRA_HIP_ERROR_OTHER, "bkv_create: out of host memory");
    kv->ctx = c;
    kv->max_rows = max_rows;
    kv->part = (float*)part;
    BkvView& v = kv->v;
    v.n_layer = (int)n_layer;
    v.n_head = (int)n_head;
    v.hd = (int)d_head;
    v.n_seq = (int)n_seq;
    v.bs = (int)block_size;
    v.n_page = (int)n_page;
    v.max_time = (int)max_time;
    v.max_blocks = (int)((max_time + block_size - 1) / block_size);
    v.codec = codec;
    v.max_work = (int)(max_rows / block_size + 2 * kBkvMaxItems);
    const size_t chunks = n_layer * n_page * n_head;
    hipError_t e = hipSuccess;
    reserve(&e, &v.pool, chunks * 2 * block_size * d_head);
    reserve(&e, &v.scales, chunks * 2);
    reserve(&e, &v.ring, n_layer * n_seq * 2 * n_head * 2 * block_size * d_head);
    reserve(&e, &v.table, n_seq * (size_t)v.max_blocks);
    reserve(&e, &v.len, n_seq);
    reserve(&e, &v.floor_, n_seq);
    reserve(&e, &v.refs, n_page);
    reserve(&e, &v.used, (n_page + 31) / 32);
    reserve(&e, &v.fresh, n_page);
    reserve(&e, &v.moves, n_page);
    reserve(&e, &v.remap, n_page);
    reserve(&e, &v.meta, BKV_META_INTS);
    reserve(&e, &v.step, kBkvMaxItems);
    reserve(&e, &v.plan, kBkvMaxItems);
    reserve(&e, &v.work, (size_t)v.max_work);
    reserve(&e, &kv->items, 4 * (size_t)kBkvMaxItems);
    if (e == hipSuccess) e = vk::launch_bkv_reset(vk::ctx_stream(c), v, true);
    if (e == hipSuccess) e = hipStreamSynchronize(vk::ctx_stream(c));
    if (e != hipSuccess) {
        release(kv);
        return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "bkv_create: %s", hipGetErrorString(e));
    }
    *out = kv;
    return VOKRA_HIP_OK;
}

void vokra_hip_bkv_destroy(vokra_hip_bkv_t* kv) {
    if (!kv) return;
    (void)hipSetDevice(vk::ctx_device(kv->ctx));
    (void)hipStreamSynchronize(vk::ctx_stream(kv->ctx));
    release(kv);
}

int vokra_hip_bkv_reset(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv) {
    BK_ST(check(c, kv, "bkv_reset"));
    BK_TRY(vk::launch_bkv_reset(vk::ctx_stream(c), kv->v, false), "launch(vk_bkv_reset)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_step_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, size_t n_rows, size_t max_count,
                           size_t max_len, const int32_t* d_seqs, const int32_t* d_starts, const int32_t* d_counts) {
    BK_ST(check(c, kv, "bkv_step"));
    BK_ST(check_items(n, "bkv_step"));
    if (n_rows > kv->max_rows)
        return ctx_fail(BAD, "bkv_step: %zu rows, the cache takes %zu a step", n_rows, kv->max_rows);
    if (n && (!d_seqs || !d_starts || !d_counts)) return ctx_fail(BAD, "bkv_step: NULL buffer");
    return step_launch(kv, n, n_rows, std::min(max_count, n_rows), max_len, d_seqs, d_starts, d_counts);
}

int vokra_hip_bkv_step(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, const int32_t* seqs, const int32_t* starts,
                       const int32_t* counts) {
    BK_ST(check(c, kv, "bkv_step"));
    BK_ST(check_items(n, "bkv_step"));
    if (n && (!seqs || !starts || !counts)) return ctx_fail(BAD, "bkv_step: NULL buffer");
    size_t n_rows = 0, max_count = 0, max_len = 0;
    for (size_t i = 0; i < n; ++i) {
        const size_t count = (size_t)std::max(counts[i], 0);  // a negative one fails its item on the device
        n_rows += count;
        max_count = std::max(max_count, count);
        max_len = std::max(max_len, (size_t)std::max(starts[i], 0) + count);
    }
    if (n_rows > kv->max_rows)
        return ctx_fail(BAD, "bkv_step: %zu rows, the cache takes %zu a step", n_rows, kv->max_rows);
    const int *ds = nullptr, *da = nullptr, *dc = nullptr;
    if (n) {
        BK_ST(stage_ids(kv, 0, seqs, n, &ds));
        BK_ST(stage_ids(kv, 1, starts, n, &da));
        BK_ST(stage_ids(kv, 2, counts, n, &dc));
    }
    BK_ST(step_launch(kv, n, n_rows, max_count, max_len, ds, da, dc));
    return status_of(kv, "bkv_step", nullptr);
}

int vokra_hip_bkv_status(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t* n_done) {
    BK_ST(check(c, kv, "bkv_status"));
    return status_of(kv, "bkv_status", n_done);
}

int vokra_hip_bkv_write_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, const float* d_k, const float* d_v) {
    BK_ST(check(c, kv, "bkv_write"));
    BK_ST(check_layer(kv, layer));
    if (kv->step_rows == 0) return VOKRA_HIP_OK;
    if (!d_k || !d_v) return ctx_fail(BAD, "bkv_write: NULL buffer");
    if (!aligned16(d_k) || !aligned16(d_v)) return ctx_fail(BAD, "bkv_write: k and v must be 16-byte aligned");
    BK_TRY(vk::launch_bkv_write(vk::ctx_stream(c), kv->v, (int)layer, (int)kv->step_rows,
                                (int)work_bound(kv, kv->step_n, kv->step_rows), d_k, d_v),
           "launch(vk_bkv_write)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_write(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, const float* k_rows,
                        const float* v_rows) {
    BK_ST(check(c, kv, "bkv_write"));
    BK_ST(check_layer(kv, layer));
    if (kv->step_rows == 0) return VOKRA_HIP_OK;
    if (!k_rows || !v_rows) return ctx_fail(BAD, "bkv_write: NULL buffer");
    const size_t n = kv->step_rows * (size_t)kv->v.n_head * (size_t)kv->v.hd;
    BK_ST(stage_rows(kv, 2 * n));
    hipStream_t s = vk::ctx_stream(c);
    BK_TRY(hipMemcpyAsync(kv->rows, k_rows, n * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BK_TRY(hipMemcpyAsync(kv->rows + n, v_rows, n * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BK_ST(vokra_hip_bkv_write_dev(c, kv, layer, kv->rows, kv->rows + n));
    BK_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_attn_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, size_t n_head_q, const float* d_q,
                           float scale, float* d_out) {
    BK_ST(check(c, kv, "bkv_attn"));
    BK_ST(check_layer(kv, layer));
    BK_ST(check_hq(kv, n_head_q));
    if (kv->step_rows == 0) return VOKRA_HIP_OK;
    if (!d_q || !d_out) return ctx_fail(BAD, "bkv_attn: NULL buffer");
    if (!aligned16(d_q) || !aligned16(d_out)) return ctx_fail(BAD, "bkv_attn: q and out must be 16-byte aligned");
    if (d_q == d_out) return ctx_fail(BAD, "bkv_attn: out overlaps q");
    return attn_launch(kv, layer, n_head_q, d_q, scale, d_out);
}

int vokra_hip_bkv_attn(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, size_t n_head_q, const float* q,
                       float scale, float* out) {
    BK_ST(check(c, kv, "bkv_attn"));
    BK_ST(check_layer(kv, layer));
    BK_ST(check_hq(kv, n_head_q));
    if (kv->step_rows == 0) return VOKRA_HIP_OK;
    if (!q || !out) return ctx_fail(BAD, "bkv_attn: NULL buffer");
    const size_t n = kv->step_rows * n_head_q * (size_t)kv->v.hd;
    BK_ST(stage_rows(kv, 2 * n));
    hipStream_t s = vk::ctx_stream(c);
    BK_TRY(hipMemcpyAsync(kv->rows, q, n * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    // rows of items that the step did not reach stay as they are in out
    BK_TRY(hipMemcpyAsync(kv->rows + n, out, n * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BK_ST(attn_launch(kv, layer, n_head_q, kv->rows, scale, kv->rows + n));
    BK_TRY(hipMemcpyAsync(out, kv->rows + n, n * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BK_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_read_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, size_t n, const int32_t* d_seqs,
                           const int32_t* d_times, float* d_k, float* d_v) {
    BK_ST(check(c, kv, "bkv_read"));
    BK_ST(check_layer(kv, layer));
    if (n > (size_t)INT32_MAX) return ctx_fail(BAD, "bkv_read: %zu rows exceed int32", n);
    if (n == 0) return VOKRA_HIP_OK;
    if (!d_seqs || !d_times || !d_k || !d_v) return ctx_fail(BAD, "bkv_read: NULL buffer");
    if (!aligned16(d_k) || !aligned16(d_v)) return ctx_fail(BAD, "bkv_read: k and v must be 16-byte aligned");
    BK_TRY(vk::launch_bkv_read(vk::ctx_stream(c), kv->v, (int)layer, (int)n, d_seqs, d_times, d_k, d_v),
           "launch(vk_bkv_read)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_read(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t layer, size_t n, const int32_t* seqs,
                       const int32_t* times, float* k_out, float* v_out) {
    BK_ST(check(c, kv, "bkv_read"));
    BK_ST(check_layer(kv, layer));
    if (n > (size_t)INT32_MAX) return ctx_fail(BAD, "bkv_read: %zu rows exceed int32", n);
    if (n == 0) return VOKRA_HIP_OK;
    if (!seqs || !times || !k_out || !v_out) return ctx_fail(BAD, "bkv_read: NULL buffer");
    const size_t w = (size_t)kv->v.n_head * (size_t)kv->v.hd, ids = (2 * n + 3) / 4 * 4;
    BK_ST(stage_rows(kv, 2 * n * w + ids));
    hipStream_t s = vk::ctx_stream(c);
    float *dk = kv->rows, *dv = dk + n * w;
    int* di = (int*)(dv + n * w);
    BK_TRY(hipMemcpyAsync(di, seqs, n * sizeof(int32_t), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BK_TRY(hipMemcpyAsync(di + n, times, n * sizeof(int32_t), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BK_ST(vokra_hip_bkv_read_dev(c, kv, layer, n, di, di + n, dk, dv));
    BK_TRY(hipMemcpyAsync(k_out, dk, n * w * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BK_TRY(hipMemcpyAsync(v_out, dv, n * w * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BK_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_fork_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, const int32_t* d_src,
                           const int32_t* d_dst) {
    BK_ST(check(c, kv, "bkv_fork"));
    BK_ST(check_items(n, "bkv_fork"));
    if (n && (!d_src || !d_dst)) return ctx_fail(BAD, "bkv_fork: NULL buffer");
    BK_TRY(vk::launch_bkv_fork(vk::ctx_stream(c), kv->v, (int)n, d_src, d_dst), "launch(vk_bkv_fork)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_fork(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, const int32_t* src, const int32_t* dst) {
    BK_ST(check(c, kv, "bkv_fork"));
    BK_ST(check_items(n, "bkv_fork"));
    if (n && (!src || !dst)) return ctx_fail(BAD, "bkv_fork: NULL buffer");
    if (n == 0) return VOKRA_HIP_OK;
    const int *a, *b;
    BK_ST(stage_ids(kv, 0, src, n, &a));
    BK_ST(stage_ids(kv, 1, dst, n, &b));
    BK_ST(vokra_hip_bkv_fork_dev(c, kv, n, a, b));
    return status_of(kv, "bkv_fork", nullptr);
}

int vokra_hip_bkv_free_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, const int32_t* d_seqs) {
    BK_ST(check(c, kv, "bkv_free"));
    BK_ST(check_items(n, "bkv_free"));
    if (n && !d_seqs) return ctx_fail(BAD, "bkv_free: NULL buffer");
    BK_TRY(vk::launch_bkv_free(vk::ctx_stream(c), kv->v, (int)n, d_seqs), "launch(vk_bkv_free)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_free(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t n, const int32_t* seqs) {
    BK_ST(check(c, kv, "bkv_free"));
    BK_ST(check_items(n, "bkv_free"));
    if (n && !seqs) return ctx_fail(BAD, "bkv_free: NULL buffer");
    if (n == 0) return VOKRA_HIP_OK;
    const int* a;
    BK_ST(stage_ids(kv, 0, seqs, n, &a));
    BK_ST(vokra_hip_bkv_free_dev(c, kv, n, a));
    return status_of(kv, "bkv_free", nullptr);
}

int vokra_hip_bkv_copy_dev(vokra_hip_ctx_t* c, vokra_hip_bkv_t* dst_kv, vokra_hip_bkv_t* src_kv, size_t n,
                           const int32_t* d_src, const int32_t* d_dst) {
    BK_ST(check(c, dst_kv, "bkv_copy"));
    BK_ST(check(c, src_kv, "bkv_copy"));
    BK_ST(check_copy(dst_kv, src_kv));
    BK_ST(check_items(n, "bkv_copy"));
    if (n && (!d_src || !d_dst)) return ctx_fail(BAD, "bkv_copy: NULL buffer");
    BK_TRY(vk::launch_bkv_copy(vk::ctx_stream(c), dst_kv->v, src_kv->v, (int)n, d_src, d_dst), "launch(vk_bkv_copy)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_copy(vokra_hip_ctx_t* c, vokra_hip_bkv_t* dst_kv, vokra_hip_bkv_t* src_kv, size_t n,
                       const int32_t* src, const int32_t* dst) {
    BK_ST(check(c, dst_kv, "bkv_copy"));
    BK_ST(check(c, src_kv, "bkv_copy"));
    BK_ST(check_copy(dst_kv, src_kv));
    BK_ST(check_items(n, "bkv_copy"));
    if (n && (!src || !dst)) return ctx_fail(BAD, "bkv_copy: NULL buffer");
    if (n == 0) return VOKRA_HIP_OK;
    const int *a, *b;
    BK_ST(stage_ids(dst_kv, 0, src, n, &a));
    BK_ST(stage_ids(dst_kv, 1, dst, n, &b));
    BK_ST(vokra_hip_bkv_copy_dev(c, dst_kv, src_kv, n, a, b));
    return status_of(dst_kv, "bkv_copy", nullptr);
}

int vokra_hip_bkv_compact(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv) {
    BK_ST(check(c, kv, "bkv_compact"));
    BK_TRY(vk::launch_bkv_compact(vk::ctx_stream(c), kv->v), "launch(vk_bkv_compact)");
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_length(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t seq, size_t* length) {
    BK_ST(check(c, kv, "bkv_length"));
    if (!length || seq >= (size_t)kv->v.n_seq) return ctx_fail(BAD, "bkv_length: sequence %zu of %d", seq, kv->v.n_seq);
    int h[2];
    BK_TRY(vk::launch_bkv_peek(vk::ctx_stream(c), kv->v, (int)seq, 0, kv->items), "launch(vk_bkv_peek)");
    BK_TRY(hipMemcpyAsync(h, kv->items, sizeof h, hipMemcpyDeviceToHost, vk::ctx_stream(c)), "hipMemcpyAsync");
    BK_TRY(hipStreamSynchronize(vk::ctx_stream(c)), "hipStreamSynchronize");
    *length = (size_t)h[0];
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_page_of(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t seq, size_t block, long* page) {
    BK_ST(check(c, kv, "bkv_page_of"));
    if (!page) return ctx_fail(BAD, "bkv_page_of: NULL argument");
    *page = -1;
    if (seq >= (size_t)kv->v.n_seq || block >= (size_t)kv->v.max_blocks) return VOKRA_HIP_OK;
    int h[2];
    BK_TRY(vk::launch_bkv_peek(vk::ctx_stream(c), kv->v, (int)seq, (int)block, kv->items), "launch(vk_bkv_peek)");
    BK_TRY(hipMemcpyAsync(h, kv->items, sizeof h, hipMemcpyDeviceToHost, vk::ctx_stream(c)), "hipMemcpyAsync");
    BK_TRY(hipStreamSynchronize(vk::ctx_stream(c)), "hipStreamSynchronize");
    *page = h[1];
    return VOKRA_HIP_OK;
}

int vokra_hip_bkv_pages(vokra_hip_ctx_t* c, vokra_hip_bkv_t* kv, size_t* free_pages, size_t* pages_in_use) {
    BK_ST(check(c, kv, "bkv_pages"));
    int m[BKV_META_INTS];
    BK_ST(read_meta(kv, m));
    if (free_pages) *free_pages = (size_t)m[BKV_FREE];
    if (pages_in_use) *pages_in_use = (size_t)(kv->v.n_page - m[BKV_FREE]);
    return VOKRA_HIP_OK;
}

}  // extern "C"
