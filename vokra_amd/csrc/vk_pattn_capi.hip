// vk_pattn_capi.hip — attention over packed sequences behind include/vokra_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/vokra_hip.h"
#include "vk_launch.h"
#include "vk_pattn.h"

struct vokra_hip_pattn {
    vokra_hip_ctx* ctx = nullptr;
    size_t seqs = 0, q_rows = 0, k_rows = 0, hq = 0, hkv = 0, hd = 0;  // at most
    void *tiles = nullptr, *meta = nullptr, *line = nullptr, *shares = nullptr, *part = nullptr;
};

namespace {

using vk::ctx_fail;
constexpr int BAD = VOKRA_HIP_ERROR_INVALID_ARGUMENT;

#define PA_TRY(call, what)                                                                                       \
    do {                                                                                                         \
        hipError_t _e = (call);                                                                                  \
        if (_e != hipSuccess)                                                                                    \
            return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "%s: %s", (what), hipGetErrorString(_e));       \
    } while (0)
#define PA_ST(x)             \
    do {                     \
        int _st = (x);       \
        if (_st) return _st; \
    } while (0)

struct Temp {
    void* p = nullptr;
    hipError_t make(size_t bytes) { return hipMalloc(&p, bytes + 16); }
    ~Temp() {
        if (p) (void)hipFree(p);
    }
};

bool meet(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na && nb && x < y + nb && y < x + na;
}

void release(vokra_hip_pattn* p) {
    for (void* x : {p->tiles, p->meta, p->line, p->shares, p->part})
        if (x) (void)hipFree(x);
    delete p;
}

// Places of tiles of `rows` rows in tiles of `size`: vk_pattn.hip's pa_q_slot, pa_k_slot.
size_t places(size_t rows, size_t size, size_t seqs) { return rows / size + seqs; }

int check_call(const vokra_hip_ctx* c, const vokra_hip_pattn* p, size_t n_seq, size_t q_rows, size_t k_rows, float scale,
               int causal, size_t window) {
    if (!c || !p || p->ctx != c) return ctx_fail(BAD, "packed_attn: bad context or plan");
    if (n_seq > p->seqs || q_rows > p->q_rows || k_rows > p->k_rows)
        return ctx_fail(BAD, "packed_attn: %zu sequences of %zu and %zu rows; the plan takes up to %zu of %zu and %zu", n_seq,
                        q_rows, k_rows, p->seqs, p->q_rows, p->k_rows);
    if (!std::isfinite(scale)) return ctx_fail(BAD, "packed_attn: scale must be finite");
    if (window && !causal) return ctx_fail(BAD, "packed_attn: a window needs causal attention");
    return VOKRA_HIP_OK;
}

int check_rows(const char* name, const float* x, size_t rows, size_t width, size_t stride) {
    if (rows == 0) return VOKRA_HIP_OK;
    if (!x) return ctx_fail(BAD, "packed_attn: %s is NULL", name);
    if (reinterpret_cast<uintptr_t>(x) % 16 != 0 || stride % 4 != 0)
        return ctx_fail(BAD, "packed_attn: rows of %s must be 16-byte aligned", name);
    if (stride < width || stride > ((size_t)1 << 23))
        return ctx_fail(BAD, "packed_attn: a row stride of %s is below its %zu values or too large", name, width);
    return VOKRA_HIP_OK;
}

}  // namespace

extern "C" {

int vokra_hip_packed_attn_create(vokra_hip_ctx_t* c, size_t max_seq, size_t max_q_rows, size_t max_k_rows,
                                 size_t n_head_q, size_t n_head_kv, size_t head_dim, vokra_hip_packed_attn_t** out) {
    if (!c || !out) return ctx_fail(BAD, "packed_attn_create: NULL argument");
    *out = nullptr;
    if (!max_seq || !max_q_rows || !max_k_rows) return ctx_fail(BAD, "packed_attn_create: every size must be > 0");
    if (head_dim != 64 && head_dim != 128)
        return ctx_fail(VOKRA_HIP_ERROR_UNSUPPORTED_OP, "packed_attn_create: head_dim %zu is not wired (64 or 128)",
                        head_dim);
    if (n_head_kv == 0 || n_head_q == 0 || n_head_q % n_head_kv != 0 || n_head_q > 1024)
        return ctx_fail(BAD, "packed_attn_create: n_head_q=%zu must be a positive multiple of n_head_kv=%zu, at most 1024",
                        n_head_q, n_head_kv);
    if (max_seq > (size_t)kPaSeqs || max_q_rows > ((size_t)1 << 20) || max_k_rows > ((size_t)1 << 20))
        return ctx_fail(BAD, "packed_attn_create: at most %d sequences of 2^20 rows in all", kPaSeqs);
    PA_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    auto* p = new (std::nothrow) vokra_hip_pattn();
    if (!p) return ctx_fail(VOKRA_HIP_ERROR_OTHER, "packed_attn_create: out of host memory");
    p->ctx = c;
    p->seqs = max_seq;
    p->q_rows = max_q_rows;
    p->k_rows = max_k_rows;
    p->hq = n_head_q;
    p->hkv = n_head_kv;
    p->hd = head_dim;
    const size_t ks = places(max_k_rows, kPaKeys, max_seq);
    const size_t qs = places(max_q_rows * (n_head_q / n_head_kv), (size_t)pa_tile_rows((int)head_dim), max_seq);
    struct {
        void** p;
        size_t bytes;
    } all[] = {{&p->tiles, ks * n_head_kv * 4 * kPaKeys * head_dim * 2},
               {&p->meta, ks * n_head_kv * sizeof(PaTileMeta)},
               {&p->line, (qs + 1) * sizeof(long long)},
               {&p->shares, kPaShares * (sizeof(PaStart) + sizeof(int)) + 3 * sizeof(long long)},
               {&p->part, vk::pattn_part_floats((int)head_dim) * sizeof(float)}};
    hipError_t e = hipSuccess;
    for (auto& x : all)
        if (e == hipSuccess) e = hipMalloc(x.p, x.bytes);
    if (e != hipSuccess) {
        (void)hipGetLastError();  // reported here
        release(p);
        return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "packed_attn_create: %s", hipGetErrorString(e));
    }
    *out = p;
    return VOKRA_HIP_OK;
}

void vokra_hip_packed_attn_destroy(vokra_hip_packed_attn_t* p) {
    if (!p) return;
    (void)hipSetDevice(vk::ctx_device(p->ctx));
    (void)hipStreamSynchronize(vk::ctx_stream(p->ctx));
    release(p);
}

int vokra_hip_packed_attn_dev(vokra_hip_ctx_t* c, vokra_hip_packed_attn_t* p, size_t n_seq, size_t n_q_rows,
                              size_t n_k_rows, size_t max_q, size_t max_k, const int32_t* d_q_offsets,
                              const int32_t* d_k_offsets, const float* d_q, size_t q_stride, const float* d_k,
                              size_t k_stride, const float* d_v, size_t v_stride, float scale, int causal,
                              size_t window, float* d_out, size_t out_stride) {
    PA_ST(check_call(c, p, n_seq, n_q_rows, n_k_rows, scale, causal, window));
    max_q = std::min(max_q, n_q_rows);
    max_k = std::min(max_k, n_k_rows);
    if (n_seq == 0 || n_q_rows == 0 || max_q == 0) return VOKRA_HIP_OK;
    if (!d_q_offsets) return ctx_fail(BAD, "packed_attn: offsets are NULL");
    const size_t wq = p->hq * p->hd, wk = p->hkv * p->hd;
    PA_ST(check_rows("q", d_q, n_q_rows, wq, q_stride));
    PA_ST(check_rows("k", d_k, n_k_rows, wk, k_stride));
    PA_ST(check_rows("v", d_v, n_k_rows, wk, v_stride));
    PA_ST(check_rows("out", d_out, n_q_rows, wq, out_stride));
    const size_t no = ((n_q_rows - 1) * out_stride + wq) * 4, ko = (n_seq + 1) * 4;
    const int32_t* koff = d_k_offsets ? d_k_offsets : d_q_offsets;
    if (meet(d_out, no, d_q, ((n_q_rows - 1) * q_stride + wq) * 4) ||
        (n_k_rows && (meet(d_out, no, d_k, ((n_k_rows - 1) * k_stride + wk) * 4) ||
                      meet(d_out, no, d_v, ((n_k_rows - 1) * v_stride + wk) * 4))) ||
        meet(d_out, no, d_q_offsets, ko) || meet(d_out, no, koff, ko))
        return ctx_fail(BAD, "packed_attn: out overlaps an input");
    PA_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    PaArgs a = {};
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.out = d_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.out_stride = out_stride;
    a.q_off = d_q_offsets;
    a.k_off = koff;
    a.n_seq = (int)n_seq;
    a.q_rows = (int)n_q_rows;
    a.k_rows = (int)n_k_rows;
    a.max_q = (int)max_q;
    a.max_k = (int)max_k;
    a.hq = (int)p->hq;
    a.hkv = (int)p->hkv;
    a.g = (int)(p->hq / p->hkv);
    a.causal = causal ? 1 : 0;
    a.window = (int)std::min<size_t>(window, (size_t)1 << 21);
    a.c = scale == 0.0f ? 1.0f : std::fabs(scale) * 1.44269504088896340736f;
    a.sign = scale == 0.0f ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
    a.tiles = (_Float16*)p->tiles;
    a.meta = (PaTileMeta*)p->meta;
    a.line = (long long*)p->line;
    a.start = (PaStart*)p->shares;
    a.ended = (int*)(a.start + kPaShares);
    a.plan = (long long*)(a.ended + kPaShares);
    a.part = (float*)p->part;
    a.k_slots = (int)places(n_k_rows, kPaKeys, n_seq);
    PA_TRY(vk::launch_pattn(vk::ctx_stream(c), (int)p->hd, a), "launch(vk_pattn)");
    return VOKRA_HIP_OK;
}

int vokra_hip_packed_attn(vokra_hip_ctx_t* c, vokra_hip_packed_attn_t* p, size_t n_seq, const int32_t* q_offsets,
                          const int32_t* k_offsets, const float* q, const float* k, const float* v, float scale,
                          int causal, size_t window, float* out) {
    if (!c || !p || p->ctx != c) return ctx_fail(BAD, "packed_attn: bad context or plan");
    if (n_seq == 0) return VOKRA_HIP_OK;
    if (!q_offsets) return ctx_fail(BAD, "packed_attn: offsets are NULL");
    if (!k_offsets) k_offsets = q_offsets;
    size_t max_q = 0, max_k = 0;
    for (int side = 0; side < 2; ++side) {
        const int32_t* off = side ? k_offsets : q_offsets;
        size_t* most = side ? &max_k : &max_q;
        for (size_t i = 0; i <= n_seq; ++i) {
            if (off[i] < 0 || (i && off[i] < off[i - 1]))
                return ctx_fail(BAD, "packed_attn: offset %zu of the %s is out of order", i, side ? "keys" : "queries");
            if (i) *most = std::max(*most, (size_t)(off[i] - off[i - 1]));
        }
    }
    const size_t nq = (size_t)q_offsets[n_seq], nk = (size_t)k_offsets[n_seq];
    PA_ST(check_call(c, p, n_seq, nq, nk, scale, causal, window));
    if (nq == 0) return VOKRA_HIP_OK;
    if (!q || !out || (nk && (!k || !v))) return ctx_fail(BAD, "packed_attn: NULL buffer");
    PA_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    hipStream_t s = vk::ctx_stream(c);
    const size_t wq = p->hq * p->hd, wk = p->hkv * p->hd;
    Temp t, ids;
    PA_TRY(t.make((2 * nq * wq + 2 * nk * wk) * sizeof(float)), "hipMalloc");
    PA_TRY(ids.make(2 * (n_seq + 1) * sizeof(int32_t)), "hipMalloc");
    float *dq = (float*)t.p, *dout = dq + nq * wq, *dk = dout + nq * wq, *dv = dk + nk * wk;
    int32_t *qo = (int32_t*)ids.p, *ko = qo + n_seq + 1;
    PA_TRY(hipMemcpyAsync(dq, q, nq * wq * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    // rows before the first sequence stay as they are in out
    PA_TRY(hipMemcpyAsync(dout, out, nq * wq * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    if (nk) {
        PA_TRY(hipMemcpyAsync(dk, k, nk * wk * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
        PA_TRY(hipMemcpyAsync(dv, v, nk * wk * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    }
    PA_TRY(hipMemcpyAsync(qo, q_offsets, (n_seq + 1) * sizeof(int32_t), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    PA_TRY(hipMemcpyAsync(ko, k_offsets, (n_seq + 1) * sizeof(int32_t), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    PA_ST(vokra_hip_packed_attn_dev(c, p, n_seq, nq, nk, max_q, max_k, qo, ko, dq, wq, dk, wk, dv, wk, scale, causal,
                                    window, dout, wq));
    PA_TRY(hipMemcpyAsync(out, dout, nq * wq * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    PA_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

}  // extern "C"
