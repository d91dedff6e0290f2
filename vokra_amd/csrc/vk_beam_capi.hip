// vk_beam_capi.hip — beam search's selection behind include/vokra_hip.h.
#include <hip/hip_runtime.h>

#include <new>

#include "../../include/vokra_hip.h"
#include "vk_beam.h"
#include "vk_launch.h"

struct vokra_hip_beam {
    vokra_hip_ctx* ctx = nullptr;
    size_t groups = 0, beams = 0, vocab = 0, out = 0;  // at most
    unsigned long long* keys = nullptr;
    BeamStat* stats = nullptr;
};

namespace {

using vk::ctx_fail;
constexpr int BAD = VOKRA_HIP_ERROR_INVALID_ARGUMENT;

#define BM_TRY(call, what)                                                                                       \
    do {                                                                                                         \
        hipError_t _e = (call);                                                                                  \
        if (_e != hipSuccess)                                                                                    \
            return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "%s: %s", (what), hipGetErrorString(_e));       \
    } while (0)
#define BM_ST(x)             \
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
    return a && b && x < y + nb && y < x + na;
}

int check(const vokra_hip_ctx* c, const vokra_hip_beam* p, size_t groups, size_t beams, size_t vocab, size_t n_out,
          size_t stride, const float* logits, const float* scores, const int32_t* ended, int32_t end_token,
          float* out_scores, int32_t* out_parents, int32_t* out_tokens, int32_t* out_ended) {
    if (!c || !p || p->ctx != c) return ctx_fail(BAD, "beam_select: bad context or plan");
    if (groups > p->groups || beams == 0 || beams > p->beams || vocab == 0 || vocab > p->vocab || n_out == 0 ||
        n_out > p->out)
        return ctx_fail(BAD, "beam_select: %zu groups of %zu beams, %zu tokens and %zu continuations; the plan takes up "
                             "to %zu, %zu, %zu and %zu",
                        groups, beams, vocab, n_out, p->groups, p->beams, p->vocab, p->out);
    if (stride < vocab || stride > ((size_t)1 << 40))
        return ctx_fail(BAD, "beam_select: row stride %zu below the vocabulary %zu or too large", stride, vocab);
    if (end_token < -1 || end_token >= (int32_t)vocab)
        return ctx_fail(BAD, "beam_select: end token %d is not in -1 .. %zu", end_token, vocab - 1);
    if (ended && end_token < 0) return ctx_fail(BAD, "beam_select: ended beams without an end token");
    if (groups == 0) return VOKRA_HIP_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens)
        return ctx_fail(BAD, "beam_select: NULL buffer");
    const size_t rows = groups * beams, in = rows * 4, out = groups * n_out * 4;
    const void* outs[4] = {out_scores, out_parents, out_tokens, out_ended};
    for (int i = 0; i < 4; ++i) {
        if (meet(outs[i], out, logits, ((rows - 1) * stride + vocab) * 4))
            return ctx_fail(BAD, "beam_select: an output overlaps the logits");
        for (int j = 0; j < i; ++j)
            if (meet(outs[i], out, outs[j], out)) return ctx_fail(BAD, "beam_select: two outputs overlap");
        const bool same = n_out == beams && ((i == 0 && out_scores == scores) || (i == 3 && out_ended == ended));
        if ((!(same && i == 0) && meet(outs[i], out, scores, in)) ||
            (!(same && i == 3) && meet(outs[i], out, ended, in)))
            return ctx_fail(BAD, "beam_select: an output overlaps scores or ended");
    }
    return VOKRA_HIP_OK;
}

}  // namespace

extern "C" {

int vokra_hip_beam_create(vokra_hip_ctx_t* c, size_t max_groups, size_t max_beams, size_t max_vocab, size_t max_out,
                          vokra_hip_beam_t** out) {
    if (!c || !out) return ctx_fail(BAD, "beam_create: NULL argument");
    *out = nullptr;
    if (!max_groups || !max_beams || !max_vocab || !max_out)
        return ctx_fail(BAD, "beam_create: every size must be > 0");
    if (max_beams > (size_t)kBeamMost || max_out > (size_t)kBeamOut || max_vocab > ((size_t)1 << 24) ||
        max_groups > 65535 / max_beams)
        return ctx_fail(BAD, "beam_create: at most %d beams, %d continuations, 2^24 tokens and 65535 rows, got %zu, %zu, "
                             "%zu and %zu x %zu",
                        kBeamMost, kBeamOut, max_beams, max_out, max_vocab, max_groups, max_beams);
    BM_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    auto* p = new (std::nothrow) vokra_hip_beam();
    if (!p) return ctx_fail(VOKRA_HIP_ERROR_OTHER, "beam_create: out of host memory");
    p->ctx = c;
    p->groups = max_groups;
    p->beams = max_beams;
    p->vocab = max_vocab;
    p->out = max_out;
    const size_t parts = max_groups * max_beams * ((max_vocab + kBeamSlice - 1) / kBeamSlice);
    hipError_t e = hipMalloc((void**)&p->keys, parts * max_out * sizeof(unsigned long long));
    if (e == hipSuccess) e = hipMalloc((void**)&p->stats, parts * sizeof(BeamStat));
    if (e != hipSuccess) {
        (void)hipGetLastError();  // reported here
        if (p->keys) (void)hipFree(p->keys);
        delete p;
        return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "beam_create: %s", hipGetErrorString(e));
    }
    *out = p;
    return VOKRA_HIP_OK;
}

void vokra_hip_beam_destroy(vokra_hip_beam_t* p) {
    if (!p) return;
    (void)hipSetDevice(vk::ctx_device(p->ctx));
    (void)hipStreamSynchronize(vk::ctx_stream(p->ctx));
    (void)hipFree(p->keys);
    (void)hipFree(p->stats);
    delete p;
}

int vokra_hip_beam_select_dev(vokra_hip_ctx_t* c, vokra_hip_beam_t* p, size_t groups, size_t beams, size_t vocab,
                              size_t n_out, size_t stride, const float* d_logits, const float* d_scores,
                              const int32_t* d_ended, int32_t end_token, float* d_out_scores, int32_t* d_out_parents,
                              int32_t* d_out_tokens, int32_t* d_out_ended) {
    BM_ST(check(c, p, groups, beams, vocab, n_out, stride, d_logits, d_scores, d_ended, end_token, d_out_scores,
                d_out_parents, d_out_tokens, d_out_ended));
    if (groups == 0) return VOKRA_HIP_OK;
    BM_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    BeamArgs a = {};
    a.logits = d_logits;
    a.stride = stride;
    a.scores = d_scores;
    a.ended = d_ended;
    a.out_scores = d_out_scores;
    a.out_parents = d_out_parents;
    a.out_tokens = d_out_tokens;
    a.out_ended = d_out_ended;
    a.keys = p->keys;
    a.stats = p->stats;
    a.groups = (int)groups;
    a.beams = (int)beams;
    a.vocab = (int)vocab;
    a.n_out = (int)n_out;
    a.end_token = end_token;
    BM_TRY(vk::launch_beam_select(vk::ctx_stream(c), a), "launch(vk_beam_select)");
    return VOKRA_HIP_OK;
}

int vokra_hip_beam_select(vokra_hip_ctx_t* c, vokra_hip_beam_t* p, size_t groups, size_t beams, size_t vocab,
                          size_t n_out, const float* logits, const float* scores, const int32_t* ended,
                          int32_t end_token, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                          int32_t* out_ended) {
    BM_ST(check(c, p, groups, beams, vocab, n_out, vocab, logits, scores, ended, end_token, out_scores, out_parents,
                out_tokens, out_ended));
    if (groups == 0) return VOKRA_HIP_OK;
    BM_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    hipStream_t s = vk::ctx_stream(c);
    const size_t rows = groups * beams, n = groups * n_out;
    Temp x, small;
    BM_TRY(x.make(rows * vocab * sizeof(float)), "hipMalloc");
    BM_TRY(small.make((2 * rows + 4 * n) * 4), "hipMalloc");
    float* d_scores = (float*)small.p;
    int32_t* d_ended = (int32_t*)(d_scores + rows);
    float* d_out = (float*)(d_ended + rows);
    int32_t* d_ids = (int32_t*)(d_out + n);
    BM_TRY(hipMemcpyAsync(x.p, logits, rows * vocab * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BM_TRY(hipMemcpyAsync(d_scores, scores, rows * 4, hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    if (ended) BM_TRY(hipMemcpyAsync(d_ended, ended, rows * 4, hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    BM_ST(vokra_hip_beam_select_dev(c, p, groups, beams, vocab, n_out, vocab, (const float*)x.p, d_scores,
                                    ended ? d_ended : nullptr, end_token, d_out, d_ids, d_ids + n,
                                    out_ended ? d_ids + 2 * n : nullptr));
    BM_TRY(hipMemcpyAsync(out_scores, d_out, n * 4, hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BM_TRY(hipMemcpyAsync(out_parents, d_ids, n * 4, hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BM_TRY(hipMemcpyAsync(out_tokens, d_ids + n, n * 4, hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    if (out_ended) BM_TRY(hipMemcpyAsync(out_ended, d_ids + 2 * n, n * 4, hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    BM_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

}  // extern "C"
