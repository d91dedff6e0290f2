// vk_step_capi.hip — rotary plans and logits rules behind include/vokra_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/vokra_hip.h"
#include "vk_launch.h"
#include "vk_step.h"

struct vokra_hip_rope {
    vokra_hip_ctx* ctx = nullptr;
    uint64_t* turn = nullptr;
    size_t hd = 0, rot = 0;
    bool pairs = false;
    float mag = 1.0f;
};

namespace {

using vk::ctx_fail;
constexpr int BAD = VOKRA_HIP_ERROR_INVALID_ARGUMENT;

#define ST_TRY(call, what)                                                                                       \
    do {                                                                                                         \
        hipError_t _e = (call);                                                                                  \
        if (_e != hipSuccess)                                                                                    \
            return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "%s: %s", (what), hipGetErrorString(_e));       \
    } while (0)
#define ST_ST(x)             \
    do {                     \
        int _st = (x);       \
        if (_st) return _st; \
    } while (0)

// A device allocation for the length of a host-array call.
struct Temp {
    void* p = nullptr;
    hipError_t make(size_t bytes) { return hipMalloc(&p, bytes + 16); }
    ~Temp() {
        if (p) (void)hipFree(p);
    }
};

// Frequency of pair j (radians per position) and the factor on turned values.
long double rope_theta(const vokra_hip_rope_config_t& f, size_t j) {
    const long double r = (long double)f.rot_dim, e = -2.0L * (long double)j / r, base = f.base, s = f.factor;
    const long double two_pi = 6.283185307179586476925286766559L;
    if (f.scaling == VOKRA_HIP_ROPE_NTK) return powl(base * powl(s, r / (r - 2.0L)), e);
    const long double th = powl(base, e);
    if (f.scaling == VOKRA_HIP_ROPE_LINEAR) return th / s;
    if (f.scaling == VOKRA_HIP_ROPE_DIVISORS) return th / (long double)f.divisors[j];
    if (f.scaling == VOKRA_HIP_ROPE_YARN) {
        const double fast = f.beta_fast != 0.0 ? f.beta_fast : 32.0, slow = f.beta_slow != 0.0 ? f.beta_slow : 1.0;
        const long double k = r / (2.0L * logl(base));
        const long double lo = std::max(floorl(k * logl((long double)f.orig_ctx / (fast * two_pi))), 0.0L);
        const long double hi = std::min(ceill(k * logl((long double)f.orig_ctx / (slow * two_pi))), r - 1.0L);
        const long double ramp = std::min(std::max(((long double)j - lo) / std::max(hi - lo, 0.001L), 0.0L), 1.0L);
        return th / s * ramp + th * (1.0L - ramp);
    }
    if (f.scaling == VOKRA_HIP_ROPE_BANDS) {
        const double lo = f.low_turns != 0.0 ? f.low_turns : 1.0, hi = f.high_turns != 0.0 ? f.high_turns : 4.0;
        const long double turns = (long double)f.orig_ctx * th / two_pi;
        const long double mix = std::min(std::max((turns - lo) / ((long double)hi - lo), 0.0L), 1.0L);
        return th / s * (1.0L - mix) + th * mix;
    }
    return th;
}

int rope_check(const vokra_hip_rope_config_t& f) {
    if (f.head_dim == 0 || f.head_dim > 65536 || f.rot_dim == 0 || f.rot_dim % 2 != 0 || f.rot_dim > f.head_dim)
        return ctx_fail(BAD, "rope_create: rot_dim %zu must be even, > 0 and at most head_dim %zu (<= 65536)", f.rot_dim,
                        f.head_dim);
    if (f.layout != VOKRA_HIP_ROPE_HALF && f.layout != VOKRA_HIP_ROPE_INTERLEAVED)
        return ctx_fail(BAD, "rope_create: unknown layout %d", f.layout);
    if (f.scaling < VOKRA_HIP_ROPE_NONE || f.scaling > VOKRA_HIP_ROPE_DIVISORS)
        return ctx_fail(BAD, "rope_create: unknown scaling %d", f.scaling);
    if (!(f.base > 1.0) || !std::isfinite(f.base)) return ctx_fail(BAD, "rope_create: base must be finite and > 1");
    if (!std::isfinite(f.magnitude) || f.magnitude < 0.0)
        return ctx_fail(BAD, "rope_create: magnitude must be finite and >= 0");
    if (f.scaling == VOKRA_HIP_ROPE_NONE) return VOKRA_HIP_OK;
    if (f.scaling == VOKRA_HIP_ROPE_DIVISORS) {
        if (!f.divisors) return ctx_fail(BAD, "rope_create: divisors is NULL");
        for (size_t j = 0; j < f.rot_dim / 2; ++j)
            if (!(f.divisors[j] > 0.0) || !std::isfinite(f.divisors[j]))
                return ctx_fail(BAD, "rope_create: divisor %zu must be finite and > 0", j);
        return VOKRA_HIP_OK;
    }
    if (!(f.factor >= 1.0) || !std::isfinite(f.factor))
        return ctx_fail(BAD, "rope_create: factor must be finite and >= 1");
    if (f.scaling == VOKRA_HIP_ROPE_NTK && f.rot_dim < 4)
        return ctx_fail(BAD, "rope_create: NTK scaling needs rot_dim >= 4");
    if (f.scaling == VOKRA_HIP_ROPE_YARN || f.scaling == VOKRA_HIP_ROPE_BANDS) {
        if (f.orig_ctx == 0) return ctx_fail(BAD, "rope_create: orig_ctx must be > 0");
        for (double x : {f.beta_fast, f.beta_slow, f.low_turns, f.high_turns})
            if (!std::isfinite(x) || x < 0.0)
                return ctx_fail(BAD, "rope_create: beta_fast, beta_slow, low_turns and high_turns must be finite and >= 0");
        const double lo = f.low_turns != 0.0 ? f.low_turns : 1.0, hi = f.high_turns != 0.0 ? f.high_turns : 4.0;
        if (f.scaling == VOKRA_HIP_ROPE_BANDS && !(lo < hi))
            return ctx_fail(BAD, "rope_create: low_turns must be below high_turns");
    }
    return VOKRA_HIP_OK;
}

// A launch has fewer than 2^32 threads, one for two values at least; sizes in bytes fit.
int rope_size(const vokra_hip_rope* p, size_t rows, size_t n_head_q, size_t n_head_k) {
    if (n_head_q > 65535 || n_head_k > 65535) return ctx_fail(BAD, "rope_apply: at most 65535 heads");
    const size_t w = (n_head_q + n_head_k) * p->hd;
    if (rows > (size_t)INT32_MAX || w > ((size_t)1 << 30) || rows * w > ((size_t)1 << 32))
        return ctx_fail(BAD, "rope_apply: more than 2^32 values, or 2^30 a row");
    return VOKRA_HIP_OK;
}

// [p, p + bytes) of two buffers meet
bool meet(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// Whether rows of two buffers meet, wa and wb floats of them, sa and sb floats from row to
// row. Rows of one stride may lie between each other; of two strides the whole ranges count.
bool rows_meet(size_t rows, const float* a, size_t wa, size_t sa, const float* b, size_t wb, size_t sb) {
    if (!meet(a, ((rows - 1) * sa + wa) * 4, b, ((rows - 1) * sb + wb) * 4)) return false;
    if (sa != sb) return true;
    // row i of a, row i + k of b: -4 wb < d + 4 k s < 4 wa, |k| < rows
    const int64_t d = (int64_t)(reinterpret_cast<uintptr_t>(b) - reinterpret_cast<uintptr_t>(a));
    const int64_t s = (int64_t)sa * 4, lo = -(int64_t)wb * 4 - d + 1, hi = (int64_t)wa * 4 - d - 1;
    const int64_t k0 = lo >= 0 ? (lo + s - 1) / s : -(-lo / s), k1 = hi >= 0 ? hi / s : -((-hi + s - 1) / s);
    return std::max(k0, 1 - (int64_t)rows) <= std::min(k1, (int64_t)rows - 1);
}

int rope_side(const vokra_hip_rope* p, const char* name, size_t rows, size_t heads, const float* x, size_t stride,
              const float* y, size_t out_stride) {
    if (heads == 0) return VOKRA_HIP_OK;
    const size_t w = heads * p->hd;
    if (!x || !y) return ctx_fail(BAD, "rope_apply: %s is NULL", name);
    if (stride < w || out_stride < w)
        return ctx_fail(BAD, "rope_apply: a row stride of %s is below its %zu values", name, w);
    if (stride > ((size_t)1 << 40) || out_stride > ((size_t)1 << 40))
        return ctx_fail(BAD, "rope_apply: a row stride of %s is too large", name);
    if (x == y) {
        if (stride != out_stride) return ctx_fail(BAD, "rope_apply: %s in place needs one row stride", name);
    } else if (rows_meet(rows, x, w, stride, y, w, out_stride)) {
        return ctx_fail(BAD, "rope_apply: %s and its output overlap without being the same", name);
    }
    return VOKRA_HIP_OK;
}

int rules_check(const vokra_hip_logits_rules_t* r, size_t rows, size_t vocab, size_t stride, const float* logits,
                const float* out, const int32_t* next) {
    if (!r) return ctx_fail(BAD, "logits_rules: rules is NULL");
    if (vocab == 0 || vocab > ((size_t)1 << 24)) return ctx_fail(BAD, "logits_rules: vocab %zu is not in 1 .. 2^24", vocab);
    if (rows > 65535) return ctx_fail(BAD, "logits_rules: at most 65535 rows, got %zu", rows);
    if (stride < vocab || stride > ((size_t)1 << 40))
        return ctx_fail(BAD, "logits_rules: row stride %zu below the vocabulary %zu or too large", stride, vocab);
    if (rows == 0) return VOKRA_HIP_OK;
    if (!logits || (!out && !next)) return ctx_fail(BAD, "logits_rules: NULL buffer");
    if (r->n_hist > (size_t)INT32_MAX || r->n_bias > (size_t)INT32_MAX)
        return ctx_fail(BAD, "logits_rules: a list exceeds int32");
    if (r->n_hist && (!r->hist || !r->hist_offsets)) return ctx_fail(BAD, "logits_rules: history without its arrays");
    if (r->n_bias && (!r->bias_ids || !r->bias || !r->bias_offsets))
        return ctx_fail(BAD, "logits_rules: biases without their arrays");
    if (r->mask && r->mask_stride != 0 && (r->mask_stride < (vocab + 31) / 32 || r->mask_stride > ((size_t)1 << 40)))
        return ctx_fail(BAD, "logits_rules: mask stride %zu below %zu words or too large", r->mask_stride,
                        (vocab + 31) / 32);
    if (out && out != logits && meet(logits, ((rows - 1) * stride + vocab) * 4, out, ((rows - 1) * stride + vocab) * 4))
        return ctx_fail(BAD, "logits_rules: logits and out overlap without being the same");
    return VOKRA_HIP_OK;
}

// Device copy of a host list; NULL stays NULL.
int to_device(hipStream_t s, Temp& t, const void* h, size_t bytes, const void** d) {
    *d = nullptr;
    if (!h) return VOKRA_HIP_OK;
    ST_TRY(t.make(bytes), "hipMalloc");
    if (bytes) ST_TRY(hipMemcpyAsync(t.p, h, bytes, hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    *d = t.p;
    return VOKRA_HIP_OK;
}

}  // namespace

extern "C" {

int vokra_hip_rope_create(vokra_hip_ctx_t* c, const vokra_hip_rope_config_t* cfg, vokra_hip_rope_t** out) {
    if (!c || !cfg || !out) return ctx_fail(BAD, "rope_create: NULL argument");
    *out = nullptr;
    ST_ST(rope_check(*cfg));
    ST_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    const size_t n = cfg->rot_dim / 2;
    auto* p = new (std::nothrow) vokra_hip_rope();
    auto* turn = new (std::nothrow) uint64_t[n];
    if (!p || !turn) {
        delete p;
        delete[] turn;
        return ctx_fail(VOKRA_HIP_ERROR_OTHER, "rope_create: out of host memory");
    }
    for (size_t j = 0; j < n; ++j) {
        const long double t = rope_theta(*cfg, j) / 6.283185307179586476925286766559L;
        const long double f = (t - floorl(t)) * 18446744073709551616.0L;  // of one turn, in 2^-64
        turn[j] = f >= 18446744073709551615.0L ? 0 : (uint64_t)roundl(f);
    }
    p->ctx = c;
    p->hd = cfg->head_dim;
    p->rot = cfg->rot_dim;
    p->pairs = cfg->layout == VOKRA_HIP_ROPE_INTERLEAVED;
    p->mag = (float)(cfg->magnitude != 0.0 ? cfg->magnitude
                     : cfg->scaling == VOKRA_HIP_ROPE_YARN ? 0.1 * std::log(cfg->factor) + 1.0
                                                           : 1.0);
    hipError_t e = hipMalloc((void**)&p->turn, n * sizeof(uint64_t));
    if (e == hipSuccess)
        e = hipMemcpyAsync(p->turn, turn, n * sizeof(uint64_t), hipMemcpyHostToDevice, vk::ctx_stream(c));
    if (e == hipSuccess) e = hipStreamSynchronize(vk::ctx_stream(c));
    delete[] turn;
    if (e != hipSuccess) {
        if (p->turn) (void)hipFree(p->turn);
        delete p;
        return ctx_fail(VOKRA_HIP_ERROR_BACKEND_UNAVAILABLE, "rope_create: %s", hipGetErrorString(e));
    }
    *out = p;
    return VOKRA_HIP_OK;
}

void vokra_hip_rope_destroy(vokra_hip_rope_t* p) {
    if (!p) return;
    (void)hipSetDevice(vk::ctx_device(p->ctx));
    (void)hipStreamSynchronize(vk::ctx_stream(p->ctx));
    (void)hipFree(p->turn);
    delete p;
}

int vokra_hip_rope_apply_dev(vokra_hip_ctx_t* c, const vokra_hip_rope_t* p, size_t rows, const int32_t* d_positions,
                             size_t n_head_q, const float* d_q, size_t q_stride, float* d_q_out, size_t q_out_stride,
                             size_t n_head_k, const float* d_k, size_t k_stride, float* d_k_out, size_t k_out_stride) {
    if (!c || !p || p->ctx != c) return ctx_fail(BAD, "rope_apply: bad context or plan");
    if (rows == 0 || n_head_q + n_head_k == 0) return VOKRA_HIP_OK;
    ST_ST(rope_size(p, rows, n_head_q, n_head_k));
    if (!d_positions) return ctx_fail(BAD, "rope_apply: positions is NULL");
    ST_ST(rope_side(p, "q", rows, n_head_q, d_q, q_stride, d_q_out, q_out_stride));
    ST_ST(rope_side(p, "k", rows, n_head_k, d_k, k_stride, d_k_out, k_out_stride));
    const size_t wq = n_head_q * p->hd, wk = n_head_k * p->hd;
    if (wq && wk &&
        (rows_meet(rows, d_q_out, wq, q_out_stride, d_k, wk, k_stride) ||
         rows_meet(rows, d_k_out, wk, k_out_stride, d_q, wq, q_stride) ||
         rows_meet(rows, d_q_out, wq, q_out_stride, d_k_out, wk, k_out_stride)))
        return ctx_fail(BAD, "rope_apply: an output overlaps the other side's input or output");
    if ((wq && meet(d_q_out, ((rows - 1) * q_out_stride + wq) * 4, d_positions, rows * 4)) ||
        (wk && meet(d_k_out, ((rows - 1) * k_out_stride + wk) * 4, d_positions, rows * 4)))
        return ctx_fail(BAD, "rope_apply: an output overlaps positions");
    ST_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    RopeArgs a = {};
    a.q = n_head_q ? d_q : d_k;  // (an absent side is given the other's address and never read)
    a.k = d_k;
    a.q_out = n_head_q ? d_q_out : d_k_out;
    a.k_out = d_k_out;
    a.q_stride = n_head_q ? q_stride : k_stride;
    a.qo_stride = n_head_q ? q_out_stride : k_out_stride;
    a.k_stride = k_stride;
    a.ko_stride = k_out_stride;
    a.positions = d_positions;
    a.turn = p->turn;
    a.mag = p->mag;
    a.rows = (int)rows;
    a.heads_q = (int)n_head_q;
    a.heads_k = (int)n_head_k;
    a.hd = (int)p->hd;
    a.rot = (int)p->rot;
    ST_TRY(vk::launch_rope_turn(vk::ctx_stream(c), a, p->pairs), "launch(vk_rope_turn)");
    return VOKRA_HIP_OK;
}

int vokra_hip_rope_apply(vokra_hip_ctx_t* c, const vokra_hip_rope_t* p, size_t rows, const int32_t* positions,
                         size_t n_head_q, const float* q, float* q_out, size_t n_head_k, const float* k,
                         float* k_out) {
    if (!c || !p || p->ctx != c) return ctx_fail(BAD, "rope_apply: bad context or plan");
    if (rows == 0 || n_head_q + n_head_k == 0) return VOKRA_HIP_OK;
    ST_ST(rope_size(p, rows, n_head_q, n_head_k));
    if (!positions || (n_head_q && (!q || !q_out)) || (n_head_k && (!k || !k_out)))
        return ctx_fail(BAD, "rope_apply: NULL buffer");
    ST_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    hipStream_t s = vk::ctx_stream(c);
    const size_t wq = n_head_q * p->hd, wk = n_head_k * p->hd;
    Temp x, pos;
    ST_TRY(x.make(rows * (wq + wk) * sizeof(float)), "hipMalloc");
    ST_TRY(pos.make(rows * sizeof(int32_t)), "hipMalloc");
    float *dq = (float*)x.p, *dk = dq + rows * wq;
    ST_TRY(hipMemcpyAsync(pos.p, positions, rows * sizeof(int32_t), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    if (wq) ST_TRY(hipMemcpyAsync(dq, q, rows * wq * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    if (wk) ST_TRY(hipMemcpyAsync(dk, k, rows * wk * sizeof(float), hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    ST_ST(vokra_hip_rope_apply_dev(c, p, rows, (const int32_t*)pos.p, n_head_q, dq, wq, dq, wq, n_head_k, dk, wk, dk,
                                   wk));
    if (wq) ST_TRY(hipMemcpyAsync(q_out, dq, rows * wq * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    if (wk) ST_TRY(hipMemcpyAsync(k_out, dk, rows * wk * sizeof(float), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    ST_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

int vokra_hip_logits_rules_dev(vokra_hip_ctx_t* c, size_t rows, size_t vocab, size_t stride, const float* d_logits,
                               const vokra_hip_logits_rules_t* rules, float* d_out, int32_t* d_next) {
    if (!c) return ctx_fail(BAD, "logits_rules: ctx is NULL");
    ST_ST(rules_check(rules, rows, vocab, stride, d_logits, d_out, d_next));
    if (rows == 0) return VOKRA_HIP_OK;
    ST_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    RulesArgs a = {};
    a.stride = stride;
    a.vocab = (int)vocab;
    a.n_hist = (int)rules->n_hist;
    a.n_bias = (int)rules->n_bias;
    a.hist = rules->hist;
    a.bias_ids = rules->bias_ids;
    a.bias = rules->bias;
    a.mask_stride = rules->mask_stride;
    if (d_next) {
        void* p = nullptr;
        ST_ST(vk::ctx_rules_part(c, &p));
        a.best = (unsigned long long*)p;
        a.done = (unsigned*)(a.best + kRulesRows);
    }
    a.rows = (int)rows;
    a.logits = d_logits;
    a.out = d_out;
    a.next = d_next;
    a.hist_off = rules->n_hist ? rules->hist_offsets : nullptr;
    a.bias_off = rules->n_bias ? rules->bias_offsets : nullptr;
    a.repetition = rules->repetition;
    a.presence = rules->presence;
    a.frequency = rules->frequency;
    a.mask = rules->mask;
    ST_TRY(vk::launch_rules(vk::ctx_stream(c), a), "launch(vk_rules)");
    return VOKRA_HIP_OK;
}

int vokra_hip_logits_rules(vokra_hip_ctx_t* c, size_t rows, size_t vocab, const float* logits,
                           const vokra_hip_logits_rules_t* rules, float* out, int32_t* next) {
    if (!c) return ctx_fail(BAD, "logits_rules: ctx is NULL");
    ST_ST(rules_check(rules, rows, vocab, vocab, logits, out, next));
    if (rows == 0) return VOKRA_HIP_OK;
    for (int side = 0; side < 2; ++side) {
        const int32_t* off = side ? rules->bias_offsets : rules->hist_offsets;
        const size_t n = side ? rules->n_bias : rules->n_hist;
        if (!n) continue;
        for (size_t r = 0; r <= rows; ++r)
            if (off[r] < 0 || (size_t)off[r] > n || (r && off[r] < off[r - 1]))
                return ctx_fail(BAD, "logits_rules: offset %zu of the %s is out of order or range", r,
                                side ? "biases" : "history");
    }
    ST_TRY(hipSetDevice(vk::ctx_device(c)), "hipSetDevice");
    hipStream_t s = vk::ctx_stream(c);
    Temp t[11];
    const void* d[9];
    vokra_hip_logits_rules_t r = *rules;
    const size_t n = rows * vocab * sizeof(float), words = (vocab + 31) / 32;
    const size_t mask_words = r.mask_stride ? (rows - 1) * r.mask_stride + words : words;
    ST_ST(to_device(s, t[0], r.n_hist ? r.hist : nullptr, r.n_hist * 4, &d[0]));
    ST_ST(to_device(s, t[1], r.n_hist ? r.hist_offsets : nullptr, (rows + 1) * 4, &d[1]));
    ST_ST(to_device(s, t[2], r.repetition, rows * 4, &d[2]));
    ST_ST(to_device(s, t[3], r.presence, rows * 4, &d[3]));
    ST_ST(to_device(s, t[4], r.frequency, rows * 4, &d[4]));
    ST_ST(to_device(s, t[5], r.n_bias ? r.bias_ids : nullptr, r.n_bias * 4, &d[5]));
    ST_ST(to_device(s, t[6], r.n_bias ? r.bias : nullptr, r.n_bias * 4, &d[6]));
    ST_ST(to_device(s, t[7], r.n_bias ? r.bias_offsets : nullptr, (rows + 1) * 4, &d[7]));
    ST_ST(to_device(s, t[8], r.mask, mask_words * 4, &d[8]));
    r.hist = (const int32_t*)d[0];
    r.hist_offsets = (const int32_t*)d[1];
    r.repetition = (const float*)d[2];
    r.presence = (const float*)d[3];
    r.frequency = (const float*)d[4];
    r.bias_ids = (const int32_t*)d[5];
    r.bias = (const float*)d[6];
    r.bias_offsets = (const int32_t*)d[7];
    r.mask = (const uint32_t*)d[8];
    ST_TRY(t[9].make(n), "hipMalloc");
    ST_TRY(t[10].make(rows * sizeof(int32_t)), "hipMalloc");
    float* x = (float*)t[9].p;
    ST_TRY(hipMemcpyAsync(x, logits, n, hipMemcpyHostToDevice, s), "hipMemcpyAsync");
    ST_ST(vokra_hip_logits_rules_dev(c, rows, vocab, vocab, x, &r, out ? x : nullptr,
                                     next ? (int32_t*)t[10].p : nullptr));
    if (out) ST_TRY(hipMemcpyAsync(out, x, n, hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    if (next) ST_TRY(hipMemcpyAsync(next, t[10].p, rows * sizeof(int32_t), hipMemcpyDeviceToHost, s), "hipMemcpyAsync");
    ST_TRY(hipStreamSynchronize(s), "hipStreamSynchronize");
    return VOKRA_HIP_OK;
}

}  // extern "C"
