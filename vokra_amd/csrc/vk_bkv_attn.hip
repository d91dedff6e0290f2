// vk_bkv_attn.hip — attention of a step's rows over the block-scaled KV cache.
//
// Row r of the step belongs to item i, at position p = start_i + (r - row0_i);
// query head h reads kv head h / (hq / n_head):
//   s_j = scale q . k_j (j <= p), out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// with k, v the values that the cache holds: 8-bit ones under their block's
// scale, f32 rows in the open block.
#include "vk_bkv.h"
#include "vk_common.h"

namespace vk {

__device__ __forceinline__ float bkv_value(const BkvView& v, uint32_t byte) {
    return v.codec == BKV_INT8 ? (float)((int)byte - 128) : __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}

// One workgroup per (row, query head): a thread per key for the scores of 256
// keys at a time, then a thread per element of the output.
__global__ __launch_bounds__(256) void vk_bkv_attn_rows(BkvView v, int layer, int hq, const float* __restrict__ q,
                                                        float scale, float* __restrict__ out) {
    __shared__ float sq[128], sp[256], red[4], so[256];
    const int r = blockIdx.x, h = blockIdx.y, hd = v.hd;
    const int n = v.meta[BKV_STEP_N];
    if (r >= v.meta[BKV_STEP_ROWS]) return;
    int i = 0;
    while (i + 1 < n && v.step[i + 1].row0 <= r) ++i;
    while (v.step[i].row0 + v.step[i].count <= r) --i;  // items without rows share a row0
    const BkvItem it = v.step[i];
    const int keys = it.start + (r - it.row0) + 1, full = (it.start + it.count) / v.bs * v.bs;
    const int head = h / (hq / v.n_head), tid = threadIdx.x;
    const size_t o = ((size_t)r * hq + h) * hd;
    if (tid < hd) sq[tid] = q[o + tid] * scale;
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    const int d = tid % hd, part = tid / hd, parts = 256 / hd;
    for (int j0 = 0; j0 < keys; j0 += 256) {
        __syncthreads();
        const int j = j0 + tid;
        float s = -INFINITY;
        if (j < keys) {
            s = 0.0f;
            if (j < full) {
                const int page = v.table[(size_t)it.seq * v.max_blocks + j / v.bs];
                const size_t chunk = ((size_t)layer * v.n_page + page) * v.n_head + head;
                const uint8_t* p = v.pool + chunk * 2 * v.bs * hd + (size_t)(j % v.bs / 16) * 16 * hd;
                for (int x = 0; x < hd; ++x) s += sq[x] * bkv_value(v, p[bkv_k_off(j & 15, x)]);
                s *= v.scales[chunk * 2];
            } else {
                const float* p = v.ring + (((((size_t)layer * v.n_seq + it.seq) * 2) * v.n_head + head) * 2 * v.bs +
                                           j % (2 * v.bs)) * hd;
                for (int x = 0; x < hd; ++x) s += sq[x] * p[x];
            }
        }
        float t = vk_group_maxf<64>(s);
        if ((tid & 63) == 0) red[tid >> 6] = t;
        __syncthreads();
        const float m1 = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        __syncthreads();
        const float e = j < keys ? expf(s - m1) : 0.0f, c = m == -INFINITY ? 0.0f : expf(m - m1);
        sp[tid] = e;
        t = vk_group_sumf<64>(e);
        if ((tid & 63) == 0) red[tid >> 6] = t;
        __syncthreads();
        l = l * c + ((red[0] + red[1]) + (red[2] + red[3]));
        m = m1;
        acc *= c;
        const int jn = min(256, keys - j0);
        for (int x = part; x < jn; x += parts) {
            const int jj = j0 + x;
            float y;
            if (jj < full) {
                const int page = v.table[(size_t)it.seq * v.max_blocks + jj / v.bs];
                const size_t chunk = ((size_t)layer * v.n_page + page) * v.n_head + head;
                const uint8_t* p = v.pool + chunk * 2 * v.bs * hd + (size_t)v.bs * hd + (size_t)(jj % v.bs / 16) * 16 * hd;
                y = bkv_value(v, p[bkv_v_off(jj & 15, d)]) * v.scales[chunk * 2 + 1];
            } else {
                y = v.ring[(((((size_t)layer * v.n_seq + it.seq) * 2 + 1) * v.n_head + head) * 2 * v.bs +
                            jj % (2 * v.bs)) * hd + d];
            }
            acc += sp[x] * y;
        }
    }
    __syncthreads();
    so[tid] = acc;
    __syncthreads();
    if (part == 0) {
        for (int x = 1; x < parts; ++x) acc += so[x * hd + d];
        out[o + d] = acc / l;
    }
}

hipError_t launch_bkv_attn(hipStream_t s, const BkvView& v, int layer, int n, int n_rows, int max_count, int max_len,
                           int hq, const float* q, float scale, float* out, float* part) {
    (void)n, (void)max_count, (void)max_len, (void)part;
    if (n_rows == 0) return hipSuccess;
    hipLaunchKernelGGL(vk_bkv_attn_rows, dim3((unsigned)n_rows, (unsigned)hq), dim3(256), 0, s, v, layer, hq, q, scale,
                       out);
    return hipGetLastError();
}

}  // namespace vk
