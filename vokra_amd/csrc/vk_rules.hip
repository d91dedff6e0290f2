// vk_rules.hip — logits through a step's rules, with the greedy choice.
//
// Per row, for token v that stands n_v times in the row's history:
//   n_v > 0:  x = x > 0 ? x / repetition : x * repetition,
//             x = x - (presence + frequency * n_v);
//   a bias for v: x = x + bias (the last one where v is given several times);
//   v not allowed by the mask: x = -inf;
// then the first largest x above -inf (a NaN never is), -1 if there is none.
//
// A workgroup takes 4096 columns of a row: counts of the history's tokens in
// them (integer adds, so their order does not matter) and the last bias entry
// of each (integer max) are gathered in LDS, then each column is read and
// written once. Bound by those 8 bytes a column.
#include "vk_common.h"
#include "vk_step.h"

namespace vk {

constexpr int RU_SLICE = 4096;

// (value desc, index asc): the first strict maximum
__device__ __forceinline__ void ru_merge(float& v, int& i, float w, int j) {
    if (w > v || (w == v && j < i)) {
        v = w;
        i = j;
    }
}
__device__ __forceinline__ void ru_reduce(float& v, int& i, float* rv, int* ri) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ru_merge(v, i, __shfl_xor(v, o, VK_WAVE), __shfl_xor(i, o, VK_WAVE));
    if ((threadIdx.x & 63) == 0) {
        rv[threadIdx.x >> 6] = v;
        ri[threadIdx.x >> 6] = i;
    }
    __syncthreads();
    for (int w = 0; w < 4; ++w) ru_merge(v, i, rv[w], ri[w]);
}

__global__ __launch_bounds__(256) void vk_rules(RulesArgs a) {
    __shared__ int count[RU_SLICE], slot[RU_SLICE];
    __shared__ float rv[4];
    __shared__ int ri[4];
    const int row = blockIdx.y, c0 = blockIdx.x * RU_SLICE, n = min(RU_SLICE, a.vocab - c0);
    const float* x = a.logits + (size_t)row * a.stride;
    for (int c = threadIdx.x; c < RU_SLICE; c += 256) count[c] = slot[c] = 0;
    __syncthreads();
    if (a.hist_off) {
        const int e = min(a.hist_off[row + 1], a.n_hist);
        for (int i = max(a.hist_off[row], 0) + (int)threadIdx.x; i < e; i += 256) {
            const int c = a.hist[i] - c0;
            if ((unsigned)c < (unsigned)n) atomicAdd(&count[c], 1);
        }
    }
    const int b0 = a.bias_off ? max(a.bias_off[row], 0) : 0;
    if (a.bias_off) {
        const int e = min(a.bias_off[row + 1], a.n_bias);
        for (int i = b0 + (int)threadIdx.x; i < e; i += 256) {
            const int c = a.bias_ids[i] - c0;
            if ((unsigned)c < (unsigned)n) atomicMax(&slot[c], i - b0 + 1);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f,
                freq = a.frequency ? a.frequency[row] : 0.0f;
    float bv = -INFINITY;
    int bi = INT_MAX;
    for (int c = threadIdx.x; c < n; c += 256) {
        float y = x[c0 + c];
        if (const int k = count[c]) {
            y = y > 0.0f ? y / rep : y * rep;
            y = y - (pres + freq * (float)k);
        }
        if (const int k = slot[c]) y = y + a.bias[b0 + k - 1];
        if (a.mask) {
            const int v = c0 + c;
            if (!((a.mask[(size_t)row * a.mask_stride + (v >> 5)] >> (v & 31)) & 1u)) y = -INFINITY;
        }
        if (a.out) a.out[(size_t)row * a.stride + c0 + c] = y;
        if (y > bv) {
            bv = y;
            bi = c0 + c;
        }
    }
    if (!a.next) return;
    ru_reduce(bv, bi, rv, ri);
    if (threadIdx.x == 0) a.part[(size_t)row * gridDim.x + blockIdx.x] = make_float2(bv, __int_as_float(bi));
}

__global__ __launch_bounds__(256) void vk_rules_next(const float2* __restrict__ part, int n, int* __restrict__ next) {
    __shared__ float rv[4];
    __shared__ int ri[4];
    float bv = -INFINITY;
    int bi = INT_MAX;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float2 p = part[(size_t)blockIdx.x * n + i];
        ru_merge(bv, bi, p.x, __float_as_int(p.y));
    }
    ru_reduce(bv, bi, rv, ri);
    if (threadIdx.x == 0) next[blockIdx.x] = bv > -INFINITY ? bi : -1;
}

int rules_slices(int vocab) { return (vocab + RU_SLICE - 1) / RU_SLICE; }

hipError_t launch_rules(hipStream_t s, const RulesArgs& a) {
    const int n = rules_slices(a.vocab);
    hipLaunchKernelGGL(vk_rules, dim3((unsigned)n, (unsigned)a.rows), dim3(256), 0, s, a);
    if (a.next) hipLaunchKernelGGL(vk_rules_next, dim3((unsigned)a.rows), dim3(256), 0, s, a.part, n, a.next);
    return hipGetLastError();
}

}  // namespace vk
