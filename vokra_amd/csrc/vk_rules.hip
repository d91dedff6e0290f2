// vk_rules.hip — logits through a step's rules, with the greedy choice.
//
// Per row, for token v that stands n_v times in the row's history:
//   n_v > 0:  x = x > 0 ? x / repetition : x * repetition,
//             x = x - (presence + frequency * n_v);
//   a bias for v: x = x + bias (the last one where v is given several times);
//   v not allowed by the mask: x = -inf;
// then the first largest x above -inf (a NaN never is), -1 if there is none.
//
// A workgroup takes 4096 columns of a row, from a 16-byte boundary on: it loads
// them, gathers the counts of the history's tokens in them (integer adds, so
// their order does not matter) and the last bias entry of each (integer max) in
// LDS meanwhile, and writes each column once. Bound by those 8 bytes a column;
// a long history is read by every workgroup of its row (from cache).
// The choice: each workgroup's best goes into the row's 64-bit maximum (value,
// then the lower index: the order of the workgroups does not matter), and the
// last of the row's workgroups writes it out and clears it for the next call.
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

__global__ __launch_bounds__(256) void vk_rules(RulesArgs a) {
    __shared__ int4 count4[RU_SLICE / 4], slot4[RU_SLICE / 4];
    __shared__ float rv[4];
    __shared__ int ri[4];
    int *count = (int*)count4, *slot = (int*)slot4;
    const int row = blockIdx.y, t = threadIdx.x;
    const float* x = a.logits + (size_t)row * a.stride;
    // column c0 + 4 k lies on a 16-byte boundary of the row
    const int c0 = (int)blockIdx.x * RU_SLICE - (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    float4 y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = c0 + 4 * (t + 256 * j);
        if (c >= 0 && c + 3 < a.vocab) {
            y[j] = *(const float4*)(x + c);
        } else {
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = c + i >= 0 && c + i < a.vocab ? x[c + i] : 0.0f;
            y[j] = make_float4(z[0], z[1], z[2], z[3]);
        }
    }
    const bool hist = a.hist_off, biased = a.bias_off;
    const int h0 = hist ? max(a.hist_off[row], 0) : 0, h1 = hist ? min(a.hist_off[row + 1], a.n_hist) : 0;
    const int b0 = biased ? max(a.bias_off[row], 0) : 0, b1 = biased ? min(a.bias_off[row + 1], a.n_bias) : 0;
    const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f,
                freq = a.frequency ? a.frequency[row] : 0.0f;
    const bool listed = h1 > h0 || b1 > b0;
    if (listed) {
#pragma unroll
        for (int j = 0; j < 4; ++j) count4[t + 256 * j] = slot4[t + 256 * j] = make_int4(0, 0, 0, 0);
        __syncthreads();
        const int lo = max(c0, 0), hi = min(c0 + RU_SLICE, a.vocab);
        // eight (two) loads in flight
        for (int i = h0 + t; i < h1; i += 8 * 256) {
            int v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = i + 256 * j < h1 ? a.hist[i + 256 * j] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v[j] >= lo && v[j] < hi) atomicAdd(&count[v[j] - c0], 1);
        }
        for (int i = b0 + t; i < b1; i += 2 * 256) {
            int v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] = i + 256 * j < b1 ? a.bias_ids[i + 256 * j] : -1;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (v[j] >= lo && v[j] < hi) atomicMax(&slot[v[j] - c0], i + 256 * j - b0 + 1);
        }
        __syncthreads();
    }
    const uint32_t* mask = a.mask ? a.mask + (size_t)row * a.mask_stride : nullptr;
    float* out = a.out ? a.out + (size_t)row * a.stride : nullptr;
    const bool vec = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0;
    float bv = -INFINITY;
    int bi = INT_MAX;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int g = t + 256 * j, c = c0 + 4 * g;
        float z[4] = {y[j].x, y[j].y, y[j].z, y[j].w};
        if (listed) {
            const int4 k4 = count4[g], s4 = slot4[g];
            const int k[4] = {k4.x, k4.y, k4.z, k4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (k[i]) {
                    z[i] = z[i] > 0.0f ? z[i] / rep : z[i] * rep;
                    z[i] = z[i] - (pres + freq * (float)k[i]);
                }
                if (s[i]) z[i] = z[i] + a.bias[b0 + s[i] - 1];
            }
        }
        if (mask) {
            // the four bits lie in one word or two
            const int w0 = max(c, 0) >> 5, w1 = min(max(c + 3, 0), a.vocab - 1) >> 5;
            const uint32_t m0 = w0 <= w1 ? mask[w0] : 0u, m1 = w0 < w1 ? mask[w1] : m0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t m = (c + i) >> 5 == w0 ? m0 : m1;
                if (!((m >> ((c + i) & 31)) & 1u)) z[i] = -INFINITY;
            }
        }
        if (c >= 0 && c + 3 < a.vocab) {
            if (out && vec) {
                *(float4*)(out + c) = make_float4(z[0], z[1], z[2], z[3]);
            } else if (out) {
#pragma unroll
                for (int i = 0; i < 4; ++i) out[c + i] = z[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (z[i] > bv) {
                    bv = z[i];
                    bi = c + i;
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i >= 0 && c + i < a.vocab) {
                    if (out) out[c + i] = z[i];
                    if (z[i] > bv) {
                        bv = z[i];
                        bi = c + i;
                    }
                }
        }
    }
    if (!a.next) return;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ru_merge(bv, bi, __shfl_xor(bv, o, VK_WAVE), __shfl_xor(bi, o, VK_WAVE));
    if ((t & 63) == 0) {
        rv[t >> 6] = bv;
        ri[t >> 6] = bi;
    }
    __syncthreads();
    if (t != 0) return;
    for (int w = 1; w < 4; ++w) ru_merge(bv, bi, rv[w], ri[w]);
    // the value's bits in the order of the values, above the lower index first; 0: nothing
    if (bv == 0.0f) bv = 0.0f;  // one zero
    const uint32_t b = __float_as_uint(bv), ord = b & 0x80000000u ? ~b : b | 0x80000000u;
    unsigned long long key = bv > -INFINITY ? ((unsigned long long)ord << 32) | (0xffffffffu - (uint32_t)bi) : 0ull;
    if (gridDim.x > 1) {
        // the maximum has been taken when its old value is here; only then this
        // workgroup is counted
        unsigned long long old = atomicMax(&a.best[row], key);
        asm volatile("" : "+v"(old)::"memory");
        if (atomicAdd(&a.done[row], 1u) != gridDim.x - 1) return;
        key = atomicExch(&a.best[row], 0ull);
        atomicExch(&a.done[row], 0u);
    }
    a.next[row] = key ? (int)(0xffffffffu - (uint32_t)key) : -1;
}

__global__ void vk_rules_clear(uint4* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        p[i] = make_uint4(0, 0, 0, 0);
}

hipError_t launch_rules_clear(hipStream_t s, void* part) {
    hipLaunchKernelGGL(vk_rules_clear, dim3(64), dim3(256), 0, s, (uint4*)part, kRulesPartBytes / 16);
    return hipGetLastError();
}

hipError_t launch_rules(hipStream_t s, const RulesArgs& a) {
    // a row may begin up to three columns before a boundary
    hipLaunchKernelGGL(vk_rules, dim3((unsigned)((a.vocab + 3 + RU_SLICE - 1) / RU_SLICE), (unsigned)a.rows), dim3(256),
                       0, s, a);
    return hipGetLastError();
}

}  // namespace vk
