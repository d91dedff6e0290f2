// vk_rules.hip — logits through a step's rules, with the greedy choice.
//
// Per row, for token v that stands n_v times in the row's history:
//   n_v > 0:  x = x > 0 ? x / repetition : x * repetition,
//             x = x - (presence + frequency * n_v);
//   a bias for v: x = x + bias (the last one where v is given several times);
//   v not allowed by the mask: x = -inf;
// then the first largest x above -inf (a NaN never is), -1 if there is none.
//
// A workgroup takes 4096 or 8192 columns of a row, from a 16-byte boundary on,
// into registers. One table in LDS, a number a column, first counts the history's
// tokens in them (integer adds, so their order does not matter) and then holds
// the last bias entry of each (integer max); each list is read by every workgroup
// of its row, from cache, and skipped where a row has none. Each column is
// read and written once, past the caches. Bound by those 8 bytes: 192 rows of 128259
// columns with up to 2048 tokens and 300 biases a row take 50 us (4.0 TB/s; 54 through
// the caches, 256 rows of 100000 with a mask 46 against 56); 32 rows of 32000 columns
// take 8.5 us, which is dependent rounds of memory. Two tables at once, filled between
// the same barriers, took 15 us longer: 33 KB of LDS leave half the waves.
// The choice: each workgroup's best goes into the row's 64-bit maximum (value,
// then the lower index: the order of the workgroups does not matter), and the
// last of the row's workgroups writes it out and clears it for the next call.
#include "vk_common.h"
#include "vk_step.h"

namespace vk {

constexpr int RU_T = 512;  // threads

// (value desc, index asc): the first strict maximum
__device__ __forceinline__ void ru_merge(float& v, int& i, float w, int j) {
    if (w > v || (w == v && j < i)) {
        v = w;
        i = j;
    }
}

// RU_VEC: 16-byte pieces a thread
template <int RU_VEC>
__global__ __launch_bounds__(RU_T) void vk_rules(RulesArgs a) {
    constexpr int RU_SLICE = 4 * RU_T * RU_VEC;
    __shared__ int4 table4[RU_SLICE / 4];
    __shared__ float rv[RU_T / 64];
    __shared__ int ri[RU_T / 64];
    int* table = (int*)table4;
    const int row = blockIdx.y, t = threadIdx.x;
    const float* x = a.logits + (size_t)row * a.stride;
    // column c0 + 4 k lies on a 16-byte boundary of the row
    const int c0 = (int)blockIdx.x * RU_SLICE - (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3);
    float y[4 * RU_VEC];
#pragma unroll
    for (int j = 0; j < RU_VEC; ++j) {
        const int c = c0 + 4 * (t + RU_T * j);
        if (c >= 0 && c + 3 < a.vocab) {
            const vk_f32x4 x4 = __builtin_nontemporal_load((const vk_f32x4*)(x + c));
            y[4 * j] = x4.x, y[4 * j + 1] = x4.y, y[4 * j + 2] = x4.z, y[4 * j + 3] = x4.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * j + i] = c + i >= 0 && c + i < a.vocab ? x[c + i] : 0.0f;
        }
    }
    const bool hist = a.hist_off, biased = a.bias_off;
    const int h0 = hist ? max(a.hist_off[row], 0) : 0, h1 = hist ? min(a.hist_off[row + 1], a.n_hist) : 0;
    const int b0 = biased ? max(a.bias_off[row], 0) : 0, b1 = biased ? min(a.bias_off[row + 1], a.n_bias) : 0;
    const float rep = a.repetition ? a.repetition[row] : 1.0f, pres = a.presence ? a.presence[row] : 0.0f,
                freq = a.frequency ? a.frequency[row] : 0.0f;
    const int lo = max(c0, 0), hi = min(c0 + RU_SLICE, a.vocab);
    int4* mine = table4 + t;  // + RU_T j: this thread's columns
    if (h1 > h0 || b1 > b0) {
#pragma unroll
        for (int j = 0; j < RU_VEC; ++j) mine[RU_T * j] = make_int4(0, 0, 0, 0);
        __syncthreads();
    }
    if (h1 > h0) {
        // (places beyond a list's end may be beyond int)
        for (unsigned i = (unsigned)h0 + t; i < (unsigned)h1; i += 8 * RU_T) {
            int v[8];  // loads in flight
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = i + RU_T * j < (unsigned)h1 ? a.hist[i + RU_T * j] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v[j] >= lo && v[j] < hi) atomicAdd(&table[v[j] - c0], 1);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RU_VEC; ++j) {
            const int4 k4 = mine[RU_T * j];
            if (!(k4.x | k4.y | k4.z | k4.w)) continue;
            float* z = &y[4 * j];
            const int k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k[i]) {
                    z[i] = z[i] > 0.0f ? z[i] / rep : z[i] * rep;
                    z[i] = z[i] - (pres + freq * (float)k[i]);
                }
            mine[RU_T * j] = make_int4(0, 0, 0, 0);
        }
    }
    if (b1 > b0) {
        if (h1 > h0) __syncthreads();
        for (unsigned i = (unsigned)b0 + t; i < (unsigned)b1; i += 2 * RU_T) {
            int v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) v[j] = i + RU_T * j < (unsigned)b1 ? a.bias_ids[i + RU_T * j] : -1;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (v[j] >= lo && v[j] < hi) atomicMax(&table[v[j] - c0], (int)(i + RU_T * j - b0) + 1);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < RU_VEC; ++j) {
            const int4 s4 = mine[RU_T * j];
            const int s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (s[i]) y[4 * j + i] = y[4 * j + i] + a.bias[b0 + s[i] - 1];
        }
    }
    const uint32_t* mask = a.mask ? a.mask + (size_t)row * a.mask_stride : nullptr;
    float* out = a.out ? a.out + (size_t)row * a.stride : nullptr;
    const bool vec = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0;
    float bv = -INFINITY;
    int bi = INT_MAX;
#pragma unroll
    for (int j = 0; j < RU_VEC; ++j) {
        const int c = c0 + 4 * (t + RU_T * j);
        float* z = &y[4 * j];
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
                __builtin_nontemporal_store(vk_f32x4{z[0], z[1], z[2], z[3]}, (vk_f32x4*)(out + c));
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
    for (int w = 1; w < RU_T / 64; ++w) ru_merge(bv, bi, rv[w], ri[w]);
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

template <int RU_VEC>
static void rules_grid(hipStream_t s, const RulesArgs& a) {
    constexpr int slice = 4 * RU_T * RU_VEC;
    // a row may begin up to three columns before a boundary
    hipLaunchKernelGGL(vk_rules<RU_VEC>, dim3((unsigned)((a.vocab + 3 + slice - 1) / slice), (unsigned)a.rows),
                       dim3(RU_T), 0, s, a);
}

hipError_t launch_rules(hipStream_t s, const RulesArgs& a) {
    // up to two workgroups of 4096 columns a CU, half the columns a thread end
    // earlier (32 rows of 32000 columns: 8.8 us against 9.8); above that, whole
    // slices halve the reads of the rows' lists (64 rows of 51866 columns: 11.2 us
    // against 12.5, 192 of 128259: 54 against 65)
    if ((size_t)a.rows * a.vocab <= (size_t)512 * 4096)
        rules_grid<2>(s, a);
    else
        rules_grid<4>(s, a);
    return hipGetLastError();
}

}  // namespace vk
