// vk_beam.hip — beam search's selection: the n best continuations of a group's beams.
//
// A live beam's continuation by token v is worth
//   total = score + (x_v - ln sum_w e^(x_w)),
// an ended beam has one, its end token at its own score. A group's n_out best go out,
// the larger total first; of equal totals the lower beam, in one beam the larger logit
// and then the lower token.
//
// Two launches. Slices: a workgroup reads 4096 or 8192 columns of a row once, into
// registers, and leaves their maximum, the sum of their exponentials and their n_out best
// columns. Merge: a workgroup a group joins the slices' sums (64 bits: totals of
// different beams are compared, and near ones have to fall in order), takes each
// beam's best from its slices' lists and the group's from its beams'.
//
// The best of a slice without a sort of it: the n_out-th largest of the 256 threads' own
// maxima bounds the n_out-th largest column from below, and hardly more than n_out columns
// reach it. They are put into LDS and ranked by counting. Where too many do (ties), they
// are taken one after the other.
//
// A logit that is NaN counts as -inf; a row with +inf has no continuations (its
// log-softmax has no value). Sums do not depend on where a row lies in memory, so
// equal rows have equal totals.
#include "vk_beam.h"
#include "vk_common.h"

namespace vk {

constexpr int BM_T = 256;     // threads of a slice
constexpr int BM_CAND = 256;  // candidates that are ranked at once
constexpr int BM_MT = 512;    // threads of a merge: eight waves, a beam each in turn
constexpr int BM_LIST = 1024; // entries of a beam's lists that a wave holds in LDS

// Values in the order of their bits, a column index that falls with it behind: the larger
// key is the better column. Key 0: none.
__device__ __forceinline__ unsigned long long bm_key(float x, int column) {
    const uint32_t b = __float_as_uint(x), ord = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((unsigned long long)ord << 32) | (0xffffffffu - (uint32_t)column);
}
__device__ __forceinline__ float bm_value(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int bm_column(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

__device__ __forceinline__ unsigned long long bm_wave_max(unsigned long long k) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long y = __shfl_xor(k, o, VK_WAVE);
        k = y > k ? y : k;
    }
    return k;
}

// A row that goes on: not ended, with a score above -inf.
__device__ __forceinline__ bool bm_live(const BeamArgs& a, int row) {
    return !(a.ended && a.ended[row]) && a.scores[row] > -INFINITY;
}

typedef float bm_f4 __attribute__((ext_vector_type(4), aligned(4)));

// E columns a thread, in runs of four
template <int E>
__global__ __launch_bounds__(BM_T) void vk_beam_slices(BeamArgs a) {
    constexpr int SLICE = BM_T * E;
    __shared__ float s_max[4], s_sorted[4][64], s_bound;
    __shared__ double s_sum[4];
    __shared__ unsigned long long s_key[BM_CAND];
    __shared__ int s_n;
    const int row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (!bm_live(a, row)) return;
    const float* x = a.logits + (size_t)row * a.stride;
    const int c0 = (int)blockIdx.x * SLICE;
    float y[E];
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
        const int c = c0 + 4 * (t + BM_T * j);
        if (c + 3 < a.vocab) {
            const bm_f4 v = __builtin_nontemporal_load((const bm_f4*)(x + c));
            y[4 * j] = v.x, y[4 * j + 1] = v.y, y[4 * j + 2] = v.z, y[4 * j + 3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * j + i] = c + i < a.vocab ? x[c + i] : -INFINITY;
        }
    }
    if (t == 0) s_n = 0;
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        if (!(y[j] == y[j])) y[j] = -INFINITY;
        if (y[j] == 0.0f) y[j] = 0.0f;  // one zero
        most = fmaxf(most, y[j]);
    }
    // the wave's maxima in falling order over its lanes
    float v = most;
#pragma unroll
    for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (int o = k >> 1; o > 0; o >>= 1) {
            const float w = __shfl_xor(v, o, VK_WAVE);
            const bool keeps_max = ((lane & o) == 0) == ((lane & k) == 0);
            v = keeps_max ? fmaxf(v, w) : fminf(v, w);
        }
    s_sorted[wave][lane] = v;
    if (lane == 0) s_max[wave] = v;
    __syncthreads();
    const float m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    // where v stands among all 256: of equal ones the lower wave's first
    int rank = lane;
#pragma unroll
    for (int o = 1; o < 4; ++o) {
        const int w = (wave + o) & 3;
        int n = 0;  // of wave w stand before v
#pragma unroll
        for (int step = 32; step > 0; step >>= 1) {
            const float u = s_sorted[w][n + step - 1];
            if (u > v || (u == v && w < wave)) n += step;
        }
        const float u = s_sorted[w][n];  // n <= 63 here
        if (u > v || (u == v && w < wave)) ++n;
        rank += n;
    }
    if (rank == a.n_out - 1) s_bound = v;
    float sum = 0.0f;
    if (m > -INFINITY)
#pragma unroll
        for (int j = 0; j < E; ++j) sum += __builtin_amdgcn_exp2f((y[j] - m) * 1.44269504088896340736f);
    double total = (double)sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o, VK_WAVE);
    if (lane == 0) s_sum[wave] = total;
    __syncthreads();
    const float bound = s_bound;
    if (most >= bound && most > -INFINITY) {
        int n = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) n += y[j] >= bound && y[j] > -INFINITY ? 1 : 0;
        int at = atomicAdd(&s_n, n);
        if (at + n <= BM_CAND)
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (y[j] >= bound && y[j] > -INFINITY)
                    s_key[at++] = bm_key(y[j], c0 + 4 * (t + BM_T * (j >> 2)) + (j & 3));
    }
    __syncthreads();
    const size_t part = (size_t)row * a.slices + blockIdx.x;
    unsigned long long* out = a.keys + part * a.n_out;
    int count = s_n;
    if (count <= BM_CAND) {
        if (t < count) {
            const unsigned long long k = s_key[t];
            int before = 0;
            for (int j = 0; j < count; ++j) before += s_key[j] > k ? 1 : 0;
            if (before < a.n_out) out[before] = k;
        }
        count = min(count, a.n_out);
    } else {
        unsigned long long last = ~0ull;
        for (count = 0; count < a.n_out; ++count) {
            unsigned long long k = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const unsigned long long w =
                    y[j] > -INFINITY ? bm_key(y[j], c0 + 4 * (t + BM_T * (j >> 2)) + (j & 3)) : 0;
                if (w < last && w > k) k = w;
            }
            k = bm_wave_max(k);
            __syncthreads();  // the round before has been read
            if (lane == 0) s_key[wave] = k;
            __syncthreads();
            k = max(max(s_key[0], s_key[1]), max(s_key[2], s_key[3]));
            if (!k) break;  // the same for all
            if (t == 0) out[count] = k;
            last = k;
        }
    }
    if (t == 0) a.stats[part] = BeamStat{(s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]), m, count};
}

// The n_out best of a beam's slices, by a wave: lists fall, so a lane looks at the heads
// of its slices (s, s + 64, ..) and the wave takes the best head, n_out times.
__global__ __launch_bounds__(BM_MT) void vk_beam_merge(BeamArgs a) {
    constexpr int WAVES = BM_MT / 64;
    __shared__ unsigned long long s_list[WAVES][BM_LIST];
    __shared__ double s_total[kBeamMost][kBeamOut];
    __shared__ int s_token[kBeamMost][kBeamOut], s_count[kBeamMost], s_ended[kBeamMost];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_out;
    for (int b = wave; b < a.beams; b += WAVES) {
        const int row = g * a.beams + b;
        const float score = a.scores[row];
        const bool ended = a.ended && a.ended[row], live = bm_live(a, row);
        if (lane == 0) s_ended[b] = ended;
        if (!live) {
            if (lane == 0) {
                s_count[b] = ended && score > -INFINITY ? 1 : 0;
                s_total[b][0] = (double)score;
                s_token[b][0] = a.end_token;
            }
            continue;
        }
        const BeamStat* st = a.stats + (size_t)row * a.slices;
        const unsigned long long* keys = a.keys + (size_t)row * a.slices * n;
        const bool staged = a.slices * n <= BM_LIST;
        if (staged) {
            for (int i = lane; i < a.slices * n; i += 64) s_list[wave][i] = keys[i];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own list: no barrier
        }
        auto key = [&](int s, int i) { return staged ? s_list[wave][s * n + i] : keys[(size_t)s * n + i]; };
        float m = -INFINITY;
        for (int s = lane; s < a.slices; s += 64) m = fmaxf(m, st[s].max);
        m = vk_group_maxf<64>(m);
        double sum = 0.0;
        for (int s = lane; s < a.slices; s += 64)
            if (st[s].max > -INFINITY) sum += st[s].sum * exp((double)st[s].max - (double)m);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, VK_WAVE);
        const double lse = (double)m + log(sum);
        // the best key of a lane's slices that is not taken yet
        int taken = 0, place = 0;
        unsigned long long last = ~0ull, mine = 0;
        auto next = [&]() {
            mine = 0;
            if (a.slices <= 64) {  // one list a lane
                if (lane < a.slices && place < st[lane].count) mine = key(lane, place++);
                return;
            }
            for (int s = lane; s < a.slices; s += 64) {
                const int c = st[s].count;
                for (int i = 0; i < c; ++i) {
                    const unsigned long long k = key(s, i);
                    if (k >= last) continue;
                    if (k > mine) mine = k;
                    break;
                }
            }
        };
        next();
        for (; taken < n; ++taken) {
            const unsigned long long k = bm_wave_max(mine);
            if (!k) break;
            const double total = (double)score + ((double)bm_value(k) - lse);
            if (!(total > -INFINITY)) break;  // NaN: the row holds +inf
            if (lane == 0) {
                s_total[b][taken] = total;
                s_token[b][taken] = bm_column(k);
            }
            last = k;
            if (mine == k) next();
        }
        if (lane == 0) s_count[b] = taken;
    }
    __syncthreads();
    if (wave != 0) return;
    int at = 0;
    const int count = lane < a.beams ? s_count[lane] : 0;
    for (int i = 0; i < n; ++i) {
        double best = at < count ? s_total[lane][at] : -INFINITY;
        int from = lane;
#pragma unroll
        for (int o = 1; o < kBeamMost; o <<= 1) {
            const double w = __shfl_xor(best, o, VK_WAVE);
            const int f = __shfl_xor(from, o, VK_WAVE);
            if (w > best || (w == best && f < from)) {
                best = w;
                from = f;
            }
        }
        const size_t o = (size_t)g * n + i;
        if (lane == from && lane < kBeamMost) {  // (from is the same in lanes 0 .. 31)
            const bool any = at < count;
            const int token = any ? s_token[lane][at] : -1;
            a.out_scores[o] = any ? (float)best : -INFINITY;
            a.out_parents[o] = any ? lane : -1;
            a.out_tokens[o] = token;
            if (a.out_ended) a.out_ended[o] = !any || s_ended[lane] || token == a.end_token ? 1 : 0;
            ++at;
        }
    }
}

hipError_t launch_beam_select(hipStream_t s, BeamArgs a) {
    const int rows = a.groups * a.beams;
    const bool small = (size_t)rows * a.vocab <= (size_t)512 * 4096;
    const int slice = small ? kBeamSlice : 2 * kBeamSlice;
    a.slices = (a.vocab + slice - 1) / slice;
    const dim3 grid((unsigned)a.slices, (unsigned)rows);
    if (small) hipLaunchKernelGGL(vk_beam_slices<16>, grid, dim3(BM_T), 0, s, a);
    else hipLaunchKernelGGL(vk_beam_slices<32>, grid, dim3(BM_T), 0, s, a);
    hipLaunchKernelGGL(vk_beam_merge, dim3((unsigned)a.groups), dim3(BM_MT), 0, s, a);
    return hipGetLastError();
}

}  // namespace vk
