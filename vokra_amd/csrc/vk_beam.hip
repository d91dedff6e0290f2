// vk_beam.hip — beam search's selection: the n best continuations of a group's beams.
//
// A live beam's continuation by token v is worth
//   total = score + (x_v - ln sum_w e^(x_w)),
// an ended beam has one, its end token at its own score. A group's n_out best go out,
// the larger total first; of equal totals the lower beam, in one beam the larger logit
// and then the lower token.
//
// Bound by reading the logits once, and by two launches: 256 rows of 128259 columns (131
// MB), 16 continuations, take 32 us for the slices (4.1 TB/s) and 12 for the merge, 320 of
// 51866, five, 17 and 6; five rows of 51865, ten, 7 and 7, which is dependent rounds of
// memory, LDS and lane permutations.
//
// Two launches. Slices: a workgroup reads up to 4096 or 8192 columns of a row once, into
// registers, and leaves their maximum, the sum of their exponentials and their n_out best
// columns. Merge: a workgroup a group joins the slices' sums (in 64 bits: totals of
// different beams are compared, and near ones have to fall in order), takes each
// beam's best from its slices' lists and the group's from its beams'.
//
// The best of a slice without a sort of it: the threads fall into at least n_out groups,
// and the least of the groups' maxima bounds the n_out-th largest column from below; a few
// times as many columns as there are groups reach it. They are put into LDS and ranked by
// counting. Where too many do (ties), they are taken one after the other.
//
// A logit that is NaN counts as -inf; a row with +inf has no continuations (its
// log-softmax has no value). Sums do not depend on where a row lies in memory, so
// equal rows have equal totals.
#include "vk_beam.h"
#include "vk_common.h"

namespace vk {

constexpr int BM_T = 256;     // threads of a slice
constexpr int BM_CAND = 512;  // candidates that are ranked at once
constexpr int BM_MT = 512;    // threads of a merge: eight waves, a beam each in turn
constexpr int BM_LIST = 1024; // entries of a beam's lists that a wave holds in LDS
constexpr int BM_FEW = 64;    // entries of a group that are all ranked

// Values in the order of their bits, a column index that falls with it behind: the larger
// key is the better column. Key 0: none.
__device__ __forceinline__ unsigned long long bm_key(float x, int column) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // one zero
    const uint32_t ord = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((unsigned long long)ord << 32) | (0xffffffffu - (uint32_t)column);
}
__device__ __forceinline__ float bm_value(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int bm_column(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

// The largest of the wave's keys, in every lane: partners by lane permutations in the VALU
// (see vk_bfly_partner; the last two steps swap rows and halves), 6 steps of some 30 cycles
// where ds_bpermute's take 150.
template <int O>
__device__ __forceinline__ void bm_partners(unsigned long long k, unsigned long long& x, unsigned long long& y) {
    const uint32_t lo = (uint32_t)k, hi = (uint32_t)(k >> 32);
    x = k;
    if constexpr (O < 16) {
        y = ((unsigned long long)(uint32_t)vk_bfly_partner<O>((int)hi) << 32) | (uint32_t)vk_bfly_partner<O>((int)lo);
    } else if constexpr (O == 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
        const auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
        x = ((unsigned long long)b[0] << 32) | a[0];
        y = ((unsigned long long)b[1] << 32) | a[1];
    } else {
        const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
        x = ((unsigned long long)b[0] << 32) | a[0];
        y = ((unsigned long long)b[1] << 32) | a[1];
    }
}
template <int O>
__device__ __forceinline__ unsigned long long bm_max_step(unsigned long long k) {
    unsigned long long x, y;
    bm_partners<O>(k, x, y);
    return y > x ? y : x;
}
__device__ __forceinline__ unsigned long long bm_wave_max(unsigned long long k) {
    k = bm_max_step<1>(k);
    k = bm_max_step<2>(k);
    k = bm_max_step<4>(k);
    k = bm_max_step<8>(k);
    k = bm_max_step<16>(k);
    return bm_max_step<32>(k);
}

// The sum over the wave likewise, in a fixed order
template <int O>
__device__ __forceinline__ double bm_sum_step(double v) {
    unsigned long long x, y;
    bm_partners<O>((unsigned long long)__double_as_longlong(v), x, y);
    return __longlong_as_double((long long)x) + __longlong_as_double((long long)y);
}
__device__ __forceinline__ double bm_wave_sum(double v) {
    v = bm_sum_step<1>(v);
    v = bm_sum_step<2>(v);
    v = bm_sum_step<4>(v);
    v = bm_sum_step<8>(v);
    v = bm_sum_step<16>(v);
    return bm_sum_step<32>(v);
}

// Doubles in the order of their bits, above 0 (0: none)
__device__ __forceinline__ unsigned long long bm_order(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// One step of the least of the groups' maxima: maxima within a group of `lanes`, least beyond
template <int O>
__device__ __forceinline__ float bm_bound_step(float v, int lanes) {
    const float w = __int_as_float(vk_bfly_partner<O>(__float_as_int(v)));
    return O < lanes ? fmaxf(v, w) : fminf(v, w);
}

// x, -inf for NaN (a maximum passes over NaN)
__device__ __forceinline__ float bm_number(float x) { return fmaxf(x, -INFINITY); }

// A row that goes on: not ended, with a score above -inf.
__device__ __forceinline__ bool bm_live(const BeamArgs& a, int row) {
    return !(a.ended && a.ended[row]) && a.scores[row] > -INFINITY;
}

typedef float bm_f4 __attribute__((ext_vector_type(4), aligned(4)));

// E columns a thread, in runs of four
template <int E>
__global__ __launch_bounds__(BM_T) void vk_beam_slices(BeamArgs a) {
    __shared__ float s_max[4], s_bound[4];
    __shared__ double s_sum[4];
    __shared__ unsigned long long s_key[BM_CAND];
    __shared__ int s_n;
    const int row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (!bm_live(a, row)) return;
    const float* x = a.logits + (size_t)row * a.stride;
    const int c0 = (int)blockIdx.x * a.width, c1 = min(c0 + a.width, a.vocab);
    float y[E];
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
        const int c = c0 + 4 * (t + BM_T * j);
        if (c + 3 < c1) {
            const bm_f4 v = *(const bm_f4*)(x + c);
            y[4 * j] = v.x, y[4 * j + 1] = v.y, y[4 * j + 2] = v.z, y[4 * j + 3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) y[4 * j + i] = c + i < c1 ? x[c + i] : -INFINITY;
        }
    }
    if (t == 0) s_n = 0;
    float most = -INFINITY, four[E / 4];  // and of each run of four
#pragma unroll
    for (int j = 0; j < E / 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[4 * j + i] = bm_number(y[4 * j + i]);
        four[j] = fmaxf(fmaxf(y[4 * j], y[4 * j + 1]), fmaxf(y[4 * j + 2], y[4 * j + 3]));
        most = fmaxf(most, four[j]);
    }
    float v = bm_bound_step<1>(most, a.group);
    v = bm_bound_step<2>(v, a.group);
    v = bm_bound_step<4>(v, a.group);
    v = bm_bound_step<8>(v, a.group);
    v = bm_bound_step<16>(v, a.group);
    v = bm_bound_step<32>(v, a.group);
    const float top = vk_group_maxf<64>(most);
    if (lane == 0) {
        s_max[wave] = top;
        s_bound[wave] = v;
    }
    __syncthreads();
    const float m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    const float bound = fminf(fminf(s_bound[0], s_bound[1]), fminf(s_bound[2], s_bound[3]));
    // e^(x - m) = 2^(x l - m l), l = log2 e: one fma and one exponential a column. m l is rounded,
    // by r, the same for all: the sum is multiplied by 2^-r at the end
    constexpr float l = 1.44269504088896340736f;
    const bool near = fabsf(m) < 16384.0f;
    const float ml = near ? m * l : 0.0f, r = near ? fmaf(m, l, -ml) : 0.0f;
    float sum = 0.0f;
    if (near) {
#pragma unroll
        for (int j = 0; j < E; ++j) sum += __builtin_amdgcn_exp2f(fmaf(y[j], l, -ml));
    } else if (m > -INFINITY) {
#pragma unroll
        for (int j = 0; j < E; ++j) sum += __builtin_amdgcn_exp2f((y[j] - m) * l);
    }
    const double total = bm_wave_sum((double)sum);
    if (lane == 0) s_sum[wave] = total;
    const float from = fmaxf(bound, -0x1.fffffep127f);  // (what is -inf is none)
    if (__any(most >= from))
#pragma unroll
        for (int j = 0; j < E / 4; ++j)
            if (four[j] >= from)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (y[4 * j + i] >= from) {
                        const int at = atomicAdd(&s_n, 1);
                        if (at < BM_CAND) s_key[at] = bm_key(y[4 * j + i], c0 + 4 * (t + BM_T * j) + i);
                    }
    __syncthreads();
    const size_t part = (size_t)row * a.slices + blockIdx.x;
    unsigned long long* out = a.keys + part * a.n_out;
    int count = s_n;
    if (count <= BM_CAND) {
        for (int i = t; i < count; i += BM_T) {
            const unsigned long long k = s_key[i];
            int before = 0;
#pragma unroll 8
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
    if (t == 0) {
        const double x = -0.69314718055994530942 * (double)r;  // below 2^-9: three terms are 2^-40
        const double all = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        a.stats[part] = BeamStat{all * (1.0 + x * (1.0 + x * (0.5 + x * 0.16666666666666667))), m, count};
    }
}

// The n_out best of a beam's slices, by a wave: lists fall, so a lane looks at the head
// of its slices' lists (s, s + 64, ..) and the wave takes the best head, n_out times. The
// beams' own lists fall too: the first wave takes the group's best from their heads likewise.
__global__ __launch_bounds__(BM_MT) void vk_beam_merge(BeamArgs a) {
    constexpr int WAVES = BM_MT / 64;
    __shared__ unsigned long long s_list[WAVES][BM_LIST];
    __shared__ unsigned long long s_some[WAVES][128], s_best[WAVES][64], s_order[BM_MT];
    __shared__ double s_total[kBeamMost][kBeamOut];
    __shared__ int s_rank[BM_MT], s_place[BM_MT], s_found, s_token[kBeamMost][kBeamOut], s_count[kBeamMost], s_ended[kBeamMost];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.n_out;
    if (threadIdx.x == 0) s_found = 0;
    for (int b = wave; b < a.beams; b += WAVES) {
        const int row = g * a.beams + b;
        const BeamStat* st = a.stats + (size_t)row * a.slices;
        const unsigned long long* keys = a.keys + (size_t)row * a.slices * n;
        // all that the beam may need, on its way at once (of a beam that has ended it is not read)
        BeamStat first = {0.0, -INFINITY, 0};
        if (lane < a.slices) first = st[lane];
        const bool staged = a.slices * n <= BM_LIST;
        if (staged)
            for (int i = lane; i < a.slices * n; i += 64) s_list[wave][i] = keys[i];
        const float score = a.scores[row];
        const bool ended = a.ended && a.ended[row], live = !ended && score > -INFINITY;
        if (lane == 0) s_ended[b] = ended;
        if (!live) {
            if (lane == 0) {
                s_count[b] = ended && score > -INFINITY ? 1 : 0;
                s_total[b][0] = (double)score;
                s_token[b][0] = a.end_token;
            }
            continue;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own list: no barrier
        auto key = [&](int s, int i) { return staged ? s_list[wave][s * n + i] : keys[(size_t)s * n + i]; };
        float m = first.max;
        for (int s = lane + 64; s < a.slices; s += 64) m = fmaxf(m, st[s].max);
        m = vk_group_maxf<64>(m);
        // e^(max - m) in f32, as the slices' exponentials (in 64 bits 0.7 us more, by its instructions alone)
        auto under = [m](float max) { return (double)__builtin_amdgcn_exp2f((max - m) * 1.44269504088896340736f); };
        double sum = first.max > -INFINITY ? first.sum * under(first.max) : 0.0;
        for (int s = lane + 64; s < a.slices; s += 64)
            if (st[s].max > -INFINITY) sum += st[s].sum * under(st[s].max);
        sum = bm_wave_sum(sum);
        const double lse = (double)m + log(sum);
        int taken = 0;
        unsigned long long got = 0;  // lane i: the i-th best
        bool few = false;
        if (staged && a.slices <= 64) {
            // the c-th entries of all lists, c n_out / slices: at least n_out entries reach the least of
            // them, and seldom more than 128: each of those is ranked by counting
            const int c = (n + a.slices - 1) / a.slices - 1;
            unsigned long long bound = lane < a.slices ? (c < first.count ? s_list[wave][lane * n + c] : 0) : ~0ull;
            bound = ~bm_wave_max(~bound);
            int found = 0;
            for (int i = lane; i < (a.slices * n + 63) / 64 * 64; i += 64) {
                const int s = i / n;
                const unsigned long long k =
                    i < a.slices * n && i - s * n < __shfl(first.count, s & 63, VK_WAVE) ? s_list[wave][i] : 0;
                const uint64_t m1 = __ballot(k && k >= bound);
                const int at = found + __popcll(m1 & ((1ull << lane) - 1));
                if (k && k >= bound && at < 128) s_some[wave][at] = k;
                found += __popcll(m1);
            }
            few = found <= 128;
            if (few) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                const unsigned long long k0 = lane < found ? s_some[wave][lane] : 0,
                                         k1 = lane + 64 < found ? s_some[wave][lane + 64] : 0;
                int b0 = 0, b1 = 0;
#pragma unroll 8
                for (int i = 0; i < found; ++i) {
                    const unsigned long long y = s_some[wave][i];
                    b0 += (int)(y > k0);
                    b1 += (int)(y > k1);
                }
                taken = min(found, n);
                if (k0 && b0 < n) s_best[wave][b0] = k0;
                if (k1 && b1 < n) s_best[wave][b1] = k1;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                got = lane < taken ? s_best[wave][lane] : 0;
            }
        }
        // else the best key of a lane's slices that is not taken yet, again and again
        int place = 0;
        unsigned long long last = ~0ull, mine = 0;
        auto next = [&]() {
            mine = 0;
            if (a.slices <= 64) {  // one list a lane
                if (place < first.count) mine = key(lane, place++);
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
        if (!few) next();
        while (!few && taken < n) {
            const unsigned long long k = bm_wave_max(mine);
            if (!k) break;
            if (lane == taken) got = k;
            last = k;
            if (mine == k) next();
            ++taken;
        }
        const double total = (double)score + ((double)bm_value(got) - lse);
        const bool there = lane < taken && total > -INFINITY;  // NaN: the row holds +inf
        if (there) {
            s_total[b][lane] = total;
            s_token[b][lane] = bm_column(got);
        }
        if (lane == 0) s_count[b] = there ? taken : 0;
    }
    __syncthreads();
    auto put = [&](int i, int b, int at, bool any) {
        const size_t o = (size_t)g * n + i;
        const int token = any ? s_token[b][at] : -1;
        a.out_scores[o] = any ? (float)s_total[b][at] : -INFINITY;
        a.out_parents[o] = any ? b : -1;
        a.out_tokens[o] = token;
        if (a.out_ended) a.out_ended[o] = !any || s_ended[b] || token == a.end_token ? 1 : 0;
    };
    if (a.beams * n <= BM_MT) {
        // ranked by counting, of equal totals the lower place first; as many threads an entry as
        // there are, a share of the others each. Of many entries those alone that reach the least
        // of the c-th ones of the F lists that are full, F c n_out or more: at least n_out
        // (twelve beams, 24 continuations: 20 -> 11.5 us; few entries are ranked sooner than
        // bounded, five of five 6.6 and 7.9)
        const int t = threadIdx.x, entries = a.beams * n;
        int found = entries;
        if (entries > BM_FEW) {
            const int count = lane < a.beams ? s_count[lane] : 0, full = __popcll(__ballot(count == n));
            const int c = full ? (n + full - 1) / full - 1 : 0;
            const unsigned long long bound = full ? ~bm_wave_max(count == n ? ~bm_order(s_total[lane][c]) : 0) : 0;
            const int b = t / n, at = t - b * n;
            const unsigned long long own = t < entries && at < s_count[b] ? bm_order(s_total[b][at]) : 0;
            if (own && own >= bound) {
                const int i = atomicAdd(&s_found, 1);
                s_order[i] = own;
                s_place[i] = t;
                s_rank[i] = 0;
            }
            __syncthreads();
            found = s_found;
        } else {
            if (t < entries) {
                const int b = t / n, at = t - b * n;
                s_order[t] = at < s_count[b] ? bm_order(s_total[b][at]) : 0;
                s_place[t] = t;
                s_rank[t] = 0;
            }
            __syncthreads();
        }
        const int parts = found ? BM_MT / found : 0, e = found ? t % found : 0, part = found ? t / found : 0;
        const unsigned long long mine = found ? s_order[e] : 0;
        const int place = found ? s_place[e] : 0;
        int before = 0;
        if (part < parts)
#pragma unroll 4
            for (int i = part; i < found; i += parts) {
                const unsigned long long y = s_order[i];
                before += (int)(y > mine) + (int)((y == mine) & (s_place[i] < place));
            }
        if (before) atomicAdd(&s_rank[e], before);
        __syncthreads();
        // (entries that are none come last, in the order of their places)
        if (t < found && s_rank[t] < n) put(s_rank[t], place / n, place % n, mine != 0);
        if (t >= found && t < n) put(t, 0, 0, false);
        return;
    }
    if (wave != 0) return;
    const int count = lane < a.beams ? s_count[lane] : 0;
    int at = 0;
    double total = count ? s_total[lane][0] : 0.0;
    for (int i = 0; i < n; ++i) {
        const unsigned long long mine = at < count ? bm_order(total) : 0, best = bm_wave_max(mine);
        const int from = __ffsll((unsigned long long)__ballot(mine == best)) - 1;  // the lowest beam
        if (lane == from) {
            put(i, lane, at, at < count);
            if (++at < count) total = s_total[lane][at];
        }
    }
}

hipError_t launch_beam_select(hipStream_t s, BeamArgs a) {
    const int rows = a.groups * a.beams;
    // up to 16 lists a beam, smaller slices end earlier (16 groups of four beams of 8192 tokens:
    // 11.1 us against 12.5; 64 of five of 51866: 23.8 against 24.3); above that, half the
    // lists to merge (one group of eight of 128259: 14.1 against 15.0, eight: 17.4 against 19.9)
    const bool small = a.vocab <= 16 * kBeamSlice;
    const int slice = small ? kBeamSlice : 2 * kBeamSlice;
    a.slices = (a.vocab + slice - 1) / slice;
    // slices of one width: all threads of each have columns (with a narrow last one its empty
    // threads bound nothing, and all of its columns are ranked: four beams of 12749 tokens 21 -> 11 us)
    a.width = ((a.vocab + a.slices - 1) / a.slices + 3) / 4 * 4;
    int groups = 4;  // of threads of a slice
    while (groups < a.n_out) groups *= 2;
    a.group = BM_T / groups;
    const dim3 grid((unsigned)a.slices, (unsigned)rows);
    if (small) hipLaunchKernelGGL(vk_beam_slices<16>, grid, dim3(BM_T), 0, s, a);
    else hipLaunchKernelGGL(vk_beam_slices<32>, grid, dim3(BM_T), 0, s, a);
    hipLaunchKernelGGL(vk_beam_merge, dim3((unsigned)a.groups), dim3(BM_MT), 0, s, a);
    return hipGetLastError();
}

}  // namespace vk
