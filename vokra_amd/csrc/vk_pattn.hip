// vk_pattn.hip — attention over packed sequences of different lengths.
//
// Sequence s has n_s query rows and m_s keys, rows of q, k, v from q_off[s], k_off[s]
// on. Row i of it stands at position p = m_s - n_s + i; query head h reads kv head
// h / G, G = hq / hkv:
//   s_j = scale q . k_j, out = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)
// over the keys j that the row sees: all, or j <= p (causal), or p - window < j <= p. A row
// that sees none gives zeros.
//
// Work: the n_s G query rows of a (sequence, kv head), row R being query R / G of head
// hk G + R % G, in tiles of 128 (hd 64) or 256 (hd 128), 32 a wave, against tiles of 64 keys.
//
// Packing (vk_pattn_pack): every K and V value as two fp16 parts, hi + lo, of the value
// times a power of two that puts its tile's largest at 2^13, in the order in which the
// matrix instructions take their operands: a tile is 64 KB (hd 128) that goes to LDS
// and registers without a shuffle. Three products for one of f32 then hold 22 bits
// whatever the values' size: hi hi + hi lo + lo hi, sums in f32.
//   S^T [keys][rows] = K q^T (q split likewise, a power of two a row);
//   its accumulators are, without leaving the lane, the operand of
//   O^T [d][rows] = V^T W^T, as V's tiles hold keys in the accumulators' order.
// Weights w = 2^(14 + s - M), s in units of log2, M the running maximum of s rounded up:
// a whole number, so what was summed is brought under a new one exactly, and seldom.
// Where a V tile's power of two is below the largest so far the weights take the
// difference, for the product alone.
//
// Even shares: the tiles' units (64 keys each, and two more for a tile's start and
// end) lie on one line, which the workgroups that the chip holds at once (two waves a
// SIMD) share evenly whatever the lengths are; a share holds whole tiles and at most two
// pieces, whose results the last share of a tile to end brings together.
#include <algorithm>

#include "vk_common.h"
#include "vk_pattn.h"

namespace vk {

typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t pa_u4 __attribute__((ext_vector_type(4)));

// A tile's start and end, in units: two documents of 5001 and 8192 rows, 32 heads over 8 of
// 128, 2.11 ms with 2, 2.07 with 3, 2.08 with 4; eight utterances of up to 1500 rows, 20 heads
// of 64, 153 us with 2, 159 with 3
constexpr int pa_cost(int hd) { return hd == 64 ? 2 : 3; }
constexpr float kNoMax = -0x1.fffffep127f;

constexpr int pa_shares(int hd) { return hd == 64 ? 512 : 256; }  // two waves a SIMD
// halves of one tile's K hi (K lo, V hi, V lo): 64 keys
constexpr int pa_part(int hd) { return kPaKeys * hd; }

// ---- sequences ---------------------------------------------------------------------

__device__ __forceinline__ bool pa_wrong(const PaArgs& a, int q0, int q1, int k0, int k1) {
    return q0 < 0 || q1 < q0 || q1 > a.q_rows || q1 - q0 > a.max_q || k0 < 0 || k1 < k0 || k1 > a.k_rows ||
           k1 - k0 > a.max_k;
}

// How many sequences, from the first on, have offsets in order and range; a sequence
// from there on is passed over. All threads of the workgroup, after a barrier; scratch:
// one int of LDS.
__device__ __forceinline__ int pa_in_order(const PaArgs& a, int* s_first) {
    if (threadIdx.x == 0) *s_first = a.n_seq;
    __syncthreads();
    for (int s = threadIdx.x; s < a.n_seq; s += (int)blockDim.x) {
        const int q0 = a.q_off[s], q1 = a.q_off[s + 1], k0 = a.k_off[s], k1 = a.k_off[s + 1];
        if (pa_wrong(a, q0, q1, k0, k1)) atomicMin(s_first, s);
    }
    __syncthreads();
    return *s_first;
}

// A piece of a tile: its units u0 .. u1 - 1.
struct PaPiece {
    int seq, head, slot;    // of the tile
    long long line;         // its place on the line
    int q0, n, k0, m;       // the sequence's rows and keys
    int row0, lo, units;    // the tile's first row, its first tile of keys, its units
    int u0, u1;
};

// Places of tiles: sequence s has those from rows-before / size + s on, which never meet
// the next one's.
template <int ROWS>
__device__ __forceinline__ int pa_q_slot(const PaArgs& a, int q0, int s) {
    return (int)((unsigned)(q0 * a.g) / ROWS) + s;  // q0 g < 2^31
}
__device__ __forceinline__ int pa_k_slot(int k0, int s) { return k0 / kPaKeys + s; }

// The keys that a tile's rows see lie in `units` tiles from `lo` on (one where there are
// none).
template <int ROWS>
__device__ __forceinline__ void pa_span(const PaArgs& a, int n, int m, int row0, int* lo, int* units) {
    const int last = min(row0 + ROWS, n * a.g) - 1;
    int k0 = 0, k1 = m;
    if (a.causal) {
        k1 = min(m, last / a.g + (m - n) + 1);
        if (a.window) k0 = max(0, row0 / a.g + (m - n) - a.window + 1);
    }
    *lo = k1 > k0 ? k0 / kPaKeys : 0;
    *units = k1 > k0 ? (k1 + kPaKeys - 1) / kPaKeys - *lo : 1;
}

// ---- packing -----------------------------------------------------------------------

// 2^e as f32, e within -126 .. 127
__device__ __forceinline__ float pa_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent that puts a largest magnitude a at 2^13 .. 2^14 when values are multiplied by
// 2^-e, which is a normal number (an a below 2^-113 is put lower); kPaNoValue for 0.
__device__ __forceinline__ int pa_exponent(float a) {
    return a == 0.0f ? kPaNoValue : max((int)(__float_as_uint(a) >> 23) - 127 - 13, -127);
}
// 2^-e for e of pa_exponent (1 for none)
__device__ __forceinline__ float pa_factor(int e) { return pa_pow2(e == kPaNoValue ? 0 : -e); }

__device__ __forceinline__ bool pa_finite(float x) { return fabsf(x) < INFINITY; }

// The largest finite magnitude of a lane's values
template <int N>
__device__ __forceinline__ float pa_most(const float (&x)[N][8]) {
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) y = fmaxf(fmaxf(fabsf(x[i][j]), fabsf(x[i][j + 1])), y);  // (passes over NaN)
    if (!(y < INFINITY)) {
        y = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) y = fmaxf(y, pa_finite(x[i][j]) ? fabsf(x[i][j]) : 0.0f);
    }
    return y;
}

// Eight values as two fp16 parts. x - hi as an fma of hi, widened on the way (one
// instruction; minus_one is -1, kept from the compiler, which would make a conversion and a
// subtraction of it): exact.
__device__ __forceinline__ float pa_minus_one() {
    float m = -1.0f;
    asm("" : "+s"(m));
    return m;
}
__device__ __forceinline__ void pa_split(const float (&x)[8], pa_u4& hi, pa_u4& lo, float minus_one) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        pa_h2 h = {(_Float16)x[2 * j], (_Float16)x[2 * j + 1]};
        asm("" : "+v"(h));  // the pair itself is what the fmas read
        const pa_h2 l = {(_Float16)fmaf((float)h.x, minus_one, x[2 * j]), (_Float16)fmaf((float)h.y, minus_one, x[2 * j + 1])};
        hi[j] = __builtin_bit_cast(uint32_t, h);
        lo[j] = __builtin_bit_cast(uint32_t, l);
    }
}

// 64 keys of a kv head, `keys` of them there, from rows kp and vp on, by 256 threads:
// taken into registers (load), then written as a tile in operand order (store), 16 bytes
// a lane and place:
//   K: [half of 32 keys][16 dims][lane]: key lane % 32, dims 8 (lane / 32) ..
//   V: [16 keys][32 dims][lane]: dim lane % 32, keys 4 (lane / 32) + 0 .. 3 and + 8 .. 11
struct PaPackLds {
    float k[4], v[4];
    unsigned long long odd[4];
};
template <int HD>
struct PaPack {
    static constexpr int N = kPaKeys * HD / 8 / 256;  // pieces of 16 bytes a thread, of K and of V
    float x[N][8], y[N][8];

    // Buffer loads: rows behind the last key read as zero, with no branch (strides are at
    // most 2^23, so 64 rows are less than 2^31 bytes).
    __device__ __forceinline__ void load(const float* kp, size_t k_stride, const float* vp, size_t v_stride, int keys) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), h = lane >> 5,
                  l = lane & 31, ks = (int)k_stride * 4, vs = (int)v_stride * 4;
        const auto rk = __builtin_amdgcn_make_buffer_rsrc((void*)kp, 0, (keys - 1) * ks + HD * 4, 0x20000);
        const auto rv = __builtin_amdgcn_make_buffer_rsrc((void*)vp, 0, (keys - 1) * vs + HD * 4, 0x20000);
        const int kl = l * ks + 32 * h, vl = 4 * h * vs + 4 * l;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int f = wave + 4 * i, at = kl + 32 * (f / (HD / 16)) * ks + 64 * (f % (HD / 16));
            const vk_f32x4 u = __builtin_bit_cast(vk_f32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, at, 0, 0));
            const vk_f32x4 w = __builtin_bit_cast(vk_f32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, at + 16, 0, 0));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = u[j];
                x[i][4 + j] = w[j];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int f = wave + 4 * i, at = vl + 16 * (f / (HD / 32)) * vs + 128 * (f % (HD / 32));
#pragma unroll
            for (int j = 0; j < 8; ++j)
                y[i][j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rv, at + ((j & 3) + 8 * (j >> 2)) * vs, 0, 0));
        }
    }

    // out: the tile; the four waves meet once
    __device__ __forceinline__ PaTileMeta store(pa_u4* out, PaPackLds& lds) {
        constexpr int P = pa_part(HD) / 8;  // 16-byte pieces of a part
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
        float ka = pa_most<N>(x), va = pa_most<N>(y);
        unsigned long long odd = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float sum = 0.0f;  // not finite if a value is not (or, harmlessly, at values near f32's end)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += fabsf(y[i][j]);
            if (!pa_finite(sum))
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!pa_finite(y[i][j])) {
                        const int f = wave + 4 * i, key = 16 * (f / (HD / 32)) + 4 * h + (j & 3) + 8 * (j >> 2);
                        odd |= 1ull << key;
                        y[i][j] = 0.0f;
                    }
        }
        ka = vk_group_max<64>(ka);
        va = vk_group_max<64>(va);
        if (__any(odd != 0))
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) odd |= __shfl_xor(odd, o, VK_WAVE);
        if (lane == 0) {
            lds.k[wave] = ka;
            lds.v[wave] = va;
            lds.odd[wave] = odd;
        }
        VK_LDS_BARRIER();
        const int ke = pa_exponent(fmaxf(fmaxf(lds.k[0], lds.k[1]), fmaxf(lds.k[2], lds.k[3])));
        const int ve = pa_exponent(fmaxf(fmaxf(lds.v[0], lds.v[1]), fmaxf(lds.v[2], lds.v[3])));
        const PaTileMeta m = {ke == kPaNoValue ? 0 : ke, ve, (lds.odd[0] | lds.odd[1]) | (lds.odd[2] | lds.odd[3])};
        const float minus_one = pa_minus_one(), kf = pa_factor(ke), vf = pa_factor(ve);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int at = (wave + 4 * i) * 64 + lane;
            pa_u4 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i][j] *= kf;
            pa_split(x[i], hi, lo, minus_one);
            out[at] = hi;
            out[P + at] = lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[i][j] *= vf;
            pa_split(y[i], hi, lo, minus_one);
            out[2 * P + at] = hi;
            out[3 * P + at] = lo;
        }
        return m;
    }
};

// The sequence whose tiles' places `slot` is among, and its rows and keys: the last of those in
// order (see pa_in_order) that begin there or before; false: none. 256 threads, one round of
// memory.
struct PaSeqLds {
    int first, seq, at[4];
};
template <class Slot>
__device__ __forceinline__ bool pa_find(const PaArgs& a, int slot, PaSeqLds& lds, PaPiece& p, Slot begins) {
    constexpr int N = kPaSeqs / 256;
    int q0[N], q1[N], k0[N], k1[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int s = threadIdx.x + 256 * i;
        if (s < a.n_seq) q0[i] = a.q_off[s], q1[i] = a.q_off[s + 1], k0[i] = a.k_off[s], k1[i] = a.k_off[s + 1];
    }
    if (threadIdx.x == 0) {
        lds.first = a.n_seq;
        lds.seq = -1;
    }
    VK_LDS_BARRIER();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int s = threadIdx.x + 256 * i;
        if (s < a.n_seq && pa_wrong(a, q0[i], q1[i], k0[i], k1[i])) atomicMin(&lds.first, s);
    }
    VK_LDS_BARRIER();
    const int n = lds.first;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int s = threadIdx.x + 256 * i;
        if (s < n && begins(q0[i], k0[i], s) <= slot) atomicMax(&lds.seq, s);
    }
    VK_LDS_BARRIER();
    p.seq = __builtin_amdgcn_readfirstlane(lds.seq);
#pragma unroll
    for (int i = 0; i < N; ++i)
        if ((int)threadIdx.x + 256 * i == p.seq) lds.at[0] = q0[i], lds.at[1] = q1[i], lds.at[2] = k0[i], lds.at[3] = k1[i];
    VK_LDS_BARRIER();
    if (p.seq < 0) return false;
    p.q0 = __builtin_amdgcn_readfirstlane(lds.at[0]);
    p.n = __builtin_amdgcn_readfirstlane(lds.at[1]) - p.q0;
    p.k0 = __builtin_amdgcn_readfirstlane(lds.at[2]);
    p.m = __builtin_amdgcn_readfirstlane(lds.at[3]) - p.k0;
    return true;
}

// One workgroup: a tile of 64 keys of one kv head. Bound by memory, which it moves twice:
// 13193 rows of 8 heads of 128 (216 MB read and written) 44 us, 6400 of 20 heads of 64 (131
// MB) 22 us.
template <int HD>
__device__ void pa_pack(const PaArgs& a, int slot, int head) {
    __shared__ PaSeqLds s_seq;
    __shared__ PaPackLds s_lds;
    PaPiece p;
    if (!pa_find(a, slot, s_seq, p, [](int, int k0, int s) { return pa_k_slot(k0, s); })) return;
    const int first = (slot - pa_k_slot(p.k0, p.seq)) * kPaKeys;
    if (first >= p.m) return;
    PaPack<HD> t;
    t.load(a.k + (size_t)(p.k0 + first) * a.k_stride + (size_t)head * HD, a.k_stride,
           a.v + (size_t)(p.k0 + first) * a.v_stride + (size_t)head * HD, a.v_stride, min(kPaKeys, p.m - first));
    const size_t place = (size_t)slot * a.hkv + head;
    const PaTileMeta meta = t.store((pa_u4*)(a.tiles + place * 4 * pa_part(HD)), s_lds);
    if (threadIdx.x == 0) a.meta[place] = meta;
}

// ---- planning ----------------------------------------------------------------------

// One workgroup: the tiles' costs in order, and where each share begins.
template <int HD>
__device__ void pa_plan(const PaArgs& a) {
    __shared__ int s_first, s_q[kPaSeqs + 1], s_k[kPaSeqs + 1];
    __shared__ long long s_wave[4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int n = pa_in_order(a, &s_first);
    for (int s = t; s <= n; s += 256) {
        s_q[s] = n ? a.q_off[s] : 0;
        s_k[s] = n ? a.k_off[s] : 0;
    }
    __syncthreads();
    const int slots = n ? pa_q_slot<pa_tile_rows(HD)>(a, s_q[n], n) : 0;  // beyond the last tile
    auto find = [&](int slot) {  // the last sequence whose places begin at or before it
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pa_q_slot<pa_tile_rows(HD)>(a, s_q[mid], mid) <= slot) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    long long before = 0;
    for (int base = 0; base < slots; base += 256) {
        const int slot = base + t;
        long long cost = 0;
        if (slot < slots) {
            const int s = find(slot), len = s_q[s + 1] - s_q[s];
            const int row0 = (slot - pa_q_slot<pa_tile_rows(HD)>(a, s_q[s], s)) * pa_tile_rows(HD);
            if (row0 < len * a.g) {
                int lo, units;
                pa_span<pa_tile_rows(HD)>(a, len, s_k[s + 1] - s_k[s], row0, &lo, &units);
                cost = units + pa_cost(HD);
            }
        }
        long long x = cost;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long y = __shfl_up(x, o, VK_WAVE);
            if (lane >= o) x += y;
        }
        __syncthreads();
        if (lane == 63) s_wave[wave] = x;
        __syncthreads();
        long long all = 0, mine = before;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < wave) mine += s_wave[w];
            all += s_wave[w];
        }
        if (slot < slots) a.line[slot] = mine + x - cost;
        before += all;
    }
    if (t == 0) a.line[slots] = before;
    const long long total = before * a.hkv;
    // two units at least: of a small call more workgroups (two sequences of up to 714 rows, 2 heads
    // of 128: 39 us, 46 with four; of 800 rows, 16 over 2: 43 and 47)
    const long long shares = total ? min((long long)pa_shares(HD), max(1ll, total / 2)) : 0;
    const long long size = shares ? (total + shares - 1) / shares : 0;
    if (t == 0) {
        a.plan[0] = size;
        a.plan[1] = total;
        a.plan[2] = n;
    }
    __syncthreads();  // line is written (and read by this workgroup alone)
    __threadfence_block();
    for (int i = t; i < pa_shares(HD); i += 256) {
        a.ended[i] = 0;
        const long long x = i * size;
        if (!size || x >= total) continue;
        // the sequence: lines of sequence s begin at hkv line[its first place]
        int lo = 0, hi = n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.line[pa_q_slot<pa_tile_rows(HD)>(a, s_q[mid], mid)] * a.hkv <= x) lo = mid;
            else hi = mid - 1;
        }
        const int s = lo, b = pa_q_slot<pa_tile_rows(HD)>(a, s_q[s], s);
        const int tiles = (int)(((long long)(s_q[s + 1] - s_q[s]) * a.g + pa_tile_rows(HD) - 1) / pa_tile_rows(HD));
        const long long l0 = a.line[b], len = a.line[b + tiles] - l0;  // (empty places behind cost nothing)
        const long long rest = x - l0 * a.hkv;
        const int head = (int)(rest / len);
        const long long in = rest - head * len;
        int tl = 0, th = tiles - 1;
        while (tl < th) {
            const int mid = (tl + th + 1) >> 1;
            if (a.line[b + mid] - l0 <= in) tl = mid;
            else th = mid - 1;
        }
        a.start[i] = PaStart{s, head, b + tl, 0, l0 * a.hkv + head * len + (a.line[b + tl] - l0)};
    }
}

template <int HD>
__global__ __launch_bounds__(256) void vk_pattn_pack(PaArgs a) {
    // planning first: it takes longest
    if (blockIdx.x == 0) {
        if (blockIdx.y == 0) pa_plan<HD>(a);
        return;
    }
    pa_pack<HD>(a, (int)blockIdx.x - 1, blockIdx.y);
}

// ---- products ----------------------------------------------------------------------

// A row's results so far, the same in the lanes l and l + 32 once the halves are summed
struct PaState {
    float m, sum;  // M; sum of w
    int e;         // O is held times 2^-e
};

// A tile's exponents by a scalar load: a vector load's wait would wait for the tiles on
// their way to LDS as well. What packing wrote is in memory since its launch ended.
__device__ __forceinline__ PaTileMeta pa_meta(const PaTileMeta* p) {
    typedef int i4 __attribute__((ext_vector_type(4)));
    const uintptr_t x = (uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x), hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    const i4 y = *(const __attribute__((address_space(4))) i4*)(((uintptr_t)hi << 32) | lo);
    return __builtin_bit_cast(PaTileMeta, y);
}

// Sum or maximum of a row's two lanes
__device__ __forceinline__ float pa_row_max(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float pa_row_sum(float v) {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

// A share's piece of partial results: O in register order [wave][16 bytes' place][lane],
// then (M, sum, e) of each row.
constexpr size_t pa_piece_floats(int hd) { return (size_t)pa_tile_rows(hd) * (hd + 4); }

// Rows of q and out go through LDS, 32 rows of 32 values a wave at a time: the matrix
// instruction wants a row a lane, a load or store of whole lines eight lanes a row. Row r's
// 16-byte piece c lies at r, c ^ (r % 8): neither way meets a bank twice. (Three sequences of
// up to 61 rows, in tiles of 128, 13.4 -> 12.6 us, 16 of up to 400 in tiles 65 -> 61; long ones as before.)
constexpr int kPaTurn = 256;  // pieces a wave
struct PaTurn {
    vk_f32x4* lds;  // the wave's
    int lane_at, row_at, sw;  // pieces of 8 rows a lane, 8 j rows on; of this lane's row
    __device__ __forceinline__ PaTurn(vk_f32x4* of_waves) {
        const int lane = threadIdx.x & 63, l = lane & 31;
        lds = of_waves + (threadIdx.x >> 6) * kPaTurn;
        lane_at = (lane & ~7) + ((lane & 7) ^ (lane >> 3));
        row_at = 8 * l;
        sw = l & 7;
    }
    __device__ __forceinline__ vk_f32x4& line(int j) { return lds[64 * j + lane_at]; }
    __device__ __forceinline__ vk_f32x4& row(int c) { return lds[row_at + (c ^ sw)]; }
    // Between the two: a wave's LDS accesses run in order, so it is the compiler's alone.
    static __device__ __forceinline__ void turn() { asm volatile("" ::: "memory"); }
};

template <int HD>
__device__ __forceinline__ void pa_store_rows(const PaArgs& a, int q0, int head, int rows, int row0,
                                              const vk_f32x16 (&o)[HD / 32], float sum, int e, PaTurn t) {
    const int lane = threadIdx.x & 63, h = lane >> 5, first = row0 + (int)(threadIdx.x >> 6) * 32;
    if (first >= rows) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // (NaN stays)
    float* out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int r = min(first + 8 * j + (lane >> 3), rows - 1), i = r / a.g;
        out[j] = a.out + (size_t)(q0 + i) * a.out_stride + (size_t)(head * a.g + r - i * a.g) * HD + 4 * (lane & 7);
    }
    const int eh = max(min(e, 254), -252) >> 1;
    const float f0 = e == kPaNoValue ? 0.0f : pa_pow2(eh), f1 = e == kPaNoValue ? 0.0f : pa_pow2(max(min(e, 254), -252) - eh);
#pragma unroll
    for (int b = 0; b < HD / 32; ++b) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            vk_f32x4 y;
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = o[b][4 * j + c] * inv * f0 * f1;
            t.row(2 * j + h) = y;
        }
        t.turn();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const vk_f32x4 y = t.line(j);
            if (first + 8 * j + (lane >> 3) < rows) *(vk_f32x4*)(out[j] + 32 * b) = y;
        }
        t.turn();
    }
}

// A sequence's offsets by scalar loads (see pa_meta; the caller wrote them before the
// launch).
__device__ __forceinline__ void pa_lengths(const PaArgs& a, PaPiece& p) {
    typedef __attribute__((address_space(4))) const int* sp;
    const sp q = (sp)(uintptr_t)a.q_off + p.seq, k = (sp)(uintptr_t)a.k_off + p.seq;
    const int q0 = q[0], q1 = q[1], k0 = k[0], k1 = k[1];
    p.q0 = q0;
    p.n = q1 - q0;
    p.k0 = k0;
    p.m = k1 - k0;
}

// The first piece of the share x0 .. x1 - 1 of the line from the tile at (seq, head,
// slot, line) on, whose sequence's lengths are there; false: none. Everything is the same
// for all threads.
template <int HD>
__device__ __forceinline__ bool pa_next(const PaArgs& a, int n_seq, long long x0, long long x1, PaPiece& p) {
    while (p.line < x1) {
        const int rows = p.n * a.g, base = pa_q_slot<pa_tile_rows(HD)>(a, p.q0, p.seq);
        p.row0 = (p.slot - base) * pa_tile_rows(HD);
        if (p.row0 >= rows) {  // the next head, or sequence
            if (rows > 0 && ++p.head < a.hkv) {
                p.slot = base;
                continue;
            }
            p.head = 0;
            if (++p.seq >= n_seq) return false;
            pa_lengths(a, p);
            p.slot = pa_q_slot<pa_tile_rows(HD)>(a, p.q0, p.seq);
            continue;
        }
        pa_span<pa_tile_rows(HD)>(a, p.n, p.m, p.row0, &p.lo, &p.units);
        const long long first = p.line + pa_cost(HD);
        p.u0 = (int)max(min(x0 - first, (long long)p.units), 0ll);
        p.u1 = (int)max(min(x1 - first, (long long)p.units), 0ll);
        if (p.u0 < p.u1) return true;
        p.line += p.units + pa_cost(HD);
        ++p.slot;
    }
    return false;
}

// A wave's 32 rows of a tile: q, as two parts of q 2^-qe in the operand order (dims 16 ks +
// 8 h .. of row l), and where they stand.
template <int HD>
struct PaWave {
    pa_u4 qh[HD / 16], ql[HD / 16];
    int qe, from, to;          // this lane's row, which sees the keys from .. to - 1
    int some_from, some_to;    // keys that a row of the wave sees,
    int all_from, all_to;      // that all of them see

    __device__ __forceinline__ void load(const PaArgs& a, const PaPiece& p, int wave, PaTurn t) {
        constexpr int KS = HD / 16;
        const int lane = threadIdx.x & 63, h = lane >> 5, l = lane & 31, rows = p.n * a.g;
        const int first = p.row0 + wave * 32, r = min(first + l, rows - 1), qi = r / a.g;
        const int off = p.m - p.n, pos0 = first / a.g + off, pos1 = min(first + 31, rows - 1) / a.g + off, pos = qi + off;
        from = some_from = all_from = 0;
        to = some_to = all_to = p.m;
        if (a.causal) {
            to = min(p.m, pos + 1);
            some_to = min(p.m, pos1 + 1);
            all_to = min(p.m, pos0 + 1);
            if (a.window) {
                from = pos - a.window + 1;
                some_from = pos0 - a.window + 1;
                all_from = pos1 - a.window + 1;
            }
        }
        if (first >= rows) some_to = 0;  // no rows
        vk_f32x4 y[HD / 32][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = min(first + 8 * j + (lane >> 3), rows - 1), i = r / a.g;
            const float* qp = a.q + (size_t)(p.q0 + i) * a.q_stride + (size_t)(p.head * a.g + r - i * a.g) * HD + 4 * (lane & 7);
#pragma unroll
            for (int b = 0; b < HD / 32; ++b) y[b][j] = *(const vk_f32x4*)(qp + 32 * b);
        }
        float x[KS][8];
#pragma unroll
        for (int b = 0; b < HD / 32; ++b) {
#pragma unroll
            for (int j = 0; j < 4; ++j) t.line(j) = y[b][j];
            t.turn();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const vk_f32x4 z = t.row(4 * (c >> 1) + 2 * h + (c & 1));
#pragma unroll
                for (int j = 0; j < 4; ++j) x[2 * b + (c >> 1)][4 * (c & 1) + j] = z[j];
            }
            t.turn();
        }
        if (a.sign != 1.0f)
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) x[s][j] *= a.sign;
        float most = 0.0f;  // (a row with a value that is not finite is NaN under any power of two)
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) most = fmaxf(fmaxf(fabsf(x[s][j]), fabsf(x[s][j + 1])), most);
        const int e = pa_exponent(pa_row_max(most));
        const float minus_one = pa_minus_one(), factor = pa_factor(e);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] *= factor;
            pa_split(x[s], qh[s], ql[s], minus_one);
        }
        qe = e == kPaNoValue ? 0 : e;
    }
    // Whether a row of the wave sees a key of the unit that begins at key kk
    __device__ __forceinline__ bool sees(int kk) const { return kk < some_to && kk + kPaKeys > some_from; }
};

// One unit: the wave's rows against the tile in LDS (K hi, K lo, V hi, V lo), whose first
// key is kk, or (NY 1) the half y0 of its keys.
template <int HD, int NY = 2>
__device__ __forceinline__ void pa_unit(const PaArgs& a, const PaPiece& x, const PaWave<HD>& w, const _Float16* tile,
                                        const PaTileMeta& meta, int kk, vk_f32x16 (&o)[HD / 32], PaState& s,
                                        float minus_one, int y0 = 0) {
    constexpr int KS = HD / 16, DB = HD / 32, P = pa_part(HD);
    const int lane = threadIdx.x & 63, h = lane >> 5, ve = meta.v_exp;
    const pa_h8* kh = (const pa_h8*)tile + lane + y0 * (KS * 64);
    const pa_h8* kl = kh + P / 8;
    const pa_h8* vh = (const pa_h8*)tile + lane + 2 * (P / 8) + y0 * (2 * DB * 64);
    const pa_h8* vl = vh + P / 8;
    constexpr vk_f32x16 zero = {};
    vk_f32x16 t[NY];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const pa_h8 qhv = __builtin_bit_cast(pa_h8, w.qh[ks]), qlv = __builtin_bit_cast(pa_h8, w.ql[ks]);
#pragma unroll
        for (int y = 0; y < NY; ++y) {
            const pa_h8 ah = kh[(y * KS + ks) * 64], al = kl[(y * KS + ks) * 64];
            t[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, qhv, ks ? t[y] : zero, 0, 0, 0);
            t[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, qlv, t[y], 0, 0, 0);
            t[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, qhv, t[y], 0, 0, 0);
        }
    }
    const int begin = w.from - kk, end = w.to - kk;  // keys of the unit that the row sees
    // (kept above 0 and below infinity, which would make NaN of -inf and of 0)
    const float c = fminf(fmaxf(__builtin_amdgcn_ldexpf(a.c, w.qe + meta.k_exp), 0x1p-126f), 0x1.fffffep127f);
    if (kk + kPaKeys > w.all_to || kk < w.all_from) {
#pragma unroll
        for (int y = 0; y < NY; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = 32 * (y0 + y) + 8 * (i >> 2) + 4 * h + (i & 3);
                t[y][i] = key < end && key >= begin ? t[y][i] : -INFINITY;
            }
    }
    // (a median with infinity, kept from the compiler, is a maximum that takes the
    // products' results as they come, where fmaxf would first quiet each)
    float inf = INFINITY;
    asm("" : "+s"(inf));
    float most = -INFINITY;
#pragma unroll
    for (int y = 0; y < NY; ++y)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            most = fmaxf(fmaxf(__builtin_amdgcn_fmed3f(t[y][i], t[y][i + 1], inf),
                               __builtin_amdgcn_fmed3f(t[y][i + 2], t[y][i + 3], inf)),
                         most);
    const float top = fmaxf(ceilf(pa_row_max(most) * c), s.m);
    const bool up = ve > s.e;  // the same for all
    if (__any(top > s.m) || up) {
        const float f = __builtin_amdgcn_exp2f(s.m - top);
        const float fo = up ? f * __builtin_amdgcn_ldexpf(1.0f, max(s.e - ve, -200)) : f;
        s.sum *= f;
        s.m = top;
        if (up) s.e = ve;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] *= fo;
    }
    const float sub = s.m - 14.0f;
#pragma unroll
    for (int y = 0; y < NY; ++y) {
#pragma unroll
        for (int i = 0; i < 16; ++i) t[y][i] = __builtin_amdgcn_exp2f(fmaf(t[y][i], c, -sub));
#pragma unroll
        for (int i = 0; i < 16; i += 4) s.sum += (t[y][i] + t[y][i + 1]) + (t[y][i + 2] + t[y][i + 3]);
    }
    if (ve < s.e) {
        const float f = __builtin_amdgcn_ldexpf(1.0f, max(ve - s.e, -200));
#pragma unroll
        for (int y = 0; y < NY; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) t[y][i] *= f;
    }
#pragma unroll
    for (int y = 0; y < 2 * NY; ++y) {
        float z[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = t[y >> 1][8 * (y & 1) + j];
        // (ahead of the other wave of the SIMD, which is at its weights: utterances 157 -> 153 us)
        if (y == 0) __builtin_amdgcn_s_setprio(1);
        pa_u4 wh, wl;
        pa_split(z, wh, wl, minus_one);
        const pa_h8 whv = __builtin_bit_cast(pa_h8, wh), wlv = __builtin_bit_cast(pa_h8, wl);
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            const pa_h8 ah = vh[(y * DB + b) * 64], al = vl[(y * DB + b) * 64];
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, whv, o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, wlv, o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, whv, o[b], 0, 0, 0);
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (meta.odd) {  // values that are not finite go to the rows that see them
        for (unsigned long long rest = meta.odd; rest; rest &= rest - 1) {
            const int key = __ffsll((unsigned long long)rest) - 1;
            const float* vp = a.v + (size_t)(x.k0 + kk + key) * a.v_stride + (size_t)x.head * HD + 4 * h;
            if (key >= end || key < begin || (NY == 1 && key >> 5 != y0)) continue;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 f = *(const float4*)(vp + 32 * b + 8 * j);
                    const float z[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!pa_finite(z[i])) o[b][4 * j + i] += z[i];
                }
        }
    }
}

// Results so far and those of other keys of the same rows: y, and (M, sum, e) in ml.
template <int DB>
__device__ __forceinline__ void pa_add(vk_f32x16 (&o)[DB], PaState& s, const vk_f32x4 (&y)[4 * DB], const vk_f32x4& ml) {
    const float m = fmaxf(s.m, ml[0]);
    const int pe = __float_as_int(ml[2]), e = max(s.e, pe);
    const float f0 = __builtin_amdgcn_exp2f(s.m - m), f1 = __builtin_amdgcn_exp2f(ml[0] - m);
    const float g0 = f0 * __builtin_amdgcn_ldexpf(1.0f, max(s.e - e, -200));
    const float g1 = f1 * __builtin_amdgcn_ldexpf(1.0f, max(pe - e, -200));
    s.sum = s.sum * f0 + ml[1] * f1;
    s.m = m;
    s.e = e;
#pragma unroll
    for (int j = 0; j < DB * 4; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j >> 2][4 * (j & 3) + c] = o[j >> 2][4 * (j & 3) + c] * g0 + y[j][c] * g1;
}

// A piece's results in memory: of this share's pieces, or of another's that has ended, which may
// be on another XCD. Past the caches that are an XCD's own (policy bit 4, sc1, as an access of
// the device's scope carries).
template <int HD>
struct PaParts {
    __amdgpu_buffer_rsrc_t r;
    int at;  // this lane's first 16 bytes of a piece
    __device__ __forceinline__ PaParts(const PaArgs& a)
        : r(__builtin_amdgcn_make_buffer_rsrc((void*)a.part, 0, (int)(2 * pa_shares(HD) * pa_piece_floats(HD) * 4), 0x20000)) {
        at = ((int)(threadIdx.x >> 6) * (HD / 8) * 64 + (int)(threadIdx.x & 63)) * 16;
    }
    __device__ __forceinline__ int state(int piece) const {
        return (int)(piece * pa_piece_floats(HD) * 4) + pa_tile_rows(HD) * HD * 4 +
               ((int)(threadIdx.x >> 6) * 32 + (int)(threadIdx.x & 31)) * 16;
    }
    __device__ __forceinline__ void put(int piece, const vk_f32x16 (&o)[HD / 32], const PaState& s) const {
        const int base = (int)(piece * pa_piece_floats(HD) * 4) + at;
#pragma unroll
        for (int b = 0; b < HD / 32; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const vk_f32x4 y = {o[b][4 * j], o[b][4 * j + 1], o[b][4 * j + 2], o[b][4 * j + 3]};
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(pa_u4, y), r, base + (b * 4 + j) * 1024, 0, 16);
            }
        if ((threadIdx.x & 32) == 0)
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(pa_u4, vk_f32x4{s.m, s.sum, __int_as_float(s.e), 0.0f}), r, state(piece), 0, 16);
    }
    __device__ __forceinline__ void add(int piece, vk_f32x16 (&o)[HD / 32], PaState& s) const {
        const int base = (int)(piece * pa_piece_floats(HD) * 4) + at;
        const vk_f32x4 ml = __builtin_bit_cast(vk_f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, state(piece), 0, 16));
        vk_f32x4 y[HD / 8];
#pragma unroll
        for (int j = 0; j < HD / 8; ++j)
            y[j] = __builtin_bit_cast(vk_f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, base + j * 1024, 0, 16));
        pa_add(o, s, y, ml);
    }
};

// Bound by the matrix instructions and the clock that they leave: two documents of 5001 and
// 8192 rows, causal, 32 heads over 8 of 128, take 2.04 ms (0.37 PFLOP/s at f32 level, 1.1 in
// fp16 products, 88% of what a large library product of fp16 reaches), 16 prompts of up
// to 2048 rows, 16 heads over 2, 315 us (0.92), eight utterances of up to 1500 rows, 20 heads
// of 64, 125 us (0.83). Loads of q ahead of a tile's end and stores that nothing waits for
// changed none of them.
// Tiles go global -> LDS directly, the next one (of the next piece, too) while this one
// is worked on: two buffers, one barrier a unit, between which the two waves of a SIMD
// run as they come, one's products beside the other's weights.
template <int HD>
__global__ __launch_bounds__(pa_tile_rows(HD) * 2) __attribute__((amdgpu_waves_per_eu(2, 2))) void vk_pattn(PaArgs a) {
    constexpr int NW = pa_tile_rows(HD) / 32, DB = HD / 32, P = pa_part(HD);
    constexpr int DMA = 8 * P / 1024 / NW;  // 1 KB loads of a tile a wave
    __shared__ __align__(16) _Float16 s_t[2][4 * P];  // K hi, K lo, V hi, V lo
    __shared__ vk_f32x4 s_turn[NW * kPaTurn];
    const PaTurn turn(s_turn);
    const PaParts<HD> parts(a);
    const int share = vk_xcd_tile(blockIdx.x, gridDim.x);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int h = lane >> 5, l = lane & 31;
    const PaStart st = a.start[share];
    const long long size = a.plan[0], total = a.plan[1];
    const int n_seq = (int)a.plan[2];
    const long long x0 = share * size, x1 = min(x0 + size, total);
    if (x0 >= x1) return;
    PaPiece p;
    p.seq = __builtin_amdgcn_readfirstlane(st.seq);
    p.head = __builtin_amdgcn_readfirstlane(st.head);
    p.slot = __builtin_amdgcn_readfirstlane(st.slot);
    p.line = st.line;
    pa_lengths(a, p);
    const float minus_one = pa_minus_one();
    auto load = [&](const PaPiece& x, int u, int buffer) __attribute__((always_inline)) {
        const size_t tile = (size_t)(pa_k_slot(x.k0, x.seq) + x.lo + u) * a.hkv + x.head;
        const char* g = (const char*)a.tiles + tile * (8 * P) + wave * (DMA * 1024) + lane * 16;
        const uint32_t to = vk_lds_addr(s_t) + buffer * (8 * P) + wave * (DMA * 1024);
#pragma unroll
        for (int i = 0; i < DMA; ++i) vk_dma_b128(g + i * 1024, to + i * 1024);
    };
    if (!pa_next<HD>(a, n_seq, x0, x1, p)) return;
    load(p, p.u0, 0);
    int buffer = 0;
    for (bool more = true; more;) {
        const int rows = p.n * a.g;
        PaWave<HD> w;
        w.load(a, p, wave, turn);
        vk_f32x16 o[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
        PaState s = {kNoMax, 0.0f, kPaNoValue};
        PaPiece next = p;
        for (int u = p.u0; u < p.u1; ++u) {
            const PaTileMeta mt = pa_meta(a.meta + (size_t)(pa_k_slot(p.k0, p.seq) + p.lo + u) * a.hkv + p.head);
            const int kk = (p.lo + u) * kPaKeys;  // its first key
            vk_wait_vm<0>();
            VK_LDS_BARRIER();  // this tile has come, the one before has been read by all
            if (u + 1 < p.u1) {
                load(p, u + 1, buffer ^ 1);
            } else {
                next.line += next.units + pa_cost(HD);
                ++next.slot;
                more = pa_next<HD>(a, n_seq, x0, x1, next);
                if (more) load(next, next.u0, buffer ^ 1);
            }
            if (w.sees(kk)) pa_unit<HD>(a, p, w, s_t[buffer], mt, kk, o, s, minus_one);
            buffer ^= 1;
        }
        s.sum = pa_row_sum(s.sum);
        if (p.u0 == 0 && p.u1 == p.units) {
            pa_store_rows<HD>(a, p.q0, p.head, rows, p.row0, o, s.sum, s.e, turn);
        } else {
            // shares owner .. owner + pieces - 1 have pieces of this tile. The last of them to end
            // joins all, in their order (of two, either order gives the same sums, so the one held
            // here need not pass through memory). All write before any counts itself, nothing
            // spins. (By a launch of its own: prompts 345 us for 335, utterances 151 for 146.)
            const long long first = p.line + pa_cost(HD);
            const int owner = (int)(first / size), pieces = (int)((first + p.units - 1) / size) - owner + 1;
            const bool two = pieces == 2;
            int* const ended = (int*)s_turn;  // (where no row of q or out is now)
            bool last = false;
            if (two) {
                if (threadIdx.x == 0)
                    *ended = __hip_atomic_load(&a.ended[owner], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                VK_LDS_BARRIER();
                last = *ended == 1;
                VK_LDS_BARRIER();
            }
            if (!last) {
                parts.put(2 * share + (p.u0 == 0 ? 1 : 0), o, s);
                vk_wait_vm<0>();
                VK_LDS_BARRIER();
                if (threadIdx.x == 0) *ended = atomicAdd(&a.ended[owner], 1);
                VK_LDS_BARRIER();
                last = *ended == pieces - 1;
                VK_LDS_BARRIER();
            }
            if (last) {
                if (!two) {
#pragma unroll
                    for (int b = 0; b < DB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
                    s = PaState{kNoMax, 0.0f, kPaNoValue};
                }
                for (int i = 0; i < pieces; ++i)
                    if (!two || i != share - owner) parts.add(2 * (owner + i) + (i == 0 ? 1 : 0), o, s);
                pa_store_rows<HD>(a, p.q0, p.head, rows, p.row0, o, s.sum, s.e, turn);
            }
        }
        p = next;
    }
}

// ---- short sequences ----------------------------------------------------------------

// Few units a tile: one launch, a workgroup a tile of 128 or 64 rows, whose threads pack
// each tile of keys into LDS themselves. Nothing is planned, split over workgroups or joined.
// ROWS 128: a wave has 32 rows. 64: two waves have 32, each half of every tile's keys.
// Bound by a wave's own steps, one after the other: loads, packing, products, weights (5.5
// us a tile of 64 keys at head size 128 and 128 rows, 4 at 64).

// Tiles of 64 rows where the chip holds them all at once (16 heads over 2 of 128, one sequence
// of 256: 24.7 us, 28.2 with 128; of 400: 36.6 and 42.9; eleven of 8 heads of up to 300, more
// than that: 51 and 34; 20 heads of 64, four of up to 226: 15.4 and 18.0)
constexpr int short_few(int hd) { return hd == 64 ? 512 : 256; }

template <int HD, int ROWS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 2 : 1, HD == 64 ? 2 : 1))) void vk_pattn_short(PaArgs a) {
    constexpr int DB = HD / 32, RG = ROWS / 32;
    __shared__ __align__(16) _Float16 s_t[4 * pa_part(HD)];
    __shared__ vk_f32x4 s_turn[4 * kPaTurn];
    __shared__ PaSeqLds s_seq;
    __shared__ PaPackLds s_lds;
    const PaTurn turn(s_turn);
    const int slot = blockIdx.x, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), rw = wave % RG, half = wave / RG;
    PaPiece p;
    p.head = blockIdx.y;
    if (!pa_find(a, slot, s_seq, p, [&](int q0, int, int s) { return pa_q_slot<ROWS>(a, q0, s); })) return;
    const int rows = p.n * a.g;
    p.row0 = (slot - pa_q_slot<ROWS>(a, p.q0, p.seq)) * ROWS;
    if (p.row0 >= rows) return;
    pa_span<ROWS>(a, p.n, p.m, p.row0, &p.lo, &p.units);
    const float minus_one = pa_minus_one();
    PaPack<HD> t;
    auto load = [&](int kk) __attribute__((always_inline)) {
        t.load(a.k + (size_t)(p.k0 + kk) * a.k_stride + (size_t)p.head * HD, a.k_stride,
               a.v + (size_t)(p.k0 + kk) * a.v_stride + (size_t)p.head * HD, a.v_stride, min(kPaKeys, p.m - kk));
    };
    int kk = p.lo * kPaKeys;
    const int end = min(p.m, (p.lo + p.units) * kPaKeys);
    if (kk < end) load(kk);
    PaWave<HD> w;
    w.load(a, p, rw, turn);
    vk_f32x16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    PaState s = {kNoMax, 0.0f, kPaNoValue};
    while (kk < end) {
        const PaTileMeta meta = t.store((pa_u4*)s_t, s_lds);  // (once all waves are through with the tile before)
        VK_LDS_BARRIER();
        if (w.sees(kk)) pa_unit<HD, RG / 2>(a, p, w, s_t, meta, kk, o, s, minus_one, half);
        kk += kPaKeys;
        if (kk < end) load(kk);
    }
    if constexpr (RG == 2) {
        VK_LDS_BARRIER();  // all are through with the tile
        vk_f32x4* po = (vk_f32x4*)s_t + rw * (HD / 8) * 64 + lane;
        if (half) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    po[(b * 4 + j) * 64] = vk_f32x4{o[b][4 * j], o[b][4 * j + 1], o[b][4 * j + 2], o[b][4 * j + 3]};
            s_turn[wave * kPaTurn + lane] = vk_f32x4{s.m, s.sum, __int_as_float(s.e), 0.0f};
        }
        VK_LDS_BARRIER();
        if (half) return;
        vk_f32x4 y[DB * 4];
#pragma unroll
        for (int j = 0; j < DB * 4; ++j) y[j] = po[j * 64];
        pa_add(o, s, y, s_turn[(wave + RG) * kPaTurn + lane]);
    }
    pa_store_rows<HD>(a, p.q0, p.head, rows, p.row0, o, pa_row_sum(s.sum), s.e, turn);
}

// ---- few rows ----------------------------------------------------------------------

// Tokens and drafts, or candidates against rows of their own: at most 16 NT query rows of a kv
// head, which see the same keys but for some at the ends. K and V are read once as they
// are, f32, straight into the operands of the f32 matrix instruction (16 x 16 x 4): nothing
// is packed.
//   S^T [16 keys][16 rows]: a lane's 16 bytes of K are one operand of four products
//     (key lane % 16, dims 16 c + 4 (lane / 16) + j; q likewise);
//   its accumulators (keys 4 (lane / 16) + i of row lane % 16) are the operand of
//   O^T [16 dims][16 rows], step i, whose other one are 16 bytes of V row 4 (lane / 16) + i:
//     dims 4 (lane % 16) + j, four products.
// A wave takes 16 keys at a time of its workgroup's range, with an online softmax of its
// own; the four merge through LDS, ranges by vk_pattn_few_join. A step's K goes on its way
// when the products of the step before have taken theirs, V likewise; steps of 16 keys
// leave room for four waves a SIMD (of 64 and 32, with two and three waves: 44 and 39 us).
// Bound by the reads of K and V: five rows each against 16 sequences of 97 to 1500 keys, 20
// heads of 64, 131 MB, take 38 us with the join from memory (3.5 TB/s). Neighbouring
// workgroups are the heads of the same keys, so that whole rows of K and V are on their
// way (ranges of one head: 44 against 41 us), and the reads go through the caches: K and V
// that stay in the last one from step to step take 31 us, 36 past them (from memory 39
// and 38).
constexpr int kFewMost = 2048;  // workgroups that leave partial results
constexpr int kFewRanges = 64;   // of a sequence (32 rows against 8000 keys, 8 heads of 128: 29 us, 43 with 128, 27 with 32;
                                 // one of 100000 keys, 16 heads over 2: 49, 46 and 78)
constexpr int kFewKeys = 16;  // of a wave's step

__device__ __forceinline__ float pa_row4_max(float v) {  // over the lanes l % 16 alike
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    return pa_row_max(v);
}
__device__ __forceinline__ float pa_row4_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return pa_row_sum(__uint_as_float(a[0]) + __uint_as_float(a[1]));
}

// The first key that a row of n, of m keys, sees
__device__ __forceinline__ int pa_few_begin(const PaArgs& a, int n, int m) {
    return a.causal && a.window ? max(0, m - n - a.window + 1) : 0;
}

// what K, V, q and o leave, and the masks of ENDS
constexpr int few_waves(int hd, int nt, bool ends) { return hd * nt == 64 ? 4 : hd * nt == 128 && !ends ? 3 : 2; }

// ENDS: rows of one sequence see different keys (causal, more than one row a sequence). Their
// masks cost a token of 32 heads over 2 of 128 against 2000 keys 42 us for 38.
template <int HD, int NT, bool ENDS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_waves(HD, NT, ENDS)))) void vk_pattn_few(PaArgs a, int per) {
    constexpr int KU = kFewKeys, QC = HD / 16, DD = HD / 64;
    __shared__ int s_first;
    __shared__ float s_m[4][16 * NT], s_l[4][16 * NT];
    __shared__ vk_f32x4 s_o[4][16 * NT][HD / 4];
    const int seq = blockIdx.z, head = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, g = lane >> 4,
              l = lane & 15;
    const int n_ok = pa_in_order(a, &s_first);
    if (seq >= n_ok) return;
    const int q0 = a.q_off[seq], n = a.q_off[seq + 1] - q0, k0 = a.k_off[seq], m = a.k_off[seq + 1] - k0;
    const int rows = n * a.g;
    if (rows == 0 || rows > 16 * NT) return;
    const int begin = pa_few_begin(a, n, m) + (int)blockIdx.y * per, end = min(begin + per, m);
    if (blockIdx.y && begin >= m) return;
    // this lane's rows see the keys from .. to - 1, all rows those of all_from .. all_to - 1
    int from[NT], to[NT];
    const int all_from = a.window ? m - a.window : 0, all_to = m - n + 1;
    vk_f32x4 q[NT][QC];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        const int r = min(16 * x + l, rows - 1), i = r / a.g;
        from[x] = ENDS && a.window ? m - n + i - a.window + 1 : 0;
        to[x] = ENDS ? min(end, m - n + i + 1) : end;
        const float* qp = a.q + (size_t)(q0 + i) * a.q_stride + (size_t)(head * a.g + r - i * a.g) * HD + 4 * g;
#pragma unroll
        for (int c = 0; c < QC; ++c) q[x][c] = *(const vk_f32x4*)(qp + 16 * c) * (a.c * a.sign);
    }
    vk_f32x4 o[NT][DD][4];
    float mx[NT], sum[NT];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        mx[x] = kNoMax;
        sum[x] = 0.0f;
#pragma unroll
        for (int d = 0; d < DD; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[x][d][j] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float* kp = a.k + (size_t)k0 * a.k_stride + (size_t)head * HD + 4 * g;
    const float* vp = a.v + (size_t)k0 * a.v_stride + (size_t)head * HD + 4 * l;
    vk_f32x4 k[QC], v[4][DD];
    auto load_k = [&](int key) __attribute__((always_inline)) {
        const float* p = kp + (size_t)min(key + l, m - 1) * a.k_stride;
#pragma unroll
        for (int x = 0; x < QC; ++x) k[x] = *(const vk_f32x4*)(p + 16 * x);
    };
    auto load_v = [&](int key) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* p = vp + (size_t)min(key + 4 * g + i, m - 1) * a.v_stride;
#pragma unroll
            for (int d = 0; d < DD; ++d) v[i][d] = *(const vk_f32x4*)(p + 64 * d);
        }
    };
    // Where rows see different keys, values of V that are not finite are taken out of the
    // product and added to the rows that see them
    auto few_odd = [&](int key) __attribute__((always_inline)) {
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DD; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!pa_finite(v[i][d][j])) {
                        odd |= 1u << (4 * g + i);
                        v[i][d][j] = 0.0f;
                    }
        if (!__any(odd != 0)) return;
#pragma unroll
        for (int b = 1; b < 64; b <<= 1) odd |= __shfl_xor(odd, b, VK_WAVE);
        for (; odd; odd &= odd - 1) {
            const int at = key + __ffs(odd) - 1;
            if (at >= end) break;
            const float* p = a.v + (size_t)(k0 + at) * a.v_stride + (size_t)head * HD + 16 * g;
#pragma unroll
            for (int d = 0; d < DD; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const vk_f32x4 f = *(const vk_f32x4*)(p + 64 * d + 4 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int x = 0; x < NT; ++x)
                            if (!pa_finite(f[j]) && at >= from[x] && at < to[x]) o[x][d][j][i] += f[j];
                }
        }
    };
    int key = begin + wave * KU;
    if (key < end) {
        load_k(key);
        load_v(key);
    }
    for (; key < end; key += 4 * KU) {
        const int next = key + 4 * KU;
        vk_f32x4 s[NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) s[x] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int y = 0; y < QC; ++y)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < NT; ++x)
                    s[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[y][j], q[x][y][j], s[x], 0, 0, 0);
        if (next < end) load_k(next);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float y = s[x][i];
                y = y > -INFINITY ? y : __builtin_nanf("");  // of a key that is not finite
                const int at = key + 4 * g + i;
                y = (!ENDS || at >= from[x]) && at < to[x] ? y : -INFINITY;
                s[x][i] = y;
                most = fmaxf(most, y);
            }
            const float top = fmaxf(pa_row4_max(most), mx[x]);
            const float f = __builtin_amdgcn_exp2f(mx[x] - top);
            mx[x] = top;
            float add = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[x][i] = __builtin_amdgcn_exp2f(s[x][i] - top);
                add += s[x][i];
            }
            sum[x] = sum[x] * f + add;
#pragma unroll
            for (int d = 0; d < DD; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[x][d][j] *= f;
        }
        if (ENDS && (key < all_from || key + KU > all_to)) few_odd(key);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < DD; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int x = 0; x < NT; ++x)
                        o[x][d][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][d][j], s[x][i], o[x][d][j], 0, 0, 0);
        if (next < end) load_v(next);
    }
    // o[x][d][j][i]: row 16 x + l, dim 64 d + 4 (4 g + i) + j
#pragma unroll
    for (int x = 0; x < NT; ++x) {
        const float all = pa_row4_sum(sum[x]);
        if (g == 0) {
            s_m[wave][16 * x + l] = mx[x];
            s_l[wave][16 * x + l] = all;
        }
#pragma unroll
        for (int d = 0; d < DD; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                s_o[wave][16 * x + l][16 * d + 4 * g + i] =
                    vk_f32x4{o[x][d][0][i], o[x][d][1][i], o[x][d][2][i], o[x][d][3][i]};
    }
    __syncthreads();
    const int ranges = max(1, (m - pa_few_begin(a, n, m) + per - 1) / per);
    float* part = a.part + (((size_t)seq * a.hkv + head) * gridDim.y + blockIdx.y) * (16 * NT) * (HD + 4);
    for (int y = t; y < rows * (HD / 4); y += 256) {
        const int r = y / (HD / 4), d = y % (HD / 4);
        float top = s_m[0][r];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
        vk_f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][r] - top);
            all += s_l[w][r] * f;
            z += s_o[w][r][d] * f;
        }
        if (ranges == 1) {
            const int i = r / a.g;
            const float inv = all == 0.0f ? 0.0f : 1.0f / all;
            *(vk_f32x4*)(a.out + (size_t)(q0 + i) * a.out_stride + (size_t)(head * a.g + r - i * a.g) * HD + 4 * d) = z * inv;
        } else {
            *(vk_f32x4*)(part + (size_t)r * (HD + 4) + 4 * d) = z;
            if (d == 0) *(float2*)(part + (size_t)r * (HD + 4) + HD) = make_float2(top, all);
        }
    }
}

// A sequence's ranges of a kv head brought together: a workgroup has 64 pieces of four
// values, its waves every fourth range, eight on their way at once. (16 rows against 8000
// keys, 8 heads of 128, 24 us in all; one workgroup a sequence and kv head, all ranges in
// turn, 99.)
template <int HD, int NT>
__global__ __launch_bounds__(256) void vk_pattn_few_join(PaArgs a, int per, int splits) {
    __shared__ int s_first;
    __shared__ float2 s_ml[4][64];
    __shared__ vk_f32x4 s_o[4][64];
    const int seq = blockIdx.z, head = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n_ok = pa_in_order(a, &s_first);
    if (seq >= n_ok) return;
    const int q0 = a.q_off[seq], n = a.q_off[seq + 1] - q0, m = a.k_off[seq + 1] - a.k_off[seq], rows = n * a.g;
    const int ranges = (m - pa_few_begin(a, n, m) + per - 1) / per, y = (int)blockIdx.x * 64 + lane;
    if (ranges < 2 || rows > 16 * NT || (int)blockIdx.x * 64 >= rows * (HD / 4)) return;
    const int r = min(y / (HD / 4), rows - 1), d = y % (HD / 4);
    const float* p = a.part + ((size_t)seq * a.hkv + head) * splits * (16 * NT) * (HD + 4) + (size_t)r * (HD + 4);
    float top = kNoMax, all = 0.0f;
    vk_f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = wave; s0 < ranges; s0 += 32) {
        float2 ml[8];
        vk_f32x4 w[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const float* x = p + (size_t)min(s0 + 4 * s, ranges - 1) * (16 * NT) * (HD + 4);
            ml[s] = *(const float2*)(x + HD);
            w[s] = *(const vk_f32x4*)(x + 4 * d);
        }
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            if (s0 + 4 * s >= ranges) break;
            const float now = fmaxf(top, ml[s].x);
            const float f = __builtin_amdgcn_exp2f(top - now), h = __builtin_amdgcn_exp2f(ml[s].x - now);
            top = now;
            all = all * f + ml[s].y * h;
            z = z * f + w[s] * h;
        }
    }
    s_ml[wave][lane] = make_float2(top, all);
    s_o[wave][lane] = z;
    __syncthreads();
    if (wave != 0 || y >= rows * (HD / 4)) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, s_ml[w][lane].x);
    all = 0.0f;
    z = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_ml[w][lane].x - top);
        all += s_ml[w][lane].y * f;
        z += s_o[w][lane] * f;
    }
    const int i = r / a.g;
    const float inv = all == 0.0f ? 0.0f : 1.0f / all;
    *(vk_f32x4*)(a.out + (size_t)(q0 + i) * a.out_stride + (size_t)(head * a.g + r - i * a.g) * HD + 4 * d) = z * inv;
}

template <int HD, int NT, bool ENDS>
static hipError_t go_few_as(hipStream_t s, const PaArgs& a) {
    // ranges of a step of all four waves at least, up to kFewRanges of them a sequence and
    // kFewMost in all if all sequences were the longest
    constexpr int step = 4 * kFewKeys;
    const long long pairs = (long long)a.n_seq * a.hkv;
    const int keys = a.causal && a.window ? std::min(a.max_k, a.window + a.max_q - 1) : a.max_k;
    const long long most = std::max<long long>(1, std::min<long long>(kFewRanges, kFewMost / pairs));
    const int per = (int)std::max<long long>(step, ((keys + most - 1) / most + step - 1) / step * step);
    const int splits = keys ? (keys + per - 1) / per : 1;
    const dim3 grid((unsigned)a.hkv, (unsigned)splits, (unsigned)a.n_seq);
    hipLaunchKernelGGL((vk_pattn_few<HD, NT, ENDS>), grid, dim3(256), 0, s, a, per);
    if (splits > 1) {
        const dim3 join((unsigned)(a.max_q * a.g * (HD / 4) + 63) / 64, (unsigned)a.hkv, (unsigned)a.n_seq);
        hipLaunchKernelGGL((vk_pattn_few_join<HD, NT>), join, dim3(256), 0, s, a, per, splits);
    }
    return hipGetLastError();
}

template <int HD, int NT>
static hipError_t go_few(hipStream_t s, const PaArgs& a) {
    return a.causal && a.max_q > 1 ? go_few_as<HD, NT, true>(s, a) : go_few_as<HD, NT, false>(s, a);
}

// ---- launchers ---------------------------------------------------------------------

size_t pattn_part_floats(int hd) { return 2 * (size_t)pa_shares(hd) * pa_piece_floats(hd); }

template <int HD>
static hipError_t go_pattn(hipStream_t s, const PaArgs& a) {
    hipLaunchKernelGGL(vk_pattn_pack<HD>, dim3((unsigned)a.k_slots + 1, (unsigned)a.hkv), dim3(256), 0, s, a);
    hipLaunchKernelGGL(vk_pattn<HD>, dim3(pa_shares(HD)), dim3(2 * pa_tile_rows(HD)), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_pattn(hipStream_t s, int hd, const PaArgs& a) {
    // few rows: each key is read by few products, packing it would move three times its bytes (16
    // sequences of 1000 keys, 20 heads of 64, of 5 rows: 33 us, 104 packed; of 32: 49 and 105; of
    // 2000 keys and four causal rows: 69 and 209; 32 rows of 8 heads of 128 against 8000 keys: 29
    // and 90; against 32 keys, in one launch either way: 10 and 12)
    const long long rows = (long long)a.max_q * a.g;
    if (rows <= kPaFewRows) {
        if (hd == 64) return rows <= 16 ? go_few<64, 1>(s, a) : go_few<64, 2>(s, a);
        return rows <= 16 ? go_few<128, 1>(s, a) : go_few<128, 2>(s, a);
    }
    // short sequences, by one launch: at head size 64 up to 512 keys (16 of 512 keys, 20 heads:
    // 82 us, 96 packed; 16 heads over 2: 67 and 61; three of up to 61: 8 and 17), at 128, where
    // a workgroup has a CU to itself, up to 448 keys (four of up to 400, 8 heads: 42 and 46, 16
    // over 2: 47 and 50; of 512: 55 and 49) and two rounds of workgroups (16 of up to 400, 16
    // over 2: 88 and 61); three of up to 61: 12 and 21
    auto tiles = [&](int rows) { return ((long long)a.q_rows * a.g / rows + a.n_seq) * a.hkv; };
    // and long ones of which a tile's rows see up to 320 (20 heads of 64, four of up to 1500, a
    // window of 100: 47 and 60, of 400: 80 and 76; 8 heads of 128, one of 1000, of 128: 29 and 45)
    const int most = a.causal && a.window && a.window + 128 / a.g <= 320 ? 320 : a.max_k;
    if (hd == 64 ? most <= 512 : most <= 448 && tiles(128) <= 512) {
        const bool few = tiles(64) <= short_few(hd);
        const dim3 grid((unsigned)(tiles(few ? 64 : 128) / a.hkv), (unsigned)a.hkv);
        if (hd == 64 && few) hipLaunchKernelGGL((vk_pattn_short<64, 64>), grid, dim3(256), 0, s, a);
        else if (hd == 64) hipLaunchKernelGGL((vk_pattn_short<64, 128>), grid, dim3(256), 0, s, a);
        else if (few) hipLaunchKernelGGL((vk_pattn_short<128, 64>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((vk_pattn_short<128, 128>), grid, dim3(256), 0, s, a);
        return hipGetLastError();
    }
    return hd == 64 ? go_pattn<64>(s, a) : go_pattn<128>(s, a);
}

}  // namespace vk
