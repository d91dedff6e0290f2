// vk_bkv_attn.hip — attention of a step's rows over the block-scaled KV cache.
//
// Row r of the step belongs to item i, at position p = start_i + (r - row0_i);
// query head h reads kv head h / G, G = hq / n_head:
//   s_j = scale q . k_j (j <= p), out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// with k, v the values that the cache holds: 8-bit ones under their block's
// scale, f32 rows in the open block.
//
// Columns: the count_i * G query rows of an item that read one kv head.
// vk_bkv_attn takes 16 or 32 of them over a range of keys; its four waves take
// the range's units of 32 keys in turn, each with an online softmax of its own,
// and merge through LDS at the end: no barrier in the key loop. A tile of 16
// columns whose keys are split over workgroups is joined by the last of them
// (111 us for six layers of 32 streams, 118 with a launch of its own for it).
// vk_bkv_attn_chunk takes 128, 32 a wave, all waves over the same units, which
// they widen to fp16 in LDS together (double buffered, one barrier a unit).
//
// vk_bkv_attn is bound by the pages' bytes where there are many (six sequences of
// 9 .. 65 thousand keys, e4m3, 32 heads over 8 of 128, up to 4 rows: 457 MB in 98
// us, 4.7 TB/s, a large copy's rate here is 4.9), by dependent rounds of memory
// (item, page, keys, results, join: 8 us) where there are few: 32 streams of 512 ..
// 4096 keys, 16 heads over 2 of 128, take 17.3 us for 38 MB. Four waves a workgroup,
// three workgroups a CU: eight waves took 28 us for those, and two units' loads in
// flight a wave spilled or left two workgroups.
// The 8-bit values are exact in fp16, so a product is two fp16 matrix
// instructions, one for each part of the f32 operand (22 bits): q in two parts
// under a power of two that puts its row's largest value at 2^14, weights in two
// parts of 2^14 w.
//   S^T [keys][columns] = K q^T: K's 16-byte loads are operand registers but for
//     the widening (the pages hold tiles in that order);
//   P's accumulator layout (4 consecutive keys a lane) is the operand layout of
//     O^T [d][columns] = V^T P^T under the key order that V's tiles use, so the
//     weights go from the softmax to the product without leaving the lane.
// Weights w = 2^(s - M) are summed as they are, M the running maximum of s, rounded
// up. For the product a block's V scale v = f 2^e (f in [1, 2)) goes into them, as w v
// 2^-E: E is the running maximum of s - M + e, rounded up, so the largest product is near
// 1 whatever the blocks' values are, a block of small values keeps its bits beside one of
// large values, and zeros (e is below that of any other block) take nothing from either.
// Two fp16 parts of 2^14 of that hold it to 2^-22, or to 2^-38 of the largest where it is
// smaller than 2^-16 of that (the largest is above 2^13 and below 2^15). M and E are whole
// numbers, so what was summed is brought under new ones exactly, and seldom. The open
// block's rows are f32 on both sides and use the f32 matrix instruction.
#include <algorithm>
#include <cmath>

#include "vk_bkv.h"
#include "vk_common.h"

namespace vk {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));

// A tile of vk_bkv_attn_chunk whose keys several shares of the work have.
struct alignas(16) BkvOpen {
    int item, tile, head, pieces;  // pieces 0: none
};

struct BkvAttnArgs {
    BkvView v;
    const float* q;
    float* out;
    float* part;        // [slot][cols][2] (max, sum), then [slot][cols][hd] outputs of a key range
    size_t part_o;      // floats before the partial outputs
    unsigned* joined;   // [tile][head] ranges that have written theirs, zero between calls
    float scale_log2;   // scale * log2(e)
    int layer, hq, g;   // g = hq / n_head
    int n, rows, count; // most items, rows, and rows an item: items beyond are passed over
    int done;           // chunks: items of so few rows are an earlier launch's
    uint32_t g_inv, splits_inv, parts_inv;  // ceil(2^32 / g) and so on: see bkv_div
    BkvOpen* open;      // of each share: the tile whose first piece is its last
    int tiles;          // chunks: places of tiles, see bkv_share
    int parts;          // tiles that an item may have
    int splits;         // key ranges an item may have (grid)
    int per;            // least units of a key range
    int cols;           // columns a slot has room for
};

constexpr int kUnit = 32;  // keys of a wave's step: two 16-token tiles

// A column tile of an item: what its workgroups work on.
struct BkvTile {
    BkvItem it;
    int c0, n;      // first column, columns
    int keys;       // keys that its last row sees
    int full;       // keys in full blocks, no more than keys rounded up to a tile
    int units, per; // units of the 8-bit part, units a key range (vk_bkv_attn)
    __device__ __forceinline__ bool one() const { return per >= units; }               // one key range
    __device__ __forceinline__ bool beyond(int s) const { return s && s * per >= units; }  // no range s
    __device__ __forceinline__ bool final(int s) const { return (s + 1) * per >= units; }  // the last range
};

// x / d for inv = ceil(2^32 / d): exact while x (d - 1) < 2^32
__device__ __forceinline__ int bkv_div(int x, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)x, inv) : x; }

// Whether the call's buffers and launches have room for an item (a captured call
// may meet a later step).
__device__ __forceinline__ bool bkv_fits(const BkvAttnArgs& a, const BkvItem& it) {
    return it.count <= a.count && it.row0 + it.count <= a.rows;
}
__device__ __forceinline__ void bkv_keys(const BkvView& v, BkvTile& t) {
    const int bs_log = 31 - __clz(v.bs);
    t.full = min((t.it.start + t.it.count) >> bs_log << bs_log, (t.keys + 15) & ~15);
    t.units = (t.full + kUnit - 1) / kUnit;
}
// A tile of vk_bkv_attn: the columns of an item, a.cols of them where it has more; false:
// none.
__device__ __forceinline__ bool bkv_tile(const BkvAttnArgs& a, int tile, BkvTile& t) {
    const int item = bkv_div(tile, a.parts_inv);
    t.it = a.v.step[item];
    t.c0 = (tile - item * a.parts) * a.cols;
    t.n = min(t.it.count * a.g - t.c0, a.cols);
    if (t.n <= 0 || !bkv_fits(a, t.it)) return false;
    t.keys = t.it.start + bkv_div(t.c0 + t.n - 1, a.g_inv) + 1;
    bkv_keys(a.v, t);
    t.per = max(a.per, (bkv_div(t.units + a.splits - 1, a.splits_inv) + 3) & ~3);
    return true;
}

constexpr int kChunkCols = 128;  // columns of a tile of vk_bkv_attn_chunk

// Columns kChunkCols * tile .. of an item; false: it has none there.
__device__ __forceinline__ bool bkv_chunk(const BkvAttnArgs& a, const BkvItem& it, int tile, BkvTile& t) {
    t.it = it;
    t.c0 = tile * kChunkCols;
    t.n = min(kChunkCols, it.count * a.g - t.c0);
    if (t.n <= 0 || it.count <= a.done || !bkv_fits(a, it)) return false;
    t.keys = it.start + (t.c0 + t.n - 1) / a.g + 1;
    bkv_keys(a.v, t);
    return true;
}

// Four stored bytes as four fp16 values.
template <int CODEC>
__device__ __forceinline__ void bkv_widen(uint32_t w, half2v& a, half2v& b) {
    if constexpr (CODEC == BKV_INT8) {
        // byte b under 0x64 is the fp16 1024 + b; the value is b - 128
        const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        a = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
    } else {
        a = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
        b = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
    }
}
template <int CODEC>
__device__ __forceinline__ half8v bkv_widen8(uint32_t w0, uint32_t w1) {
    half2v a, b, c, d;
    bkv_widen<CODEC>(w0, a, b);
    bkv_widen<CODEC>(w1, c, d);
    return half8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ uint32_t u4c(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// hi = fp16(x), lo = fp16(x - hi) of two values
__device__ __forceinline__ void bkv_split2(float x, float y, half2v& hi, half2v& lo) {
    const float2v v = {x, y};
    hi = __builtin_convertvector(v, half2v);
    // x - hi, exact; the factor is kept from the compiler, which would widen hi
    // first where one mixed-precision instruction does both
    float minus = -1.0f;
    asm("" : "+s"(minus));
    const float2v r = {fmaf((float)hi.x, minus, x), fmaf((float)hi.y, minus, y)};
    lo = __builtin_convertvector(r, half2v);
}

// sum / max over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48): a swap
// of rows of a value with itself leaves the two that meet in the lane
template <class F>
__device__ __forceinline__ float bkv_fold4(float v, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float bkv_max4(float v) {
    return bkv_fold4(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float bkv_sum4(float v) {
    return bkv_fold4(v, [](float a, float b) { return a + b; });
}
// The maxima of two values: of a in the even lane groups, of b in the odd ones (NaN where
// one is).
__device__ __forceinline__ float bkv_max_two(float a, float b) {
    auto top = [](uint32_t x, uint32_t y) { return __builtin_elementwise_maximum(__uint_as_float(x), __uint_as_float(y)); };
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    const uint32_t v = __float_as_uint(top(r[0], r[1]));
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return top(r[0], r[1]);
}
// The larger of two neighbouring groups' values, in both.
__device__ __forceinline__ float bkv_max2(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The least E, below the e of every block that holds more than zeros: 2^(14 - E) fits f32.
constexpr float kLeastE = -113.0f;

// p v, p = 2^(14 - E): the factor of a weight. A weight is 2^(E - e) at most, so one that
// would take a factor above 2^126 here is below 2^-112: it counts as less.
__device__ __forceinline__ float bkv_factor(float v, float p) { return fminf(v * p, 0x1p126f); }

// A tile's scales as the weights need them: K's (NaN where V's is: then its scores are,
// of the keys that a row sees), V's, and V's exponent (zero: -127).
struct BkvScale {
    float k, v, ve;
    __device__ __forceinline__ void set(float2 sc) {
        k = fmaf(sc.y, 0.0f, sc.x);
        v = sc.y;
        ve = (float)((int)(__float_as_uint(sc.y) >> 23) - 127);
    }
    // of lane l, in all lanes
    __device__ __forceinline__ BkvScale at(int l) const {
        auto get = [l](float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); };
        return BkvScale{get(k), get(v), get(ve)};
    }
};

// M of a column that has seen no key: no score is below it.
constexpr float kNoKey = -0x1.fffffep127f;

// Values that a workgroup on another XCD reads in this launch: past the caches
// that are the XCD's own. Four at a time by the buffer instructions, whose policy
// bit 4 (sc1) is what an access of the device's scope carries; with pairs 32 streams
// took 17.6 us, 17.1 so.
__device__ __forceinline__ void bkv_put2(float* p, float a, float b) {
    const unsigned long long v = ((unsigned long long)__float_as_uint(b) << 32) | __float_as_uint(a);
    __hip_atomic_store((unsigned long long*)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 bkv_get2(const float* p) {
    const unsigned long long v =
        __hip_atomic_load((const unsigned long long*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

__device__ __forceinline__ void bkv_put4(float* out, size_t at, vk_f32x4 x) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)out, 0, kBkvParts * 128 * 4, 0x20000);
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, x), r, (int)(at * 4), 0, 16);
}
__device__ __forceinline__ vk_f32x4 bkv_get4(const float* out, size_t at) {
    const auto r = __builtin_amdgcn_make_buffer_rsrc((void*)out, 0, kBkvParts * 128 * 4, 0x20000);
    return __builtin_bit_cast(vk_f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(at * 4), 0, 16));
}

// Values d .. d + 3 of a column from the partial results of its key ranges,
// joined in the ranges' order, B ranges' loads in flight. pm: the first range's
// (max, sum), part_o + o0: its outputs, cols columns a slot; range s > 0 is s * step -
// back slots behind. SAME: written by this launch. What is joined is an output at
// every step, so it stays in f32's range where the values do.
template <int HD, bool SAME, int B>
__device__ __forceinline__ vk_f32x4 bkv_join(const float* pm, const float* part_o, size_t o0, int ranges,
                                              int cols, int step, int back) {
    float m = kNoKey, sum = 0.0f;
    vk_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < ranges; s += B) {
        float2 ml[B];
        vk_f32x4 o[B];
#pragma unroll
        for (int x = 0; x < B; ++x) {
            const int r = min(s + x, ranges - 1);
            const size_t at = r ? (size_t)(r * step - back) * cols : 0;
            if constexpr (SAME) {
                ml[x] = bkv_get2(pm + at * 2);
                o[x] = bkv_get4(part_o, o0 + at * HD);
            } else {
                ml[x] = *(const float2*)(pm + at * 2);
                o[x] = *(const vk_f32x4*)(part_o + o0 + at * HD);
            }
        }
        float to = m;
#pragma unroll
        for (int x = 0; x < B; ++x) to = fmaxf(to, ml[x].x);
        const float before = sum * __builtin_amdgcn_exp2f(m - to);
        m = to;
        sum = before;
#pragma unroll
        for (int x = 0; x < B; ++x) {
            ml[x].y = s + x < ranges ? ml[x].y * __builtin_amdgcn_exp2f(ml[x].x - m) : 0.0f;
            sum += ml[x].y;
        }
        const float f = 1.0f / sum;
        y *= before * f;
#pragma unroll
        for (int x = 0; x < B; ++x) y += o[x] * (ml[x].y * f);
    }
    return y;
}

// One wave's query columns in blocks of 16 and what it has summed for them.
template <int HD, int C, bool CHUNKS>
struct BkvWave {
    static constexpr int U = HD / 64, DT = HD / 16;
    int col, grp;   // lane's column of a block, and its group of 16 lanes
    float qf[C];    // a score is qf (not below zero) times the product of q's parts
    int last[C];    // last key that the lane's column sees
    float M[C], L[C], E[C], P[C];  // P = 2^(14 - E)
    vk_f32x4 O[C][DT];  // [4 c + i][r]: value 64 c + 16 grp + 4 r + i of the lane's column

    // values 64 c + 16 grp + 4 r .. of the lane's column
    __device__ __forceinline__ vk_f32x4 out4(int ct, int c, int r) const {
        return vk_f32x4{O[ct][4 * c][r], O[ct][4 * c + 1][r], O[ct][4 * c + 2][r], O[ct][4 * c + 3][r]};
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            M[ct] = kNoKey;
            L[ct] = 0.0f;
            E[ct] = kLeastE;
            P[ct] = 0x1p127f;
#pragma unroll
            for (int d = 0; d < DT; ++d) O[ct][d] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // the row of the item that holds column c of the tile (c < 16 C of the kernel's; chunks: any)
    __device__ __forceinline__ int item_row(const BkvAttnArgs& a, const BkvTile& t, int c) const {
        return CHUNKS ? (t.c0 + c) / a.g : bkv_div(t.c0 + c, a.g_inv);
    }
    // place in q and out of column c of the tile (of column 0 for one beyond its columns)
    __device__ __forceinline__ size_t row(const BkvAttnArgs& a, const BkvTile& t, int head, int c) const {
        c = c < t.n ? c : 0;
        const int cc = t.c0 + c, j = item_row(a, t, c);
        return ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD;
    }
    // q of the 16 columns from c0 on: of the lane's column the values 16 i + 4 grp ..
    // (fetch_q), and their parts, k steps of 8 (split_q)
    __device__ __forceinline__ void fetch_q(const BkvAttnArgs& a, const BkvTile& t, int head, int c0,
                                            float4 (&x)[4 * U]) const {
        const float* p = a.q + row(a, t, head, c0 + col) + grp * 4;
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) x[i] = *(const float4*)(p + 16 * i);
    }
    __device__ __forceinline__ void split_q(const BkvAttnArgs& a, const BkvTile& t, int ct, int c0,
                                            const float4 (&x)[4 * U], half8v (&h8)[2 * U], half8v (&l8)[2 * U]) {
        const bool live = c0 + col < t.n;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * U; ++i)
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        top = bkv_max4(live ? top : 0.0f);
        // the largest value goes to 2^14 .. 2^15; rows below 2^-106 keep fewer bits
        const int e = min(141 - (int)(__float_as_uint(top) >> 23), 120);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        const float up = live ? copysignf(__uint_as_float((uint32_t)(127 + e) << 23), a.scale_log2) : 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * U; ++i) {
            half2v h[4], l[4];
            const float4 x0 = x[2 * i], x1 = x[2 * i + 1];
            bkv_split2(x0.x * up, x0.y * up, h[0], l[0]);
            bkv_split2(x0.z * up, x0.w * up, h[1], l[1]);
            bkv_split2(x1.x * up, x1.y * up, h[2], l[2]);
            bkv_split2(x1.z * up, x1.w * up, h[3], l[3]);
            h8[i] = half8v{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
            l8[i] = half8v{l[0].x, l[0].y, l[1].x, l[1].y, l[2].x, l[2].y, l[3].x, l[3].y};
        }
        qf[ct] = fabsf(a.scale_log2) * down;
        last[ct] = t.it.start + item_row(a, t, c0 + col);
    }
    // M and E of a column take a tile or two in, of which lanes of odd groups have one
    // and those of even groups the other: its largest score t and its V's exponent v;
    // what was summed so far shrinks
    __device__ __forceinline__ void raise(int ct, float t, float v) {
        if (__any(t - M[ct] > fminf(E[ct] - v, 0.0f))) {
            const float to = fmaxf(M[ct], ceilf(bkv_max2(t))), up = M[ct] - to, eo = E[ct] + up;
            const float ee = fmaxf(fmaxf(eo, kLeastE), ceilf(bkv_max2(t - to + v)));
            const float c = __builtin_amdgcn_exp2f(eo - ee);
            L[ct] *= __builtin_amdgcn_exp2f(up);
            M[ct] = to;
            E[ct] = ee;
            P[ct] = ldexpf(1.0f, 14 - (int)ee);
#pragma unroll
            for (int d = 0; d < DT; ++d) O[ct][d] *= c;
        }
    }
    // The column's output so far in O, with the weights' sum over its lanes. A sum of
    // weights' products may leave f32's range where no value does; this does not.
    __device__ __forceinline__ float finish(int ct) {
        const float l = bkv_sum4(L[ct]), f = l == 0.0f ? 0.0f : 1.0f / l;
        const int x = (int)E[ct] - 14;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) O[ct][d][r] = ldexpf(O[ct][d][r] * f, x);
        return l;
    }
    // raw scores of a unit (32 keys from key0 on, none from `full` on) -> the two
    // parts of 2^14 times its weights, V's scales under 2^E in them. hide: some key is
    // hidden from some column.
    __device__ __forceinline__ void weigh(int ct, vk_f32x4 (&S)[2], const BkvScale (&sc)[2], int key0, int full,
                                          bool hide, half8v& ph, half8v& pl) {
        // no factor is below zero: the largest raw score of a tile is its largest score
        const float f[2] = {sc[0].k * qf[ct], sc[1].k * qf[ct]};
        auto hidden = [&](int lim, int r) { return key0 + (r >> 2) * 16 + grp * 4 + (r & 3) >= lim; };
        auto top = [](float a, float b) { return __builtin_elementwise_maximum(a, b); };
        int lim = min(last[ct] + 1, full);
        if (hide)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (hidden(lim, r)) S[r >> 2][r & 3] = -INFINITY;
        const float t0 = top(top(top(S[0][0], S[0][1]), S[0][2]), S[0][3]);
        const float t1 = top(top(top(S[1][0], S[1][1]), S[1][2]), S[1][3]);
        raise(ct, bkv_max_two(t0, t1) * ((grp & 1 ? sc[1].k : sc[0].k) * qf[ct]), grp & 1 ? sc[1].ve : sc[0].ve);
        float e[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) e[r] = __builtin_amdgcn_exp2f(fmaf(S[r >> 2][r & 3], f[r >> 2], -M[ct]));
        if (hide) {  // also where the factor is zero or NaN
            asm("" : "+v"(lim));  // (else both branches' comparisons are made before either)
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (hidden(lim, r)) e[r] = 0.0f;
        }
        L[ct] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
        float w[8];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const float g = bkv_factor(sc[x].v, P[ct]);
#pragma unroll
            for (int r = 0; r < 4; ++r) w[4 * x + r] = e[4 * x + r] * g;
        }
        half2v h[4], l[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) bkv_split2(w[2 * r], w[2 * r + 1], h[r], l[r]);
        ph = half8v{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
        pl = half8v{l[0].x, l[0].y, l[1].x, l[1].y, l[2].x, l[2].y, l[3].x, l[3].y};
    }
    // 16 f32 rows of the open block, from key0 on; columns c0 ..
    __device__ __forceinline__ void open_rows(const BkvAttnArgs& a, const BkvTile& t, int head, int key0, int c0) {
        const BkvView& v = a.v;
        const size_t side = (size_t)v.n_head * 2 * v.bs * HD;
        const float* ring = v.ring + ((size_t)a.layer * v.n_seq + t.it.seq) * 2 * side + (size_t)head * 2 * v.bs * HD;
        const int ring_mask = 2 * v.bs - 1;
        const float* kp = ring + (size_t)((key0 + col) & ring_mask) * HD + grp * 4;
        const float* vring = ring + side;
        // V: four rows (keys 4 grp + r), values 64 c + 4 col + i as row col of product
        // 4 c + i; rows that no column sees are not used
        float vv[DT][4];
        float top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = key0 + grp * 4 + r;
            const float* p = vring + (size_t)(key & ring_mask) * HD + 4 * col;
#pragma unroll
            for (int c = 0; c < U; ++c) {
                const float4 y = *(const float4*)(p + 64 * c);
                vv[4 * c][r] = y.x, vv[4 * c + 1][r] = y.y, vv[4 * c + 2][r] = y.z, vv[4 * c + 3][r] = y.w;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (key >= t.keys) vv[d][r] = 0.0f;
                odd = odd || !(fabsf(vv[d][r]) < INFINITY);
                top = fmaxf(top, fabsf(vv[d][r]));
            }
        }
        const bool any_odd = __any(odd);
        if (any_odd) {  // of the values that are finite, at least 1
            top = 1.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(vv[d][r]) < INFINITY ? fabsf(vv[d][r]) : 0.0f);
        }
        // a power of two in the place of a block's scale, so that E weighs these
        // rows like the blocks: the largest |v| is 2^9 .. 2^10 of it (less below 2^-100)
        top = vk_group_max<64>(top);
        const int te = max((int)(__float_as_uint(top) >> 23), 27) - 136;
        const float tdown = __uint_as_float((uint32_t)(127 - te) << 23);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) vv[d][r] *= tdown;
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            const float* p = a.q + row(a, t, head, c0 + ct * 16 + col) + grp * 4;
            vk_f32x4 s4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int i = 0; i < DT; ++i) {
                const float4 x = *(const float4*)(kp + 16 * i), y = *(const float4*)(p + 16 * i);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, s4, 0, 0, 0);
            }
            float s[4], m = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] = key0 + grp * 4 + r <= last[ct] ? s4[r] * a.scale_log2 : -INFINITY;
                m = fmaxf(m, s[r]);
            }
            raise(ct, bkv_max4(m), (float)te);
            const float g = bkv_factor(__uint_as_float((uint32_t)(127 + te) << 23), P[ct]);
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[r] = __builtin_amdgcn_exp2f(s[r] - M[ct]);
                L[ct] += e[r];
                e[r] *= g;
            }
            if (!any_odd) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[d][r], e[r], O[ct][d], 0, 0, 0);
                continue;
            }
            // a value that is not finite: only the columns that see its key take it
#pragma unroll 1
            for (int x = 0; x < 16 && key0 + x < t.keys; ++x) {
                float w = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((x & 3) == r) w = __shfl(e[r], (x >> 2) * 16 + col, VK_WAVE);
                const float* p1 = vring + (size_t)((key0 + x) & ring_mask) * HD + grp * 16;
                if (key0 + x <= last[ct]) {
#pragma unroll
                    for (int c = 0; c < U; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float4 y = *(const float4*)(p1 + 64 * c + 4 * r);
                            O[ct][4 * c][r] = fmaf(w, y.x * tdown, O[ct][4 * c][r]);
                            O[ct][4 * c + 1][r] = fmaf(w, y.y * tdown, O[ct][4 * c + 1][r]);
                            O[ct][4 * c + 2][r] = fmaf(w, y.z * tdown, O[ct][4 * c + 2][r]);
                            O[ct][4 * c + 3][r] = fmaf(w, y.w * tdown, O[ct][4 * c + 3][r]);
                        }
                }
            }
        }
    }
};

// Where the tiles of one (layer, head) are: page p at base + p * stride, its
// scales at sc[p * n_head].
struct BkvPlace {
    const uint8_t* base;
    const float2* sc;
    uint32_t stride, n_head;
    __device__ __forceinline__ BkvPlace(const BkvView& v, int layer, int head, const uint8_t* pool,
                                        const float2* scales) {
        const uint32_t chunk = 2u * (uint32_t)(v.bs * v.hd);
        const size_t first = (size_t)layer * v.n_page * v.n_head + head;
        base = pool + first * chunk;
        sc = scales + first;
        n_head = (uint32_t)v.n_head;
        stride = n_head * chunk;
    }
    // tile of a page that holds key
    __device__ __forceinline__ const uint8_t* tile(int page, int key, int bs, int hd) const {
        return base + (uint64_t)(uint32_t)page * stride + (uint32_t)(((key & (bs - 1)) >> 4) * 16 * hd);
    }
    __device__ __forceinline__ float2 scale(int page) const { return sc[(uint64_t)(uint32_t)page * n_head]; }
};

constexpr int kWaves = 4;  // of the kernel below

// 16 columns: three workgroups a CU, five of heads of 64 (64 sequences of up to 448 keys,
// 20 heads: 16.3 us, 19.4 with four).
template <int HD, int CODEC, int C>
__global__ __launch_bounds__(64 * kWaves, C == 2 ? 2 : HD == 64 ? 5 : 3) void vk_bkv_attn(
    BkvAttnArgs a, const uint8_t* __restrict__ pool, const float2* __restrict__ scales) {
    using W = BkvWave<HD, C, false>;
    constexpr int U = W::U, DT = W::DT, OS = HD + 4;
    // q's parts while keys are read (16 columns: in each wave's registers instead),
    // the waves' outputs after
    __shared__ union {
        uint4 q[C > 1 ? C * U * 4 * 64 : 1];
        float o[kWaves][16][OS];
    } sh;
    __shared__ float sqf[C * 16];  // q's factor of each column
    __shared__ float2 sml[kWaves][16];
    __shared__ bool s_last;
    // ranges are the grid's slowest index: those that short items do not have come last
    const int tile = blockIdx.x, head = blockIdx.y, split = blockIdx.z;
    BkvTile t;
    if (!bkv_tile(a, tile, t) || t.beyond(split)) return;
    const BkvView& v = a.v;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bs_log = 31 - __clz(v.bs);
    W w;
    w.col = lane & 15;
    w.grp = lane >> 4;

    // this wave's units: u0, u0 + kWaves, .. below u1
    const int u0 = split * t.per + wave, u1 = min(t.units, (split + 1) * t.per);
    const int* table = v.table + (size_t)t.it.seq * v.max_blocks;
    // lane l holds the page of tile l & 1 of the wave's unit k0 + l / 2
    auto pages_from = [&](int k0) {
        const int u = min(u0 + kWaves * (k0 + (lane >> 1)), t.units - 1);
        const int key = min(u * kUnit + (lane & 1) * 16, t.full - 16);
        return table[key >> bs_log];
    };
    int pages = 0;
    if (u0 < u1) pages = pages_from(0);
    const BkvPlace place(v, a.layer, head, pool, scales);
    // zero, but a vector register to the compiler: a scale is loaded and taken apart
    // in all lanes, where scalar registers made branches of it (18.4 us against 17.6)
    int zero = 0;
    asm("" : "+v"(zero));

    uint4 kr[2][U], vr[2][U];
    const uint8_t* at[2];
    float2 sc[2];
    // the k-th unit of this wave: its tiles' places, and the loads of K (V: load_v)
    auto load_k = [&](int u, int k) {
        if (k > 0 && (k & 31) == 0) pages = pages_from(k);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int page = __builtin_amdgcn_readlane(pages, 2 * (k & 31) + x);
            at[x] = place.tile(page, min(u * kUnit + x * 16, t.full - 16), v.bs, HD);
            sc[x] = place.scale(page + zero);
#pragma unroll
            for (int i = 0; i < U; ++i) kr[x][i] = ((const uint4*)(at[x] + i * 1024))[lane];
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < U; ++i) vr[x][i] = ((const uint4*)(at[x] + v.bs * HD + i * 1024))[lane];
    };
    half8v qh[2 * U], ql[2 * U];
    float4 x[4 * U];
    if (C == 1 || wave < C) w.fetch_q(a, t, head, C == 1 ? 0 : wave * 16, x);
    w.clear();
#pragma unroll
    for (int ct = 0; ct < C; ++ct) w.last[ct] = t.it.start + w.item_row(a, t, ct * 16 + w.col);
    // The open block's rows, in the last key range: a tile a wave, from the last
    // wave down (the range's last units are few more often than not), and before
    // the wave's units: these rows wait for no page.
    const int open = t.full + (kWaves - 1 - wave) * 16;
    if (t.final(split) && open < t.keys) w.open_rows(a, t, head, open, 0);
    if (u0 < u1) {
        load_k(u0, 0);
        __builtin_amdgcn_sched_barrier(0);  // K first, as in the loop: its wait is for K alone
        load_v();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (C == 1) w.split_q(a, t, 0, 0, x, qh, ql);
    }
    if constexpr (C > 1) {
        if (wave < C) {
            w.split_q(a, t, 0, wave * 16, x, qh, ql);
            if (w.grp == 0) sqf[wave * 16 + w.col] = w.qf[0];
#pragma unroll
            for (int i = 0; i < 2 * U; ++i) {
                sh.q[((wave * 2 * U + i) * 2 + 0) * 64 + lane] = __builtin_bit_cast(uint4, qh[i]);
                sh.q[((wave * 2 * U + i) * 2 + 1) * 64 + lane] = __builtin_bit_cast(uint4, ql[i]);
            }
        }
        VK_LDS_BARRIER();
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            w.qf[ct] = sqf[ct * 16 + w.col];
            w.last[ct] = t.it.start + w.item_row(a, t, ct * 16 + w.col);
        }
    }

    for (int u = u0, k = 0; u < u1; u += kWaves, ++k) {
        // S^T of both tiles: raw scores under qf * K's scale
        vk_f32x4 S[C][2];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) S[ct][0] = S[ct][1] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 2 * U; ++i) {
            half8v ka[2];
#pragma unroll
            for (int x = 0; x < 2; ++x)
                ka[x] = bkv_widen8<CODEC>(u4c(kr[x][i >> 1], 2 * (i & 1)), u4c(kr[x][i >> 1], 2 * (i & 1) + 1));
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                half8v h8 = qh[i], l8 = ql[i];
                if constexpr (C > 1) {
                    h8 = __builtin_bit_cast(half8v, sh.q[((ct * 2 * U + i) * 2 + 0) * 64 + lane]);
                    l8 = __builtin_bit_cast(half8v, sh.q[((ct * 2 * U + i) * 2 + 1) * 64 + lane]);
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], l8, S[ct][x], 0, 0, 0);
                    S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], h8, S[ct][x], 0, 0, 0);
                }
            }
        }
        BkvScale now[2];
        now[0].set(sc[0]);
        now[1].set(sc[1]);
        const bool more = u + kWaves < u1;
        if (more) load_k(u + kWaves, k + 1);
        const bool hide = u * kUnit + kUnit > min(t.it.start + 1, t.full);
        half8v ph[C], pl[C];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) w.weigh(ct, S[ct], now, u * kUnit, t.full, hide, ph[ct], pl[ct]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const half8v va = bkv_widen8<CODEC>(u4c(vr[0][d >> 2], d & 3), u4c(vr[1][d >> 2], d & 3));
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                w.O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[ct], w.O[ct][d], 0, 0, 0);
                w.O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[ct], w.O[ct][d], 0, 0, 0);
            }
        }
        if (more) load_v();
    }

    // the waves' results of each 16 columns, merged by all threads
    const bool direct = t.one();
    const size_t slot = ((size_t)blockIdx.x * v.n_head + head) * a.splits + split;
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
        if (ct * 16 >= t.n) break;
        const float l = w.finish(ct);
        __syncthreads();  // q's parts, or the columns before, are done with
        if (w.grp == 0) sml[wave][w.col] = make_float2(w.M[ct], l);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *(vk_f32x4*)&sh.o[wave][w.col][(d >> 2) * 64 + 16 * w.grp + (d & 3) * 4] = w.out4(ct, d >> 2, d & 3);
        __syncthreads();
        constexpr int PT = 4 * kWaves, PD = HD / PT;  // threads a column, values a thread
        const int c = threadIdx.x / PT, d0 = (threadIdx.x % PT) * PD;
        if (ct * 16 + c < t.n) {
            float m = kNoKey, sum = 0.0f, f[kWaves];
#pragma unroll
            for (int x = 0; x < kWaves; ++x) m = fmaxf(m, sml[x][c].x);
#pragma unroll
            for (int x = 0; x < kWaves; ++x) {
                f[x] = sml[x][c].y * __builtin_amdgcn_exp2f(sml[x][c].x - m);
                sum += f[x];
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // 0: the range is hidden from the column
            vk_f32x4 y[PD / 4];
#pragma unroll
            for (int i = 0; i < PD / 4; ++i) {
                y[i] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kWaves; ++x) y[i] += *(const vk_f32x4*)&sh.o[x][c][d0 + 4 * i] * (f[x] * inv);
            }
            if (direct) {
                float* dst = a.out + w.row(a, t, head, ct * 16 + c) + d0;
#pragma unroll
                for (int i = 0; i < PD / 4; ++i) *(vk_f32x4*)(dst + 4 * i) = y[i];
            } else {
                const size_t at = slot * a.cols + ct * 16 + c;
                float *pm = a.part + at * 2, *po = a.part + a.part_o;
                if constexpr (C == 1) {
                    if (d0 == 0) bkv_put2(pm, m, sum);
#pragma unroll
                    for (int i = 0; i < PD / 4; ++i) bkv_put4(po, at * HD + d0 + 4 * i, y[i]);
                } else {
                    if (d0 == 0) *(float2*)pm = make_float2(m, sum);
#pragma unroll
                    for (int i = 0; i < PD / 4; ++i) *(vk_f32x4*)(po + at * HD + d0 + 4 * i) = y[i];
                }
            }
        }
    }
    if (direct || C > 1) return;
    // The tile's last workgroup to get here joins the ranges: each counts itself
    // once its results have reached memory. All write before any waits, so the
    // order in which they run does not matter, and nothing spins.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int ranges = (t.units + t.per - 1) / t.per;
    unsigned* count = a.joined + (size_t)blockIdx.x * v.n_head + head;
    if (threadIdx.x == 0) s_last = atomicAdd(count, 1u) == (unsigned)ranges - 1;
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) atomicExch(count, 0u);
    constexpr int PT = HD / 4;
    const size_t first = (slot - split) * a.cols;
    for (int c = threadIdx.x / PT; c < t.n; c += 64 * kWaves / PT) {
        const int d = (threadIdx.x % PT) * 4;
        *(vk_f32x4*)(a.out + w.row(a, t, head, c) + d) =
            bkv_join<HD, true, 8>(a.part + (first + c) * 2, a.part + a.part_o, (first + c) * HD + d, ranges, a.cols, 1,
                                  0);
    }
}

// ---- chunks ----------------------------------------------------------------------
// The call's work is one line of (head, item, tile, unit), kTileCost units more a
// tile for its start and end. Every workgroup takes an even share of the line, so
// all end together whatever the lengths are; a share holds whole tiles and at most
// two pieces, one at each end, whose results the kernel below joins. One workgroup
// for each key range of each tile left 40 % of the waves' places empty at six chunks
// of 450 .. 1030 rows over up to 4500 keys, 16 heads over 2 of 128, and finer ranges
// cost more to join than they gave: 264 us against 204 with shares.
// That call takes 186 us now: 0.39 PFLOP/s of the operator, 0.79 of fp16 products.
// Of a unit's time about a quarter each is the products and the weights, the
// rest starts, joins (15 us: 96 MB) and waits for the four waves' common units.

// The least share, in units (five sequences of up to 1000 keys and 61 rows: 30 us, 33
// with 8, 41 with 12), and a tile's start and end (2: 212 us for the call above, 5:
// 204, 12: 223).
constexpr int kLeast = 4, kTileCost = 5;

struct BkvShare {
    long long begin, end;       // on the line
    int size, index;            // of every share; of this one
    int item, tile, head, at;   // where it begins
};

// The share of workgroup w, the same on all threads; false: sh.index has none. The
// places of tiles: item i's begin at row0_i * g / kChunkCols + i (room for a partly
// filled tile each). lds: kBkvMaxItems ints and 16 more. About 3 us.
__device__ __forceinline__ bool bkv_share(const BkvAttnArgs& a, int w, int* lds, BkvShare& sh) {
    const int n = min(a.v.meta[BKV_STEP_N], a.n), t = threadIdx.x;
    int* first = lds;
    long long* sums = (long long*)(lds + kBkvMaxItems);
    for (int x = t; x < n; x += 256) first[x] = (int)((long long)a.v.step[x].row0 * a.g / kChunkCols) + x;
    __syncthreads();
    // this thread's places, and the first one's item
    const int m = (a.tiles + 255) / 256, p0 = t * m, p1 = min(p0 + m, a.tiles);
    int lo = 0, hi = n;  // the last item that begins at or before p0
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= p0) lo = mid;
        else hi = mid;
    }
    // calls f(item, tile, cost) for each tile until it returns true
    auto walk = [&](auto f) {
        if (n == 0) return;
        int i = lo;
        BkvItem it = a.v.step[i];
        for (int p = p0; p < p1; ++p) {
            while (i + 1 < n && first[i + 1] <= p) it = a.v.step[++i];
            BkvTile x;
            if (bkv_chunk(a, it, p - first[i], x) && f(i, p - first[i], x.units + kTileCost)) return;
        }
    };
    long long mine = 0;
    walk([&](int, int, int cost) {
        mine += cost;
        return false;
    });
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(upto, o, 64);
        if ((t & 63) >= o) upto += x;
    }
    if ((t & 63) == 63) sums[t >> 6] = upto;
    __syncthreads();
    long long one = 0;  // a head's
    for (int x = 0; x < 4; ++x) {
        if (x < t >> 6) upto += sums[x];
        one += sums[x];
    }
    const long long all = one * a.v.n_head;
    sh.size = (int)max((all + kBkvShares - 1) / kBkvShares, (long long)kLeast);
    const int shares = (int)((all + sh.size - 1) / sh.size);
    // neighbours on one XCD (they read the same keys)
    const int per = (shares + 7) / 8;
    sh.index = (w >> 3) < per ? (w & 7) * per + (w >> 3) : w;
    if (sh.index >= shares) return false;
    sh.begin = (long long)sh.index * sh.size;
    sh.end = min(sh.begin + sh.size, all);
    sh.head = (int)(sh.begin / one);
    const long long off = sh.begin - sh.head * one;
    int* found = (int*)(sums + 4);
    if (off >= upto - mine && off < upto) {
        long long at = upto - mine;
        walk([&](int i, int tile, int cost) {
            if (off < at + cost) {
                found[0] = i;
                found[1] = tile;
                found[2] = (int)(off - at);
                return true;
            }
            at += cost;
            return false;
        });
    }
    __syncthreads();
    sh.item = __builtin_amdgcn_readfirstlane(found[0]);
    sh.tile = __builtin_amdgcn_readfirstlane(found[1]);
    sh.at = __builtin_amdgcn_readfirstlane(found[2]);
    return true;
}

template <int HD, int CODEC>
__global__ __launch_bounds__(256, 2) void vk_bkv_attn_chunk(BkvAttnArgs a, const uint8_t* __restrict__ pool,
                                                            const float2* __restrict__ scales) {
    constexpr int C = 2;
    using W = BkvWave<HD, C, true>;
    constexpr int U = W::U, DT = W::DT;
    __shared__ uint4 kv[2][8 * U * 64];  // a unit's fragments: K [tile][k step], then V [d tile]
    static_assert(sizeof(kv) >= (kBkvMaxItems + 16) * sizeof(int), "bkv_share");
    BkvShare sh;
    if (!bkv_share(a, blockIdx.x, (int*)kv, sh)) {
        if (threadIdx.x == 0) a.open[sh.index].pieces = 0;
        return;
    }
    __syncthreads();
    const BkvView& v = a.v;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bs_log = 31 - __clz(v.bs), c0 = wave * 32;
    W w;
    w.col = lane & 15;
    w.grp = lane >> 4;
    int item = sh.item, head = sh.head, tile = sh.tile, at = sh.at;
    int left = (int)(sh.end - sh.begin);
    BkvOpen open = {0, 0, 0, 0};
    BkvItem it = v.step[item];
    for (bool begin = true; left > 0; begin = false) {
        BkvTile t;
        if (!bkv_chunk(a, it, tile, t)) {  // the next item, or the next head
            tile = 0;
            if (++item == min(v.meta[BKV_STEP_N], a.n)) {
                item = 0;
                ++head;
            }
            it = v.step[item];
            continue;
        }
        const int cost = t.units + kTileCost, to = min(cost, at + left);
        // the share with a tile's last unit ends it, also where the line does not
        if (at > 0 && at >= t.units) {
            left -= to - at;
            at = 0;
            ++tile;
            continue;
        }
        const int u0 = at, u1 = min(to, t.units);
        const bool last = to >= t.units, whole = last && at == 0;
        const int* table = v.table + (size_t)t.it.seq * v.max_blocks;
        // lane l holds the page of tile l of the units k0 .. k0 + 31 of the range
        auto pages_from = [&](int k0) {
            const int key = min((u0 + k0) * kUnit + lane * 16, t.full - 16);
            return table[key >> bs_log];
        };
        int pages = 0;
        BkvScale scale;  // of the lanes' pages
        const BkvPlace place(v, a.layer, head, pool, scales);
        if (u0 < u1) {
            pages = pages_from(0);
            scale.set(place.scale(pages));
        }
        // wave's 1 KB pieces of a unit: U = 2: K's and V's piece (tile wave / 2, half
        // wave % 2); U = 1: waves 0, 1 K's tiles, 2, 3 V's
        uint4 raw[U];
        BkvScale sc[2], sc_next[2];
        auto load = [&](int k) {
            if (k > 0 && (k & 31) == 0) {
                pages = pages_from(k);
                scale.set(place.scale(pages));
            }
            const int u = u0 + k, xw = U == 2 ? wave >> 1 : wave & 1;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int page = __builtin_amdgcn_readlane(pages, 2 * (k & 31) + x);
                sc_next[x] = scale.at(2 * (k & 31) + x);
                if (x == xw) {
                    const uint8_t* p = place.tile(page, min(u * kUnit + x * 16, t.full - 16), v.bs, HD);
                    if constexpr (U == 2) {
                        p += (wave & 1) * 1024;
                        raw[0] = ((const uint4*)p)[lane];
                        raw[1] = ((const uint4*)(p + v.bs * HD))[lane];
                    } else {
                        raw[0] = ((const uint4*)(p + (wave >> 1) * v.bs * HD))[lane];
                    }
                }
            }
        };
        auto widen_k = [&](uint4* b, const uint4& r, int x, int i) {
            b[(x * 2 * U + 2 * i) * 64 + lane] = __builtin_bit_cast(uint4, bkv_widen8<CODEC>(r.x, r.y));
            b[(x * 2 * U + 2 * i + 1) * 64 + lane] = __builtin_bit_cast(uint4, bkv_widen8<CODEC>(r.z, r.w));
        };
        auto widen_v = [&](uint4* b, const uint4& r, int x, int i) {
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                half2v p, q;
                bkv_widen<CODEC>(u4c(r, d), p, q);
                ((uint2*)&b[(4 * U + 4 * i + d) * 64 + lane])[x] =
                    make_uint2(__builtin_bit_cast(uint32_t, p), __builtin_bit_cast(uint32_t, q));
            }
        };
        auto widen = [&](int buf) {
            if constexpr (U == 2) {
                widen_k(kv[buf], raw[0], wave >> 1, wave & 1);
                widen_v(kv[buf], raw[1], wave >> 1, wave & 1);
            } else if (wave < 2) {
                widen_k(kv[buf], raw[0], wave, 0);
            } else {
                widen_v(kv[buf], raw[0], wave - 2, 0);
            }
        };
        if (u0 < u1) load(0);
        half8v qh[C][2 * U], ql[C][2 * U];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            float4 x[4 * U];
            w.fetch_q(a, t, head, c0 + ct * 16, x);
            w.split_q(a, t, ct, c0 + ct * 16, x, qh[ct], ql[ct]);
        }
        w.clear();
        // keys that the wave's columns see: all of them below `all`, none from `none` on
        const bool live = c0 < t.n;
        const int all = min(t.it.start + (t.c0 + c0) / a.g + 1, t.full);
        const int none = live ? t.it.start + (t.c0 + min(c0 + 31, t.n - 1)) / a.g + 1 : 0;
        if (u0 < u1) {
            widen(0);
            sc[0] = sc_next[0];
            sc[1] = sc_next[1];
            if (u0 + 1 < u1) load(1);
        }
        VK_LDS_BARRIER();
        for (int u = u0, k = 0; u < u1; ++u, ++k) {
            const uint4* b = kv[k & 1];
            if (u * kUnit < none) {
                vk_f32x4 S[C][2];
#pragma unroll
                for (int ct = 0; ct < C; ++ct) S[ct][0] = S[ct][1] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 2 * U; ++i) {
                    half8v ka[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) ka[x] = __builtin_bit_cast(half8v, b[(x * 2 * U + i) * 64 + lane]);
#pragma unroll
                    for (int ct = 0; ct < C; ++ct)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], ql[ct][i], S[ct][x], 0, 0, 0);
                            S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], qh[ct][i], S[ct][x], 0, 0, 0);
                        }
                }
                const bool hide = u * kUnit + kUnit > all;
                half8v ph[C], pl[C];
#pragma unroll
                for (int ct = 0; ct < C; ++ct) w.weigh(ct, S[ct], sc, u * kUnit, t.full, hide, ph[ct], pl[ct]);
                // from here to the barrier before the other workgroup's waves: it is what
                // this one's wait for (212 us against 204)
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const half8v va = __builtin_bit_cast(half8v, b[(4 * U + d) * 64 + lane]);
#pragma unroll
                    for (int ct = 0; ct < C; ++ct) {
                        w.O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[ct], w.O[ct][d], 0, 0, 0);
                        w.O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[ct], w.O[ct][d], 0, 0, 0);
                    }
                }
            }
            if (u + 1 < u1) {
                widen((k + 1) & 1);
                sc[0] = sc_next[0];
                sc[1] = sc_next[1];
                if (u + 2 < u1) load(k + 2);
            }
            VK_LDS_BARRIER();
            __builtin_amdgcn_s_setprio(0);
        }
        if (live) {
            if (last)
                for (int key0 = t.full; key0 < t.keys; key0 += 16) w.open_rows(a, t, head, key0, c0);
            const size_t slot = 2 * sh.index + !begin;
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                const int c = c0 + ct * 16 + w.col;
                const float l = w.finish(ct);
                if (c >= t.n) continue;
                float* dst = whole ? a.out + w.row(a, t, head, c) : a.part + a.part_o + (slot * kChunkCols + c) * HD;
                if (!whole && w.grp == 0) ((float2*)a.part)[slot * kChunkCols + c] = make_float2(w.M[ct], l);
#pragma unroll
                for (int d = 0; d < DT; ++d)
                    *(vk_f32x4*)(dst + (d >> 2) * 64 + 16 * w.grp + (d & 3) * 4) = w.out4(ct, d >> 2, d & 3);
            }
        }
        // a tile that begins here and goes on in later shares
        if (!last && at == 0) open = {item, tile, 2 * head + !begin, 1 + (t.units - to + sh.size - 1) / sh.size};
        left -= to - at;
        at = 0;
        ++tile;
    }
    if (threadIdx.x == 0) a.open[sh.index] = open;
}

// The pieces of a tile of chunks (share blockIdx.x has the first), HD / 4 threads a
// column. Mostly two or three: eight loads in flight made the call above 5 us longer.
template <int HD>
__global__ __launch_bounds__(256) void vk_bkv_attn_join(BkvAttnArgs a) {
    constexpr int PT = HD / 4;
    const BkvOpen o = a.open[blockIdx.x];
    if (o.pieces == 0) return;
    BkvTile t;
    bkv_chunk(a, a.v.step[o.item], o.tile, t);
    const int c = blockIdx.y * (256 / PT) + threadIdx.x / PT, d = (threadIdx.x % PT) * 4;
    if (c >= t.n) return;
    const int head = o.head >> 1, second = o.head & 1;
    const size_t first = (size_t)(2 * blockIdx.x + second) * kChunkCols + c;
    const int cc = t.c0 + c, j = cc / a.g;
    *(vk_f32x4*)(a.out + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD + d) =
        bkv_join<HD, false, 2>(a.part + first * 2, a.part + a.part_o, first * HD + d, o.pieces, kChunkCols, 2, second);
}

// The key ranges of tiles of 17 to 32 columns (their own last workgroup would take
// longer over them than a launch does): HD / 4 threads a column.
template <int HD>
__global__ __launch_bounds__(256) void vk_bkv_attn_merge(BkvAttnArgs a) {
    constexpr int PT = HD / 4;
    const int head = blockIdx.y, tile = blockIdx.x;
    BkvTile t;
    if (!bkv_tile(a, tile, t) || t.one()) return;
    const int c = blockIdx.z * (256 / PT) + threadIdx.x / PT, d = (threadIdx.x % PT) * 4;
    if (c >= t.n) return;
    const size_t first = ((size_t)blockIdx.x * a.v.n_head + head) * a.splits * a.cols + c;
    const int cc = t.c0 + c, j = bkv_div(cc, a.g_inv);
    *(vk_f32x4*)(a.out + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD + d) =
        bkv_join<HD, false, 8>(a.part + first * 2, a.part + a.part_o, first * HD + d, (t.units + t.per - 1) / t.per,
                               a.cols, 1, 0);
}

template <int HD, int CODEC>
static void go_attn(hipStream_t s, const BkvAttnArgs& a, int tc, dim3 grid) {
    const uint8_t* pool = a.v.pool;
    const float2* sc = (const float2*)a.v.scales;
    if (tc == 16) hipLaunchKernelGGL((vk_bkv_attn<HD, CODEC, 1>), grid, dim3(64 * kWaves), 0, s, a, pool, sc);
    else if (tc == 32) hipLaunchKernelGGL((vk_bkv_attn<HD, CODEC, 2>), grid, dim3(64 * kWaves), 0, s, a, pool, sc);
    else hipLaunchKernelGGL((vk_bkv_attn_chunk<HD, CODEC>), grid, dim3(256), 0, s, a, pool, sc);
}

template <int HD>
static void go_hd(hipStream_t s, const BkvAttnArgs& a, int tc, dim3 grid) {
    if (a.v.codec == BKV_INT8) go_attn<HD, BKV_INT8>(s, a, tc, grid);
    else go_attn<HD, BKV_E4M3>(s, a, tc, grid);
    constexpr unsigned CW = 256 / (HD / 4);  // columns a joining workgroup
    const unsigned cols = ((unsigned)a.cols + CW - 1) / CW;
    if (tc == kChunkCols)
        hipLaunchKernelGGL(vk_bkv_attn_join<HD>, dim3(kBkvShares, cols), dim3(256), 0, s, a);
    else if (a.splits > 1 && tc != 16)
        hipLaunchKernelGGL(vk_bkv_attn_merge<HD>, dim3(grid.x, grid.y, cols), dim3(256), 0, s, a);
}

hipError_t launch_bkv_attn(hipStream_t s, const BkvView& v, int layer, int n, int n_rows, int max_count, int max_len,
                           int hq, const float* q, float scale, float* out, float* part) {
    if (n_rows == 0 || n == 0 || max_count == 0) return hipSuccess;
    BkvAttnArgs a = {};
    a.v = v;
    a.q = q;
    a.out = out;
    a.part = part;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.layer = layer;
    a.hq = hq;
    a.g = hq / v.n_head;
    a.n = n;
    a.rows = n_rows;
    a.count = max_count;
    const long long cols = (long long)max_count * a.g;
    const int units = std::max(1, (max_len + kUnit - 1) / kUnit);
    // Tiles of 32 columns an item, or shares of tiles of 128 where those are mostly full
    // and there is work enough for all shares, in units by such tiles: 16 heads over 2
    // of 128, one prompt of 1000 rows (16 thousand) takes 30 us so and 39 by shares, one
    // of 2000 (63 thousand) 71 and 64; 8 sequences of up to 4096 keys and 16 rows, 32
    // heads over 8, 31 and 45.
    const long long parts = (cols + 31) / 32;
    const bool few = cols <= 96 || (parts * n * v.n_head * units <= 48 << 10 && cols * a.g < 1ll << 32);
    // Of those, tiles of 16, which join in their own launch, while few keys are read twice
    // for it: 16 sequences of up to 3000 keys, 4 rows, 16 heads over 2 take 15.3 us so and
    // 18.5 in tiles of 32, one of 16000 keys, 8 rows, 32 heads over 8, 24.6 and 22.
    const int tc = cols <= 16 || (few && cols * units <= 6144) ? 16 : few ? 32 : kChunkCols;
    a.part_o = (size_t)kBkvParts * 2;
    a.joined = (unsigned*)(part + (size_t)kBkvParts * (128 + 2));
    a.open = (BkvOpen*)(a.joined + kBkvShares);
    auto inv = [](int d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + (uint32_t)d - 1) / (uint32_t)d); };
    a.g_inv = inv(a.g);
    // items of up to `count` rows in tiles of tc columns, 16 or 32
    auto ranges = [&](int count, int tc) {
        BkvAttnArgs b = a;
        b.count = count;
        const int cols = count * b.g;
        b.cols = std::min(cols, tc);
        b.parts = (cols + tc - 1) / tc;
        b.parts_inv = inv(b.parts);
        const int tiles = b.parts * n;
        // Units a key range: the call's units at the longest rows' length over 512, so
        // that there are ranges for every CU (six sequences of 9 .. 65 thousand keys take
        // 99 us, over 256 142; over 1024, 32 streams of up to 4096 take 22.5 us against
        // 17.6), and 8 at least (16: one sequence of 2000 keys takes 10.8 us against 8.8).
        const long long per = std::max<long long>((long long)tiles * v.n_head * units / 512, 8);
        // Ranges: a wave's units fall with their number, the join's rounds rise with it;
        // together least near the root of twice the units (one sequence of 32768 keys, 8
        // kv heads: 45 ranges 23.5 us, 64 28.6, 16 29.7; of 12000 keys, one kv head: 27
        // 12.9, 64 14.6).
        const long long most = std::max(8, (int)std::sqrt(2.0 * units));
        b.per = (int)((std::max(per, (units + most - 1) / most) + 3) / 4 * 4);
        b.splits = (units + b.per - 1) / b.per;
        b.splits_inv = inv(b.splits);
        // More than one range only where tiles * n_head < 512 (per >= units above), and
        // then fewer than 1100 ranges of up to 32 columns in all: the workspace holds them.
        static_assert(1100 * 32 <= kBkvParts && kBkvShares == 512, "");
        const dim3 grid((unsigned)tiles, (unsigned)v.n_head, (unsigned)b.splits);
        v.hd == 64 ? go_hd<64>(s, b, tc, grid) : go_hd<128>(s, b, tc, grid);
    };
    if (tc != kChunkCols) {
        ranges(max_count, tc);
        return hipGetLastError();
    }
    // Far fewer rows than items of the most have: single tokens beside a prompt's chunk,
    // which would each take a tile of 128 columns and go first where that is much (63
    // of 200 .. 3000 keys and a chunk of 1000, 32 heads over 8: 116 us against 140; 31 of
    // up to 4096 and one of 256, 16 heads over 2: 51 against 46, so not there).
    if ((long long)n_rows * 3 <= (long long)n * max_count && (long long)n * v.n_head * units > 16 << 10 && a.g <= 32) {
        a.done = (a.g <= 16 ? 16 : 32) / a.g;
        ranges(a.done, a.g <= 16 ? 16 : 32);
    }
    static_assert(2 * kBkvShares * kChunkCols <= kBkvParts && sizeof(BkvOpen) == 16, "");
    a.tiles = (int)((long long)n_rows * a.g / kChunkCols + n);
    a.cols = kChunkCols;
    v.hd == 64 ? go_hd<64>(s, a, tc, dim3(kBkvShares)) : go_hd<128>(s, a, tc, dim3(kBkvShares));
    return hipGetLastError();
}

}  // namespace vk
