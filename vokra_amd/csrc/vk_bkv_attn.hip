// vk_bkv_attn.hip — attention of a step's rows over the block-scaled KV cache.
//
// Row r of the step belongs to item i, at position p = start_i + (r - row0_i);
// query head h reads kv head h / G, G = hq / n_head:
//   s_j = scale q . k_j (j <= p), out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
// with k, v the values that the cache holds: 8-bit ones under their block's
// scale, f32 rows in the open block.
//
// Columns: the count_i * G query rows of an item that read one kv head. A
// workgroup takes up to 16 C of them over a range of keys; its four waves take
// the range's units of 32 keys in turn, each with an online softmax of its own,
// and merge through LDS at the end: no barrier in the key loop. The 8-bit values
// are exact in fp16, so a product is two fp16 matrix instructions, one for each
// part of the f32 operand (22 bits): q in two parts under a power of two that
// puts its row's largest value at 2^14, weights in two parts of 2^14 w.
//   S^T [keys][columns] = K q^T: K's 16-byte loads are operand registers but for
//     the widening (the pages hold tiles in that order);
//   P's accumulator layout (4 consecutive keys a lane) is the operand layout of
//     O^T [d][columns] = V^T P^T under the key order that V's tiles use, so the
//     weights go from the softmax to the product without leaving the lane.
// A block's V scale f 2^e (f in [1, 2)) goes into the weights: the running
// maximum is that of s + e, so the largest weight has the largest product, and a
// block of small values keeps its bits beside one of large values; the sum of
// weights takes 2^-e back out. Two fp16 parts of 2^14 w hold a weight to 2^-22,
// or to 2^-39 of the largest where it is smaller than 2^-17 of that. The open block's rows are f32 on both sides and
// use the f32 matrix instruction.
#include <algorithm>

#include "vk_bkv.h"
#include "vk_common.h"

namespace vk {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));

struct BkvAttnArgs {
    BkvView v;
    const float* q;
    float* out;
    float* part;        // [slot][cols][2] (max, sum), then [slot][cols][hd] partial outputs
    size_t part_o;      // floats before the partial outputs
    float scale_log2;   // scale * log2(e)
    int layer, hq, g;   // g = hq / n_head
    int tile0;          // first column tile of this launch
    int chunks;         // 0: one column tile an item (at most 16 C columns); 1: as many as its columns need
    int splits;         // key ranges a column tile may have (grid)
    int cols;           // columns a slot has room for
};

constexpr int kUnit = 32;  // keys of a wave's step: two 16-token tiles

// A column tile of an item: what its workgroups work on.
struct BkvTile {
    BkvItem it;
    int c0, n;      // first column, columns
    int keys;       // keys that its last row sees
    int full;       // keys in full blocks, no more than keys rounded up to a tile
    int units, per; // units of the 8-bit part, units a key range
    int ranges;     // key ranges (at least one)
};

// Tile T of the launch's order: item T, or the item whose tiles T is one of
// (item i's begin at row0_i * g / tc + i: room for a partly filled tile each).
// Every thread returns the same; false: no such tile. sh: one int of LDS.
__device__ __forceinline__ bool bkv_tile(const BkvAttnArgs& a, int tile, int tc, int* sh, BkvTile& t) {
    const int n = a.v.meta[BKV_STEP_N];
    int i = tile, k = 0;
    if (a.chunks) {
        if (threadIdx.x == 0) *sh = -1;
        __syncthreads();
        for (int x = threadIdx.x; x < n; x += blockDim.x) {
            const BkvItem it = a.v.step[x];
            const long long lo = (long long)it.row0 * a.g / tc + x;
            const long long hi = (long long)(it.row0 + it.count) * a.g / tc + x + 1;
            if (tile >= lo && tile < hi) *sh = x;
        }
        __syncthreads();
        i = *sh;
        if (i < 0) return false;
        t.it = a.v.step[i];
        k = tile - (int)((long long)t.it.row0 * a.g / tc + i);
    } else {
        if (i >= n) return false;
        t.it = a.v.step[i];
    }
    const int cols = t.it.count * a.g;
    t.c0 = k * tc;
    t.n = min(tc, cols - t.c0);
    if (t.n <= 0) return false;
    t.keys = t.it.start + (t.c0 + t.n - 1) / a.g + 1;
    t.full = min((t.it.start + t.it.count) / a.v.bs * a.v.bs, (t.keys + 15) & ~15);
    t.units = (t.full + kUnit - 1) / kUnit;
    t.per = max(8, ((t.units + a.splits - 1) / a.splits + 3) & ~3);
    t.ranges = max(1, (t.units + t.per - 1) / t.per);
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

__device__ __forceinline__ uint32_t u4c(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// hi = fp16(x), lo = fp16(x - hi) of two values
__device__ __forceinline__ void bkv_split2(float x, float y, half2v& hi, half2v& lo) {
    const float2v v = {x, y};
    hi = __builtin_convertvector(v, half2v);
    const float2v r = {fmaf((float)hi.x, -1.0f, x), fmaf((float)hi.y, -1.0f, y)};
    lo = __builtin_convertvector(r, half2v);
}

// sum / max over the four lane groups (lanes l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float bkv_max4(float v) {
    v = fmaxf(v, __int_as_float(vk_bfly_partner<16>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(vk_bfly_partner<32>(__float_as_int(v))));
}
__device__ __forceinline__ float bkv_sum4(float v) {
    v += __int_as_float(vk_bfly_partner<16>(__float_as_int(v)));
    return v + __int_as_float(vk_bfly_partner<32>(__float_as_int(v)));
}

template <int HD, int CODEC, int C>
__global__ __launch_bounds__(256, 2) void vk_bkv_attn(BkvAttnArgs a, const uint8_t* __restrict__ pool,
                                                      const float2* __restrict__ scales) {
    constexpr int U = HD / 64, DT = HD / 16, OS = HD + 4;
    constexpr bool QL = C > 1;  // q's parts in LDS (shared by the waves), else in registers
    __shared__ uint4 sq[QL ? C * U * 4 * 64 : 1];
    __shared__ float sqf[C * 16];  // q's factor of each column
    __shared__ float so[4][16][OS];
    __shared__ float2 sml[4][16];
    __shared__ int sh;
    const int split = blockIdx.x % a.splits, head = blockIdx.y;
    const int tile = a.tile0 + (int)(blockIdx.x / a.splits);
    BkvTile t;
    if (!bkv_tile(a, tile, 16 * C, &sh, t) || split >= t.ranges) return;
    const BkvView& v = a.v;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4, bs_log = 31 - __clz(v.bs);

    // this wave's units: u0, u0 + 4, .. below u1
    const int u0 = split * t.per + wave, u1 = min(t.units, (split + 1) * t.per);
    const int* table = v.table + (size_t)t.it.seq * v.max_blocks;
    // lane l holds the page of tile l & 1 of the wave's unit k0 + l / 2
    auto pages_from = [&](int k0) {
        const int u = min(u0 + 4 * (k0 + (lane >> 1)), t.units - 1);
        const int key = min(u * kUnit + (lane & 1) * 16, t.full - 16);
        return table[key >> bs_log];
    };
    int pages = 0;
    if (u0 < u1) pages = pages_from(0);

    // q's parts: lane's 16 values d = 64 u + 16 grp .. of column `col`, two k steps of 8
    half8v qh[QL ? 1 : 2 * U], ql[QL ? 1 : 2 * U];
    auto load_q = [&](int ct, half8v* h8, half8v* l8) {
        const int c = ct * 16 + col;
        const bool live = c < t.n;
        const int cc = t.c0 + (live ? c : 0), j = cc / a.g;
        const float* p = a.q + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD + grp * 16;
        float4 x[4 * U];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) {
            x[i] = *(const float4*)(p + (i >> 2) * 64 + (i & 3) * 4);
            if (!live) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        }
        top = bkv_max4(top);
        // the largest value goes to 2^14 .. 2^15; rows below 2^-106 keep fewer bits
        const int e = min(141 - (int)(__float_as_uint(top) >> 23), 120);
        const float up = __uint_as_float((uint32_t)(127 + e) << 23), down = __uint_as_float((uint32_t)(127 - e) << 23);
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
        return a.scale_log2 * down;
    };
    float qf[C];
    if constexpr (QL) {
        for (int ct = wave; ct < C; ct += 4) {
            half8v h8[2 * U], l8[2 * U];
            const float f = load_q(ct, h8, l8);
            if (grp == 0) sqf[ct * 16 + col] = f;
#pragma unroll
            for (int i = 0; i < 2 * U; ++i) {
                sq[((ct * 2 * U + i) * 2 + 0) * 64 + lane] = __builtin_bit_cast(uint4, h8[i]);
                sq[((ct * 2 * U + i) * 2 + 1) * 64 + lane] = __builtin_bit_cast(uint4, l8[i]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int ct = 0; ct < C; ++ct) qf[ct] = sqf[ct * 16 + col];
    } else {
        qf[0] = load_q(0, qh, ql);
    }
    // last key that each of this lane's columns sees
    int last[C];
#pragma unroll
    for (int ct = 0; ct < C; ++ct) last[ct] = t.it.start + (t.c0 + ct * 16 + col) / a.g;
    const int first_last = t.it.start + t.c0 / a.g;  // the least of them

    float M[C], L[C];
    vk_f32x4 O[C][DT];
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
        M[ct] = -INFINITY;
        L[ct] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) O[ct][d] = vk_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // the running maximum of a column becomes m; what was summed so far shrinks
    auto raise = [&](int ct, float m) {
        if (__any(m > M[ct])) {
            const float to = fmaxf(M[ct], m), c = M[ct] == -INFINITY ? 0.0f : exp2f(M[ct] - to);
            M[ct] = to;
            L[ct] *= c;
#pragma unroll
            for (int d = 0; d < DT; ++d) O[ct][d] *= c;
        }
    };

    const size_t layer_page = (size_t)a.layer * v.n_page;
    uint4 kr[2][U], vr[2][U];
    float2 sc[2];
    const uint8_t *kp[2], *vp[2];
    auto at = [&](int u, int k) {  // addresses of unit u, the k-th of this wave
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int page = __builtin_amdgcn_readlane(pages, 2 * (k & 31) + x);
            const int key = min(u * kUnit + x * 16, t.full - 16);
            const size_t chunk = (layer_page + page) * v.n_head + head;
            kp[x] = pool + chunk * 2 * v.bs * HD + (size_t)((key & (v.bs - 1)) >> 4) * 16 * HD + lane * 16;
            vp[x] = kp[x] + (size_t)v.bs * HD;
            sc[x] = scales[chunk];
        }
    };
    auto load = [&](uint4 (&r)[2][U], const uint8_t* const (&p)[2]) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int u = 0; u < U; ++u) r[x][u] = *(const uint4*)(p[x] + u * 1024);
    };
    if (u0 < u1) {
        at(u0, 0);
        load(kr, kp);
        load(vr, vp);
    }
    for (int u = u0, k = 0; u < u1; u += 4, ++k) {
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
                half8v h8, l8;
                if constexpr (QL) {
                    h8 = __builtin_bit_cast(half8v, sq[((ct * 2 * U + i) * 2 + 0) * 64 + lane]);
                    l8 = __builtin_bit_cast(half8v, sq[((ct * 2 * U + i) * 2 + 1) * 64 + lane]);
                } else {
                    h8 = qh[i];
                    l8 = ql[i];
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], l8, S[ct][x], 0, 0, 0);
                    S[ct][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[x], h8, S[ct][x], 0, 0, 0);
                }
            }
        }
        float ks[2], vf[2], ve[2], back[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            ks[x] = sc[x].x;
            const uint32_t b = __float_as_uint(sc[x].y);
            const int e = (int)((b >> 23) & 255);
            const bool plain = e != 0 && e != 255;  // zero: f 0, e 0; not finite: f NaN, e 0
            vf[x] = plain ? __uint_as_float((b & 0x007fffffu) | 0x46800000u) : sc[x].y;  // f 2^14
            ve[x] = plain ? (float)(e - 127) : 0.0f;
            back[x] = plain ? __uint_as_float((uint32_t)min(254 - e, 253) << 23) : 1.0f;  // 2^-e
        }
        const bool more = u + 4 < u1;
        if (more) {
            if (((k + 1) & 31) == 0) pages = pages_from(k + 1);
            at(u + 4, k + 1);
            load(kr, kp);
        }
        const bool hide = u * kUnit + kUnit > min(first_last + 1, t.full);
        half8v ph[C], pl[C];
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            float s[8];
            float m = -INFINITY;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float f = ks[x] * qf[ct];
#pragma unroll
                for (int r = 0; r < 4; ++r) s[4 * x + r] = fmaf(S[ct][x][r], f, ve[x]);
            }
            if (hide) {
                const int lim = min(last[ct] + 1, t.full);
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (u * kUnit + (r >> 2) * 16 + grp * 4 + (r & 3) >= lim) s[r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 8; ++r) m = fmaxf(m, s[r]);
            raise(ct, bkv_max4(m));
            const float base = M[ct] == -INFINITY ? 0.0f : M[ct];
            float w[8];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(s[4 * x + r] - base);
                    sum += e;
                    w[4 * x + r] = e * vf[x];
                }
                L[ct] = fmaf(sum, back[x], L[ct]);
            }
            if (hide) {  // a hidden key has no part in a block whose scale is NaN
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (s[r] == -INFINITY) w[r] = 0.0f;
            }
            half2v h[4], l[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) bkv_split2(w[2 * r], w[2 * r + 1], h[r], l[r]);
            ph[ct] = half8v{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
            pl[ct] = half8v{l[0].x, l[0].y, l[1].x, l[1].y, l[2].x, l[2].y, l[3].x, l[3].y};
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const half8v va = bkv_widen8<CODEC>(u4c(vr[0][d >> 2], d & 3), u4c(vr[1][d >> 2], d & 3));
#pragma unroll
            for (int ct = 0; ct < C; ++ct) {
                O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[ct], O[ct][d], 0, 0, 0);
                O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[ct], O[ct][d], 0, 0, 0);
            }
        }
        if (more) load(vr, vp);
    }

    // the open block's rows: tile `wave` of them, in the last key range
    const int key0 = t.full + wave * 16;
    if (split == t.ranges - 1 && key0 < t.keys) {
        const size_t side = (size_t)v.n_head * 2 * v.bs * HD;
        const float* ring = v.ring + ((size_t)a.layer * v.n_seq + t.it.seq) * 2 * side + (size_t)head * 2 * v.bs * HD;
        const int ring_mask = 2 * v.bs - 1;
        const float* kp1 = ring + (size_t)((key0 + col) & ring_mask) * HD + grp * 4;
        const float* vring = ring + side;
        // V: four rows (keys 4 grp + r), column 16 d + col; rows that no column sees are not used
        float vv[DT][4];
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = key0 + grp * 4 + r;
            const float* p = vring + (size_t)(key & ring_mask) * HD + col;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const float y = p[16 * d];
                vv[d][r] = key < t.keys ? y : 0.0f;
                odd = odd || !(fabsf(vv[d][r]) < INFINITY);
            }
        }
        const bool any_odd = __any(odd);
        // a power of two in the place of a block's scale, so that the maximum
        // weighs these rows like the blocks: the largest |v| is 2^9 .. 2^10 of it
        float top = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(vv[d][r]));
        top = vk_group_max<64>(any_odd ? 0.0f : top);
        const int te = top < 0x1p-100f ? 0 : (int)(__float_as_uint(top) >> 23) - 136;
        const float tdown = __uint_as_float((uint32_t)(127 - te) << 23);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) vv[d][r] *= tdown;
#pragma unroll
        for (int ct = 0; ct < C; ++ct) {
            const int c = ct * 16 + col;
            const int cc = t.c0 + (c < t.n ? c : 0), j = cc / a.g;
            const float* p = a.q + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD + grp * 4;
            vk_f32x4 s4 = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                const float4 x = *(const float4*)(kp1 + 16 * i), y = *(const float4*)(p + 16 * i);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, y.x, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, y.y, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, y.z, s4, 0, 0, 0);
                s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, y.w, s4, 0, 0, 0);
            }
            float s[4], m = -INFINITY;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[r] = key0 + grp * 4 + r <= last[ct] ? fmaf(s4[r], a.scale_log2, (float)te) : -INFINITY;
                m = fmaxf(m, s[r]);
            }
            raise(ct, bkv_max4(m));
            const float base = M[ct] == -INFINITY ? 0.0f : M[ct];
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                e[r] = __builtin_amdgcn_exp2f(s[r] - base);
                L[ct] = fmaf(e[r], tdown, L[ct]);
                e[r] *= 16384.0f;
            }
            if (!any_odd) {
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        O[ct][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[d][r], e[r], O[ct][d], 0, 0, 0);
            } else {
                // a value that is not finite: only the columns that see its key take it
                for (int x = 0; x < 16 && key0 + x < t.keys; ++x) {
                    float w = 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((x & 3) == r) w = __shfl(e[r], (x >> 2) * 16 + col, VK_WAVE);
                    const float* p1 = vring + (size_t)((key0 + x) & ring_mask) * HD + grp * 4;
                    if (key0 + x <= last[ct]) {
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            const float4 y = *(const float4*)(p1 + 16 * d);
                            O[ct][d][0] = fmaf(w, y.x, O[ct][d][0]);
                            O[ct][d][1] = fmaf(w, y.y, O[ct][d][1]);
                            O[ct][d][2] = fmaf(w, y.z, O[ct][d][2]);
                            O[ct][d][3] = fmaf(w, y.w, O[ct][d][3]);
                        }
                    }
                }
            }
        }
    }

    // the four waves' results of each 16 columns, merged by all threads
    const bool direct = t.ranges == 1;
    const size_t slot = ((size_t)(tile - a.tile0) * v.n_head + head) * a.splits + split;
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
        if (ct * 16 >= t.n) break;
        const float l = bkv_sum4(L[ct]);
        if (ct > 0) __syncthreads();
        if (grp == 0) sml[wave][col] = make_float2(M[ct], l);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            *(vk_f32x4*)&so[wave][col][16 * d + 4 * grp] = O[ct][d];
        __syncthreads();
        constexpr int PER = HD / 16;  // values a thread: 16 threads a column
        const int c = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 4;
        if (ct * 16 + c < t.n) {
            float m = -INFINITY, sum = 0.0f, w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) m = fmaxf(m, sml[x][c].x);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                w[x] = sml[x][c].x == -INFINITY && sml[x][c].y == 0.0f ? 0.0f
                       : m == -INFINITY ? 1.0f : exp2f(sml[x][c].x - m);
                sum = fmaf(sml[x][c].y, w[x], sum);
            }
            const int cc = t.c0 + ct * 16 + c, j = cc / a.g;
            float* dst = direct ? a.out + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD
                                : a.part + a.part_o + (slot * a.cols + ct * 16 + c) * HD;
            const float f = direct ? 0x1p-14f / sum : 0x1p-14f;
            if (!direct && d0 == 0) ((float2*)a.part)[slot * a.cols + ct * 16 + c] = make_float2(m, sum);
#pragma unroll
            for (int b = 0; b < PER / 4; ++b) {
                const int d = d0 + 64 * b;
                vk_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (w[x] != 0.0f) y += *(const vk_f32x4*)&so[x][c][d] * w[x];
                *(vk_f32x4*)(dst + d) = y * f;
            }
        }
    }
}

// The key ranges of a column tile, merged in their order: 16 threads a column
// (HD = 64) or 32 (128).
template <int HD>
__global__ __launch_bounds__(256) void vk_bkv_attn_merge(BkvAttnArgs a, int tc) {
    __shared__ int sh;
    const int head = blockIdx.y, tile = a.tile0 + (int)blockIdx.x;
    BkvTile t;
    if (!bkv_tile(a, tile, tc, &sh, t) || t.ranges == 1) return;
    constexpr int PT = HD / 4;
    const size_t slot = ((size_t)blockIdx.x * a.v.n_head + head) * a.splits;
    for (int c = threadIdx.x / PT; c < t.n; c += 256 / PT) {
        const int d = (threadIdx.x % PT) * 4;
        float m = -INFINITY;
        for (int s = 0; s < t.ranges; ++s) m = fmaxf(m, ((const float2*)a.part)[(slot + s) * a.cols + c].x);
        float sum = 0.0f;
        vk_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < t.ranges; ++s) {
            const float2 ml = ((const float2*)a.part)[(slot + s) * a.cols + c];
            if (ml.x == -INFINITY && ml.y == 0.0f) continue;
            const float w = m == -INFINITY ? 1.0f : exp2f(ml.x - m);
            sum = fmaf(ml.y, w, sum);
            y += *(const vk_f32x4*)(a.part + a.part_o + ((slot + s) * a.cols + c) * HD + d) * w;
        }
        const int cc = t.c0 + c, j = cc / a.g;
        *(vk_f32x4*)(a.out + ((size_t)(t.it.row0 + j) * a.hq + head * a.g + (cc - j * a.g)) * HD + d) = y * (1.0f / sum);
    }
}

template <int HD, int CODEC>
static void go_attn(hipStream_t s, const BkvAttnArgs& a, int c, dim3 grid) {
    const uint8_t* pool = a.v.pool;
    const float2* sc = (const float2*)a.v.scales;
    if (c == 1) hipLaunchKernelGGL((vk_bkv_attn<HD, CODEC, 1>), grid, dim3(256), 0, s, a, pool, sc);
    else if (c == 2) hipLaunchKernelGGL((vk_bkv_attn<HD, CODEC, 2>), grid, dim3(256), 0, s, a, pool, sc);
    else hipLaunchKernelGGL((vk_bkv_attn<HD, CODEC, 4>), grid, dim3(256), 0, s, a, pool, sc);
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
    const long long cols = (long long)max_count * a.g;
    const int c = cols <= 16 ? 1 : cols <= 32 ? 2 : 4, tc = 16 * c;
    a.chunks = cols > tc;
    a.cols = a.chunks ? tc : (int)cols;
    const long long tiles = a.chunks ? (long long)n_rows * a.g / tc + n : n;
    // Key ranges of 256 keys and more, at most 64 a tile and what the workspace
    // has room for. For tiles of whole items the number does not depend on the
    // batch, so an item's rows come out the same in any batch.
    const int room = kBkvMaxParts * 16;
    const int units = (max_len + kUnit - 1) / kUnit;
    long long most = std::min<long long>(64, std::max<long long>(1, room / ((long long)v.n_head * a.cols)));
    if (a.chunks) most = std::min<long long>(most, std::max<long long>(1, 512 / (tiles * v.n_head)));
    a.splits = (int)std::min<long long>(most, std::max(1, (units + 7) / 8));
    a.part_o = (size_t)room * 2;
    // tiles a launch: what the workspace holds, and fewer than 2^24 workgroups
    const long long step = a.splits == 1 ? 1 << 20
                                         : std::max<long long>(1, room / ((long long)v.n_head * a.cols * a.splits));
    for (long long t0 = 0; t0 < tiles; t0 += step) {
        const long long now = std::min(step, tiles - t0);
        a.tile0 = (int)t0;
        const dim3 grid((unsigned)(now * a.splits), (unsigned)v.n_head);
        if (v.hd == 64) {
            if (v.codec == BKV_INT8) go_attn<64, BKV_INT8>(s, a, c, grid);
            else go_attn<64, BKV_E4M3>(s, a, c, grid);
            if (a.splits > 1)
                hipLaunchKernelGGL(vk_bkv_attn_merge<64>, dim3((unsigned)now, (unsigned)v.n_head), dim3(256), 0, s, a, tc);
        } else {
            if (v.codec == BKV_INT8) go_attn<128, BKV_INT8>(s, a, c, grid);
            else go_attn<128, BKV_E4M3>(s, a, c, grid);
            if (a.splits > 1)
                hipLaunchKernelGGL(vk_bkv_attn_merge<128>, dim3((unsigned)now, (unsigned)v.n_head), dim3(256), 0, s, a, tc);
        }
    }
    return hipGetLastError();
}

}  // namespace vk
