// vk_bkv.hip — the block-scaled KV cache for gfx950: planning (pages, lengths,
// steps), the write of rows, reading back, and the moving of pages.
//
// A page holds one block of bs tokens of one sequence, for every layer, head
// and side (K, V), in 8 bits under one f32 scale per (layer, head, side):
//   a = max |x| over the block (bs x hd values),
//   int8: scale a / 127, value rint(x * (127 / a));
//   e4m3: scale a / 448, value e4m3(x * (448 / a)),
// each operation an f32 operation rounded once, ties to even. a < 2^-100 holds
// zeros under scale 0 (127 / a would leave f32's range for the smallest a); a
// block with a value that is not finite holds zeros under a NaN scale, so it
// reads as NaN.
//
// Only a full block is rounded: the rows of the block that is still open stay
// as they came (f32, in the ring of the sequence's last two blocks). So every
// value is rounded once, by the largest value of its own block, and what the
// cache holds does not depend on how the rows were split over calls; a page
// never changes once it is written, so sequences may share it, and a fork
// copies one row of the page table and the open block's rows.
//
// Planning is one workgroup (items are at most 1024, one thread each): checks,
// prefix sums over what they take, pages from a bitmap (lowest first, so the
// result does not depend on the order of earlier frees). The
// first item that fails ends the call; the ones before it stay done.
#include <algorithm>
#include <climits>

#include "../../include/vokra_hip.h"
#include "vk_bkv.h"
#include "vk_common.h"

namespace vk {

constexpr int BKV_TPB = 1024;  // threads of the planning kernels at most

// ---- workgroup prefix sums ----------------------------------------------------

// Exclusive prefix sums of N numbers a thread over the workgroup, in place;
// totals in sum. red: N ints a wave.
template <int N>
__device__ __forceinline__ void bkv_scan(int (&v)[N], int (&sum)[N], int* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
    int x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        x[j] = v[j];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x[j], o, VK_WAVE);
            if (lane >= o) x[j] += y;
        }
    }
    __syncthreads();
    if (lane == 63)
#pragma unroll
        for (int j = 0; j < N; ++j) red[wave * N + j] = x[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        int before = 0, all = 0;
        for (int w = 0; w < waves; ++w) {
            const int t = red[w * N + j];
            if (w < wave) before += t;
            all += t;
        }
        v[j] = before + x[j] - v[j];
        sum[j] = all;
    }
}

// The last index i in [0, n) with off[i] <= k (off ascending, off[0] = 0).
__device__ __forceinline__ int bkv_find(const int* off, int n, int k) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off[mid] <= k) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Takes the `want` lowest free pages (want <= free pages) into v.fresh,
// ascending, and marks them used. Words from the hint on are searched, one a
// thread and round; the caller has checked that enough are free.
__device__ void bkv_take(const BkvView& v, int want, int* red) {
    const int words = (v.n_page + 31) / 32;
    int base = v.meta[BKV_HINT], got = 0, last = base;
    while (got < want && base < words) {
        const int w = base + (int)threadIdx.x;
        uint32_t avail = w < words ? ~v.used[w] : 0u;
        if (w == words - 1 && (v.n_page & 31)) avail &= (1u << (v.n_page & 31)) - 1u;
        int n[1] = {(int)__popc(avail)}, total[1];
        bkv_scan(n, total, red);
        int at = got + n[0];
        uint32_t taken = 0;
        while (avail && at < want) {
            const int b = __ffs(avail) - 1;
            v.fresh[at++] = w * 32 + b;
            taken |= 1u << b;
            avail &= avail - 1;
        }
        if (taken) v.used[w] |= taken;
        got += total[0];
        last = base;
        base += (int)blockDim.x;
    }
    __syncthreads();
    // every word before the last round's first is full now
    if (threadIdx.x == 0 && want > 0) v.meta[BKV_HINT] = last;
    __syncthreads();
}

// Drops one holder of a page; the last one frees it.
__device__ __forceinline__ void bkv_drop(const BkvView& v, int page) {
    if ((unsigned)page >= (unsigned)v.n_page) return;
    if (atomicSub(&v.refs[page], 1) == 1) {
        atomicAnd(&v.used[page >> 5], ~(1u << (page & 31)));
        atomicAdd(&v.meta[BKV_FREE], 1);
        atomicMin(&v.meta[BKV_HINT], page >> 5);
    }
}

// ---- reset -------------------------------------------------------------------

__global__ void vk_bkv_reset(BkvView v) {
    const size_t i0 = (size_t)blockIdx.x * blockDim.x + threadIdx.x, step = (size_t)gridDim.x * blockDim.x;
    for (size_t i = i0; i < (size_t)v.n_seq * v.max_blocks; i += step) v.table[i] = -1;
    for (size_t i = i0; i < (size_t)v.n_seq; i += step) {
        v.len[i] = 0;
        v.floor_[i] = 0;
    }
    for (size_t i = i0; i < (size_t)v.n_page; i += step) v.refs[i] = 0;
    for (size_t i = i0; i < (size_t)(v.n_page + 31) / 32; i += step) v.used[i] = 0;
    for (size_t i = i0; i < (size_t)kBkvMaxItems; i += step) v.step[i] = BkvItem{0, 0, 0, 0};
    if (i0 < BKV_META_INTS) v.meta[i0] = i0 == BKV_FREE ? v.n_page : 0;
}

__global__ void vk_bkv_fill(uint4* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x)
        p[i] = make_uint4(0, 0, 0, 0);
}

// ---- step --------------------------------------------------------------------

// Whether an item before i names id, and whether any of the n items does
// (ids in LDS, 16-byte aligned, those beyond n negative).
__device__ __forceinline__ void bkv_named(const int* ids, int n, int i, int id, bool* before, bool* any) {
    *before = *any = false;
    for (int j = 0; j < n; j += 4) {
        const int4 x = *(const int4*)(ids + j);
        const bool m[4] = {x.x == id, x.y == id, x.z == id, x.w == id};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            *any = *any || m[c];
            *before = *before || (m[c] && j + c < i);
        }
    }
}

// One thread an item; about five trips to memory, whatever the items are.
__global__ __launch_bounds__(BKV_TPB) void vk_bkv_step(BkvView v, int n, int n_rows, int max_count,
                                                       const int* __restrict__ seqs, const int* __restrict__ starts,
                                                       const int* __restrict__ counts) {
    __shared__ int red[3 * (BKV_TPB / 64)];
    __shared__ __align__(16) int s_seq[BKV_TPB];
    __shared__ int s_page[BKV_TPB + 1], s_work[BKV_TPB + 1];  // prefixes: pages taken, blocks reached
    __shared__ BkvItem s_item[BKV_TPB];
    __shared__ int s_bad, s_done;
    const int i = threadIdx.x, bs_log = 31 - __clz(v.bs);
    const int seq = i < n ? seqs[i] : -1, start = i < n ? starts[i] : 0, count = i < n ? counts[i] : 0;
    const int free_pages = v.meta[BKV_FREE];
    const bool in_range = (unsigned)seq < (unsigned)v.n_seq;
    const int len = in_range ? v.len[seq] : 0, fl = in_range ? v.floor_[seq] : 0;
    s_seq[i] = seq;
    if (i == 0) s_bad = s_done = n;
    __syncthreads();
    bool named, any;
    bkv_named(s_seq, n, i, seq, &named, &any);
    bool ok = in_range && !named && count >= 0 && count <= max_count && start >= fl && start <= len &&
              count <= v.max_time - start;
    // rows; pages: of the blocks that the step's rows fill; blocks that they reach
    const int cnt = ok ? count : 0, b0 = start >> bs_log, b1 = ok ? (start + cnt) >> bs_log : b0;
    const int need = b1 - b0;
    int at[3] = {cnt, need, cnt > 0 ? ((start + cnt - 1) >> bs_log) - b0 + 1 : 0}, sum[3];
    bkv_scan(at, sum, red);
    // up to the first item that fails, the prefixes hold no item that does
    if (at[0] + cnt > n_rows) ok = false;
    if (i < n && !ok) atomicMin(&s_bad, i);
    __syncthreads();
    const int bad = s_bad;
    if (i < bad && need > 0 && at[1] + need > free_pages) atomicMin(&s_done, i);
    s_item[i] = BkvItem{seq, start, cnt, at[0]};
    s_page[i] = at[1];
    s_work[i] = at[2];
    if (i + 1 == (int)blockDim.x) {
        s_page[i + 1] = sum[1];
        s_work[i + 1] = sum[2];
    }
    __syncthreads();
    const int done = min(s_done, bad), total = s_page[done], n_work = min(s_work[done], v.max_work);
    if (total) bkv_take(v, total, red);
    if (i < done) {
        // pages that a taken-back sequence held from its new start on
        for (int b = b0; b < len >> bs_log; ++b) {
            int* e = v.table + (size_t)seq * v.max_blocks + b;
            bkv_drop(v, *e);
            if (b >= b1) *e = -1;
        }
        const int end = start + cnt, nb = (end + v.bs - 1) >> bs_log;
        v.len[seq] = end;
        v.floor_[seq] = max(fl, (nb - 2) * v.bs);
    }
    __syncthreads();  // an entry's old page is read before its new one is there
    for (int k = i; k < total; k += (int)blockDim.x) {
        const int it = bkv_find(s_page, done, k), page = v.fresh[k];
        v.table[(size_t)s_item[it].seq * v.max_blocks + (s_item[it].start >> bs_log) + (k - s_page[it])] = page;
        v.refs[page] = 1;
    }
    for (int k = i; k < n_work; k += (int)blockDim.x) {
        const int it = bkv_find(s_work, done, k), b = k - s_work[it];
        const BkvItem m = s_item[it];
        BkvWork e;
        e.seq = m.seq;
        e.start = m.start;
        e.end = m.start + m.count;
        e.row0 = m.row0;
        e.block = (m.start >> bs_log) + b;
        e.page = (e.block + 1) * v.bs <= e.end ? v.fresh[s_page[it] + b] : -1;
        e.pad[0] = e.pad[1] = 0;
        v.work[k] = e;
    }
    for (int k = i; k < kBkvMaxItems; k += (int)blockDim.x)
        v.step[k] = k < done ? s_item[k] : BkvItem{0, 0, 0, 0};  // no rows beyond the items done
    if (i == 0) {
        atomicSub(&v.meta[BKV_FREE], total);
        v.meta[BKV_STATUS] = done == n    ? VOKRA_HIP_OK
                             : done < bad ? VOKRA_HIP_ERROR_KV_CACHE_EXHAUSTED
                                          : VOKRA_HIP_ERROR_INVALID_ARGUMENT;
        v.meta[BKV_DONE] = done;
        v.meta[BKV_STEP_N] = done;
        v.meta[BKV_WORK_N] = n_work;
    }
}

// ---- write -------------------------------------------------------------------

// f32 -> e4m3 (OCP: 4 exponent bits, 3 mantissa bits, largest 448) with
// round-to-nearest-even of |y| < 464; two values, low byte first.
__device__ __forceinline__ uint32_t bkv_e4m3_pk(float a, float b) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}
__device__ __forceinline__ float bkv_e4m3_f32(uint32_t byte) {
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}
// The stored byte of y = x * (top / a): int8 values are stored with 128 added,
// so that a byte is the low mantissa bits of an f16 in 1024 .. 1279.
template <int CODEC>
__device__ __forceinline__ uint32_t bkv_encode4(float a, float b, float c, float d) {
    if constexpr (CODEC == BKV_INT8) {
        const int ia = (int)rintf(a) + 128, ib = (int)rintf(b) + 128;
        const int ic = (int)rintf(c) + 128, id = (int)rintf(d) + 128;
        return (uint32_t)ia | ((uint32_t)ib << 8) | ((uint32_t)ic << 16) | ((uint32_t)id << 24);
    } else {
        return bkv_e4m3_pk(a, b) | (bkv_e4m3_pk(c, d) << 16);
    }
}

__device__ __forceinline__ size_t bkv_chunk(const BkvView& v, int layer, int page, int head) {
    return (((size_t)layer * v.n_page + page) * v.n_head + head);
}
__device__ __forceinline__ float* bkv_ring(const BkvView& v, int layer, int seq, int side, int head) {
    return v.ring + ((((size_t)layer * v.n_seq + seq) * 2 + side) * v.n_head + head) * (size_t)(2 * v.bs) * v.hd;
}

// One wave for each block that the step reaches, head and side. If the step
// fills the block, the wave holds it in registers (NT pieces of 16 tokens by 64
// values, 16 values a lane, in the order that the pool stores them: a lane's 16
// bytes of a piece are its own), finds its largest magnitude and stores it
// rounded: one read, one write, no LDS. The wave of the item's first block also
// puts the rows of the item's last two blocks into the ring; it alone reads ring
// rows (those that earlier steps brought), before it writes any, so no two waves
// meet there. Bound by memory, 5 bytes a value: 17.7 thousand rows of 8 heads of 128
// (K and V, blocks of 32) take 48 us, 3.8 TB/s; 64 rows take 4.4 us, which is the
// launch and three dependent rounds of memory.
template <int CODEC, int NT>
__global__ __launch_bounds__(256) void vk_bkv_write(BkvView v, int layer, int n_rows, unsigned wg0,
                                                    const float* __restrict__ k, const float* __restrict__ vv) {
    const int n_work = v.meta[BKV_WORK_N], hs = 2 * v.n_head;
    const long long unit = ((long long)wg0 + blockIdx.x) * 4 + (threadIdx.x >> 6);
    const int entry = __builtin_amdgcn_readfirstlane((int)(unit / hs));
    if (entry >= n_work) return;
    const int sub = __builtin_amdgcn_readfirstlane((int)(unit - (long long)entry * hs));
    const BkvWork e = v.work[entry];
    if (e.row0 + (e.end - e.start) > n_rows) return;  // a later step, met by a captured write
    const int side = sub & 1, head = sub >> 1, lane = threadIdx.x & 63, hd = v.hd, bs = v.bs;
    const size_t rs = (size_t)v.n_head * hd;  // floats from row to row
    const float* in = (side ? vv : k) + (size_t)e.row0 * rs + (size_t)head * hd;
    float* ring = bkv_ring(v, layer, e.seq, side, head);
    const int mask = 2 * bs - 1;
    if (e.page >= 0) {
        const int pieces = hd >> 6;  // of a tile
        float x[NT][16];
#pragma unroll
        for (int p = 0; p < NT; ++p) {
            const int t0 = e.block * bs + p / pieces * 16, d0 = p % pieces * 64;
            if (side == 0) {  // token lane % 16, values 4 (lane / 16) .. + 0, 16, 32, 48
                const int t = t0 + (lane & 15), d = d0 + (lane >> 4) * 4;
                const float* r = t >= e.start ? in + (size_t)(t - e.start) * rs + d
                                              : ring + (size_t)(t & mask) * hd + d;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 y = *(const float4*)(r + 16 * j);
                    x[p][4 * j] = y.x, x[p][4 * j + 1] = y.y, x[p][4 * j + 2] = y.z, x[p][4 * j + 3] = y.w;
                }
            } else {  // tokens 4 (lane / 16) .., values 4 (lane % 16) ..
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = t0 + (lane >> 4) * 4 + j, d = d0 + (lane & 15) * 4;
                    const float4 y = *(const float4*)(t >= e.start ? in + (size_t)(t - e.start) * rs + d
                                                                   : ring + (size_t)(t & mask) * hd + d);
                    x[p][j] = y.x, x[p][4 + j] = y.y, x[p][8 + j] = y.z, x[p][12 + j] = y.w;
                }
            }
        }
        float amax = 0.0f;
        bool odd = false;  // a value that is not finite
#pragma unroll
        for (int p = 0; p < NT; ++p)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float m = fabsf(x[p][i]);
                amax = fmaxf(amax, m);
                odd = odd || !(m < INFINITY);
            }
        amax = vk_group_max<64>(odd ? INFINITY : amax);
        const float top = CODEC == BKV_INT8 ? 127.0f : 448.0f;
        const bool holds = amax >= 0x1p-100f && amax < INFINITY;
        const float inv = holds ? top / amax : 0.0f;
        const float scale = holds ? amax / top : (amax < INFINITY ? 0.0f : __builtin_nanf(""));
        const size_t chunk = bkv_chunk(v, layer, e.page, head);
        uint4* out = (uint4*)(v.pool + (chunk * 2 + side) * bs * hd);
        if (lane == 0) v.scales[chunk * 2 + side] = scale;
#pragma unroll
        for (int p = 0; p < NT; ++p) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float z[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = holds ? x[p][4 * j + i] * inv : 0.0f;
                y[j] = bkv_encode4<CODEC>(z[0], z[1], z[2], z[3]);
            }
            out[p * 64 + lane] = make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
    if (e.block != e.start / bs) return;
    const int nb = (e.end + bs - 1) / bs, first = max(e.start, (nb - 2) * bs), q4 = hd >> 2;
    for (int g = lane; g < (e.end - first) * q4; g += 64) {
        const int t = first + g / q4, d = g % q4 * 4;
        *(float4*)(ring + (size_t)(t & mask) * hd + d) = *(const float4*)(in + (size_t)(t - e.start) * rs + d);
    }
}

// ---- read --------------------------------------------------------------------

// Row r: the values held for (seqs[r], times[r]), zeros where nothing is held. A
// workgroup takes up to 16 rows: where each is comes once into LDS, then a
// thread widens four values of each of its rows at a time (V: the row's byte of
// each word of a 16-byte piece, whose other bytes are the rows beside it), all
// rows' loads in flight. The rows go past the caches: they are what a cache cannot
// hold, the pages may be (four layers of 17.7 thousand rows of 8 heads of 128, written
// and read: 399 us against 440). Bound by memory, 5 bytes a value: those rows take 47
// us, 3.9 TB/s.
constexpr int kReadRows = 16;
__device__ __forceinline__ void bkv_stream(float* p, const float4& x) {
    __builtin_nontemporal_store(vk_f32x4{x.x, x.y, x.z, x.w}, (vk_f32x4*)p);
}
template <int CODEC>
__device__ __forceinline__ float bkv_decode1(uint32_t w) {  // the low byte of a word
    if constexpr (CODEC == BKV_INT8) return (float)(w & 255u) - 128.0f;
    else return bkv_e4m3_f32(w);
}
template <int CODEC>
__global__ __launch_bounds__(256) void vk_bkv_read(BkvView v, int layer, int n, int per, const int* __restrict__ seqs,
                                                   const int* __restrict__ times, float* __restrict__ k,
                                                   float* __restrict__ vv) {
    __shared__ int s_page[kReadRows], s_t[kReadRows], s_seq[kReadRows];  // page -1: the ring, -2: nothing
    const int r0 = blockIdx.x * per, rows = min(per, n - r0), hd = v.hd, bs = v.bs, w = v.n_head * hd;
    if ((int)threadIdx.x < rows) {
        const int seq = seqs[r0 + threadIdx.x], t = times[r0 + threadIdx.x];
        int page = -2;
        if ((unsigned)seq < (unsigned)v.n_seq && t >= 0) {
            const int len = v.len[seq], block = t / bs;
            if (t < len) page = block < len / bs ? v.table[(size_t)seq * v.max_blocks + block] : -1;
        }
        s_page[threadIdx.x] = page;
        s_t[threadIdx.x] = t;
        s_seq[threadIdx.x] = seq;
    }
    __syncthreads();
    const int w4 = w >> 2, hd_log = 31 - __clz(hd), at_once = w4 < 256 ? 256 / w4 : 1;
    const int t0 = (int)threadIdx.x, first = at_once > 1 ? t0 / w4 : 0, c0 = at_once > 1 ? t0 % w4 : t0;
    if (first >= at_once) return;
    for (int c = c0; c < w4; c += 256) {
        const int head = c * 4 >> hd_log, d = c * 4 & (hd - 1);
#pragma unroll 4
        for (int r = first; r < rows; r += at_once) {
            const int page = s_page[r], t = s_t[r];
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f), z = y;
            if (page >= 0) {
                const size_t chunk = bkv_chunk(v, layer, page, head);
                const uint8_t* p = v.pool + chunk * 2 * bs * hd + ((t & (bs - 1)) >> 4) * 16 * hd;
                const uint32_t b = *(const uint32_t*)(p + bkv_k_off(t & 15, d));
                const uint4 q = *(const uint4*)(p + bs * hd + (bkv_v_off(t & 15, d) & ~15));
                const float2 s = *(const float2*)(v.scales + chunk * 2);
                const int sh = (t & 3) * 8;
                y = make_float4(bkv_decode1<CODEC>(b) * s.x, bkv_decode1<CODEC>(b >> 8) * s.x,
                                bkv_decode1<CODEC>(b >> 16) * s.x, bkv_decode1<CODEC>(b >> 24) * s.x);
                z = make_float4(bkv_decode1<CODEC>(q.x >> sh) * s.y, bkv_decode1<CODEC>(q.y >> sh) * s.y,
                                bkv_decode1<CODEC>(q.z >> sh) * s.y, bkv_decode1<CODEC>(q.w >> sh) * s.y);
            } else if (page == -1) {
                const float* p = bkv_ring(v, layer, s_seq[r], 0, head) + (size_t)(t & (2 * bs - 1)) * hd + d;
                y = *(const float4*)p;
                z = *(const float4*)(p + (size_t)v.n_head * 2 * bs * hd);
            }
            bkv_stream(k + (size_t)(r0 + r) * w + c * 4, y);
            bkv_stream(vv + (size_t)(r0 + r) * w + c * 4, z);
        }
    }
}

// ---- fork, free, copy, compact -------------------------------------------------

// The checks that a fork and a copy share: source and destination in range,
// the destination empty, named once and no source of the call's (`same`: both
// ids are of one cache).
__device__ __forceinline__ bool bkv_pair_ok(const BkvView& dv, const BkvView& sv, bool same, int i, int n, int src,
                                            int dst, int* s_dst) {
    const bool rs = (unsigned)src < (unsigned)sv.n_seq, rd = (unsigned)dst < (unsigned)dv.n_seq;
    const int dst_len = rd ? dv.len[dst] : 1;
    s_dst[i] = dst;
    __syncthreads();
    bool named, any, before;
    bkv_named(s_dst, n, i, dst, &named, &any);
    bkv_named(s_dst, n, i, src, &before, &any);
    return rs && rd && dst_len == 0 && !named && !(same && any);
}

__global__ __launch_bounds__(BKV_TPB) void vk_bkv_fork_plan(BkvView v, int n, const int* __restrict__ srcs,
                                                            const int* __restrict__ dsts) {
    __shared__ __align__(16) int s_dst[BKV_TPB];
    __shared__ int s_bad;
    const int i = threadIdx.x;
    if (i == 0) s_bad = n;
    const int src = i < n ? srcs[i] : -1, dst = i < n ? dsts[i] : -1;
    const bool ok = bkv_pair_ok(v, v, true, i, n, src, dst, s_dst);
    if (i < n && !ok) atomicMin(&s_bad, i);
    __syncthreads();
    const int done = s_bad;
    if (i < done) {
        BkvItem it;
        it.seq = src;
        it.start = dst;
        it.count = v.len[src];
        // the fork copies the open block's rows and none before it
        it.row0 = max(v.floor_[src], it.count / v.bs * v.bs);
        v.plan[i] = it;
        v.len[dst] = it.count;
        v.floor_[dst] = it.row0;
    }
    if (i == 0) {
        v.meta[BKV_STATUS] = done == n ? VOKRA_HIP_OK : VOKRA_HIP_ERROR_INVALID_ARGUMENT;
        v.meta[BKV_DONE] = done;
        v.meta[BKV_PLAN_N] = done;
    }
}

// Rows row0 .. count - 1 of the items' sources into the rings of their
// destinations: one wave for each item, layer, head and side.
__device__ __forceinline__ void bkv_move_rows(const BkvView& dv, const BkvView& sv, long long unit) {
    const int hs = 2 * dv.n_head, per = dv.n_layer * hs, lane = threadIdx.x & 63;
    const int i = (int)(unit / per), rest = (int)(unit - (long long)i * per), layer = rest / hs, h = rest - layer * hs;
    if (i >= dv.meta[BKV_PLAN_N]) return;
    const BkvItem it = dv.plan[i];
    const float* src = bkv_ring(sv, layer, it.seq, 0, 0) + (size_t)h * 2 * sv.bs * sv.hd;
    float* dst = bkv_ring(dv, layer, it.start, 0, 0) + (size_t)h * 2 * dv.bs * dv.hd;
    const int mask = 2 * dv.bs - 1, q4 = dv.hd >> 2;
    for (int g = lane; g < (it.count - it.row0) * q4; g += 64) {
        const size_t o = (size_t)((it.row0 + g / q4) & mask) * dv.hd + g % q4 * 4;
        *(float4*)(dst + o) = *(const float4*)(src + o);
    }
}

// Workgroups below `rows`: ring rows; the others: an item's table row each.
__global__ __launch_bounds__(256) void vk_bkv_fork_rows(BkvView v, int rows) {
    if ((int)blockIdx.x < rows) {
        bkv_move_rows(v, v, (long long)blockIdx.x * 4 + (threadIdx.x >> 6));
        return;
    }
    const int i = (int)blockIdx.x - rows;
    if (i >= v.meta[BKV_PLAN_N]) return;
    const BkvItem it = v.plan[i];
    for (int b = threadIdx.x; b < it.count / v.bs; b += 256) {
        const int page = v.table[(size_t)it.seq * v.max_blocks + b];
        v.table[(size_t)it.start * v.max_blocks + b] = page;
        atomicAdd(&v.refs[page], 1);
    }
}

__global__ __launch_bounds__(BKV_TPB) void vk_bkv_free_plan(BkvView v, int n, const int* __restrict__ seqs) {
    __shared__ __align__(16) int s_seq[BKV_TPB];
    __shared__ int s_bad;
    const int i = threadIdx.x;
    if (i == 0) s_bad = n;
    const int seq = i < n ? seqs[i] : -1;
    s_seq[i] = seq;
    __syncthreads();
    if (i < n && (unsigned)seq >= (unsigned)v.n_seq) atomicMin(&s_bad, i);
    bool named, any;
    bkv_named(s_seq, n, i, seq, &named, &any);
    const bool mine = !named;
    __syncthreads();
    const int done = s_bad;
    if (i < done) {
        BkvItem it;
        it.seq = seq;
        it.start = it.row0 = 0;
        it.count = mine ? v.len[seq] : 0;  // a sequence named twice is freed once
        v.plan[i] = it;
        if (mine) {
            v.len[seq] = 0;
            v.floor_[seq] = 0;
        }
    }
    for (int k = i; k < kBkvMaxItems; k += (int)blockDim.x) v.step[k] = BkvItem{0, 0, 0, 0};
    if (i == 0) {
        v.meta[BKV_STATUS] = done == n ? VOKRA_HIP_OK : VOKRA_HIP_ERROR_INVALID_ARGUMENT;
        v.meta[BKV_DONE] = done;
        v.meta[BKV_PLAN_N] = done;
        v.meta[BKV_STEP_N] = v.meta[BKV_WORK_N] = 0;  // a step ends with a free
    }
}

__global__ __launch_bounds__(256) void vk_bkv_free_pages(BkvView v) {
    if ((int)blockIdx.x >= v.meta[BKV_PLAN_N]) return;
    const BkvItem it = v.plan[blockIdx.x];
    for (int b = blockIdx.y * 256 + threadIdx.x; b < it.count / v.bs; b += 256 * gridDim.y) {
        int* e = v.table + (size_t)it.seq * v.max_blocks + b;
        bkv_drop(v, *e);
        *e = -1;
    }
}

__global__ __launch_bounds__(BKV_TPB) void vk_bkv_copy_plan(BkvView dv, BkvView sv, int same, int n,
                                                            const int* __restrict__ srcs,
                                                            const int* __restrict__ dsts) {
    __shared__ int red[BKV_TPB / 64];
    __shared__ int off[BKV_TPB + 1], s_src[BKV_TPB];
    __shared__ __align__(16) int s_dst[BKV_TPB];
    __shared__ int s_bad, s_done;
    const int i = threadIdx.x;
    if (i == 0) s_bad = s_done = n;
    const int src = i < n ? srcs[i] : -1, dst = i < n ? dsts[i] : -1;
    const int free_pages = dv.meta[BKV_FREE];
    bool ok = bkv_pair_ok(dv, sv, same != 0, i, n, src, dst, s_dst);
    const int len = ok ? sv.len[src] : 0;
    if (len > dv.max_time) ok = false;
    const int need = ok ? len / dv.bs : 0;
    int at[1] = {need}, sum[1];
    bkv_scan(at, sum, red);
    if (i < n && !ok) atomicMin(&s_bad, i);
    off[i] = at[0];
    s_src[i] = src;
    if (i + 1 == (int)blockDim.x) off[i + 1] = sum[0];
    __syncthreads();
    const int bad = s_bad;
    if (i < bad && need > 0 && at[0] + need > free_pages) atomicMin(&s_done, i);
    __syncthreads();
    const int done = min(s_done, bad), total = off[done];
    if (total) bkv_take(dv, total, red);
    for (int k = i; k < total; k += (int)blockDim.x) {
        const int it = bkv_find(off, done, k), b = k - off[it], page = dv.fresh[k];
        dv.table[(size_t)s_dst[it] * dv.max_blocks + b] = page;
        dv.refs[page] = 1;
        dv.moves[k] = make_int2(sv.table[(size_t)s_src[it] * sv.max_blocks + b], page);
    }
    if (i < done) {
        BkvItem it;
        it.seq = src;
        it.start = dst;
        it.count = len;
        it.row0 = sv.floor_[src];
        dv.plan[i] = it;
        dv.len[dst] = len;
        dv.floor_[dst] = it.row0;
    }
    if (i == 0) {
        dv.meta[BKV_FREE] = free_pages - total;
        dv.meta[BKV_STATUS] = done == n ? VOKRA_HIP_OK
                              : done < bad ? VOKRA_HIP_ERROR_KV_CACHE_EXHAUSTED
                                           : VOKRA_HIP_ERROR_INVALID_ARGUMENT;
        dv.meta[BKV_DONE] = done;
        dv.meta[BKV_PLAN_N] = done;
        dv.meta[BKV_MOVE_N] = total;
    }
}

// The moves' bytes and scales, every layer: runs of n_head * 2 * bs * hd bytes.
// Bound by memory: 210 MB of pages move in 74 us, 5.7 TB/s read and written, some of
// it in the cache behind the L2s; with stores past the caches 30 us longer.
__global__ __launch_bounds__(256) void vk_bkv_move_pages(BkvView dv, BkvView sv) {
    const int n = dv.meta[BKV_MOVE_N];
    const size_t run = (size_t)dv.n_head * 2 * dv.bs * dv.hd;
    for (size_t e = blockIdx.x; e < (size_t)n * dv.n_layer; e += gridDim.x) {
        const int layer = (int)(e / n);
        const int2 m = dv.moves[e % n];
        const size_t sp = (size_t)layer * sv.n_page + m.x, dp = (size_t)layer * dv.n_page + m.y;
        const uint4* a = (const uint4*)(sv.pool + sp * run);
        uint4* b = (uint4*)(dv.pool + dp * run);
        for (size_t x = threadIdx.x; x < run / 16; x += 256) b[x] = a[x];
        for (int x = threadIdx.x; x < 2 * dv.n_head; x += 256)
            dv.scales[dp * 2 * dv.n_head + x] = sv.scales[sp * 2 * dv.n_head + x];
    }
}

// The ring rows of copied sequences (all that a step may still go back to).
__global__ __launch_bounds__(256) void vk_bkv_copy_rows(BkvView dv, BkvView sv) {
    bkv_move_rows(dv, sv, (long long)blockIdx.x * 4 + (threadIdx.x >> 6));
}

// u pages are in use: the k-th one at or above u moves to the k-th free one
// below u. v.fresh takes the free ones, v.moves the pairs.
__global__ __launch_bounds__(BKV_TPB) void vk_bkv_compact_plan(BkvView v) {
    __shared__ int red[2 * (BKV_TPB / 64)];
    const int u = v.n_page - v.meta[BKV_FREE], words = (v.n_page + 31) / 32;
    int holes = 0, movers = 0;
    for (int base = 0; base < words; base += BKV_TPB) {
        const int w = base + (int)threadIdx.x;
        const uint32_t bits = w < words ? v.used[w] : 0u;
        // bits of pages below u
        const int below = min(max(u - w * 32, 0), 32);
        const uint32_t low = w < words ? (below == 32 ? ~0u : (1u << below) - 1u) : 0u;
        uint32_t h = ~bits & low, m = bits & ~low;
        int at[2] = {(int)__popc(h), (int)__popc(m)}, all[2];
        bkv_scan(at, all, red);
        int ah = holes + at[0], am = movers + at[1];
        for (; h; h &= h - 1) v.fresh[ah++] = w * 32 + __ffs(h) - 1;
        for (; m; m &= m - 1) v.moves[am++].x = w * 32 + __ffs(m) - 1;
        holes += all[0];
        movers += all[1];
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += BKV_TPB) {
        const int from = v.moves[k].x, to = v.fresh[k];
        v.moves[k].y = to;
        v.remap[from] = to;
        v.refs[to] = v.refs[from];
        v.refs[from] = 0;
    }
    for (int w = threadIdx.x; w < words; w += BKV_TPB) {
        const int below = min(max(u - w * 32, 0), 32);
        v.used[w] = below == 32 ? ~0u : (1u << below) - 1u;
    }
    if (threadIdx.x == 0) {
        v.meta[BKV_MOVE_N] = movers;
        v.meta[BKV_HINT] = u / 32;
        v.meta[BKV_STATUS] = VOKRA_HIP_OK;
        v.meta[BKV_DONE] = movers;
    }
}

// Table entries of moved pages, one sequence a workgroup, and the pages that the
// current step's rows are still to be written to.
__global__ __launch_bounds__(256) void vk_bkv_compact_table(BkvView v) {
    if (v.meta[BKV_MOVE_N] == 0) return;
    const int u = v.n_page - v.meta[BKV_FREE];
    for (int seq = blockIdx.x; seq < v.n_seq; seq += gridDim.x) {
        const int nb = v.len[seq] / v.bs;
        for (int b = threadIdx.x; b < nb; b += 256) {
            int* e = v.table + (size_t)seq * v.max_blocks + b;
            if (*e >= u) *e = v.remap[*e];
        }
    }
    for (int k = blockIdx.x * 256 + threadIdx.x; k < v.meta[BKV_WORK_N]; k += gridDim.x * 256)
        if (v.work[k].page >= u) v.work[k].page = v.remap[v.work[k].page];
}

__global__ void vk_bkv_peek(BkvView v, int seq, int block, int* out) {
    out[0] = v.len[seq];
    out[1] = block < v.len[seq] / v.bs ? v.table[(size_t)seq * v.max_blocks + block] : -1;
}

// ---- launchers -----------------------------------------------------------------

hipError_t launch_bkv_part_clear(hipStream_t s, void* part) {
    hipLaunchKernelGGL(vk_bkv_fill, dim3(2048), dim3(256), 0, s, (uint4*)part, kBkvPartBytes / 16);
    return hipGetLastError();
}

hipError_t launch_bkv_reset(hipStream_t s, const BkvView& v, bool clear_data) {
    hipLaunchKernelGGL(vk_bkv_reset, dim3(256), dim3(256), 0, s, v);
    if (clear_data) {
        const size_t pages = (size_t)v.n_layer * v.n_page * v.n_head;
        const size_t pool = pages * 2 * v.bs * v.hd;
        const size_t ring = (size_t)v.n_layer * v.n_seq * 2 * v.n_head * 2 * v.bs * v.hd * sizeof(float);
        hipLaunchKernelGGL(vk_bkv_fill, dim3(2048), dim3(256), 0, s, (uint4*)v.pool, pool / 16);
        hipLaunchKernelGGL(vk_bkv_fill, dim3(2048), dim3(256), 0, s, (uint4*)v.ring, ring / 16);
        // rounded up to 16 bytes by the allocation
        hipLaunchKernelGGL(vk_bkv_fill, dim3(256), dim3(256), 0, s, (uint4*)v.scales, (pages * 8 + 15) / 16);
    }
    return hipGetLastError();
}

// Threads of a planning kernel for n items: four waves keep its barriers short.
static unsigned plan_threads(int n) { return n <= 256 ? 256 : BKV_TPB; }

hipError_t launch_bkv_step(hipStream_t s, const BkvView& v, int n, int n_rows, int max_count, const int* seqs,
                           const int* starts, const int* counts) {
    hipLaunchKernelGGL(vk_bkv_step, dim3(1), dim3(plan_threads(n)), 0, s, v, n, n_rows, max_count, seqs, starts,
                       counts);
    return hipGetLastError();
}

// Workgroups of one launch: a grid holds fewer than 2^32 threads.
constexpr long long kMaxWgs = 1 << 23;

template <int CODEC, int NT>
static void go_write(hipStream_t s, const BkvView& v, int layer, int n_rows, long long wgs, const float* k,
                     const float* vv) {
    for (long long w = 0; w < wgs; w += kMaxWgs)
        hipLaunchKernelGGL((vk_bkv_write<CODEC, NT>), dim3((unsigned)std::min(kMaxWgs, wgs - w)), dim3(256), 0, s, v,
                           layer, n_rows, (unsigned)w, k, vv);
}
template <int CODEC>
static void go_write(hipStream_t s, const BkvView& v, int layer, int n_rows, long long wgs, const float* k,
                     const float* vv) {
    switch (v.bs / 16 * (v.hd / 64)) {
    case 1: go_write<CODEC, 1>(s, v, layer, n_rows, wgs, k, vv); break;
    case 2: go_write<CODEC, 2>(s, v, layer, n_rows, wgs, k, vv); break;
    case 4: go_write<CODEC, 4>(s, v, layer, n_rows, wgs, k, vv); break;
    default: go_write<CODEC, 8>(s, v, layer, n_rows, wgs, k, vv); break;
    }
}

hipError_t launch_bkv_write(hipStream_t s, const BkvView& v, int layer, int n_rows, int work_bound, const float* k,
                            const float* vv) {
    if (work_bound == 0) return hipSuccess;
    const long long wgs = ((long long)work_bound * 2 * v.n_head + 3) / 4;
    if (v.codec == BKV_INT8) go_write<BKV_INT8>(s, v, layer, n_rows, wgs, k, vv);
    else go_write<BKV_E4M3>(s, v, layer, n_rows, wgs, k, vv);
    return hipGetLastError();
}

hipError_t launch_bkv_read(hipStream_t s, const BkvView& v, int layer, int n, const int* seqs, const int* times,
                           float* k, float* vv) {
    // rows a workgroup: up to 16, once that leaves four workgroups a CU (64 rows of 20
    // heads of 64, written and read in 8 layers: 70 us, 175 with 16; 26 thousand rows
    // of 4 heads of 128, moved and read in 8 layers: 322 us, 362 with one)
    const int per = std::min(std::max(n / 1024, 1), kReadRows);
    const size_t w = (size_t)v.n_head * v.hd;
    for (long long r = 0; r < n; r += kMaxWgs * per) {
        const int now = (int)std::min<long long>(kMaxWgs * per, n - r);
        const dim3 grid((unsigned)((now + per - 1) / per));
        if (v.codec == BKV_INT8)
            hipLaunchKernelGGL(vk_bkv_read<BKV_INT8>, grid, dim3(256), 0, s, v, layer, now, per, seqs + r, times + r,
                               k + r * w, vv + r * w);
        else
            hipLaunchKernelGGL(vk_bkv_read<BKV_E4M3>, grid, dim3(256), 0, s, v, layer, now, per, seqs + r, times + r,
                               k + r * w, vv + r * w);
    }
    return hipGetLastError();
}

// Workgroups of the ring rows of n items, four waves each. Items name a destination each,
// so no more than n_seq are done, and the rings of a cache that fits the card are fewer than
// a launch has threads for.
static unsigned row_grid(const BkvView& v, int n) {
    return (unsigned)(((long long)std::min(n, v.n_seq) * v.n_layer * 2 * v.n_head + 3) / 4);
}

hipError_t launch_bkv_fork(hipStream_t s, const BkvView& v, int n, const int* src, const int* dst) {
    hipLaunchKernelGGL(vk_bkv_fork_plan, dim3(1), dim3(plan_threads(n)), 0, s, v, n, src, dst);
    if (n) {
        const unsigned rows = row_grid(v, n);
        hipLaunchKernelGGL(vk_bkv_fork_rows, dim3(rows + (unsigned)n), dim3(256), 0, s, v, (int)rows);
    }
    return hipGetLastError();
}

hipError_t launch_bkv_free(hipStream_t s, const BkvView& v, int n, const int* seqs) {
    hipLaunchKernelGGL(vk_bkv_free_plan, dim3(1), dim3(plan_threads(n)), 0, s, v, n, seqs);
    if (n) {
        const unsigned y = (unsigned)std::min((v.max_blocks + 255) / 256, 64);
        hipLaunchKernelGGL(vk_bkv_free_pages, dim3((unsigned)n, y), dim3(256), 0, s, v);
    }
    return hipGetLastError();
}

// Workgroups of the page moves: the number of moves is known on the device only.
constexpr unsigned kMoveGrid = 2048;

hipError_t launch_bkv_copy(hipStream_t s, const BkvView& dv, const BkvView& sv, int n, const int* src,
                           const int* dst) {
    // all threads, as the pages of few items are many: 1600 pages 15 -> 11 us
    hipLaunchKernelGGL(vk_bkv_copy_plan, dim3(1), dim3(BKV_TPB), 0, s, dv, sv, (int)(dv.meta == sv.meta), n, src,
                       dst);
    if (n) {
        hipLaunchKernelGGL(vk_bkv_move_pages, dim3(kMoveGrid), dim3(256), 0, s, dv, sv);
        hipLaunchKernelGGL(vk_bkv_copy_rows, dim3(row_grid(dv, n)), dim3(256), 0, s, dv, sv);
    }
    return hipGetLastError();
}

hipError_t launch_bkv_compact(hipStream_t s, const BkvView& v) {
    hipLaunchKernelGGL(vk_bkv_compact_plan, dim3(1), dim3(BKV_TPB), 0, s, v);
    hipLaunchKernelGGL(vk_bkv_move_pages, dim3(kMoveGrid), dim3(256), 0, s, v, v);
    hipLaunchKernelGGL(vk_bkv_compact_table, dim3((unsigned)std::min(v.n_seq, 1024)), dim3(256), 0, s, v);
    return hipGetLastError();
}

hipError_t launch_bkv_peek(hipStream_t s, const BkvView& v, int seq, int block, int* out) {
    hipLaunchKernelGGL(vk_bkv_peek, dim3(1), dim3(1), 0, s, v, seq, block, out);
    return hipGetLastError();
}

}  // namespace vk
