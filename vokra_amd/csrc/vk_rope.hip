// vk_rope.hip — rotary positions of q and k by a plan: any even part of the
// head, both pair layouts, frequencies scaled for long contexts.
//
// Pair j of a head turns by pos * theta_j. The plan holds theta_j / 2pi as a
// 64-bit fraction of a turn, so pos * theta_j modulo a turn is one wrapping
// 64-bit product, exact to 2^-33 of a turn at any int32 position (an f32
// product of position and frequency is off by 2^-24 of the whole angle: a
// tenth of a radian at position 10^6). The top 32 bits give the quadrant and a
// rest in [-pi/4, pi/4], whose sine and cosine are Taylor polynomials in f32
// (degrees 9 and 10: the first terms left out are below 2e-9). They are multiplied by the
// magnitude after that, so where it is not 1 they are rounded twice: half a step of
// f32 more, for one product a pair instead of one a value.
//
// Bound by memory: 8 bytes an element moved, about 40 VALU operations a pair
// for its sine and cosine, which the heads that a thread turns share. 8191 rows of
// 32 + 8 heads of 128, half of each turned, to another buffer: 336 MB in 59 us, 5.7
// TB/s (part of them in the cache behind the L2s); 32 rows of 16 + 2 heads take 3
// us, which is dependent rounds of memory (the call 4.7, most of it the host's).
#include <algorithm>

#include "vk_common.h"
#include "vk_step.h"

namespace vk {

__device__ __forceinline__ float2 rope_cos_sin(int pos, uint64_t turn, float mag) {
    const uint64_t a = (uint64_t)(int64_t)pos * turn;
    const uint32_t u = (uint32_t)((a + 0x80000000ull) >> 32);
    const uint32_t quad = (u + 0x20000000u) >> 30;
    const float y = (float)(int32_t)(u - (quad << 30)) * 1.46291807926715968e-09f;  // 2 pi / 2^32
    const float z = y * y;
    float s = fmaf(z, 2.75573192239858907e-06f, -1.98412698412698413e-04f);
    s = fmaf(s, z, 8.33333333333333333e-03f);
    s = fmaf(s, z, -1.66666666666666667e-01f);
    s = fmaf(s * z, y, y);
    float c = fmaf(z, -2.75573192239858907e-07f, 2.48015873015873016e-05f);
    c = fmaf(c, z, -1.38888888888888889e-03f);
    c = fmaf(c, z, 4.16666666666666667e-02f);
    c = fmaf(c, z, -0.5f);
    c = fmaf(c, z, 1.0f);
    const float cq = quad & 1 ? s : c, sq = quad & 1 ? c : s;
    // quadrant 0: (c, s), 1: (-s, c), 2: (-c, -s), 3: (s, -c)
    return make_float2((quad == 1 || quad == 2 ? -cq : cq) * mag, (quad >= 2 ? -sq : sq) * mag);
}

template <bool PAST>
__device__ __forceinline__ void rope_put(float* p, vk_f32x4 x) {
    if constexpr (PAST) __builtin_nontemporal_store(x, (vk_f32x4*)p);
    else *(vk_f32x4*)p = x;
}

// A thread turns V pairs (or copies as many floats beyond rot, where the
// output is another buffer) of the heads hl, hl + HL, ...; units of a head run
// fastest over the threads, then the HL head lanes, then rows.
// V = 4 (half layout) or 2 (pairs side by side): 16-byte accesses; V = 1: any
// size and alignment. PAST: stores go past the caches.
template <int V, bool PAIRS, bool PAST>
__global__ __launch_bounds__(256) void vk_rope_turn(RopeArgs a) {
    const int units = a.units;
    const size_t g = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int per_row = units * a.head_lanes;
    const size_t row = g / per_row;
    if (row >= (size_t)a.rows) return;
    const int rest = (int)(g - row * per_row), hl = rest / units, u = rest - hl * units;
    const int half = a.rot >> 1, turn_units = half / V;
    const bool turns = u < turn_units;
    float2 cs[V];
    int i0, i1;  // the unit's elements: V at i0 and V at i1 (PAIRS: 2 V at i0)
    if (turns) {
        const int pos = a.positions[row];
#pragma unroll
        for (int j = 0; j < V; ++j) cs[j] = rope_cos_sin(pos, a.turn[u * V + j], a.mag);
        i0 = PAIRS ? 2 * u * V : u * V;
        i1 = i0 + (PAIRS ? V : half);
    } else {
        i0 = a.rot + (u - turn_units) * 2 * V;
        i1 = i0 + V;
    }
    for (int h = hl; h < a.heads_q + a.heads_k; h += a.head_lanes) {
        const bool is_q = h < a.heads_q;
        const float* x = is_q ? a.q + row * a.q_stride + (size_t)h * a.hd
                              : a.k + row * a.k_stride + (size_t)(h - a.heads_q) * a.hd;
        float* y = is_q ? a.q_out + row * a.qo_stride + (size_t)h * a.hd
                        : a.k_out + row * a.ko_stride + (size_t)(h - a.heads_q) * a.hd;
        float p[V], r[V];
        if constexpr (V == 4) {
            const float4 f = *(const float4*)(x + i0), t = *(const float4*)(x + i1);
            p[0] = f.x, p[1] = f.y, p[2] = f.z, p[3] = f.w;
            r[0] = t.x, r[1] = t.y, r[2] = t.z, r[3] = t.w;
        } else if constexpr (V == 2) {
            const float4 f = *(const float4*)(x + i0);
            p[0] = f.x, p[1] = f.y, r[0] = f.z, r[1] = f.w;
        } else {
            p[0] = x[i0];
            r[0] = i1 < a.hd ? x[i1] : 0.0f;
        }
        if (turns) {
            if constexpr (PAIRS && V == 2) {  // (p0, p1) and (r0, r1) are pairs
                const float a0 = p[0], b0 = p[1], a1 = r[0], b1 = r[1];
                p[0] = fmaf(a0, cs[0].x, -(b0 * cs[0].y));
                p[1] = fmaf(a0, cs[0].y, b0 * cs[0].x);
                r[0] = fmaf(a1, cs[1].x, -(b1 * cs[1].y));
                r[1] = fmaf(a1, cs[1].y, b1 * cs[1].x);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float f = p[j], t = r[j];
                    p[j] = fmaf(f, cs[j].x, -(t * cs[j].y));
                    r[j] = fmaf(f, cs[j].y, t * cs[j].x);
                }
            }
        }
        if constexpr (V == 4) {
            rope_put<PAST>(y + i0, vk_f32x4{p[0], p[1], p[2], p[3]});
            rope_put<PAST>(y + i1, vk_f32x4{r[0], r[1], r[2], r[3]});
        } else if constexpr (V == 2) {
            rope_put<PAST>(y + i0, vk_f32x4{p[0], p[1], r[0], r[1]});
        } else {
            y[i0] = p[0];
            if (i1 < a.hd) y[i1] = r[0];
        }
    }
}

hipError_t launch_rope_turn(hipStream_t s, RopeArgs a, bool pairs) {
    const int half = a.rot / 2, tail = a.hd - a.rot;
    // in place, the elements beyond rot stay where they are
    const bool copies = tail > 0 && (a.q_out != a.q || (a.heads_k && a.k_out != a.k));
    const uintptr_t addr = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.q_out) |
                           (a.heads_k ? reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.k_out) : 0);
    const size_t strides = a.q_stride | a.qo_stride | (a.heads_k ? a.k_stride | a.ko_stride : 0);
    const bool vec = (addr & 15) == 0 && strides % 4 == 0 && a.hd % 4 == 0;
    const int v = !vec ? 1 : pairs ? (a.rot % 4 == 0 ? 2 : 1) : (half % 4 == 0 && (!copies || tail % 8 == 0) ? 4 : 1);
    a.units = half / v + (copies ? (tail + 2 * v - 1) / (2 * v) : 0);
    // heads a thread: one where that leaves fewer than 1024 workgroups, four (sine and cosine
    // shared) from there on. The kernel's time, half layout of 128, one head a thread and
    // four: 32 rows of 18 heads 3.0 and 3.9 us, 300 rows of 40 (750 workgroups) 4.1 and
    // 4.5, 500 (1250) 5.2 and 5.0, 800 6.9 and 5.8, 2000 13.8 and 13.6
    const int heads = a.heads_q + a.heads_k;
    const size_t all = (size_t)a.rows * a.units * heads;
    a.head_lanes = all / 256 < 1024 ? heads : (heads + 3) / 4;
    // outputs that the caches cannot hold beside the inputs go past them (63 us -> 59 for
    // the call above; 1500 rows, which they hold, take 10.9 us with them and 11.2 past)
    const bool past = v > 1 && (size_t)a.rows * heads * a.hd > (size_t)32 << 20;
    const size_t threads = (size_t)a.rows * a.units * a.head_lanes;
    const dim3 grid((unsigned)((threads + 255) / 256));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
    if (v == 2) past ? go(vk_rope_turn<2, true, true>) : go(vk_rope_turn<2, true, false>);
    else if (v == 4) past ? go(vk_rope_turn<4, false, true>) : go(vk_rope_turn<4, false, false>);
    else pairs ? go(vk_rope_turn<1, true, false>) : go(vk_rope_turn<1, false, false>);
    return hipGetLastError();
}

}  // namespace vk
