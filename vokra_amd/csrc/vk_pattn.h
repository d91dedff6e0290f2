// vk_pattn.h — launcher of attention over packed sequences (vk_pattn.hip). The C-ABI
// layer (vk_pattn_capi.hip) checks what the host can see; offsets in device memory are
// checked by the kernels that read them.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

constexpr int kPaSeqs = 1024;    // sequences of a call at most
constexpr int kPaShares = 512;   // workgroups that share a call's work at most
// query rows of a tile, 32 a wave
constexpr int pa_tile_rows(int hd) { return hd == 64 ? 128 : 256; }
constexpr int kPaKeys = 64;      // keys of a tile
constexpr int kPaFewRows = 32;   // query rows of a kv head that the kernel without packing takes

// What packing leaves beside a tile of 64 keys of one kv head.
struct alignas(16) PaTileMeta {
    int k_exp, v_exp;         // its values are held times 2^-exp (v_exp kPaNoValue: all zero)
    unsigned long long odd;   // keys whose V has a value that is not finite (held as 0)
};
constexpr int kPaNoValue = -100000;

// Where a share of the work begins.
struct alignas(16) PaStart {
    int seq, head, slot;  // its first tile
    int pad;
    long long line;       // that tile's place on the line
};

struct PaArgs {
    const float *q, *k, *v;
    float* out;
    size_t q_stride, k_stride, v_stride, out_stride;  // floats from row to row
    const int *q_off, *k_off;  // [n_seq + 1]
    int n_seq, q_rows, k_rows, max_q, max_k;
    int hq, hkv, g;  // g = hq / hkv
    int causal, window;
    float c, sign;  // |scale| log2(e) and the scale's sign (0: scale 0, c 1)
    // workspace
    _Float16* tiles;         // [slot of 64 keys][kv head]: K hi, K lo, V hi, V lo in operand order
    PaTileMeta* meta;        // [slot of 64 keys][kv head]
    long long* line;         // [slot of a tile of rows + 1] cost of the tiles before, of one kv head
    PaStart* start;          // [kPaShares]
    int* ended;              // [kPaShares] pieces of the tile whose first unit a share has that have ended
    long long* plan;         // [0] a share's length, [1] the line's, [2] sequences in order
    float* part;             // partial results: [share][2] pieces
    int k_slots;             // places of tiles of keys
};

namespace vk {
size_t pattn_part_floats(int hd);
hipError_t launch_pattn(hipStream_t s, int hd, const PaArgs& a);
}  // namespace vk
