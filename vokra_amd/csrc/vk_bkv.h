// vk_bkv.h — the block-scaled KV cache: its view in device memory and the
// launchers of its kernels (vk_bkv.hip, vk_bkv_attn.hip). The C-ABI layer
// (vk_bkv_capi.hip) validates what the host can see before calling them;
// sequence ids, starts and counts in device memory are validated by the
// kernels that take them.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

constexpr int kBkvMaxItems = 1024;   // items of one call: one thread of the planning workgroup each
constexpr int kBkvParts = 1 << 17;  // query rows of which a split attention can hold a partial result
constexpr int kBkvShares = 512;  // workgroups that share a chunked attention: two a CU
// a context's partial results ((max, sum) and up to 128 values a row), counters,
// and the tiles that go on in a later share
constexpr size_t kBkvPartBytes = (size_t)kBkvParts * (128 + 2) * 4 + kBkvShares * (4 + 16);

// What planning kernels leave for the kernels of the same call or step.
// meta (int32): see the BKV_ indices.
enum {
    BKV_FREE = 0,    // pages not in use
    BKV_HINT,        // no page below word BKV_HINT of the bitmap is free
    BKV_STATUS,      // status of the last step / fork / free / copy (VOKRA_HIP_OK, _INVALID_ARGUMENT, _EXHAUSTED)
    BKV_DONE,        // its items done
    BKV_STEP_N,      // items of the current step
    BKV_WORK_N,      // blocks of the current step's write
    BKV_MOVE_N,      // page moves of the last copy / compact
    BKV_PLAN_N,      // items of the last fork / free / copy
    BKV_META_INTS = 16
};

// One item of a step: sequence, its first new row, number of rows, its first
// row in the step's packed rows. Also a fork / free / copy item: source,
// destination, source length, source floor.
struct BkvItem {
    int seq, start, count, row0;
};

// One block that an item's rows reach: what its write needs.
struct alignas(16) BkvWork {
    int seq, start, end, row0;  // the item: rows start .. end - 1, packed from row0 on
    int block, page, pad[2];    // page: of a block that the step fills, else -1
};

struct BkvView {
    // pool: [layer][page][head] chunks of 2 * bs * hd bytes, K then V, in
    // 16-token tiles (bkv_k_off / bkv_v_off); scales [layer][page][head][2]
    uint8_t* pool;
    float* scales;
    // rows of the open block and the block before it as they came, f32:
    // [layer][seq][side][head][2 * bs][hd], row t at t % (2 * bs)
    float* ring;
    int* table;      // [n_seq][max_blocks] page of each full block, -1 = none
    int* len;        // [n_seq] rows held
    int* floor_;     // [n_seq] the lowest row a step may start at
    int* refs;       // [n_page] sequences that hold the page
    uint32_t* used;  // bitmap of refs != 0
    int* fresh;      // [n_page] pages taken by the current call
    int2* moves;     // [n_page] (source page, destination page) of a copy / compact
    int* remap;      // [n_page] new page of a moved page
    int* meta;
    BkvItem* step;   // [kBkvMaxItems] the current step, no rows in entries beyond it
    BkvItem* plan;   // [kBkvMaxItems] items of the current fork / free / copy
    BkvWork* work;   // [max_work] the blocks of the current step's write
    int n_layer, n_head, hd, n_seq, bs, n_page, max_blocks, max_time, codec, max_work;
};

constexpr int BKV_INT8 = 0, BKV_E4M3 = 1;

// Byte of element (token t of the tile, d) in a 16-token K or V tile: the
// order in which the attention's matrix instructions take them, 16 bytes a
// lane, and in which 16-byte reads of rows leave them.
// K: lane (d % 16 / 4) * 16 + t holds word d % 64 / 16, byte d % 4.
// V: lane (t / 4) * 16 + d % 64 / 4 holds word d % 4 (row d % 64 / 4 of four
// products), byte t % 4.
__host__ __device__ inline int bkv_k_off(int t, int d) {
    return ((d >> 6) * 64 + ((d >> 2) & 3) * 16 + t) * 16 + ((d >> 4) & 3) * 4 + (d & 3);
}
__host__ __device__ inline int bkv_v_off(int t, int d) {
    return ((d >> 6) * 64 + (t >> 2) * 16 + ((d >> 2) & 15)) * 16 + (d & 3) * 4 + (t & 3);
}

namespace vk {
hipError_t launch_bkv_part_clear(hipStream_t s, void* part);
hipError_t launch_bkv_reset(hipStream_t s, const BkvView& v, bool clear_data);
hipError_t launch_bkv_step(hipStream_t s, const BkvView& v, int n, int n_rows, int max_count, const int* seqs,
                           const int* starts, const int* counts);
// n_rows, work_bound: at least the step's rows, blocks
hipError_t launch_bkv_write(hipStream_t s, const BkvView& v, int layer, int n_rows, int work_bound, const float* k,
                            const float* vv);
hipError_t launch_bkv_read(hipStream_t s, const BkvView& v, int layer, int n, const int* seqs, const int* times,
                           float* k, float* vv);
hipError_t launch_bkv_fork(hipStream_t s, const BkvView& v, int n, const int* src, const int* dst);
hipError_t launch_bkv_free(hipStream_t s, const BkvView& v, int n, const int* seqs);
hipError_t launch_bkv_copy(hipStream_t s, const BkvView& dst_v, const BkvView& src_v, int n, const int* src,
                           const int* dst);
hipError_t launch_bkv_compact(hipStream_t s, const BkvView& v);
// out (2 ints): length of seq, page of block
hipError_t launch_bkv_peek(hipStream_t s, const BkvView& v, int seq, int block, int* out);
// Rows of the current step (n items, n_rows rows, at most max_count each, no
// more than max_len rows held by any) against the cache; part:
// kBkvPartBytes, its counters zero.
hipError_t launch_bkv_attn(hipStream_t s, const BkvView& v, int layer, int n, int n_rows, int max_count, int max_len,
                           int hq, const float* q, float scale, float* out, float* part);
}  // namespace vk
