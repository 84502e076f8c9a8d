// Layout of the paged 4-bit KV cache in device memory, shared by its kernels and its host side (kv4.hip).
//
// The pool is [page][layer][kv head] blocks. With P positions to a page, a block holds, in this order,
//   K nibbles  [position][hd / 2 bytes]: dword c of a row holds dims 8 c .. 8 c + 7, dim 8 c + 2 p in bits
//              4 p .. 4 p + 3 and dim 8 c + 2 p + 1 sixteen bits higher: the pair (w >> 4 p) & 0x000F000F is
//              two neighbouring dims in the two halves, where the packed f16 arithmetic wants them;
//   K scales   [position][hd / 32] pairs {f16 d, f16 m} of 32 dims;
//   V nibbles  [position / 4][hd / 8][position % 4] dwords of 8 dims each: 16 bytes are four positions of the
//              same dims, since the product over positions needs neighbouring positions in one lane;
//   V d, V m   [hd / 32][position] f16 each: 16 bytes are eight positions of one group.
// Value = f16(m + q d), rounded once. 5 bits an element. Pages are whole blocks of all layers, so copying a
// page is one contiguous copy.
#pragma once

#include "common.hpp"
#include "device.hpp"

namespace aesir {

constexpr int kKv4Group = 32;  // dims per scale

// Attention work is planned for four widths of a column tile ((row, query head) columns; kv4.hip's classes). Every
// launch reads the plan of its own width, so a captured launch stays right for any later batch.
constexpr int kKv4Widths = 4;

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kNone = 0x7FFFFFFF;  // in every field of the records behind the last one

struct Kv4Seq {  // one sequence of the batch
    int32_t slot, length, rows, row0;  // length counts the new rows
    struct {
        int32_t unit0, splits, part0, pad;  // first (column tile, split) unit, splits of each tile, first partial slot
    } plan[kKv4Widths];
};
static_assert(sizeof(Kv4Seq) == 80, "descriptor");

struct Kv4Range {  // rows to read back: positions pos .. pos + rows - 1 of a sequence, to output rows row0 ..
    int32_t slot, pos, rows, row0;
};

struct Kv4Dev {
    char *pool;
    int64_t page_bytes, layer_bytes;
    int32_t page_shift, hd, nkv, nq;
    const int32_t *table;  // [max_seqs][table_stride] page ids
    int64_t table_stride;
    const Kv4Seq *seqs;    // in row order, ended by records of kNone
    float *part, *part_ml;  // split partials of a column: accumulators [hd], and (maximum, sum)

    __host__ __device__ int page_size() const { return 1 << page_shift; }
    __host__ __device__ int64_t head_bytes() const { return (int64_t)page_size() * hd / 4 * 5; }
    __device__ char *block(int64_t page, int64_t layer, int head) const {
        return pool + page * page_bytes + layer * layer_bytes + head * head_bytes();
    }
    __device__ int k_scale_off() const { return page_size() * hd / 2; }
    __device__ int v_off() const { return page_size() * hd / 8 * 5; }
    __device__ int v_d_off() const { return v_off() + page_size() * hd / 2; }
    __device__ int v_m_off() const { return v_d_off() + page_size() * hd / 16; }
};

// The two values of nibble pair p of a dword (dims 2 p and 2 p + 1) under scale d and offset m.
__device__ __forceinline__ h16x2 kv4_pair(unsigned w, int p, h16x2 d, h16x2 m) {
    const h16x2 n = as_h2(((w >> (4 * p)) & 0x000F000Fu) | 0x64006400u) - h16x2{(h16)1024.0f, (h16)1024.0f};
    return __builtin_elementwise_fma(n, d, m);  // one rounding
}
__device__ __forceinline__ h16x2 both(h16 x) { return h16x2{x, x}; }

}  // namespace aesir
