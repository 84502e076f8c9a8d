// Layout of the paged 4-bit KV cache in device memory, shared by its kernels and its host side (kv4.hip).
//
// The pool is [page][layer][kv head] blocks of P positions, each P / 32 runs of 32 positions, contiguous because a
// wave takes a run at a time. A run holds, in this order (pos in the run, c a dword of 8 dims),
//   K nibbles  [pos][c]: dim 8 c + 2 p in bits 4 p .. 4 p + 3 and dim 8 c + 2 p + 1 sixteen bits higher: the pair
//              (w >> 4 p) & 0x000F000F is two neighbouring dims in the two halves, where the packed f16
//              arithmetic wants them;
//   K scales   pairs {f16 d, f16 m} of 32 dims, [4 (pos / 8) + pos % 4][hd / 32][pos / 4 % 2]: the two that a lane
//              of the matrix instructions needs are neighbours;
//   V nibbles  [pos / 4][c][pos % 4]: 16 bytes are four positions of the same dims, since the product over
//              positions needs neighbouring positions in one lane;
//   V scales   [hd / 32][pos / 8][d, m][pos % 8] f16: 16 bytes are eight positions of one group.
// Value = f16(m + q d), rounded once. 5 bits an element. Pages are whole blocks of all layers, so copying a
// page is one contiguous copy. (With one plane of each kind to a page, scales apart from their nibbles, the
// loads of 64 sequences of about 4096 positions alone took 80 us instead of 56 for the nibbles.)
#pragma once

#include "common.hpp"
#include "device.hpp"

namespace aesir {

constexpr int kKv4Group = 32;  // dims per scale

constexpr int kKeys = 32;      // positions of a run, keys of a round of attention

// Attention work is planned for four widths of a column tile ((row, query head) columns; kv4.hip's classes), once
// for the sequences of that class and once (+ kKv4Widths) for all: a captured launch takes the latter, which stays
// right for any later batch.
constexpr int kKv4Widths = 4, kKv4Plans = 2 * kKv4Widths;

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kNone = 0x7FFFFFFF;  // in every field of the records behind the last one

struct Kv4Seq {  // one sequence of the batch
    int32_t slot, length, rows, row0;  // length counts the new rows
    // Widths 0 - 2: first step, steps (of all tiles; 0: not in the plan), steps per workgroup and log2 of the rounds of a
    // step (both the same in all). Width 3: first (tile, split) unit, splits of a tile (0: not in the plan), first
    // partial slot.
    struct {
        int32_t first, count, chunk, shift;
    } plan[kKv4Plans];
};
static_assert(sizeof(Kv4Seq) == 144, "descriptor");

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
    // the run of a position (uniform arguments give a uniform address)
    __device__ char *run(int64_t page, int64_t layer, int head, int pos) const {
        return pool + page * page_bytes + layer * layer_bytes + head * head_bytes() +
               (pos & (page_size() - 1)) / kKeys * run_bytes();
    }
    // places in a run
    __host__ __device__ int run_bytes() const { return kKeys * hd / 4 * 5; }
    __device__ int k_at(int pos, int c) const { return (pos * (hd / 8) + c) * 4; }
    __device__ int k_scale_at(int pos, int grp) const {
        return kKeys * hd / 2 + (((4 * (pos / 8) + pos % 4) * (hd / 32) + grp) * 2 + pos / 4 % 2) * 4;
    }
    __device__ int v_at(int pos, int c) const { return kKeys * hd / 8 * 5 + ((pos / 4 * (hd / 8) + c) * 4 + pos % 4) * 4; }
    __device__ int v_scale_at(int pos, int grp) const {  // d; m is 16 bytes behind
        return kKeys * hd / 8 * 9 + ((grp * (kKeys / 8) + pos / 8) * 16 + pos % 8) * 2;
    }
};

// The two values of nibble pair p of a dword (dims 2 p and 2 p + 1) under scale d and offset m.
__device__ __forceinline__ h16x2 kv4_pair(unsigned w, int p, h16x2 d, h16x2 m) {
    const h16x2 n = as_h2(((w >> (4 * p)) & 0x000F000Fu) | 0x64006400u) - h16x2{(h16)1024.0f, (h16)1024.0f};
    return __builtin_elementwise_fma(n, d, m);  // one rounding
}
__device__ __forceinline__ h16x2 both(h16 x) { return h16x2{x, x}; }

}  // namespace aesir
