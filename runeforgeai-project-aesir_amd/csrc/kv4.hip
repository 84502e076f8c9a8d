// The paged 4-bit KV cache: appending (quantizing) rows, attention over the pages, reading values back, page
// copies, and the C entry points with the bookkeeping of pages and sequences.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>

#include "kernels.hpp"
#include "kv4.hpp"
#include "kv4_pages.hpp"

namespace aesir {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ descriptors to the device
//
// Batch descriptors, page table entries and page moves are written to pinned memory by the host and fetched by
// one small launch: a copy engine's transfer costs more than the few KB it would move, and kernel arguments
// (4 KB) hold the descriptors of 28 sequences at most.
struct Kv4Upload {
    const uint32_t *src;
    uint32_t *dst;      // `words` words of src, then `fill` words of kNone
    int32_t words, fill;
    int32_t *table;     // `updates` pairs (table entry, page) behind them in src
    int32_t updates;
};

__global__ __launch_bounds__(kThreads) void kv4_upload_kernel(Kv4Upload u) {
    const int all = u.words + u.fill;
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < all + u.updates; i += gridDim.x * kThreads) {
        if (i < u.words) {
            u.dst[i] = u.src[i];
        } else if (i < all) {
            u.dst[i] = kNone;
        } else {
            const uint32_t *e = u.src + u.words + 2 * (int64_t)(i - all);
            u.table[e[0]] = (int32_t)e[1];
        }
    }
}

// The record {slot, length or position, rows, first row} that a lane's row belongs to, of records in row order ended by
// ones of kNone; rows 0 past the last. Rows do not fall from lane to lane. Lanes hold a record each and answer the wave's rows
// (few, neighbours, mostly of one record) sequence by sequence: the only memory latency is the load of the records.
__device__ __forceinline__ i32x4 find_row(const char *records, int stride, int row, int lane) {
    i32x4 mine = {0, 0, 0, 0};
    int x = __builtin_amdgcn_readlane(row, 0);  // the least row that is left
    for (int base = 0;; base += kWave) {
        const i32x4 r = *reinterpret_cast<const i32x4 *>(records + (int64_t)(base + lane) * stride);
        for (;;) {
            const int at = __popcll(__ballot(r[3] <= x)) - 1;  // the last record that starts at or before row x
            if (at == kWave - 1) break;                        // or one of the next 64
            if (at >= 0) {
                const i32x4 f = {__builtin_amdgcn_readlane(r[0], at), __builtin_amdgcn_readlane(r[1], at),
                                 __builtin_amdgcn_readlane(r[2], at), __builtin_amdgcn_readlane(r[3], at)};
                if (row >= x) mine = f;
            }
            const int next = __builtin_amdgcn_readlane(r[3], at + 1);  // of the record behind it
            const uint64_t left = __ballot(row >= next);
            if (!left) {
                if (row - mine[3] >= mine[2]) mine[2] = 0;
                return mine;
            }
            x = __builtin_amdgcn_readlane(row, __builtin_ctzll(left));
        }
        // record 63 is row x's unless the next 64 say otherwise
        const i32x4 f = {__builtin_amdgcn_readlane(r[0], kWave - 1), __builtin_amdgcn_readlane(r[1], kWave - 1),
                         __builtin_amdgcn_readlane(r[2], kWave - 1), __builtin_amdgcn_readlane(r[3], kWave - 1)};
        if (row >= x) mine = f;
    }
}

constexpr int kMaxSeqs = 4096;

// ------------------------------------------------------------------ append
//
// One thread per 8 dims of a K and of a V row (16-byte loads); the four lanes of a quad hold a group of 32, whose
// minimum and maximum they exchange by DPP. Four consecutive rows of one head are neighbouring lane groups, so a
// V tile of four positions leaves as one contiguous store. The quantization is exact: scales and levels are the
// nearest ones of the real quotients, ties to even, as their definition says. Bound by instructions (some 20 an element of
// scales, levels and packing): 8192 rows of 8 heads of 128, 13.6 us for 44 MB; one row by the launch and two reads, 3.4 us.

// The f16 nearest a double (ties to even): through f32 rounded to odd, so the second rounding decides alone.
__device__ __forceinline__ h16 nearest_half(double x) {
    float f = (float)x;
    if ((double)f != x) {
        unsigned b = __builtin_bit_cast(unsigned, f);
        if (fabs((double)f) > fabs(x)) b--;
        f = __builtin_bit_cast(float, b | 1u);
    }
    return (h16)f;
}

struct Kv4Code {
    unsigned word;  // eight 4-bit levels in the pool's order
    h16 d, m;       // the group's, in all four lanes of the quad
};

__device__ __forceinline__ Kv4Code kv4_encode(u32x4 x) {
    float v[8], mn = INFINITY, mx = -INFINITY, bad = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const h16x2 h = as_h2(x[i]);
        v[2 * i] = (float)h.x;
        v[2 * i + 1] = (float)h.y;
        if ((x[i] & 0x7C00u) == 0x7C00u || (x[i] & 0x7C000000u) == 0x7C000000u) bad = 1.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        mn = fminf(mn, v[i]);
        mx = fmaxf(mx, v[i]);
    }
    mn = fminf(mn, dpp_f<kDppXor1>(mn));
    mn = fminf(mn, dpp_f<kDppXor2>(mn));
    mx = fmaxf(mx, dpp_f<kDppXor1>(mx));
    mx = fmaxf(mx, dpp_f<kDppXor2>(mx));
    bad = fmaxf(bad, dpp_f<kDppXor1>(bad));
    bad = fmaxf(bad, dpp_f<kDppXor2>(bad));
    Kv4Code c;
    if (bad != 0.0f) {  // the group reads as NaN
        c.word = 0;
        c.d = (h16)0.0f;
        c.m = bits_to_h(0x7E00);
        return c;
    }
    // d from f32, which is within 2^-21 of the quotient: exact but where f16 is subnormal or the quotient lies by a
    // border between two f16 values
    const float step = (mx - mn) * (1.0f / 15.0f);
    h16 d = (h16)step;
    const unsigned tail = __builtin_bit_cast(unsigned, step) & 0x1FFFu;
    if (step < 0x1p-14f || tail - 0xFF0u <= 0x20u) d = nearest_half(((double)mx - (double)mn) / 15.0);
    if (mx > 60000.0f && (double)mn + 15.0 * (double)(float)d > 65504.0) d = bits_to_h((uint16_t)(h_to_bits(d) - 1));
    const float df = (float)d, inv = df > 0.0f ? __builtin_amdgcn_rcpf(df) : 0.0f;
    // t is within 2^-17 of (v - mn) / d. Levels are joined as floats: 16 bits of them are exact
    float q[8], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = (v[i] - mn) * inv;
        q[i] = rintf(t);
        far = fmaxf(far, fabsf(t - q[i]));
    }
    // Where a t could be on the other side of a border between levels, the border is compared in 64 bits (every term is
    // exact there); steps that are subnormal in f16 can leave levels past 15
    if (far > 0.5f - 0x1p-15f || (mx - mn) * inv > 15.5f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float t = (v[i] - mn) * inv, low = floorf(t);
            if (fabsf(t - low - 0.5f) < 0x1p-14f) {
                const double u = (double)v[i] - (double)mn, border = ((double)low + 0.5) * (double)df;
                q[i] = u > border || (u == border && ((int)low & 1)) ? low + 1.0f : low;
            }
            q[i] = fminf(q[i], 15.0f);
        }
    }
    const unsigned even = (unsigned)fmaf(fmaf(fmaf(q[6], 16.0f, q[4]), 16.0f, q[2]), 16.0f, q[0]);
    const unsigned odd = (unsigned)fmaf(fmaf(fmaf(q[7], 16.0f, q[5]), 16.0f, q[3]), 16.0f, q[1]);
    const unsigned w = even | odd << 16;
    c.word = w;
    c.d = d;
    c.m = (h16)mn;
    return c;
}

// What a thread of the append and read kernels works on (grid y: heads): four rows of a head are HD / 2 neighbouring threads.
template <int HD>
struct Kv4Place {
    int row, chunk;
    __device__ __forceinline__ Kv4Place() {
        const unsigned u = blockIdx.x * kThreads + threadIdx.x;
        chunk = (int)(u % (HD / 8));
        row = (int)(u / (HD / 8));
    }
};

struct Kv4AppendArgs {
    const h16 *k, *v;
    int64_t k_stride, v_stride;
    int64_t layer;
    int32_t rows;  // rows of k and v
};

template <bool VEC>
__device__ __forceinline__ u32x4 load8(const h16 *p) {
    if constexpr (VEC) {
        return ld16(p);
    } else {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (unsigned)h_to_bits(p[2 * i]) | (unsigned)h_to_bits(p[2 * i + 1]) << 16;
        return r;
    }
}

template <int HD, bool VEC>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4Dev c, Kv4AppendArgs a) {
    c.hd = HD;
    const int lane = threadIdx.x & 63, head = blockIdx.y;
    const Kv4Place<HD> q;
    const int row = q.row, chunk = q.chunk;
    // requested before the row's place is known; rows past the last repeat it
    const int64_t from = min(row, a.rows - 1), col = head * HD + 8 * chunk;
    const u32x4 kx = load8<VEC>(a.k + from * a.k_stride + col), vx = load8<VEC>(a.v + from * a.v_stride + col);
    const i32x4 s = find_row(reinterpret_cast<const char *>(c.seqs), sizeof(Kv4Seq), row, lane);
    if (row < a.rows && s[2] > 0) {  // uniform over the quad
        const int pos = s[1] - s[2] + (row - s[3]), at = pos % kKeys, grp = chunk / 4;
        char *b = c.run(c.table[(int64_t)s[0] * c.table_stride + (pos >> c.page_shift)], a.layer, head, pos);
        const Kv4Code ck = kv4_encode(kx), cv = kv4_encode(vx);
        *reinterpret_cast<unsigned *>(b + c.k_at(at, chunk)) = ck.word;
        *reinterpret_cast<unsigned *>(b + c.v_at(at, chunk)) = cv.word;
        if (chunk % 4 == 0) {
            *reinterpret_cast<h16x2 *>(b + c.k_scale_at(at, grp)) = h16x2{ck.d, ck.m};
            h16 *p = reinterpret_cast<h16 *>(b + c.v_scale_at(at, grp));
            p[0] = cv.d;
            p[8] = cv.m;
        }
    }
}

// ------------------------------------------------------------------ read
//
// The f16 values of position ranges, one thread per 8 dims of K and V. Bound by memory: 2000 positions of 32 layers and 8
// heads of 128 (344 MB with what it writes) 63 us, 5.5 TB/s.
struct Kv4ReadArgs {
    h16 *k, *v;
    int64_t k_stride, v_stride;
    int64_t layer, layers;
    const Kv4Range *ranges;  // null: `one`
    int32_t all_rows, first_row;  // output rows of a layer, first output row
    Kv4Range one;                 // the only range, without a launch that brings it to the device
};

template <bool VEC>
__device__ __forceinline__ void store8(h16 *p, u32x4 x) {
    if constexpr (VEC) {
        st16(p, x);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[2 * i] = as_h2(x[i]).x;
            p[2 * i + 1] = as_h2(x[i]).y;
        }
    }
}

__device__ __forceinline__ u32x4 kv4_decode(unsigned w, h16 d, h16 m) {
    u32x4 r;
#pragma unroll
    for (int p = 0; p < 4; p++) r[p] = h2_bits(kv4_pair(w, p, both(d), both(m)));
    return r;
}

template <int HD, bool VEC>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(Kv4Dev c, Kv4ReadArgs a) {
    c.hd = HD;
    const int lane = threadIdx.x & 63, head = blockIdx.y;
    const Kv4Place<HD> q;
    const int row = q.row, chunk = q.chunk;
    i32x4 r = {a.one.slot, a.one.pos, row < a.one.rows ? a.one.rows : 0, 0};
    if (a.ranges) r = find_row(reinterpret_cast<const char *>(a.ranges), sizeof(Kv4Range), row, lane);
    if (r[2] == 0) return;
    const int pos = r[1] + (row - r[3]), at = pos % kKeys, grp = chunk / 4;
    const int64_t page = c.table[(int64_t)r[0] * c.table_stride + (pos >> c.page_shift)];
    for (int64_t layer = blockIdx.z; layer < a.layers; layer += gridDim.z) {
        const char *b = c.run(page, a.layer + layer, head, pos);
        const unsigned kw = *reinterpret_cast<const unsigned *>(b + c.k_at(at, chunk));
        const unsigned vw = *reinterpret_cast<const unsigned *>(b + c.v_at(at, chunk));
        const h16x2 ks = *reinterpret_cast<const h16x2 *>(b + c.k_scale_at(at, grp));
        const h16 *p = reinterpret_cast<const h16 *>(b + c.v_scale_at(at, grp));
        const h16 vd = p[0], vm = p[8];
        const int64_t out = layer * a.all_rows + a.first_row + row;
        store8<VEC>(a.k + out * a.k_stride + head * HD + 8 * chunk, kv4_decode(kw, ks.x, ks.y));
        store8<VEC>(a.v + out * a.v_stride + head * HD + 8 * chunk, kv4_decode(vw, vd, vm));
    }
}

// ------------------------------------------------------------------ page copies
//
// 16 KB of a page per workgroup step, four 16-byte loads in flight per thread. Sources and destinations of one
// launch are disjoint. Bound by memory: 32 pages of 2.6 MB 25 us, 6.7 TB/s read and written (the last-level cache holds part
// of them: a copy of 8 GiB reaches 5.2).
constexpr int kCopyChunk = kThreads * 16 * 4;

__global__ __launch_bounds__(kThreads) void kv4_copy_kernel(char *pool, int64_t page_bytes, const PageMove *moves, int n) {
    const int64_t chunks = (page_bytes + kCopyChunk - 1) / kCopyChunk;
    for (int64_t u = blockIdx.x; u < chunks * n; u += gridDim.x) {
        const PageMove m = moves[u / chunks];
        const int64_t at = u % chunks * kCopyChunk + threadIdx.x * 16;
        const char *src = pool + m.src * page_bytes;
        char *dst = pool + m.dst * page_bytes;
        u32x4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (at + i * kThreads * 16 < page_bytes) x[i] = ld16(src + at + i * kThreads * 16);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (at + i * kThreads * 16 < page_bytes) st16(dst + at + i * kThreads * 16, x[i]);
    }
}

// ------------------------------------------------------------------ attention
//
// o = softmax(q k^T / sqrt(hd)) v of the batch's new rows over the positions up to their own, on the matrix
// cores. A column is one (row, query head of the KV head's group) pair. A workgroup takes a tile of 16 NC columns of one
// sequence and KV head, or a piece of its rounds of 32 keys, or pieces of several; its four or eight waves take the rounds in
// turn, each for all columns (a key is unpacked by one wave, once a tile), and meet in LDS at the end; a tile's
// pieces meet in kv4_merge_kernel. Bound by memory where there is much to read: 64 sequences of about 4096 positions, 8 KV
// heads of 128 (335 MB), 63 us and 5 for the merge, 5.4 TB/s; else by the chain of reads that a workgroup starts
// with (records, page ids, the first round) and the launches: 4.5 us for 100 positions.
//
//   scores   S^T = K q^T: a 16-key tile's A operand is unpacked nibbles; lane (i, g) holds key 8 (i / 4) + 4 t + i % 4
//            of the round (t = 0, 1) and the hd / 4 dims from g hd / 4, so one load brings its part of the row
//            and one scale serves it. With that key order a lane's results are the scores of keys 8 g .. 8 g + 7
//   softmax  f32, a running maximum and sum per column (over the lanes i, i + 16, ..: two permlane swaps); the
//            accumulator is rescaled only in rounds that raise a maximum
//   P V      O^T += V^T P^T: a lane's eight probabilities are the B operand as they are (its keys are consecutive), the A
//            operand is eight positions of one dim: the V tiles' layout. A lane unpacks the dims of one 8-dim block
//
// Unpacking gives the exact f16 values that the cache stands for (one packed multiply-add per pair). Probabilities
// are held as f16 times 2^15, 11 bits each, and only those under 2^-39 of the largest can vanish. The sum of a row's is of
// the rounded ones: weights sum to one up to f32 rounding, and finite values give finite outputs. (A second f16 term, as for
// caches of f16 values, would bring an output's error against 64 bits from 1.2 times that of its own rounding to 1.0: far below
// what 4 bits a value cost, for 1 - 11 % of single rows' and drafts' time and a third of a prompt's: 297 -> 403 us below.)
// Positions behind the last visible key are zeroed (their scales), since P = 0 times a NaN there would spread; a
// visible NaN value group (the only non-finite values there are) reaches just the columns that see it.
struct Kv4AttnArgs {
    const h16 *q;
    h16 *out;
    int64_t q_stride, out_stride;
    int64_t layer;
    int32_t rows;  // rows of q and out
    int32_t vec;   // q and out rows 16-byte aligned
    int32_t plan;  // of the batch's plans
    float scale;   // log2(e) / sqrt(hd)
};

constexpr int kMergeWaves = 4;
constexpr int64_t kMergeGrid = 1 << 22;  // workgroups at most: a launch holds under 2^32 threads

// Masks and exponents of the unpacking, one in a scalar and one in a vector register: as literals each pair would
// take an AND and an OR, since one instruction takes no two literals here.
struct Kv4Magic {
    unsigned low = 0x000F000Fu, high = 0x00F000F0u, one = 0x64006400u;
    __device__ __forceinline__ Kv4Magic() { asm("" : "+s"(low), "+s"(high), "+v"(one)); }
};

// The values of nibble P of both halves of x under scales d and offsets m.
template <int P>
__device__ __forceinline__ h16x2 kv4_values(const Kv4Magic &c, unsigned x, h16x2 d, h16x2 m) {
    h16x2 n;
    if constexpr (P % 2 == 0) {
        n = as_h2(((x >> (4 * P)) & c.low) | c.one) - both((h16)1024.0f);
    } else {  // 1024 + 16 n: no shift, the multiply-add undoes both exactly
        n = __builtin_elementwise_fma(as_h2(((x >> (4 * (P - 1))) & c.high) | c.one), both((h16)0.0625f), both((h16)-64.0f));
    }
    return __builtin_elementwise_fma(n, d, m);
}

// A lane's byte offsets in a run.
template <int HD>
struct Kv4Lane {
    static constexpr int NJ = HD / 32, NB = NJ == 8 ? 2 : 1;
    unsigned k, ks, v[NB], vs[NB];  // key 8 (i / 4) + i % 4 (the second tile's four behind); 8-dim blocks and their scales

    __device__ __forceinline__ Kv4Lane(const Kv4Dev &c, int i, int g) {
        const int key = 8 * (i / 4) + i % 4;
        k = c.k_at(key, g * NJ);
        ks = c.k_scale_at(key, g * NJ / 4);
#pragma unroll
        for (int x = 0; x < NB; x++) {
            const int block = NJ < 4 ? i % (4 * NJ) : i + 16 * x;
            v[x] = c.v_at(8 * g, block);
            vs[x] = c.v_scale_at(8 * g, block / 4);
        }
    }
};

// One lane's share of 32 keys. NT: loaded past the caches, for runs that one workgroup alone reads (64 sequences of about
// 4096 positions: 74 -> 69 us); prompts' tiles share them (307 -> 322 us).
template <int HD, bool NT>
struct Kv4Round {
    static constexpr int NJ = HD / 32, NG = NJ == 8 ? 2 : 1, NB = NJ == 8 ? 2 : 1;
    unsigned k[2][NJ];
    h16x2 ks[2][NG];
    u32x4 v[NB][2], vd[NB], vm[NB];

    static __device__ __forceinline__ u32x4 ld(const char *p) { return NT ? ld16_stream(p) : ld16(p); }

    __device__ __forceinline__ void load(const char *b, const Kv4Lane<HD> &o) {  // b: the run (uniform)
        load_k(b, o, 0);
        load_k(b, o, 1);
        load_k_scales(b, o);
#pragma unroll
        for (int x = 0; x < NB; x++) load_v(b, o, x);
    }
    __device__ __forceinline__ void load_k(const char *b, const Kv4Lane<HD> &o, int t) {  // 16 keys
        const char *p = b + (size_t)(o.k + t * 2 * HD);
        if constexpr (NJ == 1) {
            k[t][0] = *reinterpret_cast<const unsigned *>(p);
        } else if constexpr (NJ == 2) {
            const u32x2 x = *reinterpret_cast<const u32x2 *>(p);
            k[t][0] = x.x;
            k[t][1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < NJ; j += 4) {
                const u32x4 x = ld(p + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; e++) k[t][j + e] = x[e];
            }
        }
    }
    __device__ __forceinline__ void load_k_scales(const char *b, const Kv4Lane<HD> &o) {
#pragma unroll
        for (int x = 0; x < NG; x++) {
            const u32x2 s = *reinterpret_cast<const u32x2 *>(b + (size_t)(o.ks + 8 * x));
            ks[0][x] = as_h2(s.x);
            ks[1][x] = as_h2(s.y);
        }
    }
    __device__ __forceinline__ void load_v(const char *b, const Kv4Lane<HD> &o, int x) {  // 16 8-dim blocks
#pragma unroll
        for (int h = 0; h < 2; h++) v[x][h] = ld(b + (size_t)(o.v[x] + h * 2 * HD));
        vd[x] = ld(b + (size_t)o.vs[x]);
        vm[x] = ld(b + (size_t)(o.vs[x] + 16));
    }

    // The A operand of key tile t's dims 8 j .. of the lane's share.
    __device__ __forceinline__ u32x4 key_operand(const Kv4Magic &c, int t, int j) const {
        const h16x2 d = both(ks[t][j * NG / NJ].x), m = both(ks[t][j * NG / NJ].y);
        return {h2_bits(kv4_values<0>(c, k[t][j], d, m)), h2_bits(kv4_values<1>(c, k[t][j], d, m)),
                h2_bits(kv4_values<2>(c, k[t][j], d, m)), h2_bits(kv4_values<3>(c, k[t][j], d, m))};
    }

    // Zeroes the values of keys k0 + e >= keys and of NaN groups among the others; bit e of the result: key k0 + e's
    // group of value block x is NaN.
    __device__ __forceinline__ unsigned hide(int x, int k0, int keys) {
        unsigned bad = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const unsigned half = 0xFFFFu << (16 * (e % 2));
            const bool nan = ((vm[x][e / 2] >> (16 * (e % 2))) & 0x7FFFu) > 0x7C00u, hidden = k0 + e >= keys;
            if (nan || hidden) {
                vd[x][e / 2] &= ~half;
                vm[x][e / 2] &= ~half;
            }
            if (nan && !hidden) bad |= 1u << e;
        }
        return bad;
    }

    // f(p, half, A operand) for every accumulator of value block x: eight positions of one dim each.
    template <class F>
    __device__ __forceinline__ void value_operands(const Kv4Magic &c, int x, int i, F f) const {
        constexpr int NP = NJ < 4 ? NJ : 4;
        const int shift = NJ < 4 ? 4 * NJ * (i / (4 * NJ)) : 0;
        unsigned lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {  // positions 2 e, 2 e + 1: low halves (even dims) and high halves
            const unsigned w0 = v[x][e / 2][2 * (e % 2)] >> shift, w1 = v[x][e / 2][2 * (e % 2) + 1] >> shift;
            lo[e] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
            hi[e] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
        }
        auto step = [&](auto pc) {
            constexpr int P = decltype(pc)::value;
            if constexpr (P < NP) {
                u32x4 a, b;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    a[e] = h2_bits(kv4_values<P>(c, lo[e], as_h2(vd[x][e]), as_h2(vm[x][e])));
                    b[e] = h2_bits(kv4_values<P>(c, hi[e], as_h2(vd[x][e]), as_h2(vm[x][e])));
                }
                f(P, 0, a);
                f(P, 1, b);
            }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
    }
};

// What attention needs of a sequence of the batch: its record and one of its plans.
struct Kv4Found {
    int slot, length, rows, row0;
    int first, count, chunk, shift, own;
    __device__ __forceinline__ int tile_steps() const { return (((length + kKeys - 1) / kKeys - 1) >> shift) + 1; }
};

// 64 records, one a lane.
struct Kv4Records {
    i32x4 s, plan;
    __device__ __forceinline__ Kv4Records(const Kv4Seq *seqs, int p, int at) {
        const i32x4 *r = reinterpret_cast<const i32x4 *>(seqs + at);
        s = r[0];
        plan = r[1 + p];
    }
};

// The last sequence whose row0 (by_row) or plan's first is at or before x; rows and count 0 where there is none. Lanes
// hold a record each (r: the first 64); the whole wave calls it.
__device__ __forceinline__ Kv4Found find_seq(Kv4Records r, const Kv4Seq *seqs, int plan, int x, bool by_row, int lane) {
    Kv4Found f{};
    for (int base = kWave;; base += kWave) {
        const int at = __popcll(__ballot((by_row ? r.s[3] : r.plan[0]) <= x)) - 1;
        if (at >= 0) {
            f.slot = __builtin_amdgcn_readlane(r.s[0], at);
            f.length = __builtin_amdgcn_readlane(r.s[1], at);
            f.rows = __builtin_amdgcn_readlane(r.s[2], at);
            f.row0 = __builtin_amdgcn_readlane(r.s[3], at);
            f.first = __builtin_amdgcn_readlane(r.plan[0], at);
            f.count = __builtin_amdgcn_readlane(r.plan[1], at);
            f.chunk = __builtin_amdgcn_readlane(r.plan[2], at);
            const int z = __builtin_amdgcn_readlane(r.plan[3], at);
            f.shift = z & 255;
            f.own = z >> 8;
        }
        if (at < kWave - 1) break;
        r = Kv4Records(seqs, plan, base + lane);
    }
    return f;
}

// Two f16 per dword, 1 where bit 2 e (2 e + 1) of `bits` is set, as an operand of eight positions.
__device__ __forceinline__ u32x4 ones_operand(unsigned bits) {
    u32x4 r;
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = (bits >> (2 * e) & 1 ? 0x3C00u : 0u) | (bits >> (2 * e + 1) & 1 ? 0x3C000000u : 0u);
    return r;
}

// One wave's columns: 16 NC of them, column i of each 16 in lanes i, i + 16, ..
template <int HD, int NC>
struct Kv4Cols {
    static constexpr int NJ = HD / 32, NP = NJ < 4 ? NJ : 4, NB = NJ == 8 ? 2 : 1;
    u32x4 q[NC][NJ];  // dims g HD / 4 + 8 j .. of the column's query
    int limit[NC];    // last position the column sees, -1 for none
    f32x4 acc[NC][NB][NP][2];
    float m[NC], l[NC];  // running maximum (the column's), sum (the lane's share, times 2^15 as acc)

    __device__ __forceinline__ void start(const Kv4AttnArgs &a, const Kv4Found &s, int first, int G, int kvh, int i, int g) {
#pragma unroll
        for (int t = 0; t < NC; t++) {
            const int col = first + 16 * t + i, row = col / G;
            const bool live = col < s.rows * G && s.row0 + row < a.rows;
            limit[t] = live ? s.length - s.rows + row : -1;
            const h16 *p = a.q + (int64_t)(s.row0 + row) * a.q_stride + (kvh * G + col % G) * HD + g * (HD / 4);
#pragma unroll
            for (int j = 0; j < NJ; j++) q[t][j] = !live ? u32x4{0, 0, 0, 0} : a.vec ? ld16(p + 8 * j) : load8<false>(p + 8 * j);
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int x = 0; x < NB; x++)
#pragma unroll
                for (int p = 0; p < NP; p++) acc[t][x][p][0] = acc[t][x][p][1] = f32x4{0, 0, 0, 0};
        }
    }

    // Scores that a column does not see; sc[t][.][e] is that of key k0 + 32 (t / 2) + 4 (t % 2) + e.
    template <int T>
    __device__ __forceinline__ void mask(f32x4 (&sc)[T][NC], int k0) const {
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int x = 0; x < NC; x++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (k0 + kKeys * (t / 2) + 4 * (t % 2) + e > limit[x]) sc[t][x][e] = -INFINITY;
    }

    // The softmax step of T / 2 rounds; the probabilities as P V's B operands.
    template <int T>
    __device__ __forceinline__ void softmax(const f32x4 (&sc)[T][NC], float scale, u32x4 (&pb)[T / 2][NC]) {
#pragma unroll
        for (int x = 0; x < NC; x++) {
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < T; t++) mx = fmaxf(mx, fmaxf(fmaxf(sc[t][x][0], sc[t][x][1]), fmaxf(sc[t][x][2], sc[t][x][3])));
            mx = swap_pair_max<32>(swap_pair_max<16>(mx));
            if (__any(mx > m[x])) {
                const float up = fmaxf(m[x], mx), ref = up == -INFINITY ? 0.0f : up;
                const float al = __builtin_amdgcn_exp2f((m[x] - ref) * scale);
                l[x] *= al;
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int p = 0; p < NP; p++) {
                        acc[x][b][p][0] *= al;
                        acc[x][b][p][1] *= al;
                    }
                m[x] = up;
            }
            const float ref = m[x] == -INFINITY ? 0.0f : m[x];
#pragma unroll
            for (int r = 0; r < T / 2; r++) {
                float pr[8];
#pragma unroll
                for (int e = 0; e < 8; e++) pr[e] = __builtin_amdgcn_exp2f(fmaf(sc[2 * r + e / 4][x][e % 4] - ref, scale, 15.0f));
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const h16x2 w = {(h16)pr[2 * e], (h16)pr[2 * e + 1]};
                    pb[r][x][e] = h2_bits(w);
                    // the weights that P V uses, so that they sum to one (two products with one; subnormals count)
                    l[x] = __builtin_amdgcn_fdot2(w, both((h16)1.0f), l[x], false);
                }
            }
        }
    }

    // NaN for the columns that see a NaN group of value block b, in its dims; bad: the operand of ones at such positions.
    __device__ __forceinline__ void spread_nan(int b, u32x4 bad, int k0) {
#pragma unroll
        for (int x = 0; x < NC; x++) {
            const int n = min(max(limit[x] - k0 + 1, 0), 8);  // positions the column sees
            const f32x4 seen = mfma16x16x32(bad, ones_operand((1u << n) - 1), f32x4{0, 0, 0, 0});
#pragma unroll
            for (int p = 0; p < NP; p++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (seen[e] > 0.0f) acc[x][b][p][0][e] = acc[x][b][p][1][e] = NAN;
        }
    }

    __device__ __forceinline__ void sum_lanes() {
#pragma unroll
        for (int t = 0; t < NC; t++) {
            l[t] = swap_pair_sum<16>(l[t], l[t]);
            l[t] = swap_pair_sum<32>(l[t], l[t]);
        }
    }
};

// The column tile widths of the launches: 16, 32 or 64 ((row, query head of a group) pairs), and for prompts 256; at head_dim
// 256 16 and 128.
__host__ __device__ constexpr int kv4_width(int v, int hd) { return v < 3 ? 16 << v : hd == 256 ? 128 : 256; }

// The dim of accumulator (x, p, half) in matrix row r.
template <int HD>
__device__ __forceinline__ int out_dim(int r, int x, int p, int half) {
    constexpr int NJ = HD / 32;
    if constexpr (NJ < 4) return 8 * (r % (4 * NJ)) + 2 * (NJ * (r / (4 * NJ)) + p) + half;
    return 8 * (r + 16 * x) + 2 * p + half;
}

template <int HD, int NC, int NW>
__global__ __launch_bounds__(NW *kWave, NC == 1 && HD <= 128 && NW == 4 ? 3 : 1) void kv4_attention_kernel(Kv4Dev c, Kv4AttnArgs a) {
    constexpr int W = 16 * NC;
    constexpr int NJ = HD / 32, NP = NJ < 4 ? NJ : 4, NB = Kv4Round<HD, true>::NB;
    constexpr int LD = HD + 4;  // LDS row of a column
    __shared__ float ml[NW][W][2];
    __shared__ __align__(16) float ox[NW][16][LD];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = c.nq / c.nkv;
    const Kv4Lane<HD> place(c, i, g);
    const Kv4Magic magic;
    Kv4Records records(c.seqs, a.plan, lane);
    const int chunk = __builtin_amdgcn_readfirstlane(records.plan[2]);
    if (chunk == kNone) return;  // no batch
    // Workgroup b of a KV head takes steps b chunk .. (b + 1) chunk - 1 of the batch's tiles one behind the other, in
    // pieces that end where a tile does. (A step is a round, or 2^shift of them in batches of billions of rounds.)
    // A captured grid may be larger than a later batch's: its starts can pass 32 bits. 2^30 is behind every last step.
    auto start = [&](unsigned x) { return (int)min((int64_t)(x / (unsigned)c.nkv) * chunk, (int64_t)1 << 30); };
    unsigned u = blockIdx.x;
    int at = start(u), end = at + chunk;
    for (;;) {
        const int kvh = (int)(u % (unsigned)c.nkv), b = (int)(u / (unsigned)c.nkv);
        const Kv4Found s = find_seq(records, c.seqs, a.plan, at, false, lane);
        const int local = at - s.first;
        if (local >= s.count) break;  // past the last step
        const int cols = s.rows * G, steps = s.tile_steps();
        const int tile = local / steps, begin = local - tile * steps, stop = min(steps, begin + end - at);
        const bool complete = begin == 0 && stop == steps;
        const int partial = 2 * b + (at == b * chunk ? 0 : 1);  // a workgroup cuts two tiles at most
        at += stop - begin;
        const bool done = at >= end || (s.own && at - s.first >= s.count);  // (the next sequence starts in another)
        const int before = s.length - s.rows;
        const int low = before + tile * W / G;                                    // last position of the first column
        const int keys = before + min(s.rows - 1, (tile * W + W - 1) / G) + 1;     // positions the tile sees
        const int rounds = (keys + kKeys - 1) / kKeys;
        const int r0 = (begin << s.shift) + wave, r1 = min(rounds, stop << s.shift);

        // pages of this wave's next 64 rounds, one a lane
        const int32_t *table = c.table + (int64_t)s.slot * c.table_stride;
        auto page_ids = [&](int r) { return table[min(r + lane * NW, rounds - 1) * kKeys >> c.page_shift]; };
        int pages = page_ids(r0);
        Kv4Cols<HD, NC> own;
        own.start(a, s, tile * W, G, kvh, i, g);

        auto fetch = [&](int x, Kv4Round<HD, true> &d) {  // the wave's x-th round
            const int page = __builtin_amdgcn_readlane(pages, x & (kWave - 1));
            d.load(c.run(page, a.layer, kvh, (r0 + x * NW) * kKeys), place);
        };
        auto round = [&](int r, Kv4Round<HD, true> &d) {
            f32x4 sc[2][NC];
#pragma unroll
            for (int t = 0; t < 2; t++) {
#pragma unroll
                for (int x = 0; x < NC; x++) sc[t][x] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const u32x4 ka = d.key_operand(magic, t, j);
#pragma unroll
                    for (int x = 0; x < NC; x++) sc[t][x] = mfma16x16x32(ka, own.q[x][j], sc[t][x]);
                }
            }
            const bool whole = r * kKeys + kKeys - 1 <= low;  // every column sees every key (uniform)
            const int k0 = r * kKeys + 8 * g;
            unsigned bad[NB] = {};
            if (!whole) {
                own.mask(sc, k0);
#pragma unroll
                for (int x = 0; x < NB; x++) bad[x] = d.hide(x, k0, keys);
            }
            u32x4 pb[1][NC];
            own.softmax(sc, a.scale, pb);
#pragma unroll
            for (int b = 0; b < NB; b++) {
                d.value_operands(magic, b, i, [&](int p, int half, u32x4 va) {
#pragma unroll
                    for (int x = 0; x < NC; x++) own.acc[x][b][p][half] = mfma16x16x32(va, pb[0][x], own.acc[x][b][p][half]);
                });
                if (!whole && __any(bad[b] != 0)) own.spread_nan(b, ones_operand(bad[b]), k0);
            }
        };
        // A round's loads are issued before the round ahead of it is computed. The last round issues its own again (they
        // hit the cache): a load on one path only would make every wait behind it wait for all.
        const int mine = r0 < r1 ? (r1 - r0 + NW - 1) / NW : 0;
        if (mine > 0) {
            Kv4Round<HD, true> cur, next;
            fetch(0, cur);
            for (int x = 0; x < mine; x++) {
                const int y = min(x + 1, mine - 1);
                if ((y & (kWave - 1)) == 0 && y > x) pages = page_ids(r0 + y * NW);
                fetch(y, next);
                round(r0 + x * NW, cur);
                cur = next;
            }
        }

        // the waves meet: maxima and sums of all columns, then 16 columns of accumulators at a time
        own.sum_lanes();
#pragma unroll
        for (int t = 0; t < NC; t++) {
            if (g == 0) {
                ml[wave][16 * t + i][0] = own.m[t];
                ml[wave][16 * t + i][1] = own.l[t];
            }
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NC; t++) {
            float up = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; w++) up = fmaxf(up, ml[w][16 * t + i][0]);
            const float ref = up == -INFINITY ? 0.0f : up, scale = __builtin_amdgcn_exp2f((own.m[t] - ref) * a.scale);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int x = 0; x < NB; x++)
#pragma unroll
                    for (int p = 0; p < NP; p++) {
                        float *o = &ox[wave][i][out_dim<HD>(4 * g + e, x, p, 0)];
                        o[0] = own.acc[t][x][p][0][e] * scale;
                        o[1] = own.acc[t][x][p][1][e] * scale;
                    }
            __syncthreads();
            // thread: D dims of one column
            constexpr int T = NW * 4, D = HD / T;
            const int col = threadIdx.x / T, dim = threadIdx.x % T * D, gc = tile * W + 16 * t + col, row = gc / G;
            if (gc < cols && s.row0 + row < a.rows) {
                float M = -INFINITY, L = 0.0f, o[D] = {};
#pragma unroll
                for (int w = 0; w < NW; w++) M = fmaxf(M, ml[w][16 * t + col][0]);
                const float mref = M == -INFINITY ? 0.0f : M;
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    L += ml[w][16 * t + col][1] * __builtin_amdgcn_exp2f((ml[w][16 * t + col][0] - mref) * a.scale);
#pragma unroll
                    for (int d = 0; d < D; d++) o[d] += ox[w][col][dim + d];
                }
                if (complete) {
                    h16 *p = a.out + (int64_t)(s.row0 + row) * a.out_stride + (kvh * G + gc % G) * HD + dim;
                    h16 r16[D];
#pragma unroll
                    for (int d = 0; d < D; d++) r16[d] = (h16)(o[d] / L);
                    if (a.vec) {
                        __builtin_memcpy(__builtin_assume_aligned(p, 2 * D < 16 ? 2 * D : 16), r16, sizeof r16);
                    } else {
                        for (int d = 0; d < D; d++) p[d] = r16[d];
                    }
                } else {
                    const int64_t to = ((int64_t)partial * c.nkv + kvh) * W + 16 * t + col;
                    if (threadIdx.x % T == 0) *reinterpret_cast<float2 *>(c.part_ml + 2 * to) = float2{M, L};
                    __builtin_memcpy(__builtin_assume_aligned(c.part + to * HD + dim, 4 * D < 16 ? 4 * D : 16), o, sizeof o);
                }
            }
            __syncthreads();  // ox (and, before the next piece, ml) is rewritten
        }
        if (done) {
            if (a.plan < kKv4Widths) break;  // the grid is the batch's own
            u += gridDim.x;
            at = start(u);
            end = at + chunk;
        }
        records = Kv4Records(c.seqs, a.plan, lane);
    }
}

// Prompts: units of 256 columns (128 at head_dim 256), eight waves with 32 (16) of them each. The waves unpack RS rounds of keys
// and values between them, each operand once, into LDS in the order in which the matrix instructions take them (1 KB an
// operand, 16 bytes a lane, no bank conflicts); every wave then runs those rounds over its own columns, so unpacking costs
// an eighth a column and the waves never meet but at the barrier between stages. Two stages of LDS: the next is loaded
// during one and unpacked behind it. 2048 rows of 8192 positions (32 query heads of 128, 8 KV heads): 300 us, 800 TFLOP/s;
// two waves to a SIMD issue vector instructions half of the time and matrix instructions a third, mostly not at once
// (raising the priority of either phase, or sums as a product with ones, changed nothing: 296 - 310 us).
template <int HD>
__global__ __launch_bounds__(8 * kWave) void kv4_prompt_kernel(Kv4Dev c, Kv4AttnArgs a) {
    constexpr int V = 3, W = kv4_width(V, HD), NC = W / 128, NJ = HD / 32, NP = NJ < 4 ? NJ : 4;
    constexpr int NB = Kv4Round<HD, false>::NB, NG = Kv4Round<HD, false>::NG;
    constexpr int RS = HD == 256 ? 2 : 4, PARTS = 8 / RS;  // rounds per stage; waves that unpack a round
    constexpr int NK = 2 * NJ;                             // key operands of a round, and value operands
    constexpr int KR = 2;                                  // rounds per softmax step
    __shared__ __align__(16) u32x4 lds[2][RS][2 * NK][kWave];
    __shared__ __align__(16) u32x4 bad_at[2][RS][NB][kWave];
    __shared__ int any_bad[2][RS][NB];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = c.nq / c.nkv;
    const Kv4Lane<HD> place(c, i, g);
    const Kv4Magic magic;
    const int mr = wave / PARTS, part = wave % PARTS;  // the round of a stage this wave unpacks, and what of it
    for (unsigned u = blockIdx.x;; u += gridDim.x) {
        const int kvh = (int)(u % (unsigned)c.nkv), unit = (int)(u / (unsigned)c.nkv);
        const Kv4Found s = find_seq(Kv4Records(c.seqs, a.plan, lane), c.seqs, a.plan, unit, false, lane);
        const int splits = s.count, cols = s.rows * G, tiles = (cols + W - 1) / W, local = unit - s.first;
        if (local >= tiles * splits) break;
        const int tile = tiles - 1 - local / splits, split = local % splits;  // the longest first
        const int before = s.length - s.rows;
        const int low = before + tile * W / G, keys = before + min(s.rows - 1, (tile * W + W - 1) / G) + 1;
        const int rounds = (keys + kKeys - 1) / kKeys, per = ((rounds + splits - 1) / splits + RS - 1) / RS * RS;
        const int r0 = split * per, r1 = min(rounds, r0 + per), stages = r0 < r1 ? (r1 - r0 + RS - 1) / RS : 0;
        // this wave's columns: the first sees positions up to low_w, all together keys_w (none: 0)
        const int first = tile * W + wave * 16 * NC;
        const int low_w = before + first / G;
        const int keys_w = first < cols ? before + min(s.rows - 1, (first + 16 * NC - 1) / G) + 1 : 0;

        const int32_t *table = c.table + (int64_t)s.slot * c.table_stride;
        auto page_ids = [&](int st) { return table[min(r0 + (st + lane) * RS + mr, rounds - 1) * kKeys >> c.page_shift]; };
        int pages = page_ids(0);
        Kv4Cols<HD, NC> own;
        own.start(a, s, first, G, kvh, i, g);
        u32x4 raw[4];  // the next stage's share: keys and scales, or values and theirs
        auto fetch = [&](int st) {  // (rounds past the last one's page repeat it; their keys are hidden below)
            if ((st & (kWave - 1)) == 0 && st > 0) pages = page_ids(st);
            const int page = __builtin_amdgcn_readlane(pages, st & (kWave - 1));
            const char *b = c.run(page, a.layer, kvh, min(r0 + st * RS + mr, rounds - 1) * kKeys);
            Kv4Round<HD, false> d;
            if constexpr (PARTS == 2) {
                if (part == 0) {
                    d.load_k(b, place, 0);
                    d.load_k(b, place, 1);
                    d.load_k_scales(b, place);
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        raw[0][j] = d.k[0][j];
                        raw[1][j] = d.k[1][j];
                    }
                    raw[2][0] = h2_bits(d.ks[0][0]);
                    raw[2][1] = h2_bits(d.ks[1][0]);
                } else {
                    d.load_v(b, place, 0);
                    raw[0] = d.v[0][0];
                    raw[1] = d.v[0][1];
                    raw[2] = d.vd[0];
                    raw[3] = d.vm[0];
                }
            } else {
                if (part < 2) {
                    part == 0 ? d.load_k(b, place, 0) : d.load_k(b, place, 1);
                    d.load_k_scales(b, place);
#pragma unroll
                    for (int j = 0; j < NJ; j++) raw[j / 4][j % 4] = part == 0 ? d.k[0][j] : d.k[1][j];
#pragma unroll
                    for (int x = 0; x < NG; x++) raw[2][x] = h2_bits(part == 0 ? d.ks[0][x] : d.ks[1][x]);
                } else {
                    part == 2 ? d.load_v(b, place, 0) : d.load_v(b, place, NB - 1);
                    raw[0] = part == 2 ? d.v[0][0] : d.v[NB - 1][0];
                    raw[1] = part == 2 ? d.v[0][1] : d.v[NB - 1][1];
                    raw[2] = part == 2 ? d.vd[0] : d.vd[NB - 1];
                    raw[3] = part == 2 ? d.vm[0] : d.vm[NB - 1];
                }
            }
        };
        auto unpack = [&](int st) {
            u32x4(&to)[2 * NK][kWave] = lds[st & 1][mr];
            const int r = r0 + st * RS + mr;
            Kv4Round<HD, false> d;
            if (part < PARTS / 2) {
                constexpr int TILES = PARTS == 2 ? 2 : 1;  // key tiles of this wave
#pragma unroll
                for (int t = 0; t < TILES; t++) {
#pragma unroll
                    for (int j = 0; j < NJ; j++) d.k[t][j] = TILES == 2 ? raw[t][j] : raw[j / 4][j % 4];
#pragma unroll
                    for (int x = 0; x < NG; x++) d.ks[t][x] = as_h2(raw[2][TILES == 2 ? t : x]);
#pragma unroll
                    for (int j = 0; j < NJ; j++) to[(TILES == 2 ? t : part) * NJ + j][lane] = d.key_operand(magic, t, j);
                }
            } else {
                const int x = part - PARTS / 2;  // the value block
                d.v[0][0] = raw[0];
                d.v[0][1] = raw[1];
                d.vd[0] = raw[2];
                d.vm[0] = raw[3];
                if (r * kKeys + kKeys - 1 > low) {  // not seen whole by every column of the tile
                    const unsigned bad = d.hide(0, r * kKeys + 8 * g, keys);
                    const bool any = __any(bad != 0);
                    if (any) bad_at[st & 1][mr][x][lane] = ones_operand(bad);
                    if (lane == 0) any_bad[st & 1][mr][x] = any;
                }
                d.value_operands(magic, 0, i, [&](int p, int half, u32x4 v) { to[NK + (x * NP + p) * 2 + half][lane] = v; });
            }
        };

        if (stages > 0) {
            fetch(0);
            unpack(0);
        }
        for (int st = 0; st < stages; st++) {
            if (st + 1 < stages) fetch(st + 1);
            __syncthreads();  // stage st is in LDS, and stage st - 1 is used up
            for (int x = 0; x < RS; x += KR) {  // (rounds past the last are hidden keys)
                const int r = r0 + st * RS + x;
                if (r >= r1 || r * kKeys >= keys_w) break;
                f32x4 sc[2 * KR][NC];
#pragma unroll
                for (int t = 0; t < 2 * KR; t++) {
#pragma unroll
                    for (int y = 0; y < NC; y++) sc[t][y] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        const u32x4 ka = lds[st & 1][x + t / 2][t % 2 * NJ + j][lane];
#pragma unroll
                        for (int y = 0; y < NC; y++) sc[t][y] = mfma16x16x32(ka, own.q[y][j], sc[t][y]);
                    }
                }
                const int k0 = r * kKeys + 8 * g, last = (r + KR) * kKeys - 1;
                if (last > low_w) own.mask(sc, k0);
                u32x4 pb[KR][NC];
                own.softmax(sc, a.scale, pb);
#pragma unroll
                for (int z = 0; z < KR; z++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
#pragma unroll
                        for (int p = 0; p < NP; p++)
#pragma unroll
                            for (int half = 0; half < 2; half++) {
                                const u32x4 va = lds[st & 1][x + z][NK + (b * NP + p) * 2 + half][lane];
#pragma unroll
                                for (int y = 0; y < NC; y++) own.acc[y][b][p][half] = mfma16x16x32(va, pb[z][y], own.acc[y][b][p][half]);
                            }
                    }
                if (last > low) {
#pragma unroll
                    for (int z = 0; z < KR; z++)
#pragma unroll
                        for (int b = 0; b < NB; b++)
                            if ((r + z + 1) * kKeys - 1 > low && __builtin_amdgcn_readfirstlane(any_bad[st & 1][x + z][b]))
                                own.spread_nan(b, bad_at[st & 1][x + z][b][lane], k0 + z * kKeys);
                }
            }
            if (st + 1 < stages) unpack(st + 1);
        }
        __syncthreads();  // the next unit's first stage is written over this one's

        own.sum_lanes();
        constexpr int D = 2 * NP;  // neighbouring dims of a lane
#pragma unroll
        for (int t = 0; t < NC; t++) {
            const int col = first + 16 * t + i, row = col / G;
            if (own.limit[t] < 0) continue;
            const int64_t at = ((int64_t)(s.chunk + local) * c.nkv + kvh) * W + col % W;
            if (splits > 1 && g == 0) *reinterpret_cast<float2 *>(c.part_ml + 2 * at) = float2{own.m[t], own.l[t]};
#pragma unroll
            for (int x = 0; x < NB; x++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    float o[D];
#pragma unroll
                    for (int d2 = 0; d2 < D; d2++) o[d2] = own.acc[t][x][d2 / 2][d2 % 2][e];
                    const int dim = out_dim<HD>(4 * g + e, x, 0, 0);
                    if (splits == 1) {
                        h16 *p = a.out + (int64_t)(s.row0 + row) * a.out_stride + (kvh * G + col % G) * HD + dim;
                        h16 r16[D];
#pragma unroll
                        for (int d2 = 0; d2 < D; d2++) r16[d2] = (h16)(o[d2] / own.l[t]);
                        if (a.vec) {
                            __builtin_memcpy(__builtin_assume_aligned(p, 2 * D), r16, sizeof r16);
                        } else {
                            for (int d2 = 0; d2 < D; d2++) p[d2] = r16[d2];
                        }
                    } else {
                        __builtin_memcpy(__builtin_assume_aligned(c.part + at * HD + dim, 4 * D < 16 ? 4 * D : 16), o, sizeof o);
                    }
                }
        }
    }
}

// The partials of a column joined: o = sum_s 2^(scale (m_s - M)) acc_s / sum_s 2^(scale (m_s - M)) l_s. MW waves per
// (row, query head) take them in turn, eight a step, all requested before their weights are known.
template <int HD, int V, int MW>
__global__ __launch_bounds__(kMergeWaves *kWave) void kv4_merge_kernel(Kv4Dev c, Kv4AttnArgs a) {
    constexpr int D = HD >= kWave ? HD / kWave : 1, W = kv4_width(V, HD), B = 8;  // dims per lane
    __shared__ float ox[kMergeWaves][HD], mx[kMergeWaves], lx[kMergeWaves];
    const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = all % MW;
    const int G = c.nq / c.nkv;
    const unsigned columns = (unsigned)a.rows * (unsigned)c.nq;
    for (unsigned u = blockIdx.x * (kMergeWaves / MW) + all / MW; u < columns; u += gridDim.x * (kMergeWaves / MW)) {
        const int row = (int)(u / (unsigned)c.nq), head = (int)(u % (unsigned)c.nq);
        const Kv4Found s = find_seq(Kv4Records(c.seqs, a.plan, lane), c.seqs, a.plan, row, true, lane);
        // (MW of 4: uniform over the workgroup; MW of 1: no barrier follows)
        if (row - s.row0 >= s.rows || s.count == 0) continue;
        const int col = (row - s.row0) * G + head % G, tile = col / W;
        int first, splits, start = 0;  // partial slots: first, then start + 2 x (width 3: first + x)
        if constexpr (V < 3) {
            const int steps = s.tile_steps(), from = s.first + tile * steps;
            const int b0 = from / s.chunk;
            splits = (from + steps - 1) / s.chunk - b0 + 1;
            first = 2 * b0 + (from % s.chunk ? 1 : 0);
            start = 2 * b0;
        } else {
            splits = s.count;
            first = s.chunk + ((s.rows * G + W - 1) / W - 1 - tile) * splits;
        }
        if (splits <= 1) continue;
        auto slot = [&](int x) {
            const int p = V == 3 ? first + x : x == 0 ? first : start + 2 * x;
            return ((int64_t)p * c.nkv + head / G) * W + col % W;
        };
        const int dim = HD >= kWave ? lane * D : lane % HD;
        float M = -INFINITY, L = 0.0f, o[D] = {};
        for (int base = 0; base < splits; base += MW * B) {
            float p[B][D];
            float2 e[B];
#pragma unroll
            for (int j = 0; j < B; j++) {
                const int64_t at = slot(min(base + wave + MW * j, splits - 1));
                e[j] = *reinterpret_cast<const float2 *>(c.part_ml + 2 * at);
                __builtin_memcpy(p[j], __builtin_assume_aligned(c.part + at * HD + dim, 4 * D < 16 ? 4 * D : 16), sizeof p[j]);
            }
            float up = M;
#pragma unroll
            for (int j = 0; j < B; j++) up = fmaxf(up, e[j].x);  // (the last one again where there are fewer)
            const float ref = up == -INFINITY ? 0.0f : up, al = __builtin_amdgcn_exp2f((M - ref) * a.scale);
            L *= al;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] *= al;
#pragma unroll
            for (int j = 0; j < B; j++) {
                if (base + wave + MW * j >= splits) break;
                const float w = __builtin_amdgcn_exp2f((e[j].x - ref) * a.scale);
                L += w * e[j].y;
#pragma unroll
                for (int d = 0; d < D; d++) o[d] += w * p[j][d];
            }
            M = up;
        }
        if constexpr (MW == 1) {
            if (HD >= kWave || lane < HD) {
#pragma unroll
                for (int d = 0; d < D; d++) a.out[(int64_t)row * a.out_stride + head * HD + dim + d] = (h16)(o[d] / L);
            }
            continue;
        }
        if (HD >= kWave || lane < HD) {
#pragma unroll
            for (int d = 0; d < D; d++) ox[wave][dim + d] = o[d];
        }
        if (lane == 0) {
            mx[wave] = M;
            lx[wave] = L;
        }
        __syncthreads();
        float up = -INFINITY;
#pragma unroll
        for (int w = 0; w < kMergeWaves; w++) up = fmaxf(up, mx[w]);
        const float ref = up == -INFINITY ? 0.0f : up;
        for (int d = threadIdx.x; d < HD; d += kMergeWaves * kWave) {
            float x = 0.0f, l = 0.0f;
#pragma unroll
            for (int w = 0; w < kMergeWaves; w++) {
                const float z = __builtin_amdgcn_exp2f((mx[w] - ref) * a.scale);
                x += z * ox[w][d];
                l += z * lx[w];
            }
            a.out[(int64_t)row * a.out_stride + head * HD + d] = (h16)(x / l);
        }
        __syncthreads();  // ox, mx and lx are rewritten
    }
}

// What begin() plans for one width: workgroups of a KV head, their waves, the most partials of a tile.
struct Kv4Plan {
    int64_t groups = 0, splits = 1;
    int waves = 4;
};

template <int HD, int V>
int32_t launch_attention(hipStream_t st, const Kv4Dev &c, const Kv4AttnArgs &a, const Kv4Plan &p, bool captured) {
    const dim3 grid((unsigned)std::max<int64_t>(p.groups * c.nkv, 1));
    if constexpr (V == 3)
        hipLaunchKernelGGL(kv4_prompt_kernel<HD>, grid, dim3(8 * kWave), 0, st, c, a);
    else if (p.waves == 8)
        hipLaunchKernelGGL((kv4_attention_kernel<HD, 1 << V, V < 2 ? 8 : 4>), grid, dim3((V < 2 ? 8 : 4) * kWave), 0, st, c, a);
    else
        hipLaunchKernelGGL((kv4_attention_kernel<HD, 1 << V, 4>), grid, dim3(4 * kWave), 0, st, c, a);
    AESIR_LAUNCH_CHECK("kv4_attention_kernel");
    const int64_t columns = (int64_t)a.rows * c.nq;
    // a wave for a row and head with few partials, four with many (47: 16.5 -> 14.4 us in all; 12 of 40 rows: 16.3, 19.1 with four);
    // a captured call may meet a batch that is split, whatever this one is
    if (captured || p.splits > 16)
        hipLaunchKernelGGL((kv4_merge_kernel<HD, V, kMergeWaves>), dim3((unsigned)std::min(columns, kMergeGrid)), dim3(kMergeWaves * kWave), 0, st, c, a);
    else if (p.splits > 1)
        hipLaunchKernelGGL((kv4_merge_kernel<HD, V, 1>), dim3((unsigned)std::min((columns + kMergeWaves - 1) / kMergeWaves, kMergeGrid)),
                           dim3(kMergeWaves * kWave), 0, st, c, a);
    AESIR_LAUNCH_CHECK("kv4_merge_kernel");
    return AESIR_OK;
}

template <int HD>
int32_t launch_attention(hipStream_t st, const Kv4Dev &c, const Kv4AttnArgs &a, int v, const Kv4Plan &p, bool captured) {
    if (v == 3) return launch_attention<HD, 3>(st, c, a, p, captured);
    if constexpr (HD < 256) {
        if (v == 1) return launch_attention<HD, 1>(st, c, a, p, captured);
        if (v == 2) return launch_attention<HD, 2>(st, c, a, p, captured);
    }
    return launch_attention<HD, 0>(st, c, a, p, captured);
}

}  // namespace aesir

// ------------------------------------------------------------------ the cache object

using namespace aesir;

struct aesir_kv4 {
    aesir_ctx *ctx = nullptr;  // null: tables only
    int64_t layers = 0, nq = 0, nkv = 0, hd = 0, max_seq_len = 0, page = 0, pages = 0;
    PageBook book;
    Kv4Dev dev{};
    int32_t *table = nullptr;
    Kv4Seq *seqs = nullptr;
    Kv4Range *ranges = nullptr;
    PageMove *moves = nullptr;
    char *ring = nullptr;  // pinned staging, handed out front to back
    int64_t ring_at = 0;
    bool batch = false;
    int64_t batch_rows = 0;
    bool in_class[kKv4Widths] = {};             // whether the batch has sequences of a column class
    Kv4Plan plans[kKv4Plans];

    aesir_kv4(int64_t num_pages, int64_t page_size, int64_t max_seqs) : book(num_pages, page_size, max_seqs) {}
};

namespace {

constexpr int64_t kRingBytes = 1 << 20;
constexpr int64_t kMaxPages = (int64_t)1 << 27;
constexpr int64_t kPartCols = 65536;  // columns of split partials: 256 of every CU
// How attention's work is cut, with us per call of 32 query heads of 128 over 8 KV heads, one row a sequence, unless
// said otherwise:
// - a workgroup to a tile where that fills the CUs and no tile is long (merges saved: 64 sequences of about 1000
//   positions 25.5 -> 21.5, of 2000 at 4 KV heads of 64 20.5 -> 17.1; 32 of 2000 25.3 / 25.9), or where all are short (4 of
//   500, 4 KV heads of 64: 6.7, in two pieces 8.3);
// - little work that one workgroup a CU can take in pieces of their own: kFewLeast rounds or more each (8 / 12 / 16 / 32
//   rounds: one sequence of 1024 positions 8.8 / 9.5 / 10.2 / 10.5, of 4096 10.4 / 10.6 / 10.9 / 13.2), of eight
//   waves where pieces are over 16 rounds (one of 65536 positions 25.4 with four, 22.9; of 100 4.7 with four, 5.0);
// - else as many workgroups of four waves as run at once at head_dim 128 (three, two and one to a CU by the registers of 16,
//   32 and 64 columns; narrower heads leave places for more, and of head_dim 256's 512 half run at once), kLeast rounds
//   each or more (32 / 48 / 64: 24 sequences of 3000 26.0 / 25.6 / 31.0, 40 of 4000 43.1 / 43.4 / 47.3), half of that with
//   little work (12 / 24 / 48: 8 of 2048 12.7 / 12.3 / 17.6); equal shares of all tiles where starts of their own don't
//   fit (64 of 4096: 66.5 against 75.8).
constexpr int64_t kWholeRounds = 96, kShortRounds = 24;
constexpr int64_t kFewRounds = 256 * 64, kFewLeast = 8;
constexpr int64_t kGroups[3] = {768, 512, 256}, kLeast = 48;
// Rounds of a prompt's split at least (8 / 16 / 32: 128 rows over 2048 positions 28.1 / 34.2 / 51.7), and what a workgroup's
// start and the merge cost, in rounds (of 1.2 us).
constexpr int64_t kPromptRounds = 8, kPromptStart = 3, kPromptMerge = 5;
// Rounds of all tiles up to which 16-column tiles, which work side by side, beat the tile that holds all columns of a
// sequence and reads its keys once (one sequence of 2048 positions, 16 rows: 10.0 against 15.7 with 64 columns, 4.0 K
// rounds of 8000 positions 16.5 / 15.0 with 32), and up to which 32-column tiles beat the prompts' (128 rows of 2048
// positions 20.0 / 28.1, 48 of 8 sequences of 2048, 24.5 K rounds, 51 / 99; 1000 of 1000, 32 K, 58 / 48). At head_dim 256
// there are 16-column tiles (for up to 32 columns: 64 sequences of 8 rows 94 / 126) and the prompts' only: 32 columns
// would leave the registers one wave to a SIMD and spill (4 KV heads, 128 rows of 2048 positions, 8.2 K rounds, 23 / 30; 300
// of 1000, 9.6 K, 39 / 31; 16 rows of 8 sequences of 2048, 8.2 K, 41 / 32).
constexpr int64_t kNarrowRounds = 2560, kNarrowRounds256 = 6144, kPromptLeast = 28672;

struct Kv4Sizes {
    int64_t page_bytes, pool, table, seqs, ranges, moves, part, part_ml;
    int64_t total() const {
        int64_t t = 0;
        for (int64_t b : {pool, table, seqs, ranges, moves, part, part_ml}) t += (b + 255) / 256 * 256;
        return t + 256;  // the well's own alignment
    }
};

int32_t kv4_sizes(int64_t layers, int64_t nq, int64_t nkv, int64_t hd, int64_t max_seq_len, int64_t max_seqs, int64_t page,
                  int64_t pages, Kv4Sizes *z) {
    if (layers <= 0 || nq <= 0 || nkv <= 0 || hd <= 0 || max_seq_len <= 0 || max_seqs <= 0 || page <= 0 || pages <= 0)
        return fail(AESIR_ERR_INVALID, "KV4Cache: dimensions must be positive");
    if (nq % nkv != 0) return fail(AESIR_ERR_SHAPE, "KV4Cache: query heads must be a multiple of the KV heads");
    if (hd != 32 && hd != 64 && hd != 128 && hd != 256)
        return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: head_dim %lld is not 32, 64, 128 or 256", (long long)hd);
    if (page < 32 || page > 1024 || (page & (page - 1)) != 0)
        return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: page size %lld is not a power of two from 32 to 1024", (long long)page);
    if (max_seqs > kMaxSeqs) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: more than %d sequences", kMaxSeqs);
    if (max_seq_len > INT32_MAX / 2 || pages > kMaxPages || nq > 65535 || layers > 65535)
        return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    // a workgroup or more of 512 threads to a sequence and KV head; a launch holds under 2^32 threads
    if (max_seqs * nkv > 1 << 22) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    const int64_t stride = (max_seq_len + page - 1) / page;
    if (mul_checked(stride, max_seqs) > INT32_MAX) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    z->page_bytes = mul_checked(mul_checked(layers, nkv, page), hd / 4 * 5);
    z->pool = mul_checked(z->page_bytes, pages);
    if (z->pool < 0 || z->pool > (int64_t)1 << 50) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    z->table = stride * max_seqs * 4;
    z->seqs = (max_seqs + kWave) * (int64_t)sizeof(Kv4Seq);
    z->ranges = (max_seqs + kWave) * (int64_t)sizeof(Kv4Range);
    z->moves = pages * (int64_t)sizeof(PageMove);
    z->part = kPartCols * hd * 4;
    z->part_ml = kPartCols * 8;
    return AESIR_OK;
}

int32_t need_device(aesir_kv4 *kv, const char *what) {
    if (!kv) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: null cache", what);
    if (!kv->ctx) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: the cache has no context (page tables only)", what);
    return bind(kv->ctx);
}

// Calls that change the tables send host data to the device, which a replay would not send again.
int32_t not_captured(aesir_ctx *ctx, const char *what) {
    AESIR_TRY(bind(ctx));
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    AESIR_HIP_TRY(hipStreamIsCapturing(ctx->stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return fail(AESIR_ERR_INVALID, "KV4Cache.%s: not while the context's stream is being captured", what);
    return AESIR_OK;
}

int32_t can_change(aesir_kv4 *kv, const char *what) {
    clear_error();
    if (!kv) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: null cache", what);
    return kv->ctx ? not_captured(kv->ctx, what) : AESIR_OK;
}

int32_t seq_ok(aesir_kv4 *kv, const char *what, int64_t s) {
    if (s < 0 || s >= kv->book.max_seqs())
        return fail(AESIR_ERR_INVALID, "KV4Cache.%s: sequence %lld is not in [0, %lld)", what, (long long)s,
                    (long long)kv->book.max_seqs());
    return AESIR_OK;
}

// `bytes` of pinned memory that no earlier launch still reads.
int32_t stage(aesir_kv4 *kv, int64_t bytes, char **out) {
    bytes = (bytes + 15) / 16 * 16;
    if (kv->ring_at + bytes > kRingBytes) {  // once a MB: wait for the launches that read it
        AESIR_HIP_TRY(hipStreamSynchronize(kv->ctx->stream));
        kv->ring_at = 0;
    }
    *out = kv->ring + kv->ring_at;
    kv->ring_at += bytes;
    return AESIR_OK;
}

struct Run {
    void *dst;
    const void *src;
    int64_t bytes, fill;  // bytes of src, then fill bytes of kNone
};

int32_t launch_upload(aesir_kv4 *kv, const Run &run, const uint32_t *updates, int64_t n_updates) {
    if (run.bytes + run.fill + n_updates == 0) return AESIR_OK;
    char *p = nullptr;
    AESIR_TRY(stage(kv, run.bytes + n_updates * 8, &p));
    if (run.bytes) std::memcpy(p, run.src, (size_t)run.bytes);
    if (n_updates) std::memcpy(p + run.bytes, updates, (size_t)n_updates * 8);
    const Kv4Upload u{(const uint32_t *)p, (uint32_t *)run.dst, (int32_t)(run.bytes / 4), (int32_t)(run.fill / 4), kv->table,
                      (int32_t)n_updates};
    const int64_t threads = u.words + u.fill + n_updates;
    const unsigned blocks = (unsigned)std::min<int64_t>(256, (threads + kThreads - 1) / kThreads);
    hipLaunchKernelGGL(kv4_upload_kernel, dim3(blocks), dim3(kThreads), 0, kv->ctx->stream, u);
    AESIR_LAUNCH_CHECK("kv4_upload_kernel");
    return AESIR_OK;
}

// Table entries that go to the device with one launch at most.
constexpr int64_t kUpdates = kRingBytes / 4 / 8;

// Entries of the listed sequences that the device lacks.
int64_t unsynced(const aesir_kv4 *kv, const int64_t *seqs, int64_t n) {
    int64_t count = 0;
    for (int64_t i = 0; i < n; i++) count += (int64_t)kv->book.seq(seqs[i]).pages.size() - kv->book.seq(seqs[i]).synced;
    return count;
}

int32_t send(aesir_kv4 *kv, const int64_t *seqs, int64_t n, const Run &run, std::vector<uint32_t> &e) {
    for (int64_t i = 0; i < n; i++) {
        const PageBook::Seq &s = kv->book.seq(seqs[i]);
        for (int64_t j = s.synced; j < (int64_t)s.pages.size(); j++) {
            e.push_back((uint32_t)(seqs[i] * kv->dev.table_stride + j));
            e.push_back((uint32_t)s.pages[(size_t)j]);
            if ((int64_t)e.size() == 2 * kUpdates) {
                AESIR_TRY(launch_upload(kv, Run{}, e.data(), kUpdates));
                e.clear();
            }
        }
        kv->book.mark_synced(seqs[i]);  // (a sequence may be listed again)
    }
    return launch_upload(kv, run, e.data(), (int64_t)e.size() / 2);
}

// Brings the device's table rows of the listed sequences up to date, with `run` in the last launch; after a failure all of
// them are sent again. e: empty, with room for the entries (or for kUpdates).
int32_t upload(aesir_kv4 *kv, const int64_t *seqs, int64_t n, const Run &run, std::vector<uint32_t> &e) {
    const int32_t rc = send(kv, seqs, n, run, e);
    if (rc != AESIR_OK)
        for (int64_t i = 0; i < n; i++) kv->book.mark_unsynced(seqs[i]);
    return rc;
}

// n records and, behind them, at least one and up to a multiple of 64 of kNone.
template <class T>
Run records(T *dst, const T *src, int64_t n) {
    return {dst, src, n * (int64_t)sizeof(T), (kWave - n % kWave) * (int64_t)sizeof(T)};
}

// Uploads the moves and copies the pages.
int32_t copy_pages(aesir_kv4 *kv, const std::vector<PageMove> &moves) {
    if (!kv->ctx) return AESIR_OK;
    const int64_t most = kRingBytes / 4 / (int64_t)sizeof(PageMove);
    for (int64_t at = 0; at < (int64_t)moves.size(); at += most) {
        const int64_t n = std::min<int64_t>(most, (int64_t)moves.size() - at);
        const Run r{kv->moves + at, moves.data() + at, n * (int64_t)sizeof(PageMove), 0};
        AESIR_TRY(launch_upload(kv, r, nullptr, 0));
    }
    if (moves.empty()) return AESIR_OK;
    const int64_t units = (kv->dev.page_bytes + kCopyChunk - 1) / kCopyChunk * (int64_t)moves.size();
    hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)std::min<int64_t>(units, 1 << 20)), dim3(kThreads), 0, kv->ctx->stream,
                       kv->dev.pool, kv->dev.page_bytes, kv->moves, (int)moves.size());
    AESIR_LAUNCH_CHECK("kv4_copy_kernel");
    return AESIR_OK;
}

// The batch ends: captured calls that are replayed before the next begin find no rows.
int32_t end_batch(aesir_kv4 *kv) {
    if (!kv->batch) return AESIR_OK;
    kv->batch = false;
    kv->batch_rows = 0;
    if (!kv->ctx) return AESIR_OK;
    return launch_upload(kv, records<Kv4Seq>(kv->seqs, nullptr, 0), nullptr, 0);
}

template <class F>
int32_t guarded(const char *what, F f) {
    try {
        return f();
    } catch (const std::exception &) {
        return fail(AESIR_ERR_EXHAUSTED, "KV4Cache.%s: out of host memory", what);
    }
}

// f16 rows start on f16 boundaries.
int32_t pointers_ok(const char *what, const void *a, const void *b) {
    if (!a || !b) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: null tensor pointer", what);
    if (((uintptr_t)a | (uintptr_t)b) & 1) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: tensor pointer not 2-byte aligned", what);
    return AESIR_OK;
}

bool aligned16(const void *p, int64_t cols) { return ((uintptr_t)p & 15) == 0 && cols % 8 == 0; }

// Grid of the append and read kernels: a thread per 8 dims of a row and head.
dim3 rows_grid(const aesir_kv4 *kv, int64_t rows, int64_t layers) {
    return dim3((unsigned)((rows * (kv->hd / 8) + kThreads - 1) / kThreads), (unsigned)kv->nkv,
                (unsigned)std::min<int64_t>(layers, 65535));
}

#define AESIR_KV4_ROWS(kernel, vec, grid, st, dev, args)                                                          \
    switch (kv->hd * 2 + (vec)) {                                                                                 \
        case 64: hipLaunchKernelGGL((kernel<32, false>), grid, dim3(kThreads), 0, st, dev, args); break;          \
        case 65: hipLaunchKernelGGL((kernel<32, true>), grid, dim3(kThreads), 0, st, dev, args); break;           \
        case 128: hipLaunchKernelGGL((kernel<64, false>), grid, dim3(kThreads), 0, st, dev, args); break;         \
        case 129: hipLaunchKernelGGL((kernel<64, true>), grid, dim3(kThreads), 0, st, dev, args); break;          \
        case 256: hipLaunchKernelGGL((kernel<128, false>), grid, dim3(kThreads), 0, st, dev, args); break;        \
        case 257: hipLaunchKernelGGL((kernel<128, true>), grid, dim3(kThreads), 0, st, dev, args); break;         \
        case 512: hipLaunchKernelGGL((kernel<256, false>), grid, dim3(kThreads), 0, st, dev, args); break;        \
        default: hipLaunchKernelGGL((kernel<256, true>), grid, dim3(kThreads), 0, st, dev, args); break;          \
    }

// The width every sequence of the batch takes: the narrowest that holds its columns, or a narrower one with little work.
std::vector<int> column_classes(const aesir_kv4 *kv, const std::vector<Kv4Seq> &ds) {
    const int64_t G = kv->nq / kv->nkv;
    auto work = [&](int64_t W) {
        int64_t w = 0;
        for (const Kv4Seq &s : ds) w += (s.rows * G + W - 1) / W * (((int64_t)s.length + kKeys - 1) / kKeys) * kv->nkv;
        return w;
    };
    const bool large = kv->hd == 256;
    const bool narrow = work(16) <= (large ? kNarrowRounds256 : kNarrowRounds), prompts = work(32) > kPromptLeast;
    std::vector<int> c;
    for (const Kv4Seq &s : ds) {
        const int64_t cols = s.rows * G;
        if (large)
            c.push_back(narrow || cols <= 32 ? 0 : 3);
        else
            c.push_back(narrow || cols <= 16 ? 0 : cols <= 32 ? 1 : cols <= 64 ? 2 : prompts ? 3 : 1);
    }
    return c;
}

// Plan p of the batch: width p for the sequences of that class, or width p - kKv4Widths for all sequences. Workgroups
// of widths 0 - 2 get `chunk` rounds each. With `own`, sequences start workgroups of their own (firsts rounded up to a
// chunk); else they lie one behind the other, so that all workgroups have equal work and none waits for a place. Partials
// fit: only tiles that are cut have them, two at most a workgroup, and there are no more workgroups than kGroups then.
void make_plan(const aesir_kv4 *kv, int p, std::vector<Kv4Seq> &ds, const std::vector<int> &classes, Kv4Plan *out) {
    const int v = p % kKv4Widths;
    const bool all = p >= kKv4Widths;
    const int64_t W = kv4_width(v, (int)kv->hd), G = kv->nq / kv->nkv;
    auto tiles = [&](const Kv4Seq &s) -> int64_t {
        return all || classes[(size_t)(&s - ds.data())] == v ? (s.rows * G + W - 1) / W : 0;
    };
    *out = Kv4Plan{};
    if (!all && !std::count(classes.begin(), classes.end(), v)) {
        for (Kv4Seq &s : ds) s.plan[p] = {0, 0, 1, 0};
        return;
    }
    int shift = 0;
    auto rounds = [&](const Kv4Seq &s) { return (((int64_t)s.length + kKeys - 1) / kKeys + (1 << shift) - 1) >> shift; };
    auto all_work = [&] {
        int64_t w = 0;
        for (const Kv4Seq &s : ds) w += tiles(s) * rounds(s);
        return w;
    };
    int64_t work = all_work(), most = 1;
    if (v == 3) {  // equal splits of every tile: as many as make the workgroups that run one after the other on a CU shortest
        int64_t longest = 1, chunk = 0, best = INT64_MAX;
        for (const Kv4Seq &s : ds)
            if (tiles(s)) longest = std::max(longest, rounds(s));
        auto splits = [&](const Kv4Seq &s, int64_t c) { return tiles(s) ? (rounds(s) + c - 1) / c : 0; };
        for (int64_t n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
            if (n > 1 && longest / n < kPromptRounds) break;
            const int64_t c = (longest + n - 1) / n;
            int64_t units = 0, parts = 0;
            for (const Kv4Seq &s : ds) {
                units += tiles(s) * splits(s, c);
                if (splits(s, c) > 1) parts += tiles(s) * splits(s, c);
            }
            const int64_t cost = (units * kv->nkv + 255) / 256 * (c + kPromptStart) + (parts ? kPromptMerge : 0);
            if (parts * kv->nkv * W <= kPartCols && cost < best) {  // (n of 1 has none)
                best = cost;
                chunk = c;
            }
        }
        int64_t units = 0, parts = 0;
        for (Kv4Seq &s : ds) {
            const int64_t n = splits(s, chunk);
            s.plan[p] = {(int32_t)units, (int32_t)n, (int32_t)parts, 0};
            units += tiles(s) * n;
            if (n > 1) parts += tiles(s) * n;
            most = std::max(most, n);
        }
        out->groups = units;
        out->splits = most;
        return;
    }
    for (; work > INT32_MAX / 4; work = all_work()) shift++;  // ends: rows, and so tiles, are fewer
    int64_t longest = 0, count = 0;
    bool single = true;  // no sequence of several tiles
    for (const Kv4Seq &s : ds) {
        if (tiles(s)) longest = std::max(longest, rounds(s));
        count += tiles(s);
        single &= tiles(s) <= 1;
    }
    int64_t slots = 1, chunk = 1, groups = 0;
    auto cut = [&](int64_t at_once, int64_t least) {
        slots = std::max<int64_t>(1, at_once / kv->nkv);  // of a KV head
        chunk = std::max<int64_t>(std::max<int64_t>(least >> shift, 1), (work + slots - 1) / slots);
        groups = 0;
        for (const Kv4Seq &s : ds) groups += (tiles(s) * rounds(s) + chunk - 1) / chunk;
        return groups <= slots;
    };
    bool eight = false, own = true;
    const bool few = work * kv->nkv <= kFewRounds;
    if (single && shift == 0 && longest <= (count * kv->nkv >= 256 ? kWholeRounds : kShortRounds)) {
        chunk = std::max<int64_t>(longest, 1);
        eight = v < 2 && count * kv->nkv <= 256 && longest > 16;
    } else if (few && cut(256, kFewLeast)) {
        eight = v < 2 && std::min(longest, chunk) > 16;
    } else {
        own = cut(kv->hd == 256 ? kGroups[1] : kGroups[v], few ? kLeast / 2 : kLeast);
    }
    int64_t at = 0;
    for (Kv4Seq &s : ds) {
        const int64_t n = tiles(s) * rounds(s);
        if (own) at = (at + chunk - 1) / chunk * chunk;
        s.plan[p] = {(int32_t)at, (int32_t)n, (int32_t)chunk, shift + (own ? 256 : 0)};
        if (n) most = std::max(most, std::min((rounds(s) - 1) / chunk + 2, (at + n - 1) / chunk - at / chunk + 1));
        at += n;
    }
    out->groups = (at + chunk - 1) / chunk;
    out->splits = most;
    out->waves = eight ? 8 : 4;
}

int32_t kv4_begin(aesir_kv4 *kv, const int64_t *seqs, const int64_t *rows, int64_t n) {
    if (n < 0 || n > kv->book.max_seqs()) return fail(AESIR_ERR_INVALID, "KV4Cache.begin: bad sequence count");
    if (n > 0 && (!seqs || !rows)) return fail(AESIR_ERR_INVALID, "KV4Cache.begin: null argument");
    std::vector<char> seen((size_t)kv->book.max_seqs(), 0);
    int64_t total = 0;
    for (int64_t i = 0; i < n; i++) {
        AESIR_TRY(seq_ok(kv, "begin", seqs[i]));
        if (seen[(size_t)seqs[i]]++)
            return fail(AESIR_ERR_INVALID, "KV4Cache.begin: sequence %lld is listed twice", (long long)seqs[i]);
        if (rows[i] < 0) return fail(AESIR_ERR_INVALID, "KV4Cache.begin: row counts must not be negative");
        if (rows[i] > kv->max_seq_len - kv->book.seq(seqs[i]).length)
            return fail(AESIR_ERR_INVALID, "KV4Cache.begin: sequence %lld would pass %lld positions", (long long)seqs[i],
                        (long long)kv->max_seq_len);
        total += rows[i];
    }
    if (total > INT32_MAX / (kv->nq * kv->hd / 8)) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache.begin: too many rows");
    const int64_t need = kv->book.pages_needed(seqs, rows, n);
    if (need > kv->book.free_pages())
        return fail(AESIR_ERR_EXHAUSTED, "KV4Cache.begin: %lld pages needed, %lld free", (long long)need,
                    (long long)kv->book.free_pages());
    // All memory first: nothing fails between the tables' change and the launches.
    std::vector<PageMove> copies;
    std::vector<Kv4Seq> ds((size_t)n);
    std::vector<uint32_t> entries;
    copies.reserve((size_t)n);
    int64_t most = 0;
    for (int64_t i = 0; i < n; i++) {
        const PageBook::Seq &s = kv->book.seq(seqs[i]);
        kv->book.reserve(seqs[i], s.length + rows[i]);
        most += kv->book.pages_for(s.length + rows[i]) - s.synced + 1;  // one more: a last page that is copied
    }
    entries.reserve((size_t)(2 * std::min(most, kUpdates)));
    int64_t at = 0;
    for (int64_t i = 0; i < n; i++) {
        Kv4Seq &s = ds[(size_t)i];
        s = Kv4Seq{};
        s.slot = (int32_t)seqs[i];
        s.length = (int32_t)(kv->book.seq(seqs[i]).length + rows[i]);
        s.rows = (int32_t)rows[i];
        s.row0 = (int32_t)at;
        at += rows[i];
    }
    Kv4Plan plans[kKv4Plans];
    const std::vector<int> classes = column_classes(kv, ds);
    for (int p = 0; p < kKv4Plans; p++) make_plan(kv, p, ds, classes, &plans[p]);
    kv->batch = false;
    for (int64_t i = 0; i < n; i++) kv->book.grow(seqs[i], rows[i], copies);
    if (kv->ctx) {
        int32_t rc = copy_pages(kv, copies);
        if (rc == AESIR_OK) rc = upload(kv, seqs, n, records(kv->seqs, ds.data(), n), entries);
        if (rc != AESIR_OK) {
            for (int64_t i = n - 1; i >= 0; i--) kv->book.shrink(seqs[i], rows[i], copies);
            return rc;
        }
    }
    std::copy(plans, plans + kKv4Plans, kv->plans);
    kv->batch = true;
    kv->batch_rows = total;
    for (bool &b : kv->in_class) b = false;
    for (int64_t i = 0; i < n; i++)
        if (rows[i] > 0) kv->in_class[classes[(size_t)i]] = true;
    return AESIR_OK;
}

int32_t layer_ok(aesir_kv4 *kv, const char *what, int64_t layer) {
    if (layer < 0 || layer >= kv->layers) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: layer out of bounds", what);
    return AESIR_OK;
}

// The plans that attention of the batch launches, n of them: one for the sequences of each class there is. A captured call
// may meet any batch later: one launch for all sequences, as wide as its own batch's widest.
int launched(const aesir_kv4 *kv, bool captured, int (&plans)[kKv4Widths]) {
    int n = 0;
    for (int v = 0; v < kKv4Widths; v++) {
        if (!kv->batch || !kv->in_class[v]) continue;
        if (captured) n = 0;
        plans[n++] = captured ? v + kKv4Widths : v;
    }
    return n;
}

}  // namespace

extern "C" {

int64_t aesir_kv4_well_bytes(int64_t num_layers, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim, int64_t max_seq_len,
                             int64_t max_seqs, int64_t page_size, int64_t num_pages) {
    clear_error();
    Kv4Sizes z;
    const int32_t rc = kv4_sizes(num_layers, n_heads, n_kv_heads, head_dim, max_seq_len, max_seqs, page_size, num_pages, &z);
    return rc == AESIR_OK ? z.total() : rc;
}

int32_t aesir_kv4_create(aesir_ctx *ctx, int64_t num_layers, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                         int64_t max_seq_len, int64_t max_seqs, int64_t page_size, int64_t num_pages, aesir_kv4 **out) {
    clear_error();
    if (!out) return fail(AESIR_ERR_INVALID, "KV4Cache: null output handle");
    *out = nullptr;
    Kv4Sizes z;
    AESIR_TRY(kv4_sizes(num_layers, n_heads, n_kv_heads, head_dim, max_seq_len, max_seqs, page_size, num_pages, &z));
    if (ctx) AESIR_TRY(not_captured(ctx, "create"));
    return guarded("create", [&]() -> int32_t {
        auto *kv = new aesir_kv4(num_pages, page_size, max_seqs);
        kv->layers = num_layers;
        kv->nq = n_heads;
        kv->nkv = n_kv_heads;
        kv->hd = head_dim;
        kv->max_seq_len = max_seq_len;
        kv->page = page_size;
        kv->pages = num_pages;
        if (!ctx) {
            *out = kv;
            return AESIR_OK;
        }
        const int64_t mark = ctx->well_offset;
        void *p[7] = {};
        const int64_t bytes[7] = {z.pool, z.table, z.seqs, z.ranges, z.moves, z.part, z.part_ml};
        int32_t rc = AESIR_OK;
        for (int i = 0; i < 7 && rc == AESIR_OK; i++) rc = well_alloc_bytes(ctx, bytes[i], &p[i]);
        if (rc == AESIR_OK && hipHostMalloc((void **)&kv->ring, kRingBytes, hipHostMallocDefault) != hipSuccess)
            rc = fail(AESIR_ERR_HIP, "hipHostMalloc of the cache's staging memory failed");
        if (rc != AESIR_OK) {
            ctx->well_offset = mark;
            delete kv;
            return rc;
        }
        kv->ctx = ctx;
        kv->table = (int32_t *)p[1];
        kv->seqs = (Kv4Seq *)p[2];
        kv->ranges = (Kv4Range *)p[3];
        kv->moves = (PageMove *)p[4];
        Kv4Dev &d = kv->dev;
        d.pool = (char *)p[0];
        d.page_bytes = z.page_bytes;
        d.layer_bytes = z.page_bytes / num_layers;
        d.page_shift = __builtin_ctzll((unsigned long long)page_size);
        d.hd = (int32_t)head_dim;
        d.nkv = (int32_t)n_kv_heads;
        d.nq = (int32_t)n_heads;
        d.table = kv->table;
        d.table_stride = (max_seq_len + page_size - 1) / page_size;
        d.seqs = kv->seqs;
        d.part = (float *)p[5];
        d.part_ml = (float *)p[6];
        kv->batch = true;  // clears the descriptor: the well's memory may have been used before
        rc = end_batch(kv);
        if (rc != AESIR_OK) {
            (void)hipHostFree(kv->ring);
            ctx->well_offset = mark;
            delete kv;
            return rc;
        }
        ctx->live_caches++;
        *out = kv;
        return AESIR_OK;
    });
}

int32_t aesir_kv4_destroy(aesir_kv4 *kv) {
    if (!kv) return AESIR_OK;
    if (kv->ctx) {
        AESIR_TRY(not_captured(kv->ctx, "destroy"));
        (void)hipStreamSynchronize(kv->ctx->stream);  // launches may still read the staging memory
        (void)hipHostFree(kv->ring);
        kv->ctx->live_caches--;
    }
    delete kv;
    return AESIR_OK;
}

int64_t aesir_kv4_page_bytes(const aesir_kv4 *kv) { return kv ? kv->layers * kv->nkv * kv->page * (kv->hd / 4 * 5) : -1; }
int64_t aesir_kv4_free_pages(const aesir_kv4 *kv) { return kv ? kv->book.free_pages() : -1; }
int64_t aesir_kv4_length(const aesir_kv4 *kv, int64_t seq) {
    return kv && seq >= 0 && seq < kv->book.max_seqs() ? kv->book.seq(seq).length : -1;
}

int32_t aesir_kv4_pages(const aesir_kv4 *kv, int64_t seq, int64_t *pages, int64_t cap, int64_t *n) {
    clear_error();
    if (!kv || !n || cap < 0 || (cap > 0 && !pages)) return fail(AESIR_ERR_INVALID, "KV4Cache.pages: null argument");
    if (seq < 0 || seq >= kv->book.max_seqs()) return fail(AESIR_ERR_INVALID, "KV4Cache.pages: sequence out of bounds");
    const auto &v = kv->book.seq(seq).pages;
    *n = (int64_t)v.size();
    for (int64_t i = 0; i < *n && i < cap; i++) pages[i] = v[(size_t)i];
    return AESIR_OK;
}

int32_t aesir_kv4_begin(aesir_kv4 *kv, const int64_t *seqs, const int64_t *rows, int64_t n) {
    AESIR_TRY(can_change(kv, "begin"));
    return guarded("begin", [&] { return kv4_begin(kv, seqs, rows, n); });
}

int32_t aesir_kv4_plan(const aesir_kv4 *kv, int32_t captured, int64_t *widths, int64_t *pieces, int64_t cap, int64_t *n) {
    clear_error();
    if (!kv || !n || cap < 0 || (cap > 0 && (!widths || !pieces))) return fail(AESIR_ERR_INVALID, "KV4Cache.plan: null argument");
    int plans[kKv4Widths];
    *n = launched(kv, captured != 0, plans);
    for (int64_t i = 0; i < *n && i < cap; i++) {
        widths[i] = kv4_width(plans[i] % kKv4Widths, (int)kv->hd);
        pieces[i] = kv->plans[plans[i]].splits;
    }
    return AESIR_OK;
}

int32_t aesir_kv4_append(aesir_kv4 *kv, int64_t layer, const void *key, int64_t key_rows, int64_t key_cols, const void *val,
                         int64_t val_rows, int64_t val_cols) {
    AESIR_TRY(need_device(kv, "append"));
    AESIR_TRY(layer_ok(kv, "append", layer));
    if (!kv->batch) return fail(AESIR_ERR_INVALID, "KV4Cache.append: no batch (begin comes first)");
    if (key_rows != kv->batch_rows || val_rows != kv->batch_rows)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.append: the batch has %lld new rows", (long long)kv->batch_rows);
    if (kv->batch_rows == 0) return AESIR_OK;
    if (key_cols < kv->nkv * kv->hd || val_cols < kv->nkv * kv->hd)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.append: key/val rows narrower than kv_heads * head_dim");
    AESIR_TRY(pointers_ok("append", key, val));
    const Kv4AppendArgs a{(const h16 *)key, (const h16 *)val, key_cols, val_cols, layer, (int32_t)key_rows};
    const bool vec = aligned16(key, key_cols) && aligned16(val, val_cols);
    AESIR_KV4_ROWS(kv4_append_kernel, vec, rows_grid(kv, key_rows, 1), kv->ctx->stream, kv->dev, a)
    AESIR_LAUNCH_CHECK("kv4_append_kernel");
    return AESIR_OK;
}

int32_t aesir_kv4_attention(aesir_kv4 *kv, int64_t layer, const void *query, int64_t query_rows, int64_t query_cols, void *output,
                            int64_t output_rows, int64_t output_cols) {
    AESIR_TRY(need_device(kv, "attention"));
    AESIR_TRY(layer_ok(kv, "attention", layer));
    if (!kv->batch) return fail(AESIR_ERR_INVALID, "KV4Cache.attention: no batch (begin comes first)");
    if (query_rows != kv->batch_rows || output_rows != kv->batch_rows)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.attention: the batch has %lld new rows", (long long)kv->batch_rows);
    if (kv->batch_rows == 0) return AESIR_OK;
    if (query_cols < kv->nq * kv->hd || output_cols < kv->nq * kv->hd)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.attention: query/output rows narrower than heads * head_dim");
    AESIR_TRY(pointers_ok("attention", query, output));
    Kv4AttnArgs a{(const h16 *)query, (h16 *)output, query_cols, output_cols, layer, (int32_t)query_rows,
                  aligned16(query, query_cols) && aligned16(output, output_cols), 0,
                  (float)(1.4426950408889634 / std::sqrt((double)kv->hd))};
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    AESIR_HIP_TRY(hipStreamIsCapturing(kv->ctx->stream, &st));
    const bool captured = st != hipStreamCaptureStatusNone;
    int plans[kKv4Widths];
    const int n = launched(kv, captured, plans);
    for (int i = 0; i < n; i++) {
        a.plan = plans[i];
        const int v = a.plan % kKv4Widths;
        const Kv4Plan &p = kv->plans[a.plan];
        int32_t rc;
        switch (kv->hd) {
            case 32: rc = launch_attention<32>(kv->ctx->stream, kv->dev, a, v, p, captured); break;
            case 64: rc = launch_attention<64>(kv->ctx->stream, kv->dev, a, v, p, captured); break;
            case 128: rc = launch_attention<128>(kv->ctx->stream, kv->dev, a, v, p, captured); break;
            default: rc = launch_attention<256>(kv->ctx->stream, kv->dev, a, v, p, captured); break;
        }
        AESIR_TRY(rc);
    }
    return AESIR_OK;
}

int32_t aesir_kv4_read(aesir_kv4 *kv, int64_t layer, int64_t layers, const int64_t *seqs, const int64_t *pos, const int64_t *rows,
                       int64_t n, void *key, int64_t key_rows, int64_t key_cols, void *val, int64_t val_rows, int64_t val_cols) {
    if (kv && !kv->ctx) return need_device(kv, "read");
    AESIR_TRY(can_change(kv, "read"));
    if (layer < 0 || layers < 0 || layer > kv->layers - layers) return fail(AESIR_ERR_INVALID, "KV4Cache.read: layer out of bounds");
    if (n < 0 || (n > 0 && (!seqs || !pos || !rows))) return fail(AESIR_ERR_INVALID, "KV4Cache.read: null argument");
    int64_t total = 0;
    for (int64_t i = 0; i < n; i++) {
        AESIR_TRY(seq_ok(kv, "read", seqs[i]));
        const int64_t len = kv->book.seq(seqs[i]).length;
        if (pos[i] < 0 || rows[i] < 0 || pos[i] > len || rows[i] > len - pos[i])
            return fail(AESIR_ERR_INVALID, "KV4Cache.read: range [%lld, +%lld) outside sequence %lld of %lld positions",
                        (long long)pos[i], (long long)rows[i], (long long)seqs[i], (long long)len);
        total += rows[i];
        if (total > INT32_MAX / (kv->nkv * kv->hd / 8)) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache.read: too many rows");
    }
    if (key_rows != total * layers || val_rows != total * layers)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.read: %lld rows are asked for", (long long)(total * layers));
    if (total * layers == 0) return AESIR_OK;
    if (key_cols < kv->nkv * kv->hd || val_cols < kv->nkv * kv->hd)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.read: key/val rows narrower than kv_heads * head_dim");
    AESIR_TRY(pointers_ok("read", key, val));
    return guarded("read", [&]() -> int32_t {
        const bool vec = aligned16(key, key_cols) && aligned16(val, val_cols);
        std::vector<Kv4Range> r;
        int64_t first = 0;
        for (int64_t at = 0; at < n; at += kv->book.max_seqs()) {  // a launch per max_seqs ranges
            const int64_t m = std::min<int64_t>(kv->book.max_seqs(), n - at);
            r.clear();
            int64_t count = 0;
            for (int64_t i = at; i < at + m; i++) {
                r.push_back({(int32_t)seqs[i], (int32_t)pos[i], (int32_t)rows[i], (int32_t)count});
                count += rows[i];
            }
            if (count == 0) continue;
            std::vector<uint32_t> entries;
            entries.reserve((size_t)(2 * std::min(unsynced(kv, seqs + at, m), kUpdates)));
            AESIR_TRY(upload(kv, seqs + at, m, m == 1 ? Run{} : records(kv->ranges, r.data(), m), entries));
            const Kv4ReadArgs a{(h16 *)key, (h16 *)val, key_cols,     val_cols,       layer,         layers,
                                m == 1 ? nullptr : kv->ranges, (int32_t)total, (int32_t)first, r[0]};
            AESIR_KV4_ROWS(kv4_read_kernel, vec, rows_grid(kv, count, layers), kv->ctx->stream, kv->dev, a)
            AESIR_LAUNCH_CHECK("kv4_read_kernel");
            first += count;
        }
        return AESIR_OK;
    });
}

int32_t aesir_kv4_fork(aesir_kv4 *kv, int64_t src, int64_t dst) {
    AESIR_TRY(can_change(kv, "fork"));
    AESIR_TRY(seq_ok(kv, "fork", src));
    AESIR_TRY(seq_ok(kv, "fork", dst));
    if (kv->book.seq(dst).length > 0) return fail(AESIR_ERR_INVALID, "KV4Cache.fork: sequence %lld is not empty", (long long)dst);
    return guarded("fork", [&]() -> int32_t {
        AESIR_TRY(end_batch(kv));
        if (src != dst) kv->book.fork(src, dst);
        return AESIR_OK;
    });
}

int32_t aesir_kv4_copy(aesir_kv4 *kv, int64_t src, int64_t dst) {
    AESIR_TRY(can_change(kv, "copy"));
    AESIR_TRY(seq_ok(kv, "copy", src));
    AESIR_TRY(seq_ok(kv, "copy", dst));
    if (kv->book.seq(dst).length > 0) return fail(AESIR_ERR_INVALID, "KV4Cache.copy: sequence %lld is not empty", (long long)dst);
    const int64_t need = (int64_t)kv->book.seq(src).pages.size();
    if (need > kv->book.free_pages())
        return fail(AESIR_ERR_EXHAUSTED, "KV4Cache.copy: %lld pages needed, %lld free", (long long)need,
                    (long long)kv->book.free_pages());
    return guarded("copy", [&]() -> int32_t {
        AESIR_TRY(end_batch(kv));
        std::vector<PageMove> copies;
        if (src != dst) kv->book.copy(src, dst, copies);
        const int32_t rc = copy_pages(kv, copies);
        if (rc != AESIR_OK) kv->book.truncate(dst, 0);
        return rc;
    });
}

int32_t aesir_kv4_truncate(aesir_kv4 *kv, int64_t seq, int64_t length) {
    AESIR_TRY(can_change(kv, "truncate"));
    AESIR_TRY(seq_ok(kv, "truncate", seq));
    if (length < 0 || length > kv->book.seq(seq).length)
        return fail(AESIR_ERR_INVALID, "KV4Cache.truncate: length %lld is not in [0, %lld]", (long long)length,
                    (long long)kv->book.seq(seq).length);
    return guarded("truncate", [&]() -> int32_t {
        AESIR_TRY(end_batch(kv));
        kv->book.truncate(seq, length);
        return AESIR_OK;
    });
}

int32_t aesir_kv4_compact(aesir_kv4 *kv, int64_t *used_pages) {
    AESIR_TRY(can_change(kv, "compact"));
    return guarded("compact", [&]() -> int32_t {
        AESIR_TRY(end_batch(kv));
        std::vector<PageMove> moves;
        const int64_t used = kv->book.compaction(moves);
        AESIR_TRY(copy_pages(kv, moves));  // to free pages: nothing has changed if it fails
        kv->book.compact(moves);
        if (used_pages) *used_pages = used;
        return AESIR_OK;
    });
}

}  // extern "C"
