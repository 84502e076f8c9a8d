// The paged 4-bit KV cache: appending (quantizing) rows, attention over the pages, reading values back, page
// copies, and the C entry points with the bookkeeping of pages and sequences.
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
// hold too little.
struct Kv4Upload {
    const uint32_t *src;
    uint32_t *dst[3];   // contiguous runs, in the order of src
    int32_t words[3];
    int32_t *table;     // then `updates` pairs (table entry, page)
    int32_t updates;
};

__global__ __launch_bounds__(kThreads) void kv4_upload_kernel(Kv4Upload u) {
    const int all = u.words[0] + u.words[1] + u.words[2];
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < all + u.updates; i += gridDim.x * kThreads) {
        if (i >= all) {
            const uint32_t *e = u.src + all + 2 * (int64_t)(i - all);
            u.table[e[0]] = (int32_t)e[1];
            continue;
        }
        int j = i, run = 0;
        while (j >= u.words[run]) j -= u.words[run++];
        u.dst[run][j] = u.src[i];
    }
}

// Index of the last of n ascending values that is <= x (the first is 0, x >= 0), from LDS.
__device__ __forceinline__ int last_not_above(const int *v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

constexpr int kMaxSeqs = 4096;  // a batch's first rows fit LDS

// ------------------------------------------------------------------ append
//
// One thread per 8 dims of a K and of a V row (16-byte loads); the four lanes of a quad hold a group of 32, whose
// minimum and maximum they exchange by DPP. Four consecutive rows of one head are neighbouring lane groups, so a
// V tile of four positions leaves as one contiguous store. The quantization is exact: scales and levels are the
// nearest ones of the real quotients, ties to even, as their definition says.

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
    h16 d = nearest_half(((double)mx - (double)mn) / 15.0);
    if ((double)mn + 15.0 * (double)(float)d > 65504.0) d = bits_to_h((uint16_t)(h_to_bits(d) - 1));
    const float df = (float)d, inv = df > 0.0f ? 1.0f / df : 0.0f;
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        // t is within 2^-18 of (v - mn) / d; where that could cross a border between levels, the border itself
        // is compared in 64 bits (every term is exact there)
        const float t = (v[i] - mn) * inv, low = floorf(t);
        float q = rintf(t);
        if (fabsf(t - low - 0.5f) < 0x1p-15f) {
            const double u = (double)v[i] - (double)mn, border = ((double)low + 0.5) * (double)df;
            q = u > border || (u == border && ((int)low & 1)) ? low + 1.0f : low;
        }
        w |= (unsigned)fminf(q, 15.0f) << (4 * (i / 2) + 16 * (i % 2));
    }
    c.word = w;
    c.d = d;
    c.m = (h16)mn;
    return c;
}

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

template <bool VEC>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4Dev c, Kv4AppendArgs a) {
    __shared__ int row0[kMaxSeqs];
    const int n = c.head->n, total = min(c.head->total_rows, a.rows);
    for (int i = threadIdx.x; i < n; i += kThreads) row0[i] = c.row0[i];
    __syncthreads();
    const int per_row = c.hd / 8;                                       // threads per row and head
    const int64_t units = ((int64_t)total + 3) / 4 * c.nkv * 4 * per_row;  // four rows of one head together
    for (int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x; u < units; u += (int64_t)gridDim.x * kThreads) {
        const int chunk = (int)(u % per_row);
        const int64_t g = u / per_row;
        const int row = (int)(g / (4 * c.nkv)) * 4 + (int)(g % 4), head = (int)(g / 4 % c.nkv);
        if (row >= total) continue;  // uniform over the quad
        const u32x4 kx = load8<VEC>(a.k + (int64_t)row * a.k_stride + head * c.hd + 8 * chunk);
        const u32x4 vx = load8<VEC>(a.v + (int64_t)row * a.v_stride + head * c.hd + 8 * chunk);
        const Kv4Seq &s = c.seqs[last_not_above(row0, n, row)];
        const int pos = s.length - s.rows + (row - s.row0), slot = pos & (c.page_size() - 1);
        char *b = c.block(c.table[(int64_t)s.slot * c.table_stride + (pos >> c.page_shift)], a.layer, head);
        const Kv4Code ck = kv4_encode(kx), cv = kv4_encode(vx);
        reinterpret_cast<unsigned *>(b)[slot * per_row + chunk] = ck.word;
        reinterpret_cast<unsigned *>(b + c.v_off())[(slot / 4 * per_row + chunk) * 4 + slot % 4] = cv.word;
        if (chunk % 4 == 0) {
            const int grp = chunk / 4;
            reinterpret_cast<h16x2 *>(b + c.k_scale_off())[slot * (c.hd / kKv4Group) + grp] = h16x2{ck.d, ck.m};
            reinterpret_cast<h16 *>(b + c.v_d_off())[grp * c.page_size() + slot] = cv.d;
            reinterpret_cast<h16 *>(b + c.v_m_off())[grp * c.page_size() + slot] = cv.m;
        }
    }
}

// ------------------------------------------------------------------ read
//
// The f16 values of position ranges, one thread per 8 dims of K and V.
struct Kv4ReadArgs {
    h16 *k, *v;
    int64_t k_stride, v_stride;
    int64_t layer, layers;
    const Kv4Range *ranges;
    int32_t n, rows, all_rows, first_row;  // ranges, their rows, output rows of a layer, first output row
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

template <bool VEC>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(Kv4Dev c, Kv4ReadArgs a) {
    __shared__ int row0[kMaxSeqs];
    for (int i = threadIdx.x; i < a.n; i += kThreads) row0[i] = a.ranges[i].row0;
    __syncthreads();
    const int per_row = c.hd / 8;
    const int64_t per_layer = ((int64_t)a.rows + 3) / 4 * c.nkv * 4 * per_row, units = per_layer * a.layers;
    for (int64_t u = (int64_t)blockIdx.x * kThreads + threadIdx.x; u < units; u += (int64_t)gridDim.x * kThreads) {
        const int64_t layer = u / per_layer, x = u % per_layer, g = x / per_row;
        const int chunk = (int)(x % per_row);
        const int row = (int)(g / (4 * c.nkv)) * 4 + (int)(g % 4), head = (int)(g / 4 % c.nkv);
        if (row >= a.rows) continue;
        const Kv4Range r = a.ranges[last_not_above(row0, a.n, row)];
        const int pos = r.pos + (row - r.row0), slot = pos & (c.page_size() - 1), grp = chunk / 4;
        const char *b = c.block(c.table[(int64_t)r.slot * c.table_stride + (pos >> c.page_shift)], a.layer + layer, head);
        const unsigned kw = reinterpret_cast<const unsigned *>(b)[slot * per_row + chunk];
        const unsigned vw = reinterpret_cast<const unsigned *>(b + c.v_off())[(slot / 4 * per_row + chunk) * 4 + slot % 4];
        const h16x2 ks = reinterpret_cast<const h16x2 *>(b + c.k_scale_off())[slot * (c.hd / kKv4Group) + grp];
        const h16 vd = reinterpret_cast<const h16 *>(b + c.v_d_off())[grp * c.page_size() + slot];
        const h16 vm = reinterpret_cast<const h16 *>(b + c.v_m_off())[grp * c.page_size() + slot];
        const int64_t out = layer * a.all_rows + a.first_row + row;
        store8<VEC>(a.k + out * a.k_stride + head * c.hd + 8 * chunk, kv4_decode(kw, ks.x, ks.y));
        store8<VEC>(a.v + out * a.v_stride + head * c.hd + 8 * chunk, kv4_decode(vw, vd, vm));
    }
}

// ------------------------------------------------------------------ page copies
//
// 16 KB of a page per workgroup step, four 16-byte loads in flight per thread. Sources and destinations of one
// launch are disjoint.
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
// o = softmax(q k^T / sqrt(hd)) v of one row and query head over the positions up to the row's own. One wave per
// (row, query head): 64 positions a step, a lane scores one of them, then owns dims lane, lane + 64, ..
struct Kv4AttnArgs {
    const h16 *q;
    h16 *out;
    int64_t q_stride, out_stride;
    int64_t layer;
    int32_t rows;  // rows of q and out
    float scale;
};

__global__ __launch_bounds__(kWave) void kv4_attention_kernel(Kv4Dev c, Kv4AttnArgs a) {
    __shared__ int row0[kMaxSeqs];
    __shared__ float qs[256], ps[kWave];
    const int n = c.head->n, total = min(c.head->total_rows, a.rows), lane = threadIdx.x;
    for (int i = lane; i < n; i += kWave) row0[i] = c.row0[i];
    __syncthreads();
    const int groups = c.hd / kKv4Group;
    for (int64_t u = blockIdx.x; u < (int64_t)total * c.nq; u += gridDim.x) {
        const int row = (int)(u / c.nq), head = (int)(u % c.nq), kvh = head / (c.nq / c.nkv);
        const Kv4Seq s = c.seqs[last_not_above(row0, n, row)];
        const int seen = s.length - s.rows + (row - s.row0) + 1;
        __syncthreads();
        for (int d = lane; d < c.hd; d += kWave) qs[d] = (float)a.q[(int64_t)row * a.q_stride + head * c.hd + d];
        float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int p0 = 0; p0 < seen; p0 += kWave) {
            __syncthreads();
            const int pos = p0 + lane, here = min(seen - p0, kWave);
            float sc = -INFINITY;
            if (lane < here) {
                const int slot = pos & (c.page_size() - 1);
                const char *b = c.block(c.table[(int64_t)s.slot * c.table_stride + (pos >> c.page_shift)], a.layer, kvh);
                float dot = 0.0f;
                for (int g = 0; g < groups; g++) {
                    const h16x2 ks = reinterpret_cast<const h16x2 *>(b + c.k_scale_off())[slot * groups + g];
                    for (int j = 0; j < 4; j++) {
                        const u32x4 v = kv4_decode(reinterpret_cast<const unsigned *>(b)[slot * (c.hd / 8) + 4 * g + j], ks.x, ks.y);
                        for (int e = 0; e < 4; e++) {
                            dot = fmaf((float)as_h2(v[e]).x, qs[32 * g + 8 * j + 2 * e], dot);
                            dot = fmaf((float)as_h2(v[e]).y, qs[32 * g + 8 * j + 2 * e + 1], dot);
                        }
                    }
                }
                sc = dot * a.scale;
            }
            const float mn = fmaxf(m, wave_max(sc)), ref = mn == -INFINITY ? 0.0f : mn;
            const float p = expf(sc - ref), al = expf(m - ref);
            l = l * al + wave_sum(p);
            m = mn;
            ps[lane] = p;
            __syncthreads();
            for (int i = 0; i < 4; i++) {
                const int d = lane + kWave * i;
                if (d >= c.hd) break;
                acc[i] *= al;
                for (int r = 0; r < here; r++) {
                    const int q = p0 + r, slot = q & (c.page_size() - 1);
                    const char *b = c.block(c.table[(int64_t)s.slot * c.table_stride + (q >> c.page_shift)], a.layer, kvh);
                    const unsigned w = reinterpret_cast<const unsigned *>(b + c.v_off())[(slot / 4 * (c.hd / 8) + d / 8) * 4 + slot % 4];
                    const h16 vd = reinterpret_cast<const h16 *>(b + c.v_d_off())[d / 32 * c.page_size() + slot];
                    const h16 vm = reinterpret_cast<const h16 *>(b + c.v_m_off())[d / 32 * c.page_size() + slot];
                    const h16x2 v = kv4_pair(w, d % 8 / 2, both(vd), both(vm));
                    acc[i] = fmaf(ps[r], (float)(d % 2 ? v.y : v.x), acc[i]);
                }
            }
        }
        for (int i = 0; i < 4; i++) {
            const int d = lane + kWave * i;
            if (d < c.hd) a.out[(int64_t)row * a.out_stride + head * c.hd + d] = (h16)(acc[i] / l);
        }
    }
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
    Kv4Head *head = nullptr;
    Kv4Seq *seqs = nullptr;
    int32_t *row0 = nullptr;
    Kv4Range *ranges = nullptr;
    PageMove *moves = nullptr;
    char *ring = nullptr;  // pinned staging, handed out front to back
    int64_t ring_at = 0;
    bool batch = false;
    int64_t batch_rows = 0;

    aesir_kv4(int64_t num_pages, int64_t page_size, int64_t max_seqs) : book(num_pages, page_size, max_seqs) {}
};

namespace {

constexpr int64_t kRingBytes = 1 << 20;
constexpr int64_t kMaxPages = (int64_t)1 << 30;

struct Kv4Sizes {
    int64_t page_bytes, pool, table, seqs, row0, ranges, moves, part;
    int64_t total() const {
        int64_t t = 0;
        for (int64_t b : {pool, table, (int64_t)sizeof(Kv4Head), seqs, row0, ranges, moves, part}) t += (b + 255) / 256 * 256;
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
    const int64_t stride = (max_seq_len + page - 1) / page;
    if (mul_checked(stride, max_seqs) > INT32_MAX) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    z->page_bytes = mul_checked(mul_checked(layers, nkv, page), hd / 4 * 5);
    z->pool = mul_checked(z->page_bytes, pages);
    if (z->pool < 0 || z->pool > (int64_t)1 << 50) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache: a dimension is too large");
    z->table = stride * max_seqs * 4;
    z->seqs = max_seqs * (int64_t)sizeof(Kv4Seq);
    z->row0 = max_seqs * 4;
    z->ranges = max_seqs * (int64_t)sizeof(Kv4Range);
    z->moves = pages * (int64_t)sizeof(PageMove);
    z->part = 256;
    return AESIR_OK;
}

int32_t need_device(aesir_kv4 *kv, const char *what) {
    if (!kv) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: null cache", what);
    if (!kv->ctx) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: the cache has no context (page tables only)", what);
    return bind(kv->ctx);
}

// Calls that change the tables send host data to the device, which a replay would not send again.
int32_t can_change(aesir_kv4 *kv, const char *what) {
    if (!kv) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: null cache", what);
    if (!kv->ctx) {
        clear_error();
        return AESIR_OK;
    }
    AESIR_TRY(bind(kv->ctx));
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    AESIR_HIP_TRY(hipStreamIsCapturing(kv->ctx->stream, &st));
    if (st != hipStreamCaptureStatusNone)
        return fail(AESIR_ERR_INVALID, "KV4Cache.%s: not while the context's stream is being captured", what);
    return AESIR_OK;
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
    int64_t bytes;
};

int32_t launch_upload(aesir_kv4 *kv, const Run *runs, int n_runs, const uint32_t *updates, int64_t n_updates) {
    int64_t bytes = n_updates * 8;
    for (int i = 0; i < n_runs; i++) bytes += runs[i].bytes;
    if (bytes == 0) return AESIR_OK;
    char *p = nullptr;
    AESIR_TRY(stage(kv, bytes, &p));
    Kv4Upload u{};
    u.src = (const uint32_t *)p;
    u.table = kv->table;
    u.updates = (int32_t)n_updates;
    for (int i = 0; i < n_runs; i++) {
        std::memcpy(p, runs[i].src, (size_t)runs[i].bytes);
        p += runs[i].bytes;
        u.dst[i] = (uint32_t *)runs[i].dst;
        u.words[i] = (int32_t)(runs[i].bytes / 4);
    }
    if (n_updates) std::memcpy(p, updates, (size_t)n_updates * 8);
    const int64_t threads = bytes / 4 - n_updates;
    const unsigned blocks = (unsigned)std::min<int64_t>(256, (threads + kThreads - 1) / kThreads);
    hipLaunchKernelGGL(kv4_upload_kernel, dim3(blocks), dim3(kThreads), 0, kv->ctx->stream, u);
    AESIR_LAUNCH_CHECK("kv4_upload_kernel");
    return AESIR_OK;
}

// Brings the device's table rows of the listed sequences up to date, with `runs` in the last launch.
int32_t upload(aesir_kv4 *kv, const int64_t *seqs, int64_t n, const Run *runs, int n_runs) {
    const int64_t most = kRingBytes / 4 / 8;
    std::vector<uint32_t> e;
    for (int64_t i = 0; i < n; i++) {
        const PageBook::Seq &s = kv->book.seq(seqs[i]);
        for (int64_t j = s.synced; j < (int64_t)s.pages.size(); j++) {
            e.push_back((uint32_t)(seqs[i] * kv->dev.table_stride + j));
            e.push_back((uint32_t)s.pages[(size_t)j]);
            if ((int64_t)e.size() == 2 * most) {
                AESIR_TRY(launch_upload(kv, nullptr, 0, e.data(), most));
                e.clear();
            }
        }
        kv->book.mark_synced(seqs[i]);
    }
    return launch_upload(kv, runs, n_runs, e.data(), (int64_t)e.size() / 2);
}

// Uploads the moves and copies the pages.
int32_t copy_pages(aesir_kv4 *kv, const std::vector<PageMove> &moves) {
    if (!kv->ctx) return AESIR_OK;
    const int64_t most = kRingBytes / 4 / (int64_t)sizeof(PageMove);
    for (int64_t at = 0; at < (int64_t)moves.size(); at += most) {
        const int64_t n = std::min<int64_t>(most, (int64_t)moves.size() - at);
        const Run r{kv->moves + at, moves.data() + at, n * (int64_t)sizeof(PageMove)};
        AESIR_TRY(launch_upload(kv, &r, 1, nullptr, 0));
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
    const Kv4Head none{};
    const Run r{kv->head, &none, (int64_t)sizeof none};
    return launch_upload(kv, &r, 1, nullptr, 0);
}

template <class F>
int32_t guarded(const char *what, F f) {
    try {
        return f();
    } catch (const std::exception &) {
        return fail(AESIR_ERR_EXHAUSTED, "KV4Cache.%s: out of host memory", what);
    }
}

bool aligned16(const void *p, int64_t cols) { return ((uintptr_t)p & 15) == 0 && cols % 8 == 0; }

unsigned grid_for(int64_t threads) { return (unsigned)std::min<int64_t>(std::max<int64_t>((threads + kThreads - 1) / kThreads, 1), 1 << 20); }

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
    if (total > INT32_MAX / kv->nq) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache.begin: too many rows");
    const int64_t need = kv->book.pages_needed(seqs, rows, n);
    if (need > kv->book.free_pages())
        return fail(AESIR_ERR_EXHAUSTED, "KV4Cache.begin: %lld pages needed, %lld free", (long long)need,
                    (long long)kv->book.free_pages());
    std::vector<PageMove> copies;
    std::vector<Kv4Seq> ds((size_t)n);
    std::vector<int32_t> row0((size_t)n);
    copies.reserve((size_t)n);
    for (int64_t i = 0; i < n; i++) kv->book.reserve(seqs[i], kv->book.seq(seqs[i]).length + rows[i]);
    Kv4Head h{};
    h.n = (int32_t)n;
    h.total_rows = (int32_t)total;
    int64_t at = 0;
    for (int64_t i = 0; i < n; i++) {
        kv->book.grow(seqs[i], rows[i], copies);
        Kv4Seq &s = ds[(size_t)i];
        s = Kv4Seq{};
        s.slot = (int32_t)seqs[i];
        s.length = (int32_t)kv->book.seq(seqs[i]).length;
        s.rows = (int32_t)rows[i];
        s.row0 = row0[(size_t)i] = (int32_t)at;
        at += rows[i];
    }
    kv->batch = true;
    kv->batch_rows = total;
    if (!kv->ctx) return AESIR_OK;
    const Run runs[3] = {{kv->head, &h, (int64_t)sizeof h},
                         {kv->seqs, ds.data(), n * (int64_t)sizeof(Kv4Seq)},
                         {kv->row0, row0.data(), n * 4}};
    AESIR_TRY(upload(kv, seqs, n, runs, 3));
    return copy_pages(kv, copies);
}

int32_t layer_ok(aesir_kv4 *kv, const char *what, int64_t layer) {
    if (layer < 0 || layer >= kv->layers) return fail(AESIR_ERR_INVALID, "KV4Cache.%s: layer out of bounds", what);
    return AESIR_OK;
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
    if (ctx) AESIR_TRY(bind(ctx));
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
        void *p[8] = {};
        const int64_t bytes[8] = {z.pool, z.table, (int64_t)sizeof(Kv4Head), z.seqs, z.row0, z.ranges, z.moves, z.part};
        int32_t rc = AESIR_OK;
        for (int i = 0; i < 8 && rc == AESIR_OK; i++) rc = well_alloc_bytes(ctx, bytes[i], &p[i]);
        if (rc == AESIR_OK && hipHostMalloc((void **)&kv->ring, kRingBytes, hipHostMallocDefault) != hipSuccess)
            rc = fail(AESIR_ERR_HIP, "hipHostMalloc of the cache's staging memory failed");
        if (rc != AESIR_OK) {
            ctx->well_offset = mark;
            delete kv;
            return rc;
        }
        kv->ctx = ctx;
        kv->table = (int32_t *)p[1];
        kv->head = (Kv4Head *)p[2];
        kv->seqs = (Kv4Seq *)p[3];
        kv->row0 = (int32_t *)p[4];
        kv->ranges = (Kv4Range *)p[5];
        kv->moves = (PageMove *)p[6];
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
        d.head = kv->head;
        d.seqs = kv->seqs;
        d.row0 = kv->row0;
        d.part = (float *)p[7];
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
        AESIR_TRY(bind(kv->ctx));
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
    if (!key || !val) return fail(AESIR_ERR_INVALID, "KV4Cache.append: null tensor pointer");
    const Kv4AppendArgs a{(const h16 *)key, (const h16 *)val, key_cols, val_cols, layer, (int32_t)key_rows};
    const dim3 grid(grid_for((key_rows + 3) / 4 * kv->nkv * (kv->hd / 2)));
    if (aligned16(key, key_cols) && aligned16(val, val_cols))
        hipLaunchKernelGGL(kv4_append_kernel<true>, grid, dim3(kThreads), 0, kv->ctx->stream, kv->dev, a);
    else
        hipLaunchKernelGGL(kv4_append_kernel<false>, grid, dim3(kThreads), 0, kv->ctx->stream, kv->dev, a);
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
    if (!query || !output) return fail(AESIR_ERR_INVALID, "KV4Cache.attention: null tensor pointer");
    const Kv4AttnArgs a{(const h16 *)query, (h16 *)output, query_cols, output_cols, layer, (int32_t)query_rows,
                        (float)(1.0 / std::sqrt((double)kv->hd))};
    hipLaunchKernelGGL(kv4_attention_kernel, dim3((unsigned)std::min<int64_t>(query_rows * kv->nq, 1 << 20)), dim3(kWave), 0,
                       kv->ctx->stream, kv->dev, a);
    AESIR_LAUNCH_CHECK("kv4_attention_kernel");
    return AESIR_OK;
}

int32_t aesir_kv4_read(aesir_kv4 *kv, int64_t layer, int64_t layers, const int64_t *seqs, const int64_t *pos, const int64_t *rows,
                       int64_t n, void *key, int64_t key_rows, int64_t key_cols, void *val, int64_t val_rows, int64_t val_cols) {
    AESIR_TRY(need_device(kv, "read"));
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
        if (total > INT32_MAX) return fail(AESIR_ERR_UNSUPPORTED, "KV4Cache.read: too many rows");
    }
    if (key_rows != total * layers || val_rows != total * layers)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.read: %lld rows are asked for", (long long)(total * layers));
    if (total * layers == 0) return AESIR_OK;
    if (key_cols < kv->nkv * kv->hd || val_cols < kv->nkv * kv->hd)
        return fail(AESIR_ERR_SHAPE, "KV4Cache.read: key/val rows narrower than kv_heads * head_dim");
    if (!key || !val) return fail(AESIR_ERR_INVALID, "KV4Cache.read: null tensor pointer");
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
            const Run run{kv->ranges, r.data(), m * (int64_t)sizeof(Kv4Range)};
            AESIR_TRY(upload(kv, seqs + at, m, &run, 1));
            const Kv4ReadArgs a{(h16 *)key, (h16 *)val, key_cols,     val_cols,       layer,         layers,
                                kv->ranges, (int32_t)m, (int32_t)count, (int32_t)total, (int32_t)first};
            const dim3 grid(grid_for((count + 3) / 4 * kv->nkv * (kv->hd / 2) * layers));
            if (vec)
                hipLaunchKernelGGL(kv4_read_kernel<true>, grid, dim3(kThreads), 0, kv->ctx->stream, kv->dev, a);
            else
                hipLaunchKernelGGL(kv4_read_kernel<false>, grid, dim3(kThreads), 0, kv->ctx->stream, kv->dev, a);
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
        return copy_pages(kv, copies);
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
        const int64_t used = kv->book.compact(moves);
        if (used_pages) *used_pages = used;
        return copy_pages(kv, moves);
    });
}

}  // extern "C"
