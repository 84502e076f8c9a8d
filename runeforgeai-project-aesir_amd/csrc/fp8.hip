// The 8-bit floating-point path for gfx950: rows and weights as OCP e4m3 codes with an f32 scale for each block
// (1 x 128 of activations, 128 x 128 of weights), made by quantize, RMSNorm and SwiGLU kernels and multiplied on
// the matrix cores.
//
// With y the values of a block and a = max |y|: scale = f32(a / 448), code = the e4m3 number nearest 448 y / a,
// ties to even. The kernels find t = 448 y / a in f32, a few units of its last place off, and convert it; where t
// lies that near the middle of two codes it is found again in f64, so that every code is the one of
// the formula.
#include "device.hpp"
#include "kernels.hpp"
#include "mfma_gemm.hpp"

namespace aesir {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;      // elements of a block's row
constexpr float kE4m3Max = 448.0f;  // largest e4m3 number
constexpr unsigned kInfBits = 0x7f800000u;

// ------------------------------------------------------------------ codes

// Whether t, up to `near` units of the last place off, may lie on the other side of the middle of two e4m3 numbers:
// the 20 low bits of an f32 are what e4m3 drops, and its numbers below 2^-6 are as far apart as those just above,
// where adding 2^-6 takes them.
__device__ __forceinline__ bool near_middle(float t, unsigned near) {
    float v = fabsf(t);
    v = v < 0.015625f ? v + 0.015625f : v;
    return (__builtin_bit_cast(unsigned, v) & 0xfffffu) - (0x80000u - near) <= 2 * near;
}

// f32 of t cut towards zero, its last bit set where something was cut: rounding it to e4m3 gives what rounding t does.
__device__ __forceinline__ float to_odd(double t) {
    unsigned b = __builtin_bit_cast(unsigned, (float)t);
    if (fabs((double)__builtin_bit_cast(float, b)) > fabs(t)) b--;
    if ((double)__builtin_bit_cast(float, b) != t) b |= 1;
    return __builtin_bit_cast(float, b);
}

__device__ __forceinline__ u32x2 to_e4m3(const float (&t)[8]) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[4], t[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(t[6], t[7], hi, true);
    return {(unsigned)lo, (unsigned)hi};
}

// Bits of the largest |p|: as unsigned numbers those of finite values order as the values, inf's and NaN's above all.
__device__ __forceinline__ unsigned top_bits(const float (&p)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) m = max(m, __builtin_bit_cast(unsigned, p[j]) & 0x7fffffffu);
    return m;
}

// Maximum over each 16 lanes; every one gets it.
__device__ __forceinline__ unsigned row_max(unsigned m) {
    m = max(m, (unsigned)dpp_i<kDppXor1>((int)m));
    m = max(m, (unsigned)dpp_i<kDppXor2>((int)m));
    m = max(m, (unsigned)dpp_i<kDppHalfMirror>((int)m));
    return max(m, (unsigned)dpp_i<kDppMirror>((int)m));
}
__device__ __forceinline__ unsigned wave_max_u(unsigned m) {
    m = row_max(m);
    const auto r16 = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max((unsigned)r16[0], (unsigned)r16[1]);
    const auto r32 = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return max((unsigned)r32[0], (unsigned)r32[1]);
}

constexpr u32x2 kNanCodes = {0x7f7f7f7fu, 0x7f7f7f7fu};

// Codes of 8 values p that are exact in f32 with at most 22 bits (f16 numbers or products of two), top the bits of
// their block's largest |p|. t is off by at most 2 units of its last place (the quotient and the product are rounded
// once each); 448 p is exact in f64, and a quotient that is no middle is at least 2^-28 of one away from it.
__device__ __forceinline__ u32x2 codes_of(const float (&p)[8], unsigned top) {
    if (top >= kInfBits) return kNanCodes;
    const float a = __builtin_bit_cast(float, top), inv = top ? kE4m3Max / a : 0.0f;
    float t[8];
    bool near = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        t[j] = p[j] * inv;
        near |= near_middle(t[j], 4);
    }
    if (near) {
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = to_odd((double)p[j] * 448.0 / (double)a);
    }
    return to_e4m3(t);
}

// ------------------------------------------------------------------ rows

// 8 f16 elements of a row from column c on, zeros behind its `cols`. whole: every row holds whole, 16-byte aligned
// groups of 8.
__device__ __forceinline__ u32x4 load8(const h16 *row, int64_t c, int64_t cols, bool whole) {
    u32x4 v = {0, 0, 0, 0};
    if (whole) {
        if (c < cols) v = ld16(row + c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < cols) v[j / 2] |= (unsigned)h_to_bits(row[c + j]) << (16 * (j & 1));
    }
    return v;
}
__device__ __forceinline__ void store8(h16 *row, int64_t c, int64_t cols, bool whole, u32x4 v) {
    if (whole) {
        if (c < cols) st16(row + c, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < cols) row[c + j] = bits_to_h((uint16_t)(v[j / 2] >> (16 * (j & 1))));
    }
}
__device__ __forceinline__ void unpack8(u32x4 v, float (&p)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const h16x2 h = as_h2(v[j]);
        p[2 * j] = (float)h.x;
        p[2 * j + 1] = (float)h.y;
    }
}

static bool whole_rows(int64_t cols, int64_t stride, const void *p) {
    return cols % 8 == 0 && stride % 8 == 0 && ((uintptr_t)p & 15) == 0;
}
static int64_t fp8_blocks(int64_t cols) { return (cols + kFp8Block - 1) / kFp8Block; }

// ------------------------------------------------------------------ quantize

// 16 lanes a block: 8 neighbouring elements each.
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const h16 *__restrict__ x, int64_t stride, int64_t rows, int64_t cols,
                                                           bool whole, uint8_t *__restrict__ q, float *__restrict__ scales) {
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block, unit = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (unit >= rows * nb) return;
    const int64_t r = unit / nb, b = unit % nb, c = b * kFp8Block + 8 * (threadIdx.x % 16);
    float p[8];
    unpack8(load8(x + r * stride, c, cols, whole), p);
    const unsigned top = row_max(top_bits(p));
    *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = codes_of(p, top);
    if (threadIdx.x % 16 == 0)
        scales[b * rows + r] = top >= kInfBits ? __builtin_nanf("") : __builtin_bit_cast(float, top) / kE4m3Max;
}

// A workgroup per 128 x 128 block, its 16384 elements in registers between the maximum and the codes.
__global__ __launch_bounds__(256) void fp8_quantize_weight_kernel(const h16 *__restrict__ x, int64_t stride, int64_t rows,
                                                                  int64_t cols, bool whole, uint8_t *__restrict__ q,
                                                                  float *__restrict__ scales) {
    __shared__ unsigned tops[4];
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block, rb = blockIdx.x / nb, b = blockIdx.x % nb;
    const int64_t r0 = rb * kFp8Block + threadIdx.x / 16, c = b * kFp8Block + 8 * (threadIdx.x % 16);
    u32x4 v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = {0, 0, 0, 0};
        if (r0 + 16 * i < rows) v[i] = load8(x + (r0 + 16 * i) * stride, c, cols, whole);
    }
    unsigned top = 0;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        unpack8(v[i], p);
        top = max(top, top_bits(p));
    }
    top = wave_max_u(top);
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        unpack8(v[i], p);
        if (r0 + 16 * i < rows) *reinterpret_cast<u32x2 *>(q + (r0 + 16 * i) * nb * kFp8Block + c) = codes_of(p, top);
    }
    if (threadIdx.x == 0)
        scales[blockIdx.x] = top >= kInfBits ? __builtin_nanf("") : __builtin_bit_cast(float, top) / kE4m3Max;
}

int32_t launch_quantize_fp8(hipStream_t s, const void *x, int64_t stride, int64_t rows, int64_t cols, bool weight, void *q,
                            float *scales) {
    const bool whole = whole_rows(cols, stride, x);
    const int64_t nb = fp8_blocks(cols), groups = weight ? (rows + 127) / 128 * nb : (rows * nb + 15) / 16;
    if (groups > 0x7fffffff) return fail(AESIR_ERR_UNSUPPORTED, "quantize_fp8: more elements than one launch takes");
    if (weight)
        hipLaunchKernelGGL(fp8_quantize_weight_kernel, dim3((unsigned)groups), dim3(256), 0, s, (const h16 *)x, stride, rows, cols,
                           whole, (uint8_t *)q, scales);
    else
        hipLaunchKernelGGL(fp8_quantize_kernel, dim3((unsigned)groups), dim3(256), 0, s, (const h16 *)x, stride, rows, cols, whole,
                           (uint8_t *)q, scales);
    AESIR_LAUNCH_CHECK("fp8_quantize_kernel");
    return AESIR_OK;
}

// ------------------------------------------------------------------ RMSNorm

// A workgroup per row. h = f16(x + residual), y = h w / sqrt(mean h^2 + eps): the row's factor changes no code, so the
// codes are those of h w, exact in f32, and the factor goes into the scales. A row with an inf or NaN is NaN whole.
__global__ __launch_bounds__(256) void fp8_norm_kernel(const h16 *x, int64_t x_stride, const h16 *residual,
                                                       int64_t res_stride, h16 *sum, int64_t sum_stride,
                                                       const h16 *__restrict__ w, float eps, int64_t rows, int64_t cols, bool whole,
                                                       bool w_whole, uint8_t *__restrict__ q, float *__restrict__ scales) {
    __shared__ float red[4];
    const int64_t r = blockIdx.x, nb = (cols + kFp8Block - 1) / kFp8Block;
    const h16 *xr = x + r * x_stride;
    float ss = 0.0f;
    for (int64_t c = 8 * threadIdx.x; c < nb * kFp8Block; c += 2048) {
        u32x4 v = load8(xr, c, cols, whole);
        if (residual) {
            const u32x4 d = load8(residual + r * res_stride, c, cols, whole);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const h16x2 a = as_h2(v[j]), b = as_h2(d[j]);
                v[j] = h2_bits(h16x2{hadd(a.x, b.x), hadd(a.y, b.y)});
            }
            store8(sum + r * sum_stride, c, cols, whole, v);
        }
        float h[8];
        unpack8(v, h);
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(h[j], h[j], ss);
    }
    ss = block_sum<4>(ss, red);
    const float factor = 1.0f / sqrtf(ss / (float)cols + eps);
    for (int64_t c = 8 * threadIdx.x; c < nb * kFp8Block; c += 2048) {
        float p[8], g[8];
        unpack8(residual ? load8(sum + r * sum_stride, c, cols, whole) : load8(xr, c, cols, whole), p);
        unpack8(load8(w, c, cols, w_whole), g);
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] *= g[j];
        unsigned top = row_max(top_bits(p));
        if (!(ss < __builtin_inff())) top = kInfBits;
        *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = codes_of(p, top);
        if (threadIdx.x % 16 == 0)
            scales[c / kFp8Block * rows + r] =
                top >= kInfBits ? __builtin_nanf("") : __builtin_bit_cast(float, top) * factor / kE4m3Max;
    }
}

int32_t launch_rmsnorm_fp8(hipStream_t s, const void *x, int64_t x_stride, const void *residual, int64_t res_stride, void *sum,
                           int64_t sum_stride, const void *w, float eps, int64_t rows, int64_t cols, void *q, float *scales) {
    if (rows > 0x7fffffff) return fail(AESIR_ERR_UNSUPPORTED, "rmsnorm_fp8: too many rows");
    const bool whole = whole_rows(cols, x_stride, x) && (!residual || (whole_rows(cols, res_stride, residual) && whole_rows(cols, sum_stride, sum)));
    hipLaunchKernelGGL(fp8_norm_kernel, dim3((unsigned)rows), dim3(256), 0, s, (const h16 *)x, x_stride, (const h16 *)residual,
                       res_stride, (h16 *)sum, sum_stride, (const h16 *)w, eps, rows, cols, whole, whole_rows(cols, 8, w),
                       (uint8_t *)q, scales);
    AESIR_LAUNCH_CHECK("fp8_norm_kernel");
    return AESIR_OK;
}

// ------------------------------------------------------------------ SwiGLU

// y = u g / (1 + exp(-g)), at most 4 units of f32's last place off: u g is exact, the exponential is 2^hi (1 + lo ln 2)
// with hi + lo = -g log2(e), and the quotient is rounded once.
__device__ __forceinline__ float swiglu_f(float g, float u) {
    const float hi = g * -1.44269504088896341f;
    const float lo = fmaf(g, -1.44269504088896341f, -hi) + g * -1.92596299112661746e-8f;
    return u * g / (1.0f + __builtin_amdgcn_exp2f(hi) * fmaf(lo, 0.693147180559945309f, 1.0f));
}
__device__ __forceinline__ double swiglu_d(float g, float u) { return (double)u * (double)g / (1.0 + exp(-(double)g)); }

constexpr float kSwigluLeast = 0x1p-64f;  // a block of smaller values is zeros

// 16 lanes a block, as fp8_quantize_kernel. Where a quotient or the maximum is in doubt the block's lanes find all its
// values in f64.
__global__ __launch_bounds__(256) void fp8_swiglu_kernel(const h16 *__restrict__ gate, int64_t g_stride, const h16 *__restrict__ up,
                                                         int64_t u_stride, int64_t rows, int64_t cols, bool whole,
                                                         uint8_t *__restrict__ q, float *__restrict__ scales) {
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block, unit = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (unit >= rows * nb) return;
    const int64_t r = unit / nb, b = unit % nb, c = b * kFp8Block + 8 * (threadIdx.x % 16);
    float g[8], u[8], y[8];
    unpack8(load8(gate + r * g_stride, c, cols, whole), g);
    unpack8(load8(up + r * u_stride, c, cols, whole), u);
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = swiglu_f(g[j], u[j]);
    const unsigned top = row_max(top_bits(y));
    const float a = __builtin_bit_cast(float, top);
    float scale = a >= kSwigluLeast ? a / kE4m3Max : 0.0f;
    const float inv = a >= kSwigluLeast ? kE4m3Max / a : 0.0f;
    bool near = fabsf(a - kSwigluLeast) <= 0x1p-84f;
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        t[j] = y[j] * inv;
        near |= near_middle(t[j], 16);
    }
    if (row_max(near)) {
        double yd[8], m = 0.0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            yd[j] = swiglu_d(g[j], u[j]);
            m = fmax(m, fabs(yd[j]));
        }
#pragma unroll
        for (int i = 1; i < 16; i <<= 1) m = fmax(m, __shfl_xor(m, i));
        const bool some = m >= (double)kSwigluLeast;
        scale = some ? (float)(m / 448.0) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = some ? to_odd(yd[j] * 448.0 / m) : 0.0f;
    }
    const bool bad = top >= kInfBits;
    *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = bad ? kNanCodes : to_e4m3(t);
    if (threadIdx.x % 16 == 0) scales[b * rows + r] = bad ? __builtin_nanf("") : scale;
}

int32_t launch_swiglu_fp8(hipStream_t s, const void *gate, int64_t g_stride, const void *up, int64_t u_stride, int64_t rows,
                          int64_t cols, void *q, float *scales) {
    const int64_t groups = (rows * fp8_blocks(cols) + 15) / 16;
    if (groups > 0x7fffffff) return fail(AESIR_ERR_UNSUPPORTED, "swiglu_fp8: more elements than one launch takes");
    hipLaunchKernelGGL(fp8_swiglu_kernel, dim3((unsigned)groups), dim3(256), 0, s, (const h16 *)gate, g_stride, (const h16 *)up,
                       u_stride, rows, cols, whole_rows(cols, g_stride, gate) && whole_rows(cols, u_stride, up), (uint8_t *)q, scales);
    AESIR_LAUNCH_CHECK("fp8_swiglu_kernel");
    return AESIR_OK;
}

// ------------------------------------------------------------------ product

// A lane's 32 codes of a row's k-block: k-granules (16 codes) g and g + 4 of the block's 8, g = lane / 16. Any split
// of the 128 works that both operands share.
struct Frag8 {
    u32x4 lo, hi;
};
// The same as the f16 numbers they are (exact): 4 groups of 8.
struct Frag16 {
    u32x4 v[4];
};

__device__ __forceinline__ Frag16 to_f16(Frag8 f) {
    Frag16 r;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned w = i < 4 ? f.lo[i] : f.hi[i - 4];
        r.v[i / 2][2 * (i & 1)] = h2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
        r.v[i / 2][2 * (i & 1) + 1] = h2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
    return r;
}

// D = A B on one 16 x 16 x 128 tile. Lane l holds A row l % 16 and B column l % 16, and D rows 4 (l / 16) + e, column
// l % 16, in element e.
//
// The 8-bit matrix instructions do not keep all of f32: of the products of 8 neighbouring k they drop what lies under
// 2^-13 of the power of two at the largest (measured: both 16x16x128 and 16x16x32, 1.3e-5 of a sum of near normal
// products, its norm against f64), which f16 results, rounded by 2.8e-4, do not show. f32 results and products that
// wait for memory anyway take the f16 instruction, whose sums are f32, on the numbers converted; it runs at half the
// rate.
__device__ __forceinline__ f32x4 mma_block(Frag8 a, Frag8 b) {
    const i32x8 av = {(int)a.lo.x, (int)a.lo.y, (int)a.lo.z, (int)a.lo.w, (int)a.hi.x, (int)a.hi.y, (int)a.hi.z, (int)a.hi.w};
    const i32x8 bv = {(int)b.lo.x, (int)b.lo.y, (int)b.lo.z, (int)b.lo.w, (int)b.hi.x, (int)b.hi.y, (int)b.hi.z, (int)b.hi.w};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_block(const Frag16 &a, const Frag16 &b) {
    f32x4 d = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) d = mfma16x16x32(a.v[i], b.v[i], d);
    return d;
}

struct Fp8Args {
    const uint8_t *a, *b;  // codes [M][ld], [N][ld]
    const float *as, *bs;  // scales [ld / 128][M], [ceil(N / 128)][ld / 128]
    void *c;
    int64_t M, N, ldc;
    int nb;  // blocks along k
    bool f32;
};

__device__ __forceinline__ void fp8_store(const Fp8Args &p, int64_t m, int64_t n, f32x4 v) {
    if (m >= p.M) return;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= p.N) return;
        if (p.f32)
            ((float *)p.c)[m * p.ldc + n + e] = v[e];
        else
            ((h16 *)p.c)[m * p.ldc + n + e] = (h16)v[e];
    }
}

// Tile of 128 rows of A by 128 of B, 4 waves of 64 x 64, two LDS stages of one k-block. Weights are the first
// operand of the matrix instruction, so a lane's elements are 4 neighbouring columns of one row of C.
template <bool EXACT>
__global__ __launch_bounds__(256) void fp8_gemm_kernel(Fp8Args p) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t mt = (p.M + 127) / 128, m0 = blockIdx.x % mt * 128, n0 = blockIdx.x / mt * 128;
    const int64_t ld = (int64_t)p.nb * 128;
    const int rows_a = (int)min((int64_t)128, p.M - m0), rows_b = (int)min((int64_t)128, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void *)(p.a + m0 * ld), 0, (int)(rows_a * ld), kBufferDword3);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)(p.b + n0 * ld), 0, (int)(rows_b * ld), kBufferDword3);
    // a copy instruction moves 8 rows of 128 bytes: lane l fills slot l % 8 of row l / 8 with granule
    // (l % 8) ^ (row / 2 % 8), so that the 16 rows a fragment reads at once lie in different banks
    auto request = [&](int stage, int kb) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = (wave * 8 + i) % 16 * 8 + lane / 8;
            const int off = (int)(r * ld) + kb * 128 + ((lane & 7) ^ ((r >> 1) & 7)) * 16;
            uint8_t *dst = lds + stage * 32768 + (wave * 8 + i) * 1024;
            if (wave < 2)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void *)dst, 16, off, 0, 0, 0);
            else
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void *)dst, 16, off, 0, 0, 0);
        }
    };
    const int wm = wave % 2 * 64, wn = wave / 2 * 64, i16 = lane & 15;
    const int at = i16 * 128 + ((lane >> 4) ^ (i16 >> 1)) * 16;
    f32x4 acc[4][4] = {};
    request(0, 0);
    for (int kb = 0; kb < p.nb; kb++) {
        __builtin_amdgcn_s_waitcnt(vm_wait(0));
        __syncthreads();
        if (kb + 1 < p.nb) request((kb + 1) & 1, kb + 1);
        const uint8_t *la = lds + (kb & 1) * 32768 + wm * 128, *lb = lds + (kb & 1) * 32768 + 16384 + wn * 128;
        const float sb = p.bs[n0 / 128 * p.nb + kb];
        using Frag = std::conditional_t<EXACT, Frag16, Frag8>;
        auto frag = [&](const uint8_t *row) {
            const Frag8 f{ld16(row + at), ld16(row + (at ^ 64))};
            if constexpr (EXACT)
                return to_f16(f);
            else
                return f;
        };
        Frag a[4];
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t m = m0 + wm + 16 * j + i16;
            s[j] = m < p.M ? p.as[kb * p.M + m] * sb : 0.0f;
            a[j] = frag(la + 2048 * j);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const Frag b = frag(lb + 2048 * i);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const f32x4 d = mma_block(b, a[j]);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(d[e], s[j], acc[i][j][e]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) fp8_store(p, m0 + wm + 16 * j + i16, n0 + wn + 16 * i + 4 * (lane >> 4), acc[i][j]);
}

int32_t launch_gemm_fp8(hipStream_t s, const void *A, const float *as, int64_t M, const void *B, const float *bs, int64_t N,
                        int64_t K, void *C, bool f32, int64_t ldc) {
    const int64_t nb = fp8_blocks(K);
    const Fp8Args p{(const uint8_t *)A, (const uint8_t *)B, as, bs, C, M, N, ldc, (int)nb, f32};
    const int64_t tiles = (M + 127) / 128 * ((N + 127) / 128);
    if (tiles > 0x7fffffff) return fail(AESIR_ERR_UNSUPPORTED, "gemm_fp8: output larger than one launch takes");
    hipLaunchKernelGGL(f32 ? fp8_gemm_kernel<true> : fp8_gemm_kernel<false>, dim3((unsigned)tiles), dim3(256), 65536, s, p);
    AESIR_LAUNCH_CHECK("fp8_gemm_kernel");
    return AESIR_OK;
}

}  // namespace aesir
