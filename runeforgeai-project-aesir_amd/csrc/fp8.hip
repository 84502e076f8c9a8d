// The 8-bit floating-point path for gfx950: rows and weights as OCP e4m3 codes with an f32 scale for each block
// (1 x 128 of activations, 128 x 128 of weights), made by quantize, RMSNorm and SwiGLU kernels and multiplied on
// the matrix cores.
//
// With y the values of a block and a = max |y|: scale = f32(a / 448), code = the e4m3 number nearest 448 y / a,
// ties to even. The kernels find t = 448 y / a in f32, a few units of its last place off, and round both ends of an
// interval that holds the exact quotient: rounding is monotone, so where both give the same code so does the quotient.
// Elsewhere it is found again in f64, so that every code is the one of the formula: one element in 9 * 10^4 of
// quantize and RMSNorm (ends 2^-21 of it off), one in 2 * 10^4 of SwiGLU (2^-19), whose whole block is done again, one in 180.
// That is for values of many bits. Ties of two codes come often where all the values of a block are whole multiples of a
// 7 * 2^n-th of its largest and take more than e4m3's 4 bits: quantizing 28672 x 4096 weights takes 65 us if they are normal, 55 if
// they are integers up to 7, 15 or 127, and 107 if integers up to 28 or 112.
#include <algorithm>
#include <cmath>
#include <limits>

#include "device.hpp"
#include "kernels.hpp"
#include "mfma_gemm.hpp"

namespace aesir {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;      // elements of a block's row
constexpr float kE4m3Max = 448.0f;  // largest e4m3 number
constexpr unsigned kInfBits = 0x7f800000u;

// ------------------------------------------------------------------ codes

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
// The same of 8 f16 numbers, as f32 bits.
__device__ __forceinline__ unsigned top_bits(u32x4 v) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; j++) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[j] & 0x7fff7fffu));
    return __builtin_bit_cast(unsigned, (float)bits_to_h(max(m.x, m.y)));
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
// their block's largest |p|. p times 448 / a is off by at most 2^-22 of it (the reciprocal's 2^-23 and two products'
// 2^-24), so that the ends of an interval 2^-21 either way hold it; 448 p is exact in f64, and a quotient that is not the
// middle of two codes is at least 2^-28 of it away from one.
__device__ __forceinline__ u32x2 codes_of(const float (&p)[8], unsigned top) {
    if (top >= kInfBits) return kNanCodes;
    if (top == 0) return {0, 0};  // of zeros of either sign
    const float a = __builtin_bit_cast(float, top), inv = __builtin_amdgcn_rcpf(a);
    const float less = inv * (kE4m3Max * (1.0f - 0x1p-21f)), more = inv * (kE4m3Max * (1.0f + 0x1p-21f));
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        lo[j] = p[j] * less;
        hi[j] = p[j] * more;
    }
    const u32x2 c = to_e4m3(lo), d = to_e4m3(hi);
    if (((c.x ^ d.x) | (c.y ^ d.y)) == 0) return c;
#pragma unroll
    for (int j = 0; j < 8; j++) lo[j] = to_odd((double)p[j] * 448.0 / (double)a);
    return to_e4m3(lo);
}

// ------------------------------------------------------------------ rows

// 8 f16 elements of a row from column c on, zeros behind its `cols`. whole: every row holds whole, 16-byte aligned
// groups of 8. ONCE: nothing reads them again (non-temporal: SwiGLU of 4096 x 14336 60 us against 67).
template <bool ONCE = true>
__device__ __forceinline__ u32x4 load8(const h16 *row, int64_t c, int64_t cols, bool whole) {
    u32x4 v = {0, 0, 0, 0};
    if (whole) {
        if (c < cols) v = ONCE ? ld16_stream(row + c) : ld16(row + c);
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

// Rows that one launch takes: a launch has less than 2^32 threads.
constexpr int64_t kLaunchRows = (int64_t)1 << 23;

// 16 lanes a block, 8 neighbouring elements each; a workgroup has 1 << wide blocks of 16 >> wide rows at a time, kSteps
// times, all of them requested at first. Large matrices go faster by longer runs of a row, small ones by rows whose scales
// lie side by side: SwiGLU with wide 4 / 2, us: 4096 x 14336 56.1 / 60.6, 8192 x 4096 33.2 / 34.9, 4096 x 5632 25.5 / 25.0,
// 65536 x 256 31.3 / 28.2. Rows of 2048 x 4096 are quantized in 8.9 us, 2.7 of them the stores, the rest a wave's latency
// (1 step 8.9, 4 steps 9.8).
constexpr int kSteps = 2;
struct Unit {
    int64_t row, block;
    int step;  // rows between a thread's steps
};
__device__ __forceinline__ Unit unit_of(int64_t first, int wide) {
    const int g = threadIdx.x / 16, step = 16 >> wide;
    return {first + (int64_t)blockIdx.x * (step * kSteps) + (g >> wide), ((int64_t)blockIdx.y << wide) + (g & ((1 << wide) - 1)), step};
}
static int unit_wide(int64_t rows, int64_t nb) { return nb >= 16 && rows * nb >= 1 << 18 ? 4 : 2; }
static dim3 unit_grid(int64_t rows, int64_t nb, int wide) {
    const int64_t step = (16 >> wide) * kSteps;
    return dim3((unsigned)((rows + step - 1) / step), (unsigned)((nb + (1 << wide) - 1) >> wide));
}

__global__ __launch_bounds__(256) void fp8_quantize_kernel(const h16 *__restrict__ x, int64_t stride, int64_t first, int64_t rows,
                                                           int64_t cols, int wide, bool whole, uint8_t *__restrict__ q, float *__restrict__ scales) {
    const Unit u8 = unit_of(first, wide);
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block, r0 = u8.row, b = u8.block, c = b * kFp8Block + 8 * (threadIdx.x % 16);
    if (b >= nb) return;
    u32x4 v[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        v[i] = {0, 0, 0, 0};
        if (r0 + u8.step * i < rows) v[i] = load8(x + (r0 + u8.step * i) * stride, c, cols, whole);
    }
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int64_t r = r0 + u8.step * i;
        if (r >= rows) return;
        float p[8];
        unpack8(v[i], p);
        const unsigned top = row_max(top_bits(v[i]));
        *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = codes_of(p, top);
        if (threadIdx.x % 16 == 0)
            scales[b * rows + r] = top >= kInfBits ? __builtin_nanf("") : __builtin_bit_cast(float, top) / kE4m3Max;
    }
}

// A workgroup per 128 x 128 block, its 16384 elements in registers between the maximum and the codes, so memory sees
// each once: 28672 x 4096 in 70 us, 5.0 TB/s, as fast as a copy.
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
    for (int i = 0; i < 8; i++) top = max(top, top_bits(v[i]));
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
    const int64_t nb = fp8_blocks(cols);
    if (weight) {
        const int64_t groups = (rows + 127) / 128 * nb;
        if (groups >= 1 << 24) return fail(AESIR_ERR_UNSUPPORTED, "quantize_fp8: more elements than one launch takes");
        hipLaunchKernelGGL(fp8_quantize_weight_kernel, dim3((unsigned)groups), dim3(256), 0, s, (const h16 *)x, stride, rows, cols, whole,
                           (uint8_t *)q, scales);
        AESIR_LAUNCH_CHECK("fp8_quantize_weight_kernel");
        return AESIR_OK;
    }
    const int wide = unit_wide(rows, nb);
    for (int64_t first = 0; first < rows; first += kLaunchRows) {
        hipLaunchKernelGGL(fp8_quantize_kernel, unit_grid(std::min(rows - first, kLaunchRows), nb, wide), dim3(256), 0, s, (const h16 *)x, stride,
                           first, rows, cols, wide, whole, (uint8_t *)q, scales);
        AESIR_LAUNCH_CHECK("fp8_quantize_kernel");
    }
    return AESIR_OK;
}

// ------------------------------------------------------------------ RMSNorm

// A workgroup per row. h = f16(x + residual), y = h w / sqrt(mean h^2 + eps): the row's factor changes no code, so the
// codes are those of h w, exact in f32, and the factor goes into the scales. A row with an inf or NaN is NaN whole.
// V: groups of 2048 columns, which stay in registers; 0: any number of them, read twice. 8192 x 4096 with a residual in
// 44 us, 5.3 TB/s, as fast as a copy; one row of 2048 in 2.2 us, all latency.
template <int V>
__global__ __launch_bounds__(256) void fp8_norm_kernel(const h16 *x, int64_t x_stride, const h16 *residual, int64_t res_stride, h16 *sum,
                                                       int64_t sum_stride, const h16 *__restrict__ w, float eps, int64_t first,
                                                       int64_t rows, int64_t cols, bool whole, bool w_whole, uint8_t *__restrict__ q,
                                                       float *__restrict__ scales) {
    __shared__ float red[4];
    const int64_t r = first + blockIdx.x, nb = (cols + kFp8Block - 1) / kFp8Block;
    const h16 *xr = x + r * x_stride, *rr = residual + r * res_stride;
    h16 *sr = sum + r * sum_stride;
    float ss = 0.0f;
    auto add = [&](u32x4 v, u32x4 d, int64_t c) {
        float h[8];
        if (residual) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const h16x2 a = as_h2(v[j]), b = as_h2(d[j]);
                v[j] = h2_bits(h16x2{hadd(a.x, b.x), hadd(a.y, b.y)});
            }
            store8(sr, c, cols, whole, v);
        }
        unpack8(v, h);
#pragma unroll
        for (int j = 0; j < 8; j++) ss = fmaf(h[j], h[j], ss);
        return v;
    };
    float factor = 0.0f;
    auto finish = [&](u32x4 v, u32x4 g8, int64_t c) {
        float p[8], g[8];
        unpack8(v, p);
        unpack8(g8, g);
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] *= g[j];
        unsigned top = row_max(top_bits(p));
        if (!(ss < __builtin_inff())) top = kInfBits;
        *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = codes_of(p, top);
        if (threadIdx.x % 16 == 0)
            scales[c / kFp8Block * rows + r] = top >= kInfBits ? __builtin_nanf("") : __builtin_bit_cast(float, top) * factor / kE4m3Max;
    };
    const u32x4 none = {0, 0, 0, 0};
    if constexpr (V > 0) {
        u32x4 v[V], d[V], g[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int64_t c = 8 * threadIdx.x + 2048 * i;
            v[i] = load8(xr, c, cols, whole);
            d[i] = residual ? load8(rr, c, cols, whole) : none;
            g[i] = load8<false>(w, c, cols, w_whole);
        }
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = add(v[i], d[i], 8 * threadIdx.x + 2048 * i);
        ss = block_sum<4, false>(ss, red);
        factor = 1.0f / sqrtf(ss / (float)cols + eps);
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int64_t c = 8 * threadIdx.x + 2048 * i;
            if (c < nb * kFp8Block) finish(v[i], g[i], c);
        }
    } else {
        for (int64_t c = 8 * threadIdx.x; c < nb * kFp8Block; c += 2048)
            add(load8<false>(xr, c, cols, whole), residual ? load8(rr, c, cols, whole) : none, c);
        ss = block_sum<4, false>(ss, red);
        factor = 1.0f / sqrtf(ss / (float)cols + eps);
        for (int64_t c = 8 * threadIdx.x; c < nb * kFp8Block; c += 2048)
            finish(load8<false>(residual ? sr : xr, c, cols, whole), load8<false>(w, c, cols, w_whole), c);
    }
}

int32_t launch_rmsnorm_fp8(hipStream_t s, const void *x, int64_t x_stride, const void *residual, int64_t res_stride, void *sum,
                           int64_t sum_stride, const void *w, float eps, int64_t rows, int64_t cols, void *q, float *scales) {
    const bool whole = whole_rows(cols, x_stride, x) && (!residual || (whole_rows(cols, res_stride, residual) && whole_rows(cols, sum_stride, sum)));
    const auto kernel = cols <= 2048 ? fp8_norm_kernel<1> : cols <= 4096 ? fp8_norm_kernel<2> : cols <= 8192 ? fp8_norm_kernel<4> : fp8_norm_kernel<0>;
    for (int64_t first = 0; first < rows; first += kLaunchRows) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(rows - first, kLaunchRows)), dim3(256), 0, s, (const h16 *)x, x_stride,
                           (const h16 *)residual, res_stride, (h16 *)sum, sum_stride, (const h16 *)w, eps, first, rows, cols, whole,
                           whole_rows(cols, 8, w), (uint8_t *)q, scales);
        AESIR_LAUNCH_CHECK("fp8_norm_kernel");
    }
    return AESIR_OK;
}

// ------------------------------------------------------------------ SwiGLU

// y = u g / (1 + exp(-g)), off by at most 7 * 2^-24 of it: u g is exact, the exponential is 2^hi (1 + lo ln 2) with
// hi + lo = -g log2(e) (the instruction's 2^-23, a product's 2^-24), the sum 2^-24, its reciprocal 2^-23 and the product
// 2^-24.
__device__ __forceinline__ float swiglu_f(float g, float u) {
    const float hi = g * -1.44269504088896341f;
    const float lo = fmaf(g, -1.92596299112661746e-8f, fmaf(g, -1.44269504088896341f, -hi));
    const float d = fmaf(__builtin_amdgcn_exp2f(hi), fmaf(lo, 0.693147180559945309f, 1.0f), 1.0f);
    return u * g * __builtin_amdgcn_rcpf(d);
}
__device__ __forceinline__ double swiglu_d(float g, float u) { return (double)u * (double)g / (1.0 + exp(-(double)g)); }

constexpr float kSwigluLeast = 0x1p-64f;  // a block of smaller values is zeros

// Lanes as in fp8_quantize_kernel. 448 y / a is off by at most 7 + 7 + 4 times 2^-24 of it (y, a, the reciprocal and two
// products), less than 2^-19. Where a code or the maximum is in doubt the
// block's 16 lanes find all its values in f64, so a row's codes and scales do not depend on the rows beside it.
// 4096 x 14336 in 56 us, 5.3 TB/s; a copy of as many bytes takes 58.
__global__ __launch_bounds__(256) void fp8_swiglu_kernel(const h16 *__restrict__ gate, int64_t g_stride, const h16 *__restrict__ up,
                                                         int64_t u_stride, int64_t first, int64_t rows, int64_t cols, int wide, bool whole,
                                                         uint8_t *__restrict__ q, float *__restrict__ scales) {
    const Unit u8 = unit_of(first, wide);
    const int64_t nb = (cols + kFp8Block - 1) / kFp8Block, r0 = u8.row, b = u8.block, c = b * kFp8Block + 8 * (threadIdx.x % 16);
    if (b >= nb) return;
    u32x4 gv[kSteps], uv[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        gv[i] = uv[i] = {0, 0, 0, 0};
        if (r0 + u8.step * i < rows) {
            gv[i] = load8(gate + (r0 + u8.step * i) * g_stride, c, cols, whole);
            uv[i] = load8(up + (r0 + u8.step * i) * u_stride, c, cols, whole);
        }
    }
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
        const int64_t r = r0 + u8.step * i;
        if (r >= rows) return;
        float g[8], u[8], y[8];
        unpack8(gv[i], g);
        unpack8(uv[i], u);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = swiglu_f(g[j], u[j]);
        const unsigned top = row_max(top_bits(y));
        const float a = __builtin_bit_cast(float, top);
        const bool some = a >= kSwigluLeast;
        float scale = some ? a / kE4m3Max : 0.0f;
        const float inv = some ? __builtin_amdgcn_rcpf(a) : 0.0f;
        const float less = inv * (kE4m3Max * (1.0f - 0x1p-19f)), more = inv * (kE4m3Max * (1.0f + 0x1p-19f));
        float lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            lo[j] = y[j] * less;
            hi[j] = y[j] * more;
        }
        u32x2 codes = to_e4m3(lo);
        const u32x2 d = to_e4m3(hi);
        const bool bad = top >= kInfBits;
        const bool doubt = ((codes.x ^ d.x) | (codes.y ^ d.y)) != 0 || fabsf(a - kSwigluLeast) <= 0x1p-83f;
        if (bad) {
            codes = kNanCodes;
        } else if (row_max(doubt)) {
            double yd[8], m = 0.0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                yd[j] = swiglu_d(g[j], u[j]);
                m = fmax(m, fabs(yd[j]));
            }
#pragma unroll
            for (int k = 1; k < 16; k <<= 1) m = fmax(m, __shfl_xor(m, k));
            const bool some_d = m >= (double)kSwigluLeast;
            scale = some_d ? (float)(m / 448.0) : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) lo[j] = some_d ? to_odd(yd[j] * 448.0 / m) : 0.0f;
            codes = to_e4m3(lo);
        } else if (!some) {
            codes = {0, 0};  // of values of either sign
        }
        *reinterpret_cast<u32x2 *>(q + r * nb * kFp8Block + c) = codes;
        if (threadIdx.x % 16 == 0) scales[b * rows + r] = bad ? __builtin_nanf("") : scale;
    }
}

int32_t launch_swiglu_fp8(hipStream_t s, const void *gate, int64_t g_stride, const void *up, int64_t u_stride, int64_t rows,
                          int64_t cols, void *q, float *scales) {
    const bool whole = whole_rows(cols, g_stride, gate) && whole_rows(cols, u_stride, up);
    const int64_t nb = fp8_blocks(cols);
    const int wide = unit_wide(rows, nb);
    for (int64_t first = 0; first < rows; first += kLaunchRows) {
        hipLaunchKernelGGL(fp8_swiglu_kernel, unit_grid(std::min(rows - first, kLaunchRows), nb, wide), dim3(256), 0, s, (const h16 *)gate, g_stride,
                           (const h16 *)up, u_stride, first, rows, cols, wide, whole, (uint8_t *)q, scales);
        AESIR_LAUNCH_CHECK("fp8_swiglu_kernel");
    }
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
// 2^-13 of the power of two at the largest (measured: both 16x16x128 and 16x16x32). By the norm of a matrix that is 1.3e-5 of
// near normal products and 2e-5 to 3e-5 where channels differ much in size, beside f16's rounding of 2.1e-4: f16 results are
// 2.08e-4 to 2.10e-4 off f64, those of f32 sums 2.07e-4. But it goes by the size of the products, not of their sum: one result in 12
// is more than half an f16 step off, one in 50 more than a step, sums that all but cancel many steps (64 x 4096 x 14336 to
// 5207 x 744 x 128, channels as above); of results over a quarter of the root mean square one in 35 is more than half a step off,
// none more than 3. That is the choice for f16 results of many rows, which it makes up to twice as fast (8192 x 28672 x 4096 830 us,
// to f32 1631); f32 results and products of few rows, which wait for memory anyway, take the f16 instruction, whose sums are
// f32, on the numbers converted, at half the rate.
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
    int nb;     // blocks along k
    int splits; // workgroups that share a tile of C, each with a stretch of the blocks along k
    float *part;  // their sums [splits][M][N] where there are more than one
    bool f32;   // type of c
    bool quad;  // whether rows of c are 16-byte aligned
};

__device__ __forceinline__ void fp8_store(const Fp8Args &p, int64_t m, int64_t n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
    const int64_t at = m * p.ldc + n;
    if (p.quad && n + 3 < p.N) {
        if (p.f32)
            *(f32x4 *)((float *)p.c + at) = v;
        else
            *(u32x2 *)((h16 *)p.c + at) = u32x2{h2_bits(h16x2{(h16)v[0], (h16)v[1]}), h2_bits(h16x2{(h16)v[2], (h16)v[3]})};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (n + e >= p.N) return;
        if (p.f32)
            ((float *)p.c)[at + e] = v[e];
        else
            ((h16 *)p.c)[at + e] = (h16)v[e];
    }
}

constexpr int kPastBuffers = 0x70000000;  // an offset behind every buffer here, with room for a tile's rows

#define FP8_LDS(p) ((__attribute__((address_space(3))) void *)(p))

// A copy instruction fills 1 KiB of LDS, 8 rows of 128 bytes: lane l brings slot l % 8 of row l / 8, which holds granule
// (l % 8) ^ (row / 2 % 8) of the row's k-block, so that the 16 rows that a fragment reads at once lie in different banks.
// The lane's offset from the first of the 8 rows, rows `ld` bytes apart; odd: whether they are rows 8 .. 15 of 16.
__device__ __forceinline__ int copy_offset(int lane, int ld, bool odd) {
    return lane / 8 * ld + ((lane & 7) ^ ((lane >> 4) + (odd ? 4 : 0))) * 16;
}

// Lane's fragment of the 16 rows at `rows`, from LDS.
template <bool EXACT>
__device__ __forceinline__ auto read_frag(const uint8_t *rows, int at) {
    const Frag8 f{ld16(rows + at), ld16(rows + (at ^ 64))};
    if constexpr (EXACT)
        return to_f16(f);
    else
        return f;
}

// Few rows of A: every weight is used by all of them as it arrives. A workgroup owns 16 NR rows of B; its W waves take
// the k-blocks in turn, each through a ring of S stages of its own in LDS (no barriers), and their sums meet in a fixed
// order. MH: rows of A in eights.
//
// The copies bring whole lines, 8 rows of 128 bytes an instruction; fragments loaded straight to registers, 16 rows of
// 64 bytes, cost the address unit 50 cycles each (1 x 28672 x 4096 23.6 us against 20.7). A stage is read no earlier than
// its copies are counted down, and a fragment read in one turn feeds a product of that turn, so it is in registers when
// the next turn gives its stage away. Measured: 1 x 6144 x 4096 in 6.4 us, 1 x 57344 x 8192 in 68 (6.9 TB/s), 16 x 32000 x
// 2048 to f32 in 12.1; memory's rate and 3 to 4 us of starting and ending bound it.
template <int MH, int NR, int W, int S, bool EXACT>
__global__ __launch_bounds__(64 * W) void fp8_stream_kernel(Fp8Args p) {
    constexpr int MT = (MH + 1) / 2, kA = NR * 2048, kScales = kA + MH * 1024, kStage = kScales + 512, kLoads = 2 * NR + MH + 2;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NR);
    const int ld = p.nb * 128, M = (int)p.M;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void *)p.a, 0, M * ld, kBufferDword3);
    const __amdgpu_buffer_rsrc_t rb =
        __builtin_amdgcn_make_buffer_rsrc((void *)(p.b + n0 * ld), 0, (int)min((int64_t)16 * NR, p.N - n0) * ld, kBufferDword3);
    const __amdgpu_buffer_rsrc_t rsa = __builtin_amdgcn_make_buffer_rsrc((void *)p.as, 0, p.nb * M * 4, kBufferDword3);
    const __amdgpu_buffer_rsrc_t rsb = __builtin_amdgcn_make_buffer_rsrc((void *)(p.bs + n0 / 128 * p.nb), 0, p.nb * 4, kBufferDword3);
    uint8_t *ring = lds + wave * (S * kStage);
    const int even = copy_offset(lane, ld, false), odd = copy_offset(lane, ld, true);
    // blocks past the last: addresses past the buffers, which read as zeros, so that every stage has as many copies
    auto request = [&](int stage, int kb) {
        uint8_t *to = ring + stage * kStage;
        const int k = kb < p.nb ? kb * 128 : kPastBuffers;
#pragma unroll
        for (int i = 0; i < 2 * NR; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, FP8_LDS(to + i * 1024), 16, (i & 1 ? odd : even) + i * 8 * ld + k, 0, 0, 2);
#pragma unroll
        for (int i = 0; i < MH; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, FP8_LDS(to + kA + i * 1024), 16, (i & 1 ? odd : even) + i * 8 * ld + k, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsa, FP8_LDS(to + kScales), 4, kb < p.nb ? kb * M * 4 + lane * 4 : kPastBuffers, 0, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsb, FP8_LDS(to + kScales + 256), 4, kb < p.nb ? kb * 4 : kPastBuffers, 0, 0, 0);
    };
    const int at = i16 * 128 + ((lane >> 4) ^ (i16 >> 1)) * 16;
    f32x4 acc[NR][MT] = {};
#pragma unroll
    for (int i = 0; i < S - 1; i++) request(i, wave + i * W);
    int stage = 0;
    for (int kb = wave; kb < p.nb; kb += W) {
        request(stage == 0 ? S - 1 : stage - 1, kb + (S - 1) * W);
        __builtin_amdgcn_s_waitcnt(vm_wait((S - 1) * kLoads));
        const uint8_t *from = ring + stage * kStage;
        const float sb = *(const float *)(from + kScales + 256);
        decltype(read_frag<EXACT>(from, at)) b[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) b[i] = read_frag<EXACT>(from + i * 2048, at);
#pragma unroll
        for (int j = 0; j < MT; j++) {
            const float s = *(const float *)(from + kScales + (16 * j + i16) * 4) * sb;
            const auto a = read_frag<EXACT>(from + kA + j * 2048, at);
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const f32x4 d = mma_block(b[i], a);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] = fmaf(d[e], s, acc[i][j][e]);
            }
        }
        stage = stage == S - 1 ? 0 : stage + 1;
    }
    __builtin_amdgcn_s_waitcnt(vm_wait(0));
    __syncthreads();
    f32x4 *part = (f32x4 *)lds;
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) part[(wave * NR * MT + i * MT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    for (int t = wave; t < NR * MT; t += W) {
        f32x4 v = part[t * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; w++) v += part[(w * NR * MT + t) * 64 + lane];
        fp8_store(p, 16 * (t % MT) + i16, n0 + 16 * (t / MT) + 4 * (lane >> 4), v);
    }
}

// Barrier of the workgroup's waves that neither the compiler's memory operations nor its schedule cross.
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// A wave's sums to C, T's rows from (m, n) on, 16 rows at a time through a place of the wave's own in LDS, so that a
// store fills whole lines. WHOLE: all columns are C's and rows are 16-byte aligned; else element by element. Stores
// straight from the registers cost 8192 x 28672 x 4096 another 110 us, and odd rows of 2756 x 3338 x 232 27.9 us for 17.7.
template <bool WHOLE, typename T, int NF, int MF>
__device__ __forceinline__ void store_rows(const Fp8Args &p, T *c, uint8_t *lds, const f32x4 (&acc)[NF][MF], int64_t m, int64_t n, int wave,
                                           int lane) {
    constexpr int kCols = NF * 16, kStride = kCols * sizeof(T) + 16, kEach = WHOLE ? 16 / sizeof(T) : 1;
    constexpr int kLanes = kCols / kEach < 64 ? kCols / kEach : 64, kRows = 64 / kLanes;
    static_assert(16 % kRows == 0);
    uint8_t *own = lds + wave * 16 * kStride;
#pragma unroll
    for (int j = 0; j < MF; j++) {
#pragma unroll
        for (int i = 0; i < NF; i++) {
            uint8_t *to = own + (lane & 15) * kStride + (16 * i + 4 * (lane >> 4)) * sizeof(T);
            const f32x4 v = acc[i][j];
            if constexpr (sizeof(T) == 4)
                *(f32x4 *)to = v;
            else
                *(u32x2 *)to = u32x2{h2_bits(h16x2{(h16)v[0], (h16)v[1]}), h2_bits(h16x2{(h16)v[2], (h16)v[3]})};
        }
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += kRows) {
            const int r = r0 + lane / kLanes;
            T *row = c + (m + 16 * j + r) * p.ldc + n;
#pragma unroll
            for (int e = 0; e < kCols; e += kLanes * kEach) {
                const int col = e + lane % kLanes * kEach;
                const uint8_t *from = own + r * kStride + col * sizeof(T);
                if constexpr (WHOLE) {
                    if (m + 16 * j + r < p.M) st16(row + col, ld16(from));
                } else {
                    if (m + 16 * j + r < p.M && n + col < p.N) row[col] = *(const T *)from;
                }
            }
        }
    }
}

// Tile of BM rows of A by BN of B on WM x WN waves, through a ring of S stages of one k-block in LDS. Weights are the
// first operand of the matrix instruction, so a lane's elements are 4 neighbouring columns of one row of C. Per k-block a
// product of fragments starts from 0 and is added to the sums with the block's scale, 4 multiply-adds beside the 32
// cycles of a matrix instruction. ONCE: every row of B is used by one workgroup only and need not stay in the caches.
//
// Measured: 8192 x 28672 x 4096 in 820 to 890 us by the card (2.2 to 2.3 PFLOP/s), 64 x 4096 x 14336 in 17.8 (with the join below), 333 x
// 11264 x 2048 in 15.5. Of the first, matrix and vector instructions alone take 584 us at the clock they leave; reading
// fragments 90 more, since a step begins with reads that nothing covers (LDS gives 205 bytes a cycle, without
// conflicts); the copies 150, whose 64 KiB a step make a round trip of 1.5 to 1.8 us through L2, as long as a step. Tried
// and slower: two groups of waves half a step apart with all fragments in registers (985), the next step's first
// fragments read during this one's last products (256 x 256 spills, 192 x 192 with three stages 1016), several
// k-blocks a stage, touching lines in L2 ahead of the copies.
template <int BM, int BN, int WM, int WN, int S, bool EXACT, bool ONCE = false>
__global__ __launch_bounds__(64 * WM * WN) void fp8_tile_kernel(Fp8Args p) {
    constexpr int W = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16, IA = BM / 8 / W, IB = BN / 8 / W;
    constexpr int kB = BM * 128, kScales = kB + BN * 128, kStage = kScales + (BM + 64) * 4, kLoads = IA + IB + 1;
    static_assert(BM / 8 % W == 0 && BN / 8 % W == 0 && BM / 64 < W && BM % 64 == 0 && 128 % (BN / WN) == 0);
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15;
    // each XCD (workgroups go to the 8 in turn) takes a stretch of the tiles, which run through bands of 8 rows of
    // tiles of C, column by column, so that the tiles it works on at a time share rows of A and B in its L2
    const unsigned mt = (unsigned)((p.M + BM - 1) / BM), nt = (unsigned)((p.N + BN - 1) / BN), all = gridDim.x, xcd = blockIdx.x % 8;
    const unsigned place = blockIdx.x / 8 + xcd * (all / 8) + min(xcd, all % 8), split = place / (mt * nt), tile = place - split * mt * nt;
    const unsigned band = tile / (8 * nt), in_band = tile - band * 8 * nt, high = min(8u, mt - 8 * band);
    const int64_t m0 = (int64_t)(8 * band + in_band % high) * BM, n0 = (int64_t)(in_band / high) * BN;
    const int ld = p.nb * 128;
    const int rows_a = (int)min((int64_t)BM, p.M - m0), rows_b = (int)min((int64_t)BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void *)(p.a + m0 * ld), 0, rows_a * ld, kBufferDword3);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void *)(p.b + n0 * ld), 0, rows_b * ld, kBufferDword3);
    // scales: waves 0 .. BM / 64 - 1 bring those of 64 rows of A each, the others those of the tile's rows of B
    const bool sa = wave < BM / 64;
    const int nblocks = (rows_b + 127) / 128;
    const float *bs = p.bs + n0 / 128 * p.nb;
    const int scales_to = kScales + (sa ? wave : BM / 64) * 256;
    const float *scales = sa ? p.as + m0 : bs;  // of the block requested next
    const int64_t scales_step = sa ? p.M : 1;
    const int scales_bytes = sa ? rows_a * 4 : (nblocks - 1) * p.nb * 4 + 4;
    const int scales_from = sa ? min(wave * 64 + lane, rows_a - 1) * 4 : min(lane, nblocks - 1) * p.nb * 4;
    // A copy instruction fills 1 KiB of LDS, 8 rows of 128 bytes: lane l brings slot l % 8 of row l / 8, which holds
    // granule (l % 8) ^ (row / 2 % 8) of the row's k-block, so that the 16 rows that a fragment reads at once lie in
    // different banks. Rows past the last and blocks past the last are the last ones again, whose products nothing takes.
    int from[IA + IB];
#pragma unroll
    for (int i = 0; i < IA + IB; i++) {
        const int r = (i < IA ? wave * IA + i : wave * IB + i - IA) * 8 + lane / 8;
        from[i] = min(r, (i < IA ? rows_a : rows_b) - 1) * ld + ((lane & 7) ^ (r >> 1 & 7)) * 16;
    }
    const int k0 = (int)((int64_t)p.nb * split / p.splits), k1 = (int)((int64_t)p.nb * (split + 1) / p.splits);
    scales += k0 * scales_step;
    auto request = [&](int stage, int kb) {
        uint8_t *to = lds + stage * kStage;
        const int k = min(kb, k1 - 1) * 128;
#pragma unroll
        for (int i = 0; i < IA; i++) {
            const int at = from[i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, FP8_LDS(to + (wave * IA + i) * 1024), 16, at, k, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < IB; i++) {
            const int at = from[IA + i];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, FP8_LDS(to + kB + (wave * IB + i) * 1024), 16, at, k, 0, ONCE ? 2 : 0);
        }
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)scales, 0, scales_bytes, kBufferDword3);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, FP8_LDS(to + scales_to), 4, scales_from, 0, 0, 0);
        if (kb + 1 < k1) scales += scales_step;
    };
    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    const int at = i16 * 128 + ((lane >> 4) ^ (i16 >> 1)) * 16;
    using Frag = decltype(read_frag<EXACT>(lds, at));
    f32x4 acc[NF][MF] = {};
#pragma unroll
    for (int i = 0; i < S - 1; i++) request(i, k0 + i);
    int stage = 0;
    for (int kb = k0; kb < k1; kb++) {
        __builtin_amdgcn_s_waitcnt(vm_wait((S - 2) * kLoads));
        barrier();
        request(stage == 0 ? S - 1 : stage - 1, kb + S - 1);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t *la = lds + stage * kStage + wm * 128, *lb = lds + stage * kStage + kB + wn * 128;
        const float *sc = (const float *)(lds + stage * kStage + kScales);
        const float sb = sc[BM + wn / 128];
        Frag a[MF], b[3];
        float s[MF];
        b[0] = read_frag<EXACT>(lb, at);
#pragma unroll
        for (int j = 0; j < MF; j++) {
            a[j] = read_frag<EXACT>(la + 2048 * j, at);
            s[j] = sc[wm + 16 * j + i16] * sb;
            if (j == 0) b[1] = read_frag<EXACT>(lb + 2048, at);
        }
        // a product is added to its sum when the two after it have been issued; a row of B's fragment is read two rows ahead
        constexpr int D = 3, kBehind = 2;
        f32x4 d[D];
#pragma unroll
        for (int t = 0; t < MF * NF + kBehind; t++) {
            const int i = t / MF;
            if (t % MF == 0 && i + 2 < NF) b[(i + 2) % 3] = read_frag<EXACT>(lb + 2048 * (i + 2), at);
            if (t < MF * NF) d[t % D] = mma_block(b[i % 3], a[t % MF]);
            __builtin_amdgcn_sched_barrier(0);
            if (t >= kBehind) {
                const int u = t - kBehind;
#pragma unroll
                for (int e = 0; e < 4; e++) acc[u / MF][u % MF][e] = fmaf(d[u % D][e], s[u % MF], acc[u / MF][u % MF][e]);
                asm volatile("" : "+v"(acc[u / MF][u % MF]));  // here: the compiler would put all of them off to the end
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        stage = stage == S - 1 ? 0 : stage + 1;
    }
    __builtin_amdgcn_s_waitcnt(vm_wait(0));
    if (p.splits > 1) {  // sums of a stretch of k: f32 rows of N elements
        p.c = p.part + split * p.M * p.N;
        p.ldc = p.N;
        p.f32 = true;
        p.quad = p.N % 4 == 0;
    }
    barrier();  // no wave reads a stage any more
    const bool whole = p.quad && n0 + BN <= p.N;
    if (p.f32) {
        if (whole)
            store_rows<true>(p, (float *)p.c, lds, acc, m0 + wm, n0 + wn, wave, lane);
        else
            store_rows<false>(p, (float *)p.c, lds, acc, m0 + wm, n0 + wn, wave, lane);
    } else {
        if (whole)
            store_rows<true>(p, (h16 *)p.c, lds, acc, m0 + wm, n0 + wn, wave, lane);
        else
            store_rows<false>(p, (h16 *)p.c, lds, acc, m0 + wm, n0 + wn, wave, lane);
    }
}

// C from the sums of `splits` stretches of k, in their order; fewer than 2^31 elements. VEC: 4 a thread, N a multiple of 4.
// 4 x 64 x 4096 sums in 2.6 to 3.9 us, mostly the launch.
template <bool VEC>
__global__ __launch_bounds__(256) void fp8_join_kernel(Fp8Args p) {
    const unsigned e = (blockIdx.x * 256 + threadIdx.x) * (VEC ? 4 : 1), all = (unsigned)(p.M * p.N), N = (unsigned)p.N;
    if (e >= all) return;
    if constexpr (VEC) {
        f32x4 v = *(const f32x4 *)(p.part + e);
        for (int z = 1; z < p.splits; z++) v += *(const f32x4 *)(p.part + (int64_t)z * all + e);
        fp8_store(p, e / N, e % N, v);
    } else {
        float v = p.part[e];
        for (int z = 1; z < p.splits; z++) v += p.part[(int64_t)z * all + e];
        const int64_t at = e / N * p.ldc + e % N;
        if (p.f32)
            ((float *)p.c)[at] = v;
        else
            ((h16 *)p.c)[at] = (h16)v;
    }
}

template <int MH, int NR, int W, int S, bool EXACT>
static int32_t stream(hipStream_t s, const Fp8Args &p) {
    // an odd MH's last fragment reads 8 rows that are not A's, 512 bytes of them behind the stage
    constexpr int kParts = W * NR * ((MH + 1) / 2) * 1024, kRing = W * S * (NR * 2048 + MH * 1024 + 512) + MH % 2 * 512;
    constexpr int kLds = kParts > kRing ? kParts : kRing;
    static std::atomic<uint64_t> done{0};
    const auto kernel = fp8_stream_kernel<MH, NR, W, S, EXACT>;
    if (kLds > 65536) AESIR_TRY(raise_lds_limit((const void *)kernel, kLds, done));
    hipLaunchKernelGGL(kernel, dim3((unsigned)((p.N + 16 * NR - 1) / (16 * NR))), dim3(64 * W), kLds, s, p);
    AESIR_LAUNCH_CHECK("fp8_stream_kernel");
    return AESIR_OK;
}

template <int BM, int BN, int WM, int WN, int S, bool EXACT, bool ONCE = false>
static int32_t tile(hipStream_t s, const Fp8Args &p) {
    constexpr int kLds = S * ((BM + BN) * 128 + (BM + 64) * 4);
    static std::atomic<uint64_t> done{0};
    const auto kernel = fp8_tile_kernel<BM, BN, WM, WN, S, EXACT, ONCE>;
    if (kLds > 65536) AESIR_TRY(raise_lds_limit((const void *)kernel, kLds, done));
    const int64_t tiles = (p.M + BM - 1) / BM * ((p.N + BN - 1) / BN);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * p.splits)), dim3(64 * WM * WN), kLds, s, p);
    AESIR_LAUNCH_CHECK("fp8_tile_kernel");
    if (p.splits > 1) {
        const bool vec = p.N % 4 == 0;
        const unsigned groups = (unsigned)((p.M * p.N / (vec ? 4 : 1) + 255) / 256);
        hipLaunchKernelGGL(vec ? fp8_join_kernel<true> : fp8_join_kernel<false>, dim3(groups), dim3(256), 0, s, p);
        AESIR_LAUNCH_CHECK("fp8_join_kernel");
    }
    return AESIR_OK;
}

// Up to 16 rows of A: memory's rate decides. More rows of B a workgroup (NR) are fewer workgroups and fewer copies of A,
// and pay where B alone fills the 256 CUs; long rows want 8 waves along k. Measured, us of 1 / 16 rows, the taken one first:
//   4096 x 4096   NR 1, 4 waves  5.5 /  5.8, NR 2  6.0 /  6.7
//   4096 x 14336  NR 1, 8 waves 10.9 / 13.2, 4 waves 11.5 / 12.6
//   6144 x 4096   NR 2  6.8 /  7.3, NR 1  7.1 /  8.3
//   8192 x 6144   NR 2  9.4 / 10.0, NR 1  9.6 / 11.4
//   28672 x 2048  NR 2 11.3 / 12.2, NR 4 11.2 / 12.9
//   57344 x 2048  NR 2 19.0 / 20.3, NR 4 20.1 / 24.6
//   28672 x 4096  NR 4 21.2 / 23.8, NR 2 22.7 / 24.2
//   57344 x 4096  NR 4 40.1 / 46.5, NR 2 40.2 / 43.0
//   28672 x 8192  NR 1, 8 waves 36.0 / 42.4, NR 4 39.4 / 43.4
//   57344 x 8192  NR 1, 8 waves 68 / 83, NR 4 82 / 87
// The borders in k lie between those sizes, and not at the best place everywhere: of 2048 to 57344 rows of B by 1024 to 14336, one
// row's time is within 7% of the best one's but for 6144 and 8192 rows of B by 8192 and more (up to 16% behind NR 1, or NR 2 with 14336);
// 16 rows by 6144 and more are up to 26% behind NR 2 or NR 4.
template <int MH>
static int32_t stream_16(hipStream_t s, const Fp8Args &p) {
    if (p.N > 4096) {
        if (p.N <= 8192 && p.nb <= 64) return stream<MH, 2, 4, 3, true>(s, p);
        if (p.N > 8192 && p.nb <= 16) return stream<MH, 2, 4, 2, true>(s, p);
        if (p.N > 8192 && p.nb <= 32) return stream<MH, 4, 4, 2, true>(s, p);
    } else if (p.nb <= 32) {
        return stream<MH, 1, 4, 3, true>(s, p);
    }
    return stream<MH, 1, 8, 2, true>(s, p);
}

// 17 to 64 rows by at most 8192 of B: as above, with 4 waves, since the rows of A take most of a ring's stage. NR 2 pays where B
// has more than 16 rows for each CU, and more of A want fewer stages. Measured at k 4096, us of NR 1 with 2 and 3 stages, then
// of NR 2 with 2 and 3:
//   f16  24 x 4096  6.5  6.3  7.3  7.4    24 x 7168   9.7   9.7   8.2   8.4
//        40 x 4096  7.3  7.4  8.5  8.7    40 x 7168  11.7  12.9   9.4   9.7
//        64 x 4096  8.6  8.8  9.8 10.3    64 x 7168  14.9  15.5  10.7  11.2
//   f32  24 x 4096  6.8  6.3  7.8  7.7    24 x 7168   9.9   9.9   8.5   8.7
//        40 x 4096  8.1  7.9  9.2  9.5    40 x 7168  12.3  14.0   9.9  10.4
//        64 x 4096  8.9  9.4 10.1 10.6    64 x 7168  15.7  16.7  10.9  11.6
template <bool EXACT>
static int32_t stream_64(hipStream_t s, const Fp8Args &p) {
    if (p.N <= 4096)
        return p.M <= 32   ? stream<4, 1, 4, 3, EXACT>(s, p)
               : p.M <= 48 ? stream<6, 1, 4, 2, EXACT>(s, p)
                           : stream<8, 1, 4, 2, EXACT>(s, p);
    return p.M <= 32   ? stream<4, 2, 4, 3, EXACT>(s, p)
           : p.M <= 48 ? stream<6, 2, 4, 3, EXACT>(s, p)
                       : stream<8, 2, 4, 2, EXACT>(s, p);
}

// A tile's shape and how many of its workgroups a CU holds, with what a k-block takes a CU (us) that holds one of them and
// one that is full, as measured on products of 1000 to 4096 rows of 2048 to 28672 columns.
struct TileCost {
    int bm, bn, per_cu;
    float one, full;
};
constexpr TileCost kTiles[] = {{64, 64, 2, 0.28f, 0.38f}, {128, 128, 1, 0.56f, 0.56f}, {192, 128, 1, 0.72f, 0.72f}, {128, 128, 2, 0.8f, 1.07f}, {256, 256, 1, 1.73f, 1.73f}};
constexpr TileCost kExactTiles[] = {{64, 64, 2, 0.43f, 0.66f}, {128, 128, 1, 1.12f, 1.12f}, {128, 128, 2, 1.4f, 1.85f}};

constexpr int64_t kLaunchGroups = (1 << 23) - 1;  // a launch has less than 2^32 threads, a workgroup up to 512

// The tile and the number of stretches of k that the product is cut into (-1: none in one launch), by the time that they come to: rounds of
// workgroups, or what A and B take from memory at 4.5 TB/s where that is more, 4.5 us around each round, and for the
// stretches' sums another launch and their bytes.
template <int N>
static int choose_tile(const TileCost (&tiles)[N], const Fp8Args &p, int64_t part_floats, int *splits) {
    int best = -1;
    float least = std::numeric_limits<float>::infinity();
    *splits = 1;
    for (int i = 0; i < N; i++) {
        const TileCost &c = tiles[i];
        const int64_t count = (p.M + c.bm - 1) / c.bm * ((p.N + c.bn - 1) / c.bn);
        for (int z = 1; z <= 8 && count * z <= kLaunchGroups && (z == 1 || (p.nb >= 4 * z && p.M * p.N <= part_floats / z)); z *= 2) {
            const int64_t all = count * z, rounds = (all + 256 * c.per_cu - 1) / (256 * c.per_cu);
            const float step = all <= 256 ? c.one : c.full, blocks = (float)((p.nb + z - 1) / z);
            const float work = fmaxf((float)rounds * blocks * step, (float)(p.M + p.N) * (float)p.nb * (128 / 4.5e6f));
            const float t = (float)rounds * 4.5f + work + (z > 1 ? 2.2f + (float)(z * p.M * p.N) * 2.5e-6f : 0.0f);
            if (t < least) {
                least = t;
                best = i;
                *splits = z;
            }
        }
    }
    return best;
}

int32_t launch_gemm_fp8(hipStream_t s, const void *A, const float *as, int64_t M, const void *B, const float *bs, int64_t N,
                        int64_t K, void *C, bool f32, int64_t ldc, float *part, int64_t part_floats) {
    const bool quad = ldc % (f32 ? 4 : 8) == 0 && ((uintptr_t)C & 15) == 0;
    Fp8Args p{(const uint8_t *)A, (const uint8_t *)B, as, bs, C, M, N, ldc, (int)fp8_blocks(K), 1, part, f32, quad};
    const auto too_large = [] { return fail(AESIR_ERR_UNSUPPORTED, "gemm_fp8: output larger than one launch takes"); };
    if (M <= 64 && (N + 15) / 16 > kLaunchGroups) return too_large();
    if (M <= 16) return M <= 8 ? stream_16<1>(s, p) : stream_16<2>(s, p);
    if (M <= 64) {
        // Tiles of 64 x 64 share the rows of A among 64 of B. They pay once B alone makes more of them than half the CUs, or, from 33
        // rows on, cut into stretches of long rows. Measured, us streamed and in tiles, f16 then f32:
        //   24 x 8192 x 4096    9.3  13.5   9.6  14.1    64 x 8192 x 4096   11.4  13.7  11.6  15.9
        //   24 x 11264 x 4096  14.9  13.8  15.3  18.9    64 x 11264 x 4096  19.1  14.8  19.6  19.0
        //   24 x 28672 x 4096  30.3  25.6  31.0  29.1    64 x 28672 x 4096  37.9  28.6  39.2  31.5
        //   64 x 4096 x 8192   13.5  13.8  14.2  16.0    64 x 7168 x 8192   18.2  19.1  18.4  22.9
        //   64 x 4096 x 11264  18.4  16.2  19.2  19.4    64 x 7168 x 11264  23.9  23.2  24.3  28.6
        //   64 x 4096 x 14336  22.3  18.2  23.0  22.2    64 x 7168 x 14336  29.3  26.6  29.6  34.3
        //   24 x 4096 x 14336  14.6  16.4  14.7  20.9    40 x 4096 x 14336  18.4  16.9  20.1  21.3
        if (N <= 8192 && (M <= 32 || p.nb < 96)) return f32 ? stream_64<true>(s, p) : stream_64<false>(s, p);
        const TileCost one[1] = {f32 ? kExactTiles[0] : kTiles[0]};
        choose_tile(one, p, part_floats, &p.splits);
        return f32 ? tile<64, 64, 2, 2, 4, true, true>(s, p) : tile<64, 64, 2, 2, 4, false, true>(s, p);
    }
    if (f32) switch (choose_tile(kExactTiles, p, part_floats, &p.splits)) {
        case 0: return tile<64, 64, 2, 2, 4, true>(s, p);
        case 1: return tile<128, 128, 4, 2, 3, true>(s, p);
        case 2: return tile<128, 128, 2, 2, 2, true>(s, p);
        default: return too_large();
    }
    switch (choose_tile(kTiles, p, part_floats, &p.splits)) {
        case 0: return tile<64, 64, 2, 2, 4, false>(s, p);
        case 1: return tile<128, 128, 4, 2, 3, false>(s, p);
        case 2: return tile<192, 128, 4, 2, 3, false>(s, p);
        case 3: return tile<128, 128, 2, 2, 2, false>(s, p);
        case 4: return tile<256, 256, 4, 2, 2, false>(s, p);
        default: return too_large();
    }
}

}  // namespace aesir
