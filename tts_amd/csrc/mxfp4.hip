// Microscaled 4-bit floating point (MXFP4): quantisation, reading back, and the product of two
// MXFP4 operands on the gfx950 matrix cores, plain or over the taps of a 1-D convolution.
//
// Format.  Along the last dimension every 32 elements share one scale 2^s (an E8M0 byte s + 127);
// an element is a 4-bit E2M1 code for one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign.
//     s = max(floor(log2 max|x|) - 2, -127)          (2 = exponent of the largest magnitude, 4..6)
//     code = x / 2^s rounded to the nearest, ties to the even code, 6 beyond 6
// A block with an infinity or a NaN has no such scale: its byte is 255 (NaN) and its codes are 0.
//
// Layout.  A group is 128 columns: 64 bytes of codes (low nibble = even column) and one dword of
// scales.  Rows are padded with zeros to whole groups.
//     codes  [row][group][64]      scales [group][row][4]
// The scales are group-major because a matrix instruction wants, for one group, the scales of 32
// consecutive rows in 32 lanes: that is one 128-byte line here and 32 lines in row order.
#include "lowp.h"
#include "status.h"

using namespace glv;

namespace {

constexpr int kGroup = 128;       // columns of a group
constexpr int kGroupBytes = 64;   // its codes

struct Rows {  // a (batch, rows, cols) array whose last dimension is contiguous
    int64_t batch_stride, row_stride;
    int rows;  // rows of one batch entry
};

__device__ inline int64_t row_offset(const Rows& r, int row) {
    const int b = row / r.rows;
    return b * r.batch_stride + (int64_t)(row - b * r.rows) * r.row_stride;
}

// biased exponent of max|x| as float sees it (255: an infinity or a NaN is among them)
__device__ inline int top_exponent(const Eight<float>& x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __builtin_bit_cast(uint32_t, x.v[i]) & 0x7fffffffu);
    return (int)(m >> 23);
}
__device__ inline int top_exponent(const Eight<bf16>& x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, (uint32_t)(__builtin_bit_cast(uint16_t, x.v[i]) & 0x7fff));
    return (int)(m >> 7);
}
__device__ inline int top_exponent(const Eight<f16>& x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, (uint32_t)(__builtin_bit_cast(uint16_t, x.v[i]) & 0x7fff));
    if (m >= 0x7c00) return 255;
    // every finite half is a normal float, so its exponent there is the true one
    const float f = (float)__builtin_bit_cast(f16, (uint16_t)m);
    return (int)(__builtin_bit_cast(uint32_t, f) >> 23);
}

__device__ inline int scale_byte(int top) { return top == 255 ? 255 : max(top - 2, 0); }

// eight codes; the conversion takes the exponent field of `scale` as the E8M0 byte (0 included)
__device__ inline uint32_t encode(const Eight<float>& x, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.v[0], x.v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.v[2], x.v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.v[4], x.v[5], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x.v[6], x.v[7], scale, 3);
}
__device__ inline uint32_t encode(const Eight<bf16>& x, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{x.v[0], x.v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{x.v[2], x.v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{x.v[4], x.v[5]}, scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, bf16x2{x.v[6], x.v[7]}, scale, 3);
}
__device__ inline uint32_t encode(const Eight<f16>& x, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{x.v[0], x.v[1]}, scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{x.v[2], x.v[3]}, scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{x.v[4], x.v[5]}, scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, f16x2{x.v[6], x.v[7]}, scale, 3);
}

// The eight codes of this lane and its block's scale byte; a block is four neighbouring lanes.
template <typename T>
__device__ inline uint32_t quantise_eight(const Eight<T>& x, int* byte) {
    int top = top_exponent(x);
    top = max(top, __builtin_amdgcn_mov_dpp(top, 0xB1, 0xf, 0xf, true));  // quad_perm 1,0,3,2
    top = max(top, __builtin_amdgcn_mov_dpp(top, 0x4E, 0xf, 0xf, true));  // quad_perm 2,3,0,1
    const int s = scale_byte(top);
    *byte = s;
    return s == 255 ? 0u : encode(x, __builtin_bit_cast(float, (uint32_t)s << 23));
}

// Sixteen lanes a group; a workgroup takes sixteen rows of up to four groups.
template <typename T>
__global__ __launch_bounds__(256) void quantise_kernel(const T* __restrict__ x, Rows xr, int rows, int cols, int groups,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int spans = (groups + 3) / 4;
    const int rb = blockIdx.x / spans, first = (blockIdx.x - rb * spans) * 4;
    const int row = rb * 16 + (threadIdx.x >> 4);
    const int piece = threadIdx.x & 15;
    if (row >= rows) return;
    const T* src = x + row_offset(xr, row);
    for (int g = first; g < min(groups, first + 4); ++g) {
        const int col = g * kGroup + piece * 8;
        int byte;
        const uint32_t c = quantise_eight(load_eight(src + col, cols - col), &byte);
        reinterpret_cast<uint32_t*>(codes)[((int64_t)row * groups + g) * 16 + piece] = c;
        if ((piece & 3) == 0) scales[((int64_t)g * rows + row) * 4 + (piece >> 2)] = (uint8_t)byte;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void dequantise_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int rows, int cols,
                                                         int groups, T* __restrict__ out) {
    const int spans = (groups + 3) / 4;
    const int rb = blockIdx.x / spans, first = (blockIdx.x - rb * spans) * 4;
    const int row = rb * 16 + (threadIdx.x >> 4);
    const int piece = threadIdx.x & 15;
    if (row >= rows) return;
    for (int g = first; g < min(groups, first + 4); ++g) {
        const int col = g * kGroup + piece * 8;
        if (col >= cols) return;
        const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[((int64_t)row * groups + g) * 16 + piece];
        const uint32_t s = scales[((int64_t)g * rows + row) * 4 + (piece >> 2)];
        // 2^-127 is a subnormal float, 255 a NaN; the codes' own values come out of the conversion
        // exactly, and the product of the two is exact wherever T can hold it
        const float scale = __builtin_bit_cast(float, s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
        const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3)};
        Eight<T> r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = (T)(v[i >> 1][i & 1] * scale);
        store_eight(out + (int64_t)row * cols + col, r, cols - col);
    }
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
struct Product {
    const uint8_t *xc, *xs;  // quantised activations: rows = batch * T
    const uint8_t *wc, *ws;  // weights: n * taps rows of `groups` groups
    const void* bias;
    void* y;
    int rows, T, n;
    int taps, dilation, left;  // tap j of row t reads row t + j * dilation - left of its batch entry
    int groups;                // groups of one tap
    int bias_type, y_type, relu;
};

__device__ inline float load_float(const void* p, int type, int64_t i) {
    if (type == GLV_F32) return static_cast<const float*>(p)[i];
    if (type == GLV_BF16) return (float)static_cast<const bf16*>(p)[i];
    return (float)static_cast<const f16*>(p)[i];
}
__device__ inline void store_float(void* p, int type, int64_t i, float v) {
    if (type == GLV_F32)
        static_cast<float*>(p)[i] = v;
    else if (type == GLV_BF16)
        static_cast<bf16*>(p)[i] = (bf16)v;  // to nearest, ties to even, as every other store here
    else
        static_cast<f16*>(p)[i] = (f16)v;
}

// max(v, 0) that keeps a NaN
__device__ inline float relu(float v) { return v < 0.f ? 0.f : v; }

__device__ inline i32x8 widen(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// acc += W (32 rows) * X (32 rows)^T over the 64 columns of step S: lane l holds row l % 32 and, of
// the two groups of a step, group l / 32: its 32 columns of block S.  Which columns meet in one
// instruction is free as long as both operands agree, so a lane takes the four blocks of its own
// group in the four steps, and one scale dword serves them all.
template <int S>
__device__ inline f32x16 step(i32x4 w, i32x4 x, int wscale, int xscale, f32x16 acc) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(w), widen(x), acc, 4, 4, S, wscale, S, xscale);
}

// One 32 x 32 tile of y a workgroup; the waves deal the groups out among themselves two at a time
// (one for each half of the lanes) and their sums meet in LDS in a fixed order.
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void product_direct_kernel(Product p) {
    __shared__ float sums[WAVES][32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, half = lane >> 5;
    const int n_tiles = (p.n + 31) / 32;
    const int m_tile = blockIdx.x / n_tiles;
    const int n0 = (blockIdx.x - m_tile * n_tiles) * 32, m0 = m_tile * 32;
    const int n = min(n0 + r, p.n - 1), m = min(m0 + r, p.rows - 1);  // rows beyond the ends: computed, not stored
    const int t = m % p.T;
    const int all = p.taps * p.groups;
    f32x16 acc = {};
    for (int g0 = wave * 2; g0 < all; g0 += WAVES * 2) {
        const int g = g0 + half;
        const int tap = g / p.groups, gx = g - tap * p.groups;
        const int shift = tap * p.dilation - p.left;
        const bool have = g < all && t + shift >= 0 && t + shift < p.T;
        i32x4 w[4] = {}, x[4] = {};
        int wscale = 0, xscale = 0;
        if (g < all) {
            const i32x4* wp = reinterpret_cast<const i32x4*>(p.wc + ((int64_t)n * all + g) * kGroupBytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = wp[i];
            wscale = reinterpret_cast<const int*>(p.ws)[((int64_t)gx * p.n + n) * p.taps + tap];
        }
        if (have) {  // a tap outside the entry meets zeros
            const i32x4* xp = reinterpret_cast<const i32x4*>(p.xc + ((int64_t)(m + shift) * p.groups + gx) * kGroupBytes);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = xp[i];
            xscale = reinterpret_cast<const int*>(p.xs)[(int64_t)gx * p.rows + m + shift];
        }
        acc = step<0>(w[0], x[0], wscale, xscale, acc);
        acc = step<1>(w[1], x[1], wscale, xscale, acc);
        acc = step<2>(w[2], x[2], wscale, xscale, acc);
        acc = step<3>(w[3], x[3], wscale, xscale, acc);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[wave][r][8 * (i >> 2) + 4 * half + (i & 3)] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += WAVES * 64) {
        const int mm = e >> 5, nn = e & 31;
        if (m0 + mm >= p.rows || n0 + nn >= p.n) continue;
        float v = sums[0][mm][nn];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += sums[k][mm][nn];
        if (p.bias) v += load_float(p.bias, p.bias_type, n0 + nn);
        if (p.relu) v = relu(v);
        store_float(p.y, p.y_type, (int64_t)(m0 + mm) * p.n + n0 + nn, v);
    }
}


// rows sixteen at a time by groups four at a time
unsigned span_blocks(int rows, int groups) { return (unsigned)((rows + 15) / 16) * ((groups + 3) / 4); }

int quantise(const void* x, int type, Rows xr, int rows, int cols, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const int groups = (cols + kGroup - 1) / kGroup;
    const dim3 grid(span_blocks(rows, groups)), block(256);
    if (type == GLV_F32)
        hipLaunchKernelGGL(quantise_kernel<float>, grid, block, 0, st, (const float*)x, xr, rows, cols, groups, codes, scales);
    else if (type == GLV_BF16)
        hipLaunchKernelGGL(quantise_kernel<bf16>, grid, block, 0, st, (const bf16*)x, xr, rows, cols, groups, codes, scales);
    else
        hipLaunchKernelGGL(quantise_kernel<f16>, grid, block, 0, st, (const f16*)x, xr, rows, cols, groups, codes, scales);
    return launch_status("quantise_kernel");
}

// Row counts and widths are ints in the kernels, row * groups is formed in 64 bits, and every
// launch counts its workgroups in one 31-bit dimension: these limits keep all of that in range.
constexpr int64_t kMaxRows = 1 << 24;
constexpr int kMaxCols = 1 << 18;

int check_shape(const char* what, int64_t rows, int64_t cols) {
    if (rows < 0 || rows > kMaxRows)
        return report(GLV_ERR_INVALID, "%s: %lld rows outside [0, %lld]", what, (long long)rows, (long long)kMaxRows);
    if (cols < 1 || cols > kMaxCols)
        return report(GLV_ERR_INVALID, "%s: %lld columns outside [1, %d]", what, (long long)cols, kMaxCols);
    return GLV_OK;
}

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

int check_quantised(const char* what, const void* codes, const void* scales) {
    if (misaligned(codes, 16) || misaligned(scales, 4))
        return report(GLV_ERR_INVALID, "%s: codes must be 16-byte and scales 4-byte aligned", what);
    return GLV_OK;
}

int64_t quantised_bytes(int64_t rows, int64_t groups) { return rows * groups * (kGroupBytes + 4); }

}  // namespace

extern "C" int glv_mxfp4_quantize(const void* x_dev, int x_type, int batch, int rows, int cols, int64_t batch_stride,
                                  int64_t row_stride, uint8_t* codes_dev, uint8_t* scales_dev, void* stream) {
    const char* what = "glv_mxfp4_quantize";
    if (batch < 0 || rows < 0) return report(GLV_ERR_INVALID, "%s: negative batch or rows", what);
    const int64_t all = (int64_t)batch * rows;
    int rc = check_shape(what, all, cols);
    if (rc != GLV_OK) return rc;
    if (!float_type(x_type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d", what, x_type);
    if (all == 0) return GLV_OK;
    if (!x_dev || !codes_dev || !scales_dev) return report(GLV_ERR_INVALID, "%s: null argument", what);
    if (misaligned(x_dev, x_type == GLV_F32 ? 4 : 2)) return report(GLV_ERR_INVALID, "%s: x is not aligned to its elements", what);
    rc = check_quantised(what, codes_dev, scales_dev);
    if (rc != GLV_OK) return rc;
    return quantise(x_dev, x_type, Rows{batch_stride, row_stride, rows}, (int)all, cols, codes_dev, scales_dev,
                    (hipStream_t)stream);
}

extern "C" int glv_mxfp4_dequantize(const uint8_t* codes_dev, const uint8_t* scales_dev, int rows, int cols, int out_type,
                                    void* out_dev, void* stream) {
    const char* what = "glv_mxfp4_dequantize";
    int rc = check_shape(what, rows, cols);
    if (rc != GLV_OK) return rc;
    if (!float_type(out_type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d", what, out_type);
    if (rows == 0) return GLV_OK;
    if (!codes_dev || !scales_dev || !out_dev) return report(GLV_ERR_INVALID, "%s: null argument", what);
    if (misaligned(out_dev, out_type == GLV_F32 ? 4 : 2)) return report(GLV_ERR_INVALID, "%s: out is not aligned to its elements", what);
    rc = check_quantised(what, codes_dev, scales_dev);
    if (rc != GLV_OK) return rc;
    const int groups = (cols + kGroup - 1) / kGroup;
    const dim3 grid(span_blocks(rows, groups)), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (out_type == GLV_F32)
        hipLaunchKernelGGL(dequantise_kernel<float>, grid, block, 0, st, codes_dev, scales_dev, rows, cols, groups, (float*)out_dev);
    else if (out_type == GLV_BF16)
        hipLaunchKernelGGL(dequantise_kernel<bf16>, grid, block, 0, st, codes_dev, scales_dev, rows, cols, groups, (bf16*)out_dev);
    else
        hipLaunchKernelGGL(dequantise_kernel<f16>, grid, block, 0, st, codes_dev, scales_dev, rows, cols, groups, (f16*)out_dev);
    return launch_status("dequantise_kernel");
}

extern "C" int64_t glv_mxfp4_product_workspace(int x_type, int batch, int rows, int cols, int n_out, int taps) {
    if (batch < 0 || rows < 0 || n_out < 0 || taps < 1 || cols < 1 || cols > kMaxCols) return -1;
    if ((int64_t)batch * rows > kMaxRows || !(float_type(x_type) || x_type == GLV_MXFP4)) return -1;
    if (x_type == GLV_MXFP4) return 0;
    return quantised_bytes((int64_t)batch * rows, (cols + kGroup - 1) / kGroup);
}

extern "C" int glv_mxfp4_product(const void* x_dev, const uint8_t* x_scales_dev, int x_type, int batch, int rows, int cols,
                                 int64_t x_batch_stride, int64_t x_row_stride, const uint8_t* w_codes_dev,
                                 const uint8_t* w_scales_dev, int n_out, int taps, int dilation, const void* bias_dev,
                                 int bias_type, int activation, void* y_dev, int y_type, void* workspace_dev,
                                 int64_t workspace_bytes, void* stream) {
    const char* what = "glv_mxfp4_product";
    if (batch < 0 || rows < 0) return report(GLV_ERR_INVALID, "%s: negative batch or rows", what);
    const int64_t all = (int64_t)batch * rows;
    int rc = check_shape(what, all, cols);
    if (rc != GLV_OK) return rc;
    if (n_out < 0 || n_out > kMaxCols) return report(GLV_ERR_INVALID, "%s: n_out %d outside [0, %d]", what, n_out, kMaxCols);
    if (taps < 1 || dilation < 1 || (int64_t)taps * cols > kMaxCols || (int64_t)n_out * taps > kMaxRows ||
        (int64_t)(taps - 1) * dilation > kMaxRows)
        return report(GLV_ERR_INVALID, "%s: taps %d and dilation %d must be positive, taps x columns at most %d, "
                      "n_out x taps and (taps - 1) x dilation at most %lld", what, taps, dilation, kMaxCols, (long long)kMaxRows);
    if (!float_type(x_type) && x_type != GLV_MXFP4) return report(GLV_ERR_INVALID, "%s: unknown element type %d of x", what, x_type);
    if (!float_type(y_type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d of y", what, y_type);
    if (activation != GLV_ACT_NONE && activation != GLV_ACT_RELU) return report(GLV_ERR_INVALID, "%s: unknown activation %d", what, activation);
    if (bias_dev && !float_type(bias_type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d of the bias", what, bias_type);
    if (all == 0 || n_out == 0) return GLV_OK;
    if (!x_dev || !w_codes_dev || !w_scales_dev || !y_dev || (x_type == GLV_MXFP4 && !x_scales_dev))
        return report(GLV_ERR_INVALID, "%s: null argument", what);
    rc = check_quantised(what, w_codes_dev, w_scales_dev);
    if (rc != GLV_OK) return rc;
    if (misaligned(y_dev, y_type == GLV_F32 ? 4 : 2) || (bias_dev && misaligned(bias_dev, bias_type == GLV_F32 ? 4 : 2)) ||
        (x_type != GLV_MXFP4 && misaligned(x_dev, x_type == GLV_F32 ? 4 : 2)))
        return report(GLV_ERR_INVALID, "%s: an array is not aligned to its elements", what);
    hipStream_t st = (hipStream_t)stream;

    Product p = {};
    p.rows = (int)all, p.T = rows, p.n = n_out;
    p.taps = taps, p.dilation = dilation, p.left = dilation * (taps - 1) / 2;
    p.groups = (cols + kGroup - 1) / kGroup;
    p.wc = w_codes_dev, p.ws = w_scales_dev;
    p.bias = bias_dev, p.bias_type = bias_type, p.relu = activation == GLV_ACT_RELU;
    p.y = y_dev, p.y_type = y_type;
    if (x_type == GLV_MXFP4) {
        rc = check_quantised(what, x_dev, x_scales_dev);
        if (rc != GLV_OK) return rc;
        p.xc = static_cast<const uint8_t*>(x_dev), p.xs = x_scales_dev;
    } else {
        const int64_t need = quantised_bytes(all, p.groups);
        if (!workspace_dev || workspace_bytes < need)
            return report(GLV_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed (glv_mxfp4_product_workspace)", what,
                          (long long)(workspace_dev ? workspace_bytes : 0), (long long)need);
        if (misaligned(workspace_dev, 16)) return report(GLV_ERR_INVALID, "%s: the workspace is not 16-byte aligned", what);
        uint8_t* codes = static_cast<uint8_t*>(workspace_dev);
        uint8_t* scales = codes + all * p.groups * kGroupBytes;
        rc = quantise(x_dev, x_type, Rows{x_batch_stride, x_row_stride, rows}, p.rows, cols, codes, scales, st);
        if (rc != GLV_OK) return rc;
        p.xc = codes, p.xs = scales;
    }
    const int64_t tiles = ((all + 31) / 32) * ((n_out + 31) / 32);
    if (tiles > INT32_MAX) return report(GLV_ERR_INVALID, "%s: rows x n_out too large for one call", what);
    hipLaunchKernelGGL(product_direct_kernel<4>, dim3((unsigned)tiles), dim3(256), 0, st, p);
    return launch_status("product_direct_kernel");
}
