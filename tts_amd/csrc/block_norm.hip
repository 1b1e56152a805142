// The end of one block and the start of the next in one pass over the rows:
//     y = residual + scale * gate * Norm_post(u)        z = Norm_pre(y)
// with LayerNorm  N(x) = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias
// or   RMSNorm    N(x) = x / sqrt(mean(x^2) + eps) * weight + bias.
//
// A row stays in registers between its reads and its writes: sums, means and the variance (taken
// around the mean, in a second pass over the registers) are float, y enters the second norm before
// it is rounded to the element type.  What bounds it is memory: every stream is touched once.
#include "lowp.h"
#include "status.h"

using namespace glv;

namespace {

struct BlockNorm {
    const void *u, *gate, *residual;
    int64_t u_batch, u_row, gate_batch, gate_row, res_batch, res_row;
    int gate_col;  // 0: one value for the row
    const void *post_w, *post_b, *pre_w, *pre_b, *scale_vec;
    int post, pre;  // GLV_NORM_*
    float post_eps, pre_eps, scale;
    void *y, *z;
    int rows, T, cols;
};

__device__ inline float wave_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const auto s16 = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = __builtin_bit_cast(float, (unsigned)s16[0]) + __builtin_bit_cast(float, (unsigned)s16[1]);
    const unsigned c = __builtin_bit_cast(unsigned, v);
    const auto s32 = __builtin_amdgcn_permlane32_swap(c, c, false, false);
    return __builtin_bit_cast(float, (unsigned)s32[0]) + __builtin_bit_cast(float, (unsigned)s32[1]);
}

// sum over the TPR threads of a row; `slot` is a different array for every use within a kernel
template <int TPR>
__device__ inline float row_sum(float v, float* slot) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slot[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) v += slot[i];
    }
    return v;
}

// x <- Norm(x) for the row held as V pieces of eight per thread; `valid` counts columns
template <typename W, int TPR, int V, bool NARROW>
__device__ inline void normalise(float (&x)[V][8], int kind, const void* weight, const void* bias, float eps, int cols,
                                 int lane, float* slot) {
    const float inv = 1.f / (float)cols;
    if (kind == GLV_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += x[v][i];
        const float mean = row_sum<TPR>(s, slot) * inv;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[v][i] = (v * TPR + lane) * 8 + i < cols ? x[v][i] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) q += x[v][i] * x[v][i];
    const float r = rsqrtf(row_sum<TPR>(q, slot + TPR / 64) * inv + eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = (v * TPR + lane) * 8;
        if (col < cols) {
            Eight<W> w, b;
            if (weight) w = load_eight<NARROW>(static_cast<const W*>(weight), col, cols);
            if (bias) b = load_eight<NARROW>(static_cast<const W*>(bias), col, cols);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float t = x[v][i] * r;
                if (weight) t *= (float)w.v[i];
                if (bias) t += (float)b.v[i];
                x[v][i] = t;
            }
        }
    }
}

// TPR threads a row, V pieces of eight columns a thread
template <typename T, typename W, int TPR, int V, bool NARROW = false>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void block_norm_kernel(BlockNorm p) {
    __shared__ float slots[TPR > 64 ? 4 * (TPR / 64) : 1];
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    const int row = blockIdx.x * kRows + (TPR < 256 ? threadIdx.x / TPR : 0);
    const int lane = threadIdx.x % TPR;
    if (row >= p.rows) return;  // whole waves: a row is one wave here, or the workgroup
    const int b = row / p.T, t = row - b * p.T;
    const T* u = static_cast<const T*>(p.u) + b * p.u_batch + t * p.u_row;
    const T* gate = p.gate ? static_cast<const T*>(p.gate) + b * p.gate_batch + t * p.gate_row : nullptr;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + b * p.res_batch + t * p.res_row : nullptr;
    const int64_t out = (int64_t)row * p.cols;

    Eight<T> ur[V], gr[V], rr[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = (v * TPR + lane) * 8;
        ur[v] = load_eight<NARROW>(u, col, p.cols);
        if (gate && p.gate_col) gr[v] = load_eight<NARROW>(gate, col, p.cols);
        if (res) rr[v] = load_eight<NARROW>(res, col, p.cols);
    }
    float x[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[v][i] = (float)ur[v].v[i];
    if (p.post) normalise<W, TPR, V, NARROW>(x, p.post, p.post_w, p.post_b, p.post_eps, p.cols, lane, slots);
    const float row_factor = p.scale * (gate && !p.gate_col ? (float)gate[0] : 1.f);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = (v * TPR + lane) * 8;
        Eight<W> sv;
        if (p.scale_vec) sv = load_eight<NARROW>(static_cast<const W*>(p.scale_vec), col, p.cols);
        Eight<T> o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float k = x[v][i] * row_factor;
            if (gate && p.gate_col) k *= (float)gr[v].v[i];
            if (p.scale_vec) k *= (float)sv.v[i];
            if (res) k += (float)rr[v].v[i];
            x[v][i] = col + i < p.cols ? k : 0.f;
            o.v[i] = (T)k;
        }
        store_eight(static_cast<T*>(p.y) + out + col, o, p.cols - col);
    }
    if (!p.pre) return;
    normalise<W, TPR, V, NARROW>(x, p.pre, p.pre_w, p.pre_b, p.pre_eps, p.cols, lane, slots + 2 * (TPR / 64));
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int col = (v * TPR + lane) * 8;
        Eight<T> o;
#pragma unroll
        for (int i = 0; i < 8; ++i) o.v[i] = (T)x[v][i];
        store_eight(static_cast<T*>(p.z) + out + col, o, p.cols - col);
    }
}

template <typename T, typename W>
void launch(const BlockNorm& p, hipStream_t st) {
    const dim3 by4((p.rows + 3) / 4), by1(p.rows);
    if (p.cols < 8)
        hipLaunchKernelGGL((block_norm_kernel<T, W, 64, 1, true>), by4, dim3(256), 0, st, p);
    else if (p.cols <= 512)
        hipLaunchKernelGGL((block_norm_kernel<T, W, 64, 1>), by4, dim3(256), 0, st, p);
    else if (p.cols <= 1024)
        hipLaunchKernelGGL((block_norm_kernel<T, W, 64, 2>), by4, dim3(256), 0, st, p);
    else if (p.cols <= 4096)
        hipLaunchKernelGGL((block_norm_kernel<T, W, 256, 2>), by1, dim3(256), 0, st, p);
    else if (p.cols <= 8192)
        hipLaunchKernelGGL((block_norm_kernel<T, W, 256, 4>), by1, dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((block_norm_kernel<T, W, 1024, 4>), by1, dim3(1024), 0, st, p);
}

constexpr int kMaxCols = 32768;         // 1024 threads of 32 columns
constexpr int64_t kMaxRows = 1 << 24;

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
bool norm_kind(int k) { return k == GLV_NORM_NONE || k == GLV_NORM_LAYER || k == GLV_NORM_RMS; }

}  // namespace

extern "C" int glv_block_norm(const void* u_dev, int type, int batch, int rows, int cols, int64_t u_batch_stride,
                              int64_t u_row_stride, int vector_type, int post_kind, const void* post_weight_dev,
                              const void* post_bias_dev, float post_eps, const void* gate_dev, int64_t gate_batch_stride,
                              int64_t gate_row_stride, int gate_col_stride, const void* scale_dev, float scale,
                              const void* residual_dev, int64_t residual_batch_stride, int64_t residual_row_stride,
                              int pre_kind, const void* pre_weight_dev, const void* pre_bias_dev, float pre_eps, void* y_dev,
                              void* z_dev, void* stream) {
    const char* what = "glv_block_norm";
    if (batch < 0 || rows < 0 || (int64_t)batch * rows > kMaxRows)
        return report(GLV_ERR_INVALID, "%s: %d x %d rows outside [0, %lld]", what, batch, rows, (long long)kMaxRows);
    if (cols < 1 || cols > kMaxCols) return report(GLV_ERR_INVALID, "%s: cols %d outside [1, %d]", what, cols, kMaxCols);
    if (!float_type(type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d", what, type);
    if (vector_type != GLV_F32 && vector_type != type)
        return report(GLV_ERR_INVALID, "%s: weights, biases and scales are float32 or of the type of u", what);
    if (!norm_kind(post_kind) || !norm_kind(pre_kind)) return report(GLV_ERR_INVALID, "%s: unknown norm", what);
    if (!(post_eps >= 0.f) || !(pre_eps >= 0.f)) return report(GLV_ERR_INVALID, "%s: eps must be >= 0", what);
    if (gate_col_stride != 0 && gate_col_stride != 1) return report(GLV_ERR_INVALID, "%s: gate_col_stride is 0 or 1", what);
    if (batch == 0 || rows == 0) return GLV_OK;
    if (!u_dev || !y_dev || (pre_kind != GLV_NORM_NONE && !z_dev)) return report(GLV_ERR_INVALID, "%s: null argument", what);
    const size_t size = type == GLV_F32 ? 4 : 2, vsize = vector_type == GLV_F32 ? 4 : 2;
    const void* elements[] = {u_dev, gate_dev, residual_dev, y_dev, z_dev};
    const void* vectors[] = {post_weight_dev, post_bias_dev, scale_dev, pre_weight_dev, pre_bias_dev};
    for (const void* e : elements)
        if (misaligned(e, size)) return report(GLV_ERR_INVALID, "%s: an array is not aligned to its elements", what);
    for (const void* e : vectors)
        if (misaligned(e, vsize)) return report(GLV_ERR_INVALID, "%s: an array is not aligned to its elements", what);
    BlockNorm p = {};
    p.u = u_dev, p.u_batch = u_batch_stride, p.u_row = u_row_stride;
    p.gate = gate_dev, p.gate_batch = gate_batch_stride, p.gate_row = gate_row_stride, p.gate_col = gate_col_stride;
    p.residual = residual_dev, p.res_batch = residual_batch_stride, p.res_row = residual_row_stride;
    p.post = post_kind, p.post_w = post_weight_dev, p.post_b = post_bias_dev, p.post_eps = post_eps;
    p.pre = pre_kind, p.pre_w = pre_weight_dev, p.pre_b = pre_bias_dev, p.pre_eps = pre_eps;
    p.scale_vec = scale_dev, p.scale = scale;
    p.y = y_dev, p.z = z_dev;
    p.rows = batch * rows, p.T = rows, p.cols = cols;
    hipStream_t st = (hipStream_t)stream;
    if (type == GLV_F32)
        launch<float, float>(p, st);
    else if (type == GLV_BF16)
        vector_type == GLV_F32 ? launch<bf16, float>(p, st) : launch<bf16, bf16>(p, st);
    else
        vector_type == GLV_F32 ? launch<f16, float>(p, st) : launch<f16, f16>(p, st);
    return launch_status("block_norm_kernel");
}
