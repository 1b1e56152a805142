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

template <int CTRL>
__device__ inline float plus_dpp(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// sum over LANES neighbouring lanes (16, 32 or 64), in all of them
template <int LANES>
__device__ inline float lanes_sum(float v) {
    v = plus_dpp<0xB1>(v);   // quad_perm 1,0,3,2
    v = plus_dpp<0x4E>(v);   // quad_perm 2,3,0,1
    v = plus_dpp<0x141>(v);  // row_half_mirror
    v = plus_dpp<0x140>(v);  // row_mirror
    if constexpr (LANES >= 32) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
        v = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
    }
    if constexpr (LANES == 64) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
        v = __builtin_bit_cast(float, (unsigned)s[0]) + __builtin_bit_cast(float, (unsigned)s[1]);
    }
    return v;
}

// Lanes of a row: 16, 32 or 64 of a wave, or (0) all waves of the workgroup, at most 16.
template <int LANES>
struct Row {
    int lane, lanes;
    float* slots;  // LANES 0: 16 for every sum of the kernel, used once each

    __device__ float sum(float v, int use) const {
        if constexpr (LANES > 0) return lanes_sum<LANES>(v);
        v = lanes_sum<64>(v);
        float* s = slots + 16 * use;
        const int at = threadIdx.x & 15;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        return lanes_sum<16>(at < lanes >> 6 ? s[at] : 0.f);
    }
};

// A lane holds V pieces of N columns: 16 bytes of a stream each, so that what the lanes of a row touch
// at once is one run of memory.  A piece that reaches over the row's end is the row's last N columns instead,
// of which the first are another lane's: its elements [lo, hi) count, and no value has to be moved into place (which
// cost a tenth of the time at 1001 x 5000).
// NARROW: rows of fewer than N columns.
template <int N, bool NARROW>
struct Piece {
    int at, lo, hi;  // element i is column at + i

    __device__ Piece(int col, int cols) {
        if constexpr (NARROW)
            at = 0, lo = col == 0 ? 0 : N, hi = cols;
        else
            at = min(col, cols - N), lo = min(col - at, N), hi = N;
    }
    __device__ bool whole() const { return lo == 0 && hi == N; }
    template <typename T>
    __device__ Pack<T, N> fetch(const T* row) const {
        return fetch_pack<NARROW, N>(row, at, NARROW ? hi : at + N);
    }
    template <typename T>
    __device__ void store(T* row, const Pack<T, N>& r) const {
        if (whole()) {
            store_pack(row + at, r, N);
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i >= lo && i < hi) row[at + i] = r.v[i];
    }
    // zeros for what does not count
    __device__ void mask(float (&x)[N]) const {
        if (whole()) return;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i >= lo && i < hi ? x[i] : 0.f;
    }
};

// Keeps a pack as it was loaded until here: the compiler would convert it to float at its load, and hold twice the
// registers over all the sums (1001 x 5000 float16, the whole boundary: 13.8 us against 15.4).
template <typename T, int N>
__device__ inline void as_loaded(Pack<T, N>& r) {
    if constexpr (sizeof(T) == 2) {
        i32x4 w;
        static_assert(sizeof(w) == sizeof(r));
        __builtin_memcpy(&w, &r, sizeof(w));
        asm volatile("" : "+v"(w));
        __builtin_memcpy(&r, &w, sizeof(w));
    }
}

// Whether what meets the row after its sums is under way while they are formed, or is read when they are done:
// early, but for float32 rows of several waves, whose registers would leave a CU room for fewer rows (us, the whole
// boundary, early against late: 1001 x 5000 26.2 and 18.2, 4000 x 9000 185 and 154; a wave a row, 55360 x 900, 189 and
// 200), and for four eights a lane, whose would spill (8000 x 20000 float32: 1380 and 672).
template <int LANES, int EIGHTS, int N>
constexpr bool early() {
    return EIGHTS <= 2 && (LANES > 0 || N == 8);
}

// x <- Norm(x)
template <typename W, int LANES, int V, int N, bool NARROW>
__device__ inline void normalise(float (&x)[V][N], int kind, const void* weight, const void* bias, float eps, int cols,
                                 const Row<LANES>& row, int use) {
    const float inv = 1.f / (float)cols;
    auto piece = [&](int v) { return Piece<N, NARROW>((v * row.lanes + row.lane) * N, cols); };
    constexpr bool kEarly = early<LANES, V * N / 8, N>();
    Pack<W, N> w[V], b[V];
    auto fetch = [&](int v) {
        if (weight) w[v] = piece(v).fetch(static_cast<const W*>(weight));
        if (bias) b[v] = piece(v).fetch(static_cast<const W*>(bias));
    };
    if constexpr (kEarly)
#pragma unroll
        for (int v = 0; v < V; ++v) fetch(v);
#pragma unroll
    for (int v = 0; v < V; ++v) piece(v).mask(x[v]);
    if (kind == GLV_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) s += x[v][i];
        const float mean = row.sum(s, use) * inv;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int i = 0; i < N; ++i) x[v][i] -= mean;
            piece(v).mask(x[v]);
        }
    }
    float q = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) q += x[v][i] * x[v][i];
    const float r = rsqrtf(row.sum(q, use + 1) * inv + eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if constexpr (!kEarly) fetch(v);
        if (weight) as_loaded(w[v]);
        if (bias) as_loaded(b[v]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = x[v][i] * r;
            if (weight) t *= (float)w[v].v[i];
            if (bias) t += (float)b[v].v[i];
            x[v][i] = t;
        }
    }
}

// EIGHTS: columns a lane holds, in eights
template <typename T, typename W, int LANES, int EIGHTS, bool NARROW = false>
__global__ __launch_bounds__(LANES > 0 ? 256 : 1024) void block_norm_kernel(BlockNorm p) {
    __shared__ float slots[LANES > 0 ? 1 : 64];
    constexpr int N = 16 / sizeof(T), V = EIGHTS * 8 / N;
    constexpr int kRows = LANES > 0 ? 256 / LANES : 1;
    const int index = blockIdx.x * kRows + (LANES > 0 ? threadIdx.x / LANES : 0);
    // the rows behind the last are computed from the last, for their lanes take part in the sums' exchanges
    const int at = min(index, p.rows - 1);
    const Row<LANES> row{LANES > 0 ? (int)threadIdx.x % LANES : (int)threadIdx.x, LANES > 0 ? LANES : (int)blockDim.x, slots};
    const int b = at / p.T, t = at - b * p.T;
    const T* u = static_cast<const T*>(p.u) + b * p.u_batch + t * p.u_row;
    const T* gate = p.gate ? static_cast<const T*>(p.gate) + b * p.gate_batch + t * p.gate_row : nullptr;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + b * p.res_batch + t * p.res_row : nullptr;
    const int64_t out = (int64_t)at * p.cols;
    const int cols = p.cols;
    const bool stored = index < p.rows;
    auto piece = [&](int v) { return Piece<N, NARROW>((v * row.lanes + row.lane) * N, cols); };

    Pack<T, N> ur[V], gr[V], rr[V];
    constexpr bool kEarly = early<LANES, EIGHTS, N>();
    auto fetch = [&](int v) {
        if (gate && p.gate_col) gr[v] = piece(v).fetch(gate);
        if (res) rr[v] = piece(v).fetch(res);
    };
#pragma unroll
    for (int v = 0; v < V; ++v) {
        ur[v] = piece(v).fetch(u);
        if constexpr (kEarly) fetch(v);
    }
    const float row_factor = p.scale * (gate && !p.gate_col ? (float)gate[0] : 1.f);
    float x[V][N];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) x[v][i] = (float)ur[v].v[i];
    if (p.post) normalise<W, LANES, V, N, NARROW>(x, p.post, p.post_w, p.post_b, p.post_eps, cols, row, 0);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if constexpr (!kEarly) fetch(v);
        Pack<W, N> sv;
        if (p.scale_vec) sv = piece(v).fetch(static_cast<const W*>(p.scale_vec));
        if (gate && p.gate_col) as_loaded(gr[v]);
        if (res) as_loaded(rr[v]);
        Pack<T, N> o;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float k = x[v][i] * row_factor;
            if (gate && p.gate_col) k *= (float)gr[v].v[i];
            if (p.scale_vec) k *= (float)sv.v[i];
            if (res) k += (float)rr[v].v[i];
            x[v][i] = k;
            o.v[i] = (T)k;
        }
        if (stored) piece(v).store(static_cast<T*>(p.y) + out, o);
    }
    if (!p.pre) return;
    normalise<W, LANES, V, N, NARROW>(x, p.pre, p.pre_w, p.pre_b, p.pre_eps, cols, row, 2);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        Pack<T, N> o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.v[i] = (T)x[v][i];
        if (stored) piece(v).store(static_cast<T*>(p.z) + out, o);
    }
}

// The fewest lanes that hold a row: 16 or 32 leave room for the other rows of a wave (us, the whole boundary in
// float16: 32768 x 256 26.8 at 64 lanes, 19.0 at 32); beyond a wave as many waves as two eights a lane ask for (1001 x 3000
// 8.8, with four eights 11.3; 4000 x 9000 94 and 113) up to twelve, of which a CU holds two workgroups (4000 x 12200 125
// and 141), then four eights (4000 x 12400 137, with two 153).
template <typename T, typename W>
int run(const BlockNorm& p, hipStream_t st) {
    const int pieces = (p.cols + 7) / 8;  // a lane holds one, two or four of them
    const int threads = (pieces <= 1536 ? (pieces + 127) / 128 : (pieces + 255) / 256) * 64;  // of a workgroup to itself
    if (pieces > 128 && too_large(p.rows, threads)) return report(GLV_ERR_INVALID, "glv_block_norm: rows x columns too large for one call");
    auto rows_a_wave = [&](auto kernel, int lanes) {
        return launch("block_norm_kernel", kernel, dim3((unsigned)(((int64_t)p.rows * lanes + 255) / 256)), dim3(256), 0, st, p);
    };
    if (p.cols < 16 / (int)sizeof(T)) return rows_a_wave(block_norm_kernel<T, W, 16, 1, true>, 16);
    if (pieces <= 16) return rows_a_wave(block_norm_kernel<T, W, 16, 1>, 16);
    if (pieces <= 32) return rows_a_wave(block_norm_kernel<T, W, 32, 1>, 32);
    if (pieces <= 64) return rows_a_wave(block_norm_kernel<T, W, 64, 1>, 64);
    if (pieces <= 128) return rows_a_wave(block_norm_kernel<T, W, 64, 2>, 64);
    return launch("block_norm_kernel", pieces <= 1536 ? block_norm_kernel<T, W, 0, 2> : block_norm_kernel<T, W, 0, 4>, dim3(p.rows),
                  dim3(threads), 0, st, p);
}

constexpr int kMaxCols = 32768;         // 1024 threads of 32 columns
constexpr int64_t kMaxRows = 1 << 24;

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }
bool norm_kind(int k) { return k == GLV_NORM_NONE || k == GLV_NORM_LAYER || k == GLV_NORM_RMS; }

}  // namespace

extern "C" int glv_block_norm(const glv_block_norm_args* a, void* stream) {
    const char* what = "glv_block_norm";
    if (!a) return report(GLV_ERR_INVALID, "%s: null argument", what);
    const auto [u_dev, gate_dev, residual_dev, post_weight_dev, post_bias_dev, scale_dev, pre_weight_dev, pre_bias_dev, y_dev, z_dev,
                u_batch_stride, u_row_stride, gate_batch_stride, gate_row_stride, residual_batch_stride, residual_row_stride, type, batch,
                rows, cols, vector_type, post_kind, pre_kind, gate_col_stride, post_eps, pre_eps, scale] = *a;
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
    if (type == GLV_F32) return run<float, float>(p, st);
    if (type == GLV_BF16) return vector_type == GLV_F32 ? run<bf16, float>(p, st) : run<bf16, bf16>(p, st);
    return vector_type == GLV_F32 ? run<f16, float>(p, st) : run<f16, f16>(p, st);
}
