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
// scales.  Rows are padded with zeros to whole groups, and both arrays are group-major:
//     codes  [group][row][64]      scales [group][row][4]
// A product walks the groups and takes, of each, a run of rows: that is one run of memory here.  (In
// row order the codes of a stage are pieces of 64 bytes, and the scales that a matrix instruction
// wants in 32 lanes lie in 32 lines.)
#include <type_traits>

#include "lowp.h"
#include "status.h"

using namespace glv;

namespace {

constexpr int kGroup = 128;       // columns of a group
constexpr int kGroupBytes = 64;   // its codes

struct Rows {  // a (batch, rows, cols) array whose last dimension is contiguous
    int64_t batch_stride, row_stride;
    int rows;   // rows of one batch entry
    bool flat;  // there is one entry
};

__device__ inline int64_t row_offset(const Rows& r, int row) {
    if (r.flat) return row * r.row_stride;
    const int b = row / r.rows;
    return b * r.batch_stride + (int64_t)(row - b * r.rows) * r.row_stride;
}

// biased exponent of max|x| as float sees it (255: an infinity or a NaN is among them)
__device__ inline int top_exponent(const Eight<float>& x) {
    float m = 0.f;  // the maximum that keeps a NaN: three operands an instruction, signs dropped on the way in
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(m, __builtin_fabsf(x.v[i])), __builtin_fabsf(x.v[i + 1]));
    return (int)(__builtin_bit_cast(uint32_t, m) >> 23 & 255);
}
// the larger of the magnitudes' bits, two at a time: the order of the bits is that of the values
template <typename T>
__device__ inline uint32_t top_half_bits(const Eight<T>& x) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    struct Pairs {
        uint32_t w[4];
    };
    const Pairs p = __builtin_bit_cast(Pairs, x);
    u16x2 m = __builtin_bit_cast(u16x2, p.w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, p.w[i] & 0x7fff7fffu));
    return max((uint32_t)m.x, (uint32_t)m.y);
}
__device__ inline int top_exponent(const Eight<bf16>& x) { return (int)(top_half_bits(x) >> 7); }
__device__ inline int top_exponent(const Eight<f16>& x) {
    const uint32_t m = top_half_bits(x);
    // every finite half is a normal float, so its exponent there is the true one
    const float f = (float)__builtin_bit_cast(f16, (uint16_t)m);
    return m >= 0x7c00 ? 255 : (int)(__builtin_bit_cast(uint32_t, f) >> 23);
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
    const uint32_t codes = encode(x, __builtin_bit_cast(float, (uint32_t)s << 23));
    return s == 255 ? 0u : codes;
}

// Sixteen lanes a group; a workgroup takes sixteen rows of up to four groups.
template <typename T, bool NARROW>
__global__ __launch_bounds__(256) void quantise_kernel(const T* __restrict__ x, Rows xr, int rows, int cols, int groups,
                                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int spans = (groups + 3) / 4;
    const int rb = blockIdx.x / spans, first = (blockIdx.x - rb * spans) * 4;
    const int row = rb * 16 + (threadIdx.x >> 4);
    const int piece = threadIdx.x & 15;
    if (row >= rows) return;
    const T* src = x + row_offset(xr, row);
    // several loads before the first use; of float32 two, whose registers would cost waves (10560 x 1024: 8.7 us
    // against 10.1 with four; half precision 4.5 with four against 4.9 with one)
    constexpr int kDeep = sizeof(T) == 4 ? 2 : 4;
#pragma unroll
    for (int k0 = 0; k0 < 4; k0 += kDeep) {
        Eight<T> v[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const int g = first + k0 + k;
            if (g < groups) v[k] = fetch_pack<NARROW, 8>(src, g * kGroup + piece * 8, cols);
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
            const int g = first + k0 + k;
            if (g >= groups) return;
            int byte;
            const uint32_t c = quantise_eight(place_pack<NARROW>(v[k], g * kGroup + piece * 8, cols), &byte);
            const int64_t at = (int64_t)g * rows + row;
            reinterpret_cast<uint32_t*>(codes)[at * 16 + piece] = c;
            if ((piece & 3) == 0) scales[at * 4 + (piece >> 2)] = (uint8_t)byte;
        }
    }
}

// Half precision: eight columns a lane.  Float32: four and, 64 columns on, four more, so that what sixteen
// lanes store at once is one run (120000 x 4096: 445 us against 589 with runs of eight floats a lane).
template <typename T>
__global__ __launch_bounds__(256) void dequantise_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, int rows, int cols,
                                                         int groups, T* __restrict__ out) {
    const int spans = (groups + 3) / 4;
    const int rb = blockIdx.x / spans, first = (blockIdx.x - rb * spans) * 4;
    const int row = rb * 16 + (threadIdx.x >> 4);
    const int piece = threadIdx.x & 15;
    if (row >= rows) return;
    constexpr bool kWide = sizeof(T) == 4;
    uint32_t c[4], e[4];  // all loads before the first use; two codes a byte
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t at = (int64_t)(first + k) * rows + row;
        if (first + k < groups) {
            if constexpr (kWide) {
                const uint16_t* at16 = reinterpret_cast<const uint16_t*>(codes) + at * 32 + piece;
                c[k] = at16[0] | (uint32_t)at16[16] << 16;
            } else {
                c[k] = reinterpret_cast<const uint32_t*>(codes)[at * 16 + piece];
            }
            e[k] = reinterpret_cast<const uint32_t*>(scales)[at];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int col = (first + k) * kGroup + piece * (kWide ? 4 : 8);
        if (first + k >= groups) return;
        const f32x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], 1.f, 0),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], 1.f, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], 1.f, 2),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[k], 1.f, 3)};
        // 2^-127 is a subnormal float, 255 a NaN; the codes' own values come out of the conversion
        // exactly, and the product of the two is exact wherever T can hold it
        auto scale = [&](int block) {
            const uint32_t s = e[k] >> (block * 8) & 255;
            return __builtin_bit_cast(float, s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23);
        };
        T* const to = out + (int64_t)row * cols + col;
        if constexpr (kWide) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float s = scale(2 * h + (piece >> 3));
                float r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = v[2 * h + (i >> 1)][i & 1] * s;
                if (col + 64 * h + 4 <= cols) {
                    i32x4 w;
                    __builtin_memcpy(&w, r, 16);
                    store_16(to + 64 * h, w);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (col + 64 * h + i < cols) to[64 * h + i] = r[i];
                }
            }
        } else {
            const float s = scale(piece >> 2);
            Eight<T> r;
#pragma unroll
            for (int i = 0; i < 8; ++i) r.v[i] = (T)(v[i >> 1][i & 1] * s);
            store_pack(to, r, cols - col);
        }
    }
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
struct Product {
    const uint8_t *xc, *xs;  // quantised activations: rows = batch * T, or
    const void* x;           // float ones, of `cols` columns
    Rows xr;
    int cols;
    const uint8_t *wc, *ws;  // weights: n * taps rows of `groups` groups
    const void* bias;
    void* y;
    int rows, T, n;
    int taps, dilation, left;  // tap j of row t reads row t + j * dilation - left of its batch entry
    int groups;                // groups of one tap
    int bias_type, y_type;
    float least;               // 0: rectified; -infinity: as it is
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

// max(v, least) that keeps a NaN: the rectifier with least = 0, nothing with -infinity
__device__ inline float at_least(float v, float least) { return __builtin_elementwise_maximum(v, least); }

// Between a wave's writes to its own LDS and other lanes' reads of them (and back): the LDS queue keeps
// a wave's accesses in order, this keeps the compiler from changing it.
__device__ inline void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ inline i32x8 widen(i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// acc += W (32 rows) * X (32 rows)^T over 64 columns: lane l holds 32 of them, one block, of row l % 32;
// byte S of its scale dwords is that block's.  Which columns meet in one instruction is free as long
// as both operands agree: of a group's four blocks the lanes below 32 take the first two in the two
// steps, the others the last two, and a shift by 16 puts a lane's two scales in front.
template <int S>
__device__ inline f32x16 step(i32x4 w, i32x4 x, int wscale, int xscale, f32x16 acc) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(w), widen(x), acc, 4, 4, S, wscale, S, xscale);
}

// The workgroup quantises rows first .. first + span - 1 of x, whatever entries they belong to, into LDS:
//   codes [group][row][64], piece q of 16 bytes of row i at place q ^ (i / 4 % 4);  scales [group][row][4]
// Sixteen lanes that read one piece of sixteen rows in a run then touch each of the 64 banks once.
template <typename X, int THREADS>
__device__ inline void quantise_rows(const Product& p, int first, int span, uint32_t* codes, uint8_t* scales) {
    constexpr int kTeams = THREADS / 16, kDeep = sizeof(X) == 4 ? 4 : 8;  // sixteen lanes a row and group
    const int team = threadIdx.x >> 4, piece = threadIdx.x & 15, units = span * p.groups;
    // unit u is group u % groups of row u / groups; one team's units are kTeams apart
    struct Unit {
        int i, gx;
    };
    const int step_i = kTeams / p.groups, step_gx = kTeams - step_i * p.groups;
    auto next = [&](Unit u) {
        u.i += step_i, u.gx += step_gx;
        const bool over = u.gx >= p.groups;
        return Unit{u.i + over, over ? u.gx - p.groups : u.gx};
    };
    Unit at{team / p.groups, team % p.groups};
    for (int u0 = team; u0 < units; u0 += kTeams * kDeep) {
        Eight<X> v[kDeep];  // all loads before the first use
        Unit u = at;
#pragma unroll
        for (int k = 0; k < kDeep; ++k, u = next(u)) {
            if (u0 + k * kTeams >= units) break;
            v[k] = fetch_pack<false, 8>(static_cast<const X*>(p.x) + row_offset(p.xr, first + u.i), u.gx * kGroup + piece * 8, p.cols);
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k, at = next(at)) {
            if (u0 + k * kTeams >= units) break;
            int byte;
            const uint32_t c = quantise_eight(place_pack<false>(v[k], at.gx * kGroup + piece * 8, p.cols), &byte);
            const int row = at.gx * span + at.i;
            codes[(row * 4 + (((piece >> 2) ^ (at.i >> 2)) & 3)) * 4 + (piece & 3)] = c;
            if ((piece & 3) == 0) scales[row * 4 + (piece >> 2)] = (uint8_t)byte;
        }
    }
}

// Workgroup ids go round the eight XCDs; each XCD gets a contiguous run of tiles, and a run walks
// eight rows of tiles at a time, so that what an XCD's L2 holds is used by several of its CUs.
struct Tile {
    int m, n;
};
__device__ inline Tile tile_of(int id, int total, int m_tiles, int n_tiles) {
    const int q = total >> 3, rem = total & 7, xcd = id & 7;
    id = xcd * q + min(xcd, rem) + (id >> 3);
    const int band = id / (8 * n_tiles), first = band * 8, high = min(m_tiles - first, 8);
    id -= band * 8 * n_tiles;
    return Tile{first + id % high, id / high};
}

// One 32 x 32 tile of y a workgroup; the waves deal the groups out among themselves and their sums meet
// in LDS in a fixed order.  X is `void` for activations that are quantised already; otherwise the
// workgroup first quantises the rows of x that its tile reaches, all groups of them, into LDS, so that
// a small product is one launch, and every tap of a convolution finds them there.
template <typename X, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void product_direct_kernel(Product p) {
    constexpr bool kOwn = !std::is_void_v<X>;
    __shared__ float sums[WAVES][32][33];
    extern __shared__ __align__(16) uint8_t held[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, half = lane >> 5;
    const int n_tiles = (p.n + 31) / 32;
    const Tile tile = tile_of(blockIdx.x, gridDim.x, (p.rows + 31) / 32, n_tiles);
    const int n0 = tile.n * 32, m0 = tile.m * 32;
    const int n = min(n0 + r, p.n - 1), m = min(m0 + r, p.rows - 1);  // rows beyond the ends: computed, not stored
    const int rows = min(32, p.rows - m0);
    const int t = p.taps == 1 ? 0 : m % p.T;
    const int all = p.taps * p.groups;

    i32x4 w0 = {}, w1 = {};
    uint32_t wscale = 0;
    auto fetch_w = [&](int g) {
        const int tap = p.taps == 1 ? 0 : g / p.groups, gx = g - tap * p.groups;
        const int64_t row = ((int64_t)gx * p.n + n) * p.taps + tap;
        const i32x4* wp = reinterpret_cast<const i32x4*>(p.wc + row * kGroupBytes) + half * 2;
        w0 = wp[0], w1 = wp[1];
        wscale = reinterpret_cast<const uint32_t*>(p.ws)[row];
    };
    if (wave < all) fetch_w(wave);  // under way while x is quantised

    // rows first .. first + span - 1 of x, whatever entries they belong to
    const int first = max(m0 - p.left, 0);
    const int span = min(m0 + rows - 1 + (p.taps - 1) * p.dilation - p.left, p.rows - 1) - first + 1;
    uint32_t* const codes = reinterpret_cast<uint32_t*>(held);
    uint8_t* const scales = held + span * p.groups * kGroupBytes;
    if constexpr (kOwn) {
        quantise_rows<X, WAVES * 64>(p, first, span, codes, scales);
        __syncthreads();
    }

    f32x16 acc = {};
    for (int g = wave; g < all; g += WAVES) {
        const int tap = p.taps == 1 ? 0 : g / p.groups, gx = g - tap * p.groups;
        const int shift = tap * p.dilation - p.left;
        i32x4 x0 = {}, x1 = {};
        uint32_t xscale = 0;
        if ((unsigned)(t + shift) < (unsigned)p.T) {  // a tap outside the entry meets zeros
            if constexpr (kOwn) {
                const int i = m + shift - first, row = gx * span + i, place = i >> 2;
                x0 = *reinterpret_cast<const i32x4*>(codes + (row * 4 + ((half * 2 ^ place) & 3)) * 4);
                x1 = *reinterpret_cast<const i32x4*>(codes + (row * 4 + (((half * 2 + 1) ^ place) & 3)) * 4);
                xscale = *reinterpret_cast<const uint32_t*>(scales + row * 4);
            } else {
                const int64_t row = (int64_t)gx * p.rows + m + shift;
                const i32x4* xp = reinterpret_cast<const i32x4*>(p.xc + row * kGroupBytes) + half * 2;
                x0 = xp[0], x1 = xp[1];
                xscale = reinterpret_cast<const uint32_t*>(p.xs)[row];
            }
        }
        // lane l takes, of row l % 32, the blocks 2 * (l / 32) and + 1 in the two steps
        const int ws = wscale >> (half * 16), xs = xscale >> (half * 16);
        acc = step<0>(w0, x0, ws, xs, acc);
        acc = step<1>(w1, x1, ws, xs, acc);
        if (g + WAVES < all) fetch_w(g + WAVES);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[wave][r][8 * (i >> 2) + 4 * half + (i & 3)] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * rows; e += WAVES * 64) {
        const int mm = e >> 5, nn = e & 31;
        if (n0 + nn >= p.n) continue;
        float v = sums[0][mm][nn];
#pragma unroll
        for (int k = 1; k < WAVES; ++k) v += sums[k][mm][nn];
        if (p.bias) v += load_float(p.bias, p.bias_type, n0 + nn);
        store_float(p.y, p.y_type, (int64_t)(m0 + mm) * p.n + n0 + nn, at_least(v, p.least));
    }
}

// ---------------------------------------------------------------------------
// the product, large: tiles staged through LDS
// ---------------------------------------------------------------------------
// A workgroup's tile has TN rows of w and TM of x; a wave multiplies half of the w rows by 64 of x.
// TEAMS: as many such sets of waves share the groups out, each with stages of its own, and add up at the end.
// OWN (X is a float type): the workgroup quantises what its tile reaches of x into LDS before the first product.
constexpr int kHeldUnits = 392;  // pairs of a row and a group: what three workgroups of 128 x 128 find room for
template <int TM, int TN, bool OWN>
struct Tiling {
    static constexpr int kWaves = TM / 32, kThreads = 64 * kWaves, kWt = TN / 64;
    static constexpr int kStages = TM == 256 ? 4 : 3;
    static constexpr int kWavesPerSimd = TN == 128 ? 3 : 2;
    static constexpr int kStagedX = OWN ? 0 : TM;
    // one stage: the codes of one group of every row of w and of x, then their scales
    static constexpr int kW = 0, kX = TN * kGroupBytes, kWs = kX + kStagedX * kGroupBytes, kXs = kWs + TN * 4;
    static constexpr int kStage = kXs + kStagedX * 4;
    // a wave's loads for a stage: pieces of 16 rows of w and x, scales of 64 rows
    static constexpr int kLoadsW = TN / 16 / kWaves, kLoadsX = kStagedX / 16 / kWaves;
    static constexpr int kLoadsS = ((TN + kStagedX) / 64 + kWaves - 1) / kWaves;
    static constexpr int kLoads = kLoadsW + kLoadsX + kLoadsS;
    // OWN: behind the stages the codes of x, a unit of zeros, and their scales
    static constexpr int kHeld = kStages * kStage, kHeldScales = kHeld + (kHeldUnits + 1) * kGroupBytes;
    static constexpr int kBytes = OWN ? kHeldScales + (kHeldUnits + 1) * 4 : kHeld;
    static_assert(kHeld % kGroupBytes == 0, "the two pieces of a lane differ in one bit of their address");
};

template <int FROM, int TO, typename F>
__device__ inline void each(F&& f) {
    if constexpr (FROM < TO) {
        f(std::integral_constant<int, FROM>{});
        each<FROM + 1, TO>(f);
    }
}

// what a lane reads where a tap leaves its entry
__device__ __align__(64) const uint32_t g_zeros[16] = {};

// 16 (or 4) bytes a lane from memory to LDS, lane after lane from the uniform address `dst` on.  Nothing
// waits for these loads but the explicit s_waitcnt before the barrier that hands a stage over.  M0
// holds the LDS address (one wait state before its use).  It is a register that the compiler reserves and warns of in a
// list of clobbers; there it keeps a use of its own, of which these kernels have none now, from spanning a load.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ inline void to_lds(const uint8_t* base, uint32_t offset, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ inline void to_lds(const uint8_t* src, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "m0", "memory");
}

__device__ inline void dword_to_lds(const uint8_t* base, uint32_t offset, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(dst), "v"(offset), "s"(base) : "m0", "memory");
}
__device__ inline void dword_to_lds(const uint8_t* src, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(src) : "m0", "memory");
}
#pragma clang diagnostic pop

template <int WT>
struct Fragments {
    i32x4 w[WT], x[2];
};

// The wave's 32 rows (x) by 32 * WT columns (w) of accumulators through LDS of its own, so that
// a row of y leaves in pieces of 16 bytes.  Lane l holds y[m = l % 32][8 * (e / 4) + 4 * (l / 32)
// + e % 4] of every accumulator; piece q of row m lies at place q ^ m: reads and writes both
// spread over the banks.  `stream`: past the L2.
template <typename T, int WT>
__device__ inline void store_rows(const Product& p, bool stream, const f32x16 (&acc)[WT], const float* bias, uint8_t* lds, int m0, int n0, int lane) {
    constexpr int kPieces = 32 * WT * sizeof(T) / 16, kEach = 16 / sizeof(T);
    const int r = lane & 31, half = lane >> 5;
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            struct __attribute__((aligned(4 * sizeof(T)))) Four {
                T v[4];
            } four;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                four.v[e] = (T)at_least(acc[i][4 * q + e] + bias[i * 32 + 8 * q + 4 * half + e], p.least);
            const int at = (i * 32 + 8 * q + 4 * half) * sizeof(T);
            *reinterpret_cast<Four*>(lds + r * (kPieces * 16) + (((at >> 4) ^ (r & (kPieces - 1))) << 4) + (at & 15)) = four;
        }
    wave_lds_fence();
    constexpr int kRows = 64 / kPieces;  // rows that one instruction covers
    const int piece = lane % kPieces, sub = lane / kPieces;
    const int n = n0 + piece * kEach;
    T* y = static_cast<T*>(p.y) + (int64_t)(m0 + sub) * p.n + n;
    auto own = [&](int row) {
        return *reinterpret_cast<const i32x4*>(lds + row * (kPieces * 16) + ((piece ^ (row & (kPieces - 1))) << 4));
    };
    if (m0 + 32 <= p.rows && n0 + 32 * WT <= p.n) {
        // The empty statements keep the compiler from joining the two loops, which would drop the hint.
        if (stream) {
            asm volatile("; past the L2");
#pragma unroll
            for (int k = 0; k < 32; k += kRows)
                __builtin_nontemporal_store(own(k + sub), reinterpret_cast<Unaligned<T>*>(y + (int64_t)k * p.n));
            asm volatile("; past the L2");
        } else {
#pragma unroll
            for (int k = 0; k < 32; k += kRows) store_16(y + (int64_t)k * p.n, own(k + sub));
        }
        return;
    }
#pragma unroll 1
    for (int k = 0; k < 32; k += kRows) {
        if (m0 + k + sub >= p.rows) break;
        struct {
            T v[kEach];
        } v = __builtin_bit_cast(decltype(v), own(k + sub));
        T* at = y + (int64_t)k * p.n;
        if (n + kEach <= p.n) {
            store_16(at, __builtin_bit_cast(i32x4, v));
        } else {
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                if (n + e < p.n) at[e] = v.v[e];
        }
    }
}

template <int N>
__device__ inline void arrive_and_wait() {  // all but the N youngest loads are here, and every wave is
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Each wave multiplies 32 * WT rows of w by 64 of x (WT x 2 accumulators of 32 x 32); two waves share
// the rows of x.  A stage holds one group of both operands: [row][4 pieces of 16 bytes], piece q of row
// r at place q ^ (r / 4 % 4): sixteen lanes that read one piece of sixteen rows then touch each of the
// 64 banks once.  One stage is multiplied while the others are on their way.  A stage is two steps; the
// barrier stands early in the second, whose products hide the first reads of the next stage.
template <typename X, bool CONV, int TM, int TN, int TEAMS>
__global__ __launch_bounds__((Tiling<TM, TN, !std::is_void_v<X>>::kThreads * TEAMS), (TEAMS > 1 ? 2 : Tiling<TM, TN, !std::is_void_v<X>>::kWavesPerSimd)) void product_tiled_kernel(Product p) {
    constexpr bool OWN = !std::is_void_v<X>;
    using L = Tiling<TM, TN, OWN>;
    constexpr int WT = L::kWt;
    __shared__ __align__(1024) uint8_t lds[L::kBytes * TEAMS];
    __shared__ __align__(16) float bias[TN];
    const int lane = threadIdx.x & 63, id = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int team = TEAMS > 1 ? id / L::kWaves : 0, wave = id - team * L::kWaves;
    const int r = lane & 31, half = lane >> 5;
    const int m_tiles = (p.rows + TM - 1) / TM, n_tiles = (p.n + TN - 1) / TN;
    const Tile tile = tile_of(blockIdx.x, gridDim.x, m_tiles, n_tiles);
    const int n0 = tile.n * TN, m0 = tile.m * TM;
    // the team's groups: g0 .. g0 + all - 1
    const int longest = (p.taps * p.groups + TEAMS - 1) / TEAMS, g0 = team * longest;
    const int all = TEAMS > 1 ? min(longest, p.taps * p.groups - g0) : longest;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + team * L::kBytes;

    // Load i of a wave fills 16 rows from (i * waves + wave) * 16 on, lane l the place l % 4 of row l / 4.
    // Rows behind the last repeat it.
    const int place = ((lane & 3) ^ (lane >> 4)) * 16;
    uint32_t woff[L::kLoadsW], xoff[OWN ? 1 : L::kLoadsX], soff[L::kLoadsS];
    int xt[OWN ? 1 : L::kLoadsX], st = 0;
#pragma unroll
    for (int i = 0; i < L::kLoadsW; ++i)
        woff[i] = min(n0 + (i * L::kWaves + wave) * 16 + (lane >> 2), p.n - 1) * p.taps * kGroupBytes + place;
#pragma unroll
    for (int i = 0; i < L::kLoadsX; ++i) {
        const int m = min(m0 + (i * L::kWaves + wave) * 16 + (lane >> 2), p.rows - 1);
        xoff[i] = m * kGroupBytes + place;
        xt[i] = CONV ? m % p.T : 0;
    }
    // Scales, 64 rows a load: with one load a wave the first TN / 64 waves bring w's, the others x's; with two
    // every wave brings w's and then x's (four waves for two loads of x: two of them the same).
    const bool first_w = OWN || L::kLoadsS == 2 || wave < TN / 64;
    const int swave = OWN ? wave & (TN / 64 - 1) : wave;
    if constexpr (OWN) {
        soff[0] = min(n0 + swave * 64 + lane, p.n - 1) * p.taps * 4;
    } else {
        const int m = min(m0 + (L::kLoadsS == 1 ? wave - TN / 64 : wave & (TM / 64 - 1)) * 64 + lane, p.rows - 1);
        if (first_w) soff[0] = min(n0 + wave * 64 + lane, p.n - 1) * p.taps * 4;
        if (!first_w || L::kLoadsS == 2) {
            soff[L::kLoadsS - 1] = m * 4;
            st = CONV ? m % p.T : 0;
        }
    }
    // the next stage to be loaded: tap, group, and where their rows begin (counted in rows)
    int tap = TEAMS > 1 && CONV ? g0 / p.groups : 0, gx = g0 - tap * p.groups;
    const int64_t wstep = (int64_t)p.n * p.taps;
    int64_t wrow = gx * wstep + tap, xrow = (int64_t)gx * p.rows;
    // first scale load of this wave: base, bytes to the current group, bytes of a group
    const uint8_t* sbase = first_w ? p.ws : p.xs;
    const int64_t sstep = (first_w ? wstep : p.rows) * 4;
    int64_t sat = gx * sstep;
    // the loads in order: w, x, scales; after the last one on to the next group; no branches
    auto stage_part = [&](int slot, auto part) {
        constexpr int i = part, xi = i - L::kLoadsW, si = xi - L::kLoadsX;
        const uint32_t dst = lds0 + slot * L::kStage;
        const int shift = CONV ? tap * p.dilation - p.left : 0;
        const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_zeros);
        if constexpr (i < L::kLoadsW) {
            to_lds(p.wc + wrow * kGroupBytes, woff[i], dst + L::kW + (i * L::kWaves + wave) * 1024);
        } else if constexpr (xi < L::kLoadsX) {
            const uint8_t* xbase = p.xc + xrow * kGroupBytes;
            const uint32_t to = dst + L::kX + (xi * L::kWaves + wave) * 1024;
            if (CONV) {
                const bool inside = (unsigned)(xt[xi] + shift) < (unsigned)p.T;
                to_lds(inside ? xbase + (int64_t)xoff[xi] + (int64_t)shift * kGroupBytes : zeros, to);
            } else {
                to_lds(xbase, xoff[xi], to);
            }
        } else {
            // with one load a wave, x's scales follow w's as the waves follow each other
            const bool of_w = OWN || (L::kLoadsS == 1 ? first_w : si == 0);
            const uint32_t to = dst + (si == 0 ? L::kWs + swave * 256 : L::kXs + (wave & (TM / 64 - 1)) * 256);
            const uint8_t* from = si == 0 ? sbase + sat : p.xs + xrow * 4;
            if (CONV) {
                // of w the tap's own scales; of x those of the shifted row
                const int own = of_w ? tap : shift;
                const bool inside = of_w | ((unsigned)(st + shift) < (unsigned)p.T);
                dword_to_lds(inside ? from + (int64_t)soff[si] + (int64_t)own * 4 : zeros, to);
            } else {
                dword_to_lds(from, soff[si], to);
            }
        }
        if constexpr (i == L::kLoads - 1) {
            const bool last = CONV && gx == p.groups - 1;
            if (CONV) tap += last;
            gx = last ? 0 : gx + 1;
            wrow = last ? tap : wrow + wstep;
            xrow = last ? 0 : xrow + p.rows;
            sat = last ? 0 : sat + sstep;
        }
    };

#pragma unroll
    for (int c = 0; c < L::kStages; ++c)
        if (c < all) each<0, L::kLoads>([&](auto part) { stage_part(c, part); });
    const int nw = (wave & 1) * 32 * WT, mw = (wave >> 1) * 64;
    // OWN: where this lane's two rows of x lie, and the unit that the next reads of them come from (its first
    // piece; the second is the neighbour)
    int xi[2] = {}, xe[2] = {}, span = 0;
    uint32_t xat[2] = {};
    int rtap = 0, rgx = 0;
    auto seek = [&]() {
        const int shift = CONV ? rtap * p.dilation - p.left : 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const bool inside = !CONV || (unsigned)(xe[j] + shift) < (unsigned)p.T;
            const int i = xi[j] + shift, unit = inside ? rgx * span + i : kHeldUnits;
            xat[j] = L::kHeld + unit * kGroupBytes + ((half * 2 ^ (i >> 2)) & 3) * 16;
        }
    };
    if constexpr (OWN) {
        const int first = max(m0 - p.left, 0);
        span = min(min(m0 + TM, p.rows) - 1 + (p.taps - 1) * p.dilation - p.left, p.rows - 1) - first + 1;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int m = min(m0 + mw + j * 32 + r, p.rows - 1);
            xi[j] = m - first, xe[j] = CONV ? m % p.T : 0;
        }
        quantise_rows<X, L::kThreads>(p, first, span, reinterpret_cast<uint32_t*>(lds + L::kHeld), lds + L::kHeldScales);
        if (threadIdx.x < kGroupBytes / 4) reinterpret_cast<uint32_t*>(lds + L::kHeld + kHeldUnits * kGroupBytes)[threadIdx.x] = 0;
        if (threadIdx.x == 0) reinterpret_cast<uint32_t*>(lds + L::kHeldScales)[kHeldUnits] = 0;
        seek();
    }
    // asked for here, used behind the loop: no wait of its own
    static_assert(L::kThreads >= TN, "a thread for every bias");
    float own_bias = 0.f;
    if (p.bias && n0 + (int)threadIdx.x < p.n && threadIdx.x < TN) own_bias = load_float(p.bias, p.bias_type, n0 + threadIdx.x);

    // lane l takes, of row l % 32, the blocks 2 * (l / 32) and + 1 in the two steps
    uint32_t at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) at[k] = ((half * 2 + k) ^ ((r >> 2) & 3)) * 16;
    const uint32_t first_byte = team * L::kBytes;
    const uint32_t wr = first_byte + L::kW + (nw + r) * kGroupBytes, xr = first_byte + L::kX + (mw + r) * kGroupBytes;
    // the reads of a step in the order of their use: w0 x0 w1 .. x1
    constexpr int kReads = WT + 2, kProducts = WT * 2;
    auto fetch = [&](uint32_t base, int k, auto q, Fragments<WT>& f) {
        constexpr bool x = q == 1 || q == WT + 1;
        constexpr int i = q == 0 ? 0 : x ? q / (WT + 1) : q - 1;
        const uint32_t from = OWN && x ? xat[x ? i : 0] ^ (k * 16) : base + (x ? xr : wr) + at[k] + i * 32 * kGroupBytes;
        const i32x4 v = *reinterpret_cast<const i32x4*>(lds + from);
        if constexpr (x)
            f.x[i] = v;
        else
            f.w[i] = v;
    };
    int ws[WT], xs[2], wnext[WT], xnext[2];
    const uint32_t wsr = first_byte + L::kWs + (nw + r) * 4, xsr = first_byte + L::kXs + (mw + r) * 4;
    auto fetch_scales = [&](uint32_t base) {
#pragma unroll
        for (int i = 0; i < WT; ++i) wnext[i] = *reinterpret_cast<const int*>(lds + base + wsr + i * 128);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            xnext[j] = *reinterpret_cast<const int*>(lds + (OWN ? L::kHeldScales + (xat[j] - L::kHeld) / kGroupBytes * 4 : base + xsr + j * 128));
    };
    f32x16 acc[WT][2] = {};
    auto multiply = [&](auto S, auto q, const Fragments<WT>& f) {
        constexpr int i = q % WT, j = q / WT;
        acc[i][j] = step<S>(f.w[i], f.x[j], ws[i], xs[j], acc[i][j]);
    };

    Fragments<WT> fa, fb;
    if (all >= L::kStages)
        arrive_and_wait<(L::kStages - 1) * L::kLoads>();
    else
        arrive_and_wait<0>();
    each<0, kReads>([&](auto q) { fetch(0, 0, q, fa); });
    fetch_scales(0);
    int slot = 0;
    uint32_t base = 0;
    auto chunk = [&](auto more) {
        // the dword holds the group's four blocks: this lane's two go to the front
#pragma unroll
        for (int i = 0; i < WT; ++i) ws[i] = (uint32_t)wnext[i] >> (half * 16);
#pragma unroll
        for (int j = 0; j < 2; ++j) xs[j] = (uint32_t)xnext[j] >> (half * 16);
        // What is not a product is issued in the shadow of one (32 cycles each): the waves of a SIMD may come
        // through here together, so nothing else would keep the matrix core busy meanwhile.
        constexpr std::integral_constant<int, 0> first{};
        constexpr std::integral_constant<int, 1> second{};
        __builtin_amdgcn_sched_barrier(0);
        each<0, kProducts>([&](auto q) {
            multiply(first, q, fa);
            __builtin_amdgcn_sched_barrier(0);
            each<2 * q, (2 * q + 2 < kReads ? 2 * q + 2 : kReads)>([&](auto i) { fetch(base, 1, i, fb); });
            __builtin_amdgcn_sched_barrier(0);
        });
        const int freed = slot;
        each<0, kProducts>([&](auto q) {
            multiply(second, q, fb);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (q == 1) {
                // the next stage has arrived (younger ones may be under way), and this one has been read, everywhere
                if constexpr (more)
                    arrive_and_wait<(L::kStages - 2) * L::kLoads>();
                else
                    arrive_and_wait<0>();
                slot = slot == L::kStages - 1 ? 0 : slot + 1;
                base = slot * L::kStage;
                if constexpr (OWN) {
                    rgx = rgx == p.groups - 1 ? 0 : rgx + 1;
                    if (CONV) rtap = rgx > 0 ? rtap : rtap == p.taps - 1 ? 0 : rtap + 1;
                    seek();
                }
            }
            // then the next stage's first reads (behind the last stage: of whatever lies there, and nothing
            // uses them), its scales, and the loads into the stage that is free now, over the products left
            constexpr int kScales = 1 + kReads / 2 < kProducts - 2 ? 1 + kReads / 2 : kProducts - 2, kLeft = kProducts - 1 - kScales;
            if constexpr (q >= 1) each<2 * (q - 1), (2 * q < kReads ? 2 * q : kReads)>([&](auto i) { fetch(base, 0, i, fa); });
            if constexpr (q == kScales) fetch_scales(base);
            if constexpr (more && q > kScales) {
                constexpr int n = q - kScales - 1;
                each<n * L::kLoads / kLeft, (n + 1) * L::kLoads / kLeft>([&](auto part) { stage_part(freed, part); });
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // two loops, each without a branch inside: products stay on their side of the barrier
    int c = 0;
    for (; c < all - L::kStages; ++c) chunk(std::true_type{});
    for (; c < all; ++c) chunk(std::false_type{});
    if (TEAMS > 1 && all < longest) arrive_and_wait<0>();  // the other team's last barrier

    if (threadIdx.x < TN) bias[threadIdx.x] = own_bias;
    __syncthreads();
    // every read of the stages lies behind: each wave takes a part of them
    constexpr int kOwn = 32 * 32 * WT * 4;
    static_assert(L::kWaves * kOwn <= L::kBytes, "the stages (and x) hold the waves' parts of y");
    uint8_t* own = lds + id * kOwn;
    // The smaller tiles, whose y is most of the traffic, store it past the L2 where its rows are whole lines
    // (us, 30000 x 1024 x 1000: 28.2 against 31.0 through the L2, 55360 x 256 x 768: 13.9 against 15.8; but rows of 1000,
    // which share lines: 35.3 against 32.3, and 28.6 against 17.6 for 30000 x 1000 x 128).  The largest leaves L2 to
    // the operands and y alike (8192 x 8192 x 1024: 66 past it, 62 through it).
    const int y_size = p.y_type == GLV_F32 ? 4 : 2;
    const bool stream = TM == 128 && ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)p.n * y_size) & 127) == 0;
    // 32 rows of the wave's 64: of two teams each takes its half of both sums
    auto finish = [&](auto J) {
        constexpr int j = J;
        f32x16 part[WT];
#pragma unroll
        for (int i = 0; i < WT; ++i) part[i] = acc[i][j];
        if constexpr (TEAMS > 1) {
            f32x4* const to = reinterpret_cast<f32x4*>(own);
            const f32x4* const from = reinterpret_cast<const f32x4*>(lds + (id ^ L::kWaves) * kOwn);
#pragma unroll
            for (int i = 0; i < WT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    to[(i * 4 + q) * 64 + lane] = f32x4{acc[i][1 - j][4 * q], acc[i][1 - j][4 * q + 1], acc[i][1 - j][4 * q + 2], acc[i][1 - j][4 * q + 3]};
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 v = from[(i * 4 + q) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[i][4 * q + e] += v[e];
                }
            __syncthreads();
        }
        if (p.y_type == GLV_F32)
            store_rows<float>(p, stream, part, bias + nw, own, m0 + mw + j * 32, n0 + nw, lane);
        else if (p.y_type == GLV_BF16)
            store_rows<bf16>(p, stream, part, bias + nw, own, m0 + mw + j * 32, n0 + nw, lane);
        else
            store_rows<f16>(p, stream, part, bias + nw, own, m0 + mw + j * 32, n0 + nw, lane);
        wave_lds_fence();
    };
    if (TEAMS == 1 || team == 0) finish(std::integral_constant<int, 0>{});
    if (TEAMS == 1 || team == 1) finish(std::integral_constant<int, 1>{});
}

template <int TM, int TN, int TEAMS = 1, typename X = void>
int launch_tiled(const Product& p, hipStream_t st) {
    using L = Tiling<TM, TN, !std::is_void_v<X>>;
    const unsigned tiles = (unsigned)((p.rows + TM - 1) / TM) * (unsigned)((p.n + TN - 1) / TN);
    return launch("product_tiled_kernel", p.taps > 1 ? product_tiled_kernel<X, true, TM, TN, TEAMS> : product_tiled_kernel<X, false, TM, TN, TEAMS>,
                  dim3(tiles), dim3(L::kThreads * TEAMS), 0, st, p);
}

// rows sixteen at a time by groups four at a time
int64_t span_blocks(int rows, int groups) { return (int64_t)((rows + 15) / 16) * ((groups + 3) / 4); }

int quantise(const char* what, const void* x, int type, Rows xr, int rows, int cols, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const int groups = (cols + kGroup - 1) / kGroup;
    const int64_t blocks = span_blocks(rows, groups);
    if (too_large(blocks, 256)) return report(GLV_ERR_INVALID, "%s: rows x columns too large for one call", what);
    const dim3 grid((unsigned)blocks), block(256);
    auto run = [&](auto* typed) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(typed)>>;
        return launch("quantise_kernel", cols < 8 ? quantise_kernel<T, true> : quantise_kernel<T, false>, grid, block, 0, st, typed, xr, rows,
                      cols, groups, codes, scales);
    };
    if (type == GLV_F32) return run(static_cast<const float*>(x));
    return type == GLV_BF16 ? run(static_cast<const bf16*>(x)) : run(static_cast<const f16*>(x));
}

// Rows of x that one tile of `tile` rows of y reaches, at most.
int64_t reached_rows(int64_t rows, int tile, int taps, int dilation) {
    const int64_t span = tile + (int64_t)(taps - 1) * dilation;
    return span < rows ? span : rows;
}

// Four waves where there are no more groups than that, else eight.
template <typename X>
int launch_direct(const Product& p, unsigned tiles, hipStream_t st) {
    const size_t held = std::is_void_v<X> ? 0 : reached_rows(p.rows, 32, p.taps, p.dilation) * p.groups * (kGroupBytes + 4);
    const bool few = p.taps * p.groups <= 4;
    return launch("product_direct_kernel", few ? product_direct_kernel<X, 4> : product_direct_kernel<X, 8>, dim3(tiles), dim3(few ? 256 : 512),
                  held, st, p);
}

// The tile in which a product quantises its activations itself (columns of y; 0: it does not): every tile
// does so anew with the rows it reaches, against a launch and a workspace less (us, bfloat16, device).
// 32 x 32, while those are at most 256 pairs of a row and a group (32 x 4096 x 1024, 256 pairs, 5.7 against 5.8
// in two launches; 32 x 1024 x 2048, 512 pairs, 8.2 against 6.3; 165 rows, 256 -> 256, 5 taps, 80 pairs, 4.2
// against 5.6) and at most 8 M elements in all tiles together (865 x 256 x 1024, 7 M, 5.8 against 6.6; 2000 x 500 x
// 500, 16 M, 9.7 against 7.9).
// 128 x 128 and 128 x 256, where one tile spans w's rows, so that x is still read once, and x fits beside the
// stages: for narrow w from a tile a CU on (55360 x 80 x 256: 12.9 against 15.3, 120000 x 128 x 384: 26.0 against 30.6;
// 16384 x 80 x 256: 10.4 against 9.1), for wider w in one round of two a CU (55360 rows, 256 -> 256, 3 taps: 19.3
// against 21.3, 65500 x 256 x 384: 18.7 against 22.4; 32768 x 200 x 384: 17.9 against 16.4, 120000 x 200 x 384: 40.4
// against 38.2), for a workgroup's reading, multiplying and writing follow each other.
int own_tile(int64_t rows, int cols, int n_out, int taps, int dilation) {
    if (cols < 8) return 0;
    const int64_t groups = (cols + kGroup - 1) / kGroup, pairs = reached_rows(rows, 32, taps, dilation) * groups;
    const int64_t tiles = ((rows + 31) / 32) * ((n_out + 31) / 32), high = (rows + 127) / 128;
    if (pairs <= 256 && tiles * pairs * kGroup <= (int64_t)8 << 20) return 32;
    if (reached_rows(rows, 128, taps, dilation) * groups > kHeldUnits) return 0;
    if (n_out <= 128) return high >= 256 ? 128 : 0;
    return n_out <= 256 && high > 384 && high <= 512 ? 256 : 0;
}

// Row counts and widths are ints in the kernels, row * groups is formed in 64 bits, and every
// launch counts its workgroups in one dimension: these limits keep all of that in range.
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

// What both directions ask of an array; GLV_OK with *all = 0: nothing to do.
static int check_array(const char* what, const glv_mxfp4_array* a, int64_t* all) {
    if (!a) return report(GLV_ERR_INVALID, "%s: null argument", what);
    if (a->batch < 0 || a->rows < 0) return report(GLV_ERR_INVALID, "%s: negative batch or rows", what);
    *all = (int64_t)a->batch * a->rows;
    const int rc = check_shape(what, *all, a->cols);
    if (rc != GLV_OK) return rc;
    if (!float_type(a->type)) return report(GLV_ERR_INVALID, "%s: unknown element type %d", what, a->type);
    if (*all == 0) return GLV_OK;
    if (!a->data_dev || !a->codes_dev || !a->scales_dev) return report(GLV_ERR_INVALID, "%s: null argument", what);
    if (misaligned(a->data_dev, a->type == GLV_F32 ? 4 : 2)) return report(GLV_ERR_INVALID, "%s: data is not aligned to its elements", what);
    return check_quantised(what, a->codes_dev, a->scales_dev);
}

extern "C" int glv_mxfp4_quantize(const glv_mxfp4_array* a, void* stream) {
    const char* what = "glv_mxfp4_quantize";
    int64_t all = 0;
    const int rc = check_array(what, a, &all);
    if (rc != GLV_OK || all == 0) return rc;
    return quantise(what, a->data_dev, a->type, Rows{a->batch_stride, a->row_stride, a->rows, a->batch == 1}, (int)all, a->cols,
                    a->codes_dev, a->scales_dev, (hipStream_t)stream);
}

extern "C" int glv_mxfp4_dequantize(const glv_mxfp4_array* a, void* stream) {
    const char* what = "glv_mxfp4_dequantize";
    int64_t all = 0;
    const int rc = check_array(what, a, &all);
    if (rc != GLV_OK || all == 0) return rc;
    const int rows = (int)all, cols = a->cols, out_type = a->type;
    const uint8_t *codes_dev = a->codes_dev, *scales_dev = a->scales_dev;
    void* out_dev = a->data_dev;
    const int groups = (cols + kGroup - 1) / kGroup;
    const int64_t blocks = span_blocks(rows, groups);
    if (too_large(blocks, 256)) return report(GLV_ERR_INVALID, "%s: rows x columns too large for one call", what);
    const dim3 grid((unsigned)blocks), block(256);
    hipStream_t st = (hipStream_t)stream;
    auto run = [&](auto* typed) {
        using T = std::remove_pointer_t<decltype(typed)>;
        return launch("dequantise_kernel", dequantise_kernel<T>, grid, block, 0, st, codes_dev, scales_dev, rows, cols, groups, typed);
    };
    if (out_type == GLV_F32) return run((float*)out_dev);
    return out_type == GLV_BF16 ? run((bf16*)out_dev) : run((f16*)out_dev);
}

// The sizes and the type of x; GLV_OK with *all rows.
static int check_product(const char* what, const glv_mxfp4_product_args& a, int64_t* all) {
    if (a.batch < 0 || a.rows < 0) return report(GLV_ERR_INVALID, "%s: negative batch or rows", what);
    *all = (int64_t)a.batch * a.rows;
    const int rc = check_shape(what, *all, a.cols);
    if (rc != GLV_OK) return rc;
    if (a.n_out < 0 || a.n_out > kMaxCols) return report(GLV_ERR_INVALID, "%s: n_out %d outside [0, %d]", what, a.n_out, kMaxCols);
    if (a.taps < 1 || a.dilation < 1 || (int64_t)a.taps * a.cols > kMaxCols || (int64_t)a.n_out * a.taps > kMaxRows ||
        (int64_t)(a.taps - 1) * a.dilation > kMaxRows)
        return report(GLV_ERR_INVALID, "%s: taps %d and dilation %d must be positive, taps x columns at most %d, "
                      "n_out x taps and (taps - 1) x dilation at most %lld", what, a.taps, a.dilation, kMaxCols, (long long)kMaxRows);
    if (!float_type(a.x_type) && a.x_type != GLV_MXFP4) return report(GLV_ERR_INVALID, "%s: unknown element type %d of x", what, a.x_type);
    // what a launch holds: the quantiser's rows, and tiles of 128 x 128 by 256 threads (the larger ones are fewer, by more)
    if ((a.x_type != GLV_MXFP4 && too_large(span_blocks((int)*all, (a.cols + kGroup - 1) / kGroup), 256)) ||
        too_large(((*all + 127) / 128) * ((a.n_out + 127) / 128), 256))
        return report(GLV_ERR_INVALID, "%s: rows x columns or rows x n_out too large for one call", what);
    return GLV_OK;
}

extern "C" int64_t glv_mxfp4_product_workspace(const glv_mxfp4_product_args* a) {
    const char* what = "glv_mxfp4_product_workspace";
    if (!a) return report(GLV_ERR_INVALID, "%s: null argument", what);
    int64_t all = 0;
    if (check_product(what, *a, &all) != GLV_OK) return -1;
    if (a->x_type == GLV_MXFP4 || own_tile(all, a->cols, a->n_out, a->taps, a->dilation)) return 0;
    return quantised_bytes(all, (a->cols + kGroup - 1) / kGroup);
}

extern "C" int glv_mxfp4_product(const glv_mxfp4_product_args* a, void* workspace_dev, int64_t workspace_bytes, void* stream) {
    const char* what = "glv_mxfp4_product";
    if (!a) return report(GLV_ERR_INVALID, "%s: null argument", what);
    const auto [x_dev, x_scales_dev, w_codes_dev, w_scales_dev, bias_dev, y_dev, x_batch_stride, x_row_stride, x_type, batch, rows, cols,
                n_out, taps, dilation, bias_type, activation, y_type] = *a;
    int64_t all = 0;
    int rc = check_product(what, *a, &all);
    if (rc != GLV_OK) return rc;
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
    p.bias = bias_dev, p.bias_type = bias_type, p.least = activation == GLV_ACT_RELU ? 0.f : -__builtin_huge_valf();
    p.y = y_dev, p.y_type = y_type;
    const int64_t tiles = ((all + 31) / 32) * (int64_t)((n_out + 31) / 32);
    if (x_type == GLV_MXFP4) {
        rc = check_quantised(what, x_dev, x_scales_dev);
        if (rc != GLV_OK) return rc;
        p.xc = static_cast<const uint8_t*>(x_dev), p.xs = x_scales_dev;
    } else if (const int tile = own_tile(all, cols, n_out, taps, dilation)) {
        p.x = x_dev, p.xr = Rows{x_batch_stride, x_row_stride, rows, batch == 1}, p.cols = cols;
        auto run = [&](auto* typed) {
            using X = std::remove_pointer_t<decltype(typed)>;
            if (tile == 256) return launch_tiled<128, 256, 1, X>(p, st);
            if (tile == 128) return launch_tiled<128, 128, 1, X>(p, st);
            return launch_direct<X>(p, (unsigned)tiles, st);
        };
        if (x_type == GLV_F32) return run((float*)nullptr);
        return x_type == GLV_BF16 ? run((bf16*)nullptr) : run((f16*)nullptr);
    } else {
        const int64_t need = quantised_bytes(all, p.groups);
        if (!workspace_dev || workspace_bytes < need)
            return report(GLV_ERR_INVALID, "%s: workspace of %lld bytes, %lld needed (glv_mxfp4_product_workspace)", what,
                          (long long)(workspace_dev ? workspace_bytes : 0), (long long)need);
        if (misaligned(workspace_dev, 16)) return report(GLV_ERR_INVALID, "%s: the workspace is not 16-byte aligned", what);
        uint8_t* codes = static_cast<uint8_t*>(workspace_dev);
        uint8_t* scales = codes + all * p.groups * kGroupBytes;
        rc = quantise(what, x_dev, x_type, Rows{x_batch_stride, x_row_stride, rows, batch == 1}, p.rows, cols, codes, scales, st);
        if (rc != GLV_OK) return rc;
        p.xc = codes, p.xs = scales;
    }
    // Which tile, measured in us with x and y in bfloat16, quantising x included (in brackets without it):
    //                            32 x 32    128 x 128     128 x 256     256 x 256   (rows of x times rows of w)
    //    1000 x 1000 x 1024        (5.6)        (6.7)        (12.0)        (13.7)
    //    2048 x 2048 x 4096       (36.8)   19.4 (12.9)   26.6 (20.2)   32.5 (25.9)
    //    2304 x 4096 x 4096                35.5 (28.3)   39.3 (32.2)   34.8 (28.1)
    //   16384 x  256 x 1024       (15.3)   15.1 ( 8.2)   17.4 (10.1)   19.7 (12.2)
    //   20000 x  512 x 1024                30.2 (11.1)   22.7 (12.7)   23.8 (14.3)
    //   55360 x  256 x  512       (24.2)   29.7 (12.8)   23.5 (10.9)   25.1 (12.9)
    //   30000 x  640 x 1024                35.1 (18.9)   38.6 (24.7)
    //   10560 x 2048 x  512                19.8 (14.6)   22.2 (17.6)   25.8 (19.9)
    //   10560 x 4096 x 1024       (94.9)   64.4 (39.7)   47.2 (39.1)   55.3 (45.5)
    //   10560 x 2048 x 4096                71.9 (54.8)   71.6 (54.4)   77.5 (60.1)
    //    8192 x 8192 x 1024                73.0 (56.3)   62.1 (55.7)   78.9 (73.0)
    //    4096 x 4096 x 4096                49.3 (41.2)   47.2 (39.7)   45.3 (37.3)
    // 32 x 32 spreads small outputs over the chip, and takes about 3 us and 0.27 for a thousand tiles and groups; a
    // workgroup of 128 x 128 and two teams alone on its CU 5 and 0.2 a group: the rule below fits where the two meet
    // (1700 tiles of 32 x 32 for two groups, 1300 for seven, 1100 for 19, 1000 for 64: 283 x 4812 x 2061, 1359 tiles,
    // 9.8 us against 8.7; 960 tiles, 158 x 6144 x 1749, 6.8 against 7.6; 1163 x 1807 x 160, 2109 tiles, 6.6 against 6.1).
    // The hyperbola through those four points stands for no law of the card: near it the two forms are within about a tenth of each
    // other, so that a card with another clock moves the border and costs no more than that.
    // Two teams a tile, while there is a CU for every tile: a wave a SIMD alone reaches half the rate (340 x 7567 x
    // 5126, 180 tiles: 16.4 us against 19.2 with one team, 15164 x 151 x 490, 238 tiles, 6.9 against 7.6; 18227 x 187 x
    // 1375, 286 tiles, 13.7 against 11.3).  So too for a single group, of which the second team multiplies none: twice the
    // waves convert and store y (2100 x 1000 x 128 7.4 against 7.8, 8000 x 500 x 128 8.8 and 9.1, 4096 x 1024 x 64 8.0 and 7.8).
    // 128 x 128 has three workgroups on a CU to hide each other's ends, but reads twice the LDS bytes of the larger
    // tiles for a product, and where it follows a kernel bound by memory its draw makes the card lower its clock
    // (10560 x 4096 x 1024: 38 us of zeros, 64 of random values; 41 and 47 for 128 x 256).  So sums of some length take
    // 128 x 256, if it leaves no CU without work and does not reach much past w's rows, and so do shorter ones
    // that it finishes in one round of two workgroups a CU.  Long sums take the largest where its rounds, of one
    // workgroup a CU, are no longer than those of 128 x 256, half as much each.
    const int64_t groups = (int64_t)p.taps * p.groups;
    if ((tiles - 940) * (2 * groups + 5) > 6800) {
        const int64_t rows128 = (all + 127) / 128, narrow = rows128 * ((n_out + 127) / 128), mid = rows128 * ((n_out + 255) / 256);
        const int64_t wide = ((all + 255) / 256) * ((n_out + 255) / 256);
        if (groups >= 32 && 2 * ((wide + 255) / 256) <= (mid + 255) / 256) return launch_tiled<256, 256>(p, st);
        if (32 * mid <= 17 * narrow && (groups >= 8 ? mid >= 256 : mid > 384 && mid <= 512)) return launch_tiled<128, 256>(p, st);
        if (narrow <= 256) return launch_tiled<128, 128, 2>(p, st);
        return launch_tiled<128, 128>(p, st);
    }
    return launch_direct<void>(p, (unsigned)tiles, st);
}
