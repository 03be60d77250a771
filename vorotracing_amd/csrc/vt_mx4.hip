// vt_mx4.hip -- rows in 4 bits (mx4, include/vt_micro_abi.h): quantisation,
// the way back, the product of two such matrices and a head of such layers.
#include "vt_micro.h"

namespace vt {

constexpr int MX_THREADS = 256;

// Eight values a thread, the four threads of a block side by side: the
// block's largest magnitude takes two exchanges in the group of four.
template <typename T>
__global__ __launch_bounds__(MX_THREADS) void mx4_quantize_kernel(const T *__restrict__ x, int64_t x_stride,
                                                                  uint64_t groups, uint32_t width,
                                                                  uint8_t *__restrict__ codes,
                                                                  uint8_t *__restrict__ scales)
{
    const uint64_t at = (uint64_t)blockIdx.x * MX_THREADS + threadIdx.x;
    if (at >= groups) // whole groups of four threads: `groups` is a multiple of 4
        return;
    const uint32_t per_row = 4 * mx_blocks(width);
    const uint64_t row = at / per_row;
    const uint32_t k = (uint32_t)(at - row * per_row) * 8;
    Mx4Piece<T> v;
    v.load(x + (int64_t)row * x_stride + k, k < width ? width - k : 0);
    uint32_t top = 0;
    v.top(top);
    top = v.top_bits(top);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 4));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 4));
    const uint32_t c = mx4_scale(top);
    const uint32_t word = c == MX_NAN ? 0 : v.word(e8m0_value(c));
    reinterpret_cast<uint32_t *>(codes)[at] = word;
    if ((threadIdx.x & 3) == 0)
        scales[at / 4] = (uint8_t)c;
}

__device__ __forceinline__ float e2m1_value(uint32_t code)
{
    // 0, 1/2, 1, 3/2, 2, 3, 4, 6: a float's exponent and top bit, with the subnormal 1/2 apart
    const uint32_t m = code & 7;
    const float a = m < 2 ? 0.5f * (float)m : __builtin_bit_cast(float, ((m >> 1) + 126) << 23 | (m & 1) << 22);
    return code & 8 ? -a : a;
}

template <typename T>
__global__ __launch_bounds__(MX_THREADS) void mx4_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                                    const uint8_t *__restrict__ scales,
                                                                    uint64_t groups, uint32_t width,
                                                                    T *__restrict__ out)
{
    const uint64_t at = (uint64_t)blockIdx.x * MX_THREADS + threadIdx.x;
    if (at >= groups)
        return;
    const uint32_t per_row = 4 * mx_blocks(width);
    const uint64_t row = at / per_row;
    const uint32_t k = (uint32_t)(at - row * per_row) * 8;
    if (k >= width)
        return;
    const uint32_t word = reinterpret_cast<const uint32_t *>(codes)[at];
    const float s = e8m0_value(scales[at / 4]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = e2m1_value(word >> (4 * i) & 15) * s;
    store_upto8(out + row * width + k, width - k, v);
}

// One wave a tile of 32 rows of x by 32 of w, both read where they lie: a
// lane's operand of the 32x32x64 product is one block of 32 codes of one row,
// 16 bytes, with its scale.  w is the first operand, so that a lane ends with
// runs of four neighbouring outputs of one row.
template <typename Y>
__global__ __launch_bounds__(64) void mx4_linear_kernel(const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs,
                                                        uint64_t rows, uint32_t blocks,
                                                        const uint8_t *__restrict__ w, const uint8_t *__restrict__ ws,
                                                        uint32_t out, const float *__restrict__ bias, int relu,
                                                        Y *__restrict__ y)
{
    const uint32_t tiles_n = (out + 31) / 32;
    const uint64_t m0 = (uint64_t)(blockIdx.x / tiles_n) * 32;
    const uint32_t n0 = (blockIdx.x % tiles_n) * 32;
    const uint32_t r = threadIdx.x & 31, g = threadIdx.x >> 5;
    const uint64_t m = min(m0 + r, rows - 1);
    const uint32_t n = min(n0 + r, out - 1);
    f32x16 acc = {};
    for (uint32_t j0 = 0; j0 < blocks; j0 += 2) {
        const uint32_t j = j0 + g;
        u32x4 a = {}, b = {};
        uint32_t sa = 127, sb = 127;
        if (j < blocks) {
            a = *reinterpret_cast<const u32x4_any *>(w + ((uint64_t)n * blocks + j) * 16);
            b = *reinterpret_cast<const u32x4_any *>(x + (m * blocks + j) * 16);
            sa = ws[(uint64_t)n * blocks + j];
            sb = xs[m * blocks + j];
        }
        const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
        const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, acc, 4, 4, 0, (int)sa, 0, (int)sb);
    }
    if (m0 + r >= rows)
        return;
    for (int i = 0; i < 16; ++i) {
        const uint32_t o = n0 + 8 * (i / 4) + 4 * g + i % 4;
        if (o < out) {
            float v = acc[i] + (bias ? bias[o] : 0.0f);
            if (relu)
                v = v < 0.0f ? 0.0f : v; // NaN stays
            y[(m0 + r) * out + o] = (Y)v;
        }
    }
}

// ---- a head in one kernel
//
// Between its layers a head's values stay in registers: a wave takes 64 rows
// through all of them, against weights that a block puts into shared memory
// once (four layers of 256 by 256 take 140 KB).
//
// With the weights as the first operand of the 32x32x64 product, a lane ends
// with 16 outputs of one row: of 32 outputs (one block of the next layer's
// input) the lanes l and l + 32 hold one half each, n = 8 (i / 4) + 4 (l / 32)
// + i % 4 for i = 0 .. 15.  Their largest magnitude, and so the block's scale,
// is one exchange away.  Packed to codes a half is two registers, and one
// exchange of registers between the halves of the wave
// (v_permlane32_swap_b32), for the two blocks of 64 outputs, gives each lane
// the 32 codes of one block: the next layer's operand.  Its codes are in the
// order of the two halves, and the weights behind are put into the same order
// when they are staged: a sum over a block does not mind.
constexpr int MLP_THREADS = 512, MLP_R = 2; // waves of 64 rows: two operands of 32
constexpr uint32_t MLP_WIDTH = 256;         // most values between layers: four operands of 64

struct MlpLayer {
    const uint8_t *codes, *scales;
    const float *bias;
    uint32_t width, out;
    uint32_t at;     // of its tiles in shared memory, then its scales, then its biases
    uint32_t at_scales, at_bias;
};
struct MlpArgs {
    MlpLayer layer[VT_MX4_MAX_LAYERS];
    uint32_t layers;
    const void *x;
    int64_t x_stride;
    void *y;
    uint64_t rows;
};

// Layout of a layer's weights in shared memory, tiles of 32 outputs by 64
// inputs: 16 bytes for (tile, pair of blocks, half, output), a word of scales
// (one byte a pair of blocks) for (tile, half, output), a bias for each output.
// Tiles go by pairs.
inline __host__ __device__ uint32_t mlp_pairs(uint32_t width) { return (width + 63) / 64; }
inline __host__ __device__ uint32_t mlp_tiles(uint32_t out) { return 2 * mlp_pairs(out); }

__device__ __forceinline__ void mlp_stage(const MlpLayer &l, bool reorder, char *lds)
{
    const uint32_t tiles = mlp_tiles(l.out), pairs = mlp_pairs(l.width), blocks = mx_blocks(l.width);
    const uint32_t units = tiles * pairs * 64;
    constexpr uint32_t EACH = 4; // loads of a thread at once
    for (uint32_t i0 = threadIdx.x; i0 < units; i0 += EACH * MLP_THREADS) {
        u32x4 w[EACH];
        uint32_t c[EACH], at[EACH];
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) {
            const uint32_t i = i0 + e * MLP_THREADS;
            const uint32_t r = i & 31, g = i >> 5 & 1, tp = i >> 6, tile = tp / pairs, pair = tp - tile * pairs;
            const uint32_t n = tile * 32 + r, j = 2 * pair + g;
            w[e] = u32x4{};
            c[e] = 127;
            at[e] = ((tile * 2 + g) * 32 + r) * 4 + pair;
            if (i < units && n < l.out && j < blocks) {
                w[e] = *reinterpret_cast<const u32x4_any *>(l.codes + ((uint64_t)n * blocks + j) * 16);
                c[e] = l.scales[(uint64_t)n * blocks + j];
            }
        }
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) {
            const uint32_t i = i0 + e * MLP_THREADS;
            if (i >= units)
                break;
            if (reorder) { // groups of four codes 0 .. 7 to 0 2 4 6 1 3 5 7
                const u32x4 q = w[e];
                w[e][0] = (q[0] & 0xffffu) | q[1] << 16;
                w[e][1] = (q[2] & 0xffffu) | q[3] << 16;
                w[e][2] = q[0] >> 16 | (q[1] & 0xffff0000u);
                w[e][3] = q[2] >> 16 | (q[3] & 0xffff0000u);
            }
            *reinterpret_cast<u32x4 *>(lds + l.at + i * 16) = w[e];
            *reinterpret_cast<uint8_t *>(lds + l.at_scales + at[e]) = (uint8_t)c[e];
        }
    }
    for (uint32_t n = threadIdx.x; n < tiles * 32; n += MLP_THREADS)
        *reinterpret_cast<float *>(lds + l.at_bias + n * 4) = l.bias && n < l.out ? l.bias[n] : 0.0f;
}

// One layer's 32 outputs of a tile for the wave's rows: acc = bias + sum.
template <int PAIRS>
__device__ __forceinline__ void mlp_tile(const MlpLayer &l, const char *lds, uint32_t tile, const u32x4 h[MLP_R][4],
                                         const uint32_t hs[MLP_R], f32x16 acc[MLP_R])
{
    const uint32_t lane = threadIdx.x & 63, g = lane >> 5;
    const char *b = lds + l.at_bias + (tile * 32 + 4 * g) * 4;
    f32x16 init;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(b + q * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            init[4 * q + i] = v[i];
    }
    const uint32_t ws = *reinterpret_cast<const uint32_t *>(lds + l.at_scales + (tile * 64 + lane) * 4);
    const char *w = lds + l.at + tile * PAIRS * 1024 + lane * 16;
    i32x8 a[PAIRS];
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {
        const u32x4 q = *reinterpret_cast<const u32x4 *>(w + p * 1024);
        a[p] = i32x8{(int)q[0], (int)q[1], (int)q[2], (int)q[3], 0, 0, 0, 0};
    }
#pragma unroll
    for (int m = 0; m < MLP_R; ++m) {
        acc[m] = init;
#define VT_MLP_STEP(p)                                                                                                 \
    if constexpr (PAIRS > p) {                                                                                         \
        const i32x8 v = {(int)h[m][p][0], (int)h[m][p][1], (int)h[m][p][2], (int)h[m][p][3], 0, 0, 0, 0};              \
        acc[m] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[p], v, acc[m], 4, 4, p, (int)ws, p, (int)hs[m]);    \
    }
        VT_MLP_STEP(0)
        VT_MLP_STEP(1)
        VT_MLP_STEP(2)
        VT_MLP_STEP(3)
#undef VT_MLP_STEP
    }
}

// The largest of 16 outputs and 0; NaN stays.
__device__ __forceinline__ uint32_t mlp_top(const f32x16 &v)
{
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        top = __builtin_elementwise_maximum(top, (float)v[i]);
    return __builtin_bit_cast(uint32_t, top);
}

// 16 outputs through ReLU to codes, two words.
__device__ __forceinline__ void mlp_codes(const f32x16 &acc, float scale, uint32_t w[2])
{
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i)
        v[i] = acc[i];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t q = e2m1_word(v + 8 * i, scale), s = q & 0x88888888u;
        w[i] = q & ~(s - (s >> 3)); // negative codes to -0
    }
}

// 64 outputs of the wave's rows, half of a block and half of another in each
// lane, through ReLU to the next layer's operand: the lower lanes get the first
// block and its scale, the upper ones the second.
__device__ __forceinline__ u32x4 mlp_operand(const f32x16 &a, const f32x16 &b, uint32_t &scale)
{
    const auto t = __builtin_amdgcn_permlane32_swap(mlp_top(a), mlp_top(b), false, false);
    const float top = __builtin_elementwise_maximum(__builtin_bit_cast(float, (uint32_t)t[0]),
                                                    __builtin_bit_cast(float, (uint32_t)t[1]));
    const uint32_t e = __builtin_bit_cast(uint32_t, top) >> 23 & 255, c = __builtin_elementwise_sub_sat(e, 2u);
    // under the scale 255 the codes do not count; c = 0 is the subnormal 2^-127
    const uint32_t f = max(c << 23, 0x00400000u);
    const auto of = __builtin_amdgcn_permlane32_swap(f, f, false, false); // the first block's for all, the second's
    uint32_t p[2], q[2];
    mlp_codes(a, __builtin_bit_cast(float, (uint32_t)of[0]), p);
    mlp_codes(b, __builtin_bit_cast(float, (uint32_t)of[1]), q);
    const auto s0 = __builtin_amdgcn_permlane32_swap(p[0], q[0], false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap(p[1], q[1], false, false);
    scale = e == 255 ? MX_NAN : c;
    return u32x4{s0[0], s1[0], s0[1], s1[1]};
}

template <int PAIRS, int TO>
__device__ __forceinline__ void mlp_hidden(const MlpLayer &l, const char *lds, u32x4 h[MLP_R][4], uint32_t hs[MLP_R])
{
    u32x4 to[MLP_R][TO];
    uint32_t to_s[MLP_R] = {};
#pragma unroll
    for (int q = 0; q < TO; ++q) {
        f32x16 acc[2][MLP_R];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            mlp_tile<PAIRS>(l, lds, 2 * q + b, h, hs, acc[b]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int m = 0; m < MLP_R; ++m) {
            uint32_t c;
            to[m][q] = mlp_operand(acc[0][m], acc[1][m], c);
            to_s[m] |= c << (8 * q);
        }
    }
#pragma unroll
    for (int m = 0; m < MLP_R; ++m) {
#pragma unroll
        for (int q = 0; q < TO; ++q)
            h[m][q] = to[m][q];
        hs[m] = to_s[m];
    }
}

template <int PAIRS>
__device__ __forceinline__ void mlp_hidden(const MlpLayer &l, const char *lds, u32x4 h[MLP_R][4], uint32_t hs[MLP_R])
{
    switch (mlp_pairs(l.out)) {
    case 1: mlp_hidden<PAIRS, 1>(l, lds, h, hs); break;
    case 2: mlp_hidden<PAIRS, 2>(l, lds, h, hs); break;
    case 3: mlp_hidden<PAIRS, 3>(l, lds, h, hs); break;
    default: mlp_hidden<PAIRS, 4>(l, lds, h, hs); break;
    }
}

template <int PAIRS, typename Y>
__device__ __forceinline__ void mlp_last(const MlpLayer &l, const char *lds, const u32x4 h[MLP_R][4],
                                         const uint32_t hs[MLP_R], uint64_t m0, uint64_t rows, Y *y)
{
    const uint32_t r = threadIdx.x & 31, g = threadIdx.x >> 5 & 1;
    for (uint32_t t = 0; t * 32 < l.out; ++t) {
        f32x16 acc[MLP_R];
        mlp_tile<PAIRS>(l, lds, t, h, hs, acc);
#pragma unroll
        for (int m = 0; m < MLP_R; ++m) {
            const uint64_t row = m0 + 32 * m + r;
            // the halves trade runs of four, so that each has eight neighbouring outputs: 16 q + 8 g
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float a0 = acc[m][8 * q + i], a1 = acc[m][8 * q + 4 + i];
                    const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a0),
                                                                    __builtin_bit_cast(uint32_t, a1), false, false);
                    v[i] = __builtin_bit_cast(float, (uint32_t)s[0]);
                    v[4 + i] = __builtin_bit_cast(float, (uint32_t)s[1]);
                }
                const uint32_t n = t * 32 + 16 * q + 8 * g;
                if (row < rows && n < l.out)
                    store_upto8(y + row * l.out + n, l.out - n, v);
            }
        }
    }
}

// Rows of x as operands: a lane's block of 32 of row r, quantised.
template <typename T>
__device__ __forceinline__ void mlp_load(const T *x, int64_t x_stride, uint64_t m0, uint64_t rows, uint32_t width,
                                         uint32_t pair, Mx4Piece<T> v[MLP_R][4])
{
    const uint32_t r = threadIdx.x & 31, k = 64 * pair + (threadIdx.x & 32), left = k < width ? width - k : 0;
#pragma unroll
    for (int m = 0; m < MLP_R; ++m) {
        const T *at = x + (int64_t)min(m0 + 32 * m + r, rows - 1) * x_stride + k;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            v[m][i].load(at + 8 * i, left > 8 * i ? left - 8 * i : 0);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t mlp_quantize(const Mx4Piece<T> v[4], u32x4 &h)
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i].top(top);
    const uint32_t c = mx4_scale(Mx4Piece<T>::top_bits(top));
    const float scale = e8m0_value(c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = v[i].word(scale);
    return c;
}

template <typename T, typename Y>
__global__ __launch_bounds__(MLP_THREADS) void mx4_mlp_kernel(MlpArgs p)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    for (uint32_t i = 0; i < p.layers; ++i)
        mlp_stage(p.layer[i], i > 0, lds);
    __syncthreads();
    // Tiles of rows to blocks in turn, so that few of them spread over the chip. The first 64 values of the next
    // tile's rows are on their way while this one's are in the layers.
    const uint64_t step = (uint64_t)gridDim.x * (MLP_THREADS / 64) * (32 * MLP_R);
    uint64_t m0 = (blockIdx.x + (uint64_t)(threadIdx.x / 64) * gridDim.x) * (32 * MLP_R);
    const uint32_t width = p.layer[0].width, pairs = mlp_pairs(width);
    const T *x = (const T *)p.x;
    Mx4Piece<T> next[MLP_R][4];
    if (m0 < p.rows)
        mlp_load(x, p.x_stride, m0, p.rows, width, 0, next);
    for (; m0 < p.rows; m0 += step) {
        u32x4 h[MLP_R][4];
        uint32_t hs[MLP_R];
#pragma unroll
        for (int m = 0; m < MLP_R; ++m)
            hs[m] = mlp_quantize<T>(next[m], h[m][0]);
#pragma unroll
        for (uint32_t q = 1; q < 4; ++q) {
            if (q < pairs) {
                Mx4Piece<T> v[MLP_R][4];
                mlp_load(x, p.x_stride, m0, p.rows, width, q, v);
#pragma unroll
                for (int m = 0; m < MLP_R; ++m)
                    hs[m] |= mlp_quantize<T>(v[m], h[m][q]) << (8 * q);
            }
        }
        if (m0 + step < p.rows)
            mlp_load(x, p.x_stride, m0 + step, p.rows, width, 0, next);
        for (uint32_t i = 0; i + 1 < p.layers; ++i) {
            const MlpLayer &l = p.layer[i];
            switch (mlp_pairs(l.width)) {
            case 1: mlp_hidden<1>(l, lds, h, hs); break;
            case 2: mlp_hidden<2>(l, lds, h, hs); break;
            case 3: mlp_hidden<3>(l, lds, h, hs); break;
            default: mlp_hidden<4>(l, lds, h, hs); break;
            }
        }
        const MlpLayer &l = p.layer[p.layers - 1];
        switch (mlp_pairs(l.width)) {
        case 1: mlp_last<1>(l, lds, h, hs, m0, p.rows, (Y *)p.y); break;
        case 2: mlp_last<2>(l, lds, h, hs, m0, p.rows, (Y *)p.y); break;
        case 3: mlp_last<3>(l, lds, h, hs, m0, p.rows, (Y *)p.y); break;
        default: mlp_last<4>(l, lds, h, hs, m0, p.rows, (Y *)p.y); break;
        }
    }
}

// Shared memory that the layers take, and their places in it; 0 where a layer
// is too wide or the weights do not fit: those heads go layer by layer.
constexpr uint32_t MLP_LDS = 160 * 1024;
static uint32_t mlp_places(const vt_mx4_layer *layers, uint32_t num_layers, MlpLayer *to)
{
    uint64_t at = 0;
    for (uint32_t i = 0; i < num_layers; ++i) {
        const vt_mx4_layer &l = layers[i];
        if (l.width > MLP_WIDTH || (i + 1 < num_layers && l.out > MLP_WIDTH))
            return 0;
        const uint64_t tiles = mlp_tiles(l.out), pairs = mlp_pairs(l.width);
        const uint64_t scales = at + tiles * pairs * 1024, bias = scales + tiles * 256;
        if (to)
            to[i] = MlpLayer{l.codes, l.scales, l.bias, l.width, l.out, (uint32_t)at, (uint32_t)scales, (uint32_t)bias};
        at = bias + tiles * 128;
        if (at > MLP_LDS)
            return 0;
    }
    return (uint32_t)at;
}

static int launch_mlp(int x_dtype, int y_dtype, const MlpArgs &p, uint32_t lds, hipStream_t s)
{
    const uint64_t tiles = (p.rows + 32 * MLP_R - 1) / (32 * MLP_R);
    const uint32_t grid = (uint32_t)(tiles < 256 ? tiles : 256); // one block a CU
    return with_type(x_dtype, [&](auto t) -> int {
        return with_type(y_dtype, [&](auto u) -> int {
            auto kernel = mx4_mlp_kernel<decltype(t), decltype(u)>;
            if (lds > 65536)
                VT_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)MLP_LDS));
            kernel<<<grid, MLP_THREADS, lds, s>>>(p);
            VT_LAUNCH_CHECK("mx4_mlp_kernel");
            return VT_OK;
        });
    });
}

struct Mx4Rows {
    const uint8_t *codes, *scales;
};

static uint64_t align16(uint64_t n) { return (n + 15) & ~(uint64_t)15; }

static uint64_t mx4_bytes(uint64_t rows, uint32_t width) // codes, then scales
{
    const uint64_t blocks = rows * mx_blocks(width);
    return 16 * blocks + align16(blocks);
}

static int launch_quantize(int dtype, const void *x, int64_t x_stride, uint64_t rows, uint32_t width, uint8_t *codes,
                           uint8_t *scales, hipStream_t s)
{
    const uint64_t groups = rows * mx_blocks(width) * 4, grid = (groups + MX_THREADS - 1) / MX_THREADS;
    if (groups == 0)
        return VT_OK;
    VT_REQUIRE(grid < (1ull << 31), "%llu rows of %u values are too many for one call", (unsigned long long)rows, width);
    return with_type(dtype, [&](auto t) -> int {
        mx4_quantize_kernel<<<(uint32_t)grid, MX_THREADS, 0, s>>>((const decltype(t) *)x, x_stride, groups, width,
                                                                  codes, scales);
        VT_LAUNCH_CHECK("mx4_quantize_kernel");
        return VT_OK;
    });
}

static int launch_linear(Mx4Rows x, uint64_t rows, uint32_t width, Mx4Rows w, uint32_t out, const float *bias, int relu,
                         int y_dtype, void *y, hipStream_t s)
{
    const uint64_t grid = (rows + 31) / 32 * ((out + 31) / 32);
    VT_REQUIRE(grid < (1ull << 31), "%llu rows by %u outputs are too many for one call", (unsigned long long)rows, out);
    return with_type(y_dtype, [&](auto t) -> int {
        mx4_linear_kernel<<<(uint32_t)grid, 64, 0, s>>>(x.codes, x.scales, rows, mx_blocks(width), w.codes, w.scales, out,
                                                        bias, relu, (decltype(t) *)y);
        VT_LAUNCH_CHECK("mx4_linear_kernel");
        return VT_OK;
    });
}

static int linear(int x_dtype, const void *x, int64_t x_stride, const uint8_t *x_scales, uint64_t rows, uint32_t width,
                  Mx4Rows w, uint32_t out, const float *bias, int relu, int y_dtype, void *y, void *workspace,
                  hipStream_t s)
{
    Mx4Rows xr{(const uint8_t *)x, x_scales};
    if (x_dtype != VT_MX4) {
        uint8_t *codes = (uint8_t *)workspace, *scales = codes + 16 * rows * mx_blocks(width);
        if (int rc = launch_quantize(x_dtype, x, x_stride, rows, width, codes, scales, s))
            return rc;
        xr = Mx4Rows{codes, scales};
    }
    return launch_linear(xr, rows, width, w, out, bias, relu, y_dtype, y, s);
}

} // namespace vt

using namespace vt;

extern "C" int vt_mx4_quantize(int dtype, const void *x, int64_t x_stride, uint64_t rows, uint32_t width,
                               uint8_t *codes, uint8_t *scales, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || width == 0)
        return VT_OK;
    VT_REQUIRE(x && codes && scales, "null pointer argument");
    return launch_quantize(dtype, x, x_stride, rows, width, codes, scales, as_stream(stream));
}

extern "C" int vt_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint32_t width, int dtype,
                                 void *out, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || width == 0)
        return VT_OK;
    VT_REQUIRE(codes && scales && out, "null pointer argument");
    const uint64_t groups = rows * mx_blocks(width) * 4, grid = (groups + MX_THREADS - 1) / MX_THREADS;
    VT_REQUIRE(grid < (1ull << 31), "%llu rows of %u values are too many for one call", (unsigned long long)rows, width);
    return with_type(dtype, [&](auto t) -> int {
        mx4_dequantize_kernel<<<(uint32_t)grid, MX_THREADS, 0, as_stream(stream)>>>(codes, scales, groups, width,
                                                                                    (decltype(t) *)out);
        VT_LAUNCH_CHECK("mx4_dequantize_kernel");
        return VT_OK;
    });
}

extern "C" size_t vt_mx4_linear_workspace_size(int x_dtype, uint64_t rows, uint32_t width, uint32_t out)
{
    (void)out;
    return x_dtype == VT_MX4 ? 0 : mx4_bytes(rows, width);
}

extern "C" int vt_mx4_linear(int x_dtype, const void *x, int64_t x_stride, const uint8_t *x_scales, uint64_t rows,
                             uint32_t width, const uint8_t *w_codes, const uint8_t *w_scales, uint32_t out,
                             const float *bias, int relu, int y_dtype, void *y, void *workspace, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || out == 0)
        return VT_OK;
    VT_REQUIRE(y && ((x && w_codes && w_scales) || width == 0), "null pointer argument");
    VT_REQUIRE(x_dtype != VT_MX4 || x_scales || width == 0, "x in 4 bits needs its scales");
    VT_REQUIRE(x_dtype == VT_MX4 || workspace || width == 0, "null workspace");
    VT_REQUIRE(x_dtype >= VT_F32 && x_dtype <= VT_MX4, "x dtype %d is none of VT_F32, VT_F16, VT_BF16, VT_MX4", x_dtype);
    VT_REQUIRE(y_dtype >= VT_F32 && y_dtype <= VT_BF16, "y dtype %d is none of VT_F32, VT_F16, VT_BF16", y_dtype);
    return linear(x_dtype, x, x_stride, x_scales, rows, width, Mx4Rows{w_codes, w_scales}, out, bias, relu, y_dtype, y,
                  workspace, as_stream(stream));
}

// Rows of a head's layers that go through the workspace at once.
static constexpr uint64_t MLP_CHUNK = 65536;

// {bytes of the hidden values of a chunk (f32, two of them), bytes of a chunk's quantised rows}
static void mlp_sizes(uint64_t rows, const vt_mx4_layer *layers, uint32_t num_layers, uint64_t &hidden, uint64_t &quant)
{
    const uint64_t n = rows < MLP_CHUNK ? rows : MLP_CHUNK;
    hidden = quant = 0;
    for (uint32_t i = 0; i < num_layers; ++i) {
        const uint64_t q = mx4_bytes(n, layers[i].width), h = i + 1 < num_layers ? align16(4 * n * layers[i].out) : 0;
        quant = q > quant ? q : quant;
        hidden = h > hidden ? h : hidden;
    }
}

extern "C" size_t vt_mx4_mlp_workspace_size(int x_dtype, uint64_t rows, const vt_mx4_layer *layers, uint32_t num_layers)
{
    (void)x_dtype;
    if (!layers || mlp_places(layers, num_layers, nullptr))
        return 0;
    uint64_t hidden, quant;
    mlp_sizes(rows, layers, num_layers, hidden, quant);
    return hidden + quant;
}

extern "C" int vt_mx4_mlp(int x_dtype, const void *x, int64_t x_stride, uint64_t rows, const vt_mx4_layer *layers,
                          uint32_t num_layers, int y_dtype, void *y, void *workspace, vt_stream_t stream)
{
    clear_error();
    VT_REQUIRE(layers && num_layers >= 1 && num_layers <= VT_MX4_MAX_LAYERS, "1 to %d layers, got %u",
               VT_MX4_MAX_LAYERS, num_layers);
    VT_REQUIRE(x_dtype >= VT_F32 && x_dtype <= VT_BF16, "x dtype %d is none of VT_F32, VT_F16, VT_BF16", x_dtype);
    VT_REQUIRE(y_dtype >= VT_F32 && y_dtype <= VT_BF16, "y dtype %d is none of VT_F32, VT_F16, VT_BF16", y_dtype);
    for (uint32_t i = 0; i < num_layers; ++i) {
        VT_REQUIRE(layers[i].codes && layers[i].scales && layers[i].width && layers[i].out,
                   "layer %u: null weights or an empty side", i);
        VT_REQUIRE(i == 0 || layers[i].width == layers[i - 1].out, "layer %u takes %u values, the one before gives %u", i,
                   layers[i].width, layers[i - 1].out);
    }
    if (rows == 0)
        return VT_OK;
    VT_REQUIRE(x && y, "null pointer argument");
    MlpArgs p{};
    if (const uint32_t lds = mlp_places(layers, num_layers, p.layer)) {
        p.layers = num_layers;
        p.x = x;
        p.x_stride = x_stride;
        p.y = y;
        p.rows = rows;
        return launch_mlp(x_dtype, y_dtype, p, lds, as_stream(stream));
    }
    VT_REQUIRE(workspace, "null workspace");
    uint64_t hidden, quant;
    mlp_sizes(rows, layers, num_layers, hidden, quant);
    const uint64_t esize[3] = {4, 2, 2};
    const uint32_t last = num_layers - 1;
    for (uint64_t m0 = 0; m0 < rows; m0 += MLP_CHUNK) {
        const uint64_t n = rows - m0 < MLP_CHUNK ? rows - m0 : MLP_CHUNK;
        const void *h = (const char *)x + (int64_t)m0 * x_stride * (int64_t)esize[x_dtype];
        int64_t stride = x_stride;
        int type = x_dtype;
        for (uint32_t i = 0; i < num_layers; ++i) {
            const vt_mx4_layer &l = layers[i];
            void *to = i == last ? (char *)y + m0 * l.out * esize[y_dtype] : (char *)workspace + quant;
            // the rows are in 4 bits, in the workspace's front, before the product writes over the hidden values
            if (int rc = linear(type, h, stride, nullptr, n, l.width, Mx4Rows{l.codes, l.scales}, l.out, l.bias,
                                i != last, i == last ? y_dtype : VT_F32, to, workspace, as_stream(stream)))
                return rc;
            h = to;
            stride = l.out;
            type = VT_F32;
        }
    }
    return VT_OK;
}
