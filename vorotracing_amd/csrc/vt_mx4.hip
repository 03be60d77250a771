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
    float v[8];
    load_upto8(x + (int64_t)row * x_stride + k, k < width ? width - k : 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, abs_bits(v[i]));
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 4));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 4));
    const uint32_t c = mx4_scale(top);
    uint32_t word = 0;
    if (c != MX_NAN) {
        const float inv = e8m0_inverse(c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            word |= (e2m1_pair(v[2 * i] * inv, v[2 * i + 1] * inv) & 0xffu) << (8 * i);
    }
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
    if (!layers)
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
    VT_REQUIRE(x && y && workspace, "null pointer argument");
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
