// vt_ckpt8.hip -- activations that keep their input in 8 bits (ckpt8,
// include/vt_micro_abi.h) and their use in the backward pass: the slope of
// the activation, and the gradient of the weights behind it.
#include "vt_micro.h"

#include <type_traits>

namespace vt {

constexpr int ACT_THREADS = 256;

template <int ACT>
__device__ __forceinline__ float act_value(float z)
{
    if constexpr (ACT == VT_ACT_RELU)
        return z < 0.0f ? 0.0f : z; // NaN stays
    if constexpr (ACT == VT_ACT_SILU)
        return z / (1.0f + expf(-z));
    if constexpr (ACT == VT_ACT_GELU)
        return 0.5f * z * erfcf(-0.70710678118654752f * z);
    return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z)
{
    if constexpr (ACT == VT_ACT_RELU)
        return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
    if constexpr (ACT == VT_ACT_SILU) { // s + z s (1 - s), s (1 - s) = t / (1 + t)^2 with t = exp(-|z|)
        const float t = expf(-fabsf(z)), u = 1.0f / (1.0f + t);
        return (z < 0.0f ? t * u : u) + z * (t * u * u);
    }
    if constexpr (ACT == VT_ACT_GELU) // cdf + z pdf
        return 0.5f * erfcf(-0.70710678118654752f * z) + z * (0.39894228040143268f * expf(-0.5f * z * z));
    return z != z ? z : 1.0f;
}

// e4m3 codes of four values under 2^(127 - c), `inv` 2^-(c - 127): nearest
// even, zero for zeros alone, 0x7f for NaN and infinity.
__device__ __forceinline__ uint32_t e4m3_quad(const float *x, float inv)
{
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = x[i] * inv;
        // 2^-9 with x's sign where the quotient is smaller and x is not zero
        v[i] = fabsf(q) < 0x1p-9f && x[i] != 0.0f ? __builtin_copysignf(0x1p-9f, x[i]) : q;
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
    // 0xff (NaN with a sign) to 0x7f
    const uint32_t u = (uint32_t)w, low7 = u & 0x7f7f7f7fu, nan = (low7 + 0x01010101u) & 0x80808080u;
    return u & ~nan;
}

// Decode: four codes to f32 under `scale`.
__device__ __forceinline__ void e4m3_values(uint32_t w, float scale, float *v)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a[0] * scale;
    v[1] = a[1] * scale;
    v[2] = b[0] * scale;
    v[3] = b[1] * scale;
}

__device__ __forceinline__ void load_codes(const uint8_t *p, uint32_t n, uint32_t w[2])
{
    if (n >= 8) {
        const u32x2 q = *reinterpret_cast<const u32x2_any *>(p);
        w[0] = q[0];
        w[1] = q[1];
    } else {
        w[0] = w[1] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i < n)
                w[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
    }
}

// Eight values a thread, a block's four threads side by side, as the 4-bit
// quantisation.
template <typename T, int ACT>
__global__ __launch_bounds__(ACT_THREADS) void act_checkpoint_kernel(const T *__restrict__ z, int64_t z_stride,
                                                                     uint64_t groups, uint32_t width, T *__restrict__ y,
                                                                     uint8_t *__restrict__ codes,
                                                                     uint8_t *__restrict__ scales)
{
    const uint64_t at = (uint64_t)blockIdx.x * ACT_THREADS + threadIdx.x;
    if (at >= groups)
        return;
    const uint32_t per_row = 4 * mx_blocks(width);
    const uint64_t row = at / per_row;
    const uint32_t k = (uint32_t)(at - row * per_row) * 8, n = k < width ? width - k : 0;
    float v[8];
    load_upto8(z + (int64_t)row * z_stride + k, n, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = abs_bits(v[i]);
        top = max(top, b < 0x7f800000u ? b : 0u);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, 4));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, 4));
    const uint32_t e = top >> 23, c = e > 7 ? e - 7 : 0;
    if ((threadIdx.x & 3) == 0)
        scales[at / 4] = (uint8_t)c;
    if (n == 0)
        return;
    const float inv = e8m0_inverse(c);
    const uint32_t w[2] = {e4m3_quad(v, inv), e4m3_quad(v + 4, inv)};
    uint8_t *to = codes + row * width + k;
    if (n >= 8) {
        *reinterpret_cast<u32x2_any *>(to) = u32x2{w[0], w[1]};
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i < n)
                to[i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = act_value<ACT>(v[i]);
    if (ACT != VT_ACT_NONE || y)
        store_upto8(y + row * width + k, n, v);
}

// dz = dy act'(z^); without dy, z^ itself.
template <typename T, int ACT, bool SLOPE>
__global__ __launch_bounds__(ACT_THREADS) void ckpt8_read_kernel(const uint8_t *__restrict__ codes,
                                                                 const uint8_t *__restrict__ scales,
                                                                 const T *__restrict__ dy, int64_t dy_stride,
                                                                 uint64_t groups, uint32_t width, T *__restrict__ out)
{
    const uint64_t at = (uint64_t)blockIdx.x * ACT_THREADS + threadIdx.x;
    if (at >= groups)
        return;
    const uint32_t per_row = 4 * mx_blocks(width);
    const uint64_t row = at / per_row;
    const uint32_t k = (uint32_t)(at - row * per_row) * 8;
    if (k >= width)
        return;
    const uint32_t n = width - k;
    uint32_t w[2];
    load_codes(codes + row * width + k, n, w);
    const float s = e8m0_value(scales[at / 4]);
    float v[8];
    e4m3_values(w[0], s, v);
    e4m3_values(w[1], s, v + 4);
    if constexpr (SLOPE) {
        float d[8];
        load_upto8(dy + (int64_t)row * dy_stride + k, n, d);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = d[i] * act_slope<ACT>(v[i]);
    }
    store_upto8(out + row * width + k, n, v);
}

// dw[n][k] += dy[m][n] act(z^[m][k]) over one range of rows a block: a tile of
// 16 n by 16 k, one output a thread, rows staged in shared memory.
constexpr int WG_TILE = 16, WG_ROWS = 32;

template <typename T, int ACT>
__global__ __launch_bounds__(WG_TILE *WG_TILE) void weight_grad_kernel(
    const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales, const T *__restrict__ dy, int64_t dy_stride,
    uint64_t rows, uint64_t rows_per_split, uint32_t width, uint32_t out, float *__restrict__ dw, float *__restrict__ db)
{
    __shared__ float a[WG_ROWS][WG_TILE + 1], b[WG_ROWS][WG_TILE + 1];
    const uint32_t tk = threadIdx.x % WG_TILE, tn = threadIdx.x / WG_TILE;
    const uint32_t k0 = blockIdx.x * WG_TILE, n0 = blockIdx.y * WG_TILE;
    const uint64_t m1 = min(rows, (blockIdx.z + 1) * rows_per_split);
    float sum = 0.0f, sum_b = 0.0f;
    for (uint64_t m0 = blockIdx.z * rows_per_split; m0 < m1; m0 += WG_ROWS) {
        __syncthreads();
        for (int i = threadIdx.x; i < WG_ROWS * WG_TILE; i += WG_TILE * WG_TILE) {
            const uint32_t r = i / WG_TILE, c = i % WG_TILE;
            const uint64_t m = m0 + r;
            float d = 0.0f, v = 0.0f;
            if (m < m1 && n0 + c < out)
                d = (float)dy[(int64_t)m * dy_stride + n0 + c];
            if (m < m1 && k0 + c < width) {
                float q[4];
                e4m3_values(codes[m * width + k0 + c], e8m0_value(scales[m * mx_blocks(width) + (k0 + c) / MX_BLOCK]), q);
                v = act_value<ACT>(q[0]);
            }
            a[r][c] = d;
            b[r][c] = v;
        }
        __syncthreads();
        for (int r = 0; r < WG_ROWS; ++r) {
            sum = __builtin_fmaf(a[r][tn], b[r][tk], sum);
            sum_b += a[r][tn];
        }
    }
    const uint32_t n = n0 + tn, k = k0 + tk;
    if (n < out && k < width)
        dw[((uint64_t)blockIdx.z * out + n) * width + k] = sum;
    if (db && n < out && k == 0)
        db[(uint64_t)blockIdx.z * out + n] = sum_b;
}

// Joins the ranges' sums in their order.
__global__ __launch_bounds__(256) void weight_join_kernel(const float *__restrict__ parts, uint32_t splits, uint64_t n,
                                                          float *__restrict__ to)
{
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n)
        return;
    float s = 0.0f;
    for (uint32_t p = 0; p < splits; ++p)
        s += parts[p * n + i];
    to[i] = s;
}

static uint32_t weight_splits(uint64_t rows, uint32_t width, uint32_t out)
{
    const uint64_t tiles = (uint64_t)(width / WG_TILE + 1) * (out / WG_TILE + 1);
    uint64_t s = tiles < 2048 ? 2048 / tiles : 1;
    const uint64_t most = (rows + 255) / 256;
    return (uint32_t)(s < most ? s : most ? most : 1);
}

template <typename F>
static int with_act(int act, F &&f)
{
    switch (act) {
    case VT_ACT_NONE: return f(std::integral_constant<int, VT_ACT_NONE>());
    case VT_ACT_RELU: return f(std::integral_constant<int, VT_ACT_RELU>());
    case VT_ACT_SILU: return f(std::integral_constant<int, VT_ACT_SILU>());
    case VT_ACT_GELU: return f(std::integral_constant<int, VT_ACT_GELU>());
    }
    set_error("activation %d is none of VT_ACT_NONE, VT_ACT_RELU, VT_ACT_SILU, VT_ACT_GELU", act);
    return VT_ERR_INVALID;
}

static int group_grid(uint64_t rows, uint32_t width, uint64_t &groups, uint32_t &grid)
{
    groups = rows * mx_blocks(width) * 4;
    const uint64_t g = (groups + ACT_THREADS - 1) / ACT_THREADS;
    VT_REQUIRE(g < (1ull << 31), "%llu rows of %u values are too many for one call", (unsigned long long)rows, width);
    grid = (uint32_t)g;
    return VT_OK;
}

} // namespace vt

using namespace vt;

extern "C" int vt_act_checkpoint(int dtype, int act, const void *z, int64_t z_stride, uint64_t rows, uint32_t width,
                                 void *y, uint8_t *codes, uint8_t *scales, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || width == 0)
        return VT_OK;
    VT_REQUIRE(z && (y || act == VT_ACT_NONE) && codes && scales, "null pointer argument");
    uint64_t groups;
    uint32_t grid;
    if (int rc = group_grid(rows, width, groups, grid))
        return rc;
    return with_type(dtype, [&](auto t) -> int {
        return with_act(act, [&](auto a) -> int {
            typedef decltype(t) T;
            act_checkpoint_kernel<T, decltype(a)::value><<<grid, ACT_THREADS, 0, as_stream(stream)>>>(
                (const T *)z, z_stride, groups, width, (T *)y, codes, scales);
            VT_LAUNCH_CHECK("act_checkpoint_kernel");
            return VT_OK;
        });
    });
}

extern "C" int vt_ckpt8_dequantize(const uint8_t *codes, const uint8_t *scales, uint64_t rows, uint32_t width,
                                   int dtype, void *out, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || width == 0)
        return VT_OK;
    VT_REQUIRE(codes && scales && out, "null pointer argument");
    uint64_t groups;
    uint32_t grid;
    if (int rc = group_grid(rows, width, groups, grid))
        return rc;
    return with_type(dtype, [&](auto t) -> int {
        typedef decltype(t) T;
        ckpt8_read_kernel<T, VT_ACT_NONE, false><<<grid, ACT_THREADS, 0, as_stream(stream)>>>(
            codes, scales, nullptr, 0, groups, width, (T *)out);
        VT_LAUNCH_CHECK("ckpt8_read_kernel");
        return VT_OK;
    });
}

extern "C" int vt_act_input_grad(int dtype, int act, const uint8_t *codes, const uint8_t *scales, const void *dy,
                                 int64_t dy_stride, uint64_t rows, uint32_t width, void *dz, vt_stream_t stream)
{
    clear_error();
    if (rows == 0 || width == 0)
        return VT_OK;
    VT_REQUIRE(codes && scales && dy && dz, "null pointer argument");
    uint64_t groups;
    uint32_t grid;
    if (int rc = group_grid(rows, width, groups, grid))
        return rc;
    return with_type(dtype, [&](auto t) -> int {
        return with_act(act, [&](auto a) -> int {
            typedef decltype(t) T;
            ckpt8_read_kernel<T, decltype(a)::value, true><<<grid, ACT_THREADS, 0, as_stream(stream)>>>(
                codes, scales, (const T *)dy, dy_stride, groups, width, (T *)dz);
            VT_LAUNCH_CHECK("ckpt8_read_kernel");
            return VT_OK;
        });
    });
}

extern "C" size_t vt_act_weight_grad_workspace_size(uint64_t rows, uint32_t width, uint32_t out)
{
    if (out == 0)
        return 0;
    const uint32_t s = weight_splits(rows, width, out);
    return s > 1 ? (size_t)s * out * ((size_t)width + 1) * 4 : 0;
}

extern "C" int vt_act_weight_grad(int dtype, int act, const uint8_t *codes, const uint8_t *scales, const void *dy,
                                  int64_t dy_stride, uint64_t rows, uint32_t width, uint32_t out, float *dw, float *db,
                                  void *workspace, vt_stream_t stream)
{
    clear_error();
    if (out == 0)
        return VT_OK;
    VT_REQUIRE((dw || width == 0) && ((codes && scales) || rows == 0 || width == 0) && (dy || rows == 0), "null pointer argument");
    const uint32_t splits = weight_splits(rows, width, out);
    VT_REQUIRE(splits == 1 || workspace, "null workspace");
    const uint64_t n = (uint64_t)out * width, per = ((rows + splits - 1) / splits + WG_ROWS - 1) / WG_ROWS * WG_ROWS;
    float *pw = splits > 1 ? (float *)workspace : dw, *pb = !db ? nullptr : splits > 1 ? pw + splits * n : db;
    // without inputs (width 0) the tiles of k = 0 still sum db
    const dim3 grid(width ? (width + WG_TILE - 1) / WG_TILE : 1, (out + WG_TILE - 1) / WG_TILE, splits);
    const hipStream_t s = as_stream(stream);
    int rc = with_type(dtype, [&](auto t) -> int {
        return with_act(act, [&](auto a) -> int {
            typedef decltype(t) T;
            weight_grad_kernel<T, decltype(a)::value><<<grid, WG_TILE * WG_TILE, 0, s>>>(
                codes, scales, (const T *)dy, dy_stride, rows, per, width, out, pw, pb);
            VT_LAUNCH_CHECK("weight_grad_kernel");
            return VT_OK;
        });
    });
    if (rc || splits == 1)
        return rc;
    if (n) {
        weight_join_kernel<<<(uint32_t)((n + 255) / 256), 256, 0, s>>>(pw, splits, n, dw);
        VT_LAUNCH_CHECK("weight_join_kernel");
    }
    if (db) {
        weight_join_kernel<<<(out + 255) / 256, 256, 0, s>>>(pb, splits, out, db);
        VT_LAUNCH_CHECK("weight_join_kernel");
    }
    return VT_OK;
}
