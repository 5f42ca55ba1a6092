// Weight gradient behind an 8-bit product,
//
//     grad_w[k, n] = sum over rows m of x[m, k] * bf16(g[m, n]),   grad_bias[n] = sum over rows of g[m, n],
//
// x in the 8-bit format.  A scale of that format varies along the contraction here, so it cannot be left to the matrix
// unit; but a code times a power of two is a bf16 value, so x is turned into bf16 exactly on its way into LDS and the
// product runs on the bf16 matrix units: x loses nothing, g is rounded to 8 significant bits, sums are fp32.  What the
// forward has to keep for it is one byte a value.
//
// A block owns 128 x 128 of the result and a slice of the rows, 64 rows a stage.  The MFMA wants eight consecutive rows of
// one column in a lane, memory holds rows: a thread loads eight rows of four neighbouring columns, transposes them in
// registers and writes four 16-byte pieces of eight rows each.  The slices' results are added by a second launch in slice
// order; a grid of enough tiles has one slice and writes the result itself.
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 128;     // of the result, both ways
constexpr int kRows = 64;      // rows of x and g a stage

struct WgradArgs {
    const uint8_t *x, *x_scales;
    const void *g;
    float *out, *bias_out;     // slice 0's result; slice s lies s * k * n (s * n) floats behind
    int64_t g_stride, rows, rows_per_slice, k, n;
    int blocks;                // of 128 along x's rows
    int tiles_n;
};

// 16-byte piece q (eight rows) of column c in a staged tile: neighbouring columns' pieces spread over the banks both when
// columns 4 i + const are written and when 16 neighbouring ones are read
__device__ __forceinline__ int staged(int c, int q) { return c * (2 * kRows) + 16 * (q ^ (((c >> 1) ^ (c >> 4)) & 7)); }

// eight rows of four columns -> four pieces
__device__ __forceinline__ void write_columns(uint8_t *tile, int c, int q, const f32x4 (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const u32x4 piece = {bf16_pair(v[0][j], v[1][j]), bf16_pair(v[2][j], v[3][j]), bf16_pair(v[4][j], v[5][j]),
                             bf16_pair(v[6][j], v[7][j])};
        *reinterpret_cast<u32x4 *>(tile + staged(c + j, q)) = piece;
    }
}

template <typename G, bool VEC>
__global__ __launch_bounds__(256, 2) void fp8_wgrad_kernel(const WgradArgs p) {
    __shared__ __align__(16) uint8_t xt[kTile * 2 * kRows], gt[kTile * 2 * kRows];
    const int tid = (int)threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wk = wave / 2, wn = wave % 2, idx = lane % 32, half = lane / 32;
    const int kt = (int)blockIdx.x / p.tiles_n, nt = (int)blockIdx.x % p.tiles_n;
    const int64_t slice = blockIdx.y;
    const int64_t n0 = (int64_t)nt * kTile;
    const int64_t begin = slice * p.rows_per_slice;
    const int64_t end = begin + p.rows_per_slice < p.rows ? begin + p.rows_per_slice : p.rows;
    const int cq = tid % 32, oct = tid / 32;  // four columns, eight rows of a stage
    const int64_t pitch = (int64_t)p.blocks * kBlock8;
    const bool sums = kt == 0 && p.bias_out;

    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    f32x4 column_sum = {0.f, 0.f, 0.f, 0.f};

    uint32_t xc[8];
    int xe[8];
    f32x4 gv[8];
    auto fetch = [&](int64_t m0) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int64_t m = m0 + 8 * oct + r;
            xc[r] = 0;
            xe[r] = 127;
            gv[r] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (m < end) {
                xc[r] = *reinterpret_cast<const uint32_t *>(p.x + m * pitch + (int64_t)kt * kTile + 4 * cq);
                xe[r] = p.x_scales[m * p.blocks + kt];
                gv[r] = load4<VEC>(static_cast<const G *>(p.g) + m * p.g_stride, n0 + 4 * cq, p.n);
            }
        }
    };
    fetch(begin);
    for (int64_t m0 = begin; m0 < end; m0 += kRows) {
        __syncthreads();
        f32x4 xv[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) xv[r] = decode4(xc[r]) * pow2(xe[r] - 127);
        write_columns(xt, 4 * cq, oct, xv);
        write_columns(gt, 4 * cq, oct, gv);
        if (sums) {
#pragma unroll
            for (int r = 0; r < 8; ++r) column_sum += gv[r];
        }
        __syncthreads();
        if (m0 + kRows < end) fetch(m0 + kRows);
#pragma unroll
        for (int s = 0; s < kRows / 16; ++s) {
            bf16x8_t fx[2], fg[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                fx[i] = *reinterpret_cast<const bf16x8_t *>(xt + staged(64 * wk + 32 * i + idx, 2 * s + half));
#pragma unroll
            for (int j = 0; j < 2; ++j)
                fg[j] = *reinterpret_cast<const bf16x8_t *>(gt + staged(64 * wn + 32 * j + idx, 2 * s + half));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fx[i], fg[j], acc[i][j], 0, 0, 0);
        }
    }
    // register r of lane l holds row (r % 4) + 8 (r / 4) + 4 (l / 32), column l % 32 of its 32 x 32 tile
    float *out = p.out + slice * p.k * p.n;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t k = (int64_t)kt * kTile + 64 * wk + 32 * i + r % 4 + 8 * (r / 4) + 4 * half;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t n = n0 + 64 * wn + 32 * j + idx;
                if (k < p.k && n < p.n) out[k * p.n + n] = acc[i][j][r];
            }
        }
    if (sums) {
        f32x4 *parts = reinterpret_cast<f32x4 *>(xt);
        __syncthreads();
        parts[tid] = column_sum;
        __syncthreads();
        if (tid < 32) {
            for (int q = 1; q < 8; ++q) column_sum += parts[tid + 32 * q];
            store4<false>(p.bias_out + slice * p.n, n0 + 4 * cq, p.n, column_sum);
        }
    }
}

// slices that fill the chip twice over, at least 256 rows each, their results at most 256 MB
int64_t wgrad_slices(int64_t rows, int64_t k, int64_t n) {
    const int64_t tiles = (pad128(k) / kTile) * (pad128(n) / kTile);
    int64_t s = 1024 / tiles;
    const int64_t by_rows = rows / 256, by_bytes = (int64_t(1) << 26) / (k * n);
    s = s < by_rows ? s : by_rows;
    s = s < by_bytes ? s : by_bytes;
    return s < 1 ? 1 : s;
}

bool wgrad_sizes_ok(int64_t rows, int64_t k, int64_t n) {
    return rows >= 0 && k > 0 && n > 0 && k <= (1 << 20) && n <= (1 << 20) && k * n <= (int64_t(1) << 33);
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int64_t gnnagg_fp8_weight_gradient_workspace_bytes(int64_t rows, int64_t k, int64_t n) {
    if (!wgrad_sizes_ok(rows, k, n)) return 0;
    const int64_t s = wgrad_slices(rows, k, n);
    return s == 1 ? 0 : s * (k * n + n) * (int64_t)sizeof(float);
}

extern "C" int gnnagg_fp8_weight_gradient(const uint8_t *x, const uint8_t *x_scales, const void *g, int64_t g_stride,
                                          int g_dtype, float *grad_w, float *grad_bias, void *workspace,
                                          int64_t workspace_bytes, int64_t rows, int64_t k, int64_t n, void *stream) {
    GNNAGG_REQUIRE(rows >= 0 && k >= 0 && n >= 0, "negative size");
    GNNAGG_REQUIRE(known_dtype(g_dtype), "unknown dtype");
    if (k == 0 || n == 0) return GNNAGG_OK;
    if (!wgrad_sizes_ok(rows, k, n)) return fail(GNNAGG_ERR_UNSUPPORTED, "a weight of %lld x %lld", (long long)k, (long long)n);
    GNNAGG_REQUIRE(grad_w && (rows == 0 || (x && x_scales && g)), "null x/scales/g/grad_w");
    GNNAGG_REQUIRE(g_stride >= n, "a row stride is below the width");
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(x) % 4 == 0, "codes must be 4-byte aligned");
    const int64_t slices = wgrad_slices(rows, k, n), need = gnnagg_fp8_weight_gradient_workspace_bytes(rows, k, n);
    GNNAGG_REQUIRE(workspace_bytes >= need && (need == 0 || workspace) && reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
                   "workspace of %lld bytes is too small, null or misaligned", (long long)workspace_bytes);
    float *parts = slices == 1 ? grad_w : static_cast<float *>(workspace);
    float *bias_parts = !grad_bias ? nullptr : slices == 1 ? grad_bias : parts + slices * k * n;
    const int64_t per = (rows + slices - 1) / slices;
    const int64_t tiles_k = pad128(k) / kTile, tiles_n = pad128(n) / kTile;
    WgradArgs p{x, x_scales, g, parts, bias_parts, g_stride, rows, (per + kRows - 1) / kRows * kRows, k, n,
                (int)tiles_k, (int)tiles_n};
    if (tiles_k * tiles_n > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "too many tiles");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(tiles_k * tiles_n), (unsigned)slices);
    auto go = [&](auto type, auto v) {
        hipLaunchKernelGGL((fp8_wgrad_kernel<decltype(type), decltype(v)::value>), grid, dim3(256), 0, st, p);
    };
    const bool vec = vec4_rows(g, g_stride, n, g_dtype);
    if (g_dtype == GNNAGG_F32) {
        if (vec) go(float(), std::true_type());
        else go(float(), std::false_type());
    } else {
        if (vec) go(bf16_t(), std::true_type());
        else go(bf16_t(), std::false_type());
    }
    GNNAGG_HIP(hipGetLastError());
    if (slices == 1) return GNNAGG_OK;
    if (const int rc = launch_column_reduce(parts, slices, k * n, grad_w, st)) return rc;
    return grad_bias ? launch_column_reduce(bias_parts, slices, n, grad_bias, st) : GNNAGG_OK;
}
