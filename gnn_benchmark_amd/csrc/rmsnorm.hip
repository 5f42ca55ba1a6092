// RMS norm with the residual's addition, one pass over the data each way:
//
//     h = x + residual,   y = relu?(h * r * w),   r = 1 / sqrt(mean(h^2) + eps)
//
// forward: reads x and the residual once, writes h and y (or y's 8-bit codes and block scales) once.  Backward, with
// gn the gradient behind the ReLU and n the width:
//
//     grad w = sum over rows of gn * (h r),     grad h = r (gn w - (h r) mean(gn w (h r))) + grad of the residual stream
//
// TPR threads own a row (a part of a wave up to 1024 columns, a block of 256 or 1024 above), each holding NV runs of four
// consecutive columns, so a row is read once and its sums are taken from registers.  Both ways are bound by HBM; the sum
// of squares is fp64 (a v_fma_f64 per value, hidden behind the loads) because a code of the 8-bit output may hang on r's
// last place.  The weight gradient leaves each block as one partial row; a second launch adds those in a fixed order.
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y;
    uint8_t *codes, *scales;
    int64_t x_stride, residual_stride, h_stride, y_stride;
    int64_t rows, width, padded;
    double eps;
    int relu, weight_bf16;
};

struct NormBackwardArgs {
    const void *grad_y, *grad_h, *h, *weight;
    void *grad_x;
    float *partial;
    int64_t grad_y_stride, grad_h_stride, h_stride, grad_x_stride;
    int64_t rows, width;
    double eps;
    int relu, weight_bf16;
};

template <int W>
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int s = W / 2; s >= 1; s >>= 1) v += __shfl_xor(v, s, W);
    return v;
}
template <int W>
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = W / 2; s >= 1; s >>= 1) v = fmaxf(v, __shfl_xor(v, s, W));
    return v;
}

// the sum over a row's TPR threads, in every one of them; `slot`: 16 doubles of LDS where the row has a whole block
template <int TPR>
__device__ __forceinline__ double row_sum(double v, double *slot) {
    if constexpr (TPR <= 64) {
        return wave_sum<TPR>(v);
    } else {
        v = wave_sum<64>(v);
        if (threadIdx.x % 64 == 0) slot[threadIdx.x / 64] = v;
        __syncthreads();
        double s = slot[0];
#pragma unroll
        for (int q = 1; q < TPR / 64; ++q) s += slot[q];
        __syncthreads();
        return s;
    }
}

template <bool VEC>
__device__ __forceinline__ f32x4 load_weight(const void *w, int is_bf16, int64_t c, int64_t width) {
    return is_bf16 ? load4<VEC>(static_cast<const bf16_t *>(w), c, width) : load4<VEC>(static_cast<const float *>(w), c, width);
}

// h and the sum of its squares; returns r
template <int TPR, int NV>
__device__ __forceinline__ float inverse_rms(const f32x4 (&h)[NV], int64_t width, double eps, double *slot) {
    double q = 0.0;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) q = __builtin_fma((double)h[k][j], (double)h[k][j], q);
    q = row_sum<TPR>(q, slot);
    return (float)(1.0 / __builtin_sqrt(q / (double)width + eps));
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

template <typename T, int TPR, int NV, bool VEC, bool FP8>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_kernel(const NormArgs p) {
    constexpr int kGroups = block_of(TPR) / TPR;
    __shared__ double slot[16];
    const int l = (int)threadIdx.x % TPR;
    f32x4 w[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) w[k] = load_weight<VEC>(p.weight, p.weight_bf16, 4 * (l + k * TPR), p.width);
    // the threads of a row stay or leave together: shuffles and barriers never miss one
    for (int64_t row = (int64_t)blockIdx.x * kGroups + (int)threadIdx.x / TPR; row < p.rows;
         row += (int64_t)gridDim.x * kGroups) {
        const T *x = static_cast<const T *>(p.x) + row * p.x_stride;
        f32x4 h[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) h[k] = load4<VEC>(x, 4 * (l + k * TPR), p.width);
        if (p.residual) {
            const T *res = static_cast<const T *>(p.residual) + row * p.residual_stride;
            T *ho = static_cast<T *>(p.h) + row * p.h_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) h[k] = rounded(x, h[k] + load4<VEC>(res, 4 * (l + k * TPR), p.width));
#pragma unroll
            for (int k = 0; k < NV; ++k) store4<VEC>(ho, 4 * (l + k * TPR), p.width, h[k]);
        }
        const float r = inverse_rms<TPR, NV>(h, p.width, p.eps, slot);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            h[k] = h[k] * r * w[k];
            if (p.relu) {  // (a NaN stays one)
#pragma unroll
                for (int j = 0; j < 4; ++j) h[k][j] = h[k][j] < 0.0f ? 0.0f : h[k][j];
            }
        }
        if constexpr (!FP8) {
            T *y = static_cast<T *>(p.y) + row * p.y_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) store4<VEC>(y, 4 * (l + k * TPR), p.width, h[k]);
        } else {
            // Run k of the row's threads covers 4 * TPR columns: either whole blocks of 128, 32 neighbouring threads
            // each, or a part of one that the next runs complete.
            constexpr int kThreads = TPR < 32 ? TPR : 32;    // threads that share a block
            constexpr int kRuns = TPR < 32 ? 32 / TPR : 1;   // runs that share a block
            uint8_t *codes = p.codes + row * p.padded;
            uint8_t *scales = p.scales + row * (p.padded / kBlock8);
#pragma unroll
            for (int k0 = 0; k0 < NV; k0 += kRuns) {
                float top = 0.0f;
#pragma unroll
                for (int k = k0; k < k0 + kRuns && k < NV; ++k) top = fmaxf(top, finite_magnitude(h[k]));
                const int e = block_exponent(wave_max<kThreads>(top));
                const float inv = pow2(-e);
#pragma unroll
                for (int k = k0; k < k0 + kRuns; ++k) {      // (runs past NV hold a narrow row's padding)
                    const int64_t c = 4 * (l + k * TPR);
                    if (c >= p.padded) continue;
                    *reinterpret_cast<uint32_t *>(codes + c) = k < NV ? encode4(h[k < NV ? k : 0], inv) : 0u;
                    if (c % kBlock8 == 0) scales[c / kBlock8] = (uint8_t)(e + 127);
                }
            }
        }
    }
}

template <typename T, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_backward_kernel(const NormBackwardArgs p) {
    constexpr int kGroups = block_of(TPR) / TPR;
    __shared__ double slot[16];
    __shared__ f32x4 sums[kGroups > 1 ? 256 : 1];
    const int l = (int)threadIdx.x % TPR;
    f32x4 w[NV], gw_sum[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        w[k] = load_weight<VEC>(p.weight, p.weight_bf16, 4 * (l + k * TPR), p.width);
        gw_sum[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int64_t row = (int64_t)blockIdx.x * kGroups + (int)threadIdx.x / TPR; row < p.rows;
         row += (int64_t)gridDim.x * kGroups) {
        const T *hr = static_cast<const T *>(p.h) + row * p.h_stride;
        f32x4 h[NV], g[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) h[k] = load4<VEC>(hr, 4 * (l + k * TPR), p.width);
        const T *gr = static_cast<const T *>(p.grad_y) + row * p.grad_y_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) g[k] = load4<VEC>(gr, 4 * (l + k * TPR), p.width);
        const float r = inverse_rms<TPR, NV>(h, p.width, p.eps, slot);
        double s = 0.0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const f32x4 z = h[k] * r;
            if (p.relu) {  // exactly the values that the forward cut or found at zero
                const f32x4 y = z * w[k];
#pragma unroll
                for (int j = 0; j < 4; ++j) g[k][j] = y[j] > 0.0f ? g[k][j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) gw_sum[k][j] = __builtin_fmaf(g[k][j], z[j], gw_sum[k][j]);
            g[k] = g[k] * w[k];
#pragma unroll
            for (int j = 0; j < 4; ++j) s = __builtin_fma((double)g[k][j], (double)h[k][j], s);
        }
        s = row_sum<TPR>(s, slot);
        const float t = (float)(s * (double)r / (double)p.width);  // (r^3 alone would leave fp32's range for large rows)
        const T *gh = p.grad_h ? static_cast<const T *>(p.grad_h) + row * p.grad_h_stride : nullptr;
        T *out = static_cast<T *>(p.grad_x) + row * p.grad_x_stride;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            f32x4 d = (g[k] - h[k] * r * t) * r;
            if (gh) d += load4<VEC>(gh, 4 * (l + k * TPR), p.width);
            store4<VEC>(out, 4 * (l + k * TPR), p.width, d);
        }
    }
    // the block's rows' share of the weight gradient: its groups' sums in group order
    float *partial = p.partial + (int64_t)blockIdx.x * p.width;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        f32x4 total = gw_sum[k];
        if constexpr (kGroups > 1) {
            __syncthreads();
            sums[threadIdx.x] = total;
            __syncthreads();
            if (threadIdx.x < TPR)
                for (int q = 1; q < kGroups; ++q) total += sums[l + q * TPR];
        }
        if (threadIdx.x < TPR) store4<false>(partial, 4 * (l + k * TPR), p.width, total);
    }
}

// 32 columns a block, 32 slices of the partial rows, added in slice order
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float *__restrict__ partial, int64_t blocks,
                                                             int64_t width, float *__restrict__ out) {
    __shared__ float sums[32][33];
    const int col = (int)threadIdx.x % 32, slice = (int)threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    float a = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (int64_t b = slice; b < blocks; b += 32) a += partial[b * width + c];
    }
    sums[slice][col] = a;
    __syncthreads();
    if (slice == 0 && c < width) {
        for (int q = 1; q < 32; ++q) a += sums[q][col];
        out[c] = a;
    }
}

struct NormShape {
    int tpr, nv;
};

constexpr int64_t kMaxWidth = 16384;

// threads per row and runs of four columns per thread
NormShape norm_shape(int64_t width) {
    const int64_t runs = (width + 3) / 4;
    if (runs <= 8) return {8, 1};
    if (runs <= 16) return {16, 1};
    if (runs <= 32) return {16, 2};
    if (runs <= 64) return {16, 4};
    if (runs <= 128) return {32, 4};
    if (runs <= 256) return {64, 4};
    if (runs <= 512) return {256, 2};
    if (runs <= 1024) return {256, 4};
    if (runs <= 1536) return {256, 6};
    if (runs <= 2048) return {1024, 2};
    return {1024, 4};
}

template <typename F>
void for_norm_shape(const NormShape s, F &&launch) {
#define GNNAGG_NORM_SHAPE(T, N) \
    if (s.tpr == T && s.nv == N) return launch(std::integral_constant<int, T>(), std::integral_constant<int, N>());
    GNNAGG_NORM_SHAPE(8, 1)
    GNNAGG_NORM_SHAPE(16, 1)
    GNNAGG_NORM_SHAPE(16, 2)
    GNNAGG_NORM_SHAPE(16, 4)
    GNNAGG_NORM_SHAPE(32, 4)
    GNNAGG_NORM_SHAPE(64, 4)
    GNNAGG_NORM_SHAPE(256, 2)
    GNNAGG_NORM_SHAPE(256, 4)
    GNNAGG_NORM_SHAPE(256, 6)
    GNNAGG_NORM_SHAPE(1024, 2)
    GNNAGG_NORM_SHAPE(1024, 4)
#undef GNNAGG_NORM_SHAPE
}

int64_t backward_blocks(int64_t rows, int64_t width) {
    const int tpr = norm_shape(width).tpr;
    const int64_t groups = block_of(tpr) / tpr;
    const int64_t need = (rows + groups - 1) / groups;
    return need < 1024 ? need : 1024;  // four blocks a CU; 1024 partial rows are added in about 5 us
}

int check_norm(int64_t rows, int64_t width, int dtype, int weight_dtype) {
    GNNAGG_REQUIRE(rows >= 0 && width >= 0, "negative size");
    GNNAGG_REQUIRE(known_dtype(dtype) && known_dtype(weight_dtype), "unknown dtype");
    GNNAGG_REQUIRE(weight_dtype == GNNAGG_F32 || weight_dtype == dtype, "the weight is fp32 or of the rows' type");
    if (width < 1 || width > kMaxWidth)
        return fail(GNNAGG_ERR_UNSUPPORTED, "RMS norm takes widths of 1 to %lld (got %lld)", (long long)kMaxWidth,
                    (long long)width);
    return GNNAGG_OK;
}

int run_norm(const NormArgs &p, int dtype, int weight_dtype, bool fp8, hipStream_t st) {
    const bool vec = vec4_rows(p.x, p.x_stride, p.width, dtype) && vec4_rows(p.residual, p.residual_stride, p.width, dtype) &&
                     vec4_rows(p.h, p.h_stride, p.width, dtype) && vec4_rows(p.y, p.y_stride, p.width, dtype) &&
                     vec4_rows(p.weight, 4, p.width, weight_dtype);
    for_norm_shape(norm_shape(p.width), [&](auto tpr, auto nv) {
        constexpr int kTpr = decltype(tpr)::value, kNv = decltype(nv)::value, kGroups = block_of(kTpr) / kTpr;
        const int64_t need = (p.rows + kGroups - 1) / kGroups;
        const dim3 grid((unsigned)(need < 256 * 32 ? need : 256 * 32));
        auto go = [&](auto type, auto v, auto q) {
            hipLaunchKernelGGL((rms_norm_kernel<decltype(type), kTpr, kNv, decltype(v)::value, decltype(q)::value>), grid,
                               dim3(block_of(kTpr)), 0, st, p);
        };
        auto pick = [&](auto type, auto v) {
            if (fp8) go(type, v, std::true_type());
            else go(type, v, std::false_type());
        };
        if (dtype == GNNAGG_F32) {
            if (vec) pick(float(), std::true_type());
            else pick(float(), std::false_type());
        } else {
            if (vec) pick(bf16_t(), std::true_type());
            else pick(bf16_t(), std::false_type());
        }
    });
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}

}  // namespace

int launch_column_reduce(const float *partial, int64_t blocks, int64_t width, float *out, hipStream_t stream) {
    hipLaunchKernelGGL(column_reduce_kernel, dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, stream, partial, blocks,
                       width, out);
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}

}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_train_abi_version(void) { return GNNAGG_TRAIN_ABI_VERSION; }

static int norm_forward(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                        const void *weight, int weight_dtype, double eps, int relu, void *h, int64_t h_stride, void *y,
                        int64_t y_stride, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t width, int dtype,
                        bool fp8, void *stream) {
    if (const int rc = check_norm(rows, width, dtype, weight_dtype)) return rc;
    if (rows == 0) return GNNAGG_OK;
    GNNAGG_REQUIRE(x && weight && (fp8 ? codes && scales : y != nullptr), "null x/weight/output");
    GNNAGG_REQUIRE((residual != nullptr) == (h != nullptr), "h is written exactly where a residual is given");
    GNNAGG_REQUIRE(x_stride >= width && (!residual || (residual_stride >= width && h_stride >= width)) &&
                       (fp8 || y_stride >= width), "a row stride is below the width");
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 4 == 0, "codes must be 4-byte aligned");
    NormArgs p{x, residual, weight, h, y, codes, scales, x_stride, residual_stride, h_stride, y_stride,
               rows, width, pad128(width), eps, relu, weight_dtype == GNNAGG_BF16};
    return run_norm(p, dtype, weight_dtype, fp8, static_cast<hipStream_t>(stream));
}

extern "C" int gnnagg_rms_norm(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                               const void *weight, int weight_dtype, double eps, int relu, void *h, int64_t h_stride,
                               void *y, int64_t y_stride, int64_t rows, int64_t width, int dtype, void *stream) {
    return norm_forward(x, x_stride, residual, residual_stride, weight, weight_dtype, eps, relu, h, h_stride, y, y_stride,
                        nullptr, nullptr, rows, width, dtype, false, stream);
}

extern "C" int gnnagg_rms_norm_fp8(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                                   const void *weight, int weight_dtype, double eps, int relu, void *h,
                                   int64_t h_stride, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t width,
                                   int dtype, void *stream) {
    return norm_forward(x, x_stride, residual, residual_stride, weight, weight_dtype, eps, relu, h, h_stride, nullptr, 0,
                        codes, scales, rows, width, dtype, true, stream);
}

extern "C" int64_t gnnagg_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
    if (rows <= 0 || width < 1 || width > kMaxWidth) return 0;
    return backward_blocks(rows, width) * width * (int64_t)sizeof(float);
}

extern "C" int gnnagg_rms_norm_backward(const void *grad_y, int64_t grad_y_stride, const void *grad_h,
                                        int64_t grad_h_stride, const void *h, int64_t h_stride, const void *weight,
                                        int weight_dtype, double eps, int relu, void *grad_x, int64_t grad_x_stride,
                                        float *grad_weight, void *workspace, int64_t workspace_bytes, int64_t rows,
                                        int64_t width, int dtype, void *stream) {
    if (const int rc = check_norm(rows, width, dtype, weight_dtype)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GNNAGG_REQUIRE(grad_weight, "null grad_weight");
    if (rows == 0) return launch_column_reduce(nullptr, 0, width, grad_weight, st);  // zeros
    GNNAGG_REQUIRE(grad_y && h && weight && grad_x && workspace, "null grad_y/h/weight/grad_x/workspace");
    GNNAGG_REQUIRE(grad_y_stride >= width && h_stride >= width && grad_x_stride >= width && (!grad_h || grad_h_stride >= width),
                   "a row stride is below the width");
    GNNAGG_REQUIRE(workspace_bytes >= gnnagg_rms_norm_backward_workspace_bytes(rows, width) &&
                       reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
                   "workspace of %lld bytes is too small or misaligned", (long long)workspace_bytes);
    NormBackwardArgs p{grad_y, grad_h, h, weight, grad_x, static_cast<float *>(workspace), grad_y_stride, grad_h_stride,
                       h_stride, grad_x_stride, rows, width, eps, relu, weight_dtype == GNNAGG_BF16};
    const bool vec = vec4_rows(grad_y, grad_y_stride, width, dtype) && vec4_rows(grad_h, grad_h_stride, width, dtype) &&
                     vec4_rows(h, h_stride, width, dtype) && vec4_rows(grad_x, grad_x_stride, width, dtype) &&
                     vec4_rows(weight, 4, width, weight_dtype);
    const int64_t blocks = backward_blocks(rows, width);
    for_norm_shape(norm_shape(width), [&](auto tpr, auto nv) {
        constexpr int kTpr = decltype(tpr)::value, kNv = decltype(nv)::value;
        auto go = [&](auto type, auto v) {
            hipLaunchKernelGGL((rms_norm_backward_kernel<decltype(type), kTpr, kNv, decltype(v)::value>),
                               dim3((unsigned)blocks), dim3(block_of(kTpr)), 0, st, p);
        };
        if (dtype == GNNAGG_F32) {
            if (vec) go(float(), std::true_type());
            else go(float(), std::false_type());
        } else {
            if (vec) go(bf16_t(), std::true_type());
            else go(bf16_t(), std::false_type());
        }
    });
    GNNAGG_HIP(hipGetLastError());
    return launch_column_reduce(p.partial, blocks, width, grad_weight, st);
}
