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
// last place.  The weight gradient is summed in fp32 by each thread over its rows (64 bits there would double its registers;
// 62 additions for 1 M rows of 47, 1.6e-7 off) and leaves each block as one partial row; a second launch adds those in 64
// bits, in a fixed order.
// Measured: 500 009 x 256 fp32 with a residual to 8 bits 304 us = 5.4 TB/s; forward and backward of 1 000 003 x 47 fp32
// 197 us, of 8192 x 5120 bf16 with a residual 142 us = 4.7 TB/s (a copy of this machine: 4.66 TB/s).
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

struct NormArgs {
    const void *x, *residual, *weight;
    void *h, *y;
    uint8_t *codes, *scales;
    int64_t x_stride, residual_stride, h_stride, y_stride;
    int64_t rows;
    int width, padded;
    double inv_width, eps;
    int relu, weight_bf16;
};

struct NormBackwardArgs {
    const void *grad_y, *grad_h, *h, *weight;
    void *grad_x;
    float *partial;
    int64_t grad_y_stride, grad_h_stride, h_stride, grad_x_stride;
    int64_t rows;
    int width;
    double inv_width, eps;
    int relu, weight_bf16;
};

template <int W>
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int s = W / 2; s >= 1; s >>= 1) v = fmaxf(v, __shfl_xor(v, s, W));
    return v;
}

// The sums over a row's TPR threads, in every one of them, of U rows at once.  `slot`: U x 16 doubles of LDS where the row
// has a whole block; two of them, taken in turn, so that one barrier a sum is enough.
template <int TPR, int U>
__device__ __forceinline__ void row_sums(double (&v)[U], double (*slot)[16]) {
#pragma unroll
    for (int s = (TPR < 64 ? TPR : 64) / 2; s >= 1; s >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] += __shfl_xor(v[u], s, TPR < 64 ? TPR : 64);
    if constexpr (TPR > 64) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (threadIdx.x % 64 == 0) slot[u][threadIdx.x / 64] = v[u];
        lds_barrier();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = slot[u][0];
#pragma unroll
            for (int q = 1; q < TPR / 64; ++q) v[u] += slot[u][q];
        }
    }
}

// Which columns run k of a row's thread l holds: four neighbours, or, SPREAD, one of each four stretches of TPR.  Rows that
// cannot be moved in wide pieces are read and written in stretches: a store of every fourth value is a request for every
// line (1 M x 47: 133 + 193 us forward and backward, 78 + 135 in stretches).
template <int TPR, bool VEC, bool SPREAD>
struct Columns {
    template <typename T>
    static __device__ __forceinline__ typename RawOf<T>::type load(const T *row, int l, int k, int width) {
        if constexpr (!SPREAD) {
            return load4_raw<VEC>(row, 4 * (l + k * TPR), width);
        } else {
            typename RawOf<T>::type v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (4 * k + j) * TPR + l;
                const T x = row[c < width ? c : width - 1];
                if constexpr (sizeof(T) == 4) v[j] = c < width ? x : 0.0f;
                else v[j] = c < width ? x.bits : (unsigned short)0;
            }
            return v;
        }
    }
    template <typename T>
    static __device__ __forceinline__ void store(T *row, int l, int k, int width, const f32x4 v) {
        if constexpr (!SPREAD) {
            store4<VEC>(row, 4 * (l + k * TPR), width, v);
        } else {
            const f32x4 r = rounded(row, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = (4 * k + j) * TPR + l;
                if (c < width) {
                    if constexpr (sizeof(T) == 4) row[c] = r[j];
                    else row[c].bits = (unsigned short)(__float_as_uint(r[j]) >> 16);
                }
            }
        }
    }
    static __device__ __forceinline__ f32x4 weight(const void *w, int is_bf16, int l, int k, int width) {
        return is_bf16 ? widen(load(static_cast<const bf16_t *>(w), l, k, width))
                       : widen(load(static_cast<const float *>(w), l, k, width));
    }
};

// r of U rows
template <int TPR, int U, int NV>
__device__ __forceinline__ void inverse_rms(const f32x4 (&h)[U][NV], double inv_width, double eps, double (*slot)[16],
                                            float (&r)[U]) {
    double q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        q[u] = 0.0;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) q[u] = __builtin_fma((double)h[u][k][j], (double)h[u][k][j], q[u]);
    }
    row_sums<TPR, U>(q, slot);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        // 1 / sqrt: the hardware's estimate (2^-26) and a Newton step, beyond fp32 by far.  The library's square root and
        // division in 64 bits are some 60 instructions (8192 x 5120 bf16, forward: 103 us with them, 88 without).
        // (An infinite a has the root's inverse 0, a zero one infinity, and the step would make NaN of either.)
        const double a = q[u] * inv_width + eps, y = __builtin_amdgcn_rsq(a), step = __builtin_fma(-0.5 * a * y, y, 1.5);
        r[u] = (float)(step == step ? y * step : y);
    }
}

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }
// Rows a thread works on at once: narrow rows are a few hundred bytes a wave, too little on the way to hide the way.
constexpr int rows_at_once(int tpr, int nv) { return tpr > 64 ? 1 : nv == 1 ? 4 : nv == 2 ? 2 : 1; }

template <typename T, int TPR, int NV, bool VEC, bool FP8>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_kernel(const NormArgs p) {
    constexpr int kGroups = block_of(TPR) / TPR, U = rows_at_once(TPR, NV);
    constexpr bool kAhead = TPR == 256 || (TPR == 1024 && NV <= 2);  // a block's next row is asked for before its barrier
    typedef typename RawOf<T>::type Raw;
    typedef Columns<TPR, VEC, !VEC && !FP8> C;
    __shared__ double slots[2][1][16];
    const int l = (int)threadIdx.x % TPR;
    f32x4 w[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) w[k] = C::weight(p.weight, p.weight_bf16, l, k, p.width);
    Raw x[U][NV], res[U][NV];
    auto load = [&](int64_t row) {  // rows row, row + kGroups, ...; those past the end read the last one
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t m = row + u * kGroups < p.rows ? row + u * kGroups : p.rows - 1;
            const T *xr = static_cast<const T *>(p.x) + m * p.x_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) x[u][k] = C::load(xr, l, k, p.width);
            if (p.residual) {
                const T *rr = static_cast<const T *>(p.residual) + m * p.residual_stride;
#pragma unroll
                for (int k = 0; k < NV; ++k) res[u][k] = C::load(rr, l, k, p.width);
            }
        }
    };
    const int64_t stride = (int64_t)gridDim.x * kGroups * U;
    int64_t first = (int64_t)blockIdx.x * kGroups * U + (int)threadIdx.x / TPR;
    int parity = 0;
    if (kAhead) load(first);
    // the threads of a row stay or leave together (a whole block's where there is a barrier)
    for (; first < p.rows; first += stride, parity ^= 1) {
        if (!kAhead) load(first);
        f32x4 h[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < NV; ++k) h[u][k] = widen(x[u][k]);
            if (p.residual) {
#pragma unroll
                for (int k = 0; k < NV; ++k) h[u][k] = rounded(static_cast<const T *>(p.x), h[u][k] + widen(res[u][k]));
                const int64_t row = first + u * kGroups;
                if (U == 1 || row < p.rows) {
                    T *ho = static_cast<T *>(p.h) + row * p.h_stride;
#pragma unroll
                    for (int k = 0; k < NV; ++k) C::store(ho, l, k, p.width, h[u][k]);
                }
            }
        }
        if (kAhead && first + stride < p.rows) load(first + stride);
        float r[U];
        inverse_rms<TPR, U, NV>(h, p.inv_width, p.eps, slots[parity], r);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = first + u * kGroups;
            if (U > 1 && row >= p.rows) continue;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                h[u][k] = h[u][k] * r[u] * w[k];
                if (p.relu) {  // (a NaN stays one)
#pragma unroll
                    for (int j = 0; j < 4; ++j) h[u][k][j] = h[u][k][j] < 0.0f ? 0.0f : h[u][k][j];
                }
            }
            if constexpr (!FP8) {
                T *y = static_cast<T *>(p.y) + row * p.y_stride;
#pragma unroll
                for (int k = 0; k < NV; ++k) C::store(y, l, k, p.width, h[u][k]);
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
                    for (int k = k0; k < k0 + kRuns && k < NV; ++k) top = fmaxf(top, finite_magnitude(h[u][k]));
                    const int e = block_exponent(wave_max<kThreads>(top));
                    const float inv = pow2(-e);
#pragma unroll
                    for (int k = k0; k < k0 + kRuns; ++k) {      // (runs past NV hold a narrow row's padding)
                        const int c = 4 * (l + k * TPR);
                        if (c >= p.padded) continue;
                        *reinterpret_cast<uint32_t *>(codes + c) = k < NV ? encode4(h[u][k < NV ? k : 0], inv) : 0u;
                        if (c % kBlock8 == 0) scales[c / kBlock8] = (uint8_t)(e + 127);
                    }
                }
            }
        }
    }
}

template <typename T, int TPR, int NV, bool VEC>
__global__ __launch_bounds__(block_of(TPR)) void rms_norm_backward_kernel(const NormBackwardArgs p) {
    constexpr int kGroups = block_of(TPR) / TPR, U = rows_at_once(TPR, NV);
    constexpr bool kAhead = TPR == 256;
    constexpr bool kLean = TPR == 1024;  // 128 registers a thread: the weight and grad_h are read where they are used
    typedef typename RawOf<T>::type Raw;
    typedef Columns<TPR, VEC, !VEC> C;
    __shared__ double slots[2][2][1][16];
    __shared__ f32x4 sums[kGroups > 1 ? 256 : 1];
    const int l = (int)threadIdx.x % TPR;
    f32x4 w_kept[kLean ? 1 : NV], gw_sum[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (!kLean) w_kept[kLean ? 0 : k] = C::weight(p.weight, p.weight_bf16, l, k, p.width);
        gw_sum[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto weight = [&](int k) { return kLean ? C::weight(p.weight, p.weight_bf16, l, k, p.width) : w_kept[kLean ? 0 : k]; };
    Raw hx[U][NV], gx[U][NV], gh[U][NV];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t m = row + u * kGroups < p.rows ? row + u * kGroups : p.rows - 1;
            const T *hr = static_cast<const T *>(p.h) + m * p.h_stride;
            const T *gr = static_cast<const T *>(p.grad_y) + m * p.grad_y_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) hx[u][k] = C::load(hr, l, k, p.width);
#pragma unroll
            for (int k = 0; k < NV; ++k) gx[u][k] = C::load(gr, l, k, p.width);
            if (!kLean && p.grad_h) {
                const T *sr = static_cast<const T *>(p.grad_h) + m * p.grad_h_stride;
#pragma unroll
                for (int k = 0; k < NV; ++k) gh[u][k] = C::load(sr, l, k, p.width);
            }
        }
    };
    const int64_t stride = (int64_t)gridDim.x * kGroups * U;
    int64_t first = (int64_t)blockIdx.x * kGroups * U + (int)threadIdx.x / TPR;
    int parity = 0;
    if (kAhead) load(first);
    for (; first < p.rows; first += stride, parity ^= 1) {
        if (!kAhead) load(first);
        f32x4 h[U][NV], g[U][NV], more[U][NV];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                h[u][k] = widen(hx[u][k]);
                g[u][k] = widen(gx[u][k]);
                if (!kLean) more[u][k] = p.grad_h ? widen(gh[u][k]) : f32x4{0.f, 0.f, 0.f, 0.f};
            }
        if (kAhead && first + stride < p.rows) load(first + stride);
        float r[U];
        inverse_rms<TPR, U, NV>(h, p.inv_width, p.eps, slots[parity][0], r);
        double s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.0;
            const bool in = U == 1 || first + u * kGroups < p.rows;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const f32x4 z = h[u][k] * r[u], w = weight(k);
                if (p.relu) {  // exactly the values that the forward cut or found at zero
                    const f32x4 y = z * w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) g[u][k][j] = y[j] > 0.0f ? g[u][k][j] : 0.0f;
                }
                if (in) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) gw_sum[k][j] = __builtin_fmaf(g[u][k][j], z[j], gw_sum[k][j]);
                }
                g[u][k] = g[u][k] * w;
#pragma unroll
                for (int j = 0; j < 4; ++j) s[u] = __builtin_fma((double)g[u][k][j], (double)h[u][k][j], s[u]);
            }
        }
        row_sums<TPR, U>(s, slots[parity][1]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = first + u * kGroups;
            if (U > 1 && row >= p.rows) continue;
            const float t = (float)(s[u] * (double)r[u] * p.inv_width);  // (r^3 would leave fp32's range for large rows)
            T *out = static_cast<T *>(p.grad_x) + row * p.grad_x_stride;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                f32x4 d = (g[u][k] - h[u][k] * r[u] * t) * r[u];
                if (p.grad_h) d += kLean ? widen(C::load(static_cast<const T *>(p.grad_h) + row * p.grad_h_stride, l, k, p.width)) : more[u][k];
                C::store(out, l, k, p.width, d);
            }
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
        if (threadIdx.x < TPR) Columns<TPR, false, !VEC>::store(partial, l, k, p.width, total);
    }
}

// 32 columns a block, 32 slices of the partial rows, added in slice order, in 64 bits (hidden behind the loads; in 32 the
// chain would be as long as a thread's own over its rows)
__global__ __launch_bounds__(1024) void column_reduce_kernel(const float *__restrict__ partial, int64_t blocks,
                                                             int64_t width, float *__restrict__ out) {
    __shared__ double sums[32][33];
    const int col = (int)threadIdx.x % 32, slice = (int)threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    double a = 0.0;
    if (c < width) {
#pragma unroll 8
        for (int64_t b = slice; b < blocks; b += 32) a += (double)partial[b * width + c];
    }
    sums[slice][col] = a;
    __syncthreads();
    if (slice == 0 && c < width) {
        for (int q = 1; q < 32; ++q) a += sums[q][col];
        out[c] = (float)a;
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
    const int64_t at_once = block_of(tpr) / tpr * rows_at_once(tpr, norm_shape(width).nv);
    const int64_t need = (rows + at_once - 1) / at_once;
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
        constexpr int kTpr = decltype(tpr)::value, kNv = decltype(nv)::value;
        constexpr int kAtOnce = block_of(kTpr) / kTpr * rows_at_once(kTpr, kNv);
        const int64_t need = (p.rows + kAtOnce - 1) / kAtOnce;
        const int64_t most = kTpr > 64 ? 256 * 4 : 256 * 32;  // blocks that keep a row ahead stay for several rows
        const dim3 grid((unsigned)(need < most ? need : most));
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
               rows, (int)width, (int)pad128(width), 1.0 / (double)width, eps, relu, weight_dtype == GNNAGG_BF16};
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
                       h_stride, grad_x_stride, rows, (int)width, 1.0 / (double)width, eps, relu, weight_dtype == GNNAGG_BF16};
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
