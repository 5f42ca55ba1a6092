// AdamW over many tensors at once: one launch for up to kTensors of them (their addresses and sizes travel in the kernel's
// arguments: no table in device memory to fill, nothing a captured graph could find changed), one block per 4096 elements.
//
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: 28 bytes an element with fp32 states, 16 + 4/128 with 8-bit ones.  With 8-bit states half a wave holds a
// block of 128 elements, four a lane, so that a block's scale is a maximum over 32 lanes and every load and store stays
// whole: nothing is read twice.  The step counts live on the device and are raised by a launch of their own in front
// (every block of a tensor reads its count, so none of them may write it).
// Measured: 128 M elements with 8-bit states 437 us = 4.7 TB/s; 200 bf16 tensors of 60 M elements with masters 379 us =
// 4.4 TB/s; ten small tensors 9.7 us from call to call.
#include "fp8_format.h"

namespace gnnagg {
namespace {

constexpr int kTensors = 48;      // 48 records are 3.3 KB of the 4 KB a launch's arguments may take
constexpr int kChunk = 4096;      // elements per block

struct AdamwArgs {
    gnnagg_adamw_tensor t[kTensors];
    int32_t first_chunk[kTensors + 1];  // the blocks of tensor i: [first_chunk[i], first_chunk[i + 1])
    int32_t count;
    uint32_t seed, first;
    const int32_t *steps;
    const float *lr_tensor;
    float lr, beta1, beta2, rest1, rest2, eps, weight_decay;  // rest = 1 - beta, taken in 64 bits: 1 - 0.999f is 1e-5 off
    float log_beta1, log_beta2;
};
static_assert(sizeof(AdamwArgs) <= 4096, "kernel arguments");

__global__ void raise_steps_kernel(int32_t *steps, int64_t n) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) steps[i] += 1;
}

// 20 random bits of element j: a multiply-xorshift hash of j and the key of (seed, tensor, step).  The multipliers are
// published ones: the first two from C. Wellons' search for 32-bit hashes of low bias, the third a prime of Y. Collet's; the
// key's are 2^32 over the golden ratio and one of A. Appleby's.
__device__ __forceinline__ uint32_t random20(uint32_t key, uint32_t j) {
    uint32_t x = (j ^ key) * 0x7FEB352Du;
    x = (x ^ (x >> 15)) * 0x846CA68Bu;
    x = (x ^ (x >> 13)) * 0xC2B2AE3Du;
    return x >> 12;
}

// y in [0, 448] to one of its two neighbouring e4m3 values, up with the odds of the distance; above zero stays above zero
__device__ __forceinline__ float round_by_odds(float y, uint32_t bits20) {
    float t;
    if (y >= 0.015625f)  // normal codes have three mantissa bits: the 20 below them carry or are cut
        t = __uint_as_float((__float_as_uint(y) + bits20) & 0xfff00000u);
    else                 // multiples of 2^-9 below 2^-6
        t = __builtin_floorf(__builtin_fmaf(y, 512.0f, (float)bits20 * 0x1p-20f)) * 0x1p-9f;
    t = t > 448.0f ? 448.0f : t;
    t = t < 0x1p-9f ? 0x1p-9f : t;
    return y > 0.0f ? t : (y == 0.0f ? 0.0f : y);  // (NaN stays NaN)
}

__device__ __forceinline__ float half_wave_max(float v) {
#pragma unroll
    for (int s = 16; s >= 1; s >>= 1) v = fmaxf(v, __shfl_xor(v, s, 32));
    return v;
}

template <typename P, typename G, bool EIGHT, bool VEC>
__device__ __forceinline__ void update_chunk(const AdamwArgs &a, const gnnagg_adamw_tensor &t, int tensor, int64_t begin) {
    constexpr bool kMaster = sizeof(P) == 2;
    const int32_t step = a.steps[tensor];
    const float lr = a.lr_tensor ? *a.lr_tensor : a.lr;
    const float correction1 = -expm1f((float)step * a.log_beta1);
    const float correction2 = -expm1f((float)step * a.log_beta2);
    const float decay = 1.0f - lr * a.weight_decay;
    const float rate = lr / correction1;
    const float inv_correction2 = 1.0f / correction2;
    const uint32_t key = a.seed + (a.first + (uint32_t)tensor) * 0x9E3779B9u + (uint32_t)step * 0x85EBCA6Bu;

    constexpr int kRuns = kChunk / (4 * 256);
    f32x4 p[kRuns], g[kRuns], m[kRuns], v[kRuns];
    float *weights = kMaster ? t.master : static_cast<float *>(t.param);
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int64_t c = begin + 4 * ((int)threadIdx.x + 256 * k);
        g[k] = load4<VEC>(static_cast<const G *>(t.grad), c, t.n);
        p[k] = load4<VEC>(weights, c, t.n);
        if constexpr (!EIGHT) {
            m[k] = load4<VEC>(static_cast<const float *>(t.exp_avg), c, t.n);
            v[k] = load4<VEC>(static_cast<const float *>(t.exp_avg_sq), c, t.n);
        } else {
            uint32_t cm = 0, cu = 0;
            const uint8_t *mc = static_cast<const uint8_t *>(t.exp_avg), *uc = static_cast<const uint8_t *>(t.exp_avg_sq);
            if (VEC) {
                if (c < t.n) {
                    cm = *reinterpret_cast<const uint32_t *>(mc + c);
                    cu = *reinterpret_cast<const uint32_t *>(uc + c);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < t.n) {
                        cm |= (uint32_t)mc[c + j] << (8 * j);
                        cu |= (uint32_t)uc[c + j] << (8 * j);
                    }
            }
            const bool any = c < t.n;
            const float sm = any ? pow2((int)t.exp_avg_scales[c / kBlock8] - 127) : 0.0f;
            const float su = any ? pow2((int)t.exp_avg_sq_scales[c / kBlock8] - 127) : 0.0f;
            m[k] = decode4(cm) * sm;
            const f32x4 u = decode4(cu) * su;
            v[k] = u * u;
        }
    }
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int64_t c = begin + 4 * ((int)threadIdx.x + 256 * k);
        f32x4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[k][j] = a.beta1 * m[k][j] + a.rest1 * g[k][j];
            v[k][j] = a.beta2 * v[k][j] + a.rest2 * (g[k][j] * g[k][j]);
            const float denom = __builtin_sqrtf(v[k][j] * inv_correction2) + a.eps;
            p[k][j] = p[k][j] * decay - rate * m[k][j] / denom;
        }
        store4<VEC>(weights, c, t.n, p[k]);
        if constexpr (kMaster) store4<VEC>(static_cast<P *>(t.param), c, t.n, p[k]);
        if constexpr (!EIGHT) {
            store4<VEC>(static_cast<float *>(t.exp_avg), c, t.n, m[k]);
            store4<VEC>(static_cast<float *>(t.exp_avg_sq), c, t.n, v[k]);
        } else {
            // values past the end are zeros here: g, m and v were loaded as such
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = __builtin_sqrtf(v[k][j]);
            const int em = block_exponent(half_wave_max(finite_magnitude(m[k])));
            const int eu = block_exponent(half_wave_max(finite_magnitude(u)));
            const uint32_t cm = encode4(m[k], pow2(-em));
            const float inv = pow2(-eu);
#pragma unroll
            for (int j = 0; j < 4; ++j) u[j] = round_by_odds(nan_unless_finite(u[j]) * inv, random20(key, (uint32_t)(c + j)));
            const uint32_t cu = encode4(u, 1.0f);
            uint8_t *mc = static_cast<uint8_t *>(t.exp_avg), *uc = static_cast<uint8_t *>(t.exp_avg_sq);
            if (VEC) {
                if (c < t.n) {
                    *reinterpret_cast<uint32_t *>(mc + c) = cm;
                    *reinterpret_cast<uint32_t *>(uc + c) = cu;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < t.n) {
                        mc[c + j] = (uint8_t)(cm >> (8 * j));
                        uc[c + j] = (uint8_t)(cu >> (8 * j));
                    }
            }
            if (c % kBlock8 == 0 && c < t.n) {
                t.exp_avg_scales[c / kBlock8] = (uint8_t)(em + 127);
                t.exp_avg_sq_scales[c / kBlock8] = (uint8_t)(eu + 127);
            }
        }
    }
}

template <typename P, typename G, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(const AdamwArgs a) {
    const int32_t chunk = (int32_t)blockIdx.x;
    int lo = 0, hi = a.count;  // the tensor whose blocks hold this one
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.first_chunk[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    const gnnagg_adamw_tensor &t = a.t[lo];
    const int64_t begin = (int64_t)(chunk - a.first_chunk[lo]) * kChunk;
    // wide loads where the tensor's arrays are aligned for them and the chunk holds whole runs of four
    const uintptr_t places = reinterpret_cast<uintptr_t>(t.grad) * (16 / (4 * sizeof(G))) |
                             (sizeof(P) == 2 ? reinterpret_cast<uintptr_t>(t.param) * 2 | reinterpret_cast<uintptr_t>(t.master)
                                             : reinterpret_cast<uintptr_t>(t.param)) |
                             reinterpret_cast<uintptr_t>(t.exp_avg) * (EIGHT ? 4 : 1) |
                             reinterpret_cast<uintptr_t>(t.exp_avg_sq) * (EIGHT ? 4 : 1);
    const bool whole = t.n - begin >= kChunk || t.n % 4 == 0;
    if (places % 16 == 0 && whole) update_chunk<P, G, EIGHT, true>(a, t, lo, begin);
    else update_chunk<P, G, EIGHT, false>(a, t, lo, begin);
}

template <typename P, typename G>
void launch(const AdamwArgs &a, int64_t blocks, bool eight, hipStream_t st) {
    if (eight) hipLaunchKernelGGL((adamw_kernel<P, G, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((adamw_kernel<P, G, false>), dim3((unsigned)blocks), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_adamw_step(const gnnagg_adamw_tensor *tensors, int64_t count, int32_t *steps, int param_dtype,
                                 int grad_dtype, int state_bits, double lr, const float *lr_tensor, double beta1,
                                 double beta2, double eps, double weight_decay, uint32_t seed, int64_t first,
                                 void *stream) {
    GNNAGG_REQUIRE(count >= 0 && first >= 0, "negative count");
    if (count == 0) return GNNAGG_OK;
    GNNAGG_REQUIRE(tensors && steps, "null tensors/steps");
    GNNAGG_REQUIRE(known_dtype(param_dtype) && known_dtype(grad_dtype), "unknown dtype");
    GNNAGG_REQUIRE(state_bits == 32 || state_bits == 8, "states have 32 or 8 bits, not %d", state_bits);
    GNNAGG_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "beta1 and beta2 must be in [0, 1)");
    const bool eight = state_bits == 8, master = param_dtype == GNNAGG_BF16;
    for (int64_t i = 0; i < count; ++i) {
        const gnnagg_adamw_tensor &t = tensors[i];
        GNNAGG_REQUIRE(t.n >= 0, "tensor %lld: negative size", (long long)i);
        if (t.n == 0) continue;
        GNNAGG_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq, "tensor %lld: null param/grad/state", (long long)i);
        GNNAGG_REQUIRE(!eight || (t.exp_avg_scales && t.exp_avg_sq_scales), "tensor %lld: null scales", (long long)i);
        GNNAGG_REQUIRE(!master || t.master, "tensor %lld: a bf16 parameter needs its fp32 master", (long long)i);
        if (t.n > (int64_t(1) << 42)) return fail(GNNAGG_ERR_UNSUPPORTED, "tensor %lld: too many elements", (long long)i);
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(raise_steps_kernel, dim3(grid_for(count, 256)), dim3(256), 0, st, steps, count);
    GNNAGG_HIP(hipGetLastError());
    AdamwArgs a{};
    a.seed = seed;
    a.lr_tensor = lr_tensor;
    a.lr = (float)lr;
    a.beta1 = (float)beta1;
    a.beta2 = (float)beta2;
    a.rest1 = (float)(1.0 - beta1);
    a.rest2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.weight_decay = (float)weight_decay;
    a.log_beta1 = beta1 > 0.0 ? (float)__builtin_log(beta1) : -kFloatMax;
    a.log_beta2 = beta2 > 0.0 ? (float)__builtin_log(beta2) : -kFloatMax;
    for (int64_t i = 0; i < count;) {
        const int64_t begin = i;
        int64_t blocks = 0;
        for (a.count = 0; a.count < kTensors && i < count; ++a.count, ++i) {
            const int64_t need = (tensors[i].n + kChunk - 1) / kChunk;
            if (blocks + need > 0x7fffffff) break;
            a.t[a.count] = tensors[i];
            a.first_chunk[a.count] = (int32_t)blocks;
            blocks += need;
        }
        a.first_chunk[a.count] = (int32_t)blocks;
        a.first = (uint32_t)(first + begin);
        a.steps = steps + begin;
        if (blocks == 0) continue;
        if (param_dtype == GNNAGG_F32) {
            if (grad_dtype == GNNAGG_F32) launch<float, float>(a, blocks, eight, st);
            else launch<float, bf16_t>(a, blocks, eight, st);
        } else {
            if (grad_dtype == GNNAGG_F32) launch<bf16_t, float>(a, blocks, eight, st);
            else launch<bf16_t, bf16_t>(a, blocks, eight, st);
        }
        GNNAGG_HIP(hipGetLastError());
    }
    return GNNAGG_OK;
}
