// Into the 8-bit format (fp8_format.h): rows in blocks of 128 along them, weights in blocks of 128 x 128, stored twice --
// by output for the forward product, by input for the input gradient.  Streaming kernels, bound by HBM: fp32 rows cost
// 5 bytes a value, bf16 rows 3 (with four operands in turn: 300 007 x 256 fp32 68 us = 5.6 TB/s, x 172 52 us, 8192 x 4096 bf16
// 24 us = 4.2 TB/s, a bf16 weight of 4096 x 4096 in both orders 17 us; inside a layer's pass, behind kernels whose results
// are still being written back, 87 us for the first two on average, 25 and 25).
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

// Half a wave owns a block of 128 values of a row, four a lane: one wide load, a maximum over 32 lanes, one 4-byte store.
// (The maximum on the vector unit: through LDS 63 us against 56 for 300 007 x 172 fp32, 24 against 21 for 8192 x 4096 bf16,
// each on one operand again and again.)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T *__restrict__ x, int64_t x_stride,
                                                            uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                            uint32_t rows, int64_t width, uint32_t blocks) {
    const uint32_t l = threadIdx.x % 32;
    const uint64_t total = (uint64_t)rows * blocks;  // below 2^31: the host cuts longer arrays
    for (uint32_t id = blockIdx.x * 8 + threadIdx.x / 32; id < total; id += gridDim.x * 8) {
        const uint32_t row = id / blocks, block = id - row * blocks;
        const int64_t c = (int64_t)block * kBlock8 + 4 * l;
        const f32x4 v = load4<VEC>(x + (int64_t)row * x_stride, c, width);
        const int e = block_exponent(__uint_as_float(lanes_max(__float_as_uint(finite_magnitude(v)))));
        reinterpret_cast<uint32_t *>(codes)[(uint64_t)id * 32 + l] = encode4(v, pow2(-e));
        if (l == 0) scales[id] = (uint8_t)(e + 127);
    }
}

// A thread block per 128 x 128 block of W: thread t holds columns 4 (t % 32) .. + 3 of rows t / 32 + 8 i.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T *__restrict__ w, int64_t w_stride,
                                                              uint8_t *__restrict__ by_output,
                                                              uint8_t *__restrict__ by_input,
                                                              uint8_t *__restrict__ scales, int64_t k, int64_t n,
                                                              int64_t k_padded, int64_t n_padded) {
    __shared__ float tops[4];
    __shared__ uint32_t tile[kBlock8][kBlock8 / 4 + 1];  // codes, row by row; the odd pitch spreads columns over the banks
    const int64_t k0 = (int64_t)blockIdx.y * kBlock8, n0 = (int64_t)blockIdx.x * kBlock8;
    const int cq = (int)threadIdx.x % 32, r0 = (int)threadIdx.x / 32;
    f32x4 v[16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t row = k0 + r0 + 8 * i;
        v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (row < k) v[i] = load4<VEC>(w + row * w_stride, (int64_t)(n0 + 4 * cq), n);
        top = fmaxf(top, finite_magnitude(v[i]));
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
    const int e = block_exponent(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    const float inv = pow2(-e);
    if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * (n_padded / kBlock8) + blockIdx.x] = (uint8_t)(e + 127);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t row = k0 + r0 + 8 * i;
        const uint32_t c = encode4(v[i], inv);
        if (by_input && row < k) *reinterpret_cast<uint32_t *>(by_input + row * n_padded + n0 + 4 * cq) = c;
        tile[r0 + 8 * i][cq] = c;
    }
    if (!by_output) return;
    __syncthreads();
    // output column n0 + j: its 128 codes along k, four a thread
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = r0 + 8 * i;  // column of the block
        if (n0 + j >= n) continue;
        uint32_t c = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) c |= ((tile[4 * cq + q][j / 4] >> (8 * (j % 4))) & 0xffu) << (8 * q);
        *reinterpret_cast<uint32_t *>(by_output + (n0 + j) * k_padded + k0 + 4 * cq) = c;
    }
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_fp8_quantize_rows(const void *x, int64_t x_stride, uint8_t *codes, uint8_t *scales, int64_t rows,
                                        int64_t width, int dtype, void *stream) {
    GNNAGG_REQUIRE(rows >= 0 && width >= 0, "negative size");
    GNNAGG_REQUIRE(known_dtype(dtype), "unknown dtype");
    if (rows == 0 || width == 0) return GNNAGG_OK;
    GNNAGG_REQUIRE(x && codes && scales, "null x/codes/scales");
    GNNAGG_REQUIRE(x_stride >= width, "a row stride is below the width");
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 4 == 0, "codes must be 4-byte aligned");
    if (width > (int64_t(1) << 30)) return fail(GNNAGG_ERR_UNSUPPORTED, "width %lld", (long long)width);
    const int64_t blocks = pad128(width) / kBlock8;
    const bool vec = vec4_rows(x, x_stride, width, dtype);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t most = (int64_t(1) << 30) / blocks;  // rows a launch: its task numbers stay in 32 bits
    for (int64_t r = 0; r < rows; r += most) {
        const int64_t part = rows - r < most ? rows - r : most;
        const int64_t need = (part * blocks + 7) / 8;
        const dim3 grid((unsigned)(need < 256 * 64 ? need : 256 * 64));
        auto go = [&](auto type, auto v) {
            using T = decltype(type);
            hipLaunchKernelGGL((quantize_rows_kernel<T, decltype(v)::value>), grid, dim3(256), 0, st,
                               static_cast<const T *>(x) + r * x_stride, x_stride, codes + r * blocks * kBlock8,
                               scales + r * blocks, (uint32_t)part, width, (uint32_t)blocks);
        };
        if (dtype == GNNAGG_F32) {
            if (vec) go(float(), std::true_type());
            else go(float(), std::false_type());
        } else {
            if (vec) go(bf16_t(), std::true_type());
            else go(bf16_t(), std::false_type());
        }
        GNNAGG_HIP(hipGetLastError());
    }
    return GNNAGG_OK;
}

extern "C" int gnnagg_fp8_quantize_weight(const void *w, int64_t w_stride, uint8_t *codes_by_output,
                                          uint8_t *codes_by_input, uint8_t *scales, int64_t k, int64_t n, int dtype,
                                          void *stream) {
    GNNAGG_REQUIRE(k >= 0 && n >= 0, "negative size");
    GNNAGG_REQUIRE(known_dtype(dtype), "unknown dtype");
    if (k == 0 || n == 0) return GNNAGG_OK;
    GNNAGG_REQUIRE(w && scales && (codes_by_output || codes_by_input), "null w/scales/codes");
    GNNAGG_REQUIRE(w_stride >= n, "the row stride is below the width");
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(codes_by_output) % 4 == 0 && reinterpret_cast<uintptr_t>(codes_by_input) % 4 == 0,
                   "codes must be 4-byte aligned");
    const int64_t kb = pad128(k) / kBlock8, nb = pad128(n) / kBlock8;
    if (kb > 65535 || nb > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "a weight of %lld x %lld", (long long)k, (long long)n);
    const bool vec = vec4_rows(w, w_stride, n, dtype);
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto go = [&](auto type, auto v) {
        using T = decltype(type);
        hipLaunchKernelGGL((quantize_weight_kernel<T, decltype(v)::value>), dim3((unsigned)nb, (unsigned)kb), dim3(256), 0,
                           st, static_cast<const T *>(w), w_stride, codes_by_output, codes_by_input, scales, k, n,
                           kb * kBlock8, nb * kBlock8);
    };
    if (dtype == GNNAGG_F32) {
        if (vec) go(float(), std::true_type());
        else go(float(), std::false_type());
    } else {
        if (vec) go(bf16_t(), std::true_type());
        else go(bf16_t(), std::false_type());
    }
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}
