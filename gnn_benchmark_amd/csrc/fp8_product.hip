// Products of matrices in the 8-bit format (fp8_format.h):
//
//     out[m, n] = sum over blocks b of 2^(sx[m, b] + sw[b, n / 128]) sum over k in b of x[m, k] w[n, k]   (+ bias[n])
//
// in two forms, chosen by the type of the result:
//
//   bf16   v_mfma_scale_f32_*_f8f6f4 on the codes themselves.  Its scale operands are the format's own bytes: the matrix
//          unit multiplies by the two powers of two as it accumulates, in fp32, and no block's partial sum ever leaves it.
//          Of the eight products of a lane's eight neighbouring codes this instruction (and the unscaled 8-bit one) keeps
//          what lies above 2^-13 of the largest one's power of two; measured, random operands come out 1.5e-5 off (2-norm),
//          below half a percent of what storing bf16 rounds away.
//   fp32   the codes become bf16 values, scale included, in one v_cvt_scalef32_pk_bf16_fp8 for two of them -- exactly, on
//          their way from LDS into the matrix unit -- and multiply on v_mfma_f32_*_bf16: every product exact, sums fp32
//          (2e-8 off on the same operands), at half the matrix rate.
//
// Both operands have the contraction index contiguous, 128 codes = 128 bytes a block, so one pipeline stage is one block: a 128-byte piece of every row of
// the tile, copied straight from global memory into LDS (no registers between), double-buffered, one barrier a stage.
//
// w is the MFMA's first operand: a lane then owns runs of four consecutive columns of one row of the result.
//
// The 16-byte pieces of a staged row are stored at piece ^ ((row / 2) % 8): the 16 lanes of a ds_read_b128 phase read the
// same piece of 16 neighbouring rows, and two rows fill the 64 banks, so every phase touches each bank once.
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct ProductArgs {
    const uint8_t *x, *x_scales, *w, *w_scales;
    const float *bias;
    void *out;
    int64_t scale_k_stride, scale_n_stride, out_stride;
    int64_t rows, n;
    int blocks;      // of 128 along the contraction
    int vec;         // the result's rows take runs of four columns in one store
};

typedef const __attribute__((address_space(1))) void *global_ptr;
typedef __attribute__((address_space(3))) void *lds_ptr;

// 64 lanes copy 16 bytes each from their own address to `dst` + 16 * lane (dst the same in every lane)
__device__ __forceinline__ void copy_to_lds(const uint8_t *src, uint8_t *dst) {
    __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)dst, 16, 0, 0);
}

// 32 bytes at a 16-byte aligned address
__device__ __forceinline__ i32x8 load32(const uint8_t *p) {
    const i32x4 lo = *reinterpret_cast<const i32x4 *>(p), hi = *reinterpret_cast<const i32x4 *>(p + 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// eight codes, scaled, as bf16 (exact); `power`: the scale as a float
__device__ __forceinline__ bf16x8_t decode8(int lo, int hi, float power) {
    union {
        bf16x2_t h[4];
        bf16x8_t v;
    } u;
    u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, power, false);
    u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, power, true);
    u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, power, false);
    u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, power, true);
    return u.v;
}
__device__ __forceinline__ float scale_value(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// block number -> tile number: the blocks of one XCD (every eighth) take a stretch of neighbouring tiles
__device__ __forceinline__ int64_t tile_of(int64_t block, int64_t tiles) {
    const int64_t q = tiles / 8, r = tiles % 8, xcd = block % 8, i = block / 8;
    return xcd < r ? xcd * (q + 1) + i : r * (q + 1) + (xcd - r) * q + i;
}

__device__ __forceinline__ void store_run(float *row, int64_t c, int64_t n, int vec, const f32x4 v) {
    if (vec) store4<true>(row, c, n, v);
    else store4<false>(row, c, n, v);
}
__device__ __forceinline__ void store_run(bf16_t *row, int64_t c, int64_t n, int vec, const f32x4 v) {
    if (vec) store4<true>(row, c, n, v);
    else store4<false>(row, c, n, v);
}

// WM x WN tiles of 32 x 32 a wave, MW x NW waves a block
template <typename O, int WM, int WN, int MW, int NW>
__global__ __launch_bounds__(64 * MW * NW) void fp8_product_kernel(const ProductArgs p) {
    constexpr bool kExact = sizeof(O) == 4;
    constexpr int kWaves = MW * NW;
    constexpr int kM = 32 * WM * MW, kN = 32 * WN * NW;
    constexpr int kCopies = (kM + kN) / 8 / kWaves;   // copies of 8 rows a wave and stage
    static_assert((kM + kN) % (8 * kWaves) == 0 && 32 * WN <= kBlock8, "");
    extern __shared__ __align__(128) uint8_t lds[];   // two stages of (kM + kN) rows of 128 bytes
    constexpr int kStage = (kM + kN) * kBlock8;

    const int lane = (int)threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int wm = wave / NW, wn = wave % NW;
    const int idx = lane % 32, half = lane / 32;
    const int64_t tiles_n = (p.n + kN - 1) / kN;
    const int64_t tile = tile_of(blockIdx.x, gridDim.x);
    const int64_t m0 = tile / tiles_n * kM, n0 = tile % tiles_n * kN;
    const int64_t pitch = (int64_t)p.blocks * kBlock8;

    // what this lane copies: rows past the end read the last row, their results are never stored
    const uint8_t *src[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int row = (wave * kCopies + i) * 8 + lane / 8;
        const int piece = (lane % 8) ^ ((row / 2) % 8);
        const bool is_x = row < kM;
        int64_t r = is_x ? m0 + row : n0 + (row - kM);
        const int64_t last = (is_x ? p.rows : p.n) - 1;
        r = r < last ? r : last;
        src[i] = (is_x ? p.x : p.w) + r * pitch + 16 * piece;
    }
    auto fetch = [&](int stage, int block) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
            copy_to_lds(src[i] + (int64_t)block * kBlock8, lds + stage * kStage + (wave * kCopies + i) * 8 * kBlock8);
    };

    const uint8_t *xs[WM];
    int64_t wm0 = m0 + wm * 32 * WM;
#pragma unroll
    for (int i = 0; i < WM; ++i) {
        int64_t m = wm0 + 32 * i + idx;
        m = m < p.rows ? m : p.rows - 1;
        xs[i] = p.x_scales + m * p.blocks;
    }
    const int64_t wn0 = n0 + wn * 32 * WN;
    const int64_t nb = (wn0 < p.n ? wn0 : p.n - 1) / kBlock8;
    const uint8_t *ws = p.w_scales + nb * p.scale_n_stride;

    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    // byte offsets of a lane's four 16-byte pieces in a staged row of its fragment
    int piece_off[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) piece_off[q] = idx * kBlock8 + 16 * (((q / 2) * 4 + half * 2 + q % 2) ^ ((idx / 2) % 8));

    fetch(0, 0);
    int sx[WM], sw;
#pragma unroll
    for (int i = 0; i < WM; ++i) sx[i] = xs[i][0];
    sw = ws[0];
    for (int b = 0; b < p.blocks; ++b) {
        // this stage has landed (every wave waits for its own copies), and everybody is done with the other one
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const uint8_t *stage = lds + (b & 1) * kStage;
        int nx[WM], nw = 0;
        const int next = b + 1 < p.blocks ? b + 1 : b;
        if (b + 1 < p.blocks) fetch((b + 1) & 1, b + 1);
#pragma unroll
        for (int i = 0; i < WM; ++i) nx[i] = xs[i][next];
        nw = ws[next * p.scale_k_stride];
        const uint8_t *xt = stage + wm * 32 * WM * kBlock8, *wt = stage + (kM + wn * 32 * WN) * kBlock8;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x8 fx[WM], fw[WN];
#pragma unroll
            for (int j = 0; j < WN; ++j) {
                const i32x4 lo = *reinterpret_cast<const i32x4 *>(wt + 32 * j * kBlock8 + piece_off[2 * s]);
                const i32x4 hi = *reinterpret_cast<const i32x4 *>(wt + 32 * j * kBlock8 + piece_off[2 * s + 1]);
                fw[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                const i32x4 lo = *reinterpret_cast<const i32x4 *>(xt + 32 * i * kBlock8 + piece_off[2 * s]);
                const i32x4 hi = *reinterpret_cast<const i32x4 *>(xt + 32 * i * kBlock8 + piece_off[2 * s + 1]);
                fx[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            if constexpr (!kExact) {
#pragma unroll
                for (int i = 0; i < WM; ++i)
#pragma unroll
                    for (int j = 0; j < WN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[j], fx[i], acc[i][j], 0, 0, 0, sw, 0, sx[i]);
            } else {
                // a lane's codes eight at a time: the contraction in another order, the same for both operands
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    bf16x8_t hw[WN];
#pragma unroll
                    for (int j = 0; j < WN; ++j) hw[j] = decode8(fw[j][2 * t], fw[j][2 * t + 1], scale_value(sw));
#pragma unroll
                    for (int i = 0; i < WM; ++i) {
                        const bf16x8_t hx = decode8(fx[i][2 * t], fx[i][2 * t + 1], scale_value(sx[i]));
#pragma unroll
                        for (int j = 0; j < WN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hw[j], hx, acc[i][j], 0, 0, 0);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            sx[i] = nx[i];
            asm volatile("" : "+v"(sx[i]));  // (the next block's scales are loaded behind this one's products, not
        }                                    //  sunk to their first use)
        sw = nw;
        asm volatile("" : "+v"(sw));
    }

    // register r of lane l holds column (r % 4) + 8 (r / 4) + 4 (l / 32) of the tile, row l % 32
#pragma unroll
    for (int j = 0; j < WN; ++j) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int64_t c = wn0 + 32 * j + 8 * g + 4 * half;
            const f32x4 b4 = p.bias ? load4<false>(p.bias, c, p.n) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                const int64_t m = wm0 + 32 * i + idx;
                if (m >= p.rows) continue;
                const f32x4 v = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]} + b4;
                store_run(static_cast<O *>(p.out) + m * p.out_stride, c, p.n, p.vec, v);
            }
        }
    }
}

// Few rows (a token, a small batch): bound by the bytes of w and by latency.  A block owns 16 columns and 16 MT rows; its
// eight waves share the contraction, every one reading its blocks of w (128-byte rows) straight into registers, and the
// eight partial tiles are added in wave order through LDS.
template <typename O, int MT>
__global__ __launch_bounds__(512) void fp8_product_few_kernel(const ProductArgs p) {
    constexpr bool kExact = sizeof(O) == 4;
    constexpr int kWaves = 8;
    __shared__ f32x4 part[kWaves][MT][64];
    const int lane = (int)threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int idx = lane % 16, quarter = lane / 16;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16 * MT;
    const int64_t pitch = (int64_t)p.blocks * kBlock8;
    int64_t n = n0 + idx;
    n = n < p.n ? n : p.n - 1;
    const uint8_t *wr = p.w + n * pitch + 32 * quarter;
    const uint8_t *ws = p.w_scales + n0 / kBlock8 * p.scale_n_stride;
    const uint8_t *xr[MT], *xs[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        int64_t m = m0 + 16 * i + idx;
        m = m < p.rows ? m : p.rows - 1;
        xr[i] = p.x + m * pitch + 32 * quarter;
        xs[i] = p.x_scales + m * p.blocks;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int b = wave; b < p.blocks; b += kWaves) {
        const i32x8 fw = load32(wr + (int64_t)b * kBlock8);
        const int sw = ws[b * p.scale_k_stride];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const i32x8 fx = load32(xr[i] + (int64_t)b * kBlock8);
            const int sx = xs[i][b];
            if constexpr (!kExact) {
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, acc[i], 0, 0, 0, sw, 0, sx);
            } else {
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decode8(fw[2 * t], fw[2 * t + 1], scale_value(sw)),
                                                                     decode8(fx[2 * t], fx[2 * t + 1], scale_value(sx)),
                                                                     acc[i], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    // register r of lane l holds column r + 4 (l / 16) of the tile, row l % 16
    for (int t = wave; t < MT; t += kWaves) {
        f32x4 v = part[0][t][lane];
#pragma unroll
        for (int q = 1; q < kWaves; ++q) v += part[q][t][lane];
        const int64_t m = m0 + 16 * t + idx, c = n0 + 4 * quarter;
        if (m >= p.rows) continue;
        if (p.bias) v += load4<false>(p.bias, c, p.n);
        store_run(static_cast<O *>(p.out) + m * p.out_stride, c, p.n, p.vec, v);
    }
}

template <typename O, int WM, int WN, int MW, int NW>
int launch_tiles(const ProductArgs &p, hipStream_t st) {
    constexpr int kM = 32 * WM * MW, kN = 32 * WN * NW;
    constexpr size_t kLds = 2 * (size_t)(kM + kN) * kBlock8;
    const int64_t tiles = ((p.rows + kM - 1) / kM) * ((p.n + kN - 1) / kN);
    if (tiles > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "too many tiles");
    auto kernel = fp8_product_kernel<O, WM, WN, MW, NW>;
    if (kLds > 64 * 1024)
        GNNAGG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * MW * NW), kLds, st, p);
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}

template <typename O>
int launch_product(const ProductArgs &p, hipStream_t st) {
    const int64_t columns = (p.n + 15) / 16;
    if (p.rows <= 64) {
        auto few = [&](auto mt) {
            constexpr int kMt = decltype(mt)::value;
            hipLaunchKernelGGL((fp8_product_few_kernel<O, kMt>),
                               dim3((unsigned)columns, (unsigned)((p.rows + 16 * kMt - 1) / (16 * kMt))), dim3(512), 0, st, p);
        };
        if (p.rows <= 16) few(std::integral_constant<int, 1>());
        else if (p.rows <= 32) few(std::integral_constant<int, 2>());
        else few(std::integral_constant<int, 4>());
        GNNAGG_HIP(hipGetLastError());
        return GNNAGG_OK;
    }
    return launch_tiles<O, 2, 2, 2, 2>(p, st);
}

}  // namespace
}  // namespace gnnagg

using namespace gnnagg;

extern "C" int gnnagg_fp8_product(const uint8_t *x, const uint8_t *x_scales, const uint8_t *w, const uint8_t *w_scales,
                                  int64_t scale_k_stride, int64_t scale_n_stride, const float *bias, void *out,
                                  int64_t out_stride, int out_dtype, int64_t rows, int64_t k, int64_t n, void *stream) {
    GNNAGG_REQUIRE(rows >= 0 && k >= 0 && n >= 0, "negative size");
    GNNAGG_REQUIRE(known_dtype(out_dtype), "unknown dtype");
    if (rows == 0 || n == 0) return GNNAGG_OK;
    GNNAGG_REQUIRE(k > 0, "an inner width of zero");
    GNNAGG_REQUIRE(x && x_scales && w && w_scales && out, "null x/w/scales/out");
    GNNAGG_REQUIRE(out_stride >= n, "the output row stride is below the width");
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0,
                   "codes must be 16-byte aligned");
    if (k > (int64_t(1) << 31) || n > (int64_t(1) << 34)) return fail(GNNAGG_ERR_UNSUPPORTED, "a weight of %lld x %lld", (long long)k, (long long)n);
    ProductArgs p{x, x_scales, w, w_scales, bias, out, scale_k_stride, scale_n_stride, out_stride, rows, n,
                  (int)(pad128(k) / kBlock8), 0};
    p.vec = vec4_rows(out, out_stride, n, out_dtype);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return out_dtype == GNNAGG_F32 ? launch_product<float>(p, st) : launch_product<bf16_t>(p, st);
}
