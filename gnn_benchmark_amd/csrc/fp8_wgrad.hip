// Weight gradient behind an 8-bit product,
//
//     grad_w[k, n] = sum over rows m of x[m, k] * bf16(g[m, n]),   grad_bias[n] = sum over rows of g[m, n],
//
// x in the 8-bit format.  A scale of that format varies along the contraction here, so it cannot be left to the matrix
// unit; but a code times a power of two is a bf16 value, so x is turned into bf16 exactly on its way into LDS and the
// product runs on the bf16 matrix units: x loses nothing, g is rounded to 8 significant bits, sums are fp32.  What the
// forward has to keep for it is one byte a value.
//
// A block of eight waves owns 256 x 256 of the result and a slice of the rows, 32 rows a stage: with 64 x 128 of the result
// a wave, the LDS reads of a stage (6 KB a wave for 8 MFMAs' worth of a 16-row step) stay below its MFMA time, which a
// 128 x 128 block of four waves does not reach (8192 rows, 4096 x 4096, bf16 g: 0.91 ms there, 0.35 ms = 790 TFLOP/s here).  The
// MFMA wants eight consecutive rows of one column in a lane, memory holds rows: a thread loads eight rows of four
// neighbouring columns, pairs them up by bytes in registers and writes four 16-byte pieces of eight rows each.  Half the
// threads bring x, half bring g; the stage after the next is in flight from memory while the next is written to the other
// LDS buffer, one barrier a stage.  The slices' results are added by a second launch in slice order; a grid that fills the
// chip has one slice and writes the result itself.
#include <type_traits>

#include "fp8_format.h"

namespace gnnagg {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTile = 256;     // of the result, both ways
constexpr int kRows = 32;      // rows of x and g a stage
constexpr int kHalfStage = kTile * kRows * 2;   // bytes of one operand's stage
constexpr int kUnits = 256;    // compute units: a block each

struct WgradArgs {
    const uint8_t *x, *x_scales;
    const void *g;
    float *out, *bias_out;     // slice 0's result; slice s lies s * k * n (s * n) floats behind
    int64_t g_stride, rows, rows_per_slice, k, n;
    int blocks;                // of 128 along x's rows
    int tiles_n;
};

// Byte offset of 16-byte piece q (eight rows) of column c in a staged operand.  64 bytes a column; columns are exchanged
// inside their group of four and pieces inside their column.  A 16-byte LDS access takes its lanes in fours of which groups
// 0, 3, 5, 6 (and 1, 2, 4, 7) of a half-wave go together; with this order both the writes (column 4 lane + const) and the
// reads (column lane + const) of such 16 lanes fall on 16 different groups of banks.
__device__ __forceinline__ int staged(int c, int q) {
    const int u = c >> 2, v = c >> 4;
    return (c ^ (u & 3)) * (2 * kRows) + 16 * (q ^ ((u ^ (3 * (v & 1)) ^ (v >> 1)) & 3));
}

// eight rows of four columns, two bf16 values a word -> four pieces
__device__ __forceinline__ void write_columns(uint8_t *tile, int c, int q, const uint2 (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        u32x4 piece;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t a = j < 2 ? v[2 * w].x : v[2 * w].y, b = j < 2 ? v[2 * w + 1].x : v[2 * w + 1].y;
            piece[w] = __builtin_amdgcn_perm(b, a, j % 2 == 0 ? 0x05040100u : 0x07060302u);
        }
        *reinterpret_cast<u32x4 *>(tile + staged(c + j, q)) = piece;
    }
}

__device__ __forceinline__ uint32_t word(bf16x2_t h) {
    union {
        bf16x2_t h;
        uint32_t u;
    } x;
    x.h = h;
    return x.u;
}

// What a thread brings of one operand: four neighbouring columns of eight rows, in registers as they lie in memory (no
// conversion, so no wait, before they are written to LDS).  The rows are the same for a whole wave: scalar addresses.
struct XRun {
    static constexpr bool kIsX = true;
    uint32_t code[8];
    int exponent[8];
    const uint8_t *codes, *scales;   // of the operand's first row
    uint32_t column, block;          // this lane's
    int64_t pitch, blocks;           // bytes from row to row of either

    __device__ __forceinline__ XRun(const WgradArgs &p, int64_t k0, int64_t, int quad) {
        blocks = p.blocks;
        pitch = blocks * kBlock8;
        const int64_t c = k0 + 4 * quad < pitch ? k0 + 4 * quad : pitch - 4;  // (past the matrix: its results are not stored)
        column = (uint32_t)c;
        block = (uint32_t)(c / kBlock8);
        codes = p.x;
        scales = p.x_scales;
    }
    // rows first .. first + 7, those past `more` of them read the last one again
    template <bool WHOLE>
    __device__ __forceinline__ void load(int64_t first, int more) {
        const uint8_t *c = codes + first * pitch, *e = scales + first * blocks;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            code[r] = *reinterpret_cast<const uint32_t *>(scalar(c) + column);
            exponent[r] = scalar(e)[block];
            if (WHOLE || r < more) c += pitch, e += blocks;
        }
    }
    __device__ __forceinline__ void clear(int r) { code[r] = 0; }
    __device__ __forceinline__ uint2 as_bf16(int r) const {
        const float power = __uint_as_float((uint32_t)exponent[r] << 23);
        return uint2{word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[r], power, false)),
                     word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[r], power, true))};
    }
    __device__ __forceinline__ f32x4 values(int) const { return f32x4{0.f, 0.f, 0.f, 0.f}; }
};
template <typename G, bool VEC>
struct GRun {
    static constexpr bool kIsX = false;
    typedef typename std::conditional<sizeof(G) == 4, f32x4, uint2>::type Raw;
    Raw v[8];
    const G *g;
    int64_t stride;
    uint32_t column[VEC ? 1 : 4];

    __device__ __forceinline__ GRun(const WgradArgs &p, int64_t, int64_t n0, int quad) {
        g = static_cast<const G *>(p.g);
        stride = p.g_stride;
        const int64_t c = n0 + 4 * quad;
        if (VEC) {
            column[0] = (uint32_t)(c < p.n ? c : p.n - 4);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) column[VEC ? 0 : j] = (uint32_t)(c + j < p.n ? c + j : p.n - 1);
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void load(int64_t first, int more) {
        const G *at = g + first * stride;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const G *row = scalar(at);
            if constexpr (VEC) {
                v[r] = *reinterpret_cast<const Raw *>(row + column[0]);
            } else if constexpr (sizeof(G) == 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[r][j] = row[column[j]];
            } else {
                v[r] = uint2{row[column[0]].bits | (uint32_t)row[column[1]].bits << 16,
                             row[column[2]].bits | (uint32_t)row[column[3]].bits << 16};
            }
            if (WHOLE || r < more) at += stride;
        }
    }
    __device__ __forceinline__ void clear(int r) { v[r] = Raw{}; }
    __device__ __forceinline__ uint2 as_bf16(int r) const {
        if constexpr (sizeof(G) == 4) return uint2{bf16_pair(v[r].x, v[r].y), bf16_pair(v[r].z, v[r].w)};
        else return v[r];
    }
    __device__ __forceinline__ f32x4 values(int r) const {
        if constexpr (sizeof(G) == 4) return v[r];
        else return f32x4{__uint_as_float(v[r].x << 16), __uint_as_float(v[r].x & 0xffff0000u),
                          __uint_as_float(v[r].y << 16), __uint_as_float(v[r].y & 0xffff0000u)};
    }
};

struct Place {                 // of a block and a wave in the result and in the rows
    int64_t k0, n0, begin, end;
    int wk, wn, oct, lane;
    bool live, sums;           // the wave's part of the result lies inside the matrix; it adds up g's columns
};

typedef f32x16 Tiles[4][2];

template <typename Run, int SETS>
__device__ __forceinline__ void wgrad_loop(const WgradArgs &p, const Place &w, uint8_t (&lds)[2][2][kHalfStage], Tiles &acc,
                                           f32x4 &column_sum) {
    const Run empty(p, w.k0, w.n0, w.lane);
    Run raw[2] = {empty, empty};  // (the second unused with one set)
    const int idx = w.lane % 32, half = w.lane / 32;
    auto fetch = [&](auto set, int64_t m0) {
        Run &run = raw[decltype(set)::value % SETS];
        const int64_t left = w.end - 1 - (m0 + 8 * w.oct);   // rows behind the first
        if (left >= 7) run.template load<true>(m0 + 8 * w.oct, 7);
        else run.template load<false>(left >= 0 ? m0 + 8 * w.oct : w.end - 1, left < 0 ? 0 : (int)left);
    };
    auto stage = [&](auto set, int64_t m0) {
        Run &run = raw[decltype(set)::value % SETS];
        const int64_t left = w.end - m0 - 8 * w.oct;  // how many of the eight rows are the slice's
        if (left < 8) {
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r >= left) run.clear(r);
        }
        uint2 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = run.as_bf16(r);
        write_columns(lds[decltype(set)::value][Run::kIsX ? 0 : 1], 4 * w.lane, w.oct, v);
        if (!Run::kIsX && w.sums) {
#pragma unroll
            for (int r = 0; r < 8; ++r) column_sum += run.values(r);
        }
    };
    auto multiply = [&](auto set) {
        if (!w.live) return;
        const uint8_t *xt = lds[decltype(set)::value][0], *gt = lds[decltype(set)::value][1];
        // both 16-row steps' fragments are asked for before the first is multiplied
        bf16x8_t fx[kRows / 16][4], fg[kRows / 16][2];
#pragma unroll
        for (int s = 0; s < kRows / 16; ++s) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                fg[s][j] = *reinterpret_cast<const bf16x8_t *>(gt + staged(64 * w.wn + 32 * j + idx, 2 * s + half));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                fx[s][i] = *reinterpret_cast<const bf16x8_t *>(xt + staged(128 * w.wk + 32 * i + idx, 2 * s + half));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < kRows / 16; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fx[s][i], fg[s][j], acc[i][j], 0, 0, 0);
    };
    // Stage s lies in LDS buffer s % 2, s + 1 (and with two sets of registers s + 2) in registers or on its way there; as
    // s + 1 goes into the other buffer, the stage that takes its registers is asked for.  A SIMD has one wave that brings x
    // and one that brings g: the second does that first and multiplies s behind it, so that its conversions and addresses
    // run beside the first one's matrix instructions, and the other way round.
    auto step = [&](auto set, auto other, int64_t m0) {
        lds_barrier();
        if (Run::kIsX) multiply(set);
        stage(other, m0 + kRows);
        fetch(other, m0 + (1 + SETS) * kRows);
        if (!Run::kIsX) multiply(set);
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    if (w.begin >= w.end) return;
    fetch(even, w.begin);
    if (SETS == 2) fetch(odd, w.begin + kRows);
    stage(even, w.begin);
    fetch(even, w.begin + SETS * kRows);
    for (int64_t m0 = w.begin; m0 < w.end; m0 += 2 * kRows) {  // (a stage past the end holds zeros)
        step(even, odd, m0);
        step(odd, even, m0 + kRows);
    }
}

template <typename G, bool VEC>
__global__ __launch_bounds__(512, 2) void fp8_wgrad_kernel(const WgradArgs p) {
    __shared__ __align__(16) uint8_t lds[2][2][kHalfStage];   // stage parity; x, g
    const int lane = (int)threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int kt = (int)blockIdx.x / p.tiles_n, nt = (int)blockIdx.x % p.tiles_n;
    const int64_t slice = blockIdx.y;
    Place w;
    w.wk = wave / 4, w.wn = wave % 4, w.oct = wave % 4, w.lane = lane;
    w.k0 = (int64_t)kt * kTile, w.n0 = (int64_t)nt * kTile;
    w.begin = slice * p.rows_per_slice;
    w.end = w.begin + p.rows_per_slice < p.rows ? w.begin + p.rows_per_slice : p.rows;
    w.live = w.k0 + 128 * w.wk < p.k && w.n0 + 64 * w.wn < p.n;
    w.sums = kt == 0 && p.bias_out;
    const int idx = lane % 32, half = lane / 32;

    Tiles acc;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    f32x4 column_sum = {0.f, 0.f, 0.f, 0.f};

    // Waves 0-3 bring x, 4-7 bring g: the whole loop apart, with the same barriers, so that neither's registers are merged
    // with the other's (which would wait for the loads in flight).
    if (wave < 4) wgrad_loop<XRun, 2>(p, w, lds, acc, column_sum);
    else wgrad_loop<GRun<G, VEC>, sizeof(G) == 2 ? 2 : 1>(p, w, lds, acc, column_sum);  // (two sets of fp32 g would spill)

    // register r of lane l holds row (r % 4) + 8 (r / 4) + 4 (l / 32), column l % 32 of its 32 x 32 tile
    float *out = p.out + slice * p.k * p.n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t k = w.k0 + 128 * w.wk + 32 * i + r % 4 + 8 * (r / 4) + 4 * half;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t n = w.n0 + 64 * w.wn + 32 * j + idx;
                if (k < p.k && n < p.n) out[k * p.n + n] = acc[i][j][r];
            }
        }
    if (w.sums) {
        f32x4 *parts = reinterpret_cast<f32x4 *>(lds);
        const int tid = (int)threadIdx.x;
        __syncthreads();
        if (wave >= 4) parts[tid - 256] = column_sum;
        __syncthreads();
        if (tid < 64) {
            f32x4 total = parts[tid];
            for (int q = 1; q < 4; ++q) total += parts[tid + 64 * q];
            store4<false>(p.bias_out + slice * p.n, (int64_t)(w.n0 + 4 * tid), p.n, total);
        }
    }
}

// The number of slices with the least rows that a compute unit works through, a block's start and end (its result written,
// read and added once more) counted as 256 rows; slices' results at most 256 MB.
int64_t wgrad_slices(int64_t rows, int64_t k, int64_t n) {
    const int64_t tiles = ((k + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
    int64_t most = (int64_t(1) << 26) / (k * n);
    most = most < kUnits ? most : kUnits;
    int64_t best = 1, best_cost = (tiles + kUnits - 1) / kUnits * rows;
    for (int64_t s = 2; s <= most; ++s) {
        const int64_t cost = (tiles * s + kUnits - 1) / kUnits * ((rows + s - 1) / s + 256);
        if (cost < best_cost) best = s, best_cost = cost;
    }
    return best;
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
    const int64_t tiles_k = (k + kTile - 1) / kTile, tiles_n = (n + kTile - 1) / kTile;
    WgradArgs p{x, x_scales, g, parts, bias_parts, g_stride, rows, (per + kRows - 1) / kRows * kRows, k, n,
                (int)(pad128(k) / kBlock8), (int)tiles_n};
    if (tiles_k * tiles_n > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "too many tiles");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(tiles_k * tiles_n), (unsigned)slices);
    auto go = [&](auto type, auto v) {
        hipLaunchKernelGGL((fp8_wgrad_kernel<decltype(type), decltype(v)::value>), grid, dim3(512), 0, st, p);
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
