// Weight gradient behind an 8-bit product,
//
//     grad_w[k, n] = sum over rows m of x[m, k] * bf16(g[m, n]),   grad_bias[n] = sum over rows of g[m, n],
//
// x in the 8-bit format.  A scale of that format varies along the contraction here, so it cannot be left to the matrix
// unit; but a code times a power of two in [2^-124, 2^119] is a bf16 value, so x is turned into bf16 exactly on its way into
// LDS (beyond these, to bf16's subnormals and infinity) and the product runs on the bf16 matrix units: x loses nothing, g is
// rounded to 8 significant bits, sums are fp32.  What the forward has to keep for it is one byte a value.
//
// A block of eight waves owns 256 x 256 of the result and a slice of the rows, 32 rows a stage: with 64 x 128 of the result
// a wave, the LDS reads of a stage (6 KB a wave for 8 MFMAs' worth of a 16-row step) stay below its MFMA time, which a
// 128 x 128 block of four waves does not reach (8192 rows, 4096 x 4096, bf16 g: 0.91 ms there, 0.28 ms = 980 TFLOP/s here).
// The MFMA wants eight consecutive rows of one column in a lane, memory holds rows: a thread loads eight rows of four or
// eight neighbouring columns, pairs them up by bytes in registers and writes 16-byte pieces of eight rows each.  Half the
// waves bring x, half bring g; the next stage is written to the other LDS buffer, and the one after that is in flight from
// memory, while a stage is multiplied; one barrier a stage.  The slices' results are added by a second launch in slice order;
// a grid that fills the chip has one slice and writes the result itself.
//
// What bounds it: many rows and a small result, memory (1.2 M rows, 256 x 172, fp32 g: 4.6 TB/s; at 300 000 rows the slices'
// partial results and a block's start cost 30 us beside 60 of bytes).  Large results, the chain in a stage: without its
// loads from memory the 0.28 ms are 0.21, without fragments from LDS 0.24, and the matrix instructions alone take 0.16 (with
// random operands the chip's power holds them there).  Tried against that chain and slower: three LDS buffers with
// fragments read across the barrier (0.30), g copied straight to LDS three stages ahead (0.39); all parts dealt out among
// the matrix instructions gain 6 % on wide bf16 and lose 4 on fp32.  Handing g's rows on in 8 bits from these registers,
// for the input gradient's product, is no faster than the pass over g that it saves (388 / 391 us for a layer of 300 007 x
// 256 -> 172 both ways).
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

// Byte offset of 16-byte piece q (eight rows) of column c in a staged operand: four columns a 256-byte line, the line's 16
// pieces in an order of its own.  A 16-byte LDS access takes its lanes in fours of which groups 0, 3, 5, 6 (and 1, 2, 4, 7)
// of a half-wave go together; with u0..u5 the bits of the line's number these orders let such 16 lanes fall on 16 different
// pieces' banks whether they hold consecutive columns (reads), every fourth or every eighth (writes).
__device__ __forceinline__ int staged(int c, int q) {
    const int u = c >> 2;
    const int order = (u >> 1 & 1) | (u >> 1 & 2) | (u >> 2 & 4) | ((u ^ u >> 5) & 1) << 3;
    return 256 * u + 16 * ((4 * (c & 3) + q) ^ order);
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

struct Place {                 // of a block and a wave in the result and in the rows
    int64_t k0, n0, begin, end;
    int wk, wn, quarter, lane; // quarter: of the four waves that bring the same operand
    bool live, sums;           // the wave's part of the result lies inside the matrix; it adds up g's columns
};

// What a thread brings of one operand: eight rows of kCols neighbouring columns, in registers as they lie in memory (no
// conversion, so no wait, before they are written to LDS).  The loads are as wide as memory allows: a load costs the
// address and return paths much the same whatever its width, and with 4 bytes of x and 8 of g a lane these paths, not the
// matrix units, set the pace (8192 rows, 4096 x 4096, bf16 g: 0.33 ms).  With eight columns a thread two of the four waves
// hold a whole stage, and the pairs take turns.
struct XRun {
    static constexpr bool kIsX = true;
    static constexpr int kCols = 8;
    uint2 code[8];
    int exponent;                    // of row lane % 8 and this lane's block: a load for all rows, handed round below
    const uint8_t *codes, *scales;   // of the operand's first row
    uint32_t column, block;          // this lane's
    int row, oct;                    // lane % 8; which eight rows of a stage
    int64_t pitch, blocks;           // bytes from row to row of either

    __device__ __forceinline__ XRun(const WgradArgs &p, const Place &w) {
        blocks = p.blocks;
        pitch = blocks * kBlock8;
        const int64_t c = w.k0 + 8 * (w.lane % 32);
        column = (uint32_t)(c < pitch ? c : pitch - 8);   // (past the matrix: its results are not stored)
        block = column / kBlock8;
        row = w.lane % 8;
        oct = 2 * (w.quarter % 2) + w.lane / 32;
        codes = p.x;
        scales = p.x_scales;
    }
    // the stage from row m0 on; `end`: the slice's, its last row is read again for those behind it
    template <bool WHOLE>
    __device__ __forceinline__ void load(const Place &w, int64_t m0, int64_t end) {
        if (WHOLE) {
            const int64_t first = m0 + 16 * (w.quarter % 2);
            const uint8_t *c = codes + first * pitch;
            const uint32_t half = (uint32_t)(w.lane / 32) * 8;
            exponent = scalar(scales + first * blocks)[(half + row) * (uint32_t)blocks + block];
#pragma unroll
            for (int r = 0; r < 8; ++r, c += pitch)
                code[r] = *reinterpret_cast<const uint2 *>(scalar(c) + (half * (uint32_t)pitch + column));
        } else {
            const int64_t first = m0 + 8 * oct;
            exponent = scales[(first + row < end ? first + row : end - 1) * blocks + block];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                code[r] = *reinterpret_cast<const uint2 *>(codes + (first + r < end ? first + r : end - 1) * pitch + column);
        }
    }
    __device__ __forceinline__ void keep(int r, bool inside) { if (!inside) code[r] = uint2{0, 0}; }
    template <int R>
    __device__ __forceinline__ void convert(uint2 (&v)[8], int power, int half) const {
        // lane R of each sixteen lanes to all of them (they lie in one block of 128 columns)
        const float mine = __int_as_float(__builtin_amdgcn_update_dpp(0, power, 0x150 + R, 0xf, 0xf, false));
        const uint32_t c = half ? code[R].y : code[R].x;
        v[R] = uint2{word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, mine, false)),
                     word(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, mine, true))};
        if constexpr (R < 7) convert<R + 1>(v, power, half);
    }
    // columns 4 half .. 4 half + 3
    __device__ __forceinline__ void as_bf16(uint2 (&v)[8], int half) const { convert<0>(v, exponent << 23, half); }
    __device__ __forceinline__ f32x4 values(int, int) const { return f32x4{0.f, 0.f, 0.f, 0.f}; }
};

// COLS 8 (bf16 only) or 4 neighbouring columns a load; 1: four, each by itself
template <typename G, int COLS>
struct GRun {
    static constexpr bool kIsX = false;
    static constexpr int kCols = COLS == 8 ? 8 : 4;
    typedef typename std::conditional<sizeof(G) == 4 || COLS == 8, u32x4, uint2>::type Raw;
    Raw v[8];
    const G *g;
    int64_t stride;
    uint32_t column[COLS == 1 ? 4 : 1];
    int oct;

    __device__ __forceinline__ GRun(const WgradArgs &p, const Place &w) {
        g = static_cast<const G *>(p.g);
        stride = p.g_stride;
        const int64_t c = w.n0 + (COLS == 8 ? 8 * (w.lane % 32) : 4 * w.lane);
        oct = COLS == 8 ? 2 * (w.quarter % 2) + w.lane / 32 : w.quarter;
        if (COLS > 1) {
            column[0] = (uint32_t)(c < p.n ? c : p.n - COLS);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) column[COLS == 1 ? j : 0] = (uint32_t)(c + j < p.n ? c + j : p.n - 1);
        }
    }
    __device__ __forceinline__ Raw values_at(const G *row, uint32_t half) const {
        if constexpr (COLS > 1) {
            return *reinterpret_cast<const Raw *>(row + (half + column[0]));
        } else if constexpr (sizeof(G) == 4) {
            return u32x4{__float_as_uint(row[column[0]]), __float_as_uint(row[column[1]]), __float_as_uint(row[column[2]]),
                         __float_as_uint(row[column[3]])};
        } else {
            return uint2{row[column[0]].bits | (uint32_t)row[column[1]].bits << 16,
                         row[column[2]].bits | (uint32_t)row[column[3]].bits << 16};
        }
    }
    template <bool WHOLE>
    __device__ __forceinline__ void load(const Place &w, int64_t m0, int64_t end) {
        if (WHOLE) {
            const G *at = g + (m0 + (COLS == 8 ? 16 * (w.quarter % 2) : 8 * w.quarter)) * stride;
            const uint32_t half = COLS == 8 ? (uint32_t)(w.lane / 32) * 8 * (uint32_t)stride : 0;
#pragma unroll
            for (int r = 0; r < 8; ++r, at += stride) v[r] = values_at(scalar(at), half);
        } else {
            const int64_t first = m0 + 8 * oct;
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = values_at(g + (first + r < end ? first + r : end - 1) * stride, 0);
        }
    }
    __device__ __forceinline__ void keep(int r, bool inside) { if (!inside) v[r] = Raw{}; }
    __device__ __forceinline__ uint2 pair(int r, int half) const {   // bf16 g
        if constexpr (COLS == 8) return half ? uint2{v[r].z, v[r].w} : uint2{v[r].x, v[r].y};
        else return uint2{v[r].x, v[r].y};
    }
    __device__ __forceinline__ void as_bf16(uint2 (&to)[8], int half) const {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if constexpr (sizeof(G) == 4) {
                const f32x4 f = values(r, 0);
                to[r] = uint2{bf16_pair(f.x, f.y), bf16_pair(f.z, f.w)};
            } else {
                to[r] = pair(r, half);
            }
        }
    }
    __device__ __forceinline__ f32x4 values(int r, int half) const {
        if constexpr (sizeof(G) == 4) {
            return f32x4{__uint_as_float(v[r].x), __uint_as_float(v[r].y), __uint_as_float(v[r].z), __uint_as_float(v[r].w)};
        } else {
            const uint2 p = pair(r, half);
            return f32x4{__uint_as_float(p.x << 16), __uint_as_float(p.x & 0xffff0000u), __uint_as_float(p.y << 16),
                         __uint_as_float(p.y & 0xffff0000u)};
        }
    }
};

typedef f32x16 Tiles[4][2];

struct Fragments {             // of one 16-row step: a wave's 128 x 64 of the result
    bf16x8_t x[4], g[2];
};

template <typename Run>
__device__ __forceinline__ void wgrad_loop(const WgradArgs &p, const Place &w, uint8_t *lds, Tiles &acc,
                                           f32x4 (&column_sum)[2]) {
    constexpr int kTurns = Run::kCols / 4;   // a wave brings every stage, or every second one
    Run run(p, w);
    Fragments frag[2];
    const int idx = w.lane % 32, half = w.lane / 32;
    // of a SIMD's two waves, one that brings x and one that brings g, one brings the even stages and one the odd
    const int turn = Run::kIsX ? w.quarter / 2 : 1 - w.quarter / 2;
    auto fetch = [&](int64_t m0) {
        if (m0 + kRows <= w.end) run.template load<true>(w, m0, w.end);
        else run.template load<false>(w, m0, w.end);
    };
    auto stage = [&](int64_t m0, uint8_t *to) {
        if (m0 + kRows > w.end) {
            const int64_t left = w.end - m0 - 8 * run.oct;  // how many of the eight rows are the slice's
#pragma unroll
            for (int r = 0; r < 8; ++r) run.keep(r, r < left);
        }
#pragma unroll
        for (int h = 0; h < kTurns; ++h) {
            uint2 v[8];
            run.as_bf16(v, h);
            const int c = kTurns == 2 ? 8 * idx : 4 * w.lane;
            write_columns(to + (Run::kIsX ? 0 : kHalfStage), c + 4 * h, run.oct, v);
            if (!Run::kIsX && w.sums) {   // (eight rows by themselves first: a chain an eighth as long)
                f32x4 eight = run.values(0, h) + run.values(1, h);
#pragma unroll
                for (int r = 2; r < 8; r += 2) eight += run.values(r, h) + run.values(r + 1, h);
                column_sum[h] += eight;
            }
        }
    };
    auto bring = [&](int parity, int64_t m0, uint8_t *to) {   // stage m0 to LDS, the wave's next one from memory
        if (kTurns == 2 && turn != parity) return;
        stage(m0, to);
        fetch(m0 + kTurns * kRows);
    };
    auto read = [&](auto step, const uint8_t *from) {
        constexpr int s = decltype(step)::value;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            frag[s].g[j] =
                *reinterpret_cast<const bf16x8_t *>(from + kHalfStage + staged(64 * w.wn + 32 * j + idx, 2 * s + half));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            frag[s].x[i] = *reinterpret_cast<const bf16x8_t *>(from + staged(128 * w.wk + 32 * i + idx, 2 * s + half));
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](auto step) {
        constexpr int s = decltype(step)::value;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[s].x[i], frag[s].g[j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    const std::integral_constant<int, 0> even;
    const std::integral_constant<int, 1> odd;
    // A stage is multiplied out of one LDS buffer while the next is written to the other, from registers, and the stage that
    // takes these asked for.  The waves that bring g do that first and multiply behind it, so that their conversions and
    // addresses run beside the others' matrix instructions, and the other way round.
    uint8_t *now = lds, *next = lds + 2 * kHalfStage;
    auto step = [&](int parity, int64_t m0) {
        if (!Run::kIsX) bring(1 - parity, m0 + kRows, next);
        if (w.live) {
            read(even, now);
            read(odd, now);
            multiply(even);
            multiply(odd);
        }
        if (Run::kIsX) bring(1 - parity, m0 + kRows, next);
        lds_barrier();
        uint8_t *const was = now;
        now = next, next = was;
    };
    if (w.begin >= w.end) return;
    if (kTurns == 2) {
        fetch(w.begin + turn * kRows);
        if (turn == 0) bring(0, w.begin, now);
    } else {
        fetch(w.begin);
        bring(0, w.begin, now);
    }
    lds_barrier();
    for (int64_t m0 = w.begin; m0 < w.end; m0 += 2 * kRows) {  // (a stage past the end holds zeros)
        step(0, m0);
        step(1, m0 + kRows);
    }
}

template <typename G, int COLS>
__global__ __launch_bounds__(512, 2) void fp8_wgrad_kernel(const WgradArgs p) {
    __shared__ __align__(16) uint8_t lds[2 * 2 * kHalfStage];   // stages; x, g
    const int lane = (int)threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int kt = (int)blockIdx.x / p.tiles_n, nt = (int)blockIdx.x % p.tiles_n;
    const int64_t slice = blockIdx.y;
    Place w;
    w.wk = wave / 4, w.wn = wave % 4, w.quarter = wave % 4, w.lane = lane;
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
    f32x4 column_sum[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};

    // Waves 0-3 bring x, 4-7 bring g: the whole loop apart, with the same barriers, so that neither's registers are merged
    // with the other's (which would wait for the loads in flight).
    typedef GRun<G, COLS> Gradient;
    if (wave < 4) wgrad_loop<XRun>(p, w, lds, acc, column_sum);
    else wgrad_loop<Gradient>(p, w, lds, acc, column_sum);

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
    if (w.sums) {   // each wave's (with eight columns a thread, each half-wave's) sums of its rows, then all rows'
        constexpr int kParts = Gradient::kCols == 8 ? 8 : 4;
        float *parts = reinterpret_cast<float *>(lds);   // [kParts][kTile]
        const int tid = (int)threadIdx.x;
        __syncthreads();
        if (wave >= 4) {
            const int part = Gradient::kCols == 8 ? 2 * w.quarter + half : w.quarter;
            f32x4 *at = reinterpret_cast<f32x4 *>(parts + part * kTile + (Gradient::kCols == 8 ? 8 * idx : 4 * lane));
            at[0] = column_sum[0];
            if (Gradient::kCols == 8) at[1] = column_sum[1];
        }
        __syncthreads();
        if (tid < kTile && w.n0 + tid < p.n) {
            float total = parts[tid];
            for (int q = 1; q < kParts; ++q) total += parts[tid + q * kTile];
            p.bias_out[slice * p.n + w.n0 + tid] = total;
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
    GNNAGG_REQUIRE(reinterpret_cast<uintptr_t>(x) % 8 == 0, "codes must be 8-byte aligned");
    const int64_t slices = wgrad_slices(rows, k, n), need = gnnagg_fp8_weight_gradient_workspace_bytes(rows, k, n);
    GNNAGG_REQUIRE(workspace_bytes >= need && (need == 0 || workspace) && reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
                   "workspace of %lld bytes is too small, null or misaligned", (long long)workspace_bytes);
    float *parts = slices == 1 ? grad_w : static_cast<float *>(workspace);
    float *bias_parts = !grad_bias ? nullptr : slices == 1 ? grad_bias : parts + slices * k * n;
    const int64_t per = (rows + slices - 1) / slices;
    const int64_t tiles_k = (k + kTile - 1) / kTile, tiles_n = (n + kTile - 1) / kTile;
    WgradArgs p{x, x_scales, g, parts, bias_parts, g_stride, rows,
                (per + kRows - 1) / kRows * kRows, k, n, (int)(pad128(k) / kBlock8), (int)tiles_n};
    if (tiles_k * tiles_n > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "too many tiles");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(tiles_k * tiles_n), (unsigned)slices);
    auto go = [&](auto type, auto cols) {
        hipLaunchKernelGGL((fp8_wgrad_kernel<decltype(type), decltype(cols)::value>), grid, dim3(512), 0, st, p);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    const bool vec = vec4_rows(g, g_stride, n, g_dtype);
    // Sixteen bytes of bf16 a load where rows allow it and offsets of eight rows fit 32 bits (8192 rows, 4096 x 4096: 299 us
    // against 319 with eight).
    const bool wide = g_dtype == GNNAGG_BF16 && n % 8 == 0 && g_stride % 8 == 0 && g_stride < (int64_t(1) << 27) &&
                      reinterpret_cast<uintptr_t>(g) % 16 == 0;
    if (g_dtype == GNNAGG_F32) {
        if (vec) go(float(), four);
        else go(float(), one);
    } else {
        if (wide) go(bf16_t(), eight);
        else if (vec) go(bf16_t(), four);
        else go(bf16_t(), one);
    }
    GNNAGG_HIP(hipGetLastError());
    if (slices == 1) return GNNAGG_OK;
    if (const int rc = launch_column_reduce(parts, slices, k * n, grad_w, st)) return rc;
    return grad_bias ? launch_column_reduce(bias_parts, slices, n, grad_bias, st) : GNNAGG_OK;
}
