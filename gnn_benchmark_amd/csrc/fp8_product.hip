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
//   fp32   the codes become bf16 values, scale included, in one v_cvt_scalef32_pk_bf16_fp8 for two of them -- exactly
//          for scales in [2^-124, 2^119], on their way from LDS into the matrix unit -- and multiply on v_mfma_f32_*_bf16: every product exact, sums fp32
//          (2e-8 off on the same operands), at half the matrix rate.
//
// Large bf16 products are bound by the matrix unit as far as its power allows (8192^3: 0.61 ms = 1.81 PFLOP/s, with neither
// scales nor copies 0.40; to fp32 0.91 ms = 1.21 PFLOP/s), products of many rows with a small weight by memory (1 M x 512 x 256 to fp32: 0.34 ms), single
// tokens by the launch and the weight's bytes (1 x 4096 x 4096: 6.6 us on the GPU with the weight from memory, 4.2 from a cache;
// 6 to 7 from call to call).
//
// Both operands have the contraction index contiguous.  A pipeline stage is half a block of it, 64 bytes of every row of the
// tile, copied straight from global memory into one of four LDS buffers (no registers between), three stages ahead of the
// matrix unit; one barrier a stage.
//
// w is the MFMA's first operand: a lane then owns runs of four consecutive columns of one row of the result.
//
// The 16-byte pieces of a staged row are stored at piece ^ ((row / 4) % 4).  A 16-byte LDS access takes its lanes in fours
// of which groups 0, 3, 5, 6 (and 1, 2, 4, 7) of a half-wave go together; four rows fill the banks once, and with this order
// such 16 lanes, reading the same piece of their rows, touch every bank once.
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

typedef uint32_t unaligned_word __attribute__((aligned(1)));

// This wave's LDS reads are done and so are its loads and copies but the YOUNGEST ones; and so are everybody's.  (The wait
// is a builtin that the compiler counts: it waits for none of these again.)
template <int YOUNGEST>
__device__ __forceinline__ void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((YOUNGEST & 15) | (YOUNGEST >> 4) << 14 | 0x70);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

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
    constexpr int kHalf = kBlock8 / 2;                  // bytes of a row in a stage
    constexpr int kCopies = (kM + kN) / 16 / kWaves;    // copies of 16 rows a wave and stage
    static_assert((kM + kN) % (16 * kWaves) == 0 && 32 * WN <= kBlock8, "");
    extern __shared__ __align__(128) uint8_t lds[];     // four stages of (kM + kN) rows
    constexpr int kStage = (kM + kN) * kHalf;

    const int lane = (int)threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int wm = wave / NW, wn = wave % NW;
    const int idx = lane % 32, half = lane / 32;
    // neighbouring tiles: eight down, then the next column, so that the tiles at work on one XCD share both operands
    const int64_t tiles_n = (p.n + kN - 1) / kN, tiles_m = (p.rows + kM - 1) / kM;
    const int64_t tile = tile_of(blockIdx.x, gridDim.x);
    const int64_t band = tile / (8 * tiles_n), in_band = tile - band * 8 * tiles_n;
    const int64_t high = tiles_m - 8 * band < 8 ? tiles_m - 8 * band : 8;
    const int64_t m0 = (8 * band + in_band % high) * kM, n0 = in_band / high * kN;
    const int64_t pitch = (int64_t)p.blocks * kBlock8;

    // what this lane copies, from the tile's first row on: rows past the end read the last row, their results are never
    // stored
    const uint8_t *x_tile = p.x + m0 * pitch, *w_tile = p.w + n0 * pitch;
    uint32_t src[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int row = (wave * kCopies + i) * 16 + lane / 4;
        const int piece = (lane % 4) ^ ((row / 4) % 4);
        const bool is_x = row < kM;
        const int64_t last = (is_x ? p.rows - m0 : p.n - n0) - 1;
        const int r = is_x ? row : row - kM;
        src[i] = (uint32_t)((r < last ? r : last) * pitch) + 16 * piece;
    }
    auto fetch = [&](int stage, int from, int to) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
            if (i >= from && i < to) {
                const int row = (wave * kCopies + i) * 16;  // (a copy's rows are all x's or all w's)
                copy_to_lds(scalar((row < kM ? x_tile : w_tile) + (int64_t)stage * kHalf) + src[i],
                            lds + stage % 4 * kStage + row * kHalf);
            }
    };

    // A lane's scales of x: the bytes of four neighbouring blocks of its row in one (unaligned) word, for each fragment --
    // a byte for each block costs a cache line a lane and block, which took a quarter of the time (8192^3: 659 us against
    // 484 without them).  A word that would end past the array is read where the array ends, and shifted.
    const int64_t wm0 = m0 + wm * 32 * WM;
    const uint8_t *xs[WM];
    int beyond[WM];                   // blocks from which on the word would end past the array
#pragma unroll
    for (int i = 0; i < WM; ++i) {
        int64_t m = wm0 + 32 * i + idx;
        m = m < p.rows ? m : p.rows - 1;
        xs[i] = p.x_scales + m * p.blocks;
        const int64_t room = (p.rows - m) * p.blocks - 4;
        beyond[i] = room < p.blocks ? (int)room : p.blocks;
    }
    const int64_t wn0 = n0 + wn * 32 * WN;
    const int64_t nb = (wn0 < p.n ? wn0 : p.n - 1) / kBlock8;
    const uint8_t *ws = p.w_scales + nb * p.scale_n_stride;
    uint32_t four[WM];                // x's scales of the group of four blocks at work, the first block's in the low byte
    int w_next;                       // w's scale of the next block
    auto load_four = [&](int block) {
#pragma unroll
        for (int i = 0; i < WM; ++i)
            four[i] = *reinterpret_cast<const unaligned_word *>(xs[i] + (block < beyond[i] ? block : beyond[i]));
    };
    struct Scales {
        int x[WM], w;
    };

    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    // byte offsets of a lane's two 16-byte pieces in a staged row of its fragment
    int piece_off[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) piece_off[q] = idx * kHalf + 16 * ((2 * half + q) ^ ((idx / 4) % 4));
    constexpr int kPieces = 2 * (WM + WN);
    struct Fragments {
        i32x4 piece[kPieces];  // w's, then x's, two 16-byte pieces each
        __device__ __forceinline__ i32x8 get(int f) const {
            return __builtin_shufflevector(piece[2 * f], piece[2 * f + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
    };
    auto read = [&](Fragments &f, int stage, int from, int to) {
        const uint8_t *at = lds + stage % 4 * kStage;
        const uint8_t *xt = at + wm * 32 * WM * kHalf, *wt = at + (kM + wn * 32 * WN) * kHalf;
#pragma unroll
        for (int r = 0; r < kPieces; ++r)
            if (r >= from && r < to)
                f.piece[r] = *reinterpret_cast<const i32x4 *>((r < 2 * WN ? wt + 32 * (r / 2) * kHalf : xt + 32 * (r / 2 - WN) * kHalf) +
                                                              piece_off[r % 2]);
    };
    // Multiplies a stage.  `beside(q)` is called behind the q-th matrix instruction; the empty statement that names the
    // sum keeps the instruction in front of it.
    constexpr int kSteps = (kExact ? 4 : 1) * WM * WN;
    auto multiply = [&](const Fragments &f, const Scales &s, auto beside) {
        if constexpr (!kExact) {
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j) {
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(f.get(j), f.get(WN + i), acc[i][j], 0, 0, 0, s.w, 0, s.x[i]);
                    asm volatile("" : "+a"(acc[i][j]));
                    beside(i * WN + j);
                    __builtin_amdgcn_sched_barrier(0);
                }
        } else {
            // a lane's codes eight at a time: the contraction in another order, the same for both operands
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                bf16x8_t hw[WN];
#pragma unroll
                for (int j = 0; j < WN; ++j)
                    hw[j] = decode8(f.piece[2 * j + t / 2][2 * (t % 2)], f.piece[2 * j + t / 2][2 * (t % 2) + 1], scale_value(s.w));
#pragma unroll
                for (int i = 0; i < WM; ++i) {
                    const i32x4 c = f.piece[2 * (WN + i) + t / 2];
                    const bf16x8_t hx = decode8(c[2 * (t % 2)], c[2 * (t % 2) + 1], scale_value(s.x[i]));
#pragma unroll
                    for (int j = 0; j < WN; ++j) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(hw[j], hx, acc[i][j], 0, 0, 0);
                        asm volatile("" : "+a"(acc[i][j]));
                        beside((t * WM + i) * WN + j);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    // Stage s is multiplied out of registers while s + 1 is read from LDS and s + 4 is sent for into the buffer that s was
    // read from.  Reads and copies are dealt out among the matrix instructions: sent at once they fill their queues and the
    // wave waits in front of its products.
    Fragments f[2];
    auto step = [&](int s, auto part, const Scales &now, bool more) {
        constexpr int q0 = decltype(part)::value;
        multiply(f[q0], now, [&](int q) {
            read(f[1 - q0], s + 1, 2 * q * kPieces / kSteps, 2 * (q + 1) * kPieces / kSteps);  // (behind the last stage:
            if (more) fetch(s + 4, q * kCopies / kSteps, (q + 1) * kCopies / kSteps);          //  what its buffer held)
        });
    };
    const std::integral_constant<int, 0> first;
    const std::integral_constant<int, 1> second;
    auto block = [&](int b, auto more) {
        constexpr bool kMore = decltype(more)::value;
        landed<kMore ? 2 * kCopies : 0>();  // the copies of stages 2 b + 2 and 2 b + 3 may be on their way
        Scales now;
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const int at = (b & ~3) < beyond[i] ? b & ~3 : beyond[i];  // the first block in the word
            now.x[i] = (int)(four[i] >> (8 * (b - at)));               // (the low byte counts)
            if constexpr (kExact) now.x[i] &= 0xff;
        }
        now.w = w_next;
        if (b % 4 == 3 && b + 1 < p.blocks) load_four(b + 1);
        w_next = ws[(b + 1 < p.blocks ? b + 1 : b) * p.scale_k_stride];
        step(2 * b, first, now, kMore);
        landed<kMore ? 2 * kCopies : 0>();
        step(2 * b + 1, second, now, kMore);
    };
    fetch(0, 0, kCopies);
    load_four(0);
    w_next = ws[0];
    landed<0>();
    fetch(1, 0, kCopies);
    if (p.blocks > 1) {
        fetch(2, 0, kCopies);
        fetch(3, 0, kCopies);
    }
    read(f[0], 0, 0, kPieces);
    int b = 0;
    for (; b + 2 < p.blocks; ++b) block(b, std::true_type());
    for (; b < p.blocks; ++b) block(b, std::false_type());

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

// Many rows against a small weight (a layer of a graph's nodes): bound by x's and the result's bytes.  The whole weight stays
// in LDS, a persistent block a compute unit; its eight waves then work apart, with no barrier, each on 32 rows at a time
// whose codes it reads straight into registers, so that one wave's loads and stores run beside another's products
// (1 M x 512 x 256 to fp32: 0.34 ms = 4.6 TB/s; the tiled kernel, whose blocks live for eight short stages there: 0.64 ms).
// x is the first operand here: a lane holds one column of each of four tiles of 32 x 32, and as tile j takes the weight's rows
// 4 i + j, the four are neighbours in the result: 16 bytes a lane, 512 bytes a row in one store.  Rows of the weight lie
// in that order, 16 bytes further apart than they are long: 16 neighbouring ones start on 16 different groups of banks.
template <typename O, int KB>
__global__ __launch_bounds__(512, 2) void fp8_product_rows_kernel(const ProductArgs p) {
    constexpr bool kExact = sizeof(O) == 4;
    constexpr int kStages = 2 * KB;                       // of 64 along the contraction
    constexpr int kPitch = KB * kBlock8 + 16;
    extern __shared__ __align__(128) uint8_t lds[];       // the weight, then its scales [groups][KB]
    const int lane = (int)threadIdx.x % 64, idx = lane % 32, half = lane / 32;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int groups = (int)((p.n + kBlock8 - 1) / kBlock8);
    uint8_t *w_scales = lds + groups * kBlock8 * kPitch;

    // row n of the weight -> place 128 (n / 128) + 32 (n % 4) + n % 128 / 4; places without a row stay as they are, their
    // results are not stored.  A thread keeps to one piece of the row (512 threads are 64 / KB rows), eight in flight.
    constexpr int kRowPieces = 8 * KB, kRowsAtOnce = 512 / kRowPieces;
    const int q = (int)threadIdx.x % kRowPieces;
    if ((int)threadIdx.x < kRowsAtOnce * kRowPieces) {
        const uint8_t *src = p.w + 16 * q;
        for (int n0 = (int)threadIdx.x / kRowPieces; n0 < p.n; n0 += 8 * kRowsAtOnce) {
            i32x4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int n = n0 + u * kRowsAtOnce;
                v[u] = *reinterpret_cast<const i32x4 *>(src + (int64_t)(n < p.n ? n : (int)p.n - 1) * (KB * kBlock8));
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int n = n0 + u * kRowsAtOnce;
                if (n < p.n)
                    *reinterpret_cast<i32x4 *>(lds + ((n & ~127) + 32 * (n & 3) + ((n & 127) >> 2)) * kPitch + 16 * q) = v[u];
            }
        }
    }
    for (int i = threadIdx.x; i < groups * KB; i += 512)
        w_scales[i] = p.w_scales[(i % KB) * p.scale_k_stride + (i / KB) * p.scale_n_stride];
    __syncthreads();

    const int64_t tiles = (p.rows + 31) / 32, stride = (int64_t)gridDim.x * 8;
    i32x4 x[kStages][2];
    int sx[KB];
    auto load = [&](int64_t tile) {
        int64_t m = tile * 32 + idx;
        m = m < p.rows ? m : p.rows - 1;
        // a stage's four pieces of a row go to the two lanes that have it in turn (w's too: any order of the contraction
        // will do)
        const uint8_t *row = p.x + m * (KB * kBlock8) + 16 * half;
#pragma unroll
        for (int s = 0; s < kStages; ++s) {
            x[s][0] = *reinterpret_cast<const i32x4 *>(row + 64 * s);
            x[s][1] = *reinterpret_cast<const i32x4 *>(row + 64 * s + 32);
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) sx[b] = p.x_scales[m * KB + b];
    };
    f32x16 acc[4];
    auto multiply = [&](int g) {
        if constexpr (!kExact) asm volatile("" ::: "memory");  // (the weight does not change: without this its reads are
#pragma unroll                                                 //  hoisted out of the loop over tiles, and spilled)
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[j][r] = 0.0f;
        const uint8_t *wt = lds + (g * kBlock8 + idx) * kPitch + 16 * half;
        i32x4 w[2][4][2];                                 // a stage's, and the next one's on its way from LDS
        auto read = [&](int s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[s % 2][j][0] = *reinterpret_cast<const i32x4 *>(wt + 32 * j * kPitch + 64 * s);
                w[s % 2][j][1] = *reinterpret_cast<const i32x4 *>(wt + 32 * j * kPitch + 64 * s + 32);
            }
        };
        if constexpr (!kExact) read(0);
#pragma unroll
        for (int s = 0; s < kStages; ++s) {
            const int sw = w_scales[g * KB + s / 2];
            const auto &ws = w[s % 2];
            if constexpr (!kExact) {
                if (s + 1 < kStages) read(s + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        __builtin_shufflevector(x[s][0], x[s][1], 0, 1, 2, 3, 4, 5, 6, 7),
                        __builtin_shufflevector(ws[j][0], ws[j][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[j], 0, 0, 0, sx[s / 2], 0, sw);
#pragma unroll
                for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(acc[j]));  // (keeps the stages apart)
                __builtin_amdgcn_sched_barrier(0);
            } else {                                      // (decoding leaves no room for a second stage of w)
                read(s);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const bf16x8_t hx = decode8(x[s][t / 2][2 * (t % 2)], x[s][t / 2][2 * (t % 2) + 1], scale_value(sx[s / 2]));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                            hx, decode8(ws[j][t / 2][2 * (t % 2)], ws[j][t / 2][2 * (t % 2) + 1], scale_value(sw)), acc[j], 0, 0, 0);
                }
            }
        }
    };
    // register r of lane l holds row (r % 4) + 8 (r / 4) + 4 (l / 32) of the tile, column l % 32 of tile j
    auto store = [&](int64_t tile, int g) {
        const int64_t c = (int64_t)g * kBlock8 + 4 * idx;
        const f32x4 b4 = p.bias ? load4<false>(p.bias, c, p.n) : f32x4{0.f, 0.f, 0.f, 0.f};
        O *out = static_cast<O *>(p.out) + (tile * 32 + 4 * half) * p.out_stride;
        const bool whole = tile * 32 + 32 <= p.rows;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = r % 4 + 8 * (r / 4);
            if (!whole && tile * 32 + 4 * half + row >= p.rows) continue;
            const f32x4 v = f32x4{acc[0][r], acc[1][r], acc[2][r], acc[3][r]} + b4;
            store_run(out + row * p.out_stride, c, p.n, p.vec, v);
        }
    };
    int64_t tile = (int64_t)wave * gridDim.x + blockIdx.x;
    if (tile < tiles) load(tile);
    for (; tile < tiles; tile += stride) {
        for (int g = 0; g < groups; ++g) {
            multiply(g);
            if (g == groups - 1) load(tile + stride);  // in front of the stores
            store(tile, g);
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
    constexpr size_t kLds = 4 * (size_t)(kM + kN) * (kBlock8 / 2);
    const int64_t tiles = ((p.rows + kM - 1) / kM) * ((p.n + kN - 1) / kN);
    if (tiles > 0x7fffffff) return fail(GNNAGG_ERR_UNSUPPORTED, "too many tiles");
    auto kernel = fp8_product_kernel<O, WM, WN, MW, NW>;
    if (kLds > 64 * 1024)
        GNNAGG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles), dim3(64 * MW * NW), kLds, st, p);
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}

// LDS of the kernel that keeps the weight there; 0: it does not fit
inline size_t rows_lds(const ProductArgs &p) {
    if (p.blocks > 4) return 0;
    const size_t groups = (size_t)((p.n + kBlock8 - 1) / kBlock8);
    const size_t bytes = groups * kBlock8 * (p.blocks * kBlock8 + 16) + groups * p.blocks;
    return p.n <= 4096 && bytes <= 160 * 1024 ? bytes : 0;
}

template <typename O, int KB>
int launch_rows(const ProductArgs &p, hipStream_t st) {
    auto kernel = fp8_product_rows_kernel<O, KB>;
    const size_t bytes = rows_lds(p);
    GNNAGG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL(kernel, dim3(256), dim3(512), bytes, st, p);
    GNNAGG_HIP(hipGetLastError());
    return GNNAGG_OK;
}

template <typename O>
int launch_product(const ProductArgs &p, hipStream_t st) {
    const int64_t columns = (p.n + 15) / 16;
    // Few rows, or a small result: the tiled kernel would have a block for each 128 columns and rows only, this one has one
    // for each 16 columns and 64 rows, up to two a compute unit (to bf16 unless said otherwise, this kernel / tiles:
    // 65 x 1024 x 1024 4.6 / 8.1 us, 300 x 512 x 256 3.6 / 6.7, 4000 x 128 x 128 3.3 / 5.4, 512 blocks: 2000 x 512 x 256
    // 5.0 / 6.8, 128 x 4096 x 4096 27 / 27 and to fp32 27 / 34, 512 x 4096 x 1024 27 / 27 and 27 / 34; 1000 blocks:
    // 4000 x 512 x 256 7.9 / 7.0, 256 x 4096 x 4096 52 / 27, 8000 x 128 x 128 4.5 / 5.5).
    if (p.rows <= 64 || columns * ((p.rows + 63) / 64) <= 512) {
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
    // Many rows against a weight that fits LDS: one of up to 128 columns is there at once, a wider one costs more to bring
    // than it saves below about 20 000 rows (this kernel / tiles, bf16 and fp32: 4500 rows 256 x 128 4.9 / 5.8 and 5.8 / 6.7 us,
    // 512 x 128 5.6 / 6.8 and 7.0 / 8.4; 9000 rows 256 x 256 7.2 / 6.4 and 9.4 / 7.8; 16 000 rows 256 x 256 7.7 / 7.4 and
    // 11.0 / 9.8, 512 x 256 10.6 / 9.4 and 14.6 / 12.0; 20 000 rows 256 x 256 8.3 / 9.5 and 11.6 / 12.1, 512 x 256 11.7 / 12.1
    // and 15.3 / 15.0, 256 x 172 7.9 / 8.4 and 10.8 / 11.2; 60 000 rows 512 x 256 17 / 23 and 25 / 32; 1 M rows 512 x 256
    // to fp32 0.34 / 0.64 ms).
    if ((p.rows >= 20000 || p.n <= kBlock8) && rows_lds(p)) {
        if (p.blocks == 1) return launch_rows<O, 1>(p, st);
        if (p.blocks == 2) return launch_rows<O, 2>(p, st);
        if (p.blocks == 3) return launch_rows<O, 3>(p, st);
        return launch_rows<O, 4>(p, st);
    }
    // Tiles of 256 x 256 feed the matrix units better, but a compute unit holds one block of them and nothing runs beside its
    // start and end: they pay where the contraction is long and the last round of blocks is nearly full (256 / 128, bf16 and
    // fp32: 8192^3 599 / 665 and 906 / 972 us, 8192 x 16384 x 2048 269 / 337 and 400 / 495, 9000 x 5120 x 5120 252 / 313 and
    // 401 / 443, 4096^3 81 / 80 and 114 / 129, 8192 x 4096 x 4096 188 / 185 and 234 / 263; rounds a quarter empty: 6000^3 259 / 273
    // and 444 / 392, 5000 x 4096 x 4096 129 / 103 and 208 / 159; short contractions: 8192 x 2048 x 4096 118 / 88 and 145 / 149,
    // 100 000 x 1024 x 1024 218 / 203 and 291 / 278).
    const int64_t large = ((p.rows + 255) / 256) * ((p.n + 255) / 256), rounds = (large + 255) / 256;
    if (p.blocks >= 32 && 10 * large >= 9 * 256 * rounds) return launch_tiles<O, 4, 4, 2, 2>(p, st);
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
    if (k > (int64_t(1) << 23) || n > (int64_t(1) << 34)) return fail(GNNAGG_ERR_UNSUPPORTED, "a weight of %lld x %lld", (long long)k, (long long)n);
    ProductArgs p{x, x_scales, w, w_scales, bias, out, scale_k_stride, scale_n_stride, out_stride, rows, n,
                  (int)(pad128(k) / kBlock8), 0};
    p.vec = vec4_rows(out, out_stride, n, out_dtype);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return out_dtype == GNNAGG_F32 ? launch_product<float>(p, st) : launch_product<bf16_t>(p, st);
}
