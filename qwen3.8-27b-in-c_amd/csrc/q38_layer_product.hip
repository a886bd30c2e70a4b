/* Rows in 8 bits times a matrix in e4m3 (q38hip_gemm_e4m3).
 *
 * Per output, the products of a block of 128 inputs are summed by the matrix
 * unit, 16 matrix rows by 16 tokens, with the tokens' powers of two applied to
 * its operands, and the matrix block's fp32 scale joins the result to the
 * running sum by one fma.  Lane i holds 32 codes of row (token) i % 16: 16
 * neighbours from 16 (i / 16) on and 16 from 64 + 16 (i / 16) on, in both operands
 * alike, so every load is a whole 64 bytes of a row.
 *
 * 16-bit outputs: one v_mfma_scale_f32_16x16x128_f8f6f4.  The unit adds products
 * of e4m3 codes at 13 bits below the largest of a group (measured with 2^8 -
 * 2^8 + t: t is kept down to 2^-5): 1.5e-5 to 3e-5 of the result's norm, a
 * hundredth of a bf16 output's rounding and a tenth of an fp16 output's.
 * fp32 outputs would keep that error, so for them codes become bf16 values
 * (exactly; four significant bits, the token's power of two in their exponent)
 * and four v_mfma_f32_16x16x32_bf16 sum their products with all 24 bits, at
 * half the rate. */
#include <type_traits>

#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kWaves = 8;

__device__ __forceinline__ i32x8 both(i32x4 low, i32x4 high)
{
    return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
}

/* eight codes as bf16 times a power of two */
__device__ __forceinline__ bf16x8 decoded(int low, int high, float scale)
{
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, scale, true);
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1,
                                   2, 3, 4, 5, 6, 7);
}

/* the products of a block: element r is matrix row 4 (lane / 16) + r, token lane %
 * 16.  `scale` is the token's scale byte; that of the matrix operand is 1 (127). */
__device__ __forceinline__ f32x4 block_product(i32x8 matrix, i32x8 token, uint32_t scale)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(matrix, token, f32x4{}, 0, 0, 0, 127, 0, (int)scale);
}
__device__ __forceinline__ f32x4 add_scaled(f32x4 sum, f32x4 p, float factor)
{
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[r] = fmaf(p[r], factor, sum[r]);
    return sum;
}
/* Both for fp32 outputs.  The token's power of two goes into its bf16 values as far as 2^-100 and 2^100, where those and
 * their products with codes are normal, the rest of it into the block's factor. */
__device__ __forceinline__ uint32_t token_scale(uint32_t scale) { return min(max(scale, 127u - 100), 127u + 100); }
__device__ __forceinline__ float block_factor(uint32_t scale, float factor)
{
    return scale == 255u ? __uint_as_float(0x7fc00000u) : ldexpf(factor, (int)scale - (int)token_scale(scale));
}
__device__ __forceinline__ f32x4 add_exact(f32x4 sum, i32x8 matrix, i32x8 token, uint32_t scale, float factor)
{
    const float power = __uint_as_float(token_scale(scale) << 23);
    f32x4 p = {};
#pragma unroll
    for (int q = 0; q < 4; ++q)
        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(decoded(matrix[2 * q], matrix[2 * q + 1], 1.0f),
                                                    decoded(token[2 * q], token[2 * q + 1], power), p, 0, 0, 0);
    return add_scaled(sum, p, factor);
}

template <typename T>
__device__ __forceinline__ void store_output(const ProductE4M3 &a, uint32_t token, uint32_t row, float v)
{
    static_cast<T *>(a.output)[(uint64_t)token * a.output_row + row] = static_cast<T>(v);
}

/* four neighbouring rows' outputs of a token, as far as there are rows; at any alignment of elements */
template <typename T>
__device__ __forceinline__ void store_four(const ProductE4M3 &a, uint32_t token, uint32_t row, f32x4 v)
{
    if (row + 4 <= a.outputs) {
        LayerSome<T, 4> some;
#pragma unroll
        for (int i = 0; i < 4; ++i) some.e[i] = static_cast<T>(v[i]);
        *reinterpret_cast<LayerSome<T, 4> *>(static_cast<T *>(a.output) + (uint64_t)token * a.output_row + row) = some;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row + i < a.outputs) store_output<T>(a, token, row + i, v[i]);
    }
}

/* 16 bytes of neighbouring rows' outputs of a token, as far as there are rows */
template <typename T>
__device__ __forceinline__ void store_piece(const ProductE4M3 &a, uint32_t token, uint32_t row, layer_u32x4 piece)
{
    constexpr uint32_t E = 16 / sizeof(T);
    T *to = static_cast<T *>(a.output) + (uint64_t)token * a.output_row + row;
    if (row + E <= a.outputs) {
        *reinterpret_cast<LayerSome<T, E> *>(to) = __builtin_bit_cast(LayerSome<T, E>, piece);
    } else {
        T e[E];
        __builtin_memcpy(e, &piece, 16);
#pragma unroll
        for (uint32_t i = 0; i < E; ++i)
            if (row + i < a.outputs) to[i] = e[i];
    }
}

/* 16 matrix rows by up to 16 tokens to a workgroup, whose eight wavefronts take
 * every eighth block of inputs and are summed in LDS in their order: many short
 * workgroups, whose loads are all in flight at once, for matrices that a second launch would
 * not repay (one token, 5120 x 5120: 8.3 us). */
template <typename T>
__global__ void __launch_bounds__(kWaves * 64) few_kernel(ProductE4M3 a)
{
    __shared__ float sums[kWaves][4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row0 = blockIdx.x * 16;
    const uint8_t *matrix = a.weight + (uint64_t)min(row0 + lane % 16, a.outputs - 1) * a.inputs;
    const uint64_t mine = min(lane % 16, a.tokens - 1);
    const uint8_t *codes = a.codes + mine * a.inputs, *scales = a.scales + mine * a.pitch;
    const float *weight_scales = a.weight_scales + (uint64_t)(row0 / kE4M3Block) * a.blocks;
    f32x4 sum = {};
    for (uint32_t b = wave; b < a.blocks; b += kWaves) {
        const uint32_t at = b * kE4M3Block + lane / 16 * 16;
        const bool low = at < a.inputs, high = at + 64 < a.inputs;
        const auto load = [&](const uint8_t *row) {
            const i32x4 l = low ? *reinterpret_cast<const i32x4 *>(row + at) : i32x4{};
            const i32x4 h = high ? *reinterpret_cast<const i32x4 *>(row + at + 64) : i32x4{};
            return both(l, h);
        };
        const i32x8 w = load(matrix), token = load(codes);
        const float s = weight_scales[b];
        if constexpr (std::is_same_v<T, float>) sum = add_exact(sum, w, token, scales[b], block_factor(scales[b], s));
        else sum = add_scaled(sum, block_product(w, token, scales[b]), s);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][r][lane] = sum[r];
    __syncthreads();
    /* an output to a thread: token i / 16, matrix row i % 16 */
    const uint32_t r = threadIdx.x % 16, t = threadIdx.x / 16;
    if (t >= a.tokens || row0 + r >= a.outputs) return;
    float v = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) v += sums[w][r % 4][r / 4 * 16 + t];
    store_output<T>(a, t, row0 + r, v);
}

/* ---- tiles --------------------------------------------------------------------- */

#define Q38_LDS __attribute__((address_space(3)))

/* 16 bytes per lane from base + offset to LDS at `to` + 16 lane, without registers;
 * the compiler does not count it, so the kernel waits itself (tile_barrier) */
__device__ __forceinline__ void copy_to_lds(const uint8_t *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to)
                 : "memory", "m0");
}
/* the same with 4 bytes per lane */
__device__ __forceinline__ void copy_words_to_lds(const void *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(offset), "s"(base), "s"(to)
                 : "memory", "m0");
}
/* all but the last N copies of this wavefront are in LDS and what it read has
 * returned; then so for all of the workgroup */
template <int N>
__device__ __forceinline__ void tile_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

/* A workgroup of GN x GM wavefronts, each with WN x WM tiles of 16 matrix rows by
 * 16 tokens; S blocks of inputs in LDS.  A stage holds the codes of the matrix's rows
 * and of the tokens, a word with the scale bytes of each token and the factors of the
 * matrix's blocks. */
template <int N, int M, int GN, int GM, int S>
struct ProductTile {
    static constexpr int WN = N, WM = M, kWavesM = GM, kWaveCount = GN * GM, kThreads = kWaveCount * 64, kStages = S;
    static constexpr int kRows = N * 16 * GN, kTokens = M * 16 * GM;
    static constexpr int kScalesAt = (kRows + kTokens) * (int)kE4M3Block;
    static constexpr int kFactorsAt = kScalesAt + (kTokens < 64 ? 64 : kTokens) * 4;
    static constexpr int kStage = kFactorsAt + 256;
    /* copies of 1 KiB of a wavefront; the last ones of the tokens may be some wavefronts' only */
    static constexpr int kRowParts = kRows / 8 / kWaveCount, kTokenParts = (kTokens / 8 + kWaveCount - 1) / kWaveCount;
    static constexpr int kLeast = kRowParts + kTokens / 8 / kWaveCount;
    static_assert(kRowParts * kWaveCount * 8 == kRows && kTokens <= 64 * kWaveCount, "copies of a stage");
    static_assert(WN * 16 <= (int)kE4M3Block && kE4M3Block % (WN * 16) == 0, "a wavefront's rows have one factor");
};
using Tile256 = ProductTile<8, 4, 2, 4, 2>;
using Tile128 = ProductTile<4, 4, 2, 2, 3>;
using Tile64 = ProductTile<2, 4, 4, 1, 4>;
using Tile16 = ProductTile<2, 1, 4, 1, 4>;
template <typename Tile>
constexpr bool tile_is(int tile) { return (int)kProductRows[tile] == Tile::kRows && (int)kProductTokens[tile] == Tile::kTokens; }
static_assert(tile_is<Tile256>(kProductTile256) && tile_is<Tile128>(kProductTile128) && tile_is<Tile64>(kProductTile64) &&
                  tile_is<Tile16>(kProductTile16), "the plan's tiles");

/* Rows of 128 bytes in LDS; the eight 16-byte pieces of row r are turned by r / 2: the
 * 16 lanes that a 16-byte read serves together (of each 32 the lanes 0..3, 12..15,
 * 20..27, then the others) find places of their own modulo 256 bytes. */
__device__ __forceinline__ uint32_t piece_turn(uint32_t row) { return row >> 1 & 7; }

/* The first plan.whole tiles are formed by a workgroup each; of the others plan.splits
 * workgroups sum a part of the inputs each (a block at least), into
 * a.partial[tile][split][token][row].  Blocks of inputs go through stages of LDS: one is
 * read while the next ones are on their way.
 *
 * Few tokens are bound by the matrix: one token, 5120 x 34816, 35 us, 5.1 TB/s; 48 tokens, 17408 x
 * 5120, 21.6 us with the join's 4.  4096 tokens, 5120 x 34816: 704 us, 2.07 PFLOP/s.  There copying
 * the stages alone takes 640 us (330 if all came from the die's cache): a unit has room for one
 * stage of 64 KiB ahead, which arrives about when it is due; products, sums and reads from LDS
 * alone take 565, writing the results about 50.  The fma of each product's sums, under the next
 * products, costs a seventh of the matrix unit's rate with two wavefronts to a SIMD, a third with one. */
template <typename T, typename Tile>
__global__ void __launch_bounds__((Tile::kThreads), 2) tile_kernel(ProductE4M3 a, ProductPlan plan)
{
    constexpr int WN = Tile::WN, WM = Tile::WM, kWaveCount = Tile::kWaveCount, kStages = Tile::kStages;
    constexpr int kRowParts = Tile::kRowParts, kTokenParts = Tile::kTokenParts;
    __shared__ __align__(1024) uint8_t stages[kStages * Tile::kStage];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tiles_n = layer_up(a.outputs, Tile::kRows), tiles_m = layer_up(a.tokens, Tile::kTokens);

    const bool whole = blockIdx.x < plan.whole;
    const uint32_t place = whole ? die_place(blockIdx.x, plan.whole) : die_place(blockIdx.x - plan.whole, gridDim.x - plan.whole);
    const uint32_t rest = place / plan.splits, splits = whole ? 1 : plan.splits, split = whole ? 0 : place - rest * splits;
    const TilePlace tile = tile_place(whole ? place : plan.whole + rest, tiles_n, tiles_m);
    const uint32_t row0 = tile.n * Tile::kRows, token0 = tile.m * Tile::kTokens;
    const uint32_t first = (uint64_t)a.blocks * split / splits, end = (uint64_t)a.blocks * (split + 1) / splits;

    /* what this lane copies: 8 rows of 128 bytes at a time */
    const uint8_t *matrix = a.weight + (uint64_t)row0 * a.inputs, *codes = a.codes + (uint64_t)token0 * a.inputs;
    /* rows shorter than a block lie at the end of the stage's, their first codes before them too */
    const uint32_t missing = __builtin_amdgcn_readfirstlane(a.inputs < kE4M3Block ? kE4M3Block - a.inputs : 0);
    uint32_t offset[kRowParts + kTokenParts];
#pragma unroll
    for (int i = 0; i < kRowParts + kTokenParts; ++i) {
        const bool token = i >= kRowParts;
        const uint32_t r = ((token ? i - kRowParts : i) * kWaveCount + wave) * 8 + lane / 8;
        const uint32_t last = (token ? a.tokens - token0 : a.outputs - row0) - 1;
        offset[i] = min(r, last) * a.inputs + max(((lane & 7) ^ piece_turn(r)) * 16, missing) - missing;
    }
    const uint32_t stages_at = (uint32_t)(uintptr_t)(Q38_LDS const void *)stages;
    /* wavefront w copies the words of tokens 64 w on, the last one the factors */
    const bool has_scales = wave * 64 < Tile::kTokens;
    const uint8_t *scales = a.scales + (uint64_t)token0 * a.pitch;
    const uint32_t scale_offset = min(wave * 64 + lane, a.tokens - token0 - 1) * a.pitch;
    const float *factors = a.weight_scales + (uint64_t)(row0 / kE4M3Block) * a.blocks;
    constexpr uint32_t kFactors = (Tile::kRows + kE4M3Block - 1) / kE4M3Block;
    const uint32_t factor_offset = min(lane % kFactors, (a.outputs - 1) / kE4M3Block - row0 / kE4M3Block) * a.blocks * 4;
    const auto load = [&](uint32_t block, uint32_t stage_at) {
        if (has_scales) copy_words_to_lds(scales + block / 4 * 4, scale_offset, stage_at + Tile::kScalesAt + wave * 256);
        if (wave == kWaveCount - 1) copy_words_to_lds(factors + block, factor_offset, stage_at + Tile::kFactorsAt);
        /* of a row's end the last 128 codes, so nothing behind it is read */
        const uint32_t from = min(block * kE4M3Block, a.inputs + missing - kE4M3Block);
#pragma unroll
        for (int i = 0; i < kRowParts + kTokenParts; ++i)
            if (i < Tile::kLeast || (i - kRowParts) * kWaveCount + wave < Tile::kTokens / 8)
                copy_to_lds((i < kRowParts ? matrix : codes) + from, offset[i], stage_at + (i * kWaveCount + wave) * 1024);
    };

    const uint32_t wave_row = wave / Tile::kWavesM * (WN * 16), wave_token = wave % Tile::kWavesM * (WM * 16);
    /* a lane's pieces lane / 16 and 4 + lane / 16 of row lane % 16 of a tile of 16 rows; tiles
     * are 2 KiB apart, which the reads' own offsets take */
    const uint32_t piece = (lane / 16 ^ piece_turn(lane % 16)) * 16;
    uint32_t rows_at = (wave_row + lane % 16) * kE4M3Block + piece;
    uint32_t tokens_at = (Tile::kRows + wave_token + lane % 16) * kE4M3Block + piece;
    asm volatile("" : "+v"(rows_at), "+v"(tokens_at));
    f32x4 sum[WN][WM] = {};
    const uint32_t stages_end = stages_at + kStages * Tile::kStage;
    uint32_t stage_at = stages_at, load_at = stages_at, loaded = first;
    const auto load_next = [&] {
        load(loaded++, load_at);
        load_at += Tile::kStage;
        if (load_at == stages_end) load_at = stages_at;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (loaded < end) load_next();
    for (uint32_t block = first; block < end; ++block) {
        /* where fewer copies follow than the loop leaves open, all are waited for */
        if (end - block >= kStages - 1) tile_barrier<(kStages - 2) * Tile::kLeast>();
        else tile_barrier<0>();
        if (loaded < end) load_next();
        uint32_t scale[WM];
        const float factor = *(Q38_LDS const float *)(uintptr_t)(stage_at + Tile::kFactorsAt + wave_row / kE4M3Block * 4);
#pragma unroll
        for (int m = 0; m < WM; ++m)
            scale[m] = *(Q38_LDS const uint8_t *)(uintptr_t)(stage_at + Tile::kScalesAt + (wave_token + m * 16 + lane % 16) * 4 + block % 4);
        const uint32_t row_low = rows_at + stage_at, row_high = row_low ^ 64, token_low = tokens_at + stage_at, token_high = token_low ^ 64;
        stage_at += Tile::kStage;
        if (stage_at == stages_end) stage_at = stages_at;
        const auto read = [](uint32_t low, uint32_t high, int tile) {
            return both(*(Q38_LDS const i32x4 *)(uintptr_t)(low + tile * 16 * kE4M3Block),
                        *(Q38_LDS const i32x4 *)(uintptr_t)(high + tile * 16 * kE4M3Block));
        };
        i32x8 token[WM];
#pragma unroll
        for (int m = 0; m < WM; ++m) token[m] = read(token_low, token_high, m);
        if (a.inputs - block * kE4M3Block < kE4M3Block) {
            /* the stage begins with codes of the block before: they count as 0 */
            const uint32_t before = (block + 1) * kE4M3Block - a.inputs;
            const bool low = lane / 16 * 16 >= before, high = lane / 16 * 16 + 64 >= before;
#pragma unroll
            for (int m = 0; m < WM; ++m)
#pragma unroll
                for (int i = 0; i < 8; ++i) token[m][i] = (i < 4 ? low : high) ? token[m][i] : 0;
        }
        if constexpr (std::is_same_v<T, float>) {
            float factors[WM];
#pragma unroll
            for (int m = 0; m < WM; ++m) factors[m] = block_factor(scale[m], factor);
#pragma unroll
            for (int n = 0; n < WN; ++n) {
                const i32x8 rows = read(row_low, row_high, n);
#pragma unroll
                for (int m = 0; m < WM; ++m) sum[n][m] = add_exact(sum[n][m], rows, token[m], scale[m], factors[m]);
            }
        } else {
            /* a product's result takes longer than the next product's start: the sums of one
             * row of tiles are formed while the next row's products run */
            i32x8 rows = read(row_low, row_high, 0);
            f32x4 before[WM];
#pragma unroll
            for (int n = 0; n <= WN; ++n) {
                i32x8 following;
                if (n + 1 < WN) following = read(row_low, row_high, n + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int m = 0; m < WM; ++m) {
                    f32x4 now;
                    if (n < WN) now = block_product(rows, token[m], scale[m]);
                    if (n > 0) sum[n - 1][m] = add_scaled(sum[n - 1][m], before[m], factor);
                    before[m] = now;
                    __builtin_amdgcn_sched_barrier(0);
                }
                rows = following;
            }
        }
    }

    if (!whole) {
        float *part = a.partial + (uint64_t)place * (Tile::kRows * Tile::kTokens);
#pragma unroll
        for (int m = 0; m < WM; ++m) {
            const uint32_t t = wave_token + m * 16 + lane % 16;
            if (token0 + t < a.tokens) {
#pragma unroll
                for (int n = 0; n < WN; ++n)
                    *reinterpret_cast<f32x4 *>(part + t * Tile::kRows + wave_row + n * 16 + lane / 16 * 4) = sum[n][m];
            }
        }
        return;
    }
    /* A lane has four outputs of a token at a time.  Those of 16 tokens go through LDS, the
     * wavefront's own part of the stages, so that what is written is whole pieces of rows. */
    constexpr int E = 16 / (int)sizeof(T), kPieces = WN * 16 / E, kTurn = kPieces < 16 ? 16 / kPieces : 1;
    constexpr uint32_t kPart = WN * 16 * 16 * sizeof(T);
    static_assert(kPart * kWaveCount <= kStages * Tile::kStage, "a part to each wavefront");
    tile_barrier<0>();                                       /* the stages have been read */
    const uint32_t part_at = stages_at + wave * kPart;
    const auto place_of = [&](uint32_t t, uint32_t piece) { return part_at + (t * kPieces + (piece ^ t / kTurn % kPieces)) * 16; };
#pragma unroll
    for (int m = 0; m < WM; ++m) {
#pragma unroll
        for (int n = 0; n < WN; ++n) {
            const uint32_t row = n * 16 + lane / 16 * 4;
            T e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = static_cast<T>(sum[n][m][i]);
            const uint32_t at = place_of(lane % 16, row / E) + row % E * sizeof(T);
            if constexpr (sizeof(T) == 2) *(Q38_LDS layer_u32x2 *)(uintptr_t)at = __builtin_bit_cast(layer_u32x2, e);
            else *(Q38_LDS layer_u32x4 *)(uintptr_t)at = __builtin_bit_cast(layer_u32x4, e);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 64 / kPieces) {
            const uint32_t t = i + lane / kPieces, token = token0 + wave_token + m * 16 + t;
            const uint32_t row = row0 + wave_row + lane % kPieces * E;
            const layer_u32x4 piece = *(Q38_LDS const layer_u32x4 *)(uintptr_t)place_of(t, lane % kPieces);
            if (token < a.tokens) store_piece<T>(a, token, row, piece);
        }
    }
}

/* the sums of the tiles that were cut, parts in their order; a thread takes four rows of a token */
template <typename T, typename Tile>
__global__ void __launch_bounds__(256) join_kernel(ProductE4M3 a, ProductPlan plan)
{
    constexpr uint32_t kFours = Tile::kRows * Tile::kTokens / 4, kWorkgroups = kFours / 256;
    const uint32_t rest = blockIdx.x / kWorkgroups, four = blockIdx.x % kWorkgroups * 256 + threadIdx.x;
    const TilePlace tile = tile_place(plan.whole + rest, layer_up(a.outputs, Tile::kRows), layer_up(a.tokens, Tile::kTokens));
    const uint32_t token = tile.m * Tile::kTokens + four / (Tile::kRows / 4), row = tile.n * Tile::kRows + four % (Tile::kRows / 4) * 4;
    if (token >= a.tokens || row >= a.outputs) return;
    const f32x4 *part = reinterpret_cast<const f32x4 *>(a.partial) + (uint64_t)rest * plan.splits * kFours + four;
    f32x4 sum = {};
    for (uint32_t s = 0; s < plan.splits; s += 4) {
        f32x4 v[4];                                          /* asked for together */
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = part[(uint64_t)min(s + i, plan.splits - 1) * kFours];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (s + i < plan.splits) sum += v[i];
    }
    store_four<T>(a, token, row, sum);
}

template <typename T, typename Tile>
bool tiled(const ProductE4M3 &a, const ProductPlan &plan, hipStream_t stream)
{
    const uint32_t tiles = layer_up(a.outputs, Tile::kRows) * layer_up(a.tokens, Tile::kTokens), rest = tiles - plan.whole;
    if (!launch_kernel(tile_kernel<T, Tile>, dim3(plan.whole + rest * plan.splits), dim3(Tile::kThreads), stream, a, plan))
        return false;
    return !rest || launch_kernel(join_kernel<T, Tile>, dim3(rest * (Tile::kRows * Tile::kTokens / 1024)), dim3(256), stream, a, plan);
}

template <typename T>
bool product(const ProductE4M3 &a, hipStream_t stream)
{
    const ProductPlan plan = plan_product(a.tokens, a.inputs, a.outputs);
    if (plan.tile == kProductTile256) return tiled<T, Tile256>(a, plan, stream);
    if (plan.tile == kProductTile128) return tiled<T, Tile128>(a, plan, stream);
    if (plan.tile == kProductTile16) return tiled<T, Tile16>(a, plan, stream);
    if (plan.tile == kProductTile64) return tiled<T, Tile64>(a, plan, stream);
    return launch_kernel(few_kernel<T>, dim3(layer_up(a.outputs, 16)), dim3(kWaves * 64), stream, a);
}

}  // namespace

uint64_t product_e4m3_workspace_bytes(uint32_t tokens, uint64_t inputs, uint32_t outputs)
{
    return plan_product(tokens, (uint32_t)inputs, outputs).bytes;
}

bool launch_product_e4m3(const ProductE4M3 &a, hipStream_t stream)
{
    return a.type == kLayerF32 ? product<float>(a, stream) : a.type == kLayerF16 ? product<_Float16>(a, stream)
                                                                                 : product<__bf16>(a, stream);
}

}  // namespace q38
