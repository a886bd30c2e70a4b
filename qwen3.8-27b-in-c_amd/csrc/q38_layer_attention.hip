/* Causal attention of packed prompts (q38hip_prompt_attention). */
#include <type_traits>

#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

/* First row of the sequence that owns `row`, or -1 where none does: the last
 * sequence that starts at or before it, so empty ones are passed over.  Always
 * in 0 .. row, whatever the words hold. */
__device__ __forceinline__ int sequence_start(const PromptAttention &a, uint32_t row, uint32_t lane)
{
    if (a.count < 64) {                         /* one load: an offset to a lane */
        const int begin = a.row_starts[min(lane, a.count)];
        const uint32_t low = __popcll(__ballot(lane <= a.count && begin <= (int)row));
        if (low == 0 || low == a.count + 1) return -1;
        return min(max(__builtin_amdgcn_readlane(begin, low - 1), 0), (int)row);
    }
    uint32_t low = 0, high = a.count + 1;       /* row_starts[low - 1] <= row < row_starts[high] */
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (a.row_starts[mid] <= (int)row) low = mid + 1;
        else high = mid;
    }
    if (low == 0 || low == a.count + 1) return -1;
    return min(max(a.row_starts[low - 1], 0), (int)row);
}

__device__ __forceinline__ float quad_sum_f32(float v)
{
    v += __int_as_float(dpp_move<0xB1>(0, __float_as_int(v)));
    return v + __int_as_float(dpp_move<0x4E>(0, __float_as_int(v)));
}
__device__ __forceinline__ float wave_sum_f32(float v)
{
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i);
    return v;
}

/* One row of one head by one wavefront, 64 keys at a time with a running maximum;
 * only keys and values that the row sees are read.  Four lanes form a score, each
 * from 16 of every 64 bytes of a key, so a load is 16 whole pieces of 64 bytes; then a
 * lane sums D / 64 neighbouring channels of the values.
 *
 * Values are read 16 at a time, behind the row the row's own again, times the weight 0: NaN where that value is
 * infinite.  With kHidden they count as 0; without, what came out not finite is done again so (37 rows of
 * 24 heads of 256: 5.8 us, fp32 and bf16; 6.5 and 6.7 with the selects for all rows). */
template <typename T, int D, bool kWhole, bool kHidden>
__device__ __forceinline__ void attend_row(const PromptAttention &a, uint32_t row, uint32_t head, uint32_t lane)
{
    constexpr int E = 16 / (int)sizeof(T), C = D / (4 * E), kChannels = D / 64;
    const int start = sequence_start(a, row, lane);
    if (start < 0) return;
    const auto sixteen = [=](const T *from) {
        if constexpr (kWhole) return *reinterpret_cast<const layer_u32x4 *>(from);
        T e[E];
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = from[i];
        return __builtin_bit_cast(layer_u32x4, e);
    };
    const uint32_t kv = head / (a.heads / a.kv_heads), part = lane % 4 * E, channel = lane * kChannels;
    const uint64_t query = (uint64_t)row * a.query_row + (uint64_t)head * a.query_head;
    const T *keys = static_cast<const T *>(a.key) + kv * D + part, *values = static_cast<const T *>(a.value) + kv * D + channel;
    float q[C][E], out[kChannels] = {}, top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const layer_u32x4 raw = sixteen(static_cast<const T *>(a.query) + query + part + c * 4 * E);
#pragma unroll
        for (int e = 0; e < E; ++e) q[c][e] = static_cast<float>(reinterpret_cast<const T *>(&raw)[e]) * a.scale;
    }
    float gate[kChannels] = {};
    if (a.gate) {
#pragma unroll
        for (int e = 0; e < kChannels; ++e)
            gate[e] = static_cast<float>(static_cast<const T *>(a.gate)[query + channel + e]);
    }
    for (uint32_t first = start; first <= row; first += 64) {
        float s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = -INFINITY;
        /* 16-bit keys are asked for 16 at a time while the last 16 are multiplied (24 heads of 256, 37 rows: 6.0
         * instead of 8.1 us); for fp32 that costs registers and wavefronts (6.3 instead of 5.9) */
        constexpr int kInFlight = sizeof(T) == 2 ? 2 : 1;
        layer_u32x4 pieces[kInFlight][C];
        const auto ask = [&](int u) {
            const T *from = keys + (uint64_t)min(first + u * 16 + lane / 4, row) * a.key_row;
#pragma unroll
            for (int c = 0; c < C; ++c) pieces[u % kInFlight][c] = sixteen(from + c * 4 * E);
        };
        if (kInFlight > 1) ask(0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int next = u + kInFlight - 1;
            if (next < 4 && first + next * 16 <= row) ask(next);
            if (first + u * 16 > row) continue;
            const uint32_t key = first + u * 16 + lane / 4;
            const layer_u32x4 (&raw)[C] = pieces[u % kInFlight];
            float dot[2] = {};
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e)
                    dot[c % 2] = fmaf(q[c][e], static_cast<float>(reinterpret_cast<const T *>(&raw[c])[e]), dot[c % 2]);
            const float score = quad_sum_f32(dot[0] + dot[1]);
            if (key <= row) s[u] = score;
        }
        const float higher = fmaxf(top, wave_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
        /* nothing but -infinity so far: differences would be NaN, weights are 0 */
        const float base = higher == -INFINITY ? 0.0f : higher, shrink = __builtin_amdgcn_exp2f(top - base);
        top = higher;
        total *= shrink;
#pragma unroll
        for (int u = 0; u < 4; ++u) total += s[u] = __builtin_amdgcn_exp2f(s[u] - base);
        /* a score that is NaN: so are all channels, whatever follows */
        if (kHidden && __any(total != total)) break;
#pragma unroll
        for (int e = 0; e < kChannels; ++e) out[e] *= shrink;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (first + u * 16 > row) continue;
            /* behind the row itself its own value again, with the weight 0, or as 0 */
            const uint32_t seen = row - (first + u * 16) + 1;
            T v[16][kChannels];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const T *from = values + (uint64_t)min(first + u * 16 + j, row) * a.value_row;
                if constexpr (kWhole) {
                    struct Some { T e[kChannels]; } __attribute__((aligned(sizeof(T) * kChannels)));
                    const Some some = *reinterpret_cast<const Some *>(from);
#pragma unroll
                    for (int e = 0; e < kChannels; ++e) v[j][e] = some.e[e];
                } else {
#pragma unroll
                    for (int e = 0; e < kChannels; ++e) v[j][e] = from[e];
                }
            }
            const auto add = [&](auto all) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float weight = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s[u]), j * 4));
#pragma unroll
                    for (int e = 0; e < kChannels; ++e)
                        out[e] = fmaf(weight, all || (uint32_t)j < seen ? static_cast<float>(v[j][e]) : 0.0f, out[e]);
                }
            };
            if (!kHidden || seen >= 16) add(std::true_type());
            else add(std::false_type());
        }
    }
    /* the four lanes of a score each counted it */
    const float inverse = 4.0f / wave_sum_f32(total);
    if constexpr (!kHidden) {
        float nothing = 0.0f;
#pragma unroll
        for (int e = 0; e < kChannels; ++e) nothing = fmaf(out[e] * inverse, 0.0f, nothing);
        if (__any(nothing != 0.0f)) return attend_row<T, D, kWhole, true>(a, row, head, lane);
    }
    T *to = static_cast<T *>(a.output) + (uint64_t)row * a.output_row + (uint64_t)head * D + channel;
#pragma unroll
    for (int e = 0; e < kChannels; ++e) {
        float v = out[e] * inverse;
        if (a.gate) v *= sigmoid_f32(gate[e]);
        to[e] = static_cast<T>(v);
    }
}

/* A wavefront to a row and head.  Bound by latency: the offsets, then keys, then values (37 fp32 rows
 * of 24 heads of 256: 6 us). */
template <typename T, int D, bool kWhole>
__global__ void __launch_bounds__(256) row_kernel(PromptAttention a)
{
    const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= a.rows * a.heads) return;
    attend_row<T, D, kWhole, false>(a, item / a.heads, item % a.heads, threadIdx.x & 63);
}

/* ---- tiles of the matrix unit ------------------------------------------------ */

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define Q38_LDS __attribute__((address_space(3)))

__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return (uint32_t)(uintptr_t)(Q38_LDS const void *)p;
}
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at)
{
    return *(Q38_LDS const V *)(uintptr_t)at;
}
/* 16 bytes per lane from memory to LDS at `to` + 16 lane, without registers; the
 * compiler does not count it, so the kernel waits itself (tile_barrier) */
__device__ __forceinline__ void copy_to_lds(const void *from, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
/* the same from base + offset */
__device__ __forceinline__ void copy_to_lds(const void *base, uint32_t offset, uint32_t to)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(to)
                 : "memory", "m0");
}
/* what this wavefront asked for is in LDS and what it read has returned; then so
 * for all of the workgroup */
__device__ __forceinline__ void tile_barrier()
{
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* the same for what was read from and written to LDS alone */
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* c + A B over 16 bytes of a row from each lane: A's rows and B's columns are
 * lane % 32, the inner index is the lane's half and the place in the 16 bytes, in both
 * alike.  Element r of c is row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32. */
template <typename T>
__device__ __forceinline__ f32x16 multiply(u32x4 rows, u32x4 columns, f32x16 c)
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, rows), y = __builtin_bit_cast(f32x4, columns);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
        return c;
    } else if constexpr (std::is_same_v<T, _Float16>) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, rows), __builtin_bit_cast(f16x8, columns), c, 0,
                                                      0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, rows), __builtin_bit_cast(bf16x8, columns), c,
                                                       0, 0, 0);
    }
}

/* c + the two 16-bit numbers of a word, within 2^-22 of the sum */
template <typename T>
__device__ __forceinline__ float add_pair(uint32_t pair, float c)
{
    if constexpr (std::is_same_v<T, _Float16>)
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), f16x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
    else
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
}

/* the value of both halves of the wavefront, in both */
__device__ __forceinline__ float halves_max(float v)
{
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v)
{
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
/* sum and maximum over the wavefront; every lane is active (rows that a broadcast leaves out add 0) */
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v)
{
    v += dpp_move<0xB1>(0, (int)v);
    v += dpp_move<0x4E>(0, (int)v);
    v += dpp_move<0x141>(0, (int)v);
    v += dpp_move<0x140>(0, (int)v);
    v += dpp_move<0x142, 0xA>(0, (int)v);
    v += dpp_move<0x143, 0xC>(0, (int)v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v)
{
    v = row16_max(v);
    v = max(v, (uint32_t)dpp_move<0x142, 0xA>(0, (int)v));
    v = max(v, (uint32_t)dpp_move<0x143, 0xC>(0, (int)v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
/* the least of numbers above -2^30 */
__device__ __forceinline__ int wave_min(int v)
{
    return (int)(0x7fffffffu - wave_max_u32(0x7fffffffu - (uint32_t)v));
}

/* 16 bytes of a row, and to one: the results stream past the caches, which the next kernel finds empty of
 * them anyway (64 prompts of 32 rows, 32 heads of 128, bf16: 13.5 -> 11.2 us, with a reader behind 21.5 -> 19.3) */
template <bool kWhole, typename T>
__device__ __forceinline__ u32x4 load_piece(const T *from)
{
    if constexpr (kWhole) return *reinterpret_cast<const u32x4 *>(from);
    T e[16 / sizeof(T)];
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) e[i] = from[i];
    return __builtin_bit_cast(u32x4, e);
}
template <bool kWhole, typename T>
__device__ __forceinline__ void store_piece(T *to, u32x4 piece)
{
    if constexpr (kWhole) {
        __builtin_nontemporal_store(piece, reinterpret_cast<u32x4 *>(to));
    } else {
        T e[16 / sizeof(T)];
        __builtin_memcpy(e, &piece, 16);
#pragma unroll
        for (int i = 0; i < 16 / (int)sizeof(T); ++i) to[i] = e[i];
    }
}

/* Sizes of a workgroup: kWaves wavefronts of 32 columns, tiles of kKeys keys.  A
 * column is a row and one of the query heads that share a key/value head, columns of a
 * row next to each other, so all of a tile's columns read the same keys and values.
 * With kShares = 4 the four wavefronts share 32 columns: each takes a fourth of the channels in both products,
 * and the parts of the scores are joined through LDS. */
template <typename T, int D, int kShares>
struct PromptTile {
    static constexpr int kWaves = 4;
    /* Wavefronts of a SIMD, which share 512 registers a lane: two hide each other's softmax
     * (bf16, 256-wide heads, 8197 tokens: 724 us, one with twice the keys 858).  The queries and sums
     * of 256-wide fp32 heads alone fill the registers of one. */
    static constexpr int kPerUnit = D * sizeof(T) / kShares == 1024 ? 1 : 2;
    static constexpr int kKeys = sizeof(T) == 4 || D == 256 ? 32 : 64;
    static constexpr int kRowBytes = D * (int)sizeof(T);
    static constexpr int kHalf = kKeys * kRowBytes;          /* keys or values of a tile */
    static constexpr uint32_t kColumns = kWaves / kShares * 32;
};

/* Where 16-byte piece `piece` of row `row` lies in its row in LDS.  Keys are read
 * 16 bytes a lane, 16 rows together, so the turn is the row; 16-bit values are read
 * transposed, 64 bytes of four rows together, so the turn is the row modulo 4 in
 * units of 64 bytes.  Values of fp32 are read along their rows: no turn.  All turns
 * are bits of the row put elsewhere, so the turn of a sum of rows without common bits is
 * the exclusive-or of their turns. */
template <int kRowBytes>
__device__ __forceinline__ uint32_t key_turn(uint32_t row)
{
    return kRowBytes >= 256 ? row & 15 : (row >> 1) & 7;
}
template <typename T, int kRowBytes>
__device__ __forceinline__ uint32_t value_turn(uint32_t row)
{
    if (sizeof(T) == 4) return 0;
    return kRowBytes >= 256 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

/* What is not finite among the values and keys of rows first .. last, of which all columns of a wavefront see latest ..
 * earliest.  values: no row that a column may not see has one, and the others are too small for a sum of them to overflow
 * (weights are below 2^9; fp16 rows' are larger, but their values end at 2^16), so what a column's sums make of the values that it sees is
 * right.  fp16 weights may be 0 where they are small, times an infinity NaN: infinities do not count as right there.  key:
 * the first row with a NaN among its keys, which makes all channels of a column that sees it NaN.  One more pass over the rows by
 * each wavefront: 24 heads of 256, bf16, 8197 tokens 0.75 ms, with a NaN among the first row's values or keys 3.3, both of the
 * middle row 6.0; 2048 tokens 0.08 and 0.39.  Without it every column that sees one is done again: 41 ms, 4.2. */
struct Seen {
    bool values;
    int key;
};
template <typename T, int D, bool kWhole>
__device__ __forceinline__ Seen look_over(const PromptAttention &a, uint32_t kv, int first, int last, int latest, int earliest, uint32_t lane)
{
    constexpr int E = 16 / (int)sizeof(T), kPieces = D / E, kRows = 64 / kPieces, kInFlight = 4;
    const uint64_t at = kv * D + lane % kPieces * E;
    const T *keys = static_cast<const T *>(a.key) + at, *values = static_cast<const T *>(a.value) + at;
    uint32_t largest = 0, other = 0;
    int key = INT32_MAX;
    for (int from = first; from <= last; from += kInFlight * kRows) {
        u32x4 k[kInFlight], v[kInFlight];
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const uint64_t row = min(from + i * kRows + (int)(lane / kPieces), last);
            k[i] = load_piece<kWhole>(keys + row * a.key_row);
            v[i] = load_piece<kWhole>(values + row * a.value_row);
        }
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int row = min(from + i * kRows + (int)(lane / kPieces), last);
            const bool hidden = row < latest || row > earliest;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = static_cast<float>(reinterpret_cast<const T *>(&k[i])[e]);
                const uint32_t bits = __float_as_uint(static_cast<float>(reinterpret_cast<const T *>(&v[i])[e])) & 0x7fffffffu;
                if (x != x) key = min(key, row);
                if (bits < 0x7f800000u) largest = max(largest, bits);
                else if (hidden || (std::is_same_v<T, _Float16> && bits == 0x7f800000u)) other = 1;
            }
        }
    }
    key = wave_min(key);
    return {wave_max_u32(other) == 0 && __uint_as_float(wave_max_u32(largest)) * (float)(last - first + 1) < 0x1p118f, key};
}

/* Causal attention of a tile of columns.
 *
 * S^T = K Q^T leaves each lane the scores of one column, and its result has, in
 * each half of the wavefront, the keys that the second product, O^T = V^T P^T, takes
 * from that half: the weights go from one product to the other in registers.  So
 * statistics and rescaling are per lane; one exchange between the halves joins a
 * maximum.  The maximum that weights are relative to is moved only where a score
 * exceeds it by more than 2^8 (fp16: or a tile's largest is 2^12 below): then the sums are rescaled.
 *
 * Pieces of keys and values are read from LDS kAhead products early, the first of the
 * values before the softmax: a product that waits for a read of its own leaves the matrix
 * units idle (bf16, 24 heads of 256, 8197 tokens: 724 us, 797 with each read at its product).
 * That is 1.14 PFLOP/s, what a large library product of bf16 reaches; the matrix unit is busy 0.61
 * of the cycles.  fp32 (0.095 PFLOP/s of 0.154) is bound by the fp32 products themselves.  Many
 * short prompts are bound by what a tile does once: 12 of up to 1500 tokens, 32 heads of 128, 57 us.
 *
 * With kParts = 2 the workgroup has twice the wavefronts; the second half of them takes
 * every other tile of keys for the same columns, and its sums join the first's through LDS. */
template <typename T, int D, bool kWhole, int kParts, int kShares>
__global__ void __launch_bounds__((PromptTile<T, D, kShares>::kWaves * 64 * kParts), (PromptTile<T, D, kShares>::kPerUnit))
    prompt_kernel(PromptAttention a)
{
    using Tile = PromptTile<T, D, kShares>;
    constexpr int kWaves = Tile::kWaves, kRowBytes = Tile::kRowBytes, kKeys = Tile::kKeys, kHalf = Tile::kHalf;
    constexpr int kSteps = kRowBytes / 32;                   /* 16 bytes a lane each */
    constexpr int kTiles = kKeys / 32, kAhead = 3;
    constexpr int kOwnSteps = kSteps / kShares, kOwn = D / kShares;      /* of the wavefront's channels */
    static_assert(kShares == 1 || (kOwnSteps == 8 && kParts == 1 && kTiles == 1), "shares of 256 bytes");
    /* of each part keys and values, two of each; then the second part's sums and statistics */
    constexpr int kTilesBytes = kParts * 4 * kHalf, kJoinBytes = kParts > 1 ? (D / 2 + 2) * 256 * kWaves : 0;
    __shared__ __align__(1024) uint8_t tiles[kTilesBytes > kJoinBytes ? kTilesBytes : kJoinBytes];
    __shared__ int ranges[kWaves][2];
    const uint32_t lane = threadIdx.x & 63, part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWaves;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves;
    const uint32_t half = lane >> 5, low = lane & 31, share = wave % kShares;
    const uint32_t group = a.heads / a.kv_heads, kv = blockIdx.x % a.kv_heads, place = blockIdx.x / a.kv_heads;
    /* workgroups of one key/value head are eight apart where they can be, on one die's cache */
    uint32_t first, columns, row0 = 0;       /* this wavefront's first column, of how many from row row0 on */
    int start = 0;                           /* of the column's sequence */
    bool owned = true;
    /* some column of the workgroup sees keys from .. to, of the wavefront lowest .. highest, and all of
     * the wavefront see latest .. earliest */
    int from = INT32_MAX, to = -1, lowest = INT32_MAX, highest = -1, latest = 0, earliest = INT32_MAX;
    if (a.count <= 64) {
        /* A lane to a sequence.  Tiles that see most first: tile d of any sequence, as many as it
         * has, before tile d - 1 of any; behind(d) tiles are d or later of theirs. */
        const uint32_t i = min(lane, a.count - 1);
        const int begin = min(max(a.row_starts[i], 0), (int)a.rows), end = min(max(a.row_starts[i + 1], begin), (int)a.rows);
        const uint32_t mine = lane < a.count ? layer_up((uint32_t)(end - begin) * group, Tile::kColumns) : 0;
        const auto behind = [&](uint32_t d) { return wave_sum_u32(mine > d ? mine - d : 0); };
        uint32_t low_d = 0, high_d = wave_max_u32(mine), following = 0;
        if (place >= behind(0)) return;
        if (a.count == 1) low_d = high_d - 1 - place, following = place;
        else while (high_d - low_d > 1) {
            const uint32_t d = (low_d + high_d) / 2, n = behind(d);
            if (n > place) low_d = d;
            else high_d = d, following = n;
        }
        uint64_t others = __ballot(mine > low_d);
        for (uint32_t n = place - following; n; --n) others &= others - 1;
        const uint32_t sequence = __builtin_ctzll(others);
        row0 = __builtin_amdgcn_readlane(begin, sequence);
        columns = (__builtin_amdgcn_readlane(end, sequence) - row0) * group;
        first = low_d * Tile::kColumns + wave / kShares * 32;
        start = from = latest = row0;
        to = row0 + (min((low_d + 1) * Tile::kColumns, columns) - 1) / group;
        if (first < columns) {
            lowest = row0;
            highest = row0 + min(first + 31, columns - 1) / group;
            earliest = row0 + first / group;
        }
    } else {
        columns = a.rows * group;
        first = (gridDim.x / a.kv_heads - 1 - place) * Tile::kColumns + wave / kShares * 32;
    }
    struct Column {
        uint32_t row, head;
    };
    const auto column = [&](uint32_t i) {                    /* the wavefront's i-th */
        const uint32_t at = min(first + i, columns - 1);
        return Column{row0 + at / group, kv * group + at % group};
    };
    const auto [row, head] = column(low);
    if (a.count > 64) {
        const int row_first = (int)(min(first, columns - 1) / group), row_last = (int)(min(first + 31, columns - 1) / group);
        int owner = -1;
        uint32_t at = 0, end = a.count + 1;                  /* the last sequence at or before the first row */
        while (at < end) {
            const uint32_t mid = (at + end) / 2;
            if (a.row_starts[mid] <= row_first) at = mid + 1;
            else end = mid;
        }
        at = at ? at - 1 : 0;
        for (bool more = true; more && at <= a.count; at += 64) {
            const int begins = at + lane <= a.count ? a.row_starts[at + lane] : INT32_MAX;
            for (uint32_t i = 0; i < 64; ++i) {
                const int begin = __builtin_amdgcn_readlane(begins, i);
                if (begin > row_last) {
                    more = false;
                    break;
                }
                if (begin <= (int)row) start = begin, owner = (int)(at + i);
            }
        }
        start = min(max(start, 0), (int)row);
        owned = owner >= 0 && owner < (int)a.count && first + low < columns;
        lowest = wave_min(owned ? start : INT32_MAX);
        highest = -wave_min(owned ? -(int)row : 1);
        latest = -wave_min(owned ? -start : 0);
        earliest = wave_min(owned ? (int)row : INT32_MAX);
        if (lane == 0) ranges[wave][0] = lowest, ranges[wave][1] = highest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) from = min(from, ranges[w][0]), to = max(to, ranges[w][1]);
        from = __builtin_amdgcn_readfirstlane(from);
        to = __builtin_amdgcn_readfirstlane(to);
        if (to < 0) return;
    } else {
        owned = first + low < columns;
    }

    /* queries, 16 bytes of each 32, in registers throughout; a negative scale turns their sign */
    constexpr int E = 16 / (int)sizeof(T);
    u32x4 query[kOwnSteps];
    const uint64_t query_at = (uint64_t)row * a.query_row + (uint64_t)head * a.query_head;
    const float scale = fabsf(a.scale);
#pragma unroll
    for (int u = 0; u < kOwnSteps; ++u) {
        const T *p = static_cast<const T *>(a.query) + query_at + share * kOwn + (2 * u + half) * E;
        query[u] = load_piece<kWhole>(p);
        if (a.scale < 0) query[u] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    }

    const T *keys = static_cast<const T *>(a.key) + kv * D, *values = static_cast<const T *>(a.value) + kv * D;
    const uint32_t tiles_at = lds_address(tiles) + part * (4 * kHalf);
    /* The keys or values of rows `key` on into a buffer; behind the last that any column
     * sees, that one again (what lies behind the sequences may be anything).  A copy is 1 KiB:
     * kCopyRows rows, the lane's is lane_row of them. */
    constexpr int kCopyRows = 1024 / kRowBytes, kCopies = kHalf / 1024 / kWaves;
    static_assert(kCopyRows * kRowBytes == 1024 && kCopies * kWaves * 1024 == kHalf, "whole copies of each wavefront");
    const uint32_t lane_row = lane * 16 / kRowBytes, lane_piece = lane * 16 % kRowBytes / 16, wave_row = wave * kCopyRows;
    const uint32_t key_lane = lane_piece ^ key_turn<kRowBytes>(wave_row + lane_row);
    const uint32_t value_lane = lane_piece ^ value_turn<T, kRowBytes>(wave_row + lane_row);
    const auto load = [&](bool value, int key, uint32_t buffer) {
        const uint64_t stride = value ? a.value_row : a.key_row;
        const uint32_t where = tiles_at + (value ? 2 * kHalf : 0) + buffer * kHalf + wave * 1024;
        /* piece of the lane in copy i, whose rows are lane_row + wave_row + i * kWaves * kCopyRows (no common bits) */
        const auto piece = [&](int i) {
            const uint32_t r = i * kWaves * kCopyRows;
            return value ? value_lane ^ value_turn<T, kRowBytes>(r) : key_lane ^ key_turn<kRowBytes>(r);
        };
        if (kWhole && key + kKeys - 1 <= to) {
            const T *base = (value ? values : keys) + (uint64_t)(key + wave_row) * stride;
            const uint32_t lane_at = lane_row * (uint32_t)(stride * sizeof(T));
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                copy_to_lds(base, lane_at + piece(i) * 16, where + i * kWaves * 1024);
                base += kWaves * kCopyRows * stride;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int r = key + (int)(i * kWaves * kCopyRows + wave_row + lane_row);
            const T *p = (value ? values : keys) + (uint64_t)min(r, to) * stride + piece(i) * E;
            if constexpr (kWhole) {
                copy_to_lds(p, where + i * kWaves * 1024);
            } else {
                T e[E];
#pragma unroll
                for (int j = 0; j < E; ++j) e[j] = p[j];
                *(Q38_LDS u32x4 *)(uintptr_t)(where + i * kWaves * 1024 + lane * 16) = __builtin_bit_cast(u32x4, e);
            }
        }
    };

    f32x16 out[kOwn / 32] = {};
    float top = -INFINITY, base = 0.0f, total = 0.0f;
    /* Weights of fp16 rows are relative to 2^(top - 7), so at most 2^15, and the largest of each tile is at least 2^-5:
     * top follows the tiles' maxima down too (as far as `least`, 2^40 below the highest that it was), so that the
     * small weights beside a far larger one, thousands of which count, keep their 11 bits.  Within a tile those below
     * 2^-14 are in steps of 2^-24.  32 heads of 128, 8192 tokens: 550 us, 545 with weights relative to 2^top alone;
     * with kFall = 8, which scores of ordinary spread meet, 556. */
    constexpr bool kNarrow = std::is_same_v<T, _Float16>;
    constexpr float kBelow = kNarrow ? 7.0f : 0.0f, kFall = 12.0f;
    float least = -INFINITY;

    /* piece 2 u + half of key row 32 t + low; `lane_at` holds what is the lane's of its place */
    const uint32_t key_lane_at = low * kRowBytes + (half ^ key_turn<kRowBytes>(low)) * 16;
    const auto key_piece = [](uint32_t lane_at, int t, int u) {
        return lds_read<u32x4>((lane_at ^ u % 8 * 32) + t * 32 * kRowBytes + u / 8 * 256);
    };
    /* Keys 16 s on of 32 channels from 32 d on, as O^T's product takes them, 16-bit.  A transposed
     * read: 16 lanes name four rows of 16 neighbours, four lanes a row, and get a column of four
     * each.  A lane of fp32 reads one value of row 4 half and rows from there. */
    const uint32_t i16 = lane & 15, value_row = half * 4 + (sizeof(T) == 2 ? i16 / 4 : 0);
    const uint32_t value_lane_at =
        value_row * kRowBytes +
        (sizeof(T) == 2 ? (i16 & 1) * 8 + (((lane >> 4 & 1) * 2 + (i16 & 3) / 2) ^ value_turn<T, kRowBytes>(value_row)) * 16 : low * 4);
    const auto value_piece = [](uint32_t lane_at, int s, int d) {
        s16x4 part[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t turned = lane_at ^ (d % 4 * 4 ^ value_turn<T, kRowBytes>(b * 8)) * 16;
            part[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Q38_LDS s16x4 *)(uintptr_t)(turned + (s * 16 + b * 8) * kRowBytes + d / 4 * 256));
        }
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
    };

    const uint32_t span = row - start;
    /* one tile of each part at a time; where a part has none left it waits with the others */
    if (from + (int)part * kKeys <= to) {
        load(false, from + part * kKeys, 0);
        load(true, from + part * kKeys, 0);
    }
    uint32_t buffer = 0;
    for (int tile = from; tile <= to; tile += kParts * kKeys, buffer ^= 1) {
        const int key = tile + part * kKeys;
        tile_barrier();
        if (key + kParts * kKeys <= to) {
            load(false, key + kParts * kKeys, buffer ^ 1);
            load(true, key + kParts * kKeys, buffer ^ 1);
        }
        const bool sees = key <= highest && key + kKeys > lowest;
        if (kShares == 1 && !sees) continue;
        uint32_t key_at = tiles_at + buffer * kHalf + key_lane_at + share * 256;
        uint32_t value_at = tiles_at + (2 + buffer) * kHalf + value_lane_at + share * (kOwn * (uint32_t)sizeof(T));
        asm volatile("" : "+v"(key_at), "+v"(value_at));     /* turned anew for each tile: places kept would fill registers */
        f32x16 score[kTiles] = {};
        u32x4 ahead[kAhead + 1];                             /* pieces that are asked for before their products */
        if (sees) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) ahead[i] = key_piece(key_at, i % kTiles, i / kTiles);
#pragma unroll
            for (int i = 0; i < kTiles * kOwnSteps; ++i) {
                const int j = i + kAhead;
                if (j < kTiles * kOwnSteps) ahead[j % (kAhead + 1)] = key_piece(key_at, j % kTiles, j / kTiles);
                score[i % kTiles] = multiply<T>(ahead[i % (kAhead + 1)], query[i / kTiles], score[i % kTiles]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (kShares > 1) {
            /* the tile's keys have been read: their place takes the parts of the scores */
            const auto part_of = [&](uint32_t w, int i) { return tiles_at + buffer * kHalf + w * 4096 + i * 1024 + lane * 16; };
            lds_barrier();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(Q38_LDS f32x4 *)(uintptr_t)part_of(wave, i) = f32x4{score[0][4 * i], score[0][4 * i + 1], score[0][4 * i + 2], score[0][4 * i + 3]};
            lds_barrier();
            if (!sees) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f32x4 sum = lds_read<f32x4>(part_of(wave - share, i));
#pragma unroll
                for (int w = 1; w < kShares; ++w) sum += lds_read<f32x4>(part_of(wave - share + w, i));
#pragma unroll
                for (int j = 0; j < 4; ++j) score[0][4 * i + j] = sum[j];
            }
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) ahead[i] = value_piece(value_at, i / (D / 32), i % (D / 32));
        }
        if (key < latest || key + kKeys - 1 > earliest) {
            const uint32_t begin = key + 4 * half - start;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (begin + (t * 32 + r / 4 * 8 + r % 4) > span) score[t][r] = -INFINITY;
        }
        float most = score[0][0];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) most = fmaxf(most, score[t][r]);
        most = halves_max(most) * scale;
        if constexpr (kNarrow) most = fmaxf(most, least);
        if (__any(kNarrow ? (most > top + 8.0f || most < top - kFall) : most > top + 8.0f)) {
            const float before = top;
            top = kNarrow && most < top - kFall ? most : fmaxf(top, most);
            least = fmaxf(least, top - 40.0f);
            /* nothing but -infinity so far: differences would be NaN, weights are 0 */
            base = top == -INFINITY ? 0.0f : top - kBelow;
            const float shrink = __builtin_amdgcn_exp2f(before - kBelow - base);
            total *= shrink;
#pragma unroll
            for (int d = 0; d < kOwn / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) out[d][r] *= shrink;
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                score[t][r] = __builtin_amdgcn_exp2f(fmaf(score[t][r], scale, -base));
                if constexpr (sizeof(T) == 4) total += score[t][r];
            }
        if constexpr (sizeof(T) == 2) {
            /* Weights are rounded to the values' type, which the matrix unit wants: half a step of each, which mostly
             * cancels over the keys.  The total sums them as they are rounded, so that equal values stay what they are. */
            u32x4 weight[kKeys / 16];
            float sums[4] = {total, 0.0f, 0.0f, 0.0f};       /* four chains: one would be waited for */
#pragma unroll
            for (int s = 0; s < kKeys / 16; ++s) {
                T e[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = static_cast<T>(score[s / 2][s % 2 * 8 + j]);
                weight[s] = __builtin_bit_cast(u32x4, e);
#pragma unroll
                for (int j = 0; j < 4; ++j) sums[j] = add_pair<T>(weight[s][j], sums[j]);
            }
            total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < kKeys / 16 * (D / 32); ++i) {
                const int j = i + kAhead, d = i % (D / 32);
                if (j < kKeys / 16 * (D / 32)) ahead[j % (kAhead + 1)] = value_piece(value_at, j / (D / 32), j % (D / 32));
                out[d] = multiply<T>(ahead[i % (kAhead + 1)], weight[i / (D / 32)], out[d]);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int d = 0; d < kOwn / 32; ++d)
                    out[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                        lds_read<float>(value_at + (r / 4 * 8 + r % 4) * kRowBytes + d * 128), score[0][r], out[d], 0, 0, 0);
        }
    }

    if constexpr (kParts > 1) {
        tile_barrier();                                      /* the tiles have been read */
        f32x4 *sums = reinterpret_cast<f32x4 *>(tiles) + (wave * (D / 8)) * 64 + lane;
        float *statistics = reinterpret_cast<float *>(tiles + D / 2 * 256 * kWaves) + wave * 128 + lane;
        if (part) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                sums[i * 64] = f32x4{out[i / 4][i % 4 * 4], out[i / 4][i % 4 * 4 + 1], out[i / 4][i % 4 * 4 + 2], out[i / 4][i % 4 * 4 + 3]};
            statistics[0] = top;
            statistics[64] = total;
        }
        __syncthreads();
        if (part) return;
        const float other = statistics[0], higher = fmaxf(top, other), both = higher == -INFINITY ? 0.0f : higher;
        const float mine = __builtin_amdgcn_exp2f(top - both), theirs = __builtin_amdgcn_exp2f(other - both);
        total = total * mine + statistics[64] * theirs;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const f32x4 v = sums[i * 64];
#pragma unroll
            for (int j = 0; j < 4; ++j) out[i / 4][i % 4 * 4 + j] = out[i / 4][i % 4 * 4 + j] * mine + v[j] * theirs;
        }
    }

    /* A weight of 0 times a value that is not finite is NaN, so such values of rows that a
     * column does not see have got into its sums.  What came out not finite for another reason stays; the rest is done
     * again, row by row, from the rows that it sees: a tile's columns one after another, without the matrix unit (4096
     * tokens, 24 heads of 256: 0.3 ms a column). */
    const float inverse = 1.0f / halves_sum(total);
    float nothing = 0.0f;
#pragma unroll
    for (int d = 0; d < kOwn / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            out[d][r] *= inverse;
            nothing = fmaf(out[d][r], 0.0f, nothing);
        }
    const uint64_t found = __ballot(owned && nothing != 0.0f);
    uint32_t again = (uint32_t)(found | found >> 32);
    if constexpr (kShares > 1) {                             /* in any share's channels */
        if (lane == 0) ranges[wave][0] = (int)again;
        __syncthreads();
        again = 0;
#pragma unroll
        for (int w = 0; w < kShares; ++w) again |= (uint32_t)ranges[wave - share + w][0];
        again = __builtin_amdgcn_readfirstlane(again);
    }
    if (again) {
        /* of the tiles that the wavefront took */
        const int v0 = from + (lowest - from) / kKeys * kKeys, v1 = min(from + (highest - from) / kKeys * kKeys + kKeys - 1, to);
        const Seen seen = look_over<T, D, kWhole>(a, kv, v0, v1, latest, earliest, lane);
        const bool summed = inverse > 0.0f && inverse < INFINITY;
        again &= ~(uint32_t)__ballot((seen.values && summed) || (uint32_t)(seen.key - start) <= span);
    }
    const uint32_t done = (uint32_t)__ballot(owned) & ~again;

    /* A lane has four neighbours of a column at a time.  They go through LDS, where the wavefront's
     * own part has room for kChannels of its columns in fp32, so that what is read of the gate and
     * written is whole rows. */
    constexpr int kRoom = kParts == 1 ? 4 * kHalf / kWaves : D * 128;
    constexpr int kChannels = kRoom / 128 < kOwn ? kRoom / 128 : kOwn, kPieces = kChannels / E, kRows = 64 / kPieces;
    if constexpr (kParts == 1) tile_barrier();               /* the tiles have been read; of two parts each wavefront has read its own sums */
    float *turned = reinterpret_cast<float *>(tiles + wave * kRoom);
    const auto place_of = [](uint32_t r, uint32_t four) { return r * kChannels + (four ^ (r & 15)) * 4; };
    uint32_t own = low;
    asm volatile("" : "+v"(own));                            /* formed again: kept, they would fill registers of the loop */
    const auto [own_row, own_head] = column(own);
    const uint64_t output_at = (uint64_t)own_row * a.output_row + (uint64_t)own_head * D;
    const uint64_t gate_at = (uint64_t)own_row * a.query_row + (uint64_t)own_head * a.query_head;
    T *const output = static_cast<T *>(a.output);
    const T *const gate = static_cast<const T *>(a.gate);
#pragma unroll
    for (int from_channel = 0; from_channel < kOwn; from_channel += kChannels) {
#pragma unroll
        for (int d = 0; d < kChannels / 32; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x16 &v = out[from_channel / 32 + d];
                *reinterpret_cast<f32x4 *>(turned + place_of(low, d * 8 + r * 2 + half)) =
                    f32x4{v[r * 4], v[r * 4 + 1], v[r * 4 + 2], v[r * 4 + 3]};
            }
        const uint32_t piece = lane % kPieces * E, channel = share * kOwn + from_channel + piece;
        constexpr int kBatch = 32 / kRows < 8 ? 32 / kRows : 8;      /* of the gate, asked for together */
#pragma unroll
        for (int i = 0; i < 32; i += kBatch * kRows) {
            T e[kBatch][E];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const uint64_t at = __shfl(gate_at, i + b * kRows + lane / kPieces);
                if (gate) *reinterpret_cast<u32x4 *>(e[b]) = load_piece<kWhole>(gate + at + channel);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const uint32_t r = i + b * kRows + lane / kPieces;
                const uint64_t at = __shfl(output_at, r);
#pragma unroll
                for (int j = 0; j < E; j += 4) {
                    f32x4 four = *reinterpret_cast<const f32x4 *>(turned + place_of(r, (piece + j) / 4));
                    if (gate) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) four[k] *= sigmoid_f32(static_cast<float>(e[b][j + k]));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[b][j + k] = static_cast<T>(four[k]);
                }
                if (done >> r & 1) store_piece<kWhole>(output + at + channel, __builtin_bit_cast(u32x4, e[b]));
            }
        }
    }
    while (again && share == 0) {
        const uint32_t which = first + __builtin_ctz(again);
        again &= again - 1;
        attend_row<T, D, kWhole, true>(a, row0 + which / group, kv * group + which % group, lane);
    }
}

static_assert(PromptTile<float, 256, 1>::kColumns == kPromptColumns && PromptTile<float, 256, 4>::kColumns == kPromptSharedColumns,
              "the plan's columns");

template <typename T, int D>
bool attention(const PromptAttention &a, hipStream_t stream)
{
    /* 16-byte aligned rows, eight of which 32 bits span */
    const auto whole = [](const void *p, uint64_t stride) {
        return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * sizeof(T) % 16 == 0 && stride < 1u << 26;
    };
    const bool wide = whole(a.query, a.query_row) && whole(a.gate, a.query_head) && whole(a.key, a.key_row) &&
                      whole(a.value, a.value_row) && whole(a.output, a.output_row);
    const PromptPlan plan = plan_prompt(a.rows, a.heads, a.kv_heads, D, sizeof(T), a.count);
    const auto go = [&](auto kernel, uint32_t threads) { return launch_kernel(kernel, dim3(plan.workgroups), dim3(threads), stream, a); };
    if (plan.form == kPromptRows) return go(wide ? row_kernel<T, D, true> : row_kernel<T, D, false>, 256);
    if constexpr (D * sizeof(T) == 1024)
        if (plan.form == kPromptShares) return go(wide ? prompt_kernel<T, D, true, 1, 4> : prompt_kernel<T, D, false, 1, 4>, 256);
    if constexpr (D * sizeof(T) < 1024)
        if (plan.form == kPromptParts) return go(wide ? prompt_kernel<T, D, true, 2, 1> : prompt_kernel<T, D, false, 2, 1>, 512);
    return go(wide ? prompt_kernel<T, D, true, 1, 1> : prompt_kernel<T, D, false, 1, 1>, 256);
}

template <typename T>
bool attention(const PromptAttention &a, hipStream_t stream)
{
    return a.head_dim == 64 ? attention<T, 64>(a, stream) : a.head_dim == 128 ? attention<T, 128>(a, stream)
                                                                              : attention<T, 256>(a, stream);
}

}  // namespace

bool launch_prompt_attention(const PromptAttention &a, hipStream_t stream)
{
    return a.type == kLayerF32 ? attention<float>(a, stream) : a.type == kLayerF16 ? attention<_Float16>(a, stream)
                                                                                   : attention<__bf16>(a, stream);
}

}  // namespace q38
