/* Operators of a decoder layer (section 4 of include/q38hip.h): what their
 * kernels, launchers and checks share. */
#pragma once

#include <stdint.h>

#include "q38hip.h"

/* what is plain C++ here is checked on the CPU too */
#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define Q38_LAYER_HD __host__ __device__ __forceinline__
#else
#define Q38_LAYER_HD inline
#endif

namespace q38 {

/* GGML type ids of elements */
constexpr int kLayerF32 = 0, kLayerF16 = 1, kLayerBF16 = 30;

/* elements that share a scale */
constexpr uint32_t kE4M3Block = 128;

Q38_LAYER_HD constexpr uint32_t layer_up(uint32_t a, uint32_t b) { return (a + b - 1) / b; }

/* a launch has fewer than 2^32 threads along a direction of its grid */
inline bool layer_launch_holds(uint64_t workgroups, uint32_t threads) { return workgroups * threads <= 0xffffffffull; }

/* workgroups of 256 threads to a row that goes into 8 bits, eight elements a thread */
inline uint32_t quantize_parts(uint64_t width) { return (uint32_t)((width + 2047) / 2048); }
/* threads to a row that is normalised */
inline uint32_t norm_threads(uint64_t width) { return width > 8192 ? 1024 : 256; }

inline uint32_t e4m3_blocks(uint64_t width) { return (uint32_t)((width + kE4M3Block - 1) / kE4M3Block); }
inline uint32_t e4m3_pitch(uint64_t width) { return (e4m3_blocks(width) + 3) / 4 * 4; }

struct QuantizeRows {
    uint8_t *codes, *scales;
    const void *x, *gate;
    uint64_t x_row, gate_row;
    uint32_t width, pitch, rows;
};

struct NormRows {
    void *output, *total;
    uint8_t *codes, *scales;
    const void *x, *addend, *weight;
    uint64_t output_row, total_row, x_row, addend_row;
    uint32_t width, pitch, rows;
    int weight_type;
    float offset, eps;
};

struct Rotary {
    void *output;
    const void *x;
    uint64_t output_row, output_head, x_row, x_head;
    uint32_t rows, heads, head_dim, pairs;
    const int32_t *positions;
    const float *frequencies;
    float magnitude;
    bool interleaved;
};

struct ProductE4M3 {
    void *output;
    uint64_t output_row;
    const uint8_t *codes, *scales, *weight;
    const float *weight_scales;
    float *partial;
    uint32_t tokens, inputs, outputs, blocks, pitch;
    int type;
};

/* How a product is cut: tiles of so many matrix rows by tokens; `whole` of them have
 * a workgroup each, the inputs of the others are cut into `splits` parts whose sums a
 * second launch joins, from a workspace of `bytes`. */
enum { kProductFew = 0, kProductTile16, kProductTile64, kProductTile128, kProductTile256 };
constexpr uint32_t kProductRows[] = {16, 128, 128, 128, 256}, kProductTokens[] = {16, 16, 64, 128, 256};
struct ProductPlan {
    uint32_t tile, whole, splits;
    uint64_t bytes;
};
inline ProductPlan plan_product(uint32_t tokens, uint32_t inputs, uint32_t outputs)
{
    /* A second launch costs 4 us, which small matrices do not repay: few tokens by 16 rows a
     * workgroup, its wavefronts each a part of the inputs, against tiles, in us: 1 token, 5120 x 5120
     * 8.3 against 11.4, 17408 x 5120 22 against 18; 4 tokens, 5120 x 5120 9.8 against 11.3, 5120 x 14336
     * 16.7 against 14.7; 16 tokens, 5120 x 1024 7.6 against 11.6; 8 tokens, 5120 x 14336 18 against 15. */
    const uint64_t codes = (uint64_t)inputs * outputs;
    if ((tokens <= 4 && codes <= 1u << 25) || (tokens <= 16 && codes <= 1u << 23))
        return {kProductFew, 0, 1, 0};
    /* One workgroup of tiles to a compute unit.  Of the tiles that do not fill a round, each is cut
     * into as many parts as there are units, of four blocks of inputs or more. */
    constexpr uint32_t kUnits = 256;
    const uint32_t blocks = e4m3_blocks(inputs);
    const auto cut = [&](uint32_t tile) {
        const uint64_t tiles = (uint64_t)layer_up(outputs, kProductRows[tile]) * layer_up(tokens, kProductTokens[tile]), rest = tiles % kUnits;
        uint64_t splits = rest ? kUnits / rest : 1;
        if (splits > blocks / 4) splits = blocks / 4;
        if (splits < 2) return ProductPlan{tile, (uint32_t)tiles, 1, 0};
        return ProductPlan{tile, (uint32_t)(tiles - rest), (uint32_t)splits, rest * splits * kProductRows[tile] * kProductTokens[tile] * 4};
    };
    if (tokens <= 16) return cut(kProductTile16);
    /* Larger tiles move fewer bytes for a product but cut the work into larger pieces: the least of what
     * they take is taken.  A block of inputs takes 0.5, 0.82, 2.05 us (its products), or 0.84, 0.84, 1.68
     * where the matrix comes from memory for one tile of tokens; the second launch takes 6 us, the parts' sums
     * 1 us for 4 MB.  In us by tiles of 64, 128, 256 tokens: 80 x 5120 x 34816 59, 48, 69; 512 x 17408 x
     * 5120 100, 100, 69; 768 x 5120 x 14336 119, 91, 74; 1024 x 2048 x 2048 11, 25, 26; 512 x 5120 x 5120
     * 33, 31, 35; 2048 x 5120 x 5120 104, 83, 70. */
    ProductPlan best = {};
    float least = 0.0f;
    for (uint32_t tile = kProductTile64; tile <= kProductTile256; ++tile) {
        const ProductPlan plan = cut(tile);
        const float products = tile == kProductTile64 ? 0.5f : tile == kProductTile128 ? 0.82f : 2.05f;
        const float memory = kProductRows[tile] * (0.84f / 128) / layer_up(tokens, kProductTokens[tile]);
        const uint32_t rounds = plan.whole / kUnits + (plan.splits == 1 && plan.whole % kUnits ? 1 : 0);
        float us = (products > memory ? products : memory) * (rounds * blocks + (plan.splits > 1 ? layer_up(blocks, plan.splits) : 0));
        if (plan.splits > 1) us += 6.0f + plan.bytes * 2.5e-7f;
        if (tile == kProductTile64 || us < least) best = plan, least = us;
    }
    return best;
}

/* tile `place` of a product of tiles_n by tiles_m tiles: bands of four tiles of tokens,
 * along the rows */
struct TilePlace {
    uint32_t n, m;
};
Q38_LAYER_HD TilePlace tile_place(uint32_t place, uint32_t tiles_n, uint32_t tiles_m)
{
    constexpr uint32_t kHigh = 4;
    const uint32_t band = place / (kHigh * tiles_n), left = tiles_m - band * kHigh, high = left < kHigh ? left : kHigh;
    place -= band * kHigh * tiles_n;
    return {place / high, band * kHigh + place % high};
}
/* item `index` of `all` that workgroups take in turn: each of the eight dies, which workgroups go
 * round, gets a run of neighbouring items, so that its cache serves what they share */
Q38_LAYER_HD uint32_t die_place(uint32_t index, uint32_t all)
{
    constexpr uint32_t kDies = 8;
    const uint32_t die = index % kDies, share = all / kDies, more = all % kDies;
    return die * share + (die < more ? die : more) + index / kDies;
}

struct PromptAttention {
    void *output;
    const void *query, *gate, *key, *value;
    uint64_t output_row, query_row, query_head, key_row, value_row;
    const int32_t *row_starts;
    uint32_t count, rows, heads, kv_heads, head_dim;
    float scale;           /* softmax scale times log2(e) */
    int type;
};

/* How packed prompts are attended to: a wavefront to a row and head, or tiles of columns (a row and one
 * of the heads that share keys and values), with the keys in two parts or the columns shared by four
 * wavefronts. */
enum { kPromptRows = 0, kPromptTiles, kPromptParts, kPromptShares };
constexpr uint32_t kPromptColumns = 128, kPromptSharedColumns = 32;
struct PromptPlan {
    int form;
    uint32_t workgroups;
};
inline PromptPlan plan_prompt(uint32_t rows, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t element, uint32_t count)
{
    /* Few rows have few keys.  A wavefront to a row and head, against tiles, in us: 24 heads of 256
     * on 4, fp32, 64 rows 9.5 against 11.5, 128 rows 21 against 18; 5 of 256 on 5, fp32, 320 rows 32 against 35;
     * 24 of 256 bf16, 64 rows 8.1 against 11.7, 128 rows 20.7 against 13.7; 32 of 128, bf16, 64 rows 6.1
     * against 7.6, 128 rows 13.8 against 8.8, fp32 128 rows 18 against 24, 200 rows 39 against 35; 16 of 64, fp32,
     * 128 rows 8.4 against 14.7. */
    const bool full = element == 4 && head_dim == 256;
    if (rows <= (element == 4 ? 64 + head_dim : 64) && (element == 2 || rows * heads <= (full ? 2048u : 5120u)))
        return {kPromptRows, layer_up(rows * heads, 4)};
    /* a tile more for each sequence where tiles follow them */
    const uint32_t columns = rows * (heads / kv_heads), more = count <= 64 ? count : 0, spare = more * kv_heads;
    const auto tiles = [&](uint32_t size) { return (layer_up(columns, size) + more) * kv_heads; };
    const uint32_t workgroups = tiles(kPromptColumns);
    /* A tile of 256-wide fp32 heads takes 8.6 us for 32 keys, so where there are fewer tiles than units,
     * columns are shared: 5 heads on 5, 1375 tokens (60 tiles) 140 us against 364, 24 on 4, 1000 (192)
     * 175 against 272, 2048 (384) 637 against 540.  Tiles that run over sequences see few keys each, so what matters is
     * how evenly they fill the units: 24 on 4, 100 prompts, of 15 tokens (284) 42 against 49, 18 (340) 50 against 50,
     * 24 (452) 65 against 58; 5 on 5, of 100 (395) 110 against 134. */
    if (full && workgroups <= (more ? 256 + spare : 400)) return {kPromptShares, tiles(kPromptSharedColumns)};
    /* Tiles that do not fill the card twice over: both halves of the registers go to one of them,
     * unless keys are few.  Two parts against one, in us: bf16, 24 heads of 256, 1024 tokens (192
     * tiles) 38 against 42, 2048 (384) 70 against 86, 3500 (660) 179 against 163, 12 prompts of up to 300
     * (244) 29 against 22; 32 heads of 128, 700 tokens (176) 18.3 against 19.4, 2700 (680) 84 against 69, 12
     * prompts of up to 300 (328) 19 against 13; fp32, 2048 tokens (512) 283 against 365; 66 prompts of 260, 4 heads on 4
     * (540), bf16, 64-wide 24 against 17, 256-wide 63 against 48. */
    if (!full && workgroups <= 512 + spare && rows >= 256ull * count) return {kPromptParts, workgroups};
    return {kPromptTiles, workgroups};
}

#if defined(__HIPCC__)
bool launch_quantize_e4m3(const QuantizeRows &a, int type, hipStream_t stream);
bool launch_rms_norm(const NormRows &a, int type, hipStream_t stream);
bool launch_rotary(const Rotary &a, int type, hipStream_t stream);
uint64_t product_e4m3_workspace_bytes(uint32_t tokens, uint64_t inputs, uint32_t outputs);
bool launch_product_e4m3(const ProductE4M3 &a, hipStream_t stream);
bool launch_prompt_attention(const PromptAttention &a, hipStream_t stream);
#endif

}  // namespace q38
