/* Causal attention of packed prompts (q38hip_prompt_attention). */
#include "q38_kernels.h"
#include "q38_layer_device.h"

namespace q38 {

namespace {

/* First row of the sequence that owns `row`, or -1 where none does: the last
 * sequence that starts at or before it, so empty ones are passed over.  Always
 * in 0 .. row, whatever the words hold. */
__device__ __forceinline__ int sequence_start(const PromptAttention &a, uint32_t row)
{
    uint32_t low = 0, high = a.count + 1;       /* row_starts[low - 1] <= row < row_starts[high] */
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (a.row_starts[mid] <= (int)row) low = mid + 1;
        else high = mid;
    }
    if (low == 0 || low == a.count + 1) return -1;
    return min(max(a.row_starts[low - 1], 0), (int)row);
}

__device__ __forceinline__ float wave_sum_f32(float v)
{
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i);
    return v;
}

/* One row of one head by one wavefront, key by key: a lane holds D / 64
 * neighbouring channels.  One pass with a running maximum; only keys that the
 * row sees are read. */
template <typename T, int D>
__device__ __forceinline__ void attend_row(const PromptAttention &a, uint32_t row, uint32_t head, uint32_t lane)
{
    constexpr int E = D / 64;
    const int start = sequence_start(a, row);
    if (start < 0) return;
    const uint32_t kv = head / (a.heads / a.kv_heads), at = lane * E;
    const uint64_t query = (uint64_t)row * a.query_row + (uint64_t)head * a.query_head + at;
    float q[E], out[E] = {}, top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = static_cast<float>(static_cast<const T *>(a.query)[query + e]) * a.scale;
    for (uint32_t j = start; j <= row; ++j) {
        const T *key = static_cast<const T *>(a.key) + (uint64_t)j * a.key_row + kv * D + at;
        const T *value = static_cast<const T *>(a.value) + (uint64_t)j * a.value_row + kv * D + at;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], static_cast<float>(key[e]), s);
        s = wave_sum_f32(s);
        const float higher = fmaxf(top, s);
        /* nothing but -infinity so far: differences would be NaN, weights are 0 */
        const float base = higher == -INFINITY ? 0.0f : higher;
        const float shrink = exp2f(top - base), weight = exp2f(s - base);
        top = higher;
        total = fmaf(total, shrink, weight);
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = fmaf(weight, static_cast<float>(value[e]), out[e] * shrink);
    }
    T *to = static_cast<T *>(a.output) + (uint64_t)row * a.output_row + (uint64_t)head * D + at;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float v = out[e] / total;
        if (a.gate) {
            const float g = static_cast<float>(static_cast<const T *>(a.gate)[query + e]);
            v = v / (1.0f + __expf(-g));
        }
        to[e] = static_cast<T>(v);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) row_kernel(PromptAttention a)
{
    const uint32_t item = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= a.rows * a.heads) return;
    attend_row<T, D>(a, item / a.heads, item % a.heads, threadIdx.x & 63);
}

template <typename T>
bool attention(const PromptAttention &a, hipStream_t stream)
{
    const auto kernel = a.head_dim == 64 ? row_kernel<T, 64> : a.head_dim == 128 ? row_kernel<T, 128> : row_kernel<T, 256>;
    return launch_kernel(kernel, dim3(layer_up(a.rows * a.heads, 4)), dim3(256), stream, a);
}

}  // namespace

bool launch_prompt_attention(const PromptAttention &a, hipStream_t stream)
{
    return a.type == kLayerF32 ? attention<float>(a, stream) : a.type == kLayerF16 ? attention<_Float16>(a, stream)
                                                                                   : attention<__bf16>(a, stream);
}

}  // namespace q38
