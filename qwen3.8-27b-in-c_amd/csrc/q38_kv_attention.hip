/* Paged 8-bit attention: the plan of a call, and the kernel that joins the
 * parts of a token axis that was split over workgroups. */
#include "q38_kernels.h"
#include "q38_kv_attention.h"
#include "q38_kv_plan.h"

namespace q38 {

namespace {

/* One thread per (column, four channels) of a slot: the parts' sums, scaled to
 * the largest of their maxima, in part order. */
__global__ __launch_bounds__(256) void kv_join_kernel(KVAttention a, uint32_t least)
{
    const uint32_t slot = blockIdx.x, head = blockIdx.y, D = a.cache.head_dim;
    KVSlot s;
    if (!kv_slot(a, slot, s)) return;
    const uint32_t parts = kv_parts(a, (s.seen + kKVStep - 1) / kKVStep, least);
    if (parts == 1) return;
    const uint32_t at = blockIdx.z * 256 + threadIdx.x, c = at / (D / 4), d = at % (D / 4) * 4;
    if (c >= s.columns) return;
    const uint64_t first = ((uint64_t)slot * a.cache.kv_heads + head) * a.parts * a.columns + c;
    const float *stats = a.partial + (uint64_t)a.slots * a.cache.kv_heads * a.parts * a.columns * D;
    float top = -INFINITY;
    for (uint32_t p = 0; p < parts; ++p) top = fmaxf(top, stats[2 * (first + (uint64_t)p * a.columns)]);
    float total = 0.0f;
    kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t p = 0; p < parts; ++p) {
        const uint64_t row = first + (uint64_t)p * a.columns;
        const float m = stats[2 * row];
        if (m == -INFINITY) continue;
        const float keep = exp2f(m - top);
        total += kv_lower(stats[2 * row + 1], m - top);
        sum += *reinterpret_cast<const kv_float4 *>(a.partial + row * D + d) * keep;
    }
    const uint32_t column = s.column + c;
    kv_finish4(a, s.first_row + column / a.group, head * a.group + column % a.group, d, sum, total);
}

}  // namespace

uint64_t plan_kv_attention(KVAttention &a)
{
    const KVVariant variant = kv_variant(a);
    const uint32_t tile = a.type == kElementF32 ? 8 : 16;
    a.columns = variant == KVVariant::kOneTile ? tile : variant == KVVariant::kTwoTiles ? 2 * tile : 8 * tile;
    a.slots = (uint32_t)kv_slots(a.rows.total_rows, a.rows.count, a.group, a.columns, 1);
    const uint32_t least = variant == KVVariant::kColumns ? kKVLeastStepsColumns : kKVLeastStepsTokens;
    const uint64_t steps = ((uint64_t)a.cache.table_entries * a.cache.page_tokens + kKVStep - 1) / kKVStep;
    const uint64_t most = (steps + least - 1) / least, target = variant == KVVariant::kColumns ? 512 : 1024;
    const uint64_t wanted = target / ((uint64_t)a.slots * a.cache.kv_heads);
    a.parts = (uint32_t)(wanted < 1 ? 1 : wanted < most ? wanted : most);
    if (a.parts == 1) return 0;
    return (uint64_t)a.slots * a.cache.kv_heads * a.parts * a.columns * (a.cache.head_dim + 2) * sizeof(float);
}

template <int D>
bool launch_kv_attention_width(const KVAttention &a, hipStream_t stream);
extern template bool launch_kv_attention_width<64>(const KVAttention &, hipStream_t);
extern template bool launch_kv_attention_width<128>(const KVAttention &, hipStream_t);
extern template bool launch_kv_attention_width<256>(const KVAttention &, hipStream_t);

bool launch_kv_attention(const KVAttention &a, hipStream_t stream)
{
    const uint32_t D = a.cache.head_dim;
    if (!(D == 64 ? launch_kv_attention_width<64>(a, stream)
                  : D == 128 ? launch_kv_attention_width<128>(a, stream) : launch_kv_attention_width<256>(a, stream)))
        return false;
    if (a.parts == 1) return true;
    const uint32_t least = kv_variant(a) == KVVariant::kColumns ? kKVLeastStepsColumns : kKVLeastStepsTokens;
    const dim3 grid(a.slots, a.cache.kv_heads, (a.columns * (D / 4) + 255) / 256);
    return launch_kernel(kv_join_kernel, grid, dim3(256), stream, a, least);
}

}  // namespace q38
