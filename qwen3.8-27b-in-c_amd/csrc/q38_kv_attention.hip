/* Paged 8-bit attention: the plan of a call, and the kernel that joins the
 * pieces of slots that were cut along their tokens. */
#include "q38_kernels.h"
#include "q38_kv_attention.h"

namespace q38 {

namespace {

/* One output of a column's four channels is sum 2^(m_p - top) O_p over its
 * pieces, in an order that the sizes alone decide.  FEW (prompt chunks: many
 * columns of two or three pieces): a thread takes all pieces of four channels.
 * Else a workgroup takes one column, and its 1024 / D groups of threads take
 * every so-manieth piece. */
template <bool FEW>
__global__ __launch_bounds__(256) void kv_join_kernel(KVAttention a)
{
    __shared__ kv_float4 sums[FEW ? 1 : 256];
    const uint32_t slot = blockIdx.x, head = blockIdx.y, D = a.cache.head_dim, quads = D / 4, groups = 256 / quads;
    const KVRecord r = kv_records(a)[1 + slot];
    if (slot >= kv_records(a)->pieces || r.pieces < 2) return;
    const uint32_t group = threadIdx.x / quads, d = threadIdx.x % quads * 4;
    const uint32_t c = FEW ? blockIdx.z * groups + group : blockIdx.z;
    if (c >= r.columns) return;
    const float *stats = kv_stats(a, r.first_piece, head) + 2 * c, *partial = kv_partial(a, r.first_piece, head) + c * D + d;
    const uint64_t stats_step = (uint64_t)a.cache.kv_heads * a.columns * 2, step = (uint64_t)a.cache.kv_heads * a.columns * D;
    float top = -INFINITY, total = 0.0f;
    if (FEW) {
        for (uint32_t p = 0; p < r.pieces; ++p) top = fmaxf(top, stats[p * stats_step]);
        for (uint32_t p = 0; p < r.pieces; ++p) {
            const float m = stats[p * stats_step];
            if (m != -INFINITY) total += kv_lower(stats[p * stats_step + 1], m - top);
        }
    } else {
        /* the same in every wavefront */
        const uint32_t lane = threadIdx.x & 63;
        for (uint32_t p = lane; p < r.pieces; p += 64) top = fmaxf(top, stats[p * stats_step]);
        for (int by = 1; by < 64; by *= 2) top = fmaxf(top, __shfl_xor(top, by));
        for (uint32_t p = lane; p < r.pieces; p += 64) {
            const float m = stats[p * stats_step];
            if (m != -INFINITY) total += kv_lower(stats[p * stats_step + 1], m - top);
        }
        for (int by = 1; by < 64; by *= 2) total += __shfl_xor(total, by);
    }
    kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t p = FEW ? 0 : group; p < r.pieces; p += FEW ? 1 : groups) {
        const float m = stats[p * stats_step];
        const float keep = m == -INFINITY ? 0.0f : exp2f(m - top);
        sum += *reinterpret_cast<const kv_float4 *>(partial + p * step) * keep;
    }
    if (!FEW) {
        sums[threadIdx.x] = sum;
        __syncthreads();
        if (group) return;
        for (uint32_t k = 1; k < groups; ++k) sum += sums[threadIdx.x + k * quads];
    }
    const uint32_t row = kv_divide(r.rem + c, a.group_magic);
    kv_finish4(a, r.row + row, head * a.group + r.rem + c - row * a.group, d, sum, total);
}

}  // namespace

uint64_t plan_kv_attention(KVAttention &a)
{
    const KVShape shape = kv_shape(a);
    const uint32_t tile = a.type == kElementF32 ? 8 : 16, D = a.cache.head_dim, heads = a.cache.kv_heads;
    a.columns = tile * shape.tiles * (shape.columns ? 4 : 1);
    a.slots = (uint32_t)kv_slots(a.rows.total_rows, a.rows.count, a.group, a.columns, 1);
    const uint32_t most = kv_steps(a.cache.table_entries * a.cache.page_tokens);
    a.shift = 0;
    while ((uint64_t)a.slots * kv_slot_units(most, a.shift) >> 31) ++a.shift;
    a.least = a.shift ? 1 : shape.columns ? 8 : 4;
    /* as many workgroups as run at once: by LDS where wavefronts have their own
     * tokens (64 D bytes of keys and of values each), else by registers */
    const uint32_t on_a_unit = !shape.columns ? (D == 64 && shape.tiles == 2 ? 2 : 256 / D) : kv_waves(D, shape.tiles, true);
    const uint64_t units = (uint64_t)a.slots * kv_slot_units(most, a.shift), wanted = 256 * on_a_unit / heads;
    const uint64_t useful = (units + a.least - 1) / a.least;
    a.workgroups = (uint32_t)(wanted < 1 ? 1 : wanted < useful ? wanted : useful);
    a.workgroups_inverse = 1.0f / (float)a.workgroups;
    a.group_magic = kv_magic(a.group);
    if (a.workgroups == 1) return 0;
    return (a.slots + 1) * sizeof(KVRecord) +
           ((uint64_t)a.workgroups + a.slots) * heads * a.columns * (D + 2) * sizeof(float);
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
    if (a.workgroups == 1) return true;
    const bool few = kv_shape(a).columns;
    const uint32_t together = few ? 1024 / D : 1;
    return launch_kernel(few ? kv_join_kernel<true> : kv_join_kernel<false>,
                         dim3(a.slots, a.cache.kv_heads, (a.columns + together - 1) / together), dim3(256), stream, a);
}

}  // namespace q38
