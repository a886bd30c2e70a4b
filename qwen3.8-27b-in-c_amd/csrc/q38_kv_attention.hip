/* Paged 8-bit attention: the plan of a call, and the kernel that joins the
 * pieces of slots that were cut along their tokens. */
#include "q38_kernels.h"
#include "q38_kv_attention.h"

namespace q38 {

namespace {

/* One output of a column's four channels is sum 2^(m_p - top) O_p over its
 * pieces, in an order that the sizes alone decide.  Few (prompt chunks: many
 * columns of two or three pieces): a thread takes all pieces of four channels.
 * Else a workgroup takes one column after another, and its 4 THREADS / D
 * groups of threads take every so-manieth piece, so that all are read at once:
 * 1024 threads where there may be many (one sequence in 64 pieces: 6 us, 10 with
 * 256), else 256 (480 slots of a few pieces: 5 us, 16 with 1024). */
struct Column {
    uint32_t row, head;
    __device__ __forceinline__ Column(const KVAttention &a, const KVRecord &r, uint32_t kv_head, uint32_t c)
    {
        const uint32_t at = kv_divide(r.rem + c, a.group_magic);
        row = r.row + at;
        head = kv_head * a.group + r.rem + c - at * a.group;
    }
};

__global__ __launch_bounds__(256) void kv_join_few_kernel(KVAttention a)
{
    const uint32_t slot = blockIdx.x, head = blockIdx.y, D = a.cache.head_dim, quads = D / 4;
    const uint32_t c = blockIdx.z * (256 / quads) + threadIdx.x / quads, d = threadIdx.x % quads * 4;
    const KVRecord r = kv_records(a)[1 + slot];
    if (slot >= kv_records(a)->pieces || r.pieces < 2 || c >= r.columns) return;
    const float *stats = kv_stats(a, r.first_piece, head) + 2 * c, *partial = kv_partial(a, r.first_piece, head) + c * D + d;
    const uint64_t stats_step = (uint64_t)a.cache.kv_heads * a.columns * 2, step = (uint64_t)a.cache.kv_heads * a.columns * D;
    const Column column(a, r, head, c);
    const kv_float4 gate = kv_gate4(a, column.row, column.head, d);
    /* four pieces at once */
    float top = -INFINITY, total = 0.0f;
    kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t first = 0; first < r.pieces; first += 4) {
        kv_float4 part[4];
        float part_m[4], part_l[4], largest = top;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            part[k] = {0.0f, 0.0f, 0.0f, 0.0f};
            part_m[k] = -INFINITY;
            part_l[k] = 0.0f;
            if (first + k >= r.pieces) continue;
            const uint32_t at = kv_place_step(first + k);
            part[k] = *reinterpret_cast<const kv_float4 *>(partial + at * step);
            part_m[k] = stats[at * stats_step];
            part_l[k] = stats[at * stats_step + 1];
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) largest = fmaxf(largest, part_m[k]);
        auto less = [&](float m) { return m == largest ? 0.0f : m - largest; };    /* (-inf: nothing was seen) */
        total = kv_lower(total, less(top));
        sum *= exp2f(less(top));
        top = largest;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            total += kv_lower(part_l[k], less(part_m[k]));
            sum += part[k] * exp2f(less(part_m[k]));
        }
    }
    kv_finish4(a, column.row, column.head, d, sum, total, gate);
}

template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void kv_join_kernel(KVAttention a)
{
    __shared__ kv_float4 sums[THREADS];
    const uint32_t slot = blockIdx.x, head = blockIdx.y, D = a.cache.head_dim, quads = D / 4;
    const uint32_t groups = THREADS / quads, group = threadIdx.x / quads, d = threadIdx.x % quads * 4, lane = threadIdx.x & 63;
    const KVRecord r = kv_records(a)[1 + slot];
    if (slot >= kv_records(a)->pieces || r.pieces < 2) return;
    const uint64_t stats_step = (uint64_t)a.cache.kv_heads * a.columns * 2, step = (uint64_t)a.cache.kv_heads * a.columns * D;
    for (uint32_t c = blockIdx.z; c < r.columns; c += gridDim.z) {
        const float *stats = kv_stats(a, r.first_piece, head) + 2 * c;
        const float *partial = kv_partial(a, r.first_piece, head) + c * D + d;
        const Column column(a, r, head, c);
        kv_float4 gate = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!group) gate = kv_gate4(a, column.row, column.head, d);
        /* the group's first pieces are on their way while the maxima are looked at */
        constexpr uint32_t kAhead = 4;
        kv_float4 first[kAhead];
        float first_m[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t p = group + k * groups, at = kv_place_step(p);
            first[k] = {0.0f, 0.0f, 0.0f, 0.0f};
            first_m[k] = -INFINITY;
            if (p >= r.pieces) continue;
            first[k] = *reinterpret_cast<const kv_float4 *>(partial + at * step);
            first_m[k] = stats[at * stats_step];
        }
        /* maximum and total, the same in every wavefront */
        auto stat = [&](uint32_t p) { return stats + kv_place_step(p) * stats_step; };
        const float mine_m = lane < r.pieces ? stat(lane)[0] : -INFINITY;
        const float mine_l = lane < r.pieces ? stat(lane)[1] : 0.0f;
        float top = mine_m;
        for (uint32_t p = lane + 64; p < r.pieces; p += 64) top = fmaxf(top, stat(p)[0]);
        for (int by = 1; by < 64; by *= 2) top = fmaxf(top, __shfl_xor(top, by));
        auto lowered = [&](float m, float l) { return m == -INFINITY ? 0.0f : kv_lower(l, m == top ? 0.0f : m - top); };
        float total = lowered(mine_m, mine_l);
        for (uint32_t p = lane + 64; p < r.pieces; p += 64) total += lowered(stat(p)[0], stat(p)[1]);
        for (int by = 1; by < 64; by *= 2) total += __shfl_xor(total, by);
        kv_float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        auto add = [&](float m, kv_float4 o) {
            if (m != -INFINITY) sum += o * exp2f(m == top ? 0.0f : m - top);
        };
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) add(first_m[k], first[k]);
        for (uint32_t p = group + kAhead * groups; p < r.pieces; p += groups)
            add(stat(p)[0], *reinterpret_cast<const kv_float4 *>(partial + kv_place_step(p) * step));
        sums[threadIdx.x] = sum;
        for (uint32_t half = groups / 2; half; half /= 2) {
            __syncthreads();
            if (group < half) sums[threadIdx.x] = sum = sum + sums[threadIdx.x + half * quads];
        }
        if (!group) kv_finish4(a, column.row, column.head, d, sum, total, gate);
        /* the last step's `sums` are read before the next column's are written (256-wide heads:
         * the two groups of that step are two wavefronts) */
        if (c + gridDim.z < r.columns) __syncthreads();
    }
}

}  // namespace

uint64_t plan_kv_attention(KVAttention &a)
{
    const KVShape shape = kv_shape(a);
    const uint32_t tile = a.type == kElementF32 ? 8 : 16, D = a.cache.head_dim, heads = a.cache.kv_heads;
    a.columns = tile * shape.tiles * (shape.columns ? kv_workgroup_waves(D, true) : 1);
    a.slots = (uint32_t)kv_slots(a.rows.total_rows, a.rows.count, a.group, a.columns, 1);
    const uint32_t most = kv_steps(a.cache.table_entries * a.cache.page_tokens);
    a.shift = 0;
    while ((uint64_t)a.slots * kv_slot_units(most, a.shift) >> 31) ++a.shift;
    a.least = a.shift ? 1 : shape.columns ? 8 : 4;
    /* as many workgroups as run at once: by LDS where wavefronts have their own
     * tokens (64 D bytes of keys and of values each), else by registers */
    const uint32_t on_a_unit = !shape.columns ? (D == 64 && shape.tiles > 1 ? 2 : 256 / D) : D == 64 ? 4 - shape.tiles : 1;
    const uint64_t units = (uint64_t)a.slots * kv_slot_units(most, a.shift), wanted = 256 * on_a_unit / heads;
    const uint64_t useful = (units + a.least - 1) / a.least;
    a.workgroups = (uint32_t)(wanted < 1 ? 1 : wanted < useful ? wanted : useful);
    if (a.slots == 1 && kv_slot_units(most, a.shift) <= kv_small(0)) a.workgroups = 1;
    a.workgroups_inverse = 1.0f / (float)a.workgroups;
    a.group_magic = kv_magic(a.group);
    /* a table that holds short sequences only: no slot is ever cut, nothing is joined */
    a.cut = a.workgroups > 1 && kv_slot_units(most, a.shift) > kv_small(0);
    if (!a.cut) return 0;
    return (a.slots + 1) * sizeof(KVRecord) +
           2ull * a.workgroups * heads * a.columns * (D + 2) * sizeof(float);
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
    if (!a.cut) return true;
    if (kv_shape(a).columns) {
        const uint32_t together = 1024 / D;
        return launch_kernel(kv_join_few_kernel, dim3(a.slots, a.cache.kv_heads, (a.columns + together - 1) / together), dim3(256),
                             stream, a);
    }
    /* as many columns at once as a sequence has on average: workgroups without any cost a launch too */
    const uint64_t columns = ((uint64_t)a.rows.total_rows * a.group + a.rows.count - 1) / a.rows.count;
    const dim3 grid(a.slots, a.cache.kv_heads, columns < a.columns ? (uint32_t)columns : a.columns);
    return a.workgroups >= 8 * a.slots ? launch_kernel(kv_join_kernel<1024>, grid, dim3(1024), stream, a)
                                       : launch_kernel(kv_join_kernel<256>, grid, dim3(256), stream, a);
}

}  // namespace q38
