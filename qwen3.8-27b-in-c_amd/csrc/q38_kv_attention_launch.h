/* The choice among a head width's attention kernels. */
#pragma once

#include "q38_kernels.h"
#include "q38_kv_attention.h"
#include "q38_kv_plan.h"

namespace q38 {

template <bool E4M3, int D, bool SPLIT>
bool launch_kv_attention_typed(const KVAttention &a, hipStream_t stream)
{
    const KVShape shape = kv_shape(a);
    const dim3 grid(a.workgroups, a.cache.kv_heads), block(64 * kv_workgroup_waves(D, shape.columns));
    if (shape.columns)
        return launch_kernel(shape.tiles == 1 ? kv_attention_kernel<E4M3, D, 1, SPLIT, true> : kv_attention_kernel<E4M3, D, kv_most_tiles(D), SPLIT, true>,
                             grid, block, stream, a);
    if constexpr (kv_token_tiles(D) == 3)
        if (shape.tiles == 3) return launch_kernel(kv_attention_kernel<E4M3, D, 3, SPLIT, false>, grid, block, stream, a);
    return launch_kernel(shape.tiles == 1 ? kv_attention_kernel<E4M3, D, 1, SPLIT, false> : kv_attention_kernel<E4M3, D, 2, SPLIT, false>,
                         grid, block, stream, a);
}

template <int D>
bool launch_kv_attention_width(const KVAttention &a, hipStream_t stream)
{
    const bool e4m3 = a.cache.type == Q38_KV_E4M3, split = a.type == kElementF32;
    if (e4m3)
        return split ? launch_kv_attention_typed<true, D, true>(a, stream)
                     : launch_kv_attention_typed<true, D, false>(a, stream);
    return split ? launch_kv_attention_typed<false, D, true>(a, stream)
                 : launch_kv_attention_typed<false, D, false>(a, stream);
}

}  // namespace q38
