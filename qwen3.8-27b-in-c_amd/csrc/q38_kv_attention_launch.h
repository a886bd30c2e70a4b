/* The choice among a head width's attention kernels. */
#pragma once

#include "q38_kernels.h"
#include "q38_kv_attention.h"
#include "q38_kv_plan.h"

namespace q38 {

template <bool E4M3, int D, bool SPLIT>
bool launch_kv_attention_typed(const KVAttention &a, hipStream_t stream)
{
    const dim3 grid(a.slots, a.cache.kv_heads, a.parts), block(256);
    switch (kv_variant(a)) {
    case KVVariant::kOneTile:
        return launch_kernel(kv_attention_kernel<E4M3, D, 1, SPLIT, false>, grid, block, stream, a);
    case KVVariant::kTwoTiles:
        return launch_kernel(kv_attention_kernel<E4M3, D, 2, SPLIT, false>, grid, block, stream, a);
    default:
        return launch_kernel(kv_attention_kernel<E4M3, D, 2, SPLIT, true>, grid, block, stream, a);
    }
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
