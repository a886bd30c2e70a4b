/* How a paged attention call is cut into work: by sizes that the host knows. */
#pragma once

#include "q38_kv.h"

namespace q38 {

enum class KVVariant { kOneTile, kTwoTiles, kColumns };

/* columns of a sequence, on average over the call */
inline uint64_t kv_columns_each(const KVAttention &a)
{
    return ((uint64_t)a.rows.total_rows * a.group + a.rows.count - 1) / a.rows.count;
}
inline KVVariant kv_variant(const KVAttention &a)
{
    const uint64_t tile = a.type == kElementF32 ? 8 : 16, columns = kv_columns_each(a);
    return columns <= tile ? KVVariant::kOneTile : columns <= 4 * tile ? KVVariant::kTwoTiles : KVVariant::kColumns;
}

}  // namespace q38
