/* Paged 8-bit attention of 64-wide heads. */
#include "q38_kv_attention_launch.h"

namespace q38 {
template bool launch_kv_attention_width<64>(const KVAttention &, hipStream_t);
}
