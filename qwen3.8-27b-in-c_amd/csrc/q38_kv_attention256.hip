/* Paged 8-bit attention of 256-wide heads. */
#include "q38_kv_attention_launch.h"

namespace q38 {
template bool launch_kv_attention_width<256>(const KVAttention &, hipStream_t);
}
