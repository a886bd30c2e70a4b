/* C ABI of the paged 8-bit key/value cache (declared in include/q38hip.h):
 * checks of what the host can see, then the launch. */
#include "q38_kernels.h"
#include "q38_kv.h"

namespace {

using q38::abi_fail;

constexpr uint32_t kMaxExtend = 1024;
constexpr uint32_t kMaxFork = 65536;      /* every pair looks at all children */
constexpr uint32_t kMaxGridYZ = 65535;

bool power_of_two_in(uint32_t v, uint32_t low, uint32_t high) { return v >= low && v <= high && (v & (v - 1)) == 0; }

/* null where the cache is well formed, else what is wrong */
const char *cache_fault(const Q38KVPages *c)
{
    if (!c || !c->data || !c->scales || !c->refs || !c->tables || !c->lengths || !c->status) return "bad cache arguments";
    if (!c->layers || !c->pages || !c->kv_heads || !c->sequences || !c->table_entries) return "empty cache";
    if (!power_of_two_in(c->page_tokens, 16, 128)) return "page_tokens must be 16, 32, 64 or 128";
    if (!power_of_two_in(c->head_dim, 64, 256)) return "head_dim must be 64, 128 or 256";
    if (c->type != Q38_KV_INT8 && c->type != Q38_KV_E4M3) return "unknown cache type";
    if (c->layers > kMaxGridYZ || c->kv_heads > kMaxGridYZ / 2) return "too many layers or heads";
    if (c->pages > 0x7fffffffu - (1u << 14) || c->sequences > 0x7fffffffu ||
        (uint64_t)c->table_entries * c->page_tokens > 0x7fffffffull ||
        !q38::kv_launch_holds(((uint64_t)c->sequences * c->table_entries + 255) / 256, 256))
        return "cache of more than 2^31 pages, sequences or tokens, or 2^32 - 256 table entries";
    /* launches of a workgroup per 8 KiB of a page stay below 2^32 threads */
    if (q38::kv_page_bytes(*c) * c->layers > 1ull << 36) return "a page of more than 2^36 bytes in all layers";
    if (reinterpret_cast<uintptr_t>(c->data) & 15) return "cache data must be 16-byte aligned";
    return nullptr;
}

bool element_type(uint32_t type)
{
    return type == (uint32_t)q38::kElementF32 || type == (uint32_t)q38::kElementF16 || type == (uint32_t)q38::kElementBF16;
}

const char *rows_fault(const int32_t *sequences, const int32_t *row_starts, uint32_t count, uint32_t total_rows)
{
    if (!sequences || !count || !total_rows) return "bad row arguments";
    if (count > (1u << 24) || total_rows > (1u << 24)) return "more than 2^24 rows or sequences";
    if (!row_starts && total_rows % count) return "total_rows must be a multiple of count without row_starts";
    return nullptr;
}

q38::KVRows rows_of(const int32_t *sequences, const int32_t *row_starts, uint32_t count, uint32_t total_rows)
{
    return {sequences, row_starts, count, total_rows, total_rows / count};
}

/* the plan of an attention call: what is wrong, or null and the call and its workspace */
const char *plan_attention(const Q38KVPages *cache, uint32_t type, uint32_t heads, uint32_t count, uint32_t total_rows,
                           q38::KVAttention &a, uint64_t &bytes)
{
    if (const char *fault = cache_fault(cache)) return fault;
    if (!element_type(type)) return "rows must be F32, F16 or BF16";
    if (!heads || heads % cache->kv_heads) return "heads must be a multiple of kv_heads";
    if (!count || !total_rows || count > (1u << 24) || total_rows > (1u << 24)) return "bad row arguments";
    if ((uint64_t)total_rows * heads > 0x7fffffffull) return "more than 2^31 query rows";
    a = {};
    a.cache = *cache;
    a.rows = {nullptr, nullptr, count, total_rows, total_rows / count};
    a.type = (int)type;
    a.group = heads / cache->kv_heads;
    if (a.group > 32768) return "more than 32768 query heads to a key/value head";
    bytes = q38::plan_kv_attention(a);
    /* the join of slots that may be cut: 256 threads for each (1024 where they are few) */
    if (a.cut && !q38::kv_launch_holds(a.slots, 256)) return "more rows or sequences than a launch of attention's join holds";
    return nullptr;
}

}  // namespace

extern "C" int q38hip_kv_reset(const Q38KVPages *cache, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    return q38::launch_kv_reset(*cache, static_cast<hipStream_t>(stream)) ? 1 : abi_fail("cache reset kernel failed");
}

extern "C" uint64_t q38hip_kv_workspace_bytes(const Q38KVPages *cache)
{
    if (const char *fault = cache_fault(cache)) {
        abi_fail(fault);
        return 0;
    }
    return q38::kv_workspace_bytes(*cache);
}

extern "C" int q38hip_kv_extend(const Q38KVPages *cache, const int32_t *sequences, const int32_t *rows, uint32_t count,
                                void *workspace, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (!sequences || !rows || !workspace || !count) return abi_fail("bad extend arguments");
    if (count > kMaxExtend) return abi_fail("more than 1024 sequences in one extension");
    return q38::launch_kv_extend(*cache, sequences, rows, count, static_cast<int32_t *>(workspace),
                                 static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache extension kernels failed");
}

extern "C" int q38hip_kv_fork(const Q38KVPages *cache, const int32_t *parents, const int32_t *children,
                              const int32_t *lengths, uint32_t count, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (!parents || !children || !count) return abi_fail("bad fork arguments");
    if (count > kMaxFork) return abi_fail("more than 65536 sequences in one fork");
    return q38::launch_kv_fork(*cache, parents, children, lengths, count, static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache fork kernel failed");
}

extern "C" int q38hip_kv_truncate(const Q38KVPages *cache, const int32_t *sequences, const int32_t *lengths,
                                  uint32_t count, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (!sequences || !lengths || !count) return abi_fail("bad truncate arguments");
    if (!q38::kv_launch_holds(count, 256)) return abi_fail("more than 2^24 - 1 sequences in one truncation");
    return q38::launch_kv_truncate(*cache, sequences, lengths, count, static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache truncate kernel failed");
}

extern "C" int q38hip_kv_compact(const Q38KVPages *cache, void *workspace, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (!workspace) return abi_fail("bad compact arguments");
    return q38::launch_kv_compact(*cache, static_cast<int32_t *>(workspace), static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache compaction kernels failed");
}

extern "C" int q38hip_kv_copy(const Q38KVPages *cache, const int32_t *sources, const int32_t *targets, uint32_t count,
                              void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (!sources || !targets || !count || count > kMaxGridYZ) return abi_fail("bad copy arguments");
    return q38::launch_kv_copy(*cache, sources, targets, count, static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache copy kernel failed");
}

extern "C" int q38hip_kv_append(const Q38KVPages *cache, uint32_t layer, const void *key, const void *value,
                                uint32_t type, uint64_t row_stride, const int32_t *sequences, const int32_t *row_starts,
                                uint32_t count, uint32_t total_rows, void *stream)
{
    if (const char *fault = cache_fault(cache)) return abi_fail(fault);
    if (const char *fault = rows_fault(sequences, row_starts, count, total_rows)) return abi_fail(fault);
    if (!key || !value) return abi_fail("bad append arguments");
    if (!element_type(type)) return abi_fail("rows must be F32, F16 or BF16");
    if (layer >= cache->layers) return abi_fail("layer beyond the cache");
    if (total_rows > 1 && row_stride < (uint64_t)cache->kv_heads * cache->head_dim) return abi_fail("row stride too small");
    if (!q38::kv_launch_holds(q38::kv_slots(total_rows, count, 1, cache->page_tokens, 2), q38::kv_append_threads(*cache)))
        return abi_fail("more rows or sequences than a launch of append holds");
    return q38::launch_kv_append(*cache, layer, key, value, (int)type, row_stride,
                                 rows_of(sequences, row_starts, count, total_rows), static_cast<hipStream_t>(stream))
               ? 1
               : abi_fail("cache append kernel failed");
}

extern "C" uint64_t q38hip_kv_attention_workspace_bytes(const Q38KVPages *cache, uint32_t type, uint32_t heads,
                                                        uint32_t count, uint32_t total_rows)
{
    q38::KVAttention a;
    uint64_t bytes;
    if (const char *fault = plan_attention(cache, type, heads, count, total_rows, a, bytes)) {
        abi_fail(fault);
        return 0;
    }
    return bytes;
}

extern "C" int q38hip_kv_attention(const Q38KVPages *cache, uint32_t layer, void *output, const void *query,
                                   const void *gate, uint32_t type, uint32_t heads, uint64_t query_row_stride,
                                   uint64_t query_head_stride, uint64_t output_row_stride, float scale,
                                   const int32_t *sequences, const int32_t *row_starts, uint32_t count,
                                   uint32_t total_rows, void *workspace, void *stream)
{
    q38::KVAttention a;
    uint64_t bytes;
    if (const char *fault = plan_attention(cache, type, heads, count, total_rows, a, bytes)) return abi_fail(fault);
    if (const char *fault = rows_fault(sequences, row_starts, count, total_rows)) return abi_fail(fault);
    if (!output || !query) return abi_fail("bad attention arguments");
    if (layer >= cache->layers) return abi_fail("layer beyond the cache");
    if (heads > 1 && query_head_stride < cache->head_dim) return abi_fail("query head stride too small");
    if (total_rows > 1 && output_row_stride < (uint64_t)heads * cache->head_dim)
        return abi_fail("output row stride too small");
    if (bytes && !workspace) return abi_fail("this attention call needs a workspace");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return abi_fail("workspace must be 16-byte aligned");
    a.rows = rows_of(sequences, row_starts, count, total_rows);
    a.cache.data += (uint64_t)layer * cache->pages * q38::kv_page_bytes(*cache);
    a.cache.scales += (uint64_t)layer * cache->pages * 2 * cache->kv_heads;
    a.query = query;
    a.gate = gate;
    a.output = output;
    a.partial = static_cast<float *>(workspace);
    a.query_row = query_row_stride;
    a.query_head = query_head_stride;
    a.output_row = output_row_stride;
    a.page_shift = (uint32_t)__builtin_ctz(cache->page_tokens);
    a.scale = scale * 1.44269504088896340736f;
    return q38::launch_kv_attention(a, static_cast<hipStream_t>(stream)) ? 1
                                                                         : abi_fail("paged attention kernels failed");
}
