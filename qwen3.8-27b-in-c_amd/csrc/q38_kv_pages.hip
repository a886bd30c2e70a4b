/* Pages of the 8-bit cache: handing out (with a copy where a shared page is
 * about to be written), forking, cutting back and compacting, all on the
 * device: no call reads a count back.  refs[page] counts the sequences that a
 * page belongs to, 0 is a free page; the lowest free pages are handed out
 * first, so equal calls give equal tables. */
#include "q38_kernels.h"
#include "q38_kv.h"

namespace q38 {

namespace {

constexpr int kPlan = 1024;               /* threads of the one planning workgroup */
constexpr uint32_t kNear = 2048;           /* new pages of an extension that stay in LDS */
constexpr uint32_t kScanEach = 16;        /* pages per thread of one round of its scans */

/* T is a power of two */
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t T) { return (tokens + T - 1) >> (__ffs(T) - 1); }

/* exclusive prefix sum over the workgroup of kPlan threads, and the total;
 * the caller's barrier separates two uses of `sums` */
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *sums, uint32_t &total)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t run = v;
    for (int by = 1; by < 64; by *= 2) {
        const uint32_t up = (uint32_t)__shfl_up((int)run, by);
        if (lane >= (uint32_t)by) run += up;
    }
    if (lane == 63) sums[wave] = run;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < kPlan / 64; ++w) {
        before += w < wave ? sums[w] : 0;
        total += sums[w];
    }
    return before + run - v;
}

/* bit b: page first + b is free (pages past the pool are not) */
__device__ __forceinline__ uint32_t free_bits(const int32_t *refs, uint32_t first, uint32_t pages)
{
    uint32_t bits = 0;
    if (first + kScanEach <= pages && ((uintptr_t)refs & 15) == 0) {
        const int4 *p = reinterpret_cast<const int4 *>(refs + first);
#pragma unroll
        for (uint32_t b = 0; b < kScanEach / 4; ++b) {
            const int4 v = p[b];
            bits |= ((v.x == 0) | (v.y == 0) << 1 | (v.z == 0) << 2 | (v.w == 0) << 3) << (4 * b);
        }
    } else {
        for (uint32_t b = 0; b < kScanEach && first + b < pages; ++b) bits |= (uint32_t)(refs[first + b] == 0) << b;
    }
    return bits;
}

__global__ __launch_bounds__(256) void kv_reset_kernel(Q38KVPages c)
{
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (at < c.pages) c.refs[at] = 0;
    if (at < c.sequences) c.lengths[at] = 0;
    if (at < (uint64_t)c.sequences * c.table_entries) c.tables[at] = -1;
    if (at == 0) *c.status = 0;
}

/* The plan of an extension, by one workgroup: thread i has item i.  Nothing is
 * written unless every item is good and the pool has the pages.  Item i's
 * tail page is copied where other sequences still share it at its turn, that
 * is after the items before it that share it took their copies.  The pages
 * that the copy kernel moves go to pairs[i] and pairs[count + i] (-1: none). */
__global__ __launch_bounds__(kPlan) void kv_extend_kernel(Q38KVPages c, const int32_t *sequences, const int32_t *rows,
                                                          uint32_t count, int32_t *pairs, int32_t *found)
{
    __shared__ uint32_t sums[kPlan / 64];
    __shared__ int32_t ids[kPlan], tails[kPlan];
    __shared__ uint32_t offsets[kPlan + 1], lasts[kPlan];    /* first of the item's pages; table entries behind it */
    __shared__ int32_t near[kNear];                          /* the first pages found */
    __shared__ uint32_t trouble;
    const uint32_t i = threadIdx.x, T = c.page_tokens;
    uint32_t before = 0, after = 0, bad = 0, take = 0;
    int32_t id = -1, tail = -1;
    bool copy = false;
    /* the scan's first round is on its way while the items are looked at */
    const uint32_t first_bits = free_bits(c.refs, i * kScanEach, c.pages);
    if (i == 0) trouble = 0;
    if (i < count) {
        id = sequences[i];
        const int32_t more = rows[i];
        if (id < 0 || (uint32_t)id >= c.sequences || more < 0) {
            bad = Q38_KV_BAD_SEQUENCE;
        } else {
            before = kv_tokens(c, id);
            const uint64_t last = (uint64_t)before + (uint32_t)more;
            if (last > (uint64_t)c.table_entries * T) bad = Q38_KV_TABLE_FULL;
            else after = (uint32_t)last;
            if (!bad && more && (before & (T - 1))) {
                tail = kv_page(c, id, before >> (__ffs(T) - 1));
                if (tail < 0) bad = Q38_KV_BAD_PAGE;
            }
        }
    }
    ids[i] = id;
    tails[i] = tail;
    __syncthreads();
    if (i < count && !bad) {
        uint32_t turn = 0;
        for (uint32_t j = 0; j < i; ++j) {
            if (ids[j] == id) bad = Q38_KV_BAD_SEQUENCE;
            turn += tails[j] == tail;
        }
        copy = tail >= 0 && c.refs[tail] - (int32_t)turn > 1;
        if (after > before) take = pages_of(after, T) - pages_of(before, T) + copy;
    }
    if (bad) atomicOr(&trouble, bad);
    uint32_t total;
    const uint32_t offset = block_prefix(i < count ? take : 0, sums, total);
    offsets[i] = offset;
    lasts[i] = pages_of(after, T);
    if (i == 0) offsets[kPlan] = total;
    if (i < count) {
        pairs[i] = -1;
        pairs[count + i] = -1;
    }
    __syncthreads();
    if (trouble) {
        if (i == 0) atomicOr(c.status, (int32_t)trouble);
        return;
    }
    /* the lowest free pages */
    uint32_t have = 0;
    for (uint32_t first = 0; first < c.pages && have < total; first += kPlan * kScanEach) {
        uint32_t bits = first ? free_bits(c.refs, first + i * kScanEach, c.pages) : first_bits, all;
        uint32_t rank = have + block_prefix(__popc(bits), sums, all);
        for (; bits && rank < total; bits &= bits - 1, ++rank) {
            const int32_t page = (int32_t)(first + i * kScanEach + __ffs(bits) - 1);
            if (rank < kNear) near[rank] = page;
            else found[rank] = page;
        }
        have += all;
        __syncthreads();
    }
    if (have < total) {
        if (i == 0) atomicOr(c.status, Q38_KV_POOL_FULL);
        return;
    }
    __threadfence_block();
    __syncthreads();
    if (i < count && copy) {
        pairs[i] = tail;
        pairs[count + i] = offset < kNear ? near[offset] : found[offset];
        atomicSub(&c.refs[tail], 1);
    }
    for (uint32_t k = i; k < total; k += kPlan) {
        /* the item whose pages k is among: the last with offset <= k and pages of its own */
        uint32_t low = 0, high = kPlan;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (offsets[mid] <= k) low = mid;
            else high = mid;
        }
        const int32_t page = k < kNear ? near[k] : found[k];
        /* entries go up from the tail's where it is copied, else from the first new one */
        const uint32_t own = offsets[low + 1] - offsets[low];
        c.tables[(uint64_t)ids[low] * c.table_entries + (lasts[low] - own + (k - offsets[low]))] = page;
        c.refs[page] = 1;
    }
    __syncthreads();
    if (i < count) c.lengths[id] = (int32_t)after;
}

/* A slice, 32 bytes per thread, of page `source` of a layer to page `target`.
 * (A vector type of the compiler's own: an array of uint4 went through LDS.)
 * STREAM passes the caches by: for a compaction of 1.35 GB 536 us instead of 549,
 * but for 72 pages of 17 layers, which are read again at once, 49 instead of 45. */
using kv_bytes16 = uint32_t __attribute__((ext_vector_type(4)));
constexpr uint32_t kCopySlice = 256 * 16 * 2;
template <bool STREAM>
__device__ __forceinline__ void copy_slice(const Q38KVPages &c, int32_t source, int32_t target, uint32_t layer, uint32_t slice)
{
    const uint64_t bytes = kv_page_bytes(c), pages = (uint64_t)layer * c.pages;
    const kv_bytes16 *from = reinterpret_cast<const kv_bytes16 *>(c.data + (pages + source) * bytes);
    kv_bytes16 *to = reinterpret_cast<kv_bytes16 *>(c.data + (pages + target) * bytes);
    const uint32_t first = slice * (kCopySlice / 16) + threadIdx.x, second = first + 256, end = (uint32_t)(bytes / 16);
    float scale = 0.0f;
    const bool scales = slice == 0 && threadIdx.x < 2 * c.kv_heads;
    if (scales) scale = c.scales[(pages + source) * 2 * c.kv_heads + threadIdx.x];
    if (second < end) {
        const kv_bytes16 v = STREAM ? __builtin_nontemporal_load(from + first) : from[first];
        const kv_bytes16 w = STREAM ? __builtin_nontemporal_load(from + second) : from[second];
        if (STREAM) {
            __builtin_nontemporal_store(v, to + first);
            __builtin_nontemporal_store(w, to + second);
        } else {
            to[first] = v;
            to[second] = w;
        }
    } else if (first < end) {
        to[first] = from[first];
    }
    if (scales) c.scales[(pages + target) * 2 * c.kv_heads + threadIdx.x] = scale;
    if (slice == 0)
        for (uint32_t e = 256 + threadIdx.x; e < 2 * c.kv_heads; e += 256)
            c.scales[(pages + target) * 2 * c.kv_heads + e] = c.scales[(pages + source) * 2 * c.kv_heads + e];
}

__global__ __launch_bounds__(256) void kv_copy_kernel(Q38KVPages c, const int32_t *sources, const int32_t *targets)
{
    const int32_t source = sources[blockIdx.z], target = targets[blockIdx.z];
    if (source < 0 || target < 0) return;
    if ((uint32_t)source >= c.pages || (uint32_t)target >= c.pages) {
        if (threadIdx.x == 0) atomicOr(c.status, Q38_KV_BAD_PAGE);
        return;
    }
    copy_slice<false>(c, source, target, blockIdx.y, blockIdx.x);
}

/* one workgroup per pair: the child, which has to be empty, takes the first
 * tokens of its parent */
__global__ __launch_bounds__(256) void kv_fork_kernel(Q38KVPages c, const int32_t *parents, const int32_t *children,
                                                      const int32_t *lengths, uint32_t count)
{
    __shared__ uint32_t bad, taken;
    const int32_t parent = parents[blockIdx.x], child = children[blockIdx.x];
    if (threadIdx.x == 0)
        bad = parent < 0 || (uint32_t)parent >= c.sequences || child < 0 || (uint32_t)child >= c.sequences;
    __syncthreads();
    /* a sequence that the same call fills is no parent */
    for (uint32_t j = threadIdx.x; j < count; j += 256)
        if (children[j] == parent) bad = 1;
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) atomicOr(c.status, Q38_KV_BAD_SEQUENCE);
        return;
    }
    const uint32_t held = kv_tokens(c, parent);
    const uint32_t tokens = lengths ? (uint32_t)min((int64_t)held, max((int64_t)0, (int64_t)lengths[blockIdx.x])) : held;
    /* (for no tokens too: the child must be empty then as well) */
    if (threadIdx.x == 0) taken = atomicCAS(&c.lengths[child], 0, (int32_t)tokens) != 0;
    __syncthreads();
    if (taken) {
        if (threadIdx.x == 0) atomicOr(c.status, Q38_KV_NOT_EMPTY);
        return;
    }
    for (uint32_t entry = threadIdx.x; entry < pages_of(tokens, c.page_tokens); entry += 256) {
        const int32_t page = kv_page(c, parent, entry);
        c.tables[(uint64_t)child * c.table_entries + entry] = page;
        if (page >= 0) atomicAdd(&c.refs[page], 1);
        else atomicOr(c.status, Q38_KV_BAD_PAGE);
    }
}

/* one workgroup per sequence: each entry behind the new length is taken out by
 * an exchange, so a page leaves a table once even where a call repeats an id */
__global__ __launch_bounds__(256) void kv_truncate_kernel(Q38KVPages c, const int32_t *sequences, const int32_t *lengths)
{
    const int32_t id = sequences[blockIdx.x];
    if (id < 0 || (uint32_t)id >= c.sequences) {
        if (threadIdx.x == 0) atomicOr(c.status, Q38_KV_BAD_SEQUENCE);
        return;
    }
    const uint32_t held = kv_tokens(c, id);
    const uint32_t keep = min(held, (uint32_t)max(0, lengths[blockIdx.x])), T = c.page_tokens;
    __syncthreads();
    for (uint32_t entry = pages_of(keep, T) + threadIdx.x; entry < pages_of(held, T); entry += 256) {
        const int32_t page = atomicExch(&c.tables[(uint64_t)id * c.table_entries + entry], -1);
        if (page >= 0 && (uint32_t)page < c.pages) atomicSub(&c.refs[page], 1);
    }
    if (threadIdx.x == 0) atomicMin(&c.lengths[id], (int32_t)keep);
}

/* The plan of a compaction, by one workgroup: with n pages in use, the j-th
 * page in use at or above n moves to the j-th free page below n.  plan[0] = the
 * number of moves, plan[1] = n, then the targets, the sources and, for a source
 * page, its new place. */
__global__ __launch_bounds__(kPlan) void kv_compact_plan_kernel(Q38KVPages c, int32_t *plan)
{
    __shared__ uint32_t sums[kPlan / 64];
    int32_t *targets = plan + 2, *sources = targets + c.pages, *place = sources + c.pages;
    const uint32_t i = threadIdx.x;
    uint32_t free_pages = 0, all, first_bits = 0;
    for (uint64_t first = 0; first < c.pages; first += kPlan * kScanEach) {
        const uint64_t mine = first + i * kScanEach;
        const uint32_t bits = mine < c.pages ? free_bits(c.refs, (uint32_t)mine, c.pages) : 0;
        if (!first) first_bits = bits;
        free_pages += __popc(bits);
    }
    block_prefix(free_pages, sums, all);
    const uint32_t live = c.pages - all;
    __syncthreads();
    uint32_t holes = 0, movers = 0;
    for (uint64_t first = 0; first < c.pages; first += kPlan * kScanEach) {
        const uint64_t mine = first + i * kScanEach;
        uint32_t hole = 0, mover = 0;
        if (mine < c.pages) {
            const uint32_t inside = (uint32_t)min((uint64_t)kScanEach, c.pages - mine);
            const uint32_t below = mine >= live ? 0 : (uint32_t)min((uint64_t)kScanEach, live - mine);
            const uint32_t bits = first ? free_bits(c.refs, (uint32_t)mine, c.pages) : first_bits;
            hole = bits & ((1u << below) - 1);
            mover = ~bits & ((1u << inside) - 1) & ~((1u << below) - 1);
        }
        /* both ranks in one sum: a round has 2^14 pages */
        const uint32_t before = block_prefix((uint32_t)__popc(hole) | (uint32_t)__popc(mover) << 16, sums, all);
        uint32_t rank = holes + (before & 0xffffu);
        for (; hole; hole &= hole - 1) targets[rank++] = (int32_t)mine + __ffs(hole) - 1;
        rank = movers + (before >> 16);
        for (; mover; mover &= mover - 1) sources[rank++] = (int32_t)mine + __ffs(mover) - 1;
        holes += all & 0xffffu;
        movers += all >> 16;
        __syncthreads();
    }
    __threadfence_block();
    __syncthreads();
    for (uint32_t k = i; k < movers; k += kPlan) {
        const int32_t from = sources[k], to = targets[k];
        place[from] = to;
        c.refs[to] = c.refs[from];
        c.refs[from] = 0;
    }
    if (i == 0) {
        plan[0] = (int32_t)movers;
        plan[1] = (int32_t)live;
    }
}

/* the moves, and the tables after them: blockIdx.x is a slice of a layer's
 * page, blockIdx.y every so-manieth move */
__global__ __launch_bounds__(256) void kv_compact_kernel(Q38KVPages c, const int32_t *plan, uint32_t slices)
{
    const uint32_t moves = (uint32_t)plan[0], slice = blockIdx.x % slices, layer = blockIdx.x / slices;
    const int32_t live = plan[1];
    const int32_t *targets = plan + 2, *sources = targets + c.pages, *place = sources + c.pages;
    for (uint32_t k = blockIdx.y; k < moves; k += gridDim.y) copy_slice<true>(c, sources[k], targets[k], layer, slice);
    const uint64_t entries = (uint64_t)c.sequences * c.table_entries, blocks = (uint64_t)gridDim.x * gridDim.y;
    for (uint64_t e = ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; e < entries; e += blocks * 256) {
        const int32_t page = c.tables[e];
        if (page >= live && (uint32_t)page < c.pages) c.tables[e] = place[page];
    }
}

}  // namespace

bool launch_kv_reset(const Q38KVPages &c, hipStream_t stream)
{
    uint64_t most = (uint64_t)c.sequences * c.table_entries;
    most = most > c.pages ? most : c.pages;
    return launch_kernel(kv_reset_kernel, dim3((uint32_t)((most + 255) / 256)), dim3(256), stream, c);
}

uint64_t kv_workspace_bytes(const Q38KVPages &c)
{
    /* extend: 2 * kPlan pairs and up to `pages` pages; compact: 2 + 3 * pages */
    return (2ull * kPlan + 2 + 3ull * c.pages) * sizeof(int32_t);
}

static uint32_t copy_slices(const Q38KVPages &c)
{
    return (uint32_t)((kv_page_bytes(c) + kCopySlice - 1) / kCopySlice);
}

bool launch_kv_copy(const Q38KVPages &c, const int32_t *sources, const int32_t *targets, uint32_t count, hipStream_t stream)
{
    return launch_kernel(kv_copy_kernel, dim3(copy_slices(c), c.layers, count), dim3(256), stream, c, sources, targets);
}

bool launch_kv_extend(const Q38KVPages &c, const int32_t *sequences, const int32_t *rows, uint32_t count,
                      int32_t *workspace, hipStream_t stream)
{
    return launch_kernel(kv_extend_kernel, dim3(1), dim3(kPlan), stream, c, sequences, rows, count, workspace,
                         workspace + 2 * count) &&
           launch_kv_copy(c, workspace, workspace + count, count, stream);
}

bool launch_kv_fork(const Q38KVPages &c, const int32_t *parents, const int32_t *children, const int32_t *lengths,
                    uint32_t count, hipStream_t stream)
{
    return launch_kernel(kv_fork_kernel, dim3(count), dim3(256), stream, c, parents, children, lengths, count);
}

bool launch_kv_truncate(const Q38KVPages &c, const int32_t *sequences, const int32_t *lengths, uint32_t count,
                        hipStream_t stream)
{
    return launch_kernel(kv_truncate_kernel, dim3(count), dim3(256), stream, c, sequences, lengths);
}

bool launch_kv_compact(const Q38KVPages &c, int32_t *workspace, hipStream_t stream)
{
    const uint32_t slices = copy_slices(c), across = slices * c.layers, wanted = across < 8192 ? 8192 / across : 1;
    return launch_kernel(kv_compact_plan_kernel, dim3(1), dim3(kPlan), stream, c, workspace) &&
           launch_kernel(kv_compact_kernel, dim3(across, wanted < c.pages ? wanted : c.pages), dim3(256), stream, c,
                         (const int32_t *)workspace, slices);
}

}  // namespace q38
