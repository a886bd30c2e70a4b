"""Paged 8-bit key/value cache (section 3 of include/q38hip.h).

KVPages wraps the device tensors of a cache; its methods enqueue on torch's
current stream of their device, check shapes and types on the host and read
nothing back.  Ids, lengths and row offsets are int32 device tensors; what the device finds
wrong in them goes to the cache's status word (bits below), which check()
reads.

    cache = kv.KVPages.allocate(layers=17, pages=4096, page_tokens=64, kv_heads=4, head_dim=256, sequences=64,
                                table_entries=2048, kind="int8")
    cache.extend(ids, rows)                               # room for rows[i] more tokens
    cache.append(layer, key, value, ids, starts)          # [rows, 4, 256] each
    out = cache.attention(layer, query, ids, starts)      # [rows, 24, 256]
"""
import ctypes

from . import _check, lib

BAD_SEQUENCE, POOL_FULL, TABLE_FULL, BAD_PAGE, NOT_EMPTY, BAD_ROWS = 1, 2, 4, 8, 16, 32
KINDS = {"int8": 0, "e4m3": 1}
EXPORTS = ("q38hip_kv_reset", "q38hip_kv_workspace_bytes", "q38hip_kv_extend", "q38hip_kv_fork", "q38hip_kv_truncate",
           "q38hip_kv_compact", "q38hip_kv_copy", "q38hip_kv_append", "q38hip_kv_attention_workspace_bytes",
           "q38hip_kv_attention")


class Pages(ctypes.Structure):
    """Q38KVPages"""
    _fields_ = ([(name, ctypes.c_void_p) for name in ("data", "scales", "refs", "tables", "lengths", "status")] +
                [(name, ctypes.c_uint32) for name in ("layers", "pages", "page_tokens", "kv_heads", "head_dim",
                                                      "sequences", "table_entries", "type")])


_BOUND = None


def _lib():
    """the library, with the argument types of this module's functions"""
    global _BOUND
    if _BOUND is None:
        bound = lib()
        vp, u32, u64, cache = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.POINTER(Pages)
        for name, result, arguments in (
                ("reset", ctypes.c_int, [cache, vp]),
                ("workspace_bytes", u64, [cache]),
                ("extend", ctypes.c_int, [cache, vp, vp, u32, vp, vp]),
                ("fork", ctypes.c_int, [cache, vp, vp, vp, u32, vp]),
                ("truncate", ctypes.c_int, [cache, vp, vp, u32, vp]),
                ("compact", ctypes.c_int, [cache, vp, vp]),
                ("copy", ctypes.c_int, [cache, vp, vp, u32, vp]),
                ("append", ctypes.c_int, [cache, u32, vp, vp, u32, u64, vp, vp, u32, u32, vp]),
                ("attention_workspace_bytes", u64, [cache, u32, u32, u32, u32]),
                ("attention", ctypes.c_int, [cache, u32, vp, vp, vp, u32, u32, u64, u64, u64, ctypes.c_float, vp, vp, u32,
                                             u32, vp, vp])):
            function = getattr(bound, "q38hip_kv_" + name)
            function.restype, function.argtypes = result, arguments
        _BOUND = bound
    return _BOUND


class _Elsewhere:
    """the library's functions, called with a device that is not the current one"""

    def __init__(self, device):
        self._device = device

    def __getattr__(self, name):
        function = getattr(_lib(), name)

        def call(*arguments):
            with self._device:
                return function(*arguments)
        return call


def _element_types():
    import torch
    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class KVPages:
    """The tensors of a cache: data uint8 [layers, pages, 2, kv_heads,
    page_tokens, head_dim] (keys as that says, values as head_dim rows of
    page_tokens), scales float32 [layers, pages, 2, kv_heads], refs int32
    [pages], tables int32 [sequences, table_entries], lengths int32
    [sequences], status int32 [1], all on one GPU and contiguous."""

    def __init__(self, data, scales, refs, tables, lengths, status, kind):
        import torch
        if kind not in KINDS:
            raise ValueError("kind must be one of %s" % ", ".join(KINDS))
        if data.dim() != 6 or data.shape[2] != 2 or tables.dim() != 2:
            raise ValueError("expected data [layers, pages, 2, kv_heads, page_tokens, head_dim] and tables "
                             "[sequences, table_entries]")
        layers, pages, _, kv_heads, page_tokens, head_dim = data.shape
        for name, tensor, dtype, shape in (("data", data, torch.uint8, data.shape),
                                           ("scales", scales, torch.float32, (layers, pages, 2, kv_heads)),
                                           ("refs", refs, torch.int32, (pages,)),
                                           ("tables", tables, torch.int32, tables.shape),
                                           ("lengths", lengths, torch.int32, (tables.shape[0],)),
                                           ("status", status, torch.int32, (1,))):
            if tensor.dtype != dtype or tuple(tensor.shape) != tuple(shape) or not tensor.is_contiguous():
                raise ValueError("%s must be a contiguous %s tensor of shape %s" % (name, dtype, tuple(shape)))
            if tensor.device != data.device:
                raise ValueError("the cache's tensors must be on one device")
        self.data, self.scales, self.refs = data, scales, refs
        self.tables, self.lengths, self.status, self.kind = tables, lengths, status, kind
        self.layers, self.pages, self.kv_heads = layers, pages, kv_heads
        self.page_tokens, self.head_dim = page_tokens, head_dim
        self.sequences, self.table_entries = tables.shape
        self._struct = Pages(data.data_ptr(), scales.data_ptr(), refs.data_ptr(), tables.data_ptr(), lengths.data_ptr(),
                             status.data_ptr(), layers, pages, page_tokens, kv_heads, head_dim, self.sequences,
                             self.table_entries, KINDS[kind])
        self._ref = ctypes.byref(self._struct)
        self._torch, self._int32, self._device, self._types = torch, torch.int32, data.device, _element_types()
        self._index = data.get_device()
        self._bytes = {}                       # workspace of an attention call, by its sizes
        self._pages_workspace, self._words_needed = None, 0

    @classmethod
    def allocate(cls, layers, pages, page_tokens, kv_heads, head_dim, sequences, table_entries, kind="int8",
                 device="cuda"):
        """an empty cache"""
        import torch
        make = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        cache = cls(make(torch.uint8, layers, pages, 2, kv_heads, page_tokens, head_dim),
                    make(torch.float32, layers, pages, 2, kv_heads), make(torch.int32, pages),
                    make(torch.int32, sequences, table_entries), make(torch.int32, sequences), make(torch.int32, 1), kind)
        cache.reset()
        return cache

    # ---- checks ----------------------------------------------------------------

    def _stream(self):
        """torch's current stream of the cache's device"""
        return self._torch._C._cuda_getCurrentRawStream(self._index)

    def _calls(self):
        """the library's functions.  They launch on the current device, which has to be the cache's: the handle of a
        default stream is the same on all devices."""
        torch = self._torch
        return _lib() if torch._C._cuda_getDevice() == self._index else _Elsewhere(torch.cuda.device(self._index))

    def _type(self, dtype):
        kind = self._types.get(dtype)
        if kind is None:
            raise ValueError("expected float32, float16 or bfloat16 rows")
        return kind

    def _words(self, tensor, name, count=None):
        """pointer of an int32 [count] device tensor"""
        shape = tensor.shape
        if tensor.dtype != self._int32 or len(shape) != 1 or not tensor.is_contiguous():
            raise ValueError("%s must be a contiguous int32 vector" % name)
        if count is not None and shape[0] != count:
            raise ValueError("%s must have %d words" % (name, count))
        if tensor.get_device() != self._index:
            raise ValueError("%s must be on the cache's device" % name)
        return tensor.data_ptr()

    def _rows(self, sequences, row_starts, total):
        shape = sequences.shape
        count = shape[0] if len(shape) == 1 else 0
        ids = self._words(sequences, "sequences")
        starts = None if row_starts is None else self._words(row_starts, "row_starts", count + 1)
        if row_starts is None and count and total % count:
            raise ValueError("rows must be a multiple of sequences without row_starts")
        return ids, starts, count

    def _workspace(self, nbytes):
        return self._torch.empty(nbytes, dtype=self._torch.uint8, device=self._device)

    def _pages_words(self):
        """32-bit words of the workspace of extend and compact"""
        if not self._words_needed:
            self._words_needed = _lib().q38hip_kv_workspace_bytes(self._ref) // 4
        return self._words_needed

    def check(self):
        """Synchronises; raises where a call found bad ids or no room, and clears the status."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            names = ("bad sequence id", "page pool full", "table full", "page outside the pool", "fork into a sequence "
                     "that is not empty", "row offsets that decrease")
            raise RuntimeError("paged cache: " + ", ".join(n for i, n in enumerate(names) if bits >> i & 1))

    # ---- pages -------------------------------------------------------------------

    def reset(self):
        """every page free, every sequence empty"""
        _check(self._calls().q38hip_kv_reset(self._ref, self._stream()), "q38hip_kv_reset")

    def extend(self, sequences, rows):
        """sequences[i] grows by rows[i] tokens; shared last pages are copied first"""
        ids = self._words(sequences, "sequences")
        more = self._words(rows, "rows", sequences.shape[0])
        if self._pages_workspace is None:      # calls on a cache are in order, so one serves them all
            self._pages_workspace = self._workspace(4 * self._pages_words())
        _check(self._calls().q38hip_kv_extend(self._ref, ids, more, sequences.shape[0], self._pages_workspace.data_ptr(),
                                              self._stream()), "q38hip_kv_extend")

    def fork(self, parents, children, lengths=None):
        """children[i] (empty) becomes the first lengths[i] tokens (default: all) of parents[i]"""
        count = parents.shape[0]
        taken, given = self._words(parents, "parents"), self._words(children, "children", count)
        keep = None if lengths is None else self._words(lengths, "lengths", count)
        _check(self._calls().q38hip_kv_fork(self._ref, taken, given, keep, count, self._stream()), "q38hip_kv_fork")

    def truncate(self, sequences, lengths):
        """sequences[i] keeps its first lengths[i] tokens; 0 frees it"""
        count = sequences.shape[0]
        ids, keep = self._words(sequences, "sequences"), self._words(lengths, "lengths", count)
        _check(self._calls().q38hip_kv_truncate(self._ref, ids, keep, count, self._stream()), "q38hip_kv_truncate")

    def compact(self):
        """The pages in use move to the front of the pool.  Returns an int32
        [2] device tensor: the pages moved and the pages in use."""
        work = self._torch.empty(self._pages_words(), dtype=self._int32, device=self._device)
        _check(self._calls().q38hip_kv_compact(self._ref, work.data_ptr(), self._stream()), "q38hip_kv_compact")
        return work[:2]

    def copy(self, sources, targets):
        """pages sources[i] to pages targets[i], in all layers"""
        count = sources.shape[0]
        taken, given = self._words(sources, "sources"), self._words(targets, "targets", count)
        _check(self._calls().q38hip_kv_copy(self._ref, taken, given, count, self._stream()), "q38hip_kv_copy")

    # ---- rows --------------------------------------------------------------------

    def append(self, layer, key, value, sequences, row_starts=None):
        """The last rows of each sequence into one layer: key and value [rows,
        kv_heads, head_dim] with equal row strides."""
        rows, heads, dim = key.shape[0], self.kv_heads, self.head_dim
        stride = key.stride()
        if key.shape != (rows, heads, dim) or value.shape != key.shape or stride[1:] != (dim, 1) or \
                value.stride()[1:] != (dim, 1):
            raise ValueError("expected keys and values [rows, %d, %d] with contiguous heads" % (heads, dim))
        if key.dtype != value.dtype or stride[0] != value.stride(0) and rows > 1:
            raise ValueError("keys and values must have one type and row stride")
        if key.get_device() != self._index or value.get_device() != self._index:
            raise ValueError("keys and values must be on the cache's device")
        ids, starts, count = self._rows(sequences, row_starts, rows)
        kind = self._type(key.dtype)
        _check(self._calls().q38hip_kv_append(self._ref, layer, key.data_ptr(), value.data_ptr(), kind, stride[0], ids, starts,
                                              count, rows, self._stream()), "q38hip_kv_append")

    def attention(self, layer, query, sequences, row_starts=None, gate=None, scale=None, out=None):
        """Causal attention of each sequence's last rows in one layer: query
        (and gate) [rows, heads, head_dim] with contiguous channels and equal
        strides; the result [rows, heads, head_dim] in the query's type.
        Rows that row_starts leaves out are not written."""
        shape, stride, dtype = query.shape, query.stride(), query.dtype
        if len(shape) != 3 or shape[2] != self.head_dim or stride[2] != 1:
            raise ValueError("expected queries [rows, heads, %d] with contiguous channels" % self.head_dim)
        rows, heads, dim = shape
        if query.get_device() != self._index:
            raise ValueError("queries must be on the cache's device")
        if gate is not None and (gate.shape != shape or gate.stride() != stride or gate.dtype != dtype or
                                 gate.get_device() != self._index):
            raise ValueError("the gate must be laid out as the queries")
        if out is None:
            out = self._torch.empty(shape, dtype=dtype, device=self._device)
        elif out.shape != shape or out.dtype != dtype or out.get_device() != self._index or out.stride()[1:] != (dim, 1):
            raise ValueError("out must be [rows, heads, head_dim] in the queries' type with contiguous heads")
        ids, starts, count = self._rows(sequences, row_starts, rows)
        kind, bound = self._type(dtype), self._calls()
        nbytes = self._bytes.get((kind, heads, count, rows))
        if nbytes is None:
            nbytes = bound.q38hip_kv_attention_workspace_bytes(self._ref, kind, heads, count, rows)
            if len(self._bytes) >= 4096:
                self._bytes.clear()
            self._bytes[kind, heads, count, rows] = nbytes
        work = self._workspace(nbytes) if nbytes else None
        _check(bound.q38hip_kv_attention(self._ref, layer, out.data_ptr(), query.data_ptr(),
                                         None if gate is None else gate.data_ptr(), kind, heads, stride[0], stride[1],
                                         out.stride(0), dim ** -0.5 if scale is None else scale, ids, starts, count, rows,
                                         None if work is None else work.data_ptr(), self._stream()), "q38hip_kv_attention")
        return out
