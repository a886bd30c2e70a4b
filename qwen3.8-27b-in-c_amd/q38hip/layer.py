"""Operators of a decoder layer (section 4 of include/q38hip.h), for programs
that bring their own model: norm, projections in 8 bits, rotary positions and
the attention of packed prompts.

Functions check shapes and types on the host, enqueue on torch's current stream
of their tensors' device and read nothing back; there is at least one row, and
results carry no gradient.  Rows in 8 bits are a pair (codes, scales):
float8_e4m3fn [rows, width] and float8_e8m0fnu [rows, blocks of 128 rounded up to
a multiple of 4].

    y, x = layer.rms_norm(x, weight, addend=attended, e4m3=True)     # x + addend, and its norm in 8 bits
    both = layer.product(y, gate_up, gate_up_scales)                 # bfloat16 [rows, 2 * hidden]
    z = layer.quantize(both[:, hidden:], gate=both[:, :hidden])      # SwiGLU, in 8 bits
    q = layer.rotary(q, positions, frequencies)                      # [rows, heads, head_dim]
    out = layer.attention(q, k, v, row_starts)                       # causal, within each prompt
"""
import ctypes
import math
from collections import namedtuple

import torch

from . import _check, lib

EXPORTS = ("q38hip_e4m3_scale_pitch", "q38hip_quantize_e4m3", "q38hip_rms_norm", "q38hip_gemm_e4m3_workspace_bytes",
           "q38hip_gemm_e4m3", "q38hip_rotary", "q38hip_prompt_attention")
BLOCK = 128

E4M3Rows = namedtuple("E4M3Rows", "codes scales")

_CODES, _SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_BOUND = None


def _lib():
    """the library, with the argument types of this module's functions"""
    global _BOUND
    if _BOUND is None:
        bound = lib()
        vp, u32, u64, f32, i32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_float, ctypes.c_int
        for name, result, arguments in (
                ("e4m3_scale_pitch", u32, [u64]),
                ("quantize_e4m3", i32, [vp, vp, vp, u64, vp, u64, u32, u64, u32, vp]),
                ("rms_norm", i32, [vp, u64, vp, vp, vp, u64, vp, u64, vp, u64, u32, vp, u32, f32, f32, u64, u32, vp]),
                ("gemm_e4m3_workspace_bytes", u64, [u32, u64, u32]),
                ("gemm_e4m3", i32, [vp, u32, u64, vp, vp, u32, u64, vp, vp, u32, vp, vp]),
                ("rotary", i32, [vp, u64, u64, vp, u64, u64, u32, u32, u32, u32, vp, vp, u32, i32, f32, vp]),
                ("prompt_attention", i32, [vp, u64, vp, vp, u64, u64, vp, u64, vp, u64, u32, u32, u32, u32, f32, vp, u32,
                                           u32, vp])):
            function = getattr(bound, "q38hip_" + name)
            function.restype, function.argtypes = result, arguments
        _BOUND = bound
    return _BOUND


def _call(name, index, *arguments):
    """enqueues on torch's current stream of device `index`.  The library launches on the current device, which has to be
    that one: the handle of a default stream is the same on all devices."""
    function = getattr(_BOUND or _lib(), name)
    if _device() == index:
        ok = function(*arguments, _stream(index))
    else:
        with torch.cuda.device(index):
            ok = function(*arguments, _stream(index))
    if not ok:
        _check(ok, name)


def _rows(x, name):
    """(rows, width, row stride, element type, device) of rows that are contiguous each.  One look at each property: small
    calls cost what they cost the host."""
    shape, stride, index, kind = x.shape, x.stride(), x.get_device(), _TYPES.get(x.dtype)
    if len(shape) != 2 or stride[1] != 1 and shape[1] > 1:
        raise ValueError("%s must be [rows, width] with contiguous rows" % name)
    if kind is None:
        raise ValueError("%s must be float32, float16 or bfloat16" % name)
    if index < 0:
        raise ValueError("%s must be on a GPU" % name)
    return shape[0], shape[1], stride[0], kind, index


def _alike(tensor, name, x, index):
    """row stride of a tensor of x's shape, type and device with contiguous rows"""
    stride = tensor.stride()
    if tensor.shape != x.shape or tensor.dtype != x.dtype or tensor.get_device() != index or \
            stride[1] != 1 and x.shape[1] > 1:
        raise ValueError("%s must be rows of the same shape, type and device, each contiguous" % name)
    return stride[0]


def scale_pitch(width):
    """scale bytes of a row of `width` elements"""
    return -(-width // (4 * BLOCK)) * 4


def _e4m3(x, rows, width, index, into):
    """new rows in 8 bits of x's shape, or the caller's"""
    if into is None:
        into = (torch.empty_like(x, dtype=_CODES, memory_format=torch.contiguous_format),
                x.new_empty((rows, -(-width // 512) * 4), dtype=_SCALES))
    else:
        _check_e4m3(into, rows, width, index)
    return tuple.__new__(E4M3Rows, into)


def _check_e4m3(rows8, rows, width, index):
    codes, scales = rows8
    if codes.dtype != _CODES or codes.shape != (rows, width) or not codes.is_contiguous() or \
            scales.dtype != _SCALES or scales.shape != (rows, scale_pitch(width)) or not scales.is_contiguous():
        raise ValueError("rows in 8 bits must be contiguous float8_e4m3fn [%d, %d] and float8_e8m0fnu [%d, %d]"
                         % (rows, width, rows, scale_pitch(width)))
    if codes.get_device() != index or scales.get_device() != index:
        raise ValueError("rows in 8 bits must be on the device of the other tensors")


def quantize(x, gate=None, out=None):
    """x [rows, width], or x * silu(gate), in 8 bits; gate has x's shape and type, and a row stride of its own."""
    rows, width, stride, kind, index = _rows(x, "x")
    gate_row = 0 if gate is None else _alike(gate, "gate", x, index)
    out = _e4m3(x, rows, width, index, out)
    _call("q38hip_quantize_e4m3", index, out[0].data_ptr(), out[1].data_ptr(), x.data_ptr(), stride,
          None if gate is None else gate.data_ptr(), gate_row, kind, width, rows)
    return out


def rms_norm(x, weight, eps=1e-6, addend=None, offset=0.0, e4m3=False, out=None, total=None):
    """The root-mean-square norm of x [rows, width], or of x + addend, times weight + offset: in x's type, or in 8 bits
    where e4m3 is true.  With an addend the result is (norm, sum); total takes the sum, and may be x or addend."""
    rows, width, stride, kind, index = _rows(x, "x")
    weight_kind = _TYPES.get(weight.dtype)
    if weight_kind is None or weight.shape != (width,) or width > 1 and weight.stride(0) != 1 or weight.get_device() != index:
        raise ValueError("weight must be a contiguous float32, float16 or bfloat16 vector of %d elements on x's device" % width)
    if addend is not None:
        addend_row, added = _alike(addend, "addend", x, index), addend.data_ptr()
        if total is None:
            total, total_row = torch.empty_like(x, memory_format=torch.contiguous_format), width
        else:
            total_row = stride if total is x else _alike(total, "total", x, index)
        sum_at = total.data_ptr()
    elif total is None:
        addend_row = total_row = 0
        added = sum_at = None
    else:
        raise ValueError("total needs an addend")
    if e4m3:
        out = _e4m3(x, rows, width, index, out)
        to, to_row, codes, scales = None, 0, out[0].data_ptr(), out[1].data_ptr()
    else:
        if out is None:
            out, to_row = torch.empty_like(x, memory_format=torch.contiguous_format), width
        else:
            to_row = _alike(out, "out", x, index)
        to, codes, scales = out.data_ptr(), None, None
    _call("q38hip_rms_norm", index, to, to_row, codes, scales, sum_at, total_row, x.data_ptr(), stride, added, addend_row, kind,
          weight.data_ptr(), weight_kind, offset, eps, width, rows)
    return out if addend is None else (out, total)


_WORKSPACES = {}


def product(rows8, weight, weight_scales, dtype=torch.bfloat16, out=None):
    """Rows in 8 bits [rows, inputs] times weight [outputs, inputs] (float8_e4m3fn) with weight_scales [ceil(outputs /
    128), ceil(inputs / 128)] (float32): [rows, outputs] of dtype, or of out's."""
    codes = rows8[0]
    if codes.dim() != 2 or weight.dim() != 2:
        raise ValueError("expected codes [rows, inputs] and weight [outputs, inputs]")
    (rows, inputs), (outputs, columns), index = codes.shape, weight.shape, weight.get_device()
    if weight.dtype != _CODES or columns != inputs or not weight.is_contiguous() or index < 0:
        raise ValueError("weight must be contiguous float8_e4m3fn [outputs, %d] on a GPU" % inputs)
    _check_e4m3(rows8, rows, inputs, index)
    if weight_scales.dtype != torch.float32 or weight_scales.shape != (-(-outputs // BLOCK), -(-inputs // BLOCK)) or \
            not weight_scales.is_contiguous() or weight_scales.get_device() != index:
        raise ValueError("weight_scales must be contiguous float32 [%d, %d] on the weight's device"
                         % (-(-outputs // BLOCK), -(-inputs // BLOCK)))
    if out is None:
        out = weight.new_empty((rows, outputs), dtype=dtype)
        stride = outputs
    else:
        stride = out.stride()[0] if out.dim() == 2 else 0
        if out.shape != (rows, outputs) or out.get_device() != index or out.stride(1) != 1 and outputs > 1:
            raise ValueError("out must be [%d, %d] with contiguous rows on the weight's device" % (rows, outputs))
    kind, sizes = _TYPES.get(out.dtype), (rows, inputs, outputs)
    if kind is None:
        raise ValueError("the result must be float32, float16 or bfloat16")
    nbytes = _WORKSPACES.get(sizes)
    if nbytes is None:
        nbytes = _lib().q38hip_gemm_e4m3_workspace_bytes(*sizes)
        if len(_WORKSPACES) >= 4096:
            _WORKSPACES.clear()
        _WORKSPACES[sizes] = nbytes
    work = weight.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    _call("q38hip_gemm_e4m3", index, out.data_ptr(), kind, stride, codes.data_ptr(), rows8[1].data_ptr(), rows, inputs,
          weight.data_ptr(), weight_scales.data_ptr(), outputs, None if work is None else work.data_ptr())
    return out


def rotary_frequencies(turned, base=10000.0, factor=1.0, original=None, fast=32.0, slow=1.0, device=None):
    """Frequencies of the turned / 2 pairs (float32) and the magnitude for rotary(): base^(-2i / turned).  With a factor
    above 1 for longer contexts: divided by it for all pairs where `original` is None; else, with `original` the context
    that the model was trained on, pairs that turn at least `fast` times within it stay, those that turn at most `slow`
    times are divided, those between are blended linearly in the pair's index, and the magnitude is 0.1 ln(factor) + 1 (the
    method of Peng, Quesnelle, Fan and Shippole, "YaRN: Efficient Context Window Extension of Large Language Models", 2023)."""
    if turned < 2 or turned % 2 or not 1 < base < math.inf or not 1 <= factor < math.inf or not math.inf > fast > slow > 0 or \
            (original is not None and not 0 < original < math.inf):
        raise ValueError("expected an even number of channels, a base above 1, a factor of at least 1, a context above 0 and fast above "
                         "slow above 0")
    pairs = torch.arange(turned // 2, dtype=torch.float64)
    plain, magnitude = base ** (-2 * pairs / turned), 1.0
    frequencies = plain / factor
    if original is not None and factor > 1:
        # pair i turns original * base^(-2i / turned) / (2 pi) times
        at = lambda turns: turned * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), turned - 1)
        # where not even pair 0 turns more than `slow` times all are divided
        part = ((pairs - low) / max(high - low, 0.001)).clamp(0, 1) if high > 0 else torch.ones_like(pairs)
        frequencies = plain * (1 - part) + frequencies * part
        magnitude = 0.1 * math.log(factor) + 1
    return frequencies.float().to(device), magnitude


def _heads(x, name):
    """(shape, strides, element type, device) of [rows, heads, head_dim] with contiguous heads"""
    shape, stride, index, kind = x.shape, x.stride(), x.get_device(), _TYPES.get(x.dtype)
    if len(shape) != 3 or stride[2] != 1 and shape[2] > 1:
        raise ValueError("%s must be [rows, heads, head_dim] with contiguous heads" % name)
    if kind is None:
        raise ValueError("%s must be float32, float16 or bfloat16" % name)
    if index < 0:
        raise ValueError("%s must be on a GPU" % name)
    return shape, stride, kind, index


def _words(tensor, name, index):
    if tensor.dtype != torch.int32 or tensor.dim() != 1 or not tensor.is_contiguous() or tensor.get_device() != index:
        raise ValueError("%s must be a contiguous int32 vector on the device of the rows" % name)
    return tensor.shape[0]


def rotary(x, positions, frequencies, interleaved=False, magnitude=1.0, out=None):
    """Turns the first 2 * len(frequencies) channels of each head of x [rows, heads, head_dim] by positions[row] *
    frequencies[pair]; out may be x."""
    (rows, heads, dim), stride, kind, index = _heads(x, "x")
    if _words(positions, "positions", index) != rows:
        raise ValueError("positions must have %d words" % rows)
    if frequencies.dtype != torch.float32 or frequencies.dim() != 1 or not frequencies.is_contiguous() or \
            frequencies.get_device() != index:
        raise ValueError("frequencies must be a contiguous float32 vector on x's device")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        to = (heads * dim, dim)
    elif out is x:
        to = stride
    else:
        shape, to, out_kind, out_index = _heads(out, "out")
        if shape != x.shape or out_kind != kind or out_index != index:
            raise ValueError("out must be laid out as x")
    _call("q38hip_rotary", index, out.data_ptr(), to[0], to[1], x.data_ptr(), stride[0], stride[1], kind, rows, heads, dim,
          positions.data_ptr(), frequencies.data_ptr(), frequencies.shape[0], 1 if interleaved else 0, magnitude)
    return out


def _key_rows(tensor, name, query, rows, dim, index):
    """row stride of keys or values: heads next to each other"""
    shape, stride = tensor.shape, tensor.stride()
    if len(shape) != 3 or shape[0] != rows or shape[2] != dim or tensor.dtype != query.dtype or tensor.get_device() != index or \
            stride[2] != 1 or stride[1] != dim and shape[1] > 1:
        raise ValueError("%s must be [%d, kv_heads, %d] of the queries' type and device, with heads next to each other"
                         % (name, rows, dim))
    return stride[0]


def attention(query, key, value, row_starts, gate=None, scale=None, out=None):
    """Causal attention of packed prompts: sequence i owns rows row_starts[i] .. row_starts[i + 1] - 1 (int32, on the
    device).  query (and gate, laid out alike) [rows, heads, head_dim], key and value [rows, kv_heads, head_dim] with heads
    next to each other; the result is [rows, heads, head_dim] in their type.  Rows that no sequence owns are not written."""
    (rows, heads, dim), stride, kind, index = _heads(query, "query")
    key_row, value_row = _key_rows(key, "key", query, rows, dim, index), _key_rows(value, "value", query, rows, dim, index)
    if key.shape != value.shape:
        raise ValueError("keys and values must have one shape")
    if gate is not None and (gate.shape != query.shape or gate.stride() != stride or gate.dtype != query.dtype or
                             gate.get_device() != index):
        raise ValueError("the gate must be laid out as the queries")
    count = _words(row_starts, "row_starts", index) - 1
    if count < 1:
        raise ValueError("row_starts must have an offset for each sequence and one behind the last")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        out_row = heads * dim
    else:
        shape, to, out_kind, out_index = _heads(out, "out")
        if shape != query.shape or out_kind != kind or out_index != index or heads > 1 and to[1] != dim:
            raise ValueError("out must be [rows, heads, head_dim] in the queries' type, with heads next to each other")
        out_row = to[0]
    _call("q38hip_prompt_attention", index, out.data_ptr(), out_row, query.data_ptr(),
          None if gate is None else gate.data_ptr(), stride[0], stride[1], key.data_ptr(), key_row, value.data_ptr(), value_row,
          kind, heads, key.shape[1], dim, dim ** -0.5 if scale is None else scale, row_starts.data_ptr(), count, rows)
    return out
