"""Plain models of a decoder layer's operators (include/q38hip.h, section 4) in
numpy with 64-bit values, and the bounds of the kernels' errors against them."""
import numpy as np
import torch

import kv_cases as kc

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
HALF_STEP = kc.HALF_STEP
# what a value below the type's normal range may be off: half its smallest step
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}


def f64(x):
    return x.detach().double().cpu().numpy()


def rounding(want, dtype):
    return np.abs(want) * HALF_STEP[dtype] + TINY[dtype]


def check(got, want, bound):
    got = f64(got)
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    far = np.abs(got - want)
    assert (far <= bound).all(), "worst %g of its bound" % (far / bound).max()


def pitch(width):
    return -(-width // 512) * 4


def blocks_of(y):
    """y [rows, width] as [rows, blocks, 128], zeros behind the end"""
    rows, width = y.shape
    blocks = -(-width // 128)
    out = np.zeros((rows, blocks * 128))
    out[:, :width] = y
    return out.reshape(rows, blocks, 128)


def quantize(y):
    """codes (uint8) and scale bytes of float64 rows"""
    rows, width = y.shape
    part = blocks_of(y)
    bad = ~np.isfinite(part).all(2)
    largest = np.where(bad, 1.0, np.abs(np.where(np.isfinite(part), part, 0)).max(2))
    fraction, power = np.frexp(largest / 448.0)           # division by 7 * 2^6 rounds, so the border is settled exactly:
    k = np.where(largest <= np.ldexp(448.0, power - 1), power - 1, power)
    k = np.where(largest > np.ldexp(448.0, k), k + 1, k)
    k = np.where(largest == 0, -100, np.maximum(k, -100))
    codes = kc.encode(np.where(bad[:, :, None], 0, np.where(np.isfinite(part), part, 0)) / np.ldexp(1.0, k)[:, :, None], "e4m3")
    codes = np.where(bad[:, :, None], 0x7f, codes).astype(np.uint8).reshape(rows, -1)[:, :width]
    scales = np.zeros((rows, pitch(width)), dtype=np.uint8)
    scales[:, :k.shape[1]] = np.where(bad, 255, k + 127)
    return codes, scales


def check_quantized(got, y, relative):
    """Rows in 8 bits against float64 rows whose values are known to `relative`
    of themselves: a scale is the model's, or that of a largest value so much
    larger or smaller; a value is off by what was known and half a step of its
    code (2^-4 of it; below 2^-6 of the scale the steps are 2^-9)."""
    codes, scales = got.codes.view(torch.uint8).cpu().numpy(), got.scales.view(torch.uint8).cpu().numpy()
    rows, width = y.shape
    blocks = -(-width // 128)
    low, high = quantize(y * (1 - relative))[1], quantize(y * (1 + relative))[1]
    assert ((scales >= low) & (scales <= high)).all()
    scale = np.repeat(np.ldexp(1.0, scales[:, :blocks].astype(int) - 127), 128, 1)[:, :width]
    value = kc.decode(codes, "e4m3") * scale
    bound = np.abs(y) * relative + np.maximum(np.abs(y) * (1 + relative) * 2.0 ** -4, scale * 2.0 ** -10)
    far = np.abs(value - y)
    assert (far <= bound).all(), "worst %g of its bound" % (far / bound).max()


def silu(g):
    return g / (1 + np.exp(-g))


def rms_norm(total, weight, eps, offset):
    return total / np.sqrt((total * total).mean(1, keepdims=True) + eps) * (weight + offset)


def dequantize(codes, scales):
    rows, width = codes.shape
    blocks = -(-width // 128)
    scale = np.ldexp(1.0, scales[:, :blocks].astype(int) - 127)
    return kc.decode(codes, "e4m3") * np.repeat(scale, 128, 1)[:, :width]


def product(codes, scales, weight, weight_scales):
    """the product, and (the sums of its terms' magnitudes, the sums over blocks of their factors' largest magnitudes' products)"""
    x = dequantize(codes, scales)
    outputs, inputs = weight.shape
    w = kc.decode(weight, "e4m3") * np.repeat(np.repeat(weight_scales.astype(np.float64), 128, 0)[:outputs], 128, 1)[:, :inputs]
    return x @ w.T, (np.abs(x) @ np.abs(w).T, np.abs(blocks_of(x)).max(2) @ np.abs(blocks_of(w)).max(2).T)


def product_bound(want, mass, inputs, dtype):
    """A block's 128 products are exact in fp32; their sum takes 127 roundings or
    truncations (2^-23 each at most) of partial sums that its mass bounds, each
    block's scaling and addition 2 more of 2^-24, or of half the smallest fp32
    step (2^-150) where the sum is below the normal range.  For 16-bit outputs the matrix
    unit adds products of codes at 13 bits below the largest: each of a block's 128 is off
    by up to 2^-13 of that, either way; a sum of n such is off by sqrt(n) of them in
    the mean, six times that at most: 6 sqrt(128) < 68."""
    blocks = -(-inputs // 128)
    mass, largest = mass
    matrix_unit = 0 if dtype == F32 else largest * 68 * 2.0 ** -13
    return matrix_unit + mass * (127 * 2.0 ** -23 + (blocks + 2) * 2.0 ** -24) + blocks * 2.0 ** -150 + rounding(want, dtype) * 1.01


def rotary(x, positions, frequencies, interleaved, magnitude):
    pairs = len(frequencies)
    angle = np.multiply.outer(positions.astype(np.float64), frequencies.astype(np.float64))[:, None]
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    out, size = x.copy(), np.zeros_like(x)
    out[..., a] = magnitude * (x[..., a] * np.cos(angle) - x[..., b] * np.sin(angle))
    out[..., b] = magnitude * (x[..., b] * np.cos(angle) + x[..., a] * np.sin(angle))
    size[..., a] = size[..., b] = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return out, size


def rotary_bound(want, size, turns, dtype):
    """The angle in turns is formed in fp64 (two roundings of `turns`), its rest
    below half a turn rounded to fp32 (2^-26 of a turn: 2^-23 of a radian), its sine and
    cosine good to 2^-23, then three more roundings of 2^-24."""
    return size * (2.0 ** -23 + 2.0 ** -23 + 3 * 2.0 ** -24 + 2 * np.pi * turns * 2.0 ** -52) + rounding(want, dtype) * 1.01


def sequence_of(starts, rows):
    """first row of the sequence that owns each row, -1 where none does"""
    out = np.full(rows, -1)
    for a, b in zip(starts, starts[1:]):
        out[a:b] = a
    return out


def attention(query, key, value, starts, scale, gate=None):
    """outputs (nan for rows that no sequence owns), their terms' mass, and sums of the scores' magnitudes"""
    rows, heads, dim = query.shape
    group = heads // key.shape[1]
    want, mass, size = np.full(query.shape, np.nan), np.full(query.shape, np.nan), np.zeros((rows, heads))
    first = sequence_of(starts, rows)
    for a, b in zip(starts, starts[1:]):
        n = b - a
        if not n:
            continue
        hidden = np.triu(np.ones((n, n), dtype=bool), 1)
        for h in range(heads):
            q, k, v = query[a:b, h], key[a:b, h // group], value[a:b, h // group]
            scores = q @ k.T * scale
            scores[hidden] = -np.inf
            size[a:b, h] = np.where(hidden, 0, np.abs(q) @ np.abs(k).T * abs(scale)).max(1)
            weight = np.exp(scores - scores.max(1, keepdims=True))
            weight /= weight.sum(1, keepdims=True)
            want[a:b, h] = weight @ v
            mass[a:b, h] = weight @ np.abs(v)
    if gate is not None:
        share = 1 / (1 + np.exp(-gate))
        want, mass = want * share, mass * share
    return want, mass, size, first >= 0


def attention_of(query, key, value, at, scale):
    """attention() of one sequence, for its rows `at`: query holds those, key and value all rows"""
    heads, group = query.shape[1], query.shape[1] // key.shape[1]
    want, mass, size = np.empty(query.shape), np.empty(query.shape), np.empty(query.shape[:2])
    hidden = np.arange(len(key)) > np.asarray(at)[:, None]
    for h in range(heads):
        q, k, v = query[:, h], key[:, h // group], value[:, h // group]
        scores = np.where(hidden, -np.inf, q @ k.T * scale)
        size[:, h] = np.where(hidden, 0, np.abs(q) @ np.abs(k).T * abs(scale)).max(1)
        weight = np.exp(scores - scores.max(1, keepdims=True))
        weight /= weight.sum(1, keepdims=True)
        want[:, h], mass[:, h] = weight @ v, weight @ np.abs(v)
    return want, mass, size


def attention_bound(want, mass, size, dtype, longest):
    """Scores: exact products, fp32 sums of up to 256 terms (2^-24 of their sum
    each at most, 2^-24 * 32 in the mean), roundings of the scaling and of the difference to
    the maximum (2^-22); a score that is d off moves a weight by d of itself, in
    the sum and in the total.  Weights: exp2 2^-22; rounded to the rows' type,
    half a step, in the sum and the total alike (so no more than twice).  Sums
    of `longest` terms and their rescaling: 2^-24 sqrt(longest) in the mean,
    times 4.  Division and gate: 2^-21.  One rounding of the result."""
    score = size * (2.0 ** -22 + 2.0 ** -24 * 32)
    weight = 2.0 ** -22 + (HALF_STEP[dtype] if dtype != F32 else 0)
    sums = 2.0 ** -22 * np.sqrt(longest)
    return mass * (2 * score[..., None] + 2 * weight + 2 * sums + 2.0 ** -21) + rounding(want, dtype) * 1.01 + 1e-30
