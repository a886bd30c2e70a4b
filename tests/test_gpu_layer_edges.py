"""A decoder layer's operators on the GPU (q38hip.layer) at the edges: infinities, gates and scales of all sizes, sinks,
counts of sequences at which the kernels change, results in two forms at once."""
import numpy as np
import pytest
import torch

import kv_cases as kc
import layer_cases as lc
from layer_cases import BF16, F16, F32, TYPES, f64
from q38hip import layer

pytestmark = pytest.mark.gpu


def _normal(rng, *shape, dtype=F32, scale=1.0):
    return torch.from_numpy(rng.normal(size=shape) * scale).to(dtype).to("cuda")


# prompts by a wavefront to a row, by tiles, by tiles whose keys go in two parts (with 256-wide fp32 heads: whose columns four
# wavefronts share), by tiles that run over sequences
FORMS = {"rows": [50, 3], "tiles": [70] * 6, "long": [700], "many": [9, 30] * 40}


# ---- attention: values that are not finite ------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_infinite_values(device, form, dim, dtype):
    """A row that sees one infinite value in a channel has that infinity there, its own value among them, at every place of a group of
    sixteen; other channels and rows before it are as without."""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q, k, v = (_normal(rng, rows, h, dim, dtype=dtype) for h in (4, 2, 2))
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, dtype, max(lengths))
    infinite = np.zeros(want.shape)
    for a, b in zip(starts, starts[1:]):
        for i, row in enumerate(range(max(a, b - 20), b)):
            channel, sign = 3 * i + 1, 1 if i % 2 else -1
            v[row, 1, channel] = sign * np.inf
            infinite[row:b, 2:, channel] = sign
    got = f64(layer.attention(q, k, v, kc.words(starts, device)))
    assert np.array_equal(np.isinf(got) * np.sign(got), infinite)
    far = np.abs(got - want)[infinite == 0] / bound[infinite == 0]
    assert far.max() <= 1, "worst %g of its bound" % far.max()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_keys_that_are_not_numbers(device, form, dim, dtype):
    """rows that see such a key are NaN in all channels, others are as without"""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q, k, v = (_normal(rng, rows, h, dim, dtype=dtype) for h in (4, 2, 2))
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, dtype, max(lengths))
    for share in (0.0, 0.1, 0.6):
        k2, bad = k.clone(), np.zeros(want.shape, dtype=bool)
        for a, b in zip(starts, starts[1:]):
            row = a + int(share * (b - a))
            k2[row, 1, 3] = np.nan
            bad[row:b, 2:] = True
        got = f64(layer.attention(q, k2, v, kc.words(starts, device)))
        assert np.array_equal(np.isnan(got), bad)
        far = np.abs(got - want)[~bad] / bound[~bad]
        assert far.max() <= 1, "worst %g of its bound" % far.max()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_not_numbers(device, form, dim, dtype):
    """NaN and infinities among values at random places, next to each other and far apart: a channel of a row is NaN where it sees one
    NaN or two infinities of different signs, infinite where it sees infinities of one, and as without elsewhere"""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q, k, v = (_normal(rng, rows, h, dim, dtype=dtype) for h in (4, 2, 2))
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, dtype, max(lengths))
    for kinds in ((np.nan,), (np.inf, -np.inf), (np.nan, np.inf, -np.inf)):
        v2, seen = v.clone(), np.zeros((3,) + want.shape, dtype=bool)
        for a, b in zip(starts, starts[1:]):
            for row in rng.integers(a, b, size=4):
                channel, kind = int(rng.integers(dim // 2)), int(rng.integers(len(kinds)))
                v2[row, 1, channel] = kinds[kind]
        given = f64(v2)[:, 1]
        for a, b in zip(starts, starts[1:]):
            for i, found in enumerate((np.isnan(given[a:b]), given[a:b] == np.inf, given[a:b] == -np.inf)):
                seen[i, a:b, 2:] = np.logical_or.accumulate(found, 0)[:, None]
        nan = seen[0] | seen[1] & seen[2]
        got = f64(layer.attention(q, k, v2, kc.words(starts, device)))
        assert np.array_equal(np.isnan(got), nan)
        assert np.array_equal(got == np.inf, seen[1] & ~nan) and np.array_equal(got == -np.inf, seen[2] & ~nan)
        rest = ~seen.any(0)
        far = np.abs(got - want)[rest] / bound[rest]
        assert far.max() <= 1, "worst %g of its bound" % far.max()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[700], [300, 70, 260], [25, 90] * 33], ids=["two parts", "one part", "many"])
def test_sums_beyond_the_range_beside_a_nan(device, lengths, dim, dtype):
    """Values of 1e35 whose weights are up to 2^7 before they are divided: the sums of a tile leave fp32, the result does not.  A NaN in
    another channel, which all rows see, changes nothing.  Weights as in attention_bound, of terms that are all alike."""
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q, k = torch.zeros(rows, 2, dim, dtype=dtype, device=device), torch.zeros(rows, 1, dim, dtype=dtype, device=device)
    q[..., 0] = 1.0
    for a, b in zip(starts, starts[1:]):
        k[a + 16:b, 0, 0] = 4.5 * dim ** 0.5         # 2^6.5
    v = torch.full((rows, 1, dim), 1e35, dtype=dtype, device=device)
    v[starts[:-1], 0, 3] = float("nan")
    got = f64(layer.attention(q, k, v, kc.words(starts, device)))
    assert np.isnan(got[..., 3]).all()
    want, rest = float(v[1, 0, 0].double()), [c for c in range(dim) if c != 3]
    assert np.abs(got[..., rest] / want - 1).max() <= 2.0 ** -14 + (lc.HALF_STEP[BF16] if dtype == BF16 else 0)


# ---- gates of all sizes -----------------------------------------------------------------

GATES = [0.0, 1.0, -1.0, 20.0, -20.0, -40.0, 40.0, -60.0, -80.0, 87.0, -87.0, 87.5, -87.5, 88.0, -88.0, 89.0, -89.0, 90.0, -90.0, 95.0, -95.0, 100.0,
         -100.0, 103.0, -103.0, 104.0, -104.0, 1e4, -1e4, 5e4, -5e4, 1e9, -1e9, 1e30, -1e30, 3e38, -3e38, np.inf, -np.inf, np.nan]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_gates_of_all_sizes(device, form, dim, dtype):
    """Rows of a sequence have one value, a small whole number times a power of two, and keys of 0: weights are equal and sums exact, which
    leaves three roundings (the total's inverse, its product, the gate's) beside the sigmoid.  That is good to 2^-21, or to its
    smallest step where it is subnormal in fp32."""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    q = _normal(rng, starts[-1], 4, dim, dtype=dtype)
    k = torch.zeros(starts[-1], 2, dim, dtype=dtype, device=device)
    one = torch.from_numpy(rng.integers(1, 9, size=(len(lengths), 2, dim)) * np.exp2(rng.integers(-3, 4, size=(len(lengths), 2, dim))))
    v = one.repeat_interleave(torch.tensor(lengths), 0).to(dtype).to(device)
    at = torch.arange(starts[-1])[:, None, None] + torch.arange(4)[:, None] + torch.arange(dim)
    gate = torch.tensor(GATES, dtype=torch.float64)[at % len(GATES)].to(dtype)
    got = f64(layer.attention(q, k, v, kc.words(starts, device), gate=gate.to(device)))
    g, value = gate.double().numpy(), f64(v).repeat(2, 1)
    with np.errstate(over="ignore"):
        want = value / (1 + np.exp(-g))
    number = ~np.isnan(g)
    assert np.array_equal(np.isnan(got), ~number)
    bound = np.abs(want) * (2.0 ** -21 + 3 * 2.0 ** -24) + 2.0 ** -149 * (1 + value) + lc.rounding(want, dtype) * 1.01
    far = np.abs(got - want)[number] / bound[number]
    assert far.max() <= 1, "worst %g of its bound" % far.max()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("width", [1024, 1001])
def test_swiglu_of_far_gates(device, width, dtype):
    """Gates whose sigmoid leaves fp32's range and values that bring the product back into it, a block of 128 of each size; gates so
    far that nothing is left.  The error of e^-g: up to -80 its argument's two roundings (2^-18 each of an argument below 128, times
    ln 2), beyond that less."""
    rng = np.random.default_rng(width)
    sizes = np.array([-60.0, -80.0, -86.0, -88.0, -95.0, -104.0, -120.0, 100.0])
    gate = torch.from_numpy(np.repeat(sizes, 128)[:width] + rng.uniform(-0.9, 0.9, size=(3, width))).to(dtype).to(device)
    x = torch.from_numpy(rng.normal(size=(3, width)) * np.where(np.repeat(sizes, 128)[:width] < 0, 3e37, 1.0)).to(dtype).to(device)
    lc.check_quantized(layer.quantize(x, gate=gate), f64(x) * lc.silu(f64(gate)), 2.0 ** -17)
    for far in (-250.0, -1e4, -3e38):
        got = layer.quantize(x, gate=torch.full_like(gate, far))
        assert (got.codes.float() == 0).all() and (got.scales.view(torch.uint8)[:, :-(-width // 128)] == 27).all()
    got = layer.quantize(x, gate=torch.full_like(gate, -np.inf))
    assert (got.scales.view(torch.uint8)[:, :-(-width // 128)] == 255).all()


# ---- attention: keys far above the others --------------------------------------------------


def _step_bound(v, tokens, low):
    """What fp16 weights add beside half a step each: a step's weights (up to 64 keys) are off by up to 2^-20 of the step's
    largest one, which is 1 (relative to the row's largest) in the step that holds that key and `low` in the others."""
    return (64 + tokens * low) * 2.0 ** -20 * np.abs(v).max()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads,tokens", [(2, 1, 8192), (16, 4, 8192), (2, 2, 300)], ids=["two parts", "one part", "short"])
@pytest.mark.parametrize("gap", [10.0, 17.5, 21.0])
def test_sink(device, gap, heads, kv_heads, tokens, dim):
    """One key whose score is `gap` above all others' and whose value is 0, as the values of the 63 behind it: the thousands of small
    weights keep the bits of their type"""
    rng = np.random.default_rng(dim)
    q = torch.ones(tokens, heads, dim, dtype=F16, device=device)
    k = torch.zeros(tokens, kv_heads, dim, dtype=F16, device=device)
    k[0] = gap * dim ** -0.5
    v = (_normal(rng, tokens, kv_heads, dim) * 500 + 3000).to(F16)
    v[:64] = 0
    got = layer.attention(q, k, v, kc.words([0, tokens], device))
    at = np.array([0, 63, 64, 65, 100, 130, tokens // 2, tokens - 2, tokens - 1])
    want, mass, size = lc.attention_of(f64(q[at]), f64(k), f64(v), at, dim ** -0.5)
    lc.check(got[at], want, lc.attention_bound(want, mass, size, F16, tokens) + tokens * np.exp(-gap) * 2.0 ** -24 * f64(v).max())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lengths", [[1300], [200, 150, 310], [25, 90] * 33], ids=["two parts", "one part", "many"])
def test_scores_that_rise_and_fall(device, lengths, dim):
    """Steps of keys whose scores are 20 above or below the last step's, so what weights are relative to goes up and down.  Each
    step's weights are off by 2^-20 of its largest beside half a step of their own, and no step's largest is above the row's."""
    rng = np.random.default_rng(dim)
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q = _normal(rng, rows, 4, dim) * 0.3
    q[..., 0] = dim ** 0.5
    k, v = _normal(rng, rows, 2, dim) * 0.3, _normal(rng, rows, 2, dim)
    k[..., 0] = torch.from_numpy(np.repeat(rng.uniform(-20, 20, size=-(-rows // 32)), 32)[:rows, None]).to(device)
    q, k, v = q.to(F16), k.to(F16), v.to(F16)
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, F16, max(lengths)) + max(lengths) * 2.0 ** -20 * np.abs(f64(v)).max()
    lc.check(layer.attention(q, k, v, kc.words(starts, device)), want, bound)


def test_sink_within_a_step(device):
    """the small weights of the sink's own step of keys"""
    rng = np.random.default_rng(1)
    for dim in (64, 128, 256):
        lengths = [70] * 5
        starts = kc.offsets(lengths)
        q = torch.ones(350, 2, dim, dtype=F16, device=device)
        k = torch.zeros(350, 1, dim, dtype=F16, device=device)
        k[starts[:-1]] = 12.0 * dim ** -0.5
        v = (_normal(rng, 350, 1, dim) + 5).to(F16)
        v[starts[:-1]] = 0
        want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
        bound = lc.attention_bound(want, mass, size, F16, 70) + _step_bound(f64(v), 70, np.exp(-12))
        lc.check(layer.attention(q, k, v, kc.words(starts, device)), want, bound)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_equal_values_stay(device, form, dim, dtype):
    """Rows whose values are all equal give that value, whatever the weights: they are divided by the sum of what multiplies the
    values.  In fp32 sums of n weights and terms are off by 2^-24 sqrt(n) each in the mean, four times that at most, and the
    division and its product by two roundings; 16-bit results round that away."""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    q, k = _normal(rng, starts[-1], 4, dim, scale=3.0, dtype=dtype), _normal(rng, starts[-1], 2, dim, dtype=dtype)
    v = _normal(rng, len(lengths), 2, dim).repeat_interleave(torch.tensor(lengths, device=device), 0).to(dtype)
    got, want = f64(layer.attention(q, k, v, kc.words(starts, device))), f64(v).repeat(2, 1)
    bound = np.abs(want) * (8 * 2.0 ** -24 * np.sqrt(max(lengths)) + 2 * 2.0 ** -24) if dtype == F32 else np.zeros_like(want)
    assert (np.abs(got - want) <= bound).all(), "worst %g of the value" % (np.abs(got - want) / np.abs(want)).max()


# ---- product: what 16-bit outputs keep --------------------------------------------------------

# every tile size whole, cut along the inputs, and both; few tokens; rows that end inside a block
SIZES = [(1, 5120, 17), (4, 2048, 256), (9, 4112, 2050), (3, 17408, 2000), (9, 400, 33000), (33, 1024, 300), (48, 17408, 144), (65, 256, 513), (100, 1280, 1000),
         (128, 128, 128), (200, 2064, 260), (257, 896, 511), (300, 4096, 256), (66, 3600, 6050), (516, 912, 2210), (700, 528, 770), (1030, 768, 1030),
         (300, 80, 2600)]


def _half_step(want, dtype):
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(want), torch.finfo(dtype).smallest_normal)))) * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("tokens,inputs,outputs", SIZES)
def test_product_of_16_bit_outputs(device, tokens, inputs, outputs, dtype):
    """The error of all outputs together: 1e-4 of the result's norm, three times what the header states for such factors, and the
    rounding, whose square is a third of the half step's on average and, over n outputs, 8 / sqrt(n) more of it at most (its standard
    deviation is 0.9 / sqrt(n))."""
    rng = np.random.default_rng(tokens + inputs + outputs)
    rows8 = layer.quantize(_normal(rng, tokens, inputs) * torch.from_numpy(np.exp(0.7 * rng.normal(size=inputs))).float().to(device))
    weight = (_normal(rng, outputs, inputs) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.from_numpy(np.exp(rng.normal(size=(-(-outputs // 128), -(-inputs // 128)))) * 0.01).float().to(device)
    to_bytes = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
    want, _ = lc.product(to_bytes(rows8.codes), to_bytes(rows8.scales), to_bytes(weight), scales.cpu().numpy())
    want *= 2.0 ** -8                                # within fp16's range
    got = f64(layer.product(rows8, weight, scales * 2.0 ** -8, dtype))
    most = (1e-4 * np.linalg.norm(want)) ** 2 + (_half_step(want, dtype) ** 2).sum() / 3 * (1 + 8 / np.sqrt(want.size))
    assert ((got - want) ** 2).sum() <= most, "%g of its bound" % np.sqrt(((got - want) ** 2).sum() / most)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,inputs,outputs", SIZES)
def test_product_of_small_whole_numbers(device, tokens, inputs, outputs, dtype):
    """codes of -4 to 4, whose products span five bits, and scales that are powers of two: sums are exact, so every output is the exact
    one, rounded once"""
    rng = np.random.default_rng(tokens)
    blocks = -(-inputs // 128)
    codes = torch.from_numpy(rng.integers(-4, 5, size=(tokens, inputs))).float().to(torch.float8_e4m3fn).to(device)
    weight = torch.from_numpy(rng.integers(-4, 5, size=(outputs, inputs))).float().to(torch.float8_e4m3fn).to(device)
    scales = np.zeros((tokens, lc.pitch(inputs)), dtype=np.uint8)
    scales[:, :blocks] = rng.integers(125, 128, size=(tokens, blocks))
    factors = np.exp2(rng.integers(-2, 2, size=(-(-outputs // 128), blocks))).astype(np.float32)
    rows8 = (codes, torch.from_numpy(scales).to(device).view(torch.float8_e8m0fnu))
    to_bytes = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
    want, _ = lc.product(to_bytes(codes), scales, to_bytes(weight), factors)
    got = layer.product(rows8, weight, torch.from_numpy(factors).to(device), dtype)
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(dtype))


# ---- norm: rows of all sizes -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("width", [256, 2050, 8200, 24580])
def test_norm_of_rows_of_all_sizes(device, width, dtype):
    """rows whose inverse root leaves fp32's range, or is subnormal in it: the inverse rounded once, the weight's sum, two products"""
    rng = np.random.default_rng(width)
    sizes = np.array([1e-44, 1e-42, 1e-39, 1e-38, 1e-30, 1e30, 1e37, 1e38, 3.3e38])[0 if dtype == F32 else 2:]
    x = torch.from_numpy(rng.uniform(0.5, 1.0, size=(len(sizes), width)) * sizes[:, None] * rng.choice([-1.0, 1.0], size=(1, width)))
    x = x.to(dtype).to(device)
    weight = _normal(rng, width)
    want = lc.rms_norm(f64(x), f64(weight), 0.0, 0.0)
    bound = np.abs(want) * 5 * 2.0 ** -24 + lc.rounding(want, dtype) * 1.01
    lc.check(layer.rms_norm(x, weight, 0.0), want, bound)
    lc.check_quantized(layer.rms_norm(x, weight, 0.0, e4m3=True), want, 5 * 2.0 ** -24)
    assert torch.isnan(layer.rms_norm(torch.zeros_like(x), weight, 0.0)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 256), (3, 5120), (2, 2051), (2, 24584), (5, 30001)])
def test_norm_in_both_forms(device, rows, width, dtype):
    """the call that writes rows of the type and rows in 8 bits, in place too: what the calls that write one of them give"""
    rng = np.random.default_rng(width)
    x, addend, weight = _normal(rng, rows, width, dtype=dtype), _normal(rng, rows, width, dtype=dtype), _normal(rng, width)
    kind, stream = {F32: 0, F16: 1, BF16: 30}[dtype], torch.cuda.current_stream().cuda_stream
    plain, total = layer.rms_norm(x, weight, addend=addend)
    rows8 = layer.rms_norm(x, weight, addend=addend, e4m3=True)[0]
    for place in range(3):
        given, added = x.clone(), addend.clone()
        y, t = (torch.empty_like(x), added) if place == 0 else (given, torch.empty_like(x)) if place == 1 else (added, given)
        codes, scales = torch.empty_like(rows8.codes), torch.empty_like(rows8.scales)
        assert layer._lib().q38hip_rms_norm(y.data_ptr(), width, codes.data_ptr(), scales.data_ptr(), t.data_ptr(), width, given.data_ptr(), width,
                                            added.data_ptr(), width, kind, weight.data_ptr(), 0, 0.0, 1e-6, width, rows, stream)
        assert torch.equal(y, plain) and torch.equal(t, total)
        assert torch.equal(codes.view(torch.uint8), rows8.codes.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), rows8.scales.view(torch.uint8))


# ---- product: scales of all sizes ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("tokens,inputs", [(16, 384), (40, 384), (128, 384), (200, 656), (600, 656)])
def test_product_of_all_scales(device, tokens, inputs, dtype):
    """every scale byte, against matrix scales that bring the product back into fp32's range; NaN for 255"""
    rng = np.random.default_rng(tokens)
    blocks = -(-inputs // 128)
    finite = np.array([c for c in range(256) if c & 0x7f != 0x7f], dtype=np.uint8)
    codes, weight = finite[rng.integers(0, len(finite), size=(tokens, inputs))], finite[rng.integers(0, len(finite), size=(257, inputs))]
    to = lambda a, t: torch.from_numpy(a).to(device).view(t)  # noqa: E731
    for first in range(0, 256, tokens):
        scales = np.zeros((tokens, lc.pitch(inputs)), dtype=np.uint8)
        scales[:, :blocks] = ((first + np.arange(tokens)) % 256)[:, None]
        for power in (-100, -30, 30, 100):
            factors = np.full((3, blocks), 2.0 ** power, dtype=np.float32)
            # a block's largest sum times both scales within fp32's range, and its smallest
            e = scales[:, 0].astype(int) - 127
            inside = (e + power >= -126 + 18) & (e + power <= 127 - 27) & (scales[:, 0] != 255)
            # on the way to it: what is beyond 2^100 times the matrix's factor; for 16-bit outputs the sums times the tokens' alone
            inside &= np.abs(power + e - e.clip(-100, 100)) <= 126 if dtype == F32 else (e >= -126 + 18) & (e <= 127 - 27)
            got = layer.product((to(codes, torch.float8_e4m3fn), to(scales, torch.float8_e8m0fnu)), to(weight, torch.float8_e4m3fn),
                                torch.from_numpy(factors).to(device), dtype)
            assert torch.isnan(got[torch.from_numpy(scales[:, 0] == 255)]).all()
            if inside.any():
                want, mass = lc.product(codes[inside], scales[inside], weight, factors)
                lc.check(got[torch.from_numpy(inside)], want, lc.product_bound(want, mass, inputs, dtype))


# ---- rotary positions: the last bits -----------------------------------------------------------


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,dim,pairs,magnitude", [(7, 3, 256, 32, 1.0), (300, 2, 128, 64, 1.1386), (5000, 1, 80, 20, 1.25)])
def test_rotary_rounds_its_factors_once(device, rows, heads, dim, pairs, magnitude, interleaved):
    """Sine and cosine times the magnitude are rounded to fp32 once, from fp64; then two products and a sum."""
    rng = np.random.default_rng(rows)
    x = _normal(rng, rows, heads, dim)
    frequencies, _ = layer.rotary_frequencies(2 * pairs, 1e6, device=device)
    positions = rng.integers(0, 1 << 20, size=rows).astype(np.int32)
    want, size = lc.rotary(f64(x), positions, f64(frequencies), interleaved, np.float64(np.float32(magnitude)))
    bound = size * (2 * 2.0 ** -24 + 2 * np.pi * (1 << 20) / 6 * 2.0 ** -52) + lc.rounding(want, F32) * 1.01
    lc.check(layer.rotary(x, kc.words(positions, device), frequencies, interleaved, magnitude), want, bound)


# ---- attention: counts of sequences ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("count", [9, 32, 62, 63, 64, 65, 130])
def test_counts_of_sequences(device, count, dim, dtype):
    """short prompts, by rows and by tiles, empty ones among them, rows before the first and behind the last that none owns"""
    rng = np.random.default_rng(count)
    for most in (1, 40):
        lengths = rng.integers(0, most + 1, size=count)
        lengths[rng.integers(count)] = most
        starts = [2] + [2 + n for n in kc.offsets(lengths)[1:]]
        rows = starts[-1] + 3
        q, k, v = (_normal(rng, rows, h, dim, dtype=dtype) for h in (4, 2, 2))
        want, mass, size, owned = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
        out = torch.full_like(q, 7.0)
        layer.attention(q, k, v, kc.words(starts, device), out=out)
        lc.check(out[owned], want[owned], lc.attention_bound(want, mass, size, dtype, most)[owned])
        assert (out[~owned] == 7).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_long_sequences(device, dim, dtype):
    """more sequences than lanes, of a length at which keys go in two parts"""
    rng = np.random.default_rng(dim)
    lengths = [256 + int(n) for n in rng.integers(0, 9, size=66)]
    starts = kc.offsets(lengths)
    q, k, v = (_normal(rng, starts[-1], 1, dim, dtype=dtype) for _ in range(3))
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    lc.check(layer.attention(q, k, v, kc.words(starts, device)), want, lc.attention_bound(want, mass, size, dtype, max(lengths)))


@pytest.mark.parametrize("each", [21, 22], ids=["columns shared", "columns of a wavefront"])
def test_many_short_fp32_sequences(device, each):
    """100 prompts of 256-wide fp32 heads on both sides of the border between the two forms of tiles"""
    rng = np.random.default_rng(each)
    starts = kc.offsets([each] * 100)
    q, k, v = (_normal(rng, starts[-1], h, 256) for h in (24, 4, 4))
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, 1 / 16)
    lc.check(layer.attention(q, k, v, kc.words(starts, device)), want, lc.attention_bound(want, mass, size, F32, each))


# ---- attention: scales, hidden keys, offsets that change under a graph ---------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_scales_of_all_signs(device, form, dim, dtype):
    """negative, zero, so small that all weights are equal, and so large that one is all"""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    q, k, v = (_normal(rng, starts[-1], h, dim, dtype=dtype) for h in (4, 2, 2))
    for scale in (-dim ** -0.5, 0.0, 1e-42, -1e-30, 2.0):
        want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, scale)
        lc.check(layer.attention(q, k, v, kc.words(starts, device), scale=scale), want, lc.attention_bound(want, mass, size, dtype, max(lengths)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_keys_of_minus_infinity(device, form, dim, dtype):
    """keys whose scores are -infinity have no part; a row that sees nothing else is NaN"""
    rng = np.random.default_rng(dim)
    lengths = FORMS[form]
    starts = kc.offsets(lengths)
    rows = starts[-1]
    q, k, v = (_normal(rng, rows, h, dim, dtype=dtype) for h in (4, 2, 2))
    q[..., 0] = q[..., 0].abs() + 0.25
    hidden = rng.random(rows) < 0.3
    for a, b in zip(starts, starts[1:]):
        hidden[a:min(a + 3, b)] = True                   # the first rows see nothing
        hidden[a + 3:min(a + 4, b)] = False
    want, mass, size = np.full(q.shape, np.nan), np.full(q.shape, np.nan), np.zeros((rows, 4))
    query, key, value = f64(q), f64(k), f64(v)
    for a, b in zip(starts, starts[1:]):
        seen = ~hidden[a:b] & np.tri(b - a, dtype=bool)
        some = seen.any(1)
        for h in range(4):
            n, m, o = query[a:b, h], key[a:b, h // 2], value[a:b, h // 2]
            scores = np.where(seen, n @ m.T * dim ** -0.5, -np.inf)[some]
            weight = np.exp(scores - scores.max(1, keepdims=True))
            weight /= weight.sum(1, keepdims=True)
            want[a:b, h][some], mass[a:b, h][some] = weight @ o, weight @ np.abs(o)
            size[a:b, h] = np.where(seen, np.abs(n) @ np.abs(m).T * dim ** -0.5, 0).max(1)
    k[torch.from_numpy(np.flatnonzero(hidden)).to(device), :, 0] = -np.inf
    got = f64(layer.attention(q, k, v, kc.words(starts, device)))
    assert np.array_equal(np.isnan(got), np.isnan(want))
    far = np.abs(got - want) / lc.attention_bound(want, mass, size, dtype, max(lengths))
    assert np.nanmax(far) <= 1, "worst %g of its bound" % np.nanmax(far)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("count,rows", [(3, 40), (4, 700), (64, 600), (80, 900)])
def test_offsets_change_under_a_graph(device, count, rows, dtype):
    """a captured call reads the offsets when it is replayed"""
    rng = np.random.default_rng(count)
    q, k, v = (_normal(rng, rows, h, 128, dtype=dtype) for h in (4, 2, 2))
    words, out = torch.zeros(count + 1, dtype=torch.int32, device=device), torch.empty_like(q)
    side = torch.cuda.Stream(device=device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.attention(q, k, v, words, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.attention(q, k, v, words, out=out)
    for _ in range(4):
        starts = np.sort(rng.integers(0, rows + 1, size=count + 1))
        words.copy_(kc.words(starts.tolist(), device))
        out.fill_(7.0)
        graph.replay()
        want, mass, size, owned = lc.attention(f64(q), f64(k), f64(v), starts.tolist(), 128 ** -0.5)
        lc.check(out[owned], want[owned], lc.attention_bound(want, mass, size, dtype, rows)[owned])
        assert (out[~owned] == 7).all()


# ---- product: codes that are not numbers, in every type and tile ------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,inputs,outputs", [(3, 400, 40), (16, 80, 33000), (40, 400, 300), (128, 144, 8200), (300, 912, 5000), (520, 400, 513)])
def test_product_of_codes_that_are_not_numbers(device, tokens, inputs, outputs, dtype):
    """a NaN code of a token or of a matrix row, a NaN scale of either, an infinite scale: theirs are the only outputs that are not finite"""
    rng = np.random.default_rng(tokens)
    blocks = -(-inputs // 128)
    codes, weight = rng.integers(0x20, 0x50, size=(tokens, inputs)).astype(np.uint8), rng.integers(0x20, 0x50, size=(outputs, inputs)).astype(np.uint8)
    scales = np.zeros((tokens, lc.pitch(inputs)), dtype=np.uint8)
    scales[:, :blocks] = 120
    factors = np.full((-(-outputs // 128), blocks), 0.01, dtype=np.float32)
    for last in (False, True):                       # in the first block, and in the last, which may be part of one
        c, w, s, f = codes.copy(), weight.copy(), scales.copy(), factors.copy()
        at, block = (inputs - 1, blocks - 1) if last else (5, 0)
        c[1, at], w[outputs - 7, at], s[2, block] = 0x7f, 0xff, 255
        bad = np.zeros((tokens, outputs), dtype=bool)
        bad[1], bad[2], bad[:, outputs - 7] = True, True, True
        infinite = np.zeros_like(bad)
        if len(f) > 2:
            f[0, block], f[1, block] = np.nan, np.inf
            bad[:, :128], infinite[:, 128:256] = True, True
        to = lambda a, t: torch.from_numpy(a).to(device).view(t)  # noqa: E731
        got = f64(layer.product((to(c, torch.float8_e4m3fn), to(s, torch.float8_e8m0fnu)), to(w, torch.float8_e4m3fn),
                                torch.from_numpy(f).to(device), dtype))
        assert np.array_equal(np.isnan(got), bad) and np.array_equal(np.isinf(got), infinite & ~bad)


# ---- calls in other layouts ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 7, 300, 3000])
def test_heads_before_rows(device, rows, dtype):
    """queries (and gates) laid out [heads, rows, head_dim]: the same bits as [rows, heads, head_dim]"""
    rng = np.random.default_rng(rows)
    frequencies, positions = layer.rotary_frequencies(64, device=device)[0], torch.arange(rows, dtype=torch.int32, device=device)
    words = kc.words([0, rows // 3, rows], device)
    q, gate, k, v = (_normal(rng, rows, h, 128, dtype=dtype) for h in (4, 4, 2, 2))
    other = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    for interleaved in (False, True):
        want = layer.rotary(q, positions, frequencies, interleaved)
        assert torch.equal(layer.rotary(other(q), positions, frequencies, interleaved), want)
        turned = other(q)
        layer.rotary(turned, positions, frequencies, interleaved, out=turned)
        assert torch.equal(turned, want)
        into = other(torch.zeros_like(q))
        layer.rotary(q, positions, frequencies, interleaved, out=into)
        assert torch.equal(into, want)
    assert torch.equal(layer.attention(other(q), k, v, words, gate=other(gate)), layer.attention(q, k, v, words, gate=gate))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("width", [128, 1000, 24600])
def test_norm_weights_of_all_types(device, width, dtype):
    """weights of another type than the rows', at any element"""
    rng = np.random.default_rng(width)
    x = _normal(rng, 5, width, dtype=dtype)
    for kind in TYPES:
        weight = _normal(rng, width + 3, dtype=kind)
        for first in (0, 1, 3):
            part = weight[first:first + width]
            want = lc.rms_norm(f64(x), f64(part), 1e-6, 0.5)
            bound = np.abs(want) * 5 * 2.0 ** -24 + lc.rounding(want, dtype) * 1.01
            lc.check(layer.rms_norm(x, part, offset=0.5), want, bound)
            lc.check_quantized(layer.rms_norm(x, part, offset=0.5, e4m3=True), want, 5 * 2.0 ** -24)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 128), (3, 1001), (40, 5120), (2, 24600)])
def test_given_outputs(device, rows, width, dtype):
    """results into the caller's tensors, in wider rows, and in place: the same bits as into new ones"""
    rng = np.random.default_rng(width)
    x, addend, weight = _normal(rng, rows, width, dtype=dtype), _normal(rng, rows, width, dtype=dtype), _normal(rng, width)
    same = lambda a, b: torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and \
        torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))  # noqa: E731
    into = lambda: (torch.zeros(rows, width, dtype=torch.float8_e4m3fn, device=device),  # noqa: E731
                    torch.ones(rows, layer.scale_pitch(width), dtype=torch.float8_e8m0fnu, device=device))
    want = layer.quantize(x, gate=addend)
    given = into()
    got = layer.quantize(x, gate=addend, out=given)
    assert same(got, want) and got.codes is given[0] and got.scales is given[1]
    want, total = layer.rms_norm(x, weight, addend=addend, e4m3=True)
    room = torch.full((rows, width + 5), 3.0, dtype=dtype, device=device)
    got, summed = layer.rms_norm(x, weight, addend=addend, e4m3=True, out=into(), total=room[:, 2:width + 2])
    assert same(got, want) and torch.equal(summed, total) and (room[:, :2] == 3).all() and (room[:, width + 2:] == 3).all()
    want, total = layer.rms_norm(x, weight, addend=addend)
    room.fill_(3.0)
    got, summed = layer.rms_norm(x, weight, addend=addend, out=room[:, 1:width + 1])
    assert torch.equal(got, want) and torch.equal(summed, total) and (room[:, :1] == 3).all() and (room[:, width + 1:] == 3).all()
    for out, total_at in ((0, 1), (1, 0), (0, None), (1, None), (None, 0), (None, 1)):
        pair = (x.clone(), addend.clone())
        got, summed = layer.rms_norm(pair[0], weight, addend=pair[1], out=None if out is None else pair[out],
                                     total=None if total_at is None else pair[total_at])
        assert torch.equal(got, want) and torch.equal(summed, total)
    plain, alone = layer.rms_norm(x, weight), x.clone()
    assert layer.rms_norm(alone, weight, out=alone) is alone and torch.equal(alone, plain)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 5120, 37), (3, 17408, 2001), (40, 400, 301), (200, 912, 1001), (600, 528, 770)])
def test_product_into_rows_at_any_element(device, tokens, inputs, outputs, dtype):
    """outputs that begin at odd elements in rows of odd length, nothing beside them written"""
    rng = np.random.default_rng(tokens)
    rows8 = layer.quantize(_normal(rng, tokens, inputs))
    weight = (_normal(rng, outputs, inputs) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.full((-(-outputs // 128), -(-inputs // 128)), 1e-4, device=device)
    want = layer.product(rows8, weight, scales, dtype)
    for before, behind in ((1, 2), (3, 0), (0, 1)):
        room = torch.full((tokens, before + outputs + behind), 3.0, dtype=dtype, device=device)
        layer.product(rows8, weight, scales, out=room[:, before:before + outputs])
        assert torch.equal(room[:, before:before + outputs], want)
        room[:, before:before + outputs] = 3.0
        assert (room == 3).all()
