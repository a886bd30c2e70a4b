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
