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
