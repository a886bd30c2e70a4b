"""A decoder layer's operators on the GPU (q38hip.layer) against plain models in
64 bits (tests/layer_cases.py)."""
import numpy as np
import pytest
import torch

import kv_cases as kc
import layer_cases as lc
from layer_cases import BF16, F16, F32, TYPES, f64
from q38hip import kv, layer

pytestmark = pytest.mark.gpu


def _normal(rng, *shape, dtype=F32, device="cuda", spread=0.0):
    x = rng.normal(size=shape) * np.exp(spread * rng.normal(size=shape[-1:]))
    return torch.from_numpy(x).to(dtype).to(device)


def _shifted(x):
    """the same values in a tensor whose rows start at odd elements"""
    room = torch.zeros(x.numel() + x.shape[0] + 1, dtype=x.dtype, device=x.device)
    out = room[1:].as_strided(x.shape, (x[0].numel() + 1,) + x.stride()[1:])
    out.copy_(x)
    return out


# ---- rows into 8 bits ------------------------------------------------------------

SIZES = [(1, 1), (1, 16), (3, 128), (2, 130), (5, 77), (4, 2048), (3, 2056), (1, 5120), (7, 2561), (2, 17408), (33, 640)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", SIZES)
def test_quantize(device, rows, width, dtype):
    rng = np.random.default_rng(rows * 100000 + width)
    x = _normal(rng, rows, width, dtype=dtype, spread=1.0)
    codes, scales = lc.quantize(f64(x))
    for given in (x, _shifted(x)):
        got = layer.quantize(given)
        assert np.array_equal(got.codes.view(torch.uint8).cpu().numpy(), codes)
        assert np.array_equal(got.scales.view(torch.uint8).cpu().numpy(), scales)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 16), (2, 130), (5, 77), (3, 2056), (2, 17408)])
def test_swiglu(device, rows, width, dtype):
    """e^-g with its argument rounded (2^-24 of |g| <= 12 and of its product with log2 e), exp2, sum, reciprocal and two products: 2^-19"""
    rng = np.random.default_rng(rows * 100000 + width)
    both = _normal(rng, rows, 2 * width, dtype=dtype) * 2
    want = f64(both[:, width:]) * lc.silu(f64(both[:, :width]))
    lc.check_quantized(layer.quantize(both[:, width:], gate=both[:, :width]), want, 2.0 ** -19)
    gate, x = _shifted(both[:, :width].contiguous()), both[:, width:].contiguous()
    lc.check_quantized(layer.quantize(x, gate=gate), want, 2.0 ** -19)


def test_quantize_extremes(device):
    """zeros, the borders between scales, the smallest and largest magnitudes, halves between codes, infinities and NaN"""
    rows = []
    for block in ([0.0], [448.0], [np.nextafter(np.float32(448), np.float32(500))], [447.0, 464.0], [1e-38, -3e-39], [1e-45],
                  [3.4e38, -1e38], [2.0 ** -92, 449 * 2.0 ** -100], [1.0, 17 / 16, 19 / 16, 21 / 16, -23 / 16, 25 / 16],
                  [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 5 * 2.0 ** -11, 2.0 ** -6 - 2.0 ** -10], [1e30, 1e-30], [-0.0, 7.0]):
        rows.append(np.resize(np.array(block, dtype=np.float32), 128))
    x = np.stack(rows)
    codes, scales = lc.quantize(x.astype(np.float64))
    got = layer.quantize(torch.from_numpy(x).to(device))
    assert np.array_equal(got.scales.view(torch.uint8).cpu().numpy(), scales)
    same = got.codes.view(torch.uint8).cpu().numpy() == codes
    assert same.all(), np.argwhere(~same)[:5]
    bad = np.ones((3, 300), dtype=np.float32)
    bad[0, 3], bad[1, 128], bad[2, 299] = np.nan, np.inf, -np.inf
    codes, scales = lc.quantize(bad.astype(np.float64))
    for dtype in TYPES:
        got = layer.quantize(torch.from_numpy(bad).to(dtype).to(device))
        assert np.array_equal(got.scales.view(torch.uint8).cpu().numpy(), scales)
        assert np.array_equal(got.codes.view(torch.uint8).cpu().numpy(), codes)
    big = torch.tensor([[0.0, 90.0, -90.0, 1e4, -1e4, 3.0] * 8], device=device)
    got = layer.quantize(torch.ones_like(big), gate=big)
    lc.check_quantized(got, lc.silu(f64(big).clip(-700, None)), 2.0 ** -16)


# ---- norm ------------------------------------------------------------------------


def _norm_relative():
    """the inverse root rounded once, the weight's sum, two products"""
    return 5 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", SIZES + [(2, 4104), (2, 8192), (3, 8200), (1, 16392), (2, 24577), (1, 30008)])
def test_rms_norm(device, rows, width, dtype):
    rng = np.random.default_rng(rows * 100000 + width)
    x, addend = _normal(rng, rows, width, dtype=dtype, spread=0.7) * 3, _normal(rng, rows, width, dtype=dtype)
    total = (x.float() + addend.float()).to(dtype)
    for weight, offset, eps in ((_normal(rng, width), 0.0, 1e-6), (_normal(rng, width, dtype=dtype), 1.0, 1e-2)):
        for shift in (False, True):
            given = [_shifted(t) if shift else t.clone() for t in (x, addend)]      # written in place below
            plain = lc.rms_norm(f64(x), f64(weight), eps, offset)
            got = layer.rms_norm(given[0], weight, eps, offset=offset)
            assert got.dtype == dtype
            lc.check(got, plain, np.abs(plain) * _norm_relative() + lc.rounding(plain, dtype) * 1.01)
            lc.check_quantized(layer.rms_norm(given[0], weight, eps, offset=offset, e4m3=True), plain, _norm_relative())
            want = lc.rms_norm(f64(total), f64(weight), eps, offset)
            got, summed = layer.rms_norm(given[0], weight, eps, addend=given[1], offset=offset)
            assert torch.equal(summed, total)
            lc.check(got, want, np.abs(want) * _norm_relative() + lc.rounding(want, dtype) * 1.01)
            got, summed = layer.rms_norm(given[0], weight, eps, addend=given[1], offset=offset, e4m3=True, total=given[0])
            assert summed is given[0] and torch.equal(summed, total)
            lc.check_quantized(got, want, _norm_relative())
            if shift:
                given[1].copy_(addend)
                got, summed = layer.rms_norm(x, weight, eps, addend=given[1], offset=offset, total=given[1])
                assert torch.equal(given[1], total)
                lc.check(got, want, np.abs(want) * _norm_relative() + lc.rounding(want, dtype) * 1.01)


def test_norm_extremes(device):
    """rows of zeros, squares beyond fp32's range on both sides, one value that is not finite: its row alone"""
    x = torch.ones(5, 256, device=device)
    x[0], x[1], x[2] = 0, 1e25, 1e-30
    x[3, 7] = np.inf
    weight = torch.full((256,), 2.0, device=device)
    got = f64(layer.rms_norm(x, weight, 1e-6))
    assert (got[0] == 0).all() and np.allclose(got[1], 2, rtol=1e-6) and np.allclose(got[4], 2, rtol=1e-5)
    assert np.allclose(got[2], 2e-27, rtol=1e-5) and np.isnan(got[3, 7])
    rows8 = layer.rms_norm(x, weight, 1e-6, e4m3=True)
    scales = rows8.scales.view(torch.uint8).cpu().numpy()
    assert scales[0, 0] == 27 and scales[3, 0] == 255 and scales[4, 0] == 127 + 1 - 8 and (scales[:, 2:] == 0).all()


# ---- product -----------------------------------------------------------------------

PRODUCTS = [(1, 16, 1), (1, 128, 16), (1, 5120, 17), (2, 144, 130), (3, 1168, 100), (16, 2048, 256), (9, 4112, 2050), (3, 17408, 2000), (17, 400, 128), (33, 1024, 300),
            (48, 17408, 144), (64, 640, 129), (65, 256, 513), (100, 1280, 1000), (128, 128, 128), (200, 2064, 260), (257, 896, 511),
            (300, 4096, 256), (512, 384, 1024), (700, 528, 770), (2100, 272, 6010), (1030, 768, 10300),
            # every tile size whole, cut along the inputs, and both
            (9, 400, 33000), (9, 1040, 33300), (17, 912, 33320), (66, 144, 17160), (199, 912, 17160), (66, 3600, 6050), (17, 912, 35340),
            (516, 912, 22210), (199, 6672, 10090),
            # rows shorter than a block, for every tile
            (16, 16, 40), (9, 112, 76000), (40, 16, 300), (150, 48, 520), (300, 80, 2600), (600, 96, 140), (4096, 112, 4100)]


def _factors(rng, tokens, inputs, outputs):
    rows8 = layer.quantize(_normal(rng, tokens, inputs, spread=0.7))
    weight = (_normal(rng, outputs, inputs) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.from_numpy(np.exp(rng.normal(size=(-(-outputs // 128), -(-inputs // 128))))).float().to("cuda") * 0.01
    return rows8, weight, scales


def _to_bytes(t):
    return t.view(torch.uint8)


def _bytes(t):
    return _to_bytes(t).cpu().numpy()


@pytest.mark.parametrize("tokens,inputs,outputs", PRODUCTS)
def test_product(device, tokens, inputs, outputs):
    rng = np.random.default_rng(tokens * 1000 + inputs + outputs)
    rows8, weight, scales = _factors(rng, tokens, inputs, outputs)
    want, mass = lc.product(_bytes(rows8.codes), _bytes(rows8.scales), _bytes(weight), scales.cpu().numpy())
    for dtype in TYPES:
        got = layer.product(rows8, weight, scales, dtype)
        assert got.dtype == dtype
        lc.check(got, want, lc.product_bound(want, mass, inputs, dtype))
    room = torch.full((tokens, outputs + 3), 7.0, device=device)
    layer.product(rows8, weight, scales, out=room[:, :outputs])
    assert torch.equal(room[:, :outputs], layer.product(rows8, weight, scales, F32)) and (room[:, outputs:] == 7).all()


@pytest.mark.parametrize("tokens,inputs,outputs", [(1, 640, 40), (40, 2048, 256), (300, 1040, 300), (600, 512, 512)])
def test_product_of_whole_numbers(device, tokens, inputs, outputs):
    """sums of small whole numbers are exact in fp32, whatever their order: every output is the exact one"""
    rng = np.random.default_rng(tokens)
    codes = torch.from_numpy(rng.integers(-8, 9, size=(tokens, inputs))).float().to(torch.float8_e4m3fn).to(device)
    weight = torch.from_numpy(rng.integers(-8, 9, size=(outputs, inputs))).float().to(torch.float8_e4m3fn).to(device)
    scales = np.zeros((tokens, lc.pitch(inputs)), dtype=np.uint8)
    blocks = -(-inputs // 128)
    scales[:, :blocks] = rng.integers(125, 130, size=(tokens, blocks))
    factors = np.exp2(rng.integers(-2, 3, size=(-(-outputs // 128), blocks))).astype(np.float32)
    rows8 = (codes, torch.from_numpy(scales).to(device).view(torch.float8_e8m0fnu))
    want, _ = lc.product(_bytes(codes), scales, _bytes(weight), factors)
    assert np.array_equal(f64(layer.product(rows8, weight, torch.from_numpy(factors).to(device), F32)), want)


@pytest.mark.parametrize("tokens", [5, 50, 300])
def test_product_extremes(device, tokens):
    """all 256 codes, the smallest and largest scales; NaN stays in its token's and its matrix row's outputs"""
    rng = np.random.default_rng(1)
    finite = np.array([c for c in range(256) if c & 0x7f != 0x7f], dtype=np.uint8)
    codes = finite[rng.integers(0, len(finite), size=(tokens, 512))]
    weight = finite[rng.integers(0, len(finite), size=(256, 512))]
    scales = rng.choice([27, 60, 127, 150, 180], size=(tokens, 4)).astype(np.uint8)
    scales[:] = scales[:, :1]
    factors = np.array([[1e-20, 2e-20, 1e-20, 3e-20], [1.0, 2.0, 0.0, 1.0]], dtype=np.float32)
    want, mass = lc.product(codes, scales, weight, factors)
    to = lambda a, t: torch.from_numpy(a).to(device).view(t)  # noqa: E731
    args = lambda: ((to(codes, torch.float8_e4m3fn), to(scales, torch.float8_e8m0fnu)), to(weight, torch.float8_e4m3fn),  # noqa: E731
                    torch.from_numpy(factors).to(device), F32)
    lc.check(layer.product(*args()), want, lc.product_bound(want, mass, 512, F32))
    codes[1, 500], weight[200, 3] = 0x7f, 0xff
    scales[2, 1] = 255
    got = f64(layer.product(*args()))
    bad = np.zeros(got.shape, dtype=bool)
    bad[1], bad[2], bad[:, 200] = True, True, True
    assert np.array_equal(np.isnan(got), bad)


def test_product_of_many_tokens(device):
    """more tiles of tokens than 16 bits count: each token's sums are its own, so parts of the batch give the same bits"""
    rng = np.random.default_rng(9)
    tokens, inputs, outputs = 65536 * 64 + 70, 32, 18
    codes = torch.randint(0, 0x78, (tokens, inputs), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    scales = torch.randint(120, 130, (tokens, 4), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
    _, weight, factors = _factors(rng, 1, inputs, outputs)
    got = layer.product((codes, scales), weight, factors)
    for first in range(0, tokens, 1 << 20):
        part = slice(first, min(first + (1 << 20), tokens))
        assert torch.equal(layer.product((codes[part], scales[part]), weight, factors), got[part])
    tail = slice(tokens - 5, tokens)
    want, mass = lc.product(_bytes(codes[tail]), _bytes(scales[tail]), _bytes(weight), factors.cpu().numpy())
    lc.check(got[tail], want, lc.product_bound(want, mass, inputs, BF16))


# ---- rotary positions ----------------------------------------------------------------

ROTARIES = [(1, 1, 64, 32), (3, 4, 256, 32), (5, 2, 80, 10), (2, 3, 96, 48), (70, 28, 256, 32), (4, 1, 7, 3), (2, 2, 1024, 512),
            (9, 40, 128, 64), (1, 16, 64, 31), (4100, 1, 80, 20), (3001, 2, 10, 5), (2500, 1, 256, 128)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,heads,dim,pairs", ROTARIES)
def test_rotary(device, rows, heads, dim, pairs, dtype):
    rng = np.random.default_rng(rows + heads + dim)
    x = _normal(rng, rows, heads, dim, dtype=dtype)
    frequencies, _ = layer.rotary_frequencies(2 * pairs, 1e6, device=device)
    positions = rng.integers(0, 1 << 20, size=rows).astype(np.int32)
    positions[:3] = [0, (1 << 31) - 1, -5][:len(positions[:3])]
    there = torch.from_numpy(positions).to(device)
    for interleaved, magnitude in ((False, 1.0), (True, 1.25)):
        want, size = lc.rotary(f64(x), positions, frequencies.double().cpu().numpy(), interleaved, magnitude)
        bound = lc.rotary_bound(want, size, float(1 << 31) / 6, dtype)
        got = layer.rotary(x, there, frequencies, interleaved, magnitude)
        lc.check(got, want, bound)
        assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])
        turned = x.clone()
        assert layer.rotary(turned, there, frequencies, interleaved, magnitude, out=turned) is turned
        assert torch.equal(turned, got)
        # heads inside wider rows, at an odd element; queries between gates
        wide = torch.full((rows, heads * 2 * dim + 5), 3.0, dtype=dtype, device=device)
        inside = wide[:, 3:3 + heads * 2 * dim].unflatten(1, (heads, 2 * dim))[:, :, :dim]
        inside.copy_(x)
        assert torch.equal(layer.rotary(inside, there, frequencies, interleaved, magnitude), got)
        layer.rotary(inside, there, frequencies, interleaved, magnitude, out=inside)
        assert torch.equal(inside, got)
        inside.fill_(3.0)
        assert (wide == 3).all()


# ---- attention of packed prompts ------------------------------------------------------

PROMPTS = [
    # heads, kv_heads, dim, lengths
    (1, 1, 64, [1]), (24, 4, 256, [37]), (4, 2, 128, [1, 2, 3, 1, 1]), (8, 2, 128, [63, 64, 65, 15, 16, 17, 31, 33]),
    (16, 16, 64, [130, 40]), (12, 1, 128, [300]), (5, 5, 256, [190]), (40, 8, 64, [90, 0, 200, 0, 0, 7]), (6, 2, 64, [1] * 70),
    (2, 1, 256, [129, 127, 128]), (12, 2, 256, [200, 150, 90, 10]), (6, 2, 64, [0, 33, 5, 1] * 18), (8, 2, 128, [2, 40, 0, 17, 90] * 14),
    (4, 1, 256, [25, 1, 70] * 22), (5, 5, 128, [300, 280]), (3, 3, 128, [257, 255]), (6, 1, 256, [513]), (2, 2, 64, [1030]), (7, 7, 128, [700, 1, 411]),
    (4, 2, 256, [0, 330, 1, 0, 33]), (6, 3, 256, [2, 0, 9, 17] * 30),
    (24, 4, 256, [1100, 700]), (3, 1, 256, [7, 50, 0, 120] * 20), (16, 8, 256, [400, 5, 1, 64, 32, 31]),
]


def _prompt(rng, heads, kv_heads, dim, rows, dtype):
    q = _normal(rng, rows, heads, dim, dtype=dtype) * 1.5
    k, v = _normal(rng, rows, kv_heads, dim, dtype=dtype), _normal(rng, rows, kv_heads, dim, dtype=dtype, spread=0.5)
    return q, k, v, _normal(rng, rows, heads, dim, dtype=dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,dim,lengths", PROMPTS, ids=lambda v: str(v)[:24])
def test_attention(device, heads, kv_heads, dim, lengths, dtype):
    rng = np.random.default_rng(heads * 1000 + dim + len(lengths))
    starts = kc.offsets(lengths)
    q, k, v, gate = _prompt(rng, heads, kv_heads, dim, starts[-1], dtype)
    words = kc.words(starts, device)
    for g in (None, gate):
        want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5, None if g is None else f64(g))
        bound = lc.attention_bound(want, mass, size, dtype, max(lengths))
        got = layer.attention(q, k, v, words, gate=g)
        lc.check(got, want, bound)
        lc.check(layer.attention(_shifted(q), _shifted(k), _shifted(v), words, gate=None if g is None else _shifted(g)), want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_attention_in_wider_rows(device, dtype):
    """queries between their gates, keys and values in one projection's rows, an output with room; rows before the first
    and behind the last sequence stay as they were; a scale of its own"""
    rng = np.random.default_rng(4)
    starts, rows, dim = [3, 40, 40, 109], 120, 128
    wide = _normal(rng, rows, 4 * 256 + 2 * 256 + 8, dtype=dtype)
    both = wide[:, :1024].unflatten(1, (4, 256))
    q, gate = both[:, :, :dim], both[:, :, dim:]
    k, v = wide[:, 1024:1280].unflatten(1, (2, dim)), wide[:, 1280:1536].unflatten(1, (2, dim))
    room = torch.full((rows, 4 * dim + 8), 5.0, dtype=dtype, device=device)
    out = room[:, :4 * dim].unflatten(1, (4, dim))
    assert layer.attention(q, k, v, kc.words(starts, device), gate=gate, scale=0.25, out=out) is out
    want, mass, size, owned = lc.attention(f64(q), f64(k), f64(v), starts, 0.25, f64(gate))
    bound = lc.attention_bound(want, mass, size, dtype, 69)
    lc.check(out[owned], want[owned], bound[owned])
    out[owned] = 5.0
    assert (room == 5).all() and not owned[:3].any() and not owned[109:].any()


def _hidden(device, lengths, dim, dtype, at, where, bad):
    """sequence `at` has a value of its own at row `where` that is not finite: rows before it and other sequences are as without"""
    rng = np.random.default_rng(dim + len(lengths))
    starts = kc.offsets(lengths)
    q, k, v, _ = _prompt(rng, 4, 2, dim, starts[-1], dtype)
    words = kc.words(starts, device)
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, dtype, max(lengths))
    lc.check(layer.attention(q, k, v, words), want, bound)
    row, end = starts[at] + where, starts[at + 1]
    v[row, 1, 5] = bad
    got = layer.attention(q, k, v, words)
    keep = [c for c in range(dim) if c != 5]
    for part in (np.s_[:row], np.s_[row:end, :2], np.s_[row:end, 2:, keep], np.s_[end:]):
        lc.check(got[part], want[part], bound[part])
    assert not torch.isfinite(got[row:end, 2:, 5]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("lengths,at,where", [([700], 0, 430), ([280, 290], 1, 3), ([9, 30] * 40, 13, 7)], ids=["one", "two", "eighty"])
def test_attention_hidden_values(device, lengths, at, where, dtype):
    """one prompt whose keys go in parts, two, and more sequences than lanes"""
    for dim, bad in ((64, np.nan), (128, np.inf), (256, -np.inf)):
        _hidden(device, lengths, dim, dtype, at, where, bad)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("rows,count", [(40, 3), (300, 3), (300, 90)])
def test_attention_bad_offsets_stay_inside(device, rows, count, dtype):
    """Offsets that decrease, negative ones and ones behind the rows: what is written is the call's own output, nothing around it."""
    rng = np.random.default_rng(rows + count)
    q, k, v, _ = _prompt(rng, 4, 2, 64, rows, dtype)
    room = torch.full((rows + 2, 4, 64), 3.0, dtype=dtype, device=device)
    for _ in range(4):
        starts = rng.integers(-2 * rows, 3 * rows, size=count + 1)
        layer.attention(q, k, v, kc.words(starts.tolist(), device), out=room[1:-1])
        torch.cuda.synchronize()
        assert (room[0] == 3).all() and (room[-1] == 3).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_hidden_rows_have_no_part(device, dim, dtype):
    """Infinities and NaN in later rows and in other sequences have no part: rows that see none are what they are without, within
    the bound (they may be summed in another order).  A row that sees one is NaN or infinite.  Scores of the type's lowest value."""
    rng = np.random.default_rng(dim)
    lengths = [50, 100, 45, 3]
    starts = kc.offsets(lengths)
    q, k, v, _ = _prompt(rng, 4, 2, dim, starts[-1], dtype)
    words = kc.words(starts, device)
    want, mass, size, _ = lc.attention(f64(q), f64(k), f64(v), starts, dim ** -0.5)
    bound = lc.attention_bound(want, mass, size, dtype, 100)
    lc.check(layer.attention(q, k, v, words), want, bound)
    for bad in (np.nan, np.inf, -np.inf):
        k2, v2 = k.clone(), v.clone()
        v2[60, 1, 5], v2[150:, 0], k2[145:147, :] = bad, bad, np.nan
        got = layer.attention(q, k2, v2, words)
        keep = [c for c in range(dim) if c != 5]
        for part in (np.s_[:60], np.s_[60:145, :2], np.s_[60:145, 2:, keep], np.s_[150:, 2:]):
            lc.check(got[part], want[part], bound[part])
        assert not torch.isfinite(got[60:145, 2:, 5]).any() and torch.isnan(got[145:150]).all()
        assert not torch.isfinite(got[150:, :2]).any()
    # One key far above the others: its value alone; keys far below: no part.  Its score times log2 e, at most 925, is rounded
    # (2^-24 of it), so its weight is 1 + 2^-14 at most, which the rows' type may round away while the total keeps it.
    k3 = torch.zeros_like(k)
    q3 = torch.ones_like(q)
    k3[10] = 40.0
    k3[55:70] = torch.finfo(dtype).min / (2 * dim)
    got = layer.attention(q3, k3, v, words)
    alone = np.broadcast_to(f64(v[10].repeat_interleave(2, 0)), (40, 4, dim))
    lc.check(got[10:50], alone, np.abs(alone) * (2.0 ** -22 if dtype == F32 else 2.0 ** -14) + lc.rounding(alone, dtype) * 1.01)
    want, mass, size, _ = lc.attention(f64(q3), f64(k3), f64(v), starts, dim ** -0.5)
    size = np.minimum(size, 500.0)              # of the rows whose weights are not all or nothing
    lc.check(got[70:], want[70:], lc.attention_bound(want, mass, size, dtype, 100)[70:])


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 2, 64, BF16), (2, 1, 128, torch.float16), (3, 1, 256, BF16), (1, 1, 128, F32), (2, 1, 256, F32)], ids=str)
def test_attention_of_a_long_prompt(device, heads, kv_heads, dim, dtype):
    """33001 tokens behind a short prompt, at rows near tile ends and spread over it"""
    rng = np.random.default_rng(dim)
    starts, n = [0, 19, 33020], 33001
    q, k, v, _ = _prompt(rng, heads, kv_heads, dim, 33020, dtype)
    got = layer.attention(q, k, v, kc.words(starts, device))
    at = np.array([0, 1, 31, 32, 33, 63, 64, 127, 128, 4095, 4096, 16383, 16384, 32767, 32768, 33000] + list(rng.integers(0, n, size=16)))
    rows = torch.from_numpy(at + 19).to(device)
    want, mass, size = lc.attention_of(f64(q[rows]), f64(k[19:]), f64(v[19:]), at, dim ** -0.5)
    lc.check(got[rows], want, lc.attention_bound(want, mass, size, dtype, n))


# ---- far rows ---------------------------------------------------------------------------


def test_offsets_beyond_32_bits(device):
    """rows whose places pass 2^32 bytes"""
    rng = np.random.default_rng(8)
    rows, stride = 140, 1 << 25
    big = torch.empty(rows * stride, dtype=BF16, device=device)
    wide = big.as_strided((rows, 768), (stride, 1))
    near = _normal(rng, rows, 768, dtype=BF16)
    wide.copy_(near)
    got, want = layer.quantize(wide[:, :512], gate=wide[:, 256:]), layer.quantize(near[:, :512], gate=near[:, 256:])
    assert all(torch.equal(_to_bytes(a), _to_bytes(b)) for a, b in zip(got, want))
    weight = _normal(rng, 512)
    assert torch.equal(layer.rms_norm(wide[:, :512], weight), layer.rms_norm(near[:, :512].contiguous(), weight))
    heads = lambda x: (x[:, :512].unflatten(1, (8, 64)), x[:, 512:640].unflatten(1, (2, 64)), x[:, 640:].unflatten(1, (2, 64)))  # noqa: E731
    positions, frequencies = torch.arange(rows, dtype=torch.int32, device=device), layer.rotary_frequencies(64, device=device)[0]
    assert torch.equal(layer.rotary(heads(wide)[0], positions, frequencies), layer.rotary(heads(near)[0], positions, frequencies))
    words = kc.words([0, 100, 140], device)
    assert torch.equal(layer.attention(*heads(wide), words), layer.attention(*heads(near), words))
    layer.attention(*heads(near), words, out=heads(wide)[0])
    assert torch.equal(heads(wide)[0], layer.attention(*heads(near), words))
    del big, wide
    tokens, inputs = 900000, 5120
    codes = torch.zeros(tokens, inputs, dtype=torch.uint8, device=device)
    scales = torch.zeros(tokens, layer.scale_pitch(inputs), dtype=torch.uint8, device=device)
    last, matrix, factors = _factors(rng, 300, inputs, 24)
    codes[-300:], scales[-300:] = last.codes.view(torch.uint8), last.scales.view(torch.uint8)
    got = layer.product((codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)), matrix, factors, F32)
    want, mass = lc.product(_bytes(last.codes), _bytes(last.scales), _bytes(matrix), factors.cpu().numpy())
    lc.check(got[-300:], want, lc.product_bound(want, mass, inputs, F32))
    assert (got[:-300] == 0).all()


# ---- as programs use them -------------------------------------------------------------


class _Layer:
    """One decoder layer over a packed prompt, and over one new token of each sequence."""

    def __init__(self, rng, device):
        self.hidden, self.heads, self.kv_heads, self.dim, self.middle = 512, 8, 2, 64, 768
        wide = (self.heads * 2 + self.kv_heads * 2) * self.dim
        self.norms = [1 + 0.1 * _normal(rng, self.hidden) for _ in range(2)]
        self.weights = [_factors(rng, 1, i, o)[1:] for i, o in
                        ((self.hidden, wide), (self.heads * self.dim, self.hidden), (self.hidden, 2 * self.middle),
                         (self.middle, self.hidden))]
        for _, scales in self.weights:
            scales.mul_(0.02)
        self.frequencies, self.magnitude = layer.rotary_frequencies(32, 1e4, factor=4.0, original=2048, device=device)

    def __call__(self, x, attended_before, positions, attend):
        """x [rows, hidden] and the layer before's output; returns the sum and this layer's output"""
        rows, qd, kd = x.shape[0], self.heads * self.dim, self.kv_heads * self.dim
        y, x = layer.rms_norm(x, self.norms[0], addend=attended_before, e4m3=True)
        p = layer.product(y, *self.weights[0], dtype=x.dtype)
        q, gate = p[:, :2 * qd].view(rows, self.heads, 2 * self.dim).split(self.dim, 2)
        k, v = p[:, 2 * qd:2 * qd + kd].unflatten(1, (self.kv_heads, -1)), p[:, 2 * qd + kd:].unflatten(1, (self.kv_heads, -1))
        for part in (q, k):
            layer.rotary(part, positions, self.frequencies, magnitude=self.magnitude, out=part)
        out = attend(q, k, v, gate)
        y = layer.quantize(out.view(rows, qd))
        y, x = layer.rms_norm(x, self.norms[1], addend=layer.product(y, *self.weights[1], dtype=x.dtype), e4m3=True)
        p = layer.product(y, *self.weights[2], dtype=x.dtype)
        return x, layer.product(layer.quantize(p[:, self.middle:], gate=p[:, :self.middle]), *self.weights[3], dtype=x.dtype)

    def plain(self, x, attended_before, positions, starts):
        """the same in float64, with each operator's rounding of its results"""
        t = x.dtype
        near = lambda a: f64(torch.from_numpy(a).float().to(t))  # noqa: E731
        times = lambda y, w: near(lc.product(*lc.quantize(y), _bytes(w[0]), w[1].cpu().numpy())[0])  # noqa: E731
        rows, qd, kd = x.shape[0], self.heads * self.dim, self.kv_heads * self.dim
        x = near(f64(x) + f64(attended_before))
        p = times(lc.rms_norm(x, f64(self.norms[0]), 1e-6, 0.0), self.weights[0])
        q, gate = np.split(p[:, :2 * qd].reshape(rows, self.heads, -1), 2, axis=2)
        k, v = p[:, 2 * qd:2 * qd + kd].reshape(rows, self.kv_heads, -1), p[:, 2 * qd + kd:].reshape(rows, self.kv_heads, -1)
        turn = lambda a: near(lc.rotary(a, positions, f64(self.frequencies), False, self.magnitude)[0])  # noqa: E731
        out = near(lc.attention(turn(q), turn(k), v, starts, self.dim ** -0.5, gate)[0])
        x = near(x + times(out.reshape(rows, qd), self.weights[1]))
        p = times(lc.rms_norm(x, f64(self.norms[1]), 1e-6, 0.0), self.weights[2])
        return x, times(p[:, self.middle:] * lc.silu(p[:, :self.middle]), self.weights[3])


def test_layer_over_a_packed_prompt_and_a_token(device):
    """All operators in a row, with the paged cache: a packed prompt that also goes into the cache, then one new token of each
    sequence over the cache.  A relative error e in front of a rounding to 8 bits, whose steps are about 0.09 of a value, moves
    e / 0.09 of the values by a step: it comes out as sqrt(0.09 e) of the norm.  The first product's matrix unit and its outputs'
    rounding leave 6e-4 in the attention's result, so 0.7 % of its 8-bit form, half of that beside the residual, 2 % of the second
    norm's 8-bit form, 3 % of the SwiGLU, 5 % of its 8-bit form: results agree to 1 % (the sum) and 6 % (the layer's output).  The
    cache's keys and values are in 8 bits, good to 1 %: 3 % and, with e at the step's own size, 9 %."""
    rng = np.random.default_rng(11)
    block = _Layer(rng, device)
    lengths = [37, 1, 90]
    starts = kc.offsets(lengths)
    words, ids = kc.words(starts, device), kc.words([0, 1, 2], device)
    x, before = _normal(rng, 128, 512, dtype=BF16), _normal(rng, 128, 512, dtype=BF16)
    positions = np.concatenate([np.arange(n) for n in lengths]).astype(np.int32)
    cache = kv.KVPages.allocate(layers=1, pages=32, page_tokens=16, kv_heads=2, head_dim=64, sequences=3, table_entries=8)
    cache.extend(ids, kc.words(lengths, device))

    def attend(q, k, v, gate):
        cache.append(0, k, v, ids, words)
        return layer.attention(q, k, v, words, gate=gate)

    got = block(x, before, torch.from_numpy(positions).to(device), attend)
    want = block.plain(x, before, positions, starts)
    for g, w, most in zip(got, want, (0.01, 0.06)):
        assert np.linalg.norm(f64(g) - w) <= most * np.linalg.norm(w)

    # one new token each: the cache holds keys and values in 8 bits, so to a few hundredths of the whole prompt's rows
    new = [38, 2, 91]
    where = np.cumsum(new) - 1
    x2, before2 = _normal(rng, 3, 512, dtype=BF16), _normal(rng, 3, 512, dtype=BF16)
    full = [torch.cat([t for i in range(3) for t in (a[starts[i]:starts[i + 1]], b[i:i + 1])]) for a, b in ((x, x2), (before, before2))]
    positions2 = np.concatenate([np.arange(n) for n in new]).astype(np.int32)
    want = block.plain(*full, positions2, kc.offsets(new))
    cache.extend(ids, kc.words([1, 1, 1], device))

    def step(q, k, v, gate):
        cache.append(0, k, v, ids)
        return cache.attention(0, q, ids, gate=gate)

    got = block(x2, before2, kc.words(lengths, device), step)
    cache.check()
    for g, w, most in zip(got, want, (0.03, 0.09)):
        assert np.linalg.norm(f64(g) - w[where]) <= most * np.linalg.norm(w[where])


def test_streams_and_graphs(device):
    """calls on two streams at once, and captured ones replayed with other inputs between eager calls"""
    rng = np.random.default_rng(12)
    block = _Layer(rng, device)
    words = kc.words([0, 30, 64], device)
    positions = torch.arange(64, dtype=torch.int32, device=device)
    attend = lambda q, k, v, gate: layer.attention(q, k, v, words, gate=gate)  # noqa: E731
    inputs = [(_normal(rng, 64, 512, dtype=BF16), _normal(rng, 64, 512, dtype=BF16)) for _ in range(4)]
    want = [block(*i, positions, attend) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=device) for _ in range(2)]
    got = {}
    for i, pair in enumerate(inputs):
        with torch.cuda.stream(streams[i % 2]):
            got[i] = block(*pair, positions, attend)
    torch.cuda.synchronize()
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
    x, before = (t.clone() for t in inputs[0])
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream(device=device)
    with torch.cuda.stream(side):
        block(x, before, positions, attend)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = block(x, before, positions, attend)
    for i in (1, 2, 3, 1):
        x.copy_(inputs[i][0])
        before.copy_(inputs[i][1])
        graph.replay()
        eager = block(*inputs[i], positions, attend)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(out, eager, want[i]))


def test_python_refuses(device):
    x, weight = torch.zeros(3, 256, device=device), torch.ones(256, device=device)
    rows8 = layer.quantize(x)
    w8, ws = rows8.codes[:2].contiguous(), torch.ones(1, 2, device=device)
    heads, words = torch.zeros(3, 4, 64, device=device), torch.zeros(3, dtype=torch.int32, device=device)
    f = torch.ones(8, device=device)
    for call in (lambda: layer.quantize(x, gate=x.half()), lambda: layer.quantize(x, gate=x[:2]), lambda: layer.quantize(x, gate=x.cpu()),
                 lambda: layer.quantize(x, out=(rows8.codes[:2], rows8.scales)), lambda: layer.quantize(x.double()),
                 lambda: layer.rms_norm(x, weight[:255]), lambda: layer.rms_norm(x, weight.cpu()), lambda: layer.rms_norm(x, weight, total=x),
                 lambda: layer.rms_norm(x, weight, addend=x[:, :255]), lambda: layer.rms_norm(x, weight, out=x.half()),
                 lambda: layer.rms_norm(x, weight, e4m3=True, out=(rows8.codes, rows8.scales[:2])),
                 lambda: layer.product(rows8, w8, ws[:, :1]), lambda: layer.product(rows8, w8.float(), ws), lambda: layer.product(rows8, w8, ws.half()),
                 lambda: layer.product((rows8.codes.view(torch.uint8), rows8.scales), w8, ws), lambda: layer.product(rows8, w8, ws, torch.float64),
                 lambda: layer.product(rows8, w8, ws, out=torch.zeros(3, 3, device=device)),
                 lambda: layer.product((rows8.codes, rows8.scales[:, :2]), w8, ws),
                 lambda: layer.rotary(heads, words[:2], f), lambda: layer.rotary(heads, words.long(), f), lambda: layer.rotary(heads, words, f.double()),
                 lambda: layer.rotary(heads, words, f, out=heads[:2]), lambda: layer.rotary(heads, words, f.cpu()),
                 lambda: layer.attention(heads, heads[:2], heads, words), lambda: layer.attention(heads, heads, heads.half(), words),
                 lambda: layer.attention(heads, heads, heads, words.long()), lambda: layer.attention(heads, heads, heads, words[:1]),
                 lambda: layer.attention(heads, heads, heads, words, gate=heads.half()),
                 lambda: layer.attention(heads, heads, heads, words, out=heads[:, :2])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: layer.rotary(heads, words, torch.ones(33, device=device)), lambda: layer.attention(heads, heads[:, :3], heads[:, :3], words),
                 lambda: layer.quantize(x[:1].expand(3, 256)),
                 lambda: layer.product((rows8.codes[:, :120].contiguous(), rows8.scales), w8[:, :120].contiguous(), ws[:, :1].contiguous()),
                 lambda: layer.rms_norm(x, weight, eps=-1.0), lambda: layer.quantize(x[:0]), lambda: layer.rms_norm(x[:0], weight),
                 lambda: layer.product(layer.E4M3Rows(rows8.codes[:0], rows8.scales[:0]), w8, ws), lambda: layer.rotary(heads[:0], words[:0], f),
                 lambda: layer.attention(heads[:0], heads[:0], heads[:0], words), lambda: layer.attention(heads, heads, heads, words, out=heads)):
        with pytest.raises(RuntimeError):
            call()
