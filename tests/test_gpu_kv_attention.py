"""Attention over the paged 8-bit cache on the GPU (q38hip_kv_attention) against
the plain model in 64 bits (tests/kv_cases.py)."""
import numpy as np
import pytest
import torch

import kv_cases as kc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    # heads, kv_heads, dim, page, kind, type, lengths, rows
    (24, 4, 256, 16, "int8", F32, [1], [1]),
    (24, 4, 256, 64, "int8", F32, [65], [1]),
    (24, 4, 256, 64, "e4m3", F32, [700], [4]),
    (24, 4, 256, 128, "e4m3", BF16, [129, 64, 1], [1, 1, 1]),
    (24, 4, 256, 32, "int8", F16, [300, 2], [8, 2]),
    (8, 2, 128, 32, "e4m3", BF16, [63, 64, 65, 15, 16, 17, 1, 513], [1] * 8),
    (8, 2, 128, 16, "int8", F32, [63, 64, 65, 15, 16, 17, 1, 513], [1] * 8),
    (32, 8, 128, 128, "int8", BF16, [257], [3]),
    (16, 16, 64, 16, "e4m3", F16, [130, 40], [33, 40]),
    (40, 8, 64, 64, "int8", F32, [90, 7, 200], [20, 7, 1]),
    (12, 1, 128, 32, "e4m3", F32, [500], [70]),
    (5, 5, 256, 64, "int8", BF16, [190], [130]),
    (24, 4, 256, 64, "e4m3", F32, [150], [150]),
    (24, 4, 256, 64, "int8", BF16, [1100], [40]),
    (64, 1, 64, 16, "int8", F16, [33, 5], [1, 5]),
    (3, 3, 128, 128, "int8", F32, [0, 5, 0, 129], [1, 9, 3, 1]),      # rows that see nothing
    (6, 2, 64, 32, "e4m3", BF16, [10] * 70, [1, 2] * 35),             # more sequences than a wavefront
    (2, 1, 256, 16, "e4m3", F32, [6001], [2]),
]


def _case(rng, heads, kv_heads, dim, page, kind, dtype, lengths, rows, device):
    cache = kc.filled(rng, lengths, kind, page, kv_heads, dim)
    starts = kc.offsets(rows)
    q = torch.from_numpy(rng.normal(size=(starts[-1], heads, dim)) * 1.5).to(dtype)
    gate = torch.from_numpy(rng.normal(size=(starts[-1], heads, dim))).to(dtype)
    return cache, starts, q.to(device), gate.to(device)


def _compare(got, want, mass, size, dtype, longest):
    got = got.double().cpu().numpy()
    far = np.abs(got - want)
    bound = kc.tolerance(want, mass, size, dtype, longest)
    assert np.isfinite(got).all()
    assert (far <= bound).all(), "worst %g of its bound" % (far / bound).max()


@pytest.mark.parametrize("case", CASES, ids=lambda c: "%dx%dx%d-p%d-%s-%s-%s" % (c[0], c[1], c[2], c[3], c[4],
                                                                                 str(c[5])[6:], len(c[6])))
def test_attention(device, case):
    heads, kv_heads, dim, page, kind, dtype, lengths, rows = case
    rng = np.random.default_rng(len(lengths) * 1000 + heads + dim + page)
    cache, starts, q, gate = _case(rng, *case, device)
    ids = kc.words(range(len(lengths)), device)
    dev = cache.to(device)
    q64, g64 = q.double().cpu().numpy(), gate.double().cpu().numpy()
    for g in (None, gate):
        got = dev.attention(0, q, ids, kc.words(starts, device), gate=g)
        want, mass, size = cache.attention(0, q64, range(len(lengths)), starts, dim ** -0.5, None if g is None else g64)
        _compare(got, want, mass, size, dtype, max(lengths))
    if len(set(rows)) == 1:                       # equal rows need no offsets
        assert torch.equal(dev.attention(0, q, ids, gate=gate), got)
    dev.check()


@pytest.mark.parametrize("kind,dtype", [("int8", F32), ("e4m3", BF16)])
def test_strides_and_alignment(device, kind, dtype):
    """queries and gates interleaved as the engine's projection leaves them, rows
    that start at odd elements, an output with room between its rows"""
    rng = np.random.default_rng(5)
    cache = kc.filled(rng, [77, 130], kind, 32, 4, 256)
    dev, ids, starts = cache.to(device), kc.words([1, 0], device), [0, 2, 5]
    for pad, gap in ((0, 0), (3, 7)):
        wide = torch.from_numpy(rng.normal(size=(5, 24 * 512 + 2048 + pad))).to(dtype).to(device)
        both = wide[:, pad:pad + 24 * 512].unflatten(1, (24, 512))
        q, gate = both[:, :, :256], both[:, :, 256:]
        room = torch.full((5, 24 * 256 + gap), 7.0, dtype=dtype, device=device)
        out = room[:, :24 * 256].unflatten(1, (24, 256))
        got = dev.attention(0, q, ids, kc.words(starts, device), gate=gate, scale=0.05, out=out)
        assert got.data_ptr() == out.data_ptr()
        want, mass, size = cache.attention(0, q.double().cpu().numpy(), [1, 0], starts, 0.05, gate.double().cpu().numpy())
        _compare(got, want, mass, size, dtype, 130)
        assert (room[:, 24 * 256:] == 7.0).all()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_pages_that_are_not_numbers(device, kind):
    """a NaN page reaches the rows that see it, and no other"""
    rng = np.random.default_rng(6)
    cache = kc.filled(rng, [200], kind, 16, 1, 64)
    cache.scales[0, cache.tables[0, 11], 1] = np.nan          # values of tokens 176 .. 191
    starts, rows = [0, 40], 40
    q = torch.from_numpy(rng.normal(size=(rows, 2, 64))).float().to(device)
    got = cache.to(device).attention(0, q, kc.words([0], device), kc.words(starts, device)).double().cpu().numpy()
    want, _, _ = cache.attention(0, q.double().cpu().numpy(), [0], starts, 0.125)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(got[16:]).all() and np.isfinite(got[:16]).all()
    assert np.abs(got[:16] - want[:16]).max() < 1e-5


def test_large_and_small_scales(device):
    """value pages 2^60 apart, peaked and flat scores, queries of very different sizes"""
    rng = np.random.default_rng(7)
    cache = kc.filled(rng, [300], "int8", 16, 2, 64)
    for entry in range(cache.pages(300)):
        cache.scales[0, cache.tables[0, entry], 1] *= 2.0 ** (-60 if entry % 3 else 0)
    q = torch.from_numpy(rng.normal(size=(6, 4, 64)) * np.array([1e-6, 1.0, 30.0, 1e-20, 4.0, 0.0])[:, None, None]).float()
    q = q.to(device)
    got = cache.to(device).attention(0, q, kc.words([0], device), kc.words([0, 6], device))
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0], [0, 6], 0.125)
    _compare(got, want, mass, size, F32, 300)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_of_zero_beside_large_ones(device, dtype):
    """pages of zeros (the least scale there is) still count in the total"""
    rng = np.random.default_rng(17)
    cache = kc.filled(rng, [200], "int8", 16, 1, 64)
    for entry in range(cache.pages(200)):
        page = cache.tables[0, entry]
        if entry % 2:
            cache.scales[0, page, 1, 0] *= 2.0 ** 60
        else:
            cache.data[0, page, 1], cache.scales[0, page, 1] = 0, 2.0 ** -100
    q = torch.from_numpy(rng.normal(size=(3, 2, 64))).to(dtype).to(device)
    got = cache.to(device).attention(0, q, kc.words([0], device))
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0], [0, 3], 0.125)
    _compare(got, want, mass, size, dtype, 200)


def test_offsets_past_32_bits(device):
    """pages that begin more than 4 GiB into a layer, and a second layer behind it"""
    from q38hip import kv
    rng = np.random.default_rng(8)
    small = kc.filled(rng, [200], "int8", 128, 8, 256, layers=2, spare=0)
    pages, used = 8500, small.tables[0, :2].tolist()
    data = torch.empty((2, pages, 2, 8, 128, 256), dtype=torch.uint8, device=device)
    scales = torch.ones((2, pages, 2, 8), device=device)
    tables = torch.full((1, 3), -1, dtype=torch.int32, device=device)
    for entry, p in enumerate(used):
        far = pages - 1 - entry
        data[:, far] = torch.from_numpy(small.data[:, p]).to(device)
        scales[:, far] = torch.from_numpy(small.scales[:, p]).to(device)
        tables[0, entry] = far
    cache = kv.KVPages(data, scales, torch.zeros(pages, dtype=torch.int32, device=device), tables, kc.words([200], device),
                       kc.words([0], device), "int8")
    q = torch.from_numpy(rng.normal(size=(2, 8, 256))).float().to(device)
    for layer in (0, 1):
        got = cache.attention(layer, q, kc.words([0], device))
        want, mass, size = small.attention(layer, q.double().cpu().numpy(), [0], [0, 2], 256 ** -0.5)
        _compare(got, want, mass, size, F32, 200)


def test_ids_and_pages_outside_the_cache(device):
    """a bad sequence holds no tokens, a bad page is left out"""
    rng = np.random.default_rng(9)
    cache = kc.filled(rng, [48, 48], "int8", 16, 1, 64)
    q = torch.from_numpy(rng.normal(size=(4, 1, 64))).float().to(device)
    dev = cache.to(device)
    ids = kc.words([0, 99, -1, 1], device)
    dev.tables[1, 1] = 1 << 20
    got = dev.attention(0, q, ids).double().cpu().numpy()
    want, _, _ = cache.attention(0, q.double().cpu().numpy(), [0, 2, 2, 1], [0, 1, 2, 3, 4], 0.125)
    assert np.abs(got[0] - want[0]).max() < 1e-5 and not got[1:3].any()
    k, v = cache.rows_of(0, 1, 0)[:, 0], cache.rows_of(0, 1, 1)[:, 0]
    kept = np.r_[0:16, 32:48]
    w = np.exp(q[3, 0].double().cpu().numpy() @ k[kept].T * 0.125)
    assert np.abs(got[3, 0] - w @ v[kept] / w.sum()).max() < 1e-5


def test_same_bits_every_time(device):
    rng = np.random.default_rng(10)
    cache = kc.filled(rng, [3000, 900], "e4m3", 64, 2, 128)
    q = torch.from_numpy(rng.normal(size=(2, 8, 128))).float().to(device)
    dev, ids = cache.to(device), kc.words([0, 1], device)
    first = dev.attention(0, q, ids)
    for _ in range(5):
        assert torch.equal(dev.attention(0, q, ids), first)


def test_row_offsets_that_decrease(device):
    """nothing is done, and the status says so"""
    from q38hip import kv
    rng = np.random.default_rng(11)
    dev = kc.filled(rng, [48, 48, 20], "int8", 16, 2, 64).to(device)
    q = torch.from_numpy(rng.normal(size=(40, 4, 64))).float().to(device)
    out = torch.full_like(q, 3.0)
    for starts in ([0, 30, 10, 40], [40, 0, 40, 0], [0, -5, 40, 39]):
        dev.attention(0, q, kc.words([0, 1, 2], device), kc.words(starts, device), out=out)
        assert int(dev.status) == kv.BAD_ROWS
        dev.status.zero_()
        assert (out == 3.0).all()


@pytest.mark.parametrize("dim,dtype,kind", [(64, F16, "int8"), (128, F32, "e4m3"), (256, BF16, "int8")])
def test_many_sequences_of_all_lengths(device, dim, dtype, kind):
    """more sequences than a wavefront has lanes, some without tokens or rows, long ones cut between workgroups"""
    rng = np.random.default_rng(dim)
    lengths = [int(n) for n in np.exp(rng.uniform(0, np.log(1500), size=150))]
    lengths[3] = lengths[149] = 0
    rows = [int(r) for r in rng.integers(0, 4, size=150)]
    rows[0], rows[149] = 2, 1
    cache, starts, q, gate = _case(rng, 2, 1, dim, 32, kind, dtype, lengths, rows, device)
    order = [int(i) for i in rng.permutation(150)]
    got = cache.to(device).attention(0, q, kc.words(order, device), kc.words(starts, device), gate=gate)
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), order, starts, dim ** -0.5, gate.double().cpu().numpy())
    _compare(got, want, mass, size, dtype, max(lengths))


@pytest.mark.parametrize("dim,dtype,kind,heads", [(64, F32, "e4m3", 1), (64, BF16, "int8", 6), (128, F16, "e4m3", 3),
                                                  (128, F32, "int8", 1), (256, BF16, "e4m3", 2), (256, F32, "int8", 1)])
def test_prompts_that_are_cut(device, dim, dtype, kind, heads):
    """columns of several workgroups' wavefronts, cut along the tokens and joined"""
    rng = np.random.default_rng(dim + heads)
    lengths, rows = [2100, 333], [150, 333]
    cache, starts, q, gate = _case(rng, heads, 1, dim, 64, kind, dtype, lengths, rows, device)
    got = cache.to(device).attention(0, q, kc.words([0, 1], device), kc.words(starts, device), gate=gate)
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0, 1], starts, dim ** -0.5, gate.double().cpu().numpy())
    _compare(got, want, mass, size, dtype, max(lengths))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,heads,dtype", [(1, 2, F32), (2, 6, F32), (4, 6, F32), (3, 12, BF16), (60, 3, F16), (60, 3, F32)])
def test_maxima_that_rise(device, dim, rows, heads, dtype):
    """every page's scores pass those before it by more than the sums allow: they are rescaled again and again"""
    rng = np.random.default_rng(rows)
    cache = kc.filled(rng, [500], "int8", 16, 1, dim)
    direction = rng.normal(size=dim)
    for entry in range(cache.pages(500)):
        page = cache.tables[0, entry]
        x = direction * (0.5 + entry) / dim * 12 + rng.normal(size=(16, dim)) * 0.01
        scale = kc.scale_of(np.abs(x).max(), "int8")
        cache.scales[0, page, 0, 0] = scale
        cache.half(0, page, 0, 0)[:] = kc.encode(x / scale, "int8")
    q = torch.from_numpy(direction + rng.normal(size=(rows, heads, dim)) * 0.05).to(dtype).to(device)
    got = cache.to(device).attention(0, q, kc.words([0], device), scale=1.0)
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0], [0, rows], 1.0)
    _compare(got, want, mass, size, dtype, 500)


@pytest.mark.parametrize("dtype,kind,lengths,rows", [(F32, "int8", [5000, 3000], [4, 1]),
                                                     (BF16, "e4m3", [900 + 37 * i for i in range(24)], [1, 2, 1] * 8)])
def test_more_columns_than_workgroups_that_join(device, dtype, kind, lengths, rows):
    """ragged rows of 256-wide heads that are cut: a workgroup joins one column after another"""
    rng = np.random.default_rng(len(lengths))
    cache, starts, q, gate = _case(rng, 24, 4, 256, 64, kind, dtype, lengths, rows, device)
    dev, ids, ends = cache.to(device), kc.words(range(len(lengths)), device), kc.words(starts, device)
    first = dev.attention(0, q, ids, ends, gate=gate)
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), range(len(lengths)), starts, 256 ** -0.5,
                                       gate.double().cpu().numpy())
    _compare(first, want, mass, size, dtype, max(lengths))
    for _ in range(20):
        assert torch.equal(dev.attention(0, q, ids, ends, gate=gate), first)


GATES = [0.0, 20.0, -20.0, 87.0, -87.0, 90.0, -90.0, 100.0, -100.0, 104.0, -104.0, 1e4, -1e4, 5e4, -5e4, 1e9, -1e9, 1e30, -1e30, 3e38,
         -3e38, float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,heads,length,rows", [(256, 6, 20, 1), (128, 4, 6000, 2), (256, 6, 2000, 40)])
def test_gates_of_all_sizes(device, dtype, dim, heads, length, rows):
    """whole slots, cut ones and prompts; sigmoids that are subnormal in fp32 keep the bits that those have"""
    rng = np.random.default_rng(dim + rows)
    cache, starts, q, _ = _case(rng, heads, 1, dim, 64, "int8", dtype, [length], [rows], device)
    at = torch.arange(rows)[:, None, None] + torch.arange(heads)[:, None] + torch.arange(dim)
    gate = torch.tensor(GATES, dtype=torch.float64)[at % len(GATES)].to(dtype)
    got = cache.to(device).attention(0, q, kc.words([0], device), gate=gate.to(device)).double().cpu().numpy()
    with np.errstate(over="ignore"):
        want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0], starts, dim ** -0.5, gate.double().numpy())
    number = ~np.isnan(gate.double().numpy())
    assert np.array_equal(np.isnan(got), ~number)
    # the smallest steps: of the sigmoid (times the sum's size), and of the output
    value = cache.attention(0, q.double().cpu().numpy(), [0], starts, dim ** -0.5)[0]
    least = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 0.0}[dtype]
    bound = kc.tolerance(want, mass, size, dtype, length) - (1e-30 if dtype != F16 else 0) + 2.0 ** -149 * (1 + np.abs(value)) + least
    far = np.abs(got - want)[number] / bound[number]
    assert far.max() <= 1, "worst %g of its bound" % far.max()


def test_status_of_ids_and_pages(device):
    """bad ids that own rows, and bad pages that a row sees, are reported"""
    from q38hip import kv
    rng = np.random.default_rng(12)
    cache = kc.filled(rng, [48, 48, 700], "int8", 16, 1, 64)
    q = torch.from_numpy(rng.normal(size=(40, 2, 64))).float().to(device)
    for rows in (1, 40):
        for bad in (99, -1, 5):
            dev = cache.to(device)
            dev.attention(0, q[:rows], kc.words([0, bad, 2], device), kc.words([0, 0, 0, rows], device))
            assert int(dev.status) == 0                     # an id without rows
            dev.attention(0, q[:rows], kc.words([0, 2, bad], device), kc.words([0, 0, 0, rows], device))
            assert int(dev.status) == kv.BAD_SEQUENCE
        for sequence, entry, page in ((1, 0, -1), (1, 2, 1 << 20), (2, 43, -7)):
            dev = cache.to(device)
            dev.tables[0, 3] = 1 << 20                      # behind the sequence's tokens
            dev.attention(0, q[:rows], kc.words([0], device))
            assert int(dev.status) == 0
            dev.tables[sequence, entry] = page
            dev.attention(0, q[:rows], kc.words([sequence], device))
            assert int(dev.status) == kv.BAD_PAGE
