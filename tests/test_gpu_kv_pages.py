"""Append and page operations of the paged 8-bit cache on the GPU against the
plain model (tests/kv_cases.py): every code, scale, count and table entry is
equal."""
import numpy as np
import pytest
import torch

import kv_cases as kc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rows(rng, rows, heads, dim, dtype, device, size=1.0):
    x = torch.from_numpy(rng.normal(size=(rows, heads, dim)) * size).to(dtype)
    return x.to(device)


APPENDS = [
    # kind, type, kv_heads, dim, page, lengths after, rows
    ("int8", F32, 4, 256, 64, [1], [1]),
    ("int8", F32, 4, 256, 16, [17, 16, 15], [1, 1, 1]),
    ("e4m3", BF16, 2, 128, 32, [33, 64, 100], [33, 1, 70]),
    ("e4m3", F32, 1, 64, 128, [300, 7], [131, 3]),
    ("int8", F16, 3, 64, 16, [50, 0, 9, 40], [50, 0, 4, 1]),
    ("e4m3", F16, 2, 256, 128, [255], [255]),
    ("int8", BF16, 1, 128, 32, [20] * 70, [1, 3] * 35),
    ("e4m3", BF16, 2, 64, 64, [5], [9]),                   # more rows than tokens: the last five
]


@pytest.mark.parametrize("case", APPENDS, ids=lambda c: "%s-%s-%dx%d-p%d-%d" % (c[0], str(c[1])[6:], c[2], c[3], c[4], len(c[5])))
def test_append(device, case):
    kind, dtype, heads, dim, page, lengths, rows = case
    rng = np.random.default_rng(page + dim + len(lengths))
    cache = kc.filled(rng, lengths, kind, page, heads, dim, layers=2, garbage=False)
    dev = cache.to(device)
    ids = list(rng.permutation(len(lengths)))
    starts = kc.offsets([rows[i] for i in ids])
    for turn in range(2):                                  # the second values are larger: scales grow
        key = _rows(rng, starts[-1], heads, dim, dtype, device, 3.0 * 40 ** turn)
        value = _rows(rng, starts[-1], heads, dim, dtype, device, 0.2 * 40 ** turn)
        dev.append(1, key, value, kc.words(ids, device), kc.words(starts, device))
        cache.append(1, key.double().cpu().numpy(), value.double().cpu().numpy(), ids, starts)
        cache.same(dev)
    dev.check()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_token_by_token(device, kind):
    """scales that grow, shrink (and stay) and codes that follow them"""
    rng = np.random.default_rng(3)
    cache = kc.Cache(1, 4, 16, 2, 64, 1, 3, kind)
    dev = cache.to(device)
    one = kc.words([0], device)
    for token in range(40):
        assert cache.extend([0], [1])
        dev.extend(one, kc.words([1], device))
        size = 2.0 ** rng.integers(-8, 8)
        key, value = _rows(rng, 1, 2, 64, F32, device, size), _rows(rng, 1, 2, 64, F32, device, 1 / size)
        if token == 20:
            value.zero_()
        dev.append(0, key, value, one)
        cache.append(0, key.double().cpu().numpy(), value.double().cpu().numpy(), [0], [0, 1])
        cache.same(dev)


def test_append_borders(device):
    """values on the rounding borders of the codes, at the largest code, zeros and
    the smallest and largest floats"""
    for kind, largest in kc.LARGEST.items():
        cache = kc.filled(np.random.default_rng(1), [16, 32], kind, 16, 1, 64, garbage=False)
        x = np.zeros((48, 1, 64))
        x[:16, 0] = largest * np.exp2(np.arange(16) - 8)[:, None] * np.linspace(-1, 1, 64)
        x[0, 0, :16] = np.arange(16) - 7.5
        x[16:24] = 0.0
        x[24, 0, 0], x[25, 0, 0], x[26, 0, 0] = 1e-45, 3.4028234663852886e38, -3.4028234663852886e38
        x[32:48, 0] = (np.arange(16)[:, None] * 64 + np.arange(64)) / 1024 * largest
        x[47, 0, 63] = largest
        x = torch.from_numpy(x).float()
        dev = cache.to(device)
        for rows in (x, x.flip(0).contiguous()):
            r = rows.to(device)
            dev.append(0, r, r, kc.words([0, 1], device), kc.words([0, 16, 48], device))
            cache.append(0, rows.double().numpy(), rows.double().numpy(), [0, 1], [0, 16, 48])
            cache.same(dev)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_what_is_not_finite(device, kind):
    """the page's scale becomes NaN and stays so until its first token is written again"""
    rng = np.random.default_rng(4)
    cache = kc.filled(rng, [24, 5], kind, 16, 2, 64, garbage=False)
    dev = cache.to(device)
    key, value = rng.normal(size=(2, 24, 2, 64))
    key[3, 1, 7], value[20, 0, 0] = np.inf, np.nan
    for k, v, ids, starts in ((key, value, [0], [0, 24]), (key[4:8], value[4:8], [1], [0, 4]),
                              (key[3:4], value[:1], [1], [0, 1]), (key[:1], value[:1], [1], [0, 1]),
                              (key[8:13], value[8:13], [1], [0, 5])):
        k, v = torch.from_numpy(k).float().contiguous(), torch.from_numpy(v).float().contiguous()
        dev.append(0, k.to(device), v.to(device), kc.words(ids, device), kc.words(starts, device))
        cache.append(0, k.double().numpy(), v.double().numpy(), ids, starts)
        cache.same(dev)
    assert np.isnan(cache.scales).any() and np.isfinite(cache.scales[0, cache.tables[1, 0]]).all()


def test_append_strides(device):
    """keys and values inside wider rows, aligned and not"""
    rng = np.random.default_rng(5)
    for dtype in (F32, BF16):
        for pad in (0, 1):
            cache = kc.filled(rng, [40], "int8", 16, 2, 64, garbage=False)
            dev = cache.to(device)
            wide = torch.from_numpy(rng.normal(size=(21, 300 + pad))).to(dtype).to(device)
            key, value = wide[:, pad:pad + 128].unflatten(1, (2, 64)), wide[:, pad + 128:pad + 256].unflatten(1, (2, 64))
            dev.append(0, key, value, kc.words([0], device), kc.words([0, 21], device))
            cache.append(0, key.double().cpu().numpy(), value.double().cpu().numpy(), [0], [0, 21])
            cache.same(dev)


def test_append_outside_the_cache(device):
    """bad ids and pages write nothing"""
    from q38hip import kv
    rng = np.random.default_rng(6)
    cache = kc.filled(rng, [20, 20], "int8", 16, 1, 64, garbage=False)
    dev = cache.to(device)
    x = _rows(rng, 8, 1, 64, F32, device)
    dev.append(0, x, x, kc.words([99, -5], device), kc.words([0, 4, 8], device))
    cache.same(dev)
    dev.tables[0, 1] = 1 << 30
    dev.append(0, x[:4], x[:4], kc.words([0], device))
    assert torch.equal(dev.data.cpu(), torch.from_numpy(cache.data))
    assert int(dev.status) == kv.BAD_PAGE


@pytest.mark.parametrize("count", [5, 150])
def test_append_row_offsets_that_decrease(device, count):
    """nothing is written, and the status says so"""
    from q38hip import kv
    rng = np.random.default_rng(7)
    cache = kc.filled(rng, [600] * count, "int8", 16, 1, 64, garbage=False)
    dev = cache.to(device)
    x = _rows(rng, 1300, 1, 64, F32, device, 1000.0)
    up = [1250 + i % 3 for i in range(count - 5)]
    for starts in ([0, 1000, 1200, 10, 1300] + sorted(up) + [1300], [1300, 0] * (count // 2) + [1300] * (1 + count % 2),
                   [0, -5] + [40] * (count - 2) + [39]):
        assert len(starts) == count + 1
        dev.append(0, x, x, kc.words(range(count), device), kc.words(starts, device))
        assert int(dev.status) == kv.BAD_ROWS
        dev.status.zero_()
        cache.same(dev)


# ---- pages ---------------------------------------------------------------------


def _noise(rng, cache):
    cache.data[:] = rng.integers(0, 256, size=cache.shape, dtype=np.uint8)
    cache.scales[:] = rng.integers(1, 1000, size=cache.scales.shape).astype(np.float32)


def test_pages_through_a_life(device):
    """extend, fork, truncate and compact in random order, with copies on the first write"""
    rng = np.random.default_rng(11)
    cache = kc.Cache(3, 60, 16, 1, 64, 10, 12, "int8")
    _noise(rng, cache)
    dev = cache.to(device)
    done = set()
    for turn in range(120):
        what = rng.choice(["extend", "extend", "fork", "truncate", "compact"])
        if what == "extend":
            ids = list(rng.permutation(10)[:rng.integers(1, 6)])
            rows = [int(r) for r in rng.integers(0, 30, size=len(ids))]
            worked = cache.extend(ids, rows)
            dev.extend(kc.words(ids, device), kc.words(rows, device))
            assert bool(int(dev.status)) == (not worked)
            dev.status.zero_()
            done.add(("extend", worked))
        elif what == "fork":
            empty = [i for i in range(10) if cache.lengths[i] == 0]
            held = [i for i in range(10) if cache.lengths[i]]
            if not empty or not held:
                continue
            children = empty[:rng.integers(1, len(empty) + 1)]
            parents = [int(rng.choice(held)) for _ in children]
            lengths = None if turn % 2 else [int(rng.integers(0, 200)) for _ in children]
            cache.fork(parents, children, lengths)
            dev.fork(kc.words(parents, device), kc.words(children, device),
                     None if lengths is None else kc.words(lengths, device))
        elif what == "truncate":
            ids = list(rng.permutation(10)[:rng.integers(1, 4)])
            lengths = [int(rng.integers(-5, 120)) if turn % 3 else 0 for _ in ids]
            cache.truncate(ids, lengths)
            dev.truncate(kc.words(ids, device), kc.words(lengths, device))
        else:
            moved, live = cache.compact()
            assert dev.compact().tolist() == [moved, live]
        done.add(what)
        assert int(dev.status) == 0
        cache.same(dev)
    assert {("extend", True), ("extend", False), "fork", "truncate", "compact"} <= done


def test_last_owner_keeps_the_page(device):
    """of three sequences that share a partly filled page and grow together, two copy it"""
    cache = kc.Cache(2, 12, 16, 1, 64, 4, 3, "e4m3")
    _noise(np.random.default_rng(1), cache)
    dev = cache.to(device)
    for c in (cache, dev):
        w = (lambda v: kc.words(v, device)) if c is dev else list
        c.extend(w([0]), w([20]))
        c.fork(w([0, 0]), w([2, 1]))
        c.extend(w([1, 2, 0]), w([1, 13, 1]))
    cache.same(dev)
    assert cache.tables[0, 1] == 1 and cache.refs.tolist()[:5] == [3, 1, 1, 1, 1]


@pytest.mark.parametrize("offset", [0, 1])
def test_large_pool(device, offset):
    """more pages than one round of the scans, counts aligned and not"""
    from q38hip import kv
    rng = np.random.default_rng(12)
    pages = 40001
    cache = kc.Cache(1, pages, 16, 1, 64, 6, 20000, "int8")
    cache.data[:, :, 0, 0, 0, 0] = rng.integers(0, 256, size=(1, pages))
    taken = rng.permutation(pages)[:26000]
    cache.tables[5, :20000], cache.tables[4, :6000] = taken[:20000], taken[20000:]
    cache.refs[taken] = 1
    cache.lengths[5], cache.lengths[4] = 20000 * 16, 6000 * 16 - 5
    dev = cache.to(device)
    room = torch.zeros(pages + 4, dtype=torch.int32, device=device)
    room[offset:offset + pages] = dev.refs
    dev = kv.KVPages(dev.data, dev.scales, room[offset:offset + pages], dev.tables, dev.lengths, dev.status, "int8")
    for ids, rows in (([1, 2, 3], [7000 * 16, 3, 5000 * 16 + 1]), ([0], [30000]), ([4], [6]), ([0], [100])):
        worked = cache.extend(ids, rows)
        dev.extend(kc.words(ids, device), kc.words(rows, device))
        assert bool(int(dev.status)) == (not worked)
        dev.status.zero_()
        cache.same(dev)
    cache.truncate([1, 5], [16 * 50, 0])
    dev.truncate(kc.words([1, 5], device), kc.words([16 * 50, 0], device))
    moved, live = cache.compact()
    assert dev.compact().tolist() == [moved, live] and moved > 0
    cache.same(dev)


def test_status_bits(device):
    """what the device refuses: nothing changes but the status"""
    from q38hip import kv
    cache = kc.Cache(1, 6, 16, 1, 64, 4, 3, "int8")
    dev = cache.to(device)
    w = lambda *v: kc.words(v, device)  # noqa: E731
    assert cache.extend([0, 1], [30, 16])
    dev.extend(w(0, 1), w(30, 16))
    for call, bit in ((lambda: dev.extend(w(2), w(64)), kv.TABLE_FULL), (lambda: dev.extend(w(2, 3), w(48, 16)), kv.POOL_FULL),
                      (lambda: dev.extend(w(2, 2), w(1, 1)), kv.BAD_SEQUENCE), (lambda: dev.extend(w(4), w(1)), kv.BAD_SEQUENCE),
                      (lambda: dev.extend(w(2), w(-1)), kv.BAD_SEQUENCE), (lambda: dev.fork(w(0), w(1)), kv.NOT_EMPTY),
                      (lambda: dev.fork(w(0, 2), w(2, 3)), kv.BAD_SEQUENCE), (lambda: dev.fork(w(-1), w(2)), kv.BAD_SEQUENCE),
                      (lambda: dev.truncate(w(7), w(0)), kv.BAD_SEQUENCE), (lambda: dev.copy(w(0), w(6)), kv.BAD_PAGE)):
        call()
        assert int(dev.status) & bit
        with pytest.raises(RuntimeError):
            dev.check()
        if bit == kv.BAD_SEQUENCE and int(dev.lengths[2]):     # the good pair of the fork was done
            cache.fork([0], [2])
            dev.truncate(w(2), w(0))
            cache.truncate([2], [0])
        cache.same(dev)
    dev.truncate(w(0, 0, 1), w(0, 0, 0))                       # a repeated id is freed once
    cache.truncate([0, 1], [0, 0])
    cache.same(dev)


def test_fork_of_nothing(device):
    """a child that holds tokens is reported and left as it is where there is nothing to take, too"""
    from q38hip import kv
    cache = kc.Cache(1, 6, 16, 1, 64, 4, 3, "int8")
    dev = cache.to(device)
    w = lambda *v: kc.words(v, device)  # noqa: E731
    assert cache.extend([0, 1], [30, 16])
    dev.extend(w(0, 1), w(30, 16))
    for call, bits in ((lambda: dev.fork(w(2), w(3)), 0),                          # an empty parent, an empty child
                       (lambda: dev.fork(w(0), w(2), w(0)), 0),
                       (lambda: dev.fork(w(2), w(0)), kv.NOT_EMPTY),
                       (lambda: dev.fork(w(0), w(1), w(0)), kv.NOT_EMPTY),
                       (lambda: dev.fork(w(0), w(1), w(-9)), kv.NOT_EMPTY)):
        call()
        assert int(dev.status) == bits
        dev.status.zero_()
        cache.same(dev)


def test_copy_and_reset(device):
    cache = kc.Cache(2, 8, 32, 2, 128, 3, 2, "e4m3")
    _noise(np.random.default_rng(2), cache)
    dev = cache.to(device)
    dev.copy(kc.words([1, -1, 7], device), kc.words([4, 5, 0], device))
    for source, target in ((1, 4), (7, 0)):
        cache.data[:, target], cache.scales[:, target] = cache.data[:, source], cache.scales[:, source]
    cache.same(dev)
    dev.extend(kc.words([0], device), kc.words([40], device))
    dev.reset()
    cache.same(dev)


# ---- as a program uses them ---------------------------------------------------------


def test_graph_of_a_step(device):
    """extend, append and attention in one graph, replayed between eager steps"""
    from q38hip import kv
    rng = np.random.default_rng(13)
    make = lambda: kv.KVPages.allocate(1, 40, 16, 2, 64, 3, 12, "int8", device)  # noqa: E731
    graphed, eager = make(), make()
    graphed.data.zero_(), eager.data.zero_()
    ids, ones = kc.words([2, 0], device), kc.words([1, 1], device)
    x = [torch.zeros((2, n, 64), device=device) for n in (2, 2, 6)]

    def step(cache, key, value, query):
        cache.extend(ids, ones)
        cache.append(0, key, value, ids)
        return cache.attention(0, query, ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed, *x)
        graphed.reset()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(graphed, *x)
    for turn in range(37):
        for t in x:
            t.copy_(torch.from_numpy(rng.normal(size=t.shape)).float())
        graph.replay()
        want = step(eager, *x)
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn
    assert torch.equal(graphed.data[:, :6], eager.data[:, :6]) and torch.equal(graphed.lengths, eager.lengths)


def test_other_stream(device):
    """everything on a stream of its own, behind work of another stream"""
    rng = np.random.default_rng(14)
    cache = kc.filled(rng, [100, 31], "e4m3", 32, 2, 128, garbage=False)
    dev, ids = cache.to(device), kc.words([0, 1], device)
    side = torch.cuda.Stream()
    key, value = (torch.from_numpy(rng.normal(size=(2, 2, 128))).float().to(device) for _ in range(2))
    q = torch.from_numpy(rng.normal(size=(2, 8, 128))).float().to(device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dev.append(0, key, value, ids)
        got = dev.attention(0, q, ids)
    side.synchronize()
    cache.append(0, key.double().cpu().numpy(), value.double().cpu().numpy(), [0, 1], [0, 1, 2])
    cache.same(dev)
    want, mass, size = cache.attention(0, q.double().cpu().numpy(), [0, 1], [0, 1, 2], 128 ** -0.5)
    assert (np.abs(got.double().cpu().numpy() - want) <= kc.tolerance(want, mass, size, F32, 100)).all()
