"""A plain model of the paged 8-bit cache (include/q38hip.h, section 3) in
numpy with 64-bit values, and seeded inputs, shared by the kv tests."""
import numpy as np
import torch

LARGEST = {"int8": 127.0, "e4m3": 448.0}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def encode(x, kind):
    """codes (uint8) of float64 values within the type's range: one rounding, ties to even"""
    if kind == "int8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    step = np.ldexp(1.0, np.frexp(np.maximum(a, 2.0 ** -6))[1] - 4)
    return torch.from_numpy(np.copysign(np.rint(a / step) * step, x)).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def decode(codes, kind):
    codes = np.ascontiguousarray(codes)
    if kind == "int8":
        return codes.view(np.int8).astype(np.float64)
    return torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()


def scale_of(a, kind):
    """2^k, k >= -100 the least with a <= LARGEST 2^k"""
    k = -100
    while a > LARGEST[kind] * 2.0 ** k:
        k += 1
    return 2.0 ** k


class Cache:
    def __init__(self, layers, pages, page_tokens, kv_heads, head_dim, sequences, table_entries, kind):
        self.shape = (layers, pages, 2, kv_heads, page_tokens, head_dim)
        self.T, self.H, self.D, self.kind = page_tokens, kv_heads, head_dim, kind
        self.data = np.zeros(self.shape, dtype=np.uint8)
        self.scales = np.ones(self.shape[:4], dtype=np.float32)
        self.refs = np.zeros(pages, dtype=np.int32)
        self.tables = np.full((sequences, table_entries), -1, dtype=np.int32)
        self.lengths = np.zeros(sequences, dtype=np.int32)

    def half(self, layer, page, half, head):
        """codes of a block as [token][channel] (a view)"""
        block = self.data[layer, page, half, head]
        return block if half == 0 else block.reshape(self.D, self.T).T

    def pages(self, tokens):
        return -(-tokens // self.T)

    # ---- pages ------------------------------------------------------------------
    def extend(self, ids, rows):
        refs, tables, lengths = self.refs.copy(), self.tables.copy(), self.lengths.copy()
        free = list(np.flatnonzero(refs == 0))          # pages that this call frees are handed out by the next
        copies = []
        for i, r in zip(ids, rows):
            n = lengths[i]
            if n + r > self.tables.shape[1] * self.T:
                return False
            new = list(range(self.pages(n), self.pages(n + r)))
            if r and n % self.T and refs[tables[i, n // self.T]] > 1:
                new = [n // self.T] + new
                copies.append((tables[i, n // self.T], i, n // self.T))
                refs[tables[i, n // self.T]] -= 1
            for entry in new:
                if not free:
                    return False
                tables[i, entry] = free.pop(0)
                refs[tables[i, entry]] = 1
            lengths[i] = n + r
        self.refs, self.tables, self.lengths = refs, tables, lengths
        for source, i, entry in copies:
            self.data[:, tables[i, entry]] = self.data[:, source]
            self.scales[:, tables[i, entry]] = self.scales[:, source]
        return True

    def fork(self, parents, children, lengths=None):
        for j, (p, c) in enumerate(zip(parents, children)):
            n = self.lengths[p] if lengths is None else max(0, min(self.lengths[p], lengths[j]))
            self.lengths[c] = n
            self.tables[c, :self.pages(n)] = self.tables[p, :self.pages(n)]
            self.refs[self.tables[p, :self.pages(n)]] += 1

    def truncate(self, ids, lengths):
        for i, n in zip(ids, lengths):
            n = min(max(n, 0), self.lengths[i])
            for entry in range(self.pages(n), self.pages(self.lengths[i])):
                self.refs[self.tables[i, entry]] -= 1
                self.tables[i, entry] = -1
            self.lengths[i] = n

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        for source, target in zip(movers, holes):
            self.data[:, target] = self.data[:, source]
            self.scales[:, target] = self.scales[:, source]
            self.refs[target], self.refs[source] = self.refs[source], 0
            self.tables[self.tables == source] = target
        return len(movers), live

    # ---- rows -------------------------------------------------------------------
    def append(self, layer, key, value, ids, starts):
        """key, value: float64 [rows, H, D]"""
        for j, i in enumerate(ids):
            n = int(self.lengths[i])
            rows = min(starts[j + 1] - starts[j], n)
            at = n - rows
            while at < n:
                used, end = at % self.T, min(n, (at // self.T + 1) * self.T)
                page = self.tables[i, at // self.T]
                span = slice(starts[j + 1] - n + at, starts[j + 1] - n + end)
                for half, x in ((0, key[span]), (1, value[span])):
                    for h in range(self.H):
                        block, was = self.half(layer, page, half, h), float(self.scales[layer, page, half, h])
                        new = x[:, h]
                        if not np.isfinite(new).all():
                            scale = np.nan
                        else:
                            scale = scale_of(np.abs(new).max(), self.kind)
                            if used and not was <= scale:
                                scale = was
                            elif used and scale > was:
                                block[:used] = encode(decode(block[:used], self.kind) * (was / scale), self.kind)
                        self.scales[layer, page, half, h] = scale
                        block[used:used + end - at] = 0 if np.isnan(scale) else encode(new / scale, self.kind)
                at = end

    def rows_of(self, layer, seq, half):
        """float64 [tokens, H, D] of a sequence"""
        n = int(self.lengths[seq])
        out = np.zeros((n, self.H, self.D))
        for at in range(0, n, self.T):
            page = self.tables[seq, at // self.T]
            for h in range(self.H):
                values = decode(self.half(layer, page, half, h), self.kind) * float(self.scales[layer, page, half, h])
                out[at:at + self.T, h] = values[:n - at]
        return out

    def attention(self, layer, query, ids, starts, scale, gate=None):
        """float64 [rows, heads, D] of float64 queries; also the bound's
        ingredients: (sum p |v|, the largest weight p sv times sum |v| / sv),
        sv the scale of a token's page, and, per row and head, the largest sum
        |q k| scale"""
        out, mass, floor = np.zeros(query.shape), np.zeros(query.shape), np.zeros(query.shape)
        size = np.zeros(query.shape[:2])
        group = query.shape[1] // self.H
        for j, i in enumerate(ids):
            n, r = int(self.lengths[i]), starts[j + 1] - starts[j]
            if not r:
                continue
            k, v = self.rows_of(layer, i, 0), self.rows_of(layer, i, 1)
            sv = self.scales[layer, self.tables[i, np.arange(n) // self.T], 1].astype(np.float64)
            for h in range(query.shape[1]):
                q = query[starts[j]:starts[j + 1], h]
                z = q @ k[:, h // group].T * scale
                absolute = np.abs(q) @ np.abs(k[:, h // group]).T * abs(scale)
                for t in range(r):
                    seen = n - r + t + 1
                    if seen <= 0:
                        continue
                    with np.errstate(invalid="ignore"):
                        w = np.exp(z[t, :seen] - z[t, :seen].max())
                    w /= w.sum()
                    out[starts[j] + t, h] = w @ v[:seen, h // group]
                    mass[starts[j] + t, h] = w @ np.abs(v[:seen, h // group])
                    s = sv[:seen, h // group]
                    floor[starts[j] + t, h] = (w * s).max() * (np.abs(v[:seen, h // group]) / s[:, None]).sum(0)
                    size[starts[j] + t, h] = absolute[t, :seen].max()
        if gate is not None:
            sigmoid = 1 / (1 + np.exp(-gate))
            out, mass, floor = out * sigmoid, mass * sigmoid, floor * sigmoid
        return out, (mass, floor), size

    # ---- the device's copy ------------------------------------------------------
    def to(self, device):
        from q38hip import kv
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a).copy()).to(device)  # noqa: E731
        return kv.KVPages(put(self.data), put(self.scales), put(self.refs), put(self.tables), put(self.lengths),
                          torch.zeros(1, dtype=torch.int32, device=device), self.kind)

    def same(self, device_cache, data=True):
        assert np.array_equal(device_cache.lengths.cpu().numpy(), self.lengths)
        assert np.array_equal(device_cache.tables.cpu().numpy(), self.tables)
        assert np.array_equal(device_cache.refs.cpu().numpy(), self.refs)
        if data:
            assert np.array_equal(device_cache.scales.cpu().numpy(), self.scales, equal_nan=True)
            assert np.array_equal(device_cache.data.cpu().numpy(), self.data)


def words(values, device):
    return torch.tensor(list(values), dtype=torch.int32, device=device)


def offsets(rows):
    return [0] + [int(n) for n in np.cumsum(rows)]


def filled(rng, lengths, kind, page, kv_heads, head_dim, layers=1, spare=3, garbage=True):
    """A cache whose sequences hold `lengths` tokens of random codes on scattered
    pages; bytes and scales that hold no token are not numbers (e4m3) or -128"""
    pages = sum(-(-n // page) for n in lengths) + spare
    cache = Cache(layers, pages, page, kv_heads, head_dim, len(lengths) + 2, max(1, max(-(-n // page) for n in lengths)) + 1,
                  kind)
    order = list(rng.permutation(pages))
    cache.data[:] = 0x7F if kind == "e4m3" else 0x80
    cache.scales[:] = np.nan if garbage else 1.0
    for i, n in enumerate(lengths):
        cache.lengths[i] = n
        for at in range(0, n, page):
            p = order.pop()
            cache.tables[i, at // page] = p
            cache.refs[p] = 1
            for layer in range(layers):
                for half in (0, 1):
                    for h in range(kv_heads):
                        count = min(page, n - at)
                        x = rng.normal(size=(count, head_dim)) * 2.0 ** rng.integers(-4, 4)
                        scale = scale_of(np.abs(x).max(), kind)
                        cache.scales[layer, p, half, h] = scale
                        cache.half(layer, p, half, h)[:count] = encode(x / scale, kind)
    return cache


def tolerance(want, mass, size, dtype, longest):
    """Bound of an output's error.  Scores: products of exact codes with queries
    of 22 bits (fp32) or exact ones, fp32 sums of up to 256 terms (2^-24 each),
    two roundings of the scaling; a score that is d off moves a weight by d of
    itself, in the sum and in the total.  Weights: exp2 and scaling 2^-21,
    fp16 for 16-bit rows (2^-11), 22 bits for fp32 (2^-21); sums of `longest`
    terms of mean error, at most sqrt; division and gate 2^-21; one rounding
    of the result (half a step of 2^-24 where an fp16 result is subnormal).  The floor: the largest weight is 2^6 or more in fp16, whose
    smallest step is 2^-24, so every weight is within 2^-31 of the largest."""
    mass, floor = mass
    score = size * (2.0 ** -21 + 2.0 ** -24 * 32)
    weight = 2.0 ** -20 + (2.0 ** -11 if dtype != torch.float32 else 2.0 ** -21) + 2.0 ** -24 * np.sqrt(longest)
    return floor * 2.0 ** -31 + mass * (2 * score[..., None] + weight + 2.0 ** -20) + np.abs(want) * HALF_STEP[dtype] * 1.01 + \
        (2.0 ** -25 if dtype == torch.float16 else 1e-30)
