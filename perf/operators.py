"""Measured cases of the paged 8-bit key/value cache: append, attention and
page operations.

The cache is a pool of pages of `page` tokens.  A page holds, per layer and
key/value head, its keys token-major [page][dim] and its values channel-major
[dim][page] as 8-bit codes (int8, or e4m3 floats), and one scale, a power of
two, for the keys and one for the values.  A sequence is a row of the page
table and a length; a page may belong to several sequences (refs counts them).

  append     the last rows of each sequence of the call, quantised into pages
  attention  causal attention of those rows over their sequences, optionally
             times sigmoid(gate)
  branch     sequences cut back, forked and extended (pages shared until a
             sequence writes into one: then it gets its own copy)
  compact    the live pages moved to the front of the pool

With `own` false everything is plain torch on the same tensors; with `own`
true the calls go through q38hip.kv.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MIN_EXPONENT = -100


def _attention(name, kind, cache, heads, kv_heads, dim, page, count, tokens, rows, ragged=False, gate=False, empty=False):
    return {"name": name, "op": "attention", "type": kind, "cache": cache, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "count": count, "tokens": tokens, "rows": rows, "ragged": ragged, "gate": gate,
            "empty": empty}


def _append(name, kind, cache, kv_heads, dim, page, count, tokens, rows, ragged=False):
    return {"name": name, "op": "append", "type": kind, "cache": cache, "heads": kv_heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "count": count, "tokens": tokens, "rows": rows, "ragged": ragged, "gate": False,
            "empty": False}


def _pages(name, op, layers, kv_heads, dim, page, parents, children, tokens, spare):
    return {"name": name, "op": op, "layers": layers, "kv_heads": kv_heads, "dim": dim, "page": page,
            "parents": parents, "children": children, "tokens": tokens, "spare": spare}


def listed():
    return [
        # the first tokens of a chat: launch latency is all there is
        _attention("decode_short", "f32", "int8", 24, 4, 256, 16, 1, 37, 1, gate=True),
        # one sequence at the default context of the engine, its heads and gate
        _attention("decode_4k", "f32", "int8", 24, 4, 256, 64, 1, 4099, 1, gate=True),
        # a serving step over sequences of very different lengths, one of them just opened
        _attention("decode_batch", "bf16", "e4m3", 32, 8, 128, 32, 48, 16384, 1, empty=True),
        # a verify step of three drafts at the end of a long document
        _attention("verify_long", "f32", "e4m3", 24, 4, 256, 128, 1, 131075, 4, gate=True),
        # a chunk of a prompt behind an earlier part of it
        _attention("prompt_chunk", "bf16", "int8", 24, 4, 256, 64, 1, 8191, 512, gate=True),
        # short prompts of several users in one call, one head of keys for each head of queries
        _attention("prompt_ragged", "f16", "e4m3", 16, 16, 64, 16, 8, 1500, 300, ragged=True),
        # the new token of each sequence of a serving step
        _append("append_step", "f32", "int8", 4, 256, 64, 16, 6000, 1),
        # a prompt written in one call
        _append("append_prompt", "bf16", "e4m3", 8, 128, 32, 1, 4099, 4096),
        # beams of one user: every step drops the losers, forks the winners and writes a token
        _pages("branch_beam", "branch", 17, 4, 256, 16, 1, 3, 701, 64),
        # parallel samples of many prompts, the pages of all layers copied on the first write
        _pages("branch_samples", "branch", 17, 4, 256, 64, 24, 3, 2050, 40),
        # a small pool after a few sequences ended
        _pages("compact_small", "compact", 2, 8, 128, 32, 8, 0, 900, 100),
        # a pool of many sequences, about half of it free and scattered
        _pages("compact_pool", "compact", 17, 4, 256, 64, 40, 0, 3900, 900),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "branch", "compact"))
    page = rng.choice((16, 32, 64, 128))
    if op in ("branch", "compact"):
        kv_heads, dim = rng.choice(((4, 256), (8, 128), (3, 64)))
        layers, parents = rng.choice((1, 5, 17)), _log_int(rng, 1, 24)
        tokens = _log_int(rng, 20, 2000)
        children = rng.randint(1, 4) if op == "branch" else 0
        c = _pages("", op, layers, kv_heads, dim, page, parents, children, tokens, _log_int(rng, 8, 300))
    else:
        kind, cache = rng.choice(tuple(TYPES)), rng.choice(("int8", "e4m3"))
        heads, kv_heads, dim = rng.choice(((24, 4, 256), (32, 8, 128), (16, 16, 64), (12, 1, 128), (5, 5, 256), (40, 8, 64)))
        if op == "append":
            count = _log_int(rng, 1, 32)
            rows = _log_int(rng, 1, max(2, 2000 // count))
            c = _append("", kind, cache, kv_heads, dim, page, count, rows + _log_int(rng, 1, 3000), rows, rng.random() < 0.5)
        else:
            shape = rng.choice(("decode", "verify", "prompt"))
            count = _log_int(rng, 1, {"decode": 48, "verify": 16, "prompt": 8}[shape])
            rows = {"decode": 1, "verify": rng.randint(2, 8), "prompt": _log_int(rng, 9, max(10, 512 // count))}[shape]
            tokens = rows + _log_int(rng, 1, 8000 if shape == "prompt" else min(100000, 300000 // count))
            c = _attention("", kind, cache, heads, kv_heads, dim, page, count, tokens, rows, rng.random() < 0.4,
                           rng.random() < 0.4, count > 1 and rng.random() < 0.3)
    del c["name"]
    return c


# ---- sizes that follow from a case --------------------------------------------


def _lengths(c):
    """tokens of each sequence: the largest first, the others spread below it over the logarithm"""
    n = c.get("count") or c["parents"]
    low = c["tokens"] ** 0.5 if "count" in c else c["tokens"] * 0.5
    return [max(1, round(low * (c["tokens"] / low) ** (1 - i * 0.618034 % 1))) for i in range(n)]


def _rows(c):
    """rows of each sequence in the call"""
    return [min(n, 1 + (c["rows"] - 1 + i * 7919) % c["rows"]) if c["ragged"] else min(n, c["rows"])
            for i, n in enumerate(_lengths(c))]


def _tokens_of(c):
    """as _lengths, where the last sequence of an `empty` case holds nothing"""
    n = _lengths(c)
    return n[:-1] + [0] if c.get("empty") else n


def _up(a, b):
    return -(-a // b)


def work(c):
    if c["op"] in ("branch", "compact"):
        page = c["layers"] * 2 * c["kv_heads"] * (c["page"] * c["dim"] + 4)
        lengths = _lengths(c)
        if c["op"] == "branch":
            moved = sum(c["children"] for n in lengths if n % c["page"])
            entries = sum(_up(n + 1, c["page"]) * (1 + c["children"]) for n in lengths)
        else:
            entries = live = sum(_up(n, c["page"]) for n in lengths)
            spare = c["spare"] + len(lengths)
            moved = live * spare / (live + spare)
        return {"bytes": moved * page * 2 + entries * 8, "flops": 0}
    size = TYPES[c["type"]].itemsize
    lengths, rows = _tokens_of(c), _rows(c)
    token = 2 * c["kv_heads"] * c["dim"]
    pages = sum(_up(n, c["page"]) for n in lengths)
    if c["op"] == "append":
        return {"bytes": sum(rows) * token * (size + 1) + _up(sum(rows), c["page"]) * 2 * c["kv_heads"] * 4, "flops": 0}
    seen = sum(max(0, n - r + t + 1) for n, r in zip(lengths, rows) for t in range(r))
    row = c["heads"] * c["dim"] * size * (3 if c["gate"] else 2)
    return {"bytes": sum(rows) * row + sum(lengths) * token + pages * (4 + 8 * c["kv_heads"]),
            "flops": 4 * c["dim"] * c["heads"] * seen}


# ---- inputs --------------------------------------------------------------------


def _largest_exponent(a, kind):
    """least k >= MIN_EXPONENT with a <= 127 * 2^k (int8) or a <= 448 * 2^k (e4m3)"""
    bits = a.float().view(torch.int32)
    top, limit = (6, 0x7E0000) if kind == "int8" else (8, 0x600000)
    return ((bits >> 23) - 127 - top + ((bits & 0x7FFFFF) > limit)).clamp(min=MIN_EXPONENT)


def _power(k):
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _encode(x, kind):
    """codes (as bytes) of values within the range of the type"""
    if kind == "int8":
        return x.round().to(torch.int8).view(torch.uint8)
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _decode(codes, kind):
    return (codes.view(torch.int8) if kind == "int8" else codes.view(torch.float8_e4m3fn)).float()


def _typed(data, kind):
    return data.view(torch.int8) if kind == "int8" else data.view(torch.float8_e4m3fn)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    pick = lambda n: torch.randperm(n, generator=g, device=dev)  # noqa: E731
    c = dict(case)
    T, H, D = c["page"], c["kv_heads"], c["dim"]
    paged = c["op"] in ("branch", "compact")
    kind = "int8" if paged else c["cache"]
    lengths = torch.tensor(_lengths(c), device=dev)
    n = len(lengths)
    entries = (lengths + T - 1) // T
    live = int(entries.sum())
    spare = c["spare"] + n * (1 + c["children"]) if paged else 8 + live // 8
    pool, layers = live + spare, c.get("layers", 1)
    sequences = n * (1 + c.get("children", 0)) + 3
    width = int(entries.max()) + 2
    # the table: the sequences in an order of their own, their pages scattered over the pool
    tables = torch.full((sequences, width), -1, dtype=torch.int32, device=dev)
    order = pick(sequences).to(torch.int32)
    ids = order[:n].contiguous()
    where = torch.arange(width, device=dev)[None] < entries[:, None]
    part = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    part[where] = pick(pool)[:live].to(torch.int32)
    tables[ids.long()] = part
    refs = torch.zeros(pool, dtype=torch.int32, device=dev)
    refs[part[where].long()] = 1
    held = torch.zeros(sequences, dtype=torch.int32, device=dev)
    held[ids.long()] = torch.tensor(_tokens_of(c), dtype=torch.int32, device=dev)
    s = {"case": c, "kind": kind, "tables": tables, "refs": refs, "lengths": held, "ids": ids,
         "status": torch.zeros(1, dtype=torch.int32, device=dev)}
    data = torch.empty((layers, pool, 2, H, T, D), dtype=torch.uint8, device=dev)
    scales = torch.empty((layers, pool, 2, H), dtype=torch.float32, device=dev)
    if paged:
        for layer in range(layers):
            data[layer].random_(0, 256, generator=g)
        scales.copy_(_power(torch.randint(-12, 3, scales.shape, generator=g, device=dev)))
        if c["op"] == "compact":
            s.update(tables0=tables.clone(), refs0=refs.clone())
        else:
            s["parents"] = ids.repeat(c["children"])
            s["forks"] = order[n:n * (1 + c["children"])].contiguous()
            s["all"] = torch.cat((s["forks"], ids))
            s["back"] = torch.cat((torch.zeros_like(s["forks"]), lengths.to(torch.int32)))
            s["ones"] = torch.ones_like(s["all"])
    else:
        # keys with a few large channels, values whose size differs from page to page
        channel = torch.exp(0.5 * normal(H, 1, D))
        for half in (0, 1):
            x = normal(pool, H, T, D) * (channel if half == 0 else torch.exp(0.7 * normal(pool, H, 1, 1)))
            scale = _power(_largest_exponent(x.abs().amax((2, 3)), kind))
            x /= scale[:, :, None, None]
            if half:
                x = x.transpose(2, 3).contiguous().view(pool, H, T, D)
            data[0, :, half] = _encode(x, kind)
            scales[0, :, half] = scale
        rows = torch.tensor(_rows(c), device=dev)
        s["starts"] = torch.cat((rows.new_zeros(1), rows.cumsum(0))).to(torch.int32)
        total, t = sum(_rows(c)), TYPES[c["type"]]
        if c["op"] == "append":
            s["key"] = (normal(total, H, D) * channel[:, 0]).to(t)
            s["value"] = (normal(total, H, D) * torch.exp(0.7 * normal(total, H, 1))).to(t)
        else:
            s["query"] = (normal(total, c["heads"], D) * 1.5).to(t)
            s["gate"] = normal(total, c["heads"], D).to(t) if c["gate"] else None
    s.update(data=data, scales=scales)
    if own:
        s["cache"] = _package().KVPages(data, scales, refs, tables, held, s["status"], kind)
    return s


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.8-27b-in-c_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from q38hip import kv
    return kv


# ---- one pass --------------------------------------------------------------------


def run(s):
    op = s["case"]["op"]
    if own:
        cache = s["cache"]
        if op == "attention":
            return {"out": cache.attention(0, s["query"], s["ids"], s["starts"], gate=s["gate"])}
        if op == "append":
            cache.append(0, s["key"], s["value"], s["ids"], s["starts"])
            return {"codes": _typed(s["data"], s["kind"]), "scales": s["scales"]}
        if op == "branch":
            cache.truncate(s["all"], s["back"])
            cache.fork(s["parents"], s["forks"])
            cache.extend(s["all"], s["ones"])
        else:
            s["tables"].copy_(s["tables0"])
            s["refs"].copy_(s["refs0"])
            cache.compact()
    elif op == "attention":
        return {"out": _plain_attention(s)}
    elif op == "append":
        _plain_append(s)
        return {"codes": _typed(s["data"], s["kind"]), "scales": s["scales"]}
    elif op == "branch":
        _plain_truncate(s, s["all"], s["back"])
        _plain_fork(s, s["parents"], s["forks"])
        _plain_extend(s, s["all"], s["ones"])
    else:
        # the pool as the sequences that ended left it; the pages that move stay intact at their old places
        s["tables"].copy_(s["tables0"])
        s["refs"].copy_(s["refs0"])
        _plain_compact(s)
    return {"tables": s["tables"], "lengths": s["lengths"], "refs": s["refs"], "data": s["data"], "scales": s["scales"]}


def _plain_attention(s):
    c, dev = s["case"], s["data"].device
    T, H, D, S = c["page"], c["kv_heads"], c["dim"], len(s["ids"])
    G, R, E = c["heads"] // H, max(_rows(c)), _up(c["tokens"], T)
    n = s["lengths"][s["ids"].long()].long()
    starts = s["starts"].long()
    r = starts[1:] - starts[:-1]
    page = s["tables"][s["ids"].long(), :E].long().clamp(min=0)
    scale = s["scales"][0][page]
    key = _decode(s["data"][0, :, 0][page], s["kind"]) * scale[:, :, 0, :, None, None]
    key = key.permute(0, 2, 1, 3, 4).reshape(S, H, E * T, D)
    value = _decode(s["data"][0, :, 1][page], s["kind"]).view(S, E, H, D, T) * scale[:, :, 1, :, None, None]
    value = value.permute(0, 2, 1, 4, 3).reshape(S, H, E * T, D)
    t = torch.arange(R, device=dev)
    row = (starts[:-1, None] + t).clamp(max=len(s["query"]) - 1)
    query = s["query"].float()[row].view(S, R, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, R * G, D)
    scores = torch.matmul(query, key.transpose(2, 3).contiguous()) * D ** -0.5
    last = n[:, None] - r[:, None] + t
    seen = torch.arange(E * T, device=dev) <= last[:, :, None]
    scores = scores.view(S, H, R, G, E * T).masked_fill_(~seen[:, None, :, None], -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=-1e30))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(S, H, R * G, E * T), value).view(S, H, R, G, D)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 2, 1, 3, 4).reshape(S, R, c["heads"], D)[t < r[:, None]]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(TYPES[c["type"]])


def _plain_append(s):
    c, dev, kind = s["case"], s["data"].device, s["kind"]
    T, H, D, S = c["page"], c["kv_heads"], c["dim"], len(s["ids"])
    n = s["lengths"][s["ids"].long()].long()
    starts = s["starts"].long()
    first = n - (starts[1:] - starts[:-1])
    entry = first[:, None] // T + torch.arange(_up(max(_rows(c)) - 1, T) + 1, device=dev)
    touched = entry * T < n[:, None]
    page = s["tables"][s["ids"].long()[:, None], entry.clamp(max=s["tables"].shape[1] - 1)].long().clamp(min=0)
    position = entry[:, :, None] * T + torch.arange(T, device=dev)
    new = (position >= first[:, None, None]) & (position < n[:, None, None])
    old = position < first[:, None, None]
    row = (starts[:-1, None, None] + position - first[:, None, None]).clamp(0, len(s["key"]) - 1)
    new5, old5 = new[:, :, None, :, None], old[:, :, None, :, None]
    for half, x in ((0, s["key"]), (1, s["value"])):
        x = x.float()[row].permute(0, 1, 3, 2, 4)                      # [sequence, page, head, token, dim]
        finite = (x.isfinite() | ~new5).all(-1).all(-1)
        x = torch.where(new5 & x.isfinite(), x, 0.0)
        was = s["scales"][0, page, half]
        now = _power(_largest_exponent(x.abs().amax((3, 4)), kind))
        now = torch.where(finite, now, math.nan)
        has_old = old.any(-1)[:, :, None]
        now = torch.where(has_old & ~(now > was) & ~now.isnan() | has_old & was.isnan(), was, now)
        codes = s["data"][0, page, half]
        if half:
            codes = codes.view(S, -1, H, D, T).transpose(3, 4)
        grown = _encode(_decode(codes, kind) * (was / now)[..., None, None].nan_to_num(1.0, 1.0, 1.0).clamp(max=1.0), kind)
        fresh = _encode((x / now[..., None, None]).nan_to_num(0.0), kind)
        grows = (has_old & (now > was))[..., None, None]
        codes = torch.where(new5, fresh, torch.where(old5 & grows, grown, codes))
        if half:
            codes = codes.transpose(3, 4).contiguous().view(S, -1, H, T, D)
        s["data"][0, page[touched], half] = codes[touched]
        s["scales"][0, page[touched], half] = now[touched]


def _plain_truncate(s, ids, lengths):
    ids, T = ids.long(), s["case"]["page"]
    lengths = torch.minimum(s["lengths"][ids], lengths)
    table = s["tables"][ids]
    entry = torch.arange(table.shape[1], device=table.device)
    drop = (entry >= ((lengths + T - 1) // T)[:, None]) & (table >= 0)
    pages = table[drop].long()
    s["refs"].index_add_(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    s["tables"][ids] = table.masked_fill(drop, -1)
    s["lengths"][ids] = lengths


def _plain_fork(s, parents, children):
    table = s["tables"][parents.long()]
    pages = table[table >= 0].long()
    s["refs"].index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    s["tables"][children.long()] = table
    s["lengths"][children.long()] = s["lengths"][parents.long()]


def _plain_extend(s, ids, rows):
    ids, T, refs = ids.long(), s["case"]["page"], s["refs"]
    before = s["lengths"][ids].long()
    after = before + rows
    table = s["tables"][ids].long()
    tail = torch.where(before % T != 0, table.gather(1, (before // T).clamp(max=table.shape[1] - 1)[:, None])[:, 0], -1)
    turn = ((tail[:, None] == tail[None]) & (tail >= 0)).tril(-1).sum(1)
    copy = (tail >= 0) & (refs[tail.clamp(min=0)] - turn > 1)
    begin = torch.where(copy, before // T, (before + T - 1) // T)
    entry = torch.arange(table.shape[1], device=table.device)
    fresh = (entry >= begin[:, None]) & (entry < ((after + T - 1) // T)[:, None])
    pages = (refs == 0).nonzero()[: int(fresh.sum()), 0]
    table[fresh] = pages
    source = tail[copy]
    target = table.gather(1, (before // T).clamp(max=table.shape[1] - 1)[:, None])[:, 0][copy]
    s["data"][:, target] = s["data"][:, source]
    s["scales"][:, target] = s["scales"][:, source]
    refs.index_add_(0, source, torch.full_like(source, -1, dtype=torch.int32))
    refs[pages] = 1
    s["tables"][ids] = table.to(torch.int32)
    s["lengths"][ids] = after.to(torch.int32)


def _plain_compact(s):
    refs = s["refs"]
    used = refs > 0
    live = int(used.sum())
    holes = (~used[:live]).nonzero()[:, 0]
    movers = used[live:].nonzero()[:, 0] + live
    s["data"][:, holes] = s["data"][:, movers]
    s["scales"][:, holes] = s["scales"][:, movers]
    place = torch.arange(len(refs), device=refs.device, dtype=torch.int32)
    place[movers] = holes.to(torch.int32)
    refs[holes] = refs[movers]
    refs[movers] = 0
    s["tables"].copy_(torch.where(s["tables"] >= 0, place[s["tables"].long().clamp(min=0)], s["tables"]))


# ---- the definition, in 64 bits ----------------------------------------------------


def exact(case, seed):
    if case["op"] not in ("attention", "append"):
        return None
    s = prepare(case, seed)
    c, T, H, D = case, case["page"], case["kv_heads"], case["dim"]
    ends = [0]
    for r in _rows(c):
        ends.append(ends[-1] + r)
    sizes = _tokens_of(c)
    if c["op"] == "append":
        codes = _typed(s["data"], s["kind"])[0].double().reshape(-1, 2, H, T * D)
        scales = s["scales"][0].double()
        largest = 127.0 if s["kind"] == "int8" else 448.0
        snap = torch.round if s["kind"] == "int8" else _nearest_e4m3
        for i, seq in enumerate(s["ids"].tolist()):
            n, r = sizes[i], ends[i + 1] - ends[i]
            at = n - r
            while at < n:
                page, used = int(s["tables"][seq, at // T]), at % T
                end = min(n, (at // T + 1) * T)
                rows = slice(ends[i] + at - (n - r), ends[i] + end - (n - r))
                for half, x in ((0, s["key"][rows].double()), (1, s["value"][rows].double())):
                    m, k = torch.frexp((x.abs().amax((0, 2)) / largest).clamp(min=2.0 ** -120))
                    size = _power64((k - (m == 0.5).int()).clamp(min=MIN_EXPONENT))
                    was = scales[page, half]
                    size = torch.maximum(size, was) if used else size
                    block = codes[page, half].view(H, D, T).transpose(1, 2) if half else codes[page, half].view(H, T, D)
                    if used:
                        block[:, :used] = snap(block[:, :used] * (was / size)[:, None, None])
                    block[:, used:used + end - at] = snap(x.transpose(0, 1) / size[:, None, None])
                    scales[page, half] = size
                at = end
        shape = s["data"].shape
        return {"codes": codes.view(shape) if s["kind"] != "int8" else None, "scales": scales[None]}
    out = torch.zeros((ends[-1], c["heads"], D), dtype=torch.float64, device="cuda")
    G = c["heads"] // H
    for i, seq in enumerate(s["ids"].tolist()):
        n, r = sizes[i], ends[i + 1] - ends[i]
        if not n or not r:
            continue
        pages = s["tables"][seq, : _up(n, T)].long()
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - r, n, device="cuda")[:, None]
        for h in range(H):
            codes = _typed(s["data"][0], s["kind"])[pages][:, :, h].double()
            sizes_h = s["scales"][0, pages, :, h].double()[:, :, None, None]
            k = (codes[:, 0] * sizes_h[:, 0]).reshape(-1, D)[:n]
            v = (codes[:, 1].reshape(-1, D, T) * sizes_h[:, 1]).transpose(1, 2).reshape(-1, D)[:n]
            for j in range(h * G, (h + 1) * G):
                z = s["query"][ends[i]:ends[i + 1], j].double() @ k.t().contiguous() / math.sqrt(D)
                out[ends[i]:ends[i + 1], j] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v
    if s["gate"] is not None:
        out /= 1 + torch.exp(-s["gate"].double())
    return {"out": out}


def _power64(k):
    return ((k.long() + 1023) << 52).view(torch.float64)


def _nearest_e4m3(x):
    """the nearest multiple of the spacing of e4m3 at |x| (2^-9 below 2^-6), ties to an even multiple"""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = _power64(e - 4)
    return torch.round(x / step) * step
