"""Measured cases of a decoder layer's operators over rows in 8 bits and over
packed prompts.

Rows in 8 bits are e4m3 codes with one power of two for each 128 neighbours of
a row (scales [rows, blocks rounded up to 4], e8m0): 2^k, k >= -100 the least
with the largest magnitude of the block <= 448 * 2^k.

  norm       root-mean-square norm of a row, after the residual's addition,
             into rows in 8 bits or into the rows' type
  quantize   rows into 8 bits, multiplied by silu(gate) on the way (SwiGLU)
  product    rows in 8 bits times a weight matrix in e4m3, [outputs, inputs],
             with an fp32 scale for each 128 x 128 block
  rotary     rotary positions: pairs of channels turned by position * frequency,
             interleaved or a half apart, in the first channels of each head
  attention  causal attention of packed prompts of different lengths, grouped
             heads, optionally times sigmoid(gate)

With `own` false everything is plain torch on the same tensors; with `own`
true the calls go through q38hip.layer.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 128
MIN_EXPONENT = -100
EPS = 1e-6


def _norm(name, kind, rows, width, add=True, e4m3=True, offset=0.0):
    return {"name": name, "op": "norm", "type": kind, "rows": rows, "width": width, "add": add, "e4m3": e4m3, "offset": offset}


def _quantize(name, kind, rows, width, gate=True):
    return {"name": name, "op": "quantize", "type": kind, "rows": rows, "width": width, "gate": gate}


def _product(name, kind, rows, inputs, outputs):
    return {"name": name, "op": "product", "type": kind, "rows": rows, "inputs": inputs, "outputs": outputs}


def _rotary(name, kind, rows, heads, dim, turned, interleaved, first, factor=1.0):
    return {"name": name, "op": "rotary", "type": kind, "rows": rows, "heads": heads, "dim": dim, "turned": turned,
            "interleaved": interleaved, "first": first, "factor": factor}


def _attention(name, kind, heads, kv_heads, dim, count, tokens, gate=False):
    return {"name": name, "op": "attention", "type": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "count": count,
            "tokens": tokens, "gate": gate}


def listed():
    return [
        # one new token of a chat in front of a projection: launch latency is all there is
        _norm("norm_token", "bf16", 1, 5120),
        # a whole prompt in front of a projection
        _norm("norm_prompt", "bf16", 4096, 5120),
        # the feed-forward's middle in a serving step of many sequences
        _quantize("swiglu_step", "bf16", 48, 17408),
        # the same over a prompt
        _quantize("swiglu_prompt", "bf16", 4096, 17408),
        # one token through the gate and up matrices
        _product("product_token", "bf16", 1, 5120, 34816),
        # a serving step through the down matrix
        _product("product_batch", "bf16", 48, 17408, 5120),
        # a prompt through the gate and up matrices
        _product("product_prompt", "bf16", 4096, 5120, 34816),
        # queries and keys of a serving step, a quarter of the head turned
        _rotary("rotary_step", "f32", 16, 28, 256, 64, False, 6000),
        # queries and keys of a prompt late in a long document, whole heads of neighbouring pairs
        _rotary("rotary_prompt", "bf16", 8192, 40, 128, 128, True, 250000, 4.0),
        # the first question of a chat
        _attention("attention_short", "f32", 24, 4, 256, 1, 37, gate=True),
        # prompts of several users in one call
        _attention("attention_packed", "bf16", 32, 8, 128, 12, 1500),
        # one long prompt
        _attention("attention_prompt", "bf16", 24, 4, 256, 1, 8197, gate=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "quantize", "product", "product", "rotary", "attention", "attention"))
    kind = rng.choice(tuple(TYPES))
    if op in ("norm", "quantize"):
        width = rng.choice((5120, 6144, 17408, 2048, _log_int(rng, 64, 20000), 16 * _log_int(rng, 4, 1200)))
        rows = _log_int(rng, 1, min(6000, 40000000 // width))
        c = _norm("", kind, rows, width, rng.random() < 0.7, rng.random() < 0.6, rng.choice((0.0, 1.0))) if op == "norm" else \
            _quantize("", kind, rows, width, rng.random() < 0.7)
    elif op == "product":
        inputs = rng.choice((5120, 6144, 17408, 2048, 16 * _log_int(rng, 4, 1200)))
        outputs = rng.choice((5120, 14336, 17408, _log_int(rng, 16, 40000)))
        rows = rng.choice((_log_int(rng, 1, 16), _log_int(rng, 8, 128), _log_int(rng, 64, 4096)))
        rows = max(1, min(rows, int(7e11) // (inputs * outputs)))
        c = _product("", kind, rows, inputs, outputs)
    elif op == "rotary":
        heads, dim = rng.choice(((28, 256), (40, 128), (32, 64), (9, 96), (1, 80)))
        turned = rng.choice((dim, dim // 2, dim // 4 // 2 * 2))
        rows = _log_int(rng, 1, max(2, 40000000 // (heads * dim)))
        c = _rotary("", kind, rows, heads, dim, turned, rng.random() < 0.5, _log_int(rng, 1, 1000000), rng.choice((1.0, 4.0, 32.0)))
    else:
        heads, kv_heads, dim = rng.choice(((24, 4, 256), (32, 8, 128), (16, 16, 64), (12, 1, 128), (5, 5, 256), (40, 8, 64)))
        count = _log_int(rng, 1, 24)
        tokens = _log_int(rng, 1, 4000 if count == 1 else 8000 // count)
        c = _attention("", kind, heads, kv_heads, dim, count, tokens, rng.random() < 0.4)
    del c["name"]
    return c


# ---- sizes that follow from a case --------------------------------------------


def _up(a, b):
    return -(-a // b)


def _pitch(width):
    return _up(_up(width, BLOCK), 4) * 4


def _lengths(c):
    """tokens of each sequence: the largest first, the others spread below it over the logarithm"""
    low = c["tokens"] ** 0.5
    return [max(1, round(low * (c["tokens"] / low) ** (1 - i * 0.618034 % 1))) for i in range(c["count"])]


def work(c):
    size = TYPES[c["type"]].itemsize
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        out = n + c["rows"] * _up(c["width"], BLOCK) if c["e4m3"] else n * size
        return {"bytes": n * size * (3 if c["add"] else 1) + c["width"] * 4 + out, "flops": 5 * n}
    if c["op"] == "quantize":
        n = c["rows"] * c["width"]
        return {"bytes": n * size * (2 if c["gate"] else 1) + n + c["rows"] * _up(c["width"], BLOCK), "flops": 6 * n}
    if c["op"] == "product":
        m, k, n = c["rows"], c["inputs"], c["outputs"]
        return {"bytes": k * n + _up(k, BLOCK) * (_up(n, BLOCK) * 4 + m) + m * (k + n * size), "flops": 2 * m * k * n}
    if c["op"] == "rotary":
        n = c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * size + c["rows"] * 4 + c["turned"] * 2, "flops": 3 * c["rows"] * c["heads"] * c["turned"]}
    lengths = _lengths(c)
    row = c["heads"] * c["dim"] * (3 if c["gate"] else 2) + 2 * c["kv_heads"] * c["dim"]
    return {"bytes": sum(lengths) * row * size + (c["count"] + 1) * 4,
            "flops": 4 * c["dim"] * c["heads"] * sum(n * (n + 1) // 2 for n in lengths)}


# ---- inputs --------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    c, t = dict(case), TYPES[case["type"]]
    s = {"case": c}
    if c["op"] == "norm":
        # a residual stream: a few channels far larger than the others
        channel = torch.exp(0.8 * normal(c["width"]))
        s["x"] = (normal(c["rows"], c["width"]) * channel * 3).to(t)
        s["addend"] = normal(c["rows"], c["width"]).to(t) if c["add"] else None
        s["weight"] = 1 - c["offset"] + 0.2 * normal(c["width"])
    elif c["op"] == "quantize":
        if c["gate"]:
            # the two halves of one projection's output
            both = (normal(c["rows"], 2 * c["width"]) * 2).to(t)
            s["gate"], s["x"] = both[:, :c["width"]], both[:, c["width"]:]
        else:
            s["gate"], s["x"] = None, (normal(c["rows"], c["width"]) * torch.exp(normal(c["rows"], 1))).to(t)
    elif c["op"] == "product":
        m, k, n = c["rows"], c["inputs"], c["outputs"]
        s["codes"], s["scales"] = _plain_quantize(normal(m, k) * torch.exp(0.5 * normal(k)))
        blocks = (_up(n, BLOCK), _up(k, BLOCK))
        # codes whose blocks reach the type's largest value, and the blocks' scales
        s["weight"] = (normal(n, k) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s["weight_scales"] = torch.exp(0.3 * normal(*blocks)) * (0.01 / math.sqrt(k))
    elif c["op"] == "rotary":
        s["x"] = normal(c["rows"], c["heads"], c["dim"]).to(t)
        # the tokens of a prompt from its place in the document on, or of many sequences
        at = torch.arange(c["rows"], device=dev) if c["rows"] > 64 else torch.randint(0, 1000, (c["rows"],), generator=g, device=dev)
        s["positions"] = (at + c["first"] + seed % 7).to(torch.int32)
        pairs = torch.arange(0, c["turned"], 2, dtype=torch.float64, device=dev)
        s["frequencies"] = (1000000.0 ** (-pairs / c["turned"]) / c["factor"]).float()
        s["magnitude"] = 1.0 if c["factor"] == 1 else 0.1 * math.log(c["factor"]) + 1
    else:
        lengths = torch.tensor(_lengths(c), device=dev)
        total = int(lengths.sum())
        s["starts"] = torch.cat((lengths.new_zeros(1), lengths.cumsum(0))).to(torch.int32)
        channel = torch.exp(0.5 * normal(c["kv_heads"], c["dim"]))
        s["query"] = (normal(total, c["heads"], c["dim"]) * 1.5).to(t)
        s["key"] = (normal(total, c["kv_heads"], c["dim"]) * channel).to(t)
        s["value"] = (normal(total, c["kv_heads"], c["dim"]) * torch.exp(0.7 * normal(total, c["kv_heads"], 1))).to(t)
        s["gate"] = normal(total, c["heads"], c["dim"]).to(t) if c["gate"] else None
    return s


_LAYER = None


def _layer():
    global _LAYER
    if _LAYER is None:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen3.8-27b-in-c_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        from q38hip import layer
        _LAYER = layer
    return _LAYER


# ---- one pass --------------------------------------------------------------------


def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        layer = _layer()
        if op == "norm":
            y = layer.rms_norm(s["x"], s["weight"], EPS, addend=s["addend"], offset=c["offset"], e4m3=c["e4m3"])
            return _norm_outputs(c, *(y if c["add"] else (y, None)))
        if op == "quantize":
            codes, scales = layer.quantize(s["x"], gate=s["gate"])
            return {"codes": codes, "scales": scales}
        if op == "product":
            return {"out": layer.product((s["codes"], s["scales"]), s["weight"], s["weight_scales"], TYPES[c["type"]])}
        if op == "rotary":
            return {"out": layer.rotary(s["x"], s["positions"], s["frequencies"], interleaved=c["interleaved"],
                                        magnitude=s["magnitude"])}
        return {"out": layer.attention(s["query"], s["key"], s["value"], s["starts"], gate=s["gate"])}
    if op == "norm":
        return _norm_outputs(c, *_plain_norm(s))
    if op == "quantize":
        x = s["x"].float()
        if s["gate"] is not None:
            gate = s["gate"].float()
            x = gate / (1 + torch.exp(-gate)) * x
        codes, scales = _plain_quantize(x)
        return {"codes": codes, "scales": scales}
    if op == "product":
        return {"out": _plain_product(s)}
    if op == "rotary":
        return {"out": _plain_rotary(s)}
    return {"out": _plain_attention(s)}


def _norm_outputs(c, y, total):
    out = {"codes": y[0], "scales": y[1]} if c["e4m3"] else {"out": y}
    if c["add"]:
        out["total"] = total
    return out


def _plain_quantize(x):
    """codes and scales of fp32 rows"""
    rows, width = x.shape
    blocks, pitch = _up(width, BLOCK), _pitch(width)
    y = torch.nn.functional.pad(x, (0, blocks * BLOCK - width)).view(rows, blocks, BLOCK)
    bits = y.abs().amax(2).view(torch.int32)
    # 448 = 1.75 * 2^8
    k = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=MIN_EXPONENT)
    codes = (y * ((127 - k) << 23).view(torch.float32)[:, :, None]).view(rows, blocks * BLOCK)[:, :width]
    scales = torch.zeros((rows, pitch), dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = k + 127
    return codes.to(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _plain_norm(s):
    c, x, total = s["case"], s["x"], None
    if s["addend"] is not None:
        x = total = (x.float() + s["addend"].float()).to(x.dtype)
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * (s["weight"] + c["offset"])
    return (_plain_quantize(y) if c["e4m3"] else y.to(s["x"].dtype)), total


def _spread(scales, rows, width):
    """scales of 128 x 128 blocks for each value"""
    return scales.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :width]


def _plain_product(s):
    m, k = s["codes"].shape
    scales = s["scales"].view(torch.uint8)[:, :_up(k, BLOCK)].to(torch.int32) << 23
    x = s["codes"].float() * scales.view(torch.float32).repeat_interleave(BLOCK, 1)[:, :k]
    w = s["weight"].float() * _spread(s["weight_scales"], len(s["weight"]), k)
    return torch.matmul(x, w.t()).to(TYPES[s["case"]["type"]])


def _plain_rotary(s):
    c = s["case"]
    x, n = s["x"].float(), s["case"]["turned"]
    # the angles of far positions need 64 bits
    angle = (s["positions"].double()[:, None] * s["frequencies"].double())[:, None]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if c["interleaved"] else (x[..., :n // 2], x[..., n // 2:n])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((p, q), -1).flatten(2) if c["interleaved"] else torch.cat((p, q), -1)
    return torch.cat((turned, x[..., n:]), -1).to(s["x"].dtype)


def _plain_attention(s):
    c = s["case"]
    heads, groups, n = c["heads"], c["kv_heads"], len(s["query"])
    at = torch.arange(n, device=s["query"].device)
    sequence = torch.bucketize(at, s["starts"][1:], right=True)
    seen = (sequence[:, None] == sequence) & (at[:, None] >= at)
    query = s["query"].float().permute(1, 0, 2).reshape(groups, heads // groups * n, c["dim"])
    key = s["key"].float().permute(1, 2, 0).contiguous()
    scores = torch.matmul(query, key).view(groups, heads // groups, n, n) * c["dim"] ** -0.5
    scores.masked_fill_(~seen, -math.inf)
    weight = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weight.sum(-1, keepdim=True)
    value = s["value"].float().permute(1, 0, 2).contiguous()
    out = torch.matmul(weight.view(groups, heads // groups * n, n), value).view(groups, heads // groups, n, c["dim"]) / total
    out = out.permute(2, 0, 1, 3).reshape(n, heads, c["dim"])
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    return out.to(s["query"].dtype)


# ---- the definitions in 64 bits --------------------------------------------------


def _exact_codes(y):
    """values in units of their block's scale, before their rounding to e4m3, and the scales"""
    rows, width = y.shape
    blocks = _up(width, BLOCK)
    codes = torch.empty_like(y)
    scales = torch.full((rows, _pitch(width)), 2.0 ** -127, dtype=torch.float64, device=y.device)
    for i in range(blocks):
        part = y[:, i * BLOCK:(i + 1) * BLOCK]
        # 448 = 0.875 * 2^9: the least k with largest <= 448 * 2^k, from largest / 448 = f * 2^e, 0.5 <= f < 1
        f, e = torch.frexp(part.abs().amax(1) / 448)
        k = torch.where(f == 0.5, e - 1, e).clamp(min=MIN_EXPONENT)
        unit = torch.ldexp(torch.ones_like(f), torch.where(f == 0, torch.full_like(k, MIN_EXPONENT), k))
        codes[:, i * BLOCK:(i + 1) * BLOCK] = part / unit[:, None]
        scales[:, i] = unit
    return codes, scales


def exact(case, seed):
    s = prepare(case, seed)
    c, op = s["case"], case["op"]
    if op == "norm":
        x, total = s["x"].double(), None
        if s["addend"] is not None:
            # the sum is an output of its own: what is normalised is what is stored
            total = x + s["addend"].double()
            x = total.float().to(s["x"].dtype).double()
        mean = torch.linalg.vector_norm(x, dim=1).square() / c["width"]
        y = x / torch.sqrt(mean + EPS)[:, None] * (s["weight"].double() + c["offset"])
        return _norm_outputs(c, _exact_codes(y) if c["e4m3"] else y, total)
    if op == "quantize":
        y = s["x"].double()
        if s["gate"] is not None:
            y = y * s["gate"].double() * torch.sigmoid(s["gate"].double())
        codes, scales = _exact_codes(y)
        return {"codes": codes, "scales": scales}
    if op == "product":
        m, k = s["codes"].shape
        out = torch.zeros((m, c["outputs"]), dtype=torch.float64, device=s["codes"].device)
        for i in range(_up(k, BLOCK)):
            part = slice(i * BLOCK, (i + 1) * BLOCK)
            x = s["codes"][:, part].double() * s["scales"][:, i].double()[:, None]
            w = s["weight"][:, part].double() * s["weight_scales"][:, i].double().repeat_interleave(BLOCK)[:c["outputs"], None]
            out.addmm_(x, w.t())
        return {"out": out}
    if op == "rotary":
        n = c["turned"]
        turn = torch.polar(torch.full((1,), s["magnitude"], dtype=torch.float64, device=s["x"].device),
                           torch.outer(s["positions"].double(), s["frequencies"].double()))[:, None]
        out = s["x"].double()
        if c["interleaved"]:
            z = torch.view_as_complex(out[..., :n].unflatten(-1, (n // 2, 2)).contiguous()) * turn
            out[..., 0:n:2], out[..., 1:n:2] = z.real, z.imag
        else:
            z = torch.complex(out[..., :n // 2], out[..., n // 2:n]) * turn
            out[..., :n // 2], out[..., n // 2:n] = z.real, z.imag
        return {"out": out}
    starts = s["starts"].tolist()
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=s["query"].device)
    for a, b in zip(starts, starts[1:]):
        hidden = torch.ones((b - a, b - a), dtype=torch.bool, device=out.device).triu_(1)
        for h in range(c["heads"]):
            j = h * c["kv_heads"] // c["heads"]
            scores = s["query"][a:b, h].double() @ s["key"][a:b, j].double().t() / math.sqrt(c["dim"])
            weight = torch.softmax(scores.masked_fill_(hidden, -math.inf), 1)
            out[a:b, h] = weight @ s["value"][a:b, j].double()
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return {"out": out}
