"""What a decoder layer's operators refuse on the host (section 4 of
include/q38hip.h, q38hip/layer.py), and the frequencies of rotary positions."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import q38hip
from q38hip import layer

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096            # an aligned address that no refused call follows
BIG = (1 << 24) + 16


def test_exports():
    declared = open(os.path.join(ROOT, "include", "q38hip.h")).read()
    for name in layer.EXPORTS:
        assert name + "(" in declared and hasattr(q38hip.lib(), name)


def _refused(name, good, changes):
    """a call of the C function with each change of its arguments is refused, with a message"""
    function = getattr(layer._lib(), name)
    for change in changes:
        arguments = dict(good, **change)
        assert set(arguments) == set(good), change
        assert function(*arguments.values()) == 0 and q38hip.last_error(), change


def test_pitch():
    lib = layer._lib()
    for width in (1, 127, 128, 129, 512, 513, 5120, 17408, 1 << 24):
        assert lib.q38hip_e4m3_scale_pitch(width) == layer.scale_pitch(width) == -(-width // 512) * 4
    assert lib.q38hip_e4m3_scale_pitch(0) == 0 and lib.q38hip_e4m3_scale_pitch((1 << 24) + 1) == 0


def test_quantize_refuses():
    good = dict(codes=2 * P, scales=3 * P, x=P, x_row=128, gate=None, gate_row=0, type=0, width=128, rows=2, stream=None)
    _refused("q38hip_quantize_e4m3", good, [
        dict(codes=None), dict(scales=None), dict(x=None), dict(type=2), dict(width=0), dict(rows=0), dict(width=BIG, x_row=BIG),
        dict(rows=BIG), dict(x_row=127), dict(gate=P, gate_row=127), dict(x=P + 2), dict(x=P + 1, type=1), dict(gate=P + 2, gate_row=128),
        dict(rows=1 << 23, width=1 << 18, x_row=1 << 18), dict(rows=1 << 24, width=4096, x_row=4096), dict(codes=P),
        dict(gate=2 * P, gate_row=128)])


def test_norm_refuses():
    good = dict(output=P, output_row=256, codes=None, scales=None, total=None, total_row=0, x=2 * P, x_row=256, addend=None,
                addend_row=0, type=30, weight=3 * P, weight_type=0, offset=0.0, eps=1e-6, width=256, rows=3, stream=None)
    added = dict(addend=4 * P, addend_row=256, total=5 * P, total_row=256)
    _refused("q38hip_rms_norm", good, [
        dict(output=None), dict(codes=P), dict(scales=P), dict(addend=P, addend_row=256), dict(total=P, total_row=256), dict(x=None),
        dict(weight=None), dict(type=3), dict(weight_type=12), dict(width=0), dict(rows=0), dict(rows=BIG), dict(width=BIG),
        dict(x_row=255), dict(output_row=255), dict(added, addend_row=255), dict(added, total_row=200),
        dict(added, total=P), dict(added, total=2 * P, total_row=512), dict(added, total=4 * P, total_row=512),
        dict(output=2 * P, output_row=512), dict(added, output=4 * P, output_row=512), dict(eps=-1.0), dict(eps=math.nan),
        dict(eps=math.inf), dict(offset=math.nan), dict(x=2 * P + 1), dict(weight=3 * P + 2), dict(output=P + 1),
        dict(added, addend=4 * P + 1), dict(added, total=5 * P + 1),
        dict(codes=2 * P, scales=7 * P), dict(codes=P, scales=7 * P), dict(added, codes=4 * P, scales=7 * P),
        dict(added, codes=5 * P, scales=7 * P), dict(rows=1 << 23, width=16384, x_row=16384, output_row=16384)])


def test_product_refuses():
    good = dict(output=4 * P, type=30, output_row=256, codes=P, scales=P, tokens=2, inputs=128, weight=2 * P, weight_scales=P, rows=256,
                workspace=None, stream=None)
    _refused("q38hip_gemm_e4m3", good, [
        dict(output=None), dict(type=8), dict(output_row=255), dict(codes=None), dict(scales=None), dict(weight=None),
        dict(weight_scales=None), dict(tokens=0), dict(inputs=0), dict(rows=0), dict(inputs=120), dict(inputs=129), dict(tokens=BIG),
        dict(inputs=BIG), dict(rows=BIG, output_row=BIG), dict(tokens=1 << 20, rows=1 << 20, output_row=1 << 20), dict(codes=P + 8),
        dict(weight=P + 4), dict(scales=P + 2), dict(weight_scales=P + 2), dict(output=P + 1), dict(workspace=P + 8),
        dict(output=P), dict(output=2 * P)])
    lib = layer._lib()
    for sizes in ((0, 128, 16), (1, 0, 16), (1, 128, 0), (1, 100, 16), (BIG, 128, 16)):
        assert lib.q38hip_gemm_e4m3_workspace_bytes(*sizes) == 0 and q38hip.last_error()


def test_rotary_refuses():
    good = dict(output=P, output_row=512, output_head=128, x=2 * P, x_row=512, x_head=128, type=1, rows=3, heads=4, dim=128,
                positions=P, frequencies=P, pairs=32, interleaved=0, magnitude=1.0, stream=None)
    _refused("q38hip_rotary", good, [
        dict(output=None), dict(x=None), dict(positions=None), dict(frequencies=None), dict(type=7), dict(rows=0), dict(heads=0),
        dict(dim=0), dict(pairs=0), dict(pairs=65), dict(dim=2048, x_head=2048, output_head=2048), dict(heads=1 << 14), dict(rows=BIG),
        dict(x_head=127), dict(output_head=127), dict(x_row=100), dict(output_row=100), dict(x=P + 1), dict(output=P + 1),
        dict(positions=P + 2), dict(frequencies=P + 1), dict(output=2 * P, output_row=1024), dict(output=2 * P, output_head=256),
        dict(magnitude=math.inf), dict(rows=1 << 24)])


def test_attention_refuses():
    good = dict(output=2 * P, output_row=512, query=P, gate=None, query_row=512, query_head=128, key=P, key_row=256, value=P,
                value_row=256, type=30, heads=4, kv_heads=2, dim=128, scale=1.0, starts=P, count=1, rows=8, stream=None)
    _refused("q38hip_prompt_attention", good, [
        dict(output=None), dict(query=None), dict(key=None), dict(value=None), dict(starts=None), dict(type=2), dict(dim=96),
        dict(dim=512), dict(heads=0), dict(kv_heads=0), dict(heads=3), dict(count=0), dict(rows=0), dict(count=BIG), dict(rows=BIG),
        dict(heads=1 << 20, kv_heads=2, rows=1 << 12, output_row=1 << 30), dict(query_head=127), dict(query_row=127), dict(key_row=255),
        dict(value_row=255), dict(output_row=511), dict(output=P + 1), dict(gate=P + 1), dict(key=P + 1), dict(starts=P + 2),
        dict(scale=math.nan), dict(heads=65536, kv_heads=65536, rows=1), dict(output=P), dict(gate=2 * P), dict(key=2 * P),
        dict(value=2 * P)])


def test_python_refuses():
    x = torch.zeros(3, 256)
    half, weight = x.half(), torch.ones(256)
    rows8 = (torch.zeros(3, 256, dtype=torch.float8_e4m3fn), torch.zeros(3, 4, dtype=torch.float8_e8m0fnu))
    heads, words = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: layer.quantize(x), lambda: layer.quantize(x.int()), lambda: layer.quantize(x[0]),
                 lambda: layer.quantize(x.t()), lambda: layer.rms_norm(x, weight), lambda: layer.rms_norm(x.t(), weight),
                 lambda: layer.product(rows8, rows8[0], torch.ones(1, 2)),
                 lambda: layer.product(rows8, rows8[0][:, :128], torch.ones(1, 1)),
                 lambda: layer.rotary(heads, words, torch.ones(8)), lambda: layer.rotary(heads[0], words, torch.ones(8)),
                 lambda: layer.attention(heads, heads, heads, words), lambda: layer.attention(heads[0], heads, heads, words),
                 lambda: layer.attention(heads.int(), heads, heads, words),
                 lambda: layer.rotary_frequencies(0), lambda: layer.rotary_frequencies(7), lambda: layer.rotary_frequencies(8, 1.0),
                 lambda: layer.rotary_frequencies(8, factor=0.5), lambda: layer.rotary_frequencies(8, factor=2, original=0)):
        with pytest.raises(ValueError):
            call()
    assert half.dtype == torch.float16


def test_frequencies():
    plain, magnitude = layer.rotary_frequencies(64, 1e6)
    assert magnitude == 1.0 and plain.dtype == torch.float32
    want = 1e6 ** (-np.arange(0, 64, 2) / 64)
    assert np.array_equal(plain.numpy(), want.astype(np.float32))
    slower, magnitude = layer.rotary_frequencies(64, 1e6, factor=4)
    assert magnitude == 1.0 and np.array_equal(slower.numpy(), (want / 4).astype(np.float32))
    original = 32768
    mixed, magnitude = layer.rotary_frequencies(64, 1e6, factor=4, original=original)
    assert magnitude == pytest.approx(0.1 * math.log(4) + 1)
    turns = original * want / (2 * np.pi)
    share = mixed.numpy() / want
    assert (share[turns >= 64] == 1).all() or np.allclose(share[turns >= 64], 1, rtol=2.0 ** -23)
    assert np.allclose(share[turns <= 0.5], 0.25, rtol=2.0 ** -23)
    assert (np.diff(share) <= 2.0 ** -22).all() and share.min() >= 0.25 * (1 - 2.0 ** -23)
    same, magnitude = layer.rotary_frequencies(64, 1e6, factor=1.0, original=original)
    assert magnitude == 1.0 and torch.equal(same, plain)


PLAN_CHECK = r"""
#include <cstdio>
#include <vector>
#include "q38_layer.h"
using namespace q38;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s (%u %u %u)\n", __LINE__, #x, m, k, n); return 1; } } while (0)
static uint32_t state = 777;
static uint32_t draw(uint32_t n) { state = state * 1664525u + 1013904223u; return (state >> 8) % n; }
int main()
{
    unsigned seen[5][3] = {};
    uint32_t m = 0, k = 0, n = 0;
    for (int i = 0; i < 30000; ++i) {
        m = draw(3) ? 1 + draw(1 + draw(5000)) : 1 + draw(70);
        k = 16 * (1 + draw(1 + draw(1200)));
        n = 1 + draw(1 + draw(40000));
        const ProductPlan p = plan_product(m, k, n);
        const uint32_t blocks = e4m3_blocks(k);
        CHECK(p.tile <= kProductTile256);
        if (p.tile == kProductFew) { CHECK(m <= 16); CHECK(p.splits == 1 && p.bytes == 0); ++seen[0][0]; continue; }
        const uint32_t tiles_n = layer_up(n, kProductRows[p.tile]), tiles_m = layer_up(m, kProductTokens[p.tile]);
        const uint64_t tiles = (uint64_t)tiles_n * tiles_m, rest = tiles - p.whole;
        CHECK(p.whole <= tiles && p.splits >= 1 && (p.splits == 1) == (rest == 0));
        CHECK(p.splits == 1 || blocks / p.splits >= 4);
        CHECK(p.bytes == (p.splits == 1 ? 0 : rest * p.splits * kProductRows[p.tile] * kProductTokens[p.tile] * 4));
        ++seen[p.tile][p.splits == 1 ? 0 : p.whole ? 1 : 2];
        /* every tile once, whole or cut, and every block of inputs of a cut one once */
        if (i % 16 == 0) {
            std::vector<unsigned> got(tiles);
            for (uint32_t b = 0; b < p.whole; ++b) {
                const TilePlace t = tile_place(die_place(b, p.whole), tiles_n, tiles_m);
                CHECK(t.n < tiles_n && t.m < tiles_m);
                got[t.n + (uint64_t)t.m * tiles_n] += blocks;
            }
            const uint32_t all = (uint32_t)rest * p.splits;
            for (uint32_t b = 0; b < all; ++b) {
                const uint32_t place = die_place(b, all), tile = place / p.splits, split = place % p.splits;
                const TilePlace t = tile_place(p.whole + tile, tiles_n, tiles_m);
                const uint32_t from = (uint64_t)blocks * split / p.splits, to = (uint64_t)blocks * (split + 1) / p.splits;
                CHECK(t.n < tiles_n && t.m < tiles_m && from < to);
                got[t.n + (uint64_t)t.m * tiles_n] += to - from;
            }
            for (unsigned g : got) CHECK(g == blocks);
        }
    }
    for (int t = 0; t < 5; ++t) std::printf("%u %u %u\n", seen[t][0], seen[t][1], seen[t][2]);
    return 0;
}
"""


def test_product_plans(tmp_path):
    """every tile of a product is formed once, every plan is met by some size"""
    source = tmp_path / "plan.cpp"
    source.write_text(PLAN_CHECK)
    program = str(tmp_path / "plan")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "qwen3.8-27b-in-c_amd", "csrc"), str(source), "-o", program], check=True)
    run = subprocess.run([program], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
    seen = [[int(v) for v in line.split()] for line in run.stdout.split("\n") if line]
    assert seen[0][0] and all(all(row) for row in seen[1:]), seen


LIMIT_CHECK = r"""
#include <cstdio>
#include "q38_layer.h"
using namespace q38;
int main()
{
    const uint64_t widths[] = {1, 128, 2048, 2049, 4096, 8192, 8193, 17408, 1u << 20, 1u << 24};
    for (uint64_t width : widths) {
        const uint64_t parts = (width + 2047) / 2048, quantized = ((1u << 24) - 1) / parts, normed = width > 8192 ? (1u << 22) - 1 : (1u << 24) - 1;
        if (!layer_launch_holds(quantized * quantize_parts(width), 256) || layer_launch_holds((quantized + 1) * quantize_parts(width), 256) ||
            !layer_launch_holds(normed, norm_threads(width)) || layer_launch_holds(normed + 1, norm_threads(width))) {
            std::printf("width %llu\n", (unsigned long long)width);
            return 1;
        }
    }
    return !layer_launch_holds((1u << 24) - 1, 256) || layer_launch_holds(1u << 24, 256);
}
"""


def _run_cpp(tmp_path, text):
    source, program = tmp_path / "check.cpp", str(tmp_path / "check")
    source.write_text(text)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I" + os.path.join(ROOT, "include"),
                    "-I" + os.path.join(ROOT, "qwen3.8-27b-in-c_amd", "csrc"), str(source), "-o", program], check=True)
    run = subprocess.run([program], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
    return run.stdout


def test_limits_are_the_documented_ones(tmp_path):
    """the most rows that the header names fit a launch and one more does not; the calls refuse those"""
    declared = " ".join(open(os.path.join(ROOT, "include", "q38hip.h")).read().replace("*", " ").split())
    for limit in ("rows ceil(width / 2048) below 2^24", "rows below 2^24, with widths above 8192 below 2^22",
                  "heads head_dim <= 2^20, rows below 2^24"):
        assert limit in declared, limit
    _run_cpp(tmp_path, LIMIT_CHECK)
    norm = dict(output=P, output_row=8193, codes=None, scales=None, total=None, total_row=0, x=2 * P, x_row=8193, addend=None,
                addend_row=0, type=30, weight=3 * P, weight_type=0, offset=0.0, eps=1e-6, width=8193, rows=1 << 22, stream=None)
    _refused("q38hip_rms_norm", norm, [dict(), dict(width=1, rows=1 << 24)])
    quantize = dict(codes=2 * P, scales=3 * P, x=P, x_row=2049, gate=None, gate_row=0, type=0, width=2049, rows=1 << 23, stream=None)
    _refused("q38hip_quantize_e4m3", quantize, [dict(), dict(width=1, rows=1 << 24)])


PROMPT_CHECK = r"""
#include <cstdio>
#include <initializer_list>
#include "q38_layer.h"
using namespace q38;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main()
{
    /* more sequences than lanes have no spare tiles: both sides of 400 and 512 real ones */
    CHECK(plan_prompt(100 * 30, 24, 4, 256, 4, 100).form == kPromptTiles && plan_prompt(100 * 30, 24, 4, 256, 4, 100).workgroups == 564);
    CHECK(plan_prompt(2133, 24, 4, 256, 4, 100).form == kPromptShares && plan_prompt(2133, 24, 4, 256, 4, 100).workgroups == 4 * 400);
    CHECK(plan_prompt(2134, 24, 4, 256, 4, 100).form == kPromptTiles && plan_prompt(2134, 24, 4, 256, 4, 100).workgroups == 4 * 101);
    CHECK(plan_prompt(65536, 1, 1, 128, 2, 100).form == kPromptParts && plan_prompt(65537, 1, 1, 128, 2, 100).form == kPromptTiles);
    /* up to 64 they have one each for each key/value head */
    CHECK(plan_prompt(1365, 24, 4, 256, 4, 10).form == kPromptShares && plan_prompt(1365, 24, 4, 256, 4, 10).workgroups == 4 * 266);
    CHECK(plan_prompt(1366, 24, 4, 256, 4, 10).form == kPromptTiles && plan_prompt(1366, 24, 4, 256, 4, 10).workgroups == 4 * 75);
    CHECK(plan_prompt(16384, 4, 4, 128, 2, 64).form == kPromptParts && plan_prompt(16385, 4, 4, 128, 2, 64).form == kPromptTiles);
    /* keys that are few on average go in one part, whatever the count */
    CHECK(plan_prompt(25599, 1, 1, 128, 2, 100).form == kPromptTiles && plan_prompt(25600, 1, 1, 128, 2, 100).form == kPromptParts);
    CHECK(plan_prompt(1 << 16, 1, 1, 64, 2, 1 << 24).form == kPromptTiles);
    CHECK(plan_prompt(300, 65535, 65535, 256, 4, 1 << 17).form == kPromptTiles);
    /* every launch of the sizes that are taken holds its threads, and has a tile or a wavefront for every row and head */
    for (uint32_t rows = 1; rows <= 1u << 24; rows += 1 + rows / 3)
        for (uint32_t heads = 1; heads <= 65535; heads += 1 + heads / 2)
            for (uint32_t kv = 1; kv <= heads; ++kv)
                if (heads % kv == 0 && (uint64_t)rows * heads <= 1u << 30)
                    for (uint32_t dim = 64; dim <= 256; dim *= 2)
                        for (uint32_t element = 2; element <= 4; element += 2)
                            for (uint32_t count : {1u, 64u, 65u, 1000u, 1u << 24}) {
                                const PromptPlan p = plan_prompt(rows, heads, kv, dim, element, count);
                                CHECK(layer_launch_holds(p.workgroups, p.form == kPromptParts ? 512 : 256));
                                if (p.form == kPromptRows) { CHECK(p.workgroups * 4ull >= (uint64_t)rows * heads); continue; }
                                const uint64_t tiles = ((uint64_t)rows * (heads / kv) + (p.form == kPromptShares ? 31 : 127)) / (p.form == kPromptShares ? 32 : 128);
                                CHECK(p.workgroups == (tiles + (count <= 64 ? count : 0)) * kv);
                            }
    return 0;
}
"""


def test_prompt_plans(tmp_path):
    """which form of attention is taken on both sides of each border, and that all launches hold it"""
    _run_cpp(tmp_path, PROMPT_CHECK)


def test_attention_refuses_scales_beyond_the_exponent():
    """scores are taken times scale * log2(e), which has to be finite too"""
    good = dict(output=2 * P, output_row=512, query=P, gate=None, query_row=512, query_head=128, key=P, key_row=256, value=P,
                value_row=256, type=30, heads=4, kv_heads=2, dim=128, scale=1.0, starts=P, count=1, rows=8, stream=None)
    _refused("q38hip_prompt_attention", good, [dict(scale=s) for s in (3e38, -3e38, 2.4e38, math.inf, -math.inf, math.nan)])
    for scale in (3e38, math.inf):
        assert layer._lib().q38hip_prompt_attention(*dict(good, scale=scale).values()) == 0
        assert q38hip.last_error() == "scale must be finite, at most 2^127"


def test_blended_frequencies_at_the_ends():
    """contexts in which no pair turns `slow` times, or all turn `fast` times; the borders themselves; arguments that have no blend"""
    plain = layer.rotary_frequencies(64, 1e4)[0]
    for original in (1, 3, 6):                   # pair 0 turns original / (2 pi) < 1 times: all are divided
        assert torch.equal(layer.rotary_frequencies(64, 1e4, factor=4.0, original=original)[0], layer.rotary_frequencies(64, 1e4, factor=4.0)[0])
    for original in (10 ** 7, 10 ** 9):          # the last pair turns original / (2 pi) * 1e4^(-62 / 64) > 32 times: all stay
        assert torch.equal(layer.rotary_frequencies(64, 1e4, factor=4.0, original=original)[0], plain)
    for original in (7, 50, 200, 4096, 100000, 600000):
        for turned in (2, 4, 64, 128):
            want = 1e4 ** (-np.arange(0, turned, 2) / turned)
            share = layer.rotary_frequencies(turned, 1e4, factor=4.0, original=original)[0].double().numpy() / want
            turns = original * want / (2 * np.pi)
            assert np.allclose(share[turns >= 32], 1, rtol=2.0 ** -23) and np.allclose(share[turns <= 1], 0.25, rtol=2.0 ** -23)
            assert (np.diff(share) <= 2.0 ** -22).all() and (share <= 1 + 2.0 ** -23).all() and (share >= 0.25 - 2.0 ** -23).all()
    for bad in (dict(fast=1.0, slow=1.0), dict(fast=1.0, slow=2.0), dict(slow=0.0), dict(slow=-1.0), dict(fast=math.nan), dict(fast=math.inf),
                dict(original=math.nan), dict(original=math.inf), dict(factor=math.inf), dict(factor=math.nan), dict(base=math.inf)):
        with pytest.raises(ValueError):
            layer.rotary_frequencies(64, **dict(dict(factor=4.0, original=4096), **bad))


def test_outputs_that_are_inputs_are_refused():
    """every output and workspace against every other tensor of its call, but for what may be in place; the message says so"""
    at = {name: (i + 1) * 16 * P for i, name in enumerate("abcdefghi")}
    calls = {
        "q38hip_quantize_e4m3": (dict(codes=at["a"], scales=at["b"], x=at["c"], x_row=128, gate=at["d"], gate_row=128, type=0, width=128, rows=2,
                                      stream=None), ("codes", "scales"), ("x", "gate"), ()),
        "q38hip_rms_norm": (dict(output=at["a"], output_row=256, codes=at["b"], scales=at["c"], total=at["d"], total_row=256, x=at["e"], x_row=256,
                                 addend=at["f"], addend_row=256, type=30, weight=at["g"], weight_type=0, offset=0.0, eps=1e-6, width=256, rows=3,
                                 stream=None), ("output", "codes", "scales", "total"), ("x", "addend", "weight"),
                            (("output", "x"), ("output", "addend"), ("total", "x"), ("total", "addend"))),
        "q38hip_gemm_e4m3": (dict(output=at["a"], type=30, output_row=256, codes=at["b"], scales=at["c"], tokens=2, inputs=128, weight=at["d"],
                                  weight_scales=at["e"], rows=256, workspace=at["f"], stream=None), ("output", "workspace"),
                             ("codes", "scales", "weight", "weight_scales"), ()),
        "q38hip_rotary": (dict(output=at["a"], output_row=512, output_head=128, x=at["b"], x_row=512, x_head=128, type=1, rows=3, heads=4, dim=128,
                               positions=at["c"], frequencies=at["d"], pairs=32, interleaved=0, magnitude=1.0, stream=None), ("output",),
                          ("x", "positions", "frequencies"), (("output", "x"),)),
        "q38hip_prompt_attention": (dict(output=at["a"], output_row=512, query=at["b"], gate=at["c"], query_row=512, query_head=128, key=at["d"],
                                         key_row=256, value=at["e"], value_row=256, type=30, heads=4, kv_heads=2, dim=128, scale=1.0,
                                         starts=at["f"], count=1, rows=8, stream=None), ("output",), ("query", "gate", "key", "value", "starts"), ())}
    for name, (good, outputs, inputs, allowed) in calls.items():
        for output in outputs:
            for other in outputs + inputs:
                if other != output and (output, other) not in allowed:
                    _refused(name, good, [{output: good[other]}])
                    assert " must " in q38hip.last_error() and "kernel failed" not in q38hip.last_error(), (name, output, other)
