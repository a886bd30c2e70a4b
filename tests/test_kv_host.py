"""What the paged cache refuses on the host, and its index arithmetic
(csrc/q38_kv.h) compiled for the CPU: work slots of ragged batches, bad ids and
pages, scale exponents."""
import ctypes
import glob
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import kv_cases as kc
import q38hip
from q38hip import kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _cache(**change):
    words = ctypes.create_string_buffer(4096 + 16)
    at = (ctypes.addressof(words) + 15) // 16 * 16
    fields = dict(data=at, scales=at, refs=at, tables=at, lengths=at, status=at, layers=1, pages=4, page_tokens=16, kv_heads=2,
                  head_dim=64, sequences=2, table_entries=2, type=0)
    fields.update(change)
    cache = kv.Pages(**fields)
    cache.keep = words
    return cache


BAD_CACHES = [dict(data=0), dict(status=0), dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(sequences=0),
              dict(table_entries=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256), dict(head_dim=32),
              dict(head_dim=96), dict(head_dim=512), dict(type=2), dict(pages=0x80000000), dict(table_entries=0x10000000),
              dict(kv_heads=40000), dict(layers=70000), dict(sequences=0x80000000),
              dict(kv_heads=32767, layers=65535, page_tokens=128, head_dim=256)]


@pytest.mark.parametrize("change", BAD_CACHES, ids=str)
def test_bad_caches_are_refused(change):
    lib, p = kv._lib(), 4096
    cache = ctypes.byref(_cache(**change))
    calls = (lambda: lib.q38hip_kv_reset(cache, None), lambda: lib.q38hip_kv_workspace_bytes(cache),
             lambda: lib.q38hip_kv_extend(cache, p, p, 1, p, None), lambda: lib.q38hip_kv_fork(cache, p, p, None, 1, None),
             lambda: lib.q38hip_kv_truncate(cache, p, p, 1, None), lambda: lib.q38hip_kv_compact(cache, p, None),
             lambda: lib.q38hip_kv_copy(cache, p, p, 1, None),
             lambda: lib.q38hip_kv_append(cache, 0, p, p, 0, 128, p, None, 1, 1, None),
             lambda: lib.q38hip_kv_attention_workspace_bytes(cache, 0, 2, 1, 1),
             lambda: lib.q38hip_kv_attention(cache, 0, p, p, None, 0, 2, 128, 64, 128, 1.0, p, None, 1, 1, p, None))
    for call in calls:
        assert call() == 0 and q38hip.last_error()


def test_bad_arguments_are_refused():
    lib, p = kv._lib(), 4096
    cache = ctypes.byref(_cache())
    append = dict(layer=0, key=p, value=p, type=0, stride=128, ids=p, starts=None, count=1, total=1)
    for change in (dict(key=None), dict(value=None), dict(type=2), dict(layer=1), dict(ids=None), dict(count=0), dict(total=0),
                   dict(total=3, count=2), dict(total=2, stride=127), dict(total=1 << 25), dict(count=1 << 25, starts=p)):
        a = dict(append, **change)
        assert not lib.q38hip_kv_append(cache, a["layer"], a["key"], a["value"], a["type"], a["stride"], a["ids"], a["starts"],
                                        a["count"], a["total"], None), change
    good = dict(layer=0, out=p, query=p, gate=None, type=0, heads=4, row=256, head=64, to=256, ids=p, starts=None, count=1,
                total=1, work=p)
    for change in (dict(out=None), dict(query=None), dict(type=8), dict(heads=3), dict(heads=0), dict(layer=5), dict(head=63),
                   dict(total=2, to=255), dict(ids=None), dict(total=0), dict(count=0), dict(total=5, count=2), dict(work=None),
                   dict(work=p + 4)):
        a = dict(good, **change)
        assert not lib.q38hip_kv_attention(cache, a["layer"], a["out"], a["query"], a["gate"], a["type"], a["heads"], a["row"],
                                           a["head"], a["to"], 1.0, a["ids"], a["starts"], a["count"], a["total"], a["work"],
                                           None) or change.get("work", p) is None and not \
            lib.q38hip_kv_attention_workspace_bytes(cache, 0, 4, 1, 1), change
    assert not lib.q38hip_kv_extend(cache, p, p, 1025, p, None)
    assert not lib.q38hip_kv_extend(cache, p, None, 1, p, None)
    assert not lib.q38hip_kv_extend(cache, p, p, 1, None, None)
    assert not lib.q38hip_kv_fork(cache, p, None, None, 1, None)
    assert not lib.q38hip_kv_truncate(cache, p, None, 1, None)
    assert not lib.q38hip_kv_compact(cache, None, None)
    assert not lib.q38hip_kv_copy(cache, p, p, 0, None)


def test_launches_that_a_grid_cannot_hold_are_refused():
    lib, p = kv._lib(), 4096
    assert not lib.q38hip_kv_fork(ctypes.byref(_cache()), p, p, None, 65537, None)
    assert "65536" in q38hip.last_error()
    page = dict(kv_heads=32767, page_tokens=128, head_dim=256)          # 2 GiB less 64 KiB
    assert lib.q38hip_kv_workspace_bytes(ctypes.byref(_cache(layers=32, **page)))
    assert not lib.q38hip_kv_workspace_bytes(ctypes.byref(_cache(layers=33, **page)))
    assert "all layers" in q38hip.last_error()


def test_python_checks():
    plain = kc.Cache(1, 4, 16, 2, 64, 2, 2, "int8").to("cpu")
    ids = kc.words([0], "cpu")
    row = torch.zeros(1, 2, 64)
    for call in (lambda: kv.KVPages(plain.data, plain.scales, plain.refs, plain.tables, plain.lengths, plain.status, "int4"),
                 lambda: kv.KVPages(plain.data[0], plain.scales, plain.refs, plain.tables, plain.lengths, plain.status, "int8"),
                 lambda: kv.KVPages(plain.data, plain.scales[:, :2], plain.refs, plain.tables, plain.lengths, plain.status, "int8"),
                 lambda: kv.KVPages(plain.data, plain.scales, plain.refs.long(), plain.tables, plain.lengths, plain.status, "int8"),
                 lambda: plain.append(0, row, row.half(), ids), lambda: plain.append(0, row.double(), row.double(), ids),
                 lambda: plain.append(0, row[:, :1], row, ids), lambda: plain.append(0, row, row, ids.long()),
                 lambda: plain.append(0, torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), kc.words([0, 1], "cpu")),
                 lambda: plain.append(0, row, row, ids, kc.words([0], "cpu")),
                 lambda: plain.attention(0, row[..., :32], ids), lambda: plain.attention(0, row.int(), ids),
                 lambda: plain.attention(0, row, ids, gate=row.half()), lambda: plain.attention(0, row, ids, out=row.half()),
                 lambda: plain.attention(0, row[0], ids), lambda: plain.extend(ids, kc.words([1, 2], "cpu")),
                 lambda: plain.fork(ids, ids.long()), lambda: plain.truncate(ids, kc.words([], "cpu"))):
        with pytest.raises(ValueError):
            call()


def test_exports():
    declared = open(os.path.join(ROOT, "include", "q38hip.h")).read()
    for name in kv.EXPORTS:
        assert name + "(" in declared and hasattr(q38hip.lib(), name)
    assert ctypes.sizeof(kv.Pages) == 6 * 8 + 8 * 4


INDEX_CHECK = r"""
#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <vector>
#include "q38_kv.h"
using namespace q38;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
static uint32_t state = 12345;
static uint32_t draw(uint32_t n) { state = state * 1664525u + 1013904223u; return (state >> 8) % n; }
int main()
{
    /* every item of every sequence has a slot of its own sequence, and the slots suffice */
    for (int trial = 0; trial < 3000; ++trial) {
        const uint32_t count = 1 + draw(40), per_row = 1 + draw(12), unit = 1u << draw(8), T = 16u << draw(4);
        std::vector<int32_t> starts(1, 0), ids(count, 0);
        for (uint32_t i = 0; i < count; ++i) starts.push_back(starts.back() + draw(trial % 3 ? 4 : 200));
        const uint32_t total = starts.back();
        if (!total) continue;
        const KVRows rows{ids.data(), starts.data(), count, total, total / count};
        for (uint32_t i = 0; i < count; ++i) {
            const uint32_t b = kv_row_start(rows, i), e = kv_row_start(rows, i + 1);
            const uint32_t items = ((e - b) * per_row + unit - 1) / unit;
            CHECK(kv_slot_base(b, i, per_row, unit, 1) + items <= kv_slot_base(e, i + 1, per_row, unit, 1));
            for (uint32_t first = 0; first < 2 * T; ++first) {
                const uint32_t pages = e > b ? (first + e - b + T - 1) / T - first / T : 0;
                CHECK(kv_slot_base(b, i, 1, T, 2) + pages <= kv_slot_base(e, i + 1, 1, T, 2));
            }
        }
        CHECK(kv_slot_base(total, count, per_row, unit, 1) <= kv_slots(total, count, per_row, unit, 1));
        CHECK(kv_slot_base(total, count, 1, T, 2) <= kv_slots(total, count, 1, T, 2));
    }
    /* a slot of an append holds each of a sequence's pages once, and with offsets that decrease it still
     * stays within a page and within its sequence's rows */
    for (int trial = 0; trial < 20000; ++trial) {
        const uint32_t count = 1 + draw(12), shift = 4 + draw(4), T = 1u << shift, entries = 1 + draw(200);
        const bool rising = trial % 2;
        std::vector<int32_t> starts(1, rising ? 0 : draw(100)), ids(count, 0);
        std::vector<uint32_t> tokens;
        for (uint32_t i = 0; i < count; ++i) {
            starts.push_back(rising ? starts.back() + draw(200) : draw(2) ? draw(4000) : starts.back() + draw(300));
            tokens.push_back(draw(4) ? draw(entries * T + 1) : draw(3));
        }
        const uint32_t total = rising ? starts.back() : 4000;
        if (!total) continue;
        const KVRows rows{ids.data(), starts.data(), count, total, 0};
        std::vector<uint32_t> written(count, 0);
        for (uint32_t slot = 0; slot < kv_slots(total, count, 1, T, 2); ++slot) {
            uint32_t before = 0;           /* as many bases as lie at or before the slot: the sequence, if they rise */
            for (uint32_t i = 0; i < count; ++i) before += kv_slot_base(kv_row_start(rows, i), i, 1, T, 2) <= slot;
            if (!before) continue;
            const uint32_t i = before - 1, b = kv_row_start(rows, i), e = kv_row_start(rows, i + 1);
            const KVPageRows p = kv_page_rows(b, e, tokens[i], slot, kv_slot_base(b, i, 1, T, 2), shift, entries);
            if (!p.some) continue;
            CHECK(p.entry < entries && p.from < p.to && p.to <= T && p.entry * T + p.to <= tokens[i]);
            const uint32_t row = e - tokens[i] + p.entry * T;
            CHECK((int32_t)(row + p.from) >= (int32_t)b && row + p.to <= e);
            written[i] += p.to - p.from;
        }
        for (uint32_t i = 0; rising && i < count; ++i) {
            const uint32_t n = starts[i + 1] - starts[i];
            CHECK(written[i] == (n < tokens[i] ? n : tokens[i]));
        }
    }
    /* offsets that are not: never past the rows */
    int32_t odd[4] = {-7, 3, 1 << 30, 2}, id = 0;
    const KVRows rows{&id, odd, 3, 10, 3};
    for (uint32_t i = 0; i < 4; ++i) CHECK(kv_row_start(rows, i) <= 10);
    const KVRows even{&id, nullptr, 3, 12, 4};
    for (uint32_t i = 0; i < 4; ++i) CHECK(kv_row_start(even, i) == 4 * i);
    /* ids, lengths and pages outside the cache */
    int32_t tables[6] = {0, 4, 5, -1, 0x7fffffff, (int32_t)0x80000000}, lengths[2] = {33, 1000};
    Q38KVPages c{};
    c.tables = tables;
    c.lengths = lengths;
    c.pages = 5;
    c.page_tokens = 16;
    c.sequences = 2;
    c.table_entries = 3;
    c.kv_heads = 4;
    c.head_dim = 256;
    CHECK(kv_tokens(c, 0) == 33 && kv_tokens(c, 1) == 48 && kv_tokens(c, 2) == 0 && kv_tokens(c, -1) == 0);
    lengths[0] = -3;
    CHECK(kv_tokens(c, 0) == 0);
    CHECK(kv_page(c, 0, 0) == 0 && kv_page(c, 0, 1) == 4 && kv_page(c, 0, 2) == -1 && kv_page(c, 0, 3) == -1);
    CHECK(kv_page(c, 1, 0) == -1 && kv_page(c, 1, 1) == -1 && kv_page(c, 1, 2) == -1);
    CHECK(kv_page_bytes(c) == 2 * 4 * 16 * 256 && kv_block(c, 0x7ffffffe, 1, 3) == (0x7ffffffeull * 2 + 1) * 4 + 3);
    /* scale exponents: the least that holds the value */
    for (int e4m3 = 0; e4m3 < 2; ++e4m3) {
        const double most = e4m3 ? 448 : 127;
        for (uint32_t bits = 0; bits < 0x7f800000u; bits += 9973) {
            float v;
            __builtin_memcpy(&v, &bits, 4);
            const int k = kv_scale_exponent(bits, e4m3);
            CHECK(v <= std::ldexp(most, k) && k >= -100 && k <= 122);
            CHECK(k == -100 || v > std::ldexp(most, k - 1));
        }
        for (int e = -80; e < 110; ++e)
            for (int step = -1; step <= 1; ++step) {
                float v = (float)std::ldexp(most, e);
                uint32_t bits;
                __builtin_memcpy(&bits, &v, 4);
                CHECK(kv_scale_exponent(bits + step, e4m3) == (step > 0 ? e + 1 : e));
            }
    }
    std::puts("ok");
    return 0;
}
"""


def test_index_arithmetic(tmp_path):
    source, program = tmp_path / "kv_index.cpp", tmp_path / "kv_index"
    source.write_text(INDEX_CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "qwen3.8-27b-in-c_amd", "csrc"), str(source),
                    "-o", str(program)], check=True)
    assert subprocess.run([str(program)], capture_output=True, text=True, timeout=120).stdout == "ok\n"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_model_of_the_codes(kind):
    """the plain model's own encoding: every code stands for itself, and borders go to even"""
    codes = np.arange(256, dtype=np.uint8)
    values = kc.decode(codes, kind)
    fine = np.isfinite(values) & ((values != -128) | (kind != "int8"))
    assert np.array_equal(kc.decode(kc.encode(values[fine], kind), kind), values[fine])
    steps = np.unique(values[fine])
    middle = (steps[1:] + steps[:-1]) / 2
    got = kc.decode(kc.encode(middle, kind), kind)
    assert np.isin(got, steps).all() and (np.abs(got - middle) == (steps[1:] - steps[:-1]) / 2).all()
    want = torch.from_numpy(middle).float()
    want = want.round() if kind == "int8" else want.to(torch.float8_e4m3fn).float()
    assert np.array_equal(got, want.double().numpy())


WORK_CHECK = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "q38_kv_plan.h"
using namespace q38;
#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
static uint32_t state = 54321;
static uint32_t draw(uint32_t n) { state = state * 1664525u + 1013904223u; return (state >> 8) % n; }
struct Slot { uint32_t at, each, steps; };
int main()
{
    /* divisions by a group */
    for (uint32_t d = 1; d <= 32768; d = d < 70 ? d + 1 : d * 2 - d / 3)
        for (uint32_t n = 0; n < d + 256; n += 1 + n / 300) CHECK(kv_divide(n, kv_magic(d)) == n / d);
    /* ranges: workgroups of them hold all units, and one less would not */
    for (int trial = 0; trial < 200000; ++trial) {
        const uint32_t units = draw(2) ? draw(100000) : (draw(1 << 24) << 7) + draw(128), groups = 1 + draw(1024), least = 1 + draw(8);
        const uint32_t chunk = kv_chunk(units, groups, 1.0f / (float)groups, least);
        CHECK(chunk >= least && (uint64_t)chunk * groups >= units);
        CHECK(chunk == least || chunk <= units / groups * (1 + 1e-6) + 2);
    }
    /* every step of every slot is in one piece, its pieces are counted, and each has a place of its own */
    for (int trial = 0; trial < 4000; ++trial) {
        const uint32_t shift = trial % 5 ? 0 : draw(4), groups = 1 + draw(40), least = shift ? 1 : 4;
        std::vector<Slot> slots;
        uint32_t total = 0;
        for (uint32_t n = 1 + draw(30); n; --n) {
            const uint32_t most = draw(3) ? draw(20) : draw(600), each = kv_slot_units(most, shift);
            for (uint32_t k = 1 + draw(3); k; --k) {              /* slots of one sequence: the last rows see all steps */
                slots.push_back({total, each, most - (most ? draw(most < 3 ? most : 3) : 0)});
                total += each;
            }
        }
        const uint32_t chunk = kv_chunk(total, groups, 1.0f / (float)groups, least), small = kv_small(chunk);
        std::vector<uint32_t> reached(slots.size(), 0), pieces(slots.size(), 0), firsts(slots.size(), 0);
        std::vector<uint32_t> places(slots.size(), 0);
        std::vector<char> used(2 * groups, 0);
        for (uint32_t w = 0; w < groups; ++w) {
            const uint64_t begin = (uint64_t)w * chunk, end64 = begin + chunk;
            if (begin >= total) break;
            const uint32_t end = end64 < total ? (uint32_t)end64 : total;
            for (uint32_t k = 0; k < slots.size(); ++k) {
                const Slot &s = slots[k];
                if (s.at >= end || s.at + s.each <= begin) continue;
                const KVPiece p = kv_piece(s.at, s.each, s.steps, (uint32_t)begin, end, small, shift);
                if (!p.some) continue;
                CHECK(p.first == reached[k] && p.last >= p.first && p.last <= s.steps);
                reached[k] = p.last;
                ++pieces[k];
                CHECK(p.first_piece == (pieces[k] == 1));
                if (p.first_piece) firsts[k] = p.whole ? 1 : kv_pieces(p.units, chunk, s.at + s.each, s.each);
                CHECK(!p.whole || p.last == s.steps);
                if (p.whole) continue;
                const uint32_t place = kv_place(w, p.first_piece);
                CHECK(place < used.size() && !used[place]);
                used[place] = 1;
                if (p.first_piece) places[k] = place;
                CHECK(place == places[k] + kv_place_step(pieces[k] - 1));
            }
        }
        for (uint32_t k = 0; k < slots.size(); ++k) CHECK(reached[k] == slots[k].steps && pieces[k] >= 1 && pieces[k] == firsts[k]);
    }
    std::puts("ok");
    return 0;
}
"""


def test_work_split(tmp_path):
    """how the tokens of a paged attention call are cut between workgroups (csrc/q38_kv_plan.h)"""
    source, program = tmp_path / "kv_work.cpp", tmp_path / "kv_work"
    source.write_text(WORK_CHECK)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror",
                    "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "qwen3.8-27b-in-c_amd", "csrc"), str(source),
                    "-o", str(program)], check=True)
    assert subprocess.run([str(program)], capture_output=True, text=True, timeout=120).stdout == "ok\n"


def test_too_many_query_heads_are_refused():
    cache = ctypes.byref(_cache(kv_heads=1))
    assert kv._lib().q38hip_kv_attention_workspace_bytes(cache, 0, 32769, 1, 1) == 0
    assert "32768" in q38hip.last_error()


def test_workspace_follows_the_workgroups():
    """only slots that are cut need room, and they are no more than the workgroups, however long the prompt"""
    cache = ctypes.byref(_cache(kv_heads=4, head_dim=256, page_tokens=64, table_entries=1024, pages=2048))
    sizes = [kv._lib().q38hip_kv_attention_workspace_bytes(cache, 30, 24, 1, rows) for rows in (1, 512, 4096, 32768)]
    assert 0 < sizes[0] < sizes[1] and max(sizes) < 80e6 and sizes[3] - sizes[2] < 1e6
    short = ctypes.byref(_cache(kv_heads=4, head_dim=256, page_tokens=16, table_entries=8, pages=64))
    assert kv._lib().q38hip_kv_attention_workspace_bytes(short, 0, 24, 2, 2) == 0


def test_loads_to_lds_wait_for_their_base():
    """a load to LDS that reads M0 needs a wait state behind the scalar write of M0; the compiler adds none inside
    inline assembly"""
    found = 0
    for path in glob.glob(os.path.join(ROOT, "qwen3.8-27b-in-c_amd", "csrc", "*.h*")):
        for block in re.findall(r'asm volatile\(((?:\s*"(?:[^"\\]|\\.)*")+)', open(path).read()):
            lines = [line.strip() for line in "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block)).replace("\\t", " ").split("\\n")]
            for at, line in enumerate(lines):
                if re.match(r"s_\w+ m0\b", line):
                    found += 1
                    assert lines[at + 1].startswith("s_nop"), (path, lines)
    assert found


def _assembly(tmp_path, name):
    """the device assembly of one of csrc's files, with the flags that it is built with"""
    package = os.path.join(ROOT, "qwen3.8-27b-in-c_amd")
    lines = subprocess.run(["make", "-n", "-B", "-C", package], capture_output=True, text=True, check=True).stdout.splitlines()
    command = next(line for line in lines if line.endswith("/" + name + ".o") and " -c " in line).split()
    command[command.index("-c")] = "-S"
    command[command.index("-o") + 1] = str(tmp_path / (name + ".s"))
    subprocess.run(command + ["--offload-device-only"], check=True, capture_output=True)
    return (tmp_path / (name + ".s")).read_text()


def _registers(text):
    found = set()
    for kind, first, last, single, number in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        found |= {(kind, n) for n in range(int(first), int(last) + 1)} if kind else {(single, int(number))}
    return found


def _touched_too_soon(body, states):
    """vector instructions that touch the registers of a product in inline assembly, which the compiler does not see,
    fewer than `states` wait states behind it, over all branches; and the number of such products"""
    code, labels, inside = [], {}, False
    for line in body.split("\n"):
        inside = "#ASMSTART" in line or inside and "#ASMEND" not in line
        text = line.split(";")[0].strip()
        if text.endswith(":"):
            labels[text[:-1]] = len(code)
        elif text and not text.startswith("."):
            code.append((text, inside))
    products = [at for at, (text, own) in enumerate(code) if own and text.startswith("v_mfma")]
    bad = []
    for product in products:
        written, ways, known = _registers(code[product][0].split(",")[0]), [(product + 1, 0)], set()
        while ways:
            at, waited = ways.pop()
            while at < len(code) and waited < states and (at, waited) not in known:
                known.add((at, waited))
                text, own = code[at]
                what = text.split()[0]
                if what == "s_nop":
                    waited += int(text.split()[1])
                if what.startswith(("v_", "ds_", "global_", "scratch_")) and not (own and what.startswith("v_mfma")) and \
                        _registers(text) & written:
                    bad.append((code[product][0], text, waited))
                    break
                if what.startswith("s_cbranch"):
                    ways.append((labels[text.split()[1]], waited + 1))
                at, waited = labels[text.split()[1]] if what == "s_branch" else at + 1, waited + 1
    return bad, len(products)


def test_sums_are_left_alone_until_they_are_written(tmp_path):
    """256-wide attention multiplies into accumulation registers by inline assembly: whatever the compiler does with
    them comes eight wait states behind the product, as it does behind the compiler's own"""
    text = _assembly(tmp_path, "q38_kv_attention256")
    kernels = re.findall(r"^(_ZN3q38\w*kv_attention_kernel\w*):(.*?)^\.Lfunc_end", text, re.S | re.M)
    products = 0
    for name, body in kernels:
        bad, count = _touched_too_soon(body, 8)
        assert not bad, (name, bad[:3])
        products += count
    assert len(kernels) == 16 and products


def test_calls_of_more_threads_than_a_launch_are_refused():
    """2^32 threads or more along the grid: refused on the host, before anything is enqueued"""
    lib, p = kv._lib(), 4096

    def refused(ok, *words):
        assert not ok and "failed" not in q38hip.last_error(), q38hip.last_error()
        for word in words:
            assert word in q38hip.last_error(), q38hip.last_error()

    # append: rows / page_tokens + 2 sequences workgroups of page_tokens * head_dim / 32 threads
    wide = ctypes.byref(_cache(page_tokens=128, head_dim=256, kv_heads=1))
    refused(lib.q38hip_kv_append(wide, 0, p, p, 0, 256, p, p, 1 << 21, 1 << 21, None), "append", "sequences")
    refused(lib.q38hip_kv_append(wide, 0, p, p, 0, 256, p, p, 1 << 24, 1 << 24, None), "append", "sequences")
    refused(lib.q38hip_kv_append(ctypes.byref(_cache(kv_heads=1, page_tokens=128)), 0, p, p, 0, 64, p, None, 1 << 24, 1 << 24, None),
            "append", "sequences")
    refused(lib.q38hip_kv_truncate(ctypes.byref(_cache()), p, p, 1 << 24, None), "2^24")
    # attention: the join of slots that may be cut has a workgroup of 256 threads for each of them
    long = ctypes.byref(_cache(kv_heads=1, table_entries=1 << 16))
    for count, total in ((1 << 24, 1 << 24), ((1 << 24) - 1, 1 << 24)):
        refused(lib.q38hip_kv_attention_workspace_bytes(long, 0, 8, count, total), "attention", "sequences")
        refused(lib.q38hip_kv_attention(long, 0, p, p, None, 0, 8, 512, 64, 512, 1.0, p, p, count, total, p, None), "attention")
    assert lib.q38hip_kv_attention_workspace_bytes(long, 0, 1, 1 << 20, 1 << 20)
    # reset: a thread for each table entry
    most = dict(sequences=1 << 14, table_entries=1 << 18)
    refused(lib.q38hip_kv_reset(ctypes.byref(_cache(**most)), None), "table")
    refused(lib.q38hip_kv_reset(ctypes.byref(_cache(sequences=0xffffffff // 255, table_entries=255)), None), "table")


def test_calls_are_made_on_the_device_of_the_cache(monkeypatch):
    """a default stream's handle names no device: whatever device is current, a call is made with the cache's"""
    plain = kc.Cache(1, 4, 16, 2, 64, 2, 2, "int8").to("cpu")            # (its device index is -1)
    ids, more, row, heads = kc.words([0], "cpu"), kc.words([1], "cpu"), torch.zeros(1, 2, 64), torch.zeros(1, 4, 64)
    current, calls = [3], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *what):
            current.pop()

    class Library:
        def __getattr__(self, name):
            if name.endswith("workspace_bytes"):
                return lambda *arguments: 64
            return lambda *arguments: calls.append((name, current[-1], arguments[-1])) or 1

    class Torch:
        empty = staticmethod(torch.empty)
        uint8 = torch.uint8

        class _C:
            _cuda_getDevice = staticmethod(lambda: current[-1])
            _cuda_getCurrentRawStream = staticmethod(lambda index: 1000 + index)

        class cuda:
            device = Device

    monkeypatch.setattr(kv, "_lib", Library)
    plain._torch = Torch
    for now in (3, -1):
        current[:] = [now]
        calls.clear()
        plain.reset()
        plain.extend(ids, more)
        plain.fork(ids, ids)
        plain.truncate(ids, ids)
        plain.compact()
        plain.copy(ids, ids)
        plain.append(0, row, row, ids)
        plain.attention(0, heads, ids, gate=heads)
        assert [name[len("q38hip_kv_"):] for name, _, _ in calls] == ["reset", "extend", "fork", "truncate", "compact", "copy",
                                                                      "append", "attention"]
        assert all(device == -1 and stream == 999 for _, device, stream in calls), calls
        assert current == [now]
