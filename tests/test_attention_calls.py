"""Argument checks, builds and grids of rotary positions, the cache's appending and attention (host/attention_ops.h) and their
binding, on the CPU: every call that include/gyro_attention.h refuses, none of which reaches a launch."""
import ctypes as C
import math
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest
import torch

from gyrodx import engine
from gyrodx.engine import NO_ROTARY, AttentionDesc, Cache, CacheAppendDesc, Engine, RotaryDesc, Rows
from gyrodx.rotary import frequencies
from test_abi import declared, exported

ROOT = Path(__file__).resolve().parents[1]
BUILD = ROOT / "gyro-dx_amd" / "build"

SHIM = r"""
#include "attention_ops.h"
using namespace gyro;
template <class F> static int run(char *why, F f) {
    try { f(); return 0; } catch (const NativeError &e) { std::strncpy(why, e.what(), 199); return e.code; }
}
static void tell(const Launch &l, uint32_t *out, char *why) {
    out[0] = l.x; out[1] = l.y; out[2] = l.next_x; out[3] = l.next_y;
    std::memcpy(out + 4, l.c.w, sizeof(l.c.w));
    std::strncpy(why, l.kernel ? l.kernel : "", 199);
}
static AttentionOps ops(uint32_t pairs) {
    AttentionOps o;
    Rotary r;
    r.table.handle = reinterpret_cast<gd_buffer *>(64);
    r.pairs = pairs;
    o.rotaries.push_back(r);
    return o;
}
extern "C" int plan_frequencies(const double *f, uint32_t pairs, uint32_t layout, float scale, uint64_t *out, char *why) {
    return run(why, [&] { std::vector<uint64_t> t; AttentionOps::describe(f, pairs, layout, scale, t); std::copy(t.begin(), t.end(), out); });
}
extern "C" int plan_rotary(const gm_rotary_desc *d, uint32_t n, uint32_t pairs, uint32_t *out, char *why) {
    return run(why, [&] { tell(ops(pairs).turned(*d, n), out, why); });
}
extern "C" int plan_append(const gm_cache_append_desc *d, uint32_t n, uint32_t pairs, uint32_t *out, char *why) {
    return run(why, [&] { tell(ops(pairs).append(*d, n), out, why); });
}
// The launches' grids, then the constants; their names, one after another.
extern "C" int plan_attention(const gm_attention_desc *d, uint32_t n, uint32_t, uint32_t *out, char *why) {
    return run(why, [&] {
        const Launches l = AttentionOps::attention(*d, n);
        std::string names;
        out[0] = l.count;
        for (int i = 0; i < l.count; ++i) {
            out[1 + 2 * i] = l.step[i].x;
            out[2 + 2 * i] = l.step[i].y;
            names += std::string(l.step[i].kernel) + " ";
        }
        std::memcpy(out + 9, l.c.w, sizeof(l.c.w));
        std::strncpy(why, names.c_str(), 199);
    });
}
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("ops")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "gyro-dx_amd" / "host"), "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    L = C.CDLL(str(d / "shim.so"))
    L.plan_frequencies.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32, C.c_float, C.c_void_p, C.c_char_p]
    return L


A = 0x100000  # an address that no check may follow


def rows(type=1, stride=1 << 20, data=A):
    return Rows(data, stride, type)


def cache(**kw):
    d = Cache(k=A, v=2 * A, type=1, pages=100, page_size=16, kv_heads=2, head_dim=64, page_stride=2 * 16 * 64, head_stride=16 * 64,
              token_stride=64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def call(f, d, n, pairs=16):
    why, out = C.create_string_buffer(200), (C.c_uint32 * 70)()
    rc = f(C.byref(d), n, pairs, out, why)
    return rc, why.value.decode(), list(out)


def refused_each(f, good, bads, n=3):
    for g in good:
        rc, why, _ = call(f, g, n)
        assert rc == 0, why
    for b in bads:
        m = n
        if isinstance(b, tuple):
            b, m = b
        rc, why, _ = call(f, b, m)
        assert rc < 0 and why


def test_header_is_exported():
    names = declared("gyro_attention.h", "gm_")
    assert len(names) == 6, names
    assert not set(names) - exported(BUILD / "libgyro_moe.so")


def test_struct_layouts():
    """Offsets of the header's structs (64-bit pointers)."""
    assert C.sizeof(Cache) == 64 and Cache.type.offset == 16 and Cache.page_stride.offset == 40
    assert C.sizeof(RotaryDesc) == 72 and RotaryDesc.x.offset == 16 and RotaryDesc.positions.offset == 64
    assert C.sizeof(CacheAppendDesc) == 192 and CacheAppendDesc.k.offset == 80 and CacheAppendDesc.slots.offset == 176
    assert C.sizeof(AttentionDesc) == 192 and AttentionDesc.heads.offset == 112 and AttentionDesc.table.offset == 136
    assert AttentionDesc.table_width.offset == 168 and AttentionDesc.workspace.offset == 176


# ---- frequencies ----

def test_frequency_table(shim):
    """The table's fractions of a turn are the frequencies' own to the last of 64 places."""
    turn = 2 * Fraction("3.14159265358979323846264338327950288419716939937510")
    f = np.array([1.0, 0.1, 1e-4, 3.7e-9, 0.0, -0.25, 6.2, 12345.678, 2.0 ** 30, 1e-19, -1e-30])
    out, why = (C.c_uint64 * len(f))(), C.create_string_buffer(200)
    assert shim.plan_frequencies(f.ctypes.data, len(f), 0, 1.0, out, why) == 0
    for v, got in zip(f, out):
        turns = Fraction(float(v)) / turn
        want = (turns - math.floor(turns)) * 2 ** 64
        off = abs(want - got)
        # x87 divides to 64 bits: turns above one lose as many places.
        assert min(off, 2 ** 64 - off) <= 1 + abs(float(turns)), (v, got, float(want))


def test_frequency_refusals(shim):
    f = np.ones(600)
    ok = lambda f=f, pairs=4, layout=0, scale=1.0: shim.plan_frequencies(  # noqa: E731
        None if f is None else f.ctypes.data, pairs, layout, scale, (C.c_uint64 * 600)(), C.create_string_buffer(200))
    assert ok() == 0 and ok(pairs=512, layout=1, scale=-0.5) == 0
    for bad in (dict(f=None), dict(pairs=0), dict(pairs=513), dict(layout=2), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(f=np.array([1, np.nan, 1, 1.0])), dict(f=np.array([1, np.inf, 1, 1.0])), dict(f=np.array([1, 1, 1, 2.0 ** 31]))):
        assert ok(**bad) < 0


def test_frequencies():
    f, s = frequencies(8)
    assert s == 1 and np.allclose(f, [1, 1e-1, 1e-2, 1e-3], rtol=1e-15)
    f, s = frequencies(8, scaling="linear", factor=4)
    assert s == 1 and np.allclose(f, [0.25, 0.025, 0.0025, 0.00025], rtol=1e-15)
    f, s = frequencies(8, scaling="base", factor=4)
    assert s == 1 and np.allclose(f[0], 1) and np.allclose(f[-1], 1e-3 / 4, rtol=1e-14)
    f, s = frequencies(128, scaling="bands", factor=16, context=4096)
    plain, _ = frequencies(128)
    turns = 4096 * plain / (2 * np.pi)
    assert np.isclose(s, 0.1 * np.log(16) + 1)
    assert np.array_equal(f[turns >= 32], plain[turns >= 32]) and np.allclose(f[turns <= 1], plain[turns <= 1] / 16, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((f < plain) & (f > plain / 16))[between].all()
    assert np.array_equal(frequencies(2, scaling="base", factor=4)[0], [1.0])
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, factor=0.0), dict(dim=8, base=-1.0),
                dict(dim=8, slow=4.0, fast=2.0), dict(dim=8, context=0)):
        with pytest.raises(ValueError):
            frequencies(**bad)


# ---- rotary, append ----

def rotary(**kw):
    d = RotaryDesc(rotary=0, heads=4, head_dim=64, positions_64=1, x=rows(), y=rows(0, data=2 * A), positions=A)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_rotary_refusals(shim):
    refused_each(shim.plan_rotary,
                 [rotary(), rotary(y=rows()), rotary(head_dim=32), rotary(head_dim=1024), rotary(positions_64=0, positions=A + 4)],
                 [rotary(rotary=1), rotary(rotary=NO_ROTARY), rotary(heads=0), rotary(head_dim=0), rotary(head_dim=31), rotary(head_dim=1025),
                  rotary(x=Rows()), rotary(y=Rows()), rotary(x=rows(3)), rotary(y=rows(data=A + 1)), rotary(y=rows(stride=255, data=2 * A)),
                  rotary(y=rows(0)), rotary(y=rows(stride=1 << 19)), rotary(positions=None), rotary(positions=A + 4),
                  rotary(positions_64=0, positions=A + 2), rotary(x=rows(stride=1 << 41)), (rotary(heads=1 << 20), 1 << 11),
                  rotary(heads=(1 << 20) + 1)])
    assert call(shim.plan_rotary, rotary(), 0)[2][0] == 0
    assert call(shim.plan_rotary, rotary(y=rows(0, stride=0, data=2 * A)), 1)[0] == 0  # one row's stride is not used


def append(**kw):
    d = CacheAppendDesc(cache=cache(), rotary=0, heads=8, slots_64=1, positions_64=1, k=rows(), v=rows(), q=rows(data=3 * A),
                        q_out=rows(0, data=4 * A), slots=A, positions=A)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_append_refusals(shim):
    none = dict(heads=0, q=Rows(), q_out=Rows())
    by_tokens = dict(head_stride=64, token_stride=2 * 64)
    refused_each(shim.plan_append,
                 [append(), append(**none), append(rotary=NO_ROTARY, positions=None), append(q_out=rows(data=3 * A)),
                  append(cache=cache(**by_tokens)), append(cache=cache(type=0)), append(cache=cache(type=2, pages=1, page_stride=0)),
                  append(cache=cache(kv_heads=1, head_stride=0)), append(cache=cache(page_size=1, token_stride=0, head_stride=64)),
                  append(cache=cache(head_dim=57)), append(slots_64=0, slots=A + 4)],
                 [append(rotary=1), append(positions=None), append(positions=A + 4), append(slots=None), append(slots=A + 4),
                  append(slots_64=0, slots=A + 2), append(k=Rows()), append(v=Rows()), append(k=rows(0)), append(v=rows(2)),
                  append(q=rows(0, data=3 * A)), append(heads=0), append(q=Rows()), append(q_out=Rows()), append(heads=8, q=Rows(), q_out=Rows()),
                  append(q_out=rows(0, data=3 * A)), append(q_out=rows(stride=511, data=4 * A)),
                  *[append(cache=cache(**c)) for c in (dict(k=None), dict(v=None), dict(k=A + 1), dict(type=3), dict(pages=0), dict(page_size=0),
                                                       dict(kv_heads=0), dict(head_dim=0), dict(pages=1 << 27), dict(head_dim=30),
                                                       dict(head_dim=1025), dict(page_stride=1 << 41), dict(token_stride=63),
                                                       dict(head_stride=16 * 64 - 1), dict(page_stride=2 * 16 * 64 - 1),
                                                       dict(head_stride=64), dict(token_stride=0), dict(type=0, v=A + 2))],
                  (append(), 1 << 28)])
    assert call(shim.plan_append, append(), 0)[2][0] == 0


@pytest.mark.parametrize("pairs,dim", [(1, 2), (1, 1024), (512, 1024), (16, 64), (10, 80), (64, 128), (5, 11), (3, 7)])
def test_rotary_grids(shim, pairs, dim):
    """Every unit of every head of every token has a thread, and the grid fits."""
    for n in (1, 3, 64, 1023, 100000, (1 << 31) // 12):
        for heads, kv in ((1, 0), (32, 0), (8, 2), (0, 1)):
            if n * (heads + 2 * kv) >= 1 << 31:
                continue
            if kv:
                none = dict(heads=0, q=Rows(), q_out=Rows()) if not heads else dict(heads=heads)
                c = cache(kv_heads=kv, head_dim=dim, token_stride=dim, head_stride=16 * dim, page_stride=16 * dim * kv)
                rc, why, out = call(shim.plan_append, append(cache=c, **none), n, pairs)
            else:
                rc, why, out = call(shim.plan_rotary, rotary(heads=heads, head_dim=dim), n, pairs)
            assert rc == 0, why
            x, y, w = out[0], out[1], out[4:]
            sharers, units, turns, narrow = w[42], w[43], w[44], w[45]
            assert 1 <= x <= 65535 and 1 <= y <= 65535
            assert units >= -(-pairs // 8) + -(-(dim - 2 * pairs) // 16) and units * 16 >= dim
            assert units <= 256 and sharers * turns * 2 * ((64 if narrow else 256) // units) >= heads + 2 * kv
            assert not narrow or pairs <= 128 and sharers == 1 and n > 2048
            assert x * y >= (-(-n // 4) if narrow else n * sharers)


# ---- attention ----

def attention(**kw):
    d = AttentionDesc(cache=cache(), q=rows(), out=rows(data=3 * A), heads=8, sequences=3, longest=1, causal=1, window=0, scale=0.125,
                      table=A, table_stride=7, lengths=A, starts=None, table_width=7, workspace=A, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_attention_refusals(shim):
    refused_each(shim.plan_attention,
                 [attention(), attention(out=rows()), attention(sequences=1, longest=3), attention(starts=A, sequences=5, longest=2),
                  attention(window=5), attention(causal=0), attention(cache=cache(type=0), q=rows(0), out=rows(0)),
                  attention(cache=cache(head_dim=256)), attention(cache=cache(head_dim=8)), attention(heads=2),
                  attention(table_width=1, workspace=None, workspace_bytes=0)],
                 [attention(heads=0), attention(heads=3), attention(cache=cache(head_dim=60)), attention(cache=cache(head_dim=264)),
                  attention(q=Rows()), attention(out=Rows()), attention(q=rows(0)), attention(out=rows(2)), attention(q=rows(data=A + 1)),
                  attention(out=rows(stride=511, data=3 * A)), attention(out=rows(stride=1 << 19)), attention(sequences=0),
                  attention(longest=0), attention(longest=4, starts=A), attention(longest=2), attention(sequences=2),
                  attention(lengths=None), attention(lengths=A + 2), attention(starts=A + 1), attention(table=None), attention(table=A + 2),
                  attention(table_width=0), attention(table_width=1 << 27), attention(table_stride=1 << 41), attention(causal=0, window=4),
                  attention(scale=0.0), attention(scale=-1.0), attention(scale=float("nan")), attention(scale=float("inf")),
                  attention(table_width=1000, workspace=None), attention(table_width=1000, workspace=A + 128),
                  attention(table_width=1000, workspace_bytes=4096), attention(heads=64, table_width=5000, workspace=None),
                  attention(heads=64, table_width=5000, workspace_bytes=1 << 20), attention(cache=cache(pages=0)), attention(cache=cache(type=3)),
                  attention(cache=cache(pages=1 << 27)), (attention(sequences=1 << 28, longest=1), 1 << 28)])
    assert call(shim.plan_attention, attention(), 0)[2][0] == 0


@pytest.mark.parametrize("type", [0, 1, 2])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (1, 1, 8), (64, 1, 256), (32, 8, 128), (40, 40, 72), (700, 700, 64)])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_launches(shim, type, heads, kv, dim, ragged):
    """Sequences of few rows and of many go to their kernels, the grids cover every row and part, and the workspace serves
    every call."""
    most = engine.lib().gm_attention_workspace(heads, kv, dim)
    c, group = cache(type=type, kv_heads=kv, head_dim=dim), heads // kv
    few_bytes, part = 2048 * 16 * 4 * (dim + 2), 128 * 4 * (dim + 2)
    assert most == few_bytes + 4352 + (32 << 18) + 1024 * part
    for sequences, longest in ((1, 1), (1, 5), (1, 4096), (3, 1), (64, 1), (64, 7), (300, 100), (5000, 1), (2, 100000)):
        if sequences * longest * group > 128 * 250000 or sequences * longest * heads > 1 << 30:
            continue
        for width in (1, 3, 60, 1000, 30000000):
            d = attention(cache=c, q=rows(type), out=rows(type, data=3 * A), heads=heads, sequences=sequences, longest=longest, table_width=width,
                          workspace_bytes=most, starts=A if ragged else None)
            rc, names, out = call(shim.plan_attention, d, sequences * longest)
            assert rc == 0, names
            names, w = names.split(), out[9:]
            grids = {name: out[1 + 2 * i] * out[2 + 2 * i] for i, name in enumerate(names)}
            assert len(names) == out[0] and all(1 <= v <= 65535 for v in out[1:1 + 2 * out[0]])
            pairs = -(-longest * group // 16) * sequences * kv
            many = bool(type) and longest * group > 16 and (pairs > 512 or pairs * width * 16 > 1 << 18)
            size = 64 if dim <= 64 else 128 if dim <= 128 else 256
            short = type and size < 256 and f"attend_short_{'?bh'[type]}{size}" in names
            build = "f32_" if not type else ("short_" if short else "few_") + "?bh"[type]
            assert not short or width * 16 <= min(2048, max(896, 16 * (sequences * kv if many else pairs)))
            few = f"attend_{build}{size}"
            tile = "attend_tile_%s%d" % ("?bh"[type], size)
            listed = many and sequences * -(-longest * group // 128) > 1024
            assert names[:1] == ["attend_plan"] if listed else "attend_plan" not in names
            assert (few in names) == (not many or ragged) and (tile in names) == bool(many)
            assert w[46] == (17 if many else 0)
            join = 0
            if few in names:
                split, tiles, keys, least = w[41], w[42], w[44], w[45]
                assert keys == (16 if not type and dim > 64 else 32)
                assert tiles == 1 if many else tiles * 16 >= longest * group > (tiles - 1) * 16
                # A group for every entry and head, and for what splits add: of each entry less than its share of `split`.
                assert split in (0, 256, 512, 1024) and grids[few] >= sequences * tiles * kv + split
                assert not split or (sequences * tiles <= 1024 and width * 16 > w[57] * keys and least >= 1)
                if split:
                    most_rows = min(16, longest * group)
                    assert w[56] == most_rows
                    join = w[47]
                    assert join >= min(sequences * tiles, split // kv) * kv * most_rows
            assert w[47] == join
            if many:
                tokens = sequences * longest * group
                units = min(sequences * -(-longest * group // 128), tokens // 128 + min(sequences, tokens // 17)) + 512 // kv
                assert grids[tile] > units * kv and units < 1 << 18
                assert w[50] | w[51] << 32 == A + few_bytes + 4352 + (32 << 18)
                assert w[54] * kv * part <= 1024 * part and w[55] == (32 if dim > 128 else 64)
                assert grids["attend_join"] >= join + 1024
                if listed:
                    assert grids["attend_plan"] == 1 and w[48] | w[49] << 32 == A + few_bytes and grids[tile] >= w[53] * kv > units * kv
                else:
                    assert w[48] == w[49] == 0 and w[28] == -(-longest * group // 128)
            else:
                assert ("attend_join" in names) == bool(join) and (not join or grids["attend_join"] >= join)


def test_page_division(shim):
    """The kernels' division by the page size, of key numbers up to the largest."""
    rng = np.random.default_rng(3)
    for size in (1, 2, 3, 5, 7, 16, 24, 48, 100, 255, 256, 257, 1000, 4095, 65537, (1 << 20) - 1, 1 << 20, (1 << 29) - 1):
        width = max(1, ((1 << 29) - 1) // size)
        c = cache(page_size=size, pages=2, token_stride=64, head_stride=size * 64, page_stride=size * 128)
        rc, why, out = call(shim.plan_attention, attention(cache=c, table_width=width, table_stride=width), 3)
        assert rc == 0, why
        shift, reciprocal = out[9 + 52], out[9 + 59]
        i = np.concatenate([np.arange(5), rng.integers(0, 1 << 29, 100000), [(1 << 29) - 1], *(np.arange(1, 50) * size + k for k in (-1, 0, 1))])
        i = np.unique(np.clip(i, 0, (1 << 29) - 1)).astype(object)
        assert all(((int(v) << 3) * reciprocal >> 32) >> shift == int(v) // size for v in i), size


@pytest.mark.parametrize("kw,small", [
    (dict(), 1), (dict(pages=1 << 20, page_stride=2048), 1), (dict(pages=(1 << 20) + 1, page_stride=2048), 0),
    (dict(type=0, pages=1 << 19, page_stride=2048), 1), (dict(type=0, pages=(1 << 19) + 1, page_stride=2048), 0),
    (dict(pages=2, page_stride=1 << 40), 0), (dict(pages=1, page_stride=1 << 40), 1), (dict(pages=1 << 26, page_stride=1 << 40), 0),
    (dict(head_stride=(1 << 31) - 100 * 2048), 1), (dict(head_stride=1 << 31), 0), (dict(pages=1, page_size=2, token_stride=1 << 31), 0)])
def test_cache_spans(shim, kw, small):
    """Caches whose last byte 32 bits reach are told from larger ones, whatever the strides."""
    c = cache(**kw)
    t = c.type
    rc, why, out = call(shim.plan_attention, attention(cache=c, q=rows(t), out=rows(t, data=3 * A)), 3)
    assert rc == 0 and out[9 + 38] == 1 + 2 * small, why


def test_workspace_of_no_shape():
    f = engine.lib().gm_attention_workspace
    assert f(0, 1, 64) == f(8, 0, 64) == f(8, 3, 64) == f(8, 8, 0) == f(8, 8, 264) == 0


# ---- the binding's own checks ----

@pytest.fixture
def eng():
    """An engine without a device: tensors on the CPU pass its device check, and a call that passes every check ends
    at the missing handle."""
    e = Engine.__new__(Engine)
    e._h, e.adapter, e._matrices = C.c_void_p(), -1, {}
    return e


def reached(f, *args, **kw):
    with pytest.raises(RuntimeError, match="no engine"):
        f(*args, **kw)


def refused(f, *args, **kw):
    with pytest.raises((ValueError, KeyError)):
        f(*args, **kw)


def test_binding_rotary(eng):
    x, p = torch.zeros(3, 64), torch.zeros(3, dtype=torch.int64)
    reached(eng.add_rotary, [1.0, 0.5])
    refused(eng.add_rotary, [1.0], layout="other")
    refused(eng.add_rotary, [[1.0]])
    reached(eng.rotary, 0, x, p, x, heads=4)
    reached(eng.rotary, 0, torch.zeros(3, 100)[:, 4:68], p.int(), x.half(), heads=1)
    for bad in ((0, x, p, x, 0), (0, x, p, x, 3), (0, x, p, x, -4), (0, x, p[:2], x, 4), (0, x, p.float(), x, 4), (0, x, p, x[:2], 4),
                (0, x, p, x[:, :32], 4), (0, x.double(), p, x, 4), (0, x, p, torch.zeros(64, 3).T, 4), (-1, x, p, x, 4), (1 << 32, x, p, x, 4)):
        refused(eng.rotary, *bad)
    for bad in (-1, 1 << 32):
        refused(eng.release_rotary, bad)
    eng.adapter = 0
    refused(eng.rotary, 0, x, p, x, heads=4)


def test_binding_append(eng):
    kc, vc = torch.zeros(5, 2, 16, 8), torch.zeros(5, 2, 16, 8)
    k, s = torch.zeros(3, 16), torch.zeros(3, dtype=torch.int64)
    q = torch.zeros(3, 32)
    reached(eng.cache_append, k, k, kc, vc, s)
    reached(eng.cache_append, k, k, kc, vc, s.int(), rotary=0, positions=s, q=q, q_out=q.half())
    tokens = [torch.zeros(5, 16, 2, 8).transpose(1, 2) for _ in range(2)]
    reached(eng.cache_append, k, k, *tokens, s)
    for args, kw in (((k, k, kc, vc[:4], s), {}), ((k, k, kc, vc.half(), s), {}), ((k, k, kc, tokens[1], s), {}), ((k, k, kc[0], vc[0], s), {}),
                     ((k[:, :8], k, kc, vc, s), {}), ((k, k[:2], kc, vc, s), {}), ((k, k, kc, vc, s[:2]), {}), ((k, k, kc, vc, s.float()), {}),
                     ((k, k, kc, vc, s), dict(rotary=0)), ((k, k, kc, vc, s), dict(q=q)), ((k, k, kc, vc, s), dict(q_out=q)),
                     ((k, k, kc, vc, s), dict(q=q[:, :30], q_out=q[:, :30])), ((k, k, kc, vc, s), dict(q=q, q_out=q[:, :16])),
                     ((k, k, kc, vc, s), dict(rotary=0, positions=s[:1])), ((k, k, kc.double(), vc.double(), s), {}),
                     ((k, k, kc.transpose(2, 3), vc.transpose(2, 3), s), {})):
        refused(eng.cache_append, *args, **kw)
    eng.adapter = 0
    refused(eng.cache_append, k, k, kc, vc, s)


def test_binding_attention(eng):
    kc, vc = torch.zeros(5, 2, 16, 8), torch.zeros(5, 2, 16, 8)
    q, table, lengths = torch.zeros(6, 32), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    starts, ws = torch.zeros(4, dtype=torch.int32), torch.zeros(512, dtype=torch.uint8)
    good = (q, kc, vc, table, lengths, q)
    reached(eng.attention, *good)
    reached(eng.attention, *good, ws, starts=starts, longest=2, window=3, scale=1.0)
    reached(eng.attention, q, kc, vc, torch.zeros(3, 9, dtype=torch.int32)[:, 2:6], lengths, q, causal=False)
    for at, bad in ((0, q[:, :30]), (0, q[0]), (0, q.double()), (1, kc.half()), (2, vc[:, :1]), (3, table.long()), (3, table[0]),
                    (3, torch.zeros(4, 3, dtype=torch.int32).T), (4, lengths[:2]), (4, lengths.long()), (5, q[:5]), (5, q[:, :16])):
        refused(eng.attention, *(bad if i == at else a for i, a in enumerate(good)))
    for kw in (dict(starts=starts), dict(starts=starts[:3], longest=2), dict(starts=starts.long(), longest=2), dict(window=-1),
               dict(window=1 << 32), dict(longest=1 << 32), dict(workspace=torch.zeros(4))):
        refused(eng.attention, *good, **kw)
    refused(eng.attention, q[:5], kc, vc, table, lengths, q[:5])  # not three equal sequences
    for bad in (-1, 1 << 32):
        refused(Engine.attention_workspace, bad, 1, 8)
    eng.adapter = 0
    refused(eng.attention, *good)


def test_default_stream_is_torchs_current(eng, monkeypatch):
    """A call without a stream goes to torch's current one on the engine's GPU, one with a stream to that."""
    queued = []

    class Library:
        def __getattr__(self, name):
            return lambda *args: queued.append((name, args[-1])) or 0

    class Stream:
        cuda_stream = 0x5150

    monkeypatch.setattr(engine, "lib", Library)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: Stream if device == -1 else None)
    x, i = torch.zeros(3, 16), torch.zeros(3, dtype=torch.int32)
    kc = torch.zeros(5, 2, 16, 8)
    for kw, want in (({}, 0x5150), (dict(stream=0), 0), (dict(stream=7), 7)):
        eng.rotary(0, x, i, x, heads=2, **kw)
        eng.cache_append(x, x, kc, kc, i, **kw)
        eng.attention(x, kc, kc, torch.zeros(3, 1, dtype=torch.int32), i, x, **kw)
        assert queued == [("gm_rotary", want), ("gm_cache_append", want), ("gm_attention", want)]
        queued.clear()
