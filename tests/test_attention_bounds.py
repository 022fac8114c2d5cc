"""Where the host's checks and choices for rotary positions, the cache and attention end (host/attention_ops.h), on the CPU."""
import ctypes as C
import math
from fractions import Fraction

import numpy as np
import pytest
import torch
from gyrodx import engine
from gyrodx.engine import AttentionDesc, Engine
from test_attention_calls import A, append, attention, cache, call, rows, shim  # noqa: F401 (a fixture)


@pytest.mark.parametrize("type", [1, 2])
def test_unaligned_caches(shim, type):  # noqa: F811
    """Loads straight to LDS want addresses that are multiples of four bytes: a cache with others goes to the kernels that load to
    registers, all its rows in tiles of 16."""
    plain = dict(type=type, pages=100, page_stride=2 * 16 * 64 + 2, head_stride=16 * 64 + 2, token_stride=66)
    for kw, direct in ((dict(), True), (dict(k=A + 2), False), (dict(v=2 * A + 2), False), (dict(k=A + 4, v=2 * A + 12), True),
                       (dict(page_stride=2049), False), (dict(head_stride=1025), False), (dict(token_stride=65), False),
                       (dict(pages=1, page_stride=2049), True), (dict(kv_heads=1, head_stride=1025), True),
                       (dict(page_size=1, token_stride=65), True), (dict(page_stride=1 << 40), True), (dict(page_stride=(1 << 40) - 1), False)):
        c = cache(**{**plain, **kw})
        d = attention(cache=c, q=rows(type), out=rows(type, data=3 * A), heads=32 * c.kv_heads, sequences=2, longest=300, starts=A, table_width=1000)
        rc, names, out = call(shim.plan_attention, d, 600)
        assert rc == 0, names
        names = names.split()
        assert any(n.startswith("attend_tile") for n in names) == direct, (kw, names)
        if not direct:
            assert names[0].startswith("attend_few") and out[9 + 42] == 300 * 32 // 16 and out[9 + 46] == 0
            assert out[1] * out[2] >= 2 * 600 * c.kv_heads


def test_frequencies_of_many_turns(shim):  # noqa: F811
    """The table is off by half of its last place, 2^-65 of a turn (and 2^-21 of that place for digits of 2 pi behind 128 bits and
    what is cut off), however many turns a position is: at positions below 2^36 angles are exact to 2^-29 of a turn before fp32."""
    turn = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    rng = np.random.default_rng(7)
    f = np.concatenate([[0.0, -0.0, 5e-324, 2.0 ** -64, 1e-19, 0.5, 1, 6.283185307179586, 2.0 ** 30, 2.0 ** 31 - 2.0 ** -21, -1e9, 12345.678],
                        rng.uniform(-1, 1, 200) * 2.0 ** rng.uniform(-70, 31, 200)])
    out, why = (C.c_uint64 * len(f))(), C.create_string_buffer(200)
    assert shim.plan_frequencies(f.ctypes.data, len(f), 0, 1.0, out, why) == 0
    for v, got in zip(f, out):
        turns = Fraction(float(v)) / turn
        off = abs((turns - math.floor(turns)) * 2 ** 64 - got)
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 2 ** 21), (v, got, float(off))


def test_keys_and_values_of_one_address(shim):  # noqa: F811
    """Appending keys and values to one array would leave either's: refused. Attention may read one array as both."""
    d = append()
    assert call(shim.plan_append, d, 3)[0] == 0
    d.cache.v = d.cache.k
    rc, why, _ = call(shim.plan_append, d, 3)
    assert rc < 0 and "cache" in why
    d = attention()
    d.cache.v = d.cache.k
    assert call(shim.plan_attention, d, 3)[0] == 0


def test_scales(shim):  # noqa: F811
    """The kernels' scale is times log2 e: one that leaves fp32 by that would make scores of zero NaN, and is refused."""
    for scale, ok in ((2.3e38, True), (2.4e38, False), (3.4e38, False), (1e-44, True)):
        assert (call(shim.plan_attention, attention(scale=scale), 3)[0] == 0) == ok, scale


def test_binding_takes_any_bound(monkeypatch):
    """A host's fixed bound on a sequence's tokens may be above the tokens of a call: no sequence has more than all of them, which
    is what the library is told (it refuses more)."""
    seen = []

    class Library:
        def gm_attention(self, handle, desc, n, on):
            seen.append((AttentionDesc.from_buffer_copy(desc).longest, n))
            return 0

    monkeypatch.setattr(engine, "lib", Library)
    e = Engine.__new__(Engine)
    e._h, e.adapter, e._matrices = C.c_void_p(), -1, {}
    x, kc = torch.zeros(6, 16), torch.zeros(5, 2, 16, 8)
    table, lengths, starts = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for longest in (2, 6, 7, 4096):
        e.attention(x, kc, kc, table, lengths, x, starts=starts, longest=longest, stream=0)
    assert seen == [(2, 6), (6, 6), (6, 6), (6, 6)]
    e.attention(x, kc, kc, table, lengths, x, longest=7, stream=0)  # without starts: every sequence has as many
    assert seen[-1] == (7, 6)


def test_limits_as_stated(shim):  # noqa: F811
    """`longest` up to n, and tiles of 16 rows of the longest sequence times all of them and the cache's heads below 2^31 in fp32."""
    d = dict(heads=8, starts=A, table_width=100)
    fp32 = cache(type=0, kv_heads=8, page_stride=8 * 1024)
    for sequences, longest, n, ok in ((5000, 1 << 18, 1 << 20, True), (5000, 1 << 20, 1 << 20, False), (1 << 14, 1 << 18, 1 << 20, False),
                                      ((1 << 14) - 1, 1 << 18, 1 << 20, True), (1, 1 << 21, 1 << 20, False)):
        assert (sequences * -(-longest // 16) * 8 < 1 << 31 and longest <= n) == ok
        rc, why, _ = call(shim.plan_attention, attention(cache=fp32, q=rows(0), out=rows(0, data=3 * A), sequences=sequences, longest=longest, **d), n)
        assert (rc == 0) == ok, (sequences, longest, why)
