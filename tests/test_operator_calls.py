"""The operators' argument checks, builds and grids (host/row_ops.h) and their binding, on the CPU: every call that the
headers refuse, none of which reaches a launch, and the layout sizes of matrices."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import op_reference as ref
from gyrodx import engine
from gyrodx.engine import BlockNormDesc, Engine, LogprobsDesc, MatrixDesc, Rows
from test_abi import declared, exported

ROOT = Path(__file__).resolve().parents[1]
BUILD = ROOT / "gyro-dx_amd" / "build"

SHIM = r"""
#include "row_ops.h"
using namespace gyro;
template <class F> static int run(char *why, F f) {
    try { f(); return 0; } catch (const NativeError &e) { std::strncpy(why, e.what(), 199); return e.code; }
}
static void tell(const Launch &l, uint32_t *out, char *why) {
    out[0] = l.x; out[1] = l.y;
    std::memcpy(out + 2, l.c.w, sizeof(l.c.w));
    std::strncpy(why, l.kernel ? l.kernel : "", 199);
}
extern "C" int plan_matrix(const gm_matrix_desc *d, uint64_t *out, char *why) {
    return run(why, [&] { Matrix m = RowOps::describe(*d); out[0] = RowOps::layout(m); out[1] = m.tiles; out[2] = m.chunks;
                          out[3] = m.scales; out[4] = m.minima; });
}
extern "C" int plan_linear(const gm_matrix_desc *d, const gm_rows *x, uint32_t n, const gm_rows *y, uint32_t act,
                           uint32_t accumulate, float scale, uint32_t *out, char *why) {
    return run(why, [&] { Matrix m = RowOps::describe(*d); RowOps::layout(m);
                          tell(RowOps::linear(m, 256, *x, n, *y, act, accumulate, scale), out, why); });
}
extern "C" int plan_norm(const gm_block_norm_desc *d, uint32_t n, uint32_t *out, char *why) {
    return run(why, [&] { tell(RowOps::block_norm(*d, n), out, why); });
}
extern "C" int plan_logprobs(const gm_logprobs_desc *d, uint32_t n, uint32_t *out, char *why) {
    return run(why, [&] { tell(RowOps::logprobs(*d, n), out, why); });
}
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    d = tmp_path_factory.mktemp("ops")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(ROOT / "include"), "-I",
                    str(ROOT / "gyro-dx_amd" / "host"), "-o", str(d / "shim.so"), str(d / "shim.cpp")], check=True)
    L = C.CDLL(str(d / "shim.so"))
    L.plan_linear.argtypes = [C.c_void_p, C.c_void_p, C.c_uint32, C.c_void_p, C.c_uint32, C.c_uint32, C.c_float, C.c_void_p,
                              C.c_char_p]
    return L


A = 0x10000  # an address that no check may follow


def rows(type=0, stride=1 << 20, data=A):
    return Rows(data, stride, type)


def matrix(fmt=0, rows=64, cols=256, group=32, **more):
    d = MatrixDesc(fmt, rows, cols, group, quants=A)
    if fmt == 2:
        d.scales = A
    for k, v in more.items():
        setattr(d, k, v)
    return d


def call(f, *args):
    why, out = C.create_string_buffer(200), (C.c_uint32 * 62)()
    rc = f(*[C.byref(a) if isinstance(a, C.Structure) else a for a in args], out, why)
    return rc, why.value.decode(), out[0], out[1]


def test_header_is_exported():
    names = declared("gyro_ops.h", "gm_")
    assert len(names) == 7, names
    assert not set(names) - exported(BUILD / "libgyro_moe.so")


def test_struct_layouts():
    """Offsets of the header's structs (64-bit pointers)."""
    assert C.sizeof(Rows) == 24 and Rows.stride.offset == 8 and Rows.type.offset == 16
    assert C.sizeof(MatrixDesc) == 64 and MatrixDesc.quants.offset == 16 and MatrixDesc.up_quants.offset == 40
    assert C.sizeof(BlockNormDesc) == 168 and BlockNormDesc.h.offset == 16 and BlockNormDesc.post_weight.offset == 136
    assert C.sizeof(LogprobsDesc) == 128 and LogprobsDesc.tokens.offset == 48 and LogprobsDesc.workspace.offset == 112


@pytest.mark.parametrize("d,tiles,chunks,per,mins", [
    (matrix(), 4, 2, 4, 0), (matrix(rows=17, cols=32), 2, 1, 4, 0), (matrix(1, rows=16, cols=160), 1, 2, 4, 1),
    (matrix(2, group=64, cols=192), 4, 2, 2, 0), (matrix(2, group=128, mins=A), 4, 2, 1, 1),
    (matrix(rows=17, up_quants=A), 4, 2, 4, 0)])
def test_matrix_layout(shim, d, tiles, chunks, per, mins):
    out, why = (C.c_uint64 * 5)(), C.create_string_buffer(200)
    assert shim.plan_matrix(C.byref(d), out, why) == 0, why.value
    units = tiles * chunks
    assert list(out) == [units * (1024 + 32 * per * (1 + mins)), tiles, chunks, units * 1024, units * (1024 + 32 * per)]


@pytest.mark.parametrize("d", [
    matrix(3), matrix(group=64), matrix(1, group=128), matrix(2, group=16), matrix(2, group=256, cols=512),
    matrix(rows=0), matrix(cols=0), matrix(cols=48), matrix(2, group=128, cols=192), matrix(quants=None),
    matrix(2, scales=None), matrix(scales=A), matrix(mins=A), matrix(up_scales=A), matrix(2, up_scales=A),
    matrix(2, up_quants=A), matrix(2, up_quants=A, up_scales=A, mins=A), matrix(2, up_quants=A, up_scales=A, up_mins=A),
    matrix(rows=1 << 26, cols=256), matrix(rows=1 << 27, cols=32), matrix(rows=1, cols=1 << 21)])
def test_matrix_refusals(shim, d):
    out, why = (C.c_uint64 * 5)(), C.create_string_buffer(200)
    assert shim.plan_matrix(C.byref(d), out, why) < 0 and why.value


def test_linear_refusals(shim):
    m, g = matrix(), matrix(up_quants=A)
    ok = lambda d=m, x=rows(), n=4, y=rows(), act=0, acc=0, scale=1.0: call(shim.plan_linear, d, x, n, y, act, acc, scale)  # noqa: E731
    assert ok()[0] == 0 and ok()[2] >= 1
    assert ok(n=0)[0] == 0 and ok(n=0)[2] == 0
    assert ok(x=rows(stride=1 << 30), n=1)[0] == 0  # one row's stride is not used
    assert ok(x=rows(stride=0))[0] == 0 and ok(y=rows(stride=0), n=1)[0] == 0
    for bad in (dict(x=rows(data=None)), dict(y=rows(data=None)), dict(x=rows(type=3)), dict(y=rows(type=7)),
                dict(x=rows(data=A + 2)), dict(y=rows(type=1, data=A + 1)), dict(y=rows(stride=63)), dict(act=3),
                dict(d=g, act=1), dict(n=(1 << 18) + 1), dict(x=rows(stride=1 << 41)), dict(x=rows(stride=(1 << 24) + 1)), dict(y=rows(stride=1 << 41))):
        rc, why, *_ = ok(**bad)
        assert rc < 0 and why, bad


def test_linear_grids(shim):
    """Any token count and matrix fits the grid's 65535 groups a dimension."""
    for fmt, r, c in ((0, 1, 32), (0, 131072, 2048), (2, 100003, 2560), (0, 1 << 22, 1024), (0, (1 << 24) - 240, 128),
                      (0, 1 << 24, 32), (0, 50 << 20, 32)):
        for type in (0, 1, 2):
            for n in (1, 5, 6, 64, 1023, 1 << 18):
                rc, why, x, y = call(shim.plan_linear, matrix(fmt, r, c), rows(type), n, rows(stride=r), 0, 0, 1.0)
                assert rc == 0 and 1 <= x <= 65535 and 1 <= y <= 65535, (r, c, type, n, why, x, y)


def test_linear_builds(shim):
    """Few tokens or few rows take mv_q4, many mm_q4 by 16 to 64 tokens a group (16 to 48 of fp32 ones)."""
    def plan(r, c, type, n, fmt=0, group=32):
        rc, why, x, y = call(shim.plan_linear, matrix(fmt, r, c, group), rows(type), n, rows(stride=r), 0, 0, 1.0)
        out, why = (C.c_uint32 * 62)(), C.create_string_buffer(200)
        m, a, b = matrix(fmt, r, c, group), rows(type), rows(stride=r)
        assert shim.plan_linear(C.byref(m), C.byref(a), n, C.byref(b), 0, 0, 1.0, out, why) == 0
        return why.value.decode(), out[2 + 26], x, y
    assert plan(2048, 512, 0, 1)[0] == "mv_q4" and plan(2048, 512, 0, 1, 2, 128)[0] == "mv_q4"
    for type in (0, 1, 2):
        assert plan(131072, 2048, type, 1)[0] == "mv_q4" and plan(512, 2048, type, 64)[0] == "mv_q4"
        for n in (12, 20, 30, 45, 64, 150, 1023):
            name, t, x, y = plan(40000, 128, type, n, 2, 64)
            if n > (5, 16, 8)[type]:
                assert name == "mm_q4_" + "fbh"[type] + "64" and 1 <= t <= (3, 4, 4)[type]
                assert x == 157 and y * 16 * t >= n > (y - 1) * 16 * t
    tokens = [[plan(r, g, type, n, 2 if g > 32 else 0, g)[1] for r, n in
               ((100003, 30), (100003, 45), (100003, 64), (8000, 1000), (8000, 500), (8000, 700))]
              for type in (1, 2) for g in (32, 64, 128)]
    assert all(t == [2, 3, 4, 4, 2, 3] for t in tokens), tokens
    for g, want in ((32, [1, 2, 2, 2, 2]), (64, [1, 2, 3, 2, 3]), (128, [1, 2, 3, 2, 3])):
        assert [plan(r, 128, 0, n, 2 if g > 32 else 0, g)[1] for r, n in
                ((40000, 12), (100003, 30), (100003, 45), (8000, 1000), (8000, 700))] == want
    assert plan(40000, 64, 1, 20)[0] == "mm_q4_b32" and plan(40000, 64, 2, 12)[0] == "mm_q4_h32"


def norm(**kw):
    d = BlockNormDesc(E=100, post=0, h=rows(), x=rows(), out=rows(), normed=rows(), post_eps=1e-6, pre_eps=1e-6, scale=1.0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_block_norm_refusals(shim):
    none = Rows()
    for good in (norm(), norm(h=none), norm(out=none), norm(normed=none), norm(post=1, post_weight=A), norm(E=16384),
                 norm(gate_kind=3, gate=rows(1))):
        assert call(shim.plan_norm, good, 3)[0] == 0
    assert call(shim.plan_norm, norm(), 0)[2] == 0
    assert call(shim.plan_norm, norm(), 70000)[2:] == (65535, 2)
    for bad in (norm(E=0), norm(E=16385), norm(out=none, normed=none), norm(x=none), norm(x=rows(9)), norm(h=rows(data=A + 1)),
                norm(out=rows(stride=99)), norm(normed=rows(stride=0)), norm(gate_kind=4, gate=rows()),
                norm(gate_kind=1), norm(gate_kind=1, gate=rows(), gate_act=1), norm(h=none, gate_kind=1, gate=rows()),
                norm(h=none, post=1), norm(post_weight=A), norm(post=1, post_weight=A + 2), norm(pre_weight=A + 1),
                norm(post_eps=-1.0), norm(pre_eps=float("nan"))):
        rc, why, *_ = call(shim.plan_norm, bad, 3)
        assert rc < 0 and why


def lp(n=3, **kw):
    d = LogprobsDesc(logits=rows(), V=1000, given=1, top=5, tokens_64=1, scale=1.0, tokens=A, tokens_stride=1, logprobs=A,
                     logprobs_stride=1, entropy=A, top_ids=A, top_logprobs=A, top_stride=5, workspace=A, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_logprobs_refusals(shim):
    for good in (lp(), lp(given=0, tokens=None, logprobs=None), lp(top=0, top_ids=None, top_logprobs=None), lp(entropy=None),
                 lp(V=5), lp(V=70000, top=64, given=64, top_stride=64, logprobs_stride=64, tokens_stride=64)):
        rc, why, *_ = call(shim.plan_logprobs, good, 3)
        assert rc == 0, why
    assert call(shim.plan_logprobs, lp(), 0)[2] == 0
    assert call(shim.plan_logprobs, lp(), 200000)[2:] == (65535, 4)
    for bad in (lp(V=0), lp(V=1 << 31), lp(logits=Rows()), lp(logits=rows(5)), lp(logits=rows(data=A + 1)), lp(scale=0.0),
                lp(scale=-1.0), lp(scale=float("nan")), lp(scale=float("inf")), lp(given=65), lp(top=65), lp(V=4),
                lp(tokens=None), lp(logprobs=None), lp(tokens=A + 4), lp(tokens_64=0, tokens=A + 2), lp(logprobs=A + 2),
                lp(logprobs_stride=0), lp(top_ids=None), lp(top_logprobs=None), lp(top_ids=A + 1), lp(top_stride=4),
                lp(entropy=A + 2), lp(given=0, top=0, entropy=None)):
        rc, why, *_ = call(shim.plan_logprobs, bad, 3)
        assert rc < 0 and why


# ---- the binding's own checks ----

@pytest.fixture
def eng():
    """An engine without a device: tensors on the CPU pass its device check, and a call that passes every check ends
    at the missing handle."""
    e = Engine.__new__(Engine)
    e._h, e.adapter, e._matrices = C.c_void_p(), -1, {0: (64, 96)}
    return e


def reached(f, *args, **kw):
    with pytest.raises(RuntimeError, match="no engine"):
        f(*args, **kw)


def refused(f, *args, **kw):
    with pytest.raises((ValueError, KeyError)):
        f(*args, **kw)


def test_binding_linear(eng):
    x, y = torch.zeros(3, 96), torch.zeros(3, 64)
    reached(eng.linear, 0, x, y)
    reached(eng.linear, 0, torch.zeros(3, 100)[:, 4:], y.half())
    for bad in ((1, x, y), (0, x[:, :95], y), (0, x, y[:2]), (0, x.double(), y), (0, x, y.int()), (0, x, torch.zeros(64, 3).T),
                (0, x[0], y)):
        refused(eng.linear, *bad)
    refused(eng.linear, 0, x, y, act="gelu")
    eng.adapter = 0
    refused(eng.linear, 0, x, y)


def test_binding_matrix(eng):
    q, s = np.zeros((4, 32), np.uint8), np.zeros((4, 2), np.float16)
    reached(eng.add_matrix, "q4", 4, 64, (q, s, None))
    reached(eng.add_matrix, "q4", 4, 64, (q, s, s), up=(q, s, s))
    reached(eng.add_matrix, "q4_0", 4, 64, np.zeros((4, 36), np.uint8))
    for bad in (("q5", 4, 64, q), ("q4", 4, 64, (q, s)), ("q4", 4, 64, (q.astype(np.int8), s, None)), ("q4", 4, 64, (q[:3], s, None)),
                ("q4", 4, 64, (q, s.astype(np.float32), None)), ("q4", 4, 64, (q, s, s[:1])), ("q4_0", 4, 64, q),
                ("q4_1", 4, 64, np.zeros((4, 36), np.uint8)), ("q4", 0, 64, (q, s, None)), ("q4", 4, 48, (q, s, None))):
        refused(eng.add_matrix, *bad)


def test_binding_block_norm(eng):
    x, w = torch.zeros(3, 8), torch.zeros(8)
    reached(eng.block_norm, x, x, x, x, post=True, post_weight=w, gate=torch.zeros(3, 1), pre_weight=w)
    reached(eng.block_norm, None, x, None, x.half(), gate=None)
    for kw in (dict(gate=torch.zeros(2, 8)), dict(gate=torch.zeros(8)), dict(gate=torch.zeros(3, 1), gate_act="tanh"),
               dict(pre_weight=w[:7]), dict(pre_weight=w.half()), dict(post_weight=torch.zeros(16)[::2]), dict(normed=x[:2])):
        refused(eng.block_norm, x, x, x, **kw)
    refused(eng.block_norm, x[:2], x, x)


def test_binding_logprobs(eng):
    x, t, o = torch.zeros(3, 50), torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 1)
    ids, top = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)
    reached(eng.logprobs, x, tokens=t, logprob=o, entropy=torch.zeros(3), top_ids=ids, top_logprobs=top)
    for kw in (dict(tokens=t), dict(logprob=o), dict(tokens=t.double(), logprob=o), dict(tokens=t, logprob=o.half()),
               dict(tokens=t[:2], logprob=o), dict(entropy=torch.zeros(2)), dict(top_ids=ids), dict(top_logprobs=top),
               dict(top_ids=ids.long(), top_logprobs=top), dict(top_ids=ids, top_logprobs=top[:, :3]),
               dict(entropy=torch.zeros(3), workspace=torch.zeros(4))):
        refused(eng.logprobs, x, **kw)


def test_workspace_sizes():
    f = engine.lib().gm_logprobs_workspace
    assert f(0, 1000, 5) == 0
    for n in (1, 5, 64, 1023, 70000):
        for V in (1, 50, 4096, 131072):
            assert f(n, V, 0) <= f(n, V, min(V, 64)) < 1 << 40


@pytest.mark.parametrize("V", [1000, 4097, 9000, 40000, 131072, (1 << 31) - 1])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_workspace_serves_smaller_batches(shim, V, top):
    """The workspace of the largest batch is enough for every smaller one, and no more than some batch needs."""
    f = engine.lib().gm_logprobs_workspace
    sizes = [*range(70), 85, 86, 127, 128, 129, 204, 205, 255, 256, 257, 341, 342, 511, 512, 513, 700, 1024, 1025, 70000]

    def taken(n, bytes):
        return call(shim.plan_logprobs, lp(V=V, top=top, top_stride=top, workspace_bytes=bytes), n)[0] == 0

    for i, n in enumerate(sizes):
        assert all(taken(m, f(n, V, top)) for m in sizes[:i + 1]), n
    most = f(70000, V, top)
    assert most <= 1024 * (16 + 8 * (top + 1))
    assert most == 0 or any(not taken(m, most - 1) for m in range(1, 1025))


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
    x, y = torch.zeros(3, 96), torch.zeros(3, 64)
    for kw, want in (({}, 0x5150), (dict(stream=0), 0), (dict(stream=7), 7)):
        eng.linear(0, x, y, **kw)
        eng.block_norm(None, x, x, **kw)
        eng.logprobs(x, entropy=torch.zeros(3), **kw)
        assert queued == [("gm_linear", want), ("gm_block_norm", want), ("gm_logprobs", want)]
        queued.clear()
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: False)
    eng.linear(0, x, y)
    assert queued == [("gm_linear", 0)]


def test_counts_past_32_bits(eng):
    """Rows, sizes and indices that the library's 32-bit counts cannot hold are refused, not cut to their low bits."""
    many, row = (1 << 32) + 1, torch.zeros(1, 96)
    x, y = row.expand(many, 96), torch.zeros(1, 64).expand(many, 64)
    long = torch.zeros(1).expand(1, (1 << 32) + 8)
    refused(eng.linear, 0, x, y)
    refused(eng.block_norm, None, x, x)
    refused(eng.logprobs, x, entropy=torch.zeros(1).expand(many))
    for f, args in ((eng.block_norm, (None, long, long)), (eng.logprobs, (long,)), (eng.release_matrix, (1 << 32,)),
                    (eng.release_matrix, (-1,)), (Engine.logprobs_workspace, (1 << 32, 1000)), (Engine.logprobs_workspace, (-1, 1000)),
                    (Engine.logprobs_workspace, (4, (1 << 32) + 1000, 5)), (eng.add_matrix, ("q4_0", (1 << 32) + 4, 64, None))):
        with pytest.raises(ValueError, match="32-bit"):
            f(*args)


def test_block_norm_in_place_layouts(shim):
    """Outputs at an input's address have its type and stride; one row has no stride."""
    def takes(n, **kw):
        apart = dict(h=rows(data=A), x=rows(data=2 * A), out=rows(data=3 * A), normed=rows(data=4 * A))
        return call(shim.plan_norm, norm(**{**apart, **kw}), n)[0] == 0

    for to, at in (("out", 2 * A), ("normed", A), ("out", A), ("normed", 2 * A)):
        assert takes(3, **{to: rows(data=at)}) and takes(1, **{to: rows(data=at, stride=100)})
        assert not takes(3, **{to: rows(data=at, stride=100)})
        assert not takes(3, **{to: rows(1, data=at)}) and not takes(1, **{to: rows(2, data=at)})
    assert takes(3, out=rows(1, data=3 * A, stride=100))
    assert takes(3, h=Rows(), out=Rows()) and takes(3, h=Rows(), normed=Rows())


@pytest.mark.parametrize("case", ref.SECOND_RUNS)
def test_second_runs(shim, case):
    """The products that tests run for it do take the few-token kernel with more runs of rows than groups."""
    r, cols, fmt, group, mins, gated, x, n, whole = case
    d = matrix(engine.MATRIX_FORMATS[fmt], r, cols, group, mins=A if mins and fmt == "q4" else None)
    if gated:
        d.up_quants = A
        d.up_scales, d.up_mins = d.scales, d.mins
    type, out, why = ("f32", "bf16", "f16").index(x), (C.c_uint32 * 62)(), C.create_string_buffer(200)
    a, b = rows(type, 1 << 12), rows(stride=r)
    assert shim.plan_linear(C.byref(d), C.byref(a), n, C.byref(b), 0, 0, 1.0, out, why) == 0
    tiles, chunks, wk = out[2 + 6], out[2 + 7], out[2 + 26]
    runs, operands = -(-tiles // (2 * (8 // wk))), n * (3, 1, 2)[type]
    assert why.value.decode() == ("mv_q4_m" if mins else "mv_q4") and out[1] == 1 and runs > out[0]
    assert whole == ((81920 - 8 * 2 * operands * 64) // (operands * 256) >= chunks)
