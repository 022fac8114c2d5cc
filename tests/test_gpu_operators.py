"""The operators around the MoE layers (gm_linear, gm_block_norm, gm_logprobs) on the GPU against plain forms in
64 bits: formats, types, sizes from one token to hundreds, odd sizes, strides and alignments, rows that a
mask leaves empty, infinities and NaNs, captured graphs, and a run of them together.

Tolerances. linear: with small integers as activations, powers of two as scales and integer minima every
partial sum is a multiple of 1/4 below 2^22, so the result is exact in fp32 whatever the order. Otherwise a product goes
through at most 32 + 32 roundings in a group's two matrix products, one per group after that and 12 where slices and
parts meet, each of at most a unit of fp32's last place of a partial sum of at most 55 |s| sum |x| + |m| sum |x| (q + 16
plus 24): (76 + groups) 2^-23 of their total. Where the corrections are added to the sums, in fours, that is at most
two more a group, for roundings of half as much: within the same. block_norm: a sum of at most 16384 squares (64 adds
per lane and 10 across them, halved by the root) and at most 24 roundings: 64 2^-24 of each term. logprobs: S sums V
positive terms, at most V / 256 + 32 in a row, each term within 4 2^-24 (1 + |d|); z, m and log S round once each.
Outputs in 16 bits add half a step of their type."""
import numpy as np
import pytest
import torch

import op_reference as ref
from gyrodx.engine import Engine

pytestmark = pytest.mark.gpu
ULP = 2.0 ** -24


@pytest.fixture(scope="module")
def eng():
    e = Engine(max_tok=8)
    yield e
    e.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- linear ----------------------------------------------------------------------------------------

def add(eng, rng, fmt, rows, cols, group, mins, gated, exact):
    mats = [ref.random_matrix(rng, fmt, rows, cols, group, mins, exact) for _ in range(2 if gated else 1)]
    index = eng.add_matrix(fmt, rows, cols, mats[0][0], up=mats[1][0] if gated else None, group=group)
    return index, mats


def integers(rng, n, cols, cut=None):
    """Small whole activations."""
    x = rng.integers(-3, 4, (n, cols)).astype(np.float64)
    return torch.from_numpy(x)


FORMATS = [("q4_0", 32, False), ("q4_1", 32, True), ("q4", 32, False), ("q4", 64, True), ("q4", 64, False),
           ("q4", 128, True), ("q4", 128, False)]


@pytest.mark.parametrize("fmt,group,mins", FORMATS)
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
def test_linear_exact(eng, fmt, group, mins, x):
    rng = np.random.default_rng(group + len(fmt) + ord(x[0]))
    for rows, cols, n in ((1, group, 1), (16, 128, 1), (17, 3 * 128 + group, 2), (100, 1024, 6), (300, 2560, 16),
                          (1000, 512, 9), (33, 128 * 9, 37)):
        print(f"linear exact {fmt} group {group} mins {mins} x {x}: {rows} x {cols}, {n} tokens", flush=True)
        index, ((_, W, _, _),) = add(eng, rng, fmt, rows, cols, group, mins, False, True)
        xs = integers(rng, n, cols, x)
        xd, _ = ref.wide_rows(xs, ref.DTYPES[x], pad=8)
        yd, buf = ref.wide_rows(torch.zeros(n, rows), torch.float32, pad=3, fill=7.0)
        eng.linear(index, xd, yd, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(yd.cpu().double(), xs @ W.T)
        assert ref.untouched(buf, yd, 7.0)
        eng.release_matrix(index)


def linear_bound(mats, x, cols, group):
    _, _, s, m = mats
    return (76 + cols // group) * 2 * ULP * (x.abs() @ (55 * s + m).T)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f32", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols,n,fmt,group,mins", [
    (48, 512, 1, "q4_0", 32, False), (640, 2560, 3, "q4_1", 32, True), (1024, 2048, 5, "q4", 64, True),
    (500, 640, 8, "q4", 128, False), (129, 4128, 16, "q4_0", 32, False), (2048, 512, 33, "q4", 32, True),
    (77, 8192, 70, "q4", 128, True), (520, 2048, 130, "q4_1", 32, True)])
def test_linear(eng, rows, cols, n, fmt, group, mins, xt, yt, gated):
    rng = np.random.default_rng(rows + cols + n)
    print(f"linear {rows} x {cols}, {n} tokens, {fmt} {group} {mins}, {xt} -> {yt}, gated {gated}", flush=True)
    index, mats = add(eng, rng, fmt, rows, cols, group, mins, gated, False)
    xs = torch.from_numpy(rng.standard_normal((n, cols)))
    xs[:, ::61] *= 20
    xd, _ = ref.wide_rows(xs, ref.DTYPES[xt], pad=rng.integers(0, 9))
    x = xd.cpu().double()
    yd, buf = ref.wide_rows(torch.zeros(n, rows), ref.DTYPES[yt], pad=1, fill=3.0)
    eng.linear(index, xd, yd, stream=stream())
    torch.cuda.synchronize()
    y = x @ mats[0][1].T
    bound = linear_bound(mats[0], x, cols, group)
    if gated:
        u, bu = x @ mats[1][1].T, linear_bound(mats[1], x, cols, group)
        # |silu'| <= 1.1; expf and the division round a few times.
        bound = 1.1 * bound * u.abs() + bu * (ref.silu(y).abs() + 1.1 * bound) + 16 * ULP * (ref.silu(y) * u).abs()
        y = ref.silu(y) * u
    bound = bound + ref.half_step(ref.DTYPES[yt]) * (y.abs() + bound) + 1e-7 * (yt == "f16")
    err = (yd.cpu().double() - y).abs()
    print(f"  err / bound {float((err / bound).max()):.4f}, rel rms {float(err.norm() / y.norm()):.2e}", flush=True)
    assert (err <= bound).all()
    if yt == "f32":
        # Roundings are as often up as down: their sum stays near the root of their number, sqrt(76 + groups) 2^-24
        # of a partial sum's size, at most 55 / 4.6 (the rms of q - 8) of the result's.
        assert err.norm() <= (2.0 if gated else 1.0) * 12 * np.sqrt(76 + cols // group) * ULP * y.norm()
    assert ref.untouched(buf, yd, 3.0)
    eng.release_matrix(index)


# Shapes whose products take the many-token kernels, by 16, 32, 48 and 64 tokens a group (test_operator_calls.py).
MANY = [(40000, 1, 12), (100003, 1, 30), (100003, 1, 45), (100003, 1, 64), (8000, 3, 1000), (8000, 5, 500), (8000, 3, 700)]


@pytest.mark.parametrize("fmt,group,mins", FORMATS)
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
def test_linear_many_tokens_exact(eng, fmt, group, mins, x):
    rng = np.random.default_rng(7 * group + len(fmt) + ord(x[0]))
    for rows, groups, n in MANY:
        n += 8 * (x == "bf16" and n == 12)
        cols = groups * group
        print(f"many tokens exact {fmt} group {group} mins {mins} x {x}: {rows} x {cols}, {n} tokens", flush=True)
        index, ((_, W, _, _),) = add(eng, rng, fmt, rows, cols, group, mins, False, True)
        xs = integers(rng, n, cols, x)
        xd, _ = ref.wide_rows(xs, ref.DTYPES[x], pad=3, shift=1)
        yd, buf = ref.wide_rows(torch.zeros(n, rows), torch.float32, pad=5, shift=3, fill=7.0)
        eng.linear(index, xd, yd, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(yd.cpu().double(), xs @ W.T)
        assert ref.untouched(buf, yd, 7.0)
        eng.release_matrix(index)


@pytest.mark.parametrize("group,mins", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
def test_linear_many_tokens_chunks(eng, group, mins, x):
    """One to eight chunks of 128 columns, the last one whole or not, by 16 to 64 tokens a group."""
    rng = np.random.default_rng(group + ord(x[0]))
    for chunks in range(1, 9):
        for cols in {128 * chunks, 128 * chunks - (96 if group == 32 else 64 if group == 64 else 0)}:
            index, ((_, W, _, _),) = add(eng, rng, "q4", 30001, cols, group, mins, False, True)
            for n in (17, 30, 47, 60):
                print(f"chunks, group {group} mins {mins} x {x}: {cols} columns, {n} tokens", flush=True)
                xs = integers(rng, n, cols)
                yd = torch.zeros(n, 30001, device="cuda")
                eng.linear(index, xs.to(ref.DTYPES[x]).cuda(), yd, stream=stream())
                assert torch.equal(yd.cpu().double(), xs @ W.T)
            eng.release_matrix(index)


def test_linear_many_tokens_graph(eng):
    """A captured product of many tokens, replayed with eager ones of other inputs between."""
    rng = np.random.default_rng(12)
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", 20000, 640, 32, False, False, True)
    xs = [integers(rng, 40, 640) for _ in range(4)]
    x, y, other = torch.zeros(40, 640, device="cuda"), torch.zeros(40, 20000, device="cuda"), torch.zeros(40, 20000, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        eng.linear(index, x, y, stream=stream())
    for i in range(4):
        x.copy_(xs[i])
        g.replay()
        eng.linear(index, xs[i - 1].float().cuda(), other, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(y.cpu().double(), xs[i] @ W.T) and torch.equal(other.cpu().double(), xs[i - 1] @ W.T)
    eng.release_matrix(index)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("rows,cols,n,fmt,group,mins", [(20001, 640, 50, "q4_0", 32, False), (20001, 384, 70, "q4", 128, True),
                                                        (6007, 1088, 200, "q4", 64, False), (30010, 96, 20, "q4_1", 32, True)])
def test_linear_many_tokens(eng, rows, cols, n, fmt, group, mins, xt, yt, gated):
    test_linear(eng, rows, cols, n, fmt, group, mins, xt, yt, gated)


@pytest.mark.parametrize("yt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["none", "silu", "sigmoid"])
def test_linear_many_tokens_epilogue(eng, act, yt):
    """Activation, scale and accumulation of the many-token kernels, rows not in fours, added to what y held."""
    rng = np.random.default_rng(15)
    rows, cols, n = 40003, 64, 33
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", rows, cols, 32, False, False, True)
    xs = integers(rng, n, cols)
    y0 = torch.from_numpy(rng.standard_normal((n, rows)))
    for accumulate in (False, True):
        yd, buf = ref.wide_rows(y0, ref.DTYPES[yt], pad=1, shift=1, fill=2.0)
        held = yd.cpu().double()
        eng.linear(index, xs.bfloat16().cuda(), yd, act=act, accumulate=accumulate, scale=0.03125, stream=stream())
        z = 0.03125 * (xs @ W.T)
        want = {"none": z, "silu": ref.silu(z), "sigmoid": torch.sigmoid(z)}[act]
        part = want.abs() + z.abs() + 1
        want = want + held if accumulate else want
        err = (yd.cpu().double() - want).abs()
        assert (err <= 8 * ULP * (part + want.abs()) + half_step(ref.DTYPES[yt]) * (want.abs() + 1e-6) + 1e-7 * (yt == "f16")).all()
        assert ref.untouched(buf, yd, 2.0)
    eng.release_matrix(index)


@pytest.mark.parametrize("act", ["none", "silu", "sigmoid"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_linear_epilogue(eng, act, accumulate):
    rng = np.random.default_rng(5)
    rows, cols, n = 130, 256, 4
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", rows, cols, 32, False, False, True)
    xs = integers(rng, n, cols, "f32")
    y0 = torch.from_numpy(rng.standard_normal((n, rows))).float()
    yd = y0.cuda()
    eng.linear(index, xs.float().cuda(), yd, act=act, accumulate=accumulate, scale=0.03125, stream=stream())
    z = 0.03125 * (xs @ W.T)
    want = {"none": z, "silu": ref.silu(z), "sigmoid": torch.sigmoid(z)}[act]
    want = want + y0.double() if accumulate else want
    err = (yd.cpu().double() - want).abs()
    assert (err <= 8 * ULP * (want.abs() + (want - y0).abs() + z.abs() + 1)).all()
    eng.release_matrix(index)


@pytest.mark.parametrize("xt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift,pad", [(1, 0), (3, 5), (0, 4), (2, 1)])
def test_linear_alignment(eng, xt, shift, pad):
    rng = np.random.default_rng(shift + pad)
    rows, cols, n = 70, 352, 7
    index, ((_, W, _, _),) = add(eng, rng, "q4_1", rows, cols, 32, True, False, True)
    xs = integers(rng, n, cols, xt)
    xd, _ = ref.wide_rows(xs, ref.DTYPES[xt], pad=pad, shift=shift)
    yd, buf = ref.wide_rows(torch.zeros(n, rows), torch.float32, pad=pad, shift=shift, fill=9.0)
    eng.linear(index, xd, yd, stream=stream())
    assert torch.equal(yd.cpu().double(), xs @ W.T)
    assert ref.untouched(buf, yd, 9.0)
    eng.release_matrix(index)


def test_linear_broadcast_and_empty(eng):
    rng = np.random.default_rng(1)
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", 40, 96, 32, False, False, True)
    xs = integers(rng, 1, 96, "f32")
    yd = torch.zeros(9, 40, device="cuda")
    eng.linear(index, xs.float().cuda().expand(9, 96), yd, stream=stream())
    assert torch.equal(yd.cpu().double(), (xs @ W.T).expand(9, 40))
    eng.linear(index, torch.zeros(0, 96, device="cuda"), torch.zeros(0, 40, device="cuda"), stream=stream())
    eng.release_matrix(index)


@pytest.mark.parametrize("n,rows", [(3, 200), (40, 200), (40, 20000)])
@pytest.mark.parametrize("xt", ["f32", "bf16", "f16"])
def test_linear_nonfinite_token(eng, xt, n, rows):
    """Of a token with an infinity or a NaN no output is finite; the others keep their bits."""
    rng = np.random.default_rng(2)
    index, _ = add(eng, rng, "q4", rows, 640, 64, True, False, False)
    xs = torch.from_numpy(rng.standard_normal((n, 640))).to(ref.DTYPES[xt]).cuda()
    clean, dirty = torch.zeros(n, rows, device="cuda"), torch.zeros(n, rows, device="cuda")
    eng.linear(index, xs, clean, stream=stream())
    for value in (float("inf"), float("-inf"), float("nan")):
        xs[1, 333] = value
        eng.linear(index, xs, dirty, stream=stream())
        assert not torch.isfinite(dirty[1]).any()
        keep = [t for t in range(n) if t != 1]
        assert torch.equal(dirty[keep], clean[keep])
    eng.release_matrix(index)


@pytest.mark.parametrize("n,rows", [(4, 64), (50, 64), (50, 20000)])
@pytest.mark.parametrize("xt,sizes", [("f32", (1e-30, 1e-5, 1.0, 1e20)), ("bf16", (1e-30, 1e-5, 1e20)),
                                      ("f16", (1e-7, 1e-5, 1.0, 5000.0))])
def test_linear_wide_range(eng, xt, sizes, n, rows):
    """Activations keep all their bits, at any size: fp32's 24, binary16's below its normal range."""
    rng = np.random.default_rng(3)
    index, (mats,) = add(eng, rng, "q4_0", rows, 256, 32, False, False, False)
    for size in sizes:
        x = torch.from_numpy(rng.standard_normal((n, 256)) * size).to(ref.DTYPES[xt])
        yd = torch.zeros(n, rows, device="cuda")
        eng.linear(index, x.cuda(), yd, stream=stream())
        y = x.double() @ mats[1].T
        assert ((yd.cpu().double() - y).abs() <= linear_bound(mats, x.double(), 256, 32) + ULP * y.abs()).all()
    eng.release_matrix(index)


@pytest.mark.parametrize("n,rows", [(4, 64), (50, 64), (50, 20000)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("xt,sizes", [("f32", (1e-30, 1.0, 1e20)), ("bf16", (1e-30, 1e20)), ("f16", (1e-7, 1e-5, 5000.0))])
def test_linear_minima_wide_range(eng, xt, sizes, group, n, rows):
    """The sums that minima multiply keep all bits as well."""
    rng = np.random.default_rng(5)
    index, (mats,) = add(eng, rng, "q4", rows, 384, group, True, False, False)
    for size in sizes:
        x = torch.from_numpy(rng.standard_normal((n, 384)) * size).to(ref.DTYPES[xt])
        yd = torch.zeros(n, rows, device="cuda")
        eng.linear(index, x.cuda(), yd, stream=stream())
        y = x.double() @ mats[1].T
        assert ((yd.cpu().double() - y).abs() <= linear_bound(mats, x.double(), 384, group) + ULP * y.abs()).all()
    eng.release_matrix(index)


def far_rows(n, width, stride, dtype):
    """[n, width] zeros whose rows are `stride` values apart (memory between them untouched)."""
    view = torch.empty((n - 1) * stride + width, dtype=dtype, device="cuda").as_strided((n, width), (stride, 1))
    view.zero_()
    return view


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("n,rows", [(70, 40), (70, 20000)])
def test_linear_far_rows(eng, xt, n, rows):
    """Inputs and outputs whose offsets pass 32 bits, in few and in many tokens' kernels."""
    rng = np.random.default_rng(6)
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", rows, 160, 32, False, False, True)
    xs = integers(rng, n, 160)
    x = far_rows(n, 160, 1 << 24, ref.DTYPES[xt])
    x.copy_(xs)
    y = far_rows(n, rows, (1 << 25) + 3, torch.bfloat16)
    eng.linear(index, x, y, stream=stream())
    assert torch.equal(y.cpu(), (xs @ W.T).bfloat16())
    eng.release_matrix(index)


def test_norm_and_logprobs_far_rows(eng):
    n, stride = 20, (1 << 28) + 1
    x, out = far_rows(n, 100, stride, torch.bfloat16), far_rows(n, 100, stride, torch.bfloat16)
    xs = torch.randn(n, 100, generator=torch.Generator().manual_seed(1)).bfloat16()
    x.copy_(xs)
    near = torch.zeros(n, 100, dtype=torch.bfloat16, device="cuda")
    eng.block_norm(None, xs.cuda(), None, near, stream=stream())
    eng.block_norm(None, x, None, out, stream=stream())
    assert torch.equal(out, near) and near.abs().sum() > 0
    a, b = ([torch.zeros(n, 3, dtype=torch.int32, device="cuda"), torch.zeros(n, 3, device="cuda"), torch.zeros(n, device="cuda")]
            for _ in range(2))
    for t, (ids, top, entropy) in ((xs.cuda(), a), (x, b)):
        eng.logprobs(t, top_ids=ids, top_logprobs=top, entropy=entropy, stream=stream())
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[2].min() > 0


def test_matrix_indices(eng):
    rng = np.random.default_rng(4)
    first, ((_, W, _, _),) = add(eng, rng, "q4_0", 32, 64, 32, False, False, True)
    second, ((_, W2, _, _),) = add(eng, rng, "q4_0", 48, 96, 32, False, False, True)
    assert first != second
    eng.release_matrix(first)
    with pytest.raises(RuntimeError, match="no such matrix"):
        eng.release_matrix(first)
    third, ((_, W3, _, _),) = add(eng, rng, "q4_0", 16, 32, 32, False, False, True)
    for index, W, cols in ((second, W2, 96), (third, W3, 32)):
        xs = integers(rng, 2, cols, "f32")
        yd = torch.zeros(2, W.shape[0], device="cuda")
        eng.linear(index, xs.float().cuda(), yd, stream=stream())
        assert torch.equal(yd.cpu().double(), xs @ W.T)
        eng.release_matrix(index)


# ---- block norm ------------------------------------------------------------------------------------

def norm_case(eng, rng, n, E, ht, st, nt, gate, gate_act, post, weights, pad, shift=0, in_place=False):
    g = lambda *s: torch.from_numpy(rng.standard_normal(s))  # noqa: E731
    h, _ = ref.wide_rows(g(n, E) * 0.3, ref.DTYPES[ht], pad=pad, shift=shift)
    x, _ = ref.wide_rows(g(n, E) * 2, ref.DTYPES[st], pad=pad, shift=shift)
    pw = (1 + 0.1 * g(E)).float().cuda() if post and weights else None
    nw = (1 + 0.1 * g(E)).float().cuda() if weights else None
    shape = {None: None, "token": (n, 1), "channel": (1, E), "value": (n, E)}[gate]
    gt = None if shape is None else g(*shape).to(ref.DTYPES[ht]).cuda()
    v, z, part = ref.block_norm(h.cpu(), x.cpu(), post, None if pw is None else pw.cpu(), 1e-5,
                                None if gt is None else gt.cpu(), gate_act, 0.7, None if nw is None else nw.cpu(), 1e-6)
    if in_place:
        out, ob, normed, nb = x, None, h, None
    else:
        out, ob = ref.wide_rows(torch.zeros(n, E), ref.DTYPES[st], pad=pad, shift=shift, fill=5.0)
        normed, nb = ref.wide_rows(torch.zeros(n, E), ref.DTYPES[nt], pad=pad, shift=shift, fill=5.0)
    eng.block_norm(h, x, out, normed, post=post, post_weight=pw, post_eps=1e-5, gate=gt, gate_act=gate_act, scale=0.7,
                   pre_weight=nw, pre_eps=1e-6, stream=stream())
    dv = 2 * ULP * v.abs() + 64 * ULP * part.abs()
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * (1 if nw is None else nw.cpu().double())
    dz = 64 * ULP * z.abs() + dv * r.abs() + z.abs() * (dv.norm(dim=-1, keepdim=True) / v.norm(dim=-1, keepdim=True).clamp_min(1e-30))
    for got, want, d in ((out, v, dv), (normed, z, dz)):
        t = got.dtype
        tiny = 2.0 ** -25 if t == torch.float16 else 0.0
        assert ((got.cpu().double() - want).abs() <= d + half_step(t) * (want.abs() + d) + tiny).all()
    if not in_place:
        assert ref.untouched(ob, out, 5.0) and ref.untouched(nb, normed, 5.0)


def half_step(t):
    return 0.0 if t == torch.float32 else ref.half_step(t)


@pytest.mark.parametrize("n,E", [(1, 1), (1, 2048), (3, 7), (5, 2560), (17, 2047), (2, 4096), (3, 4097), (2, 16384),
                                 (300, 128), (9, 8200)])
@pytest.mark.parametrize("gate,gate_act", [(None, "none"), ("token", "sigmoid"), ("channel", "none"), ("value", "sigmoid")])
def test_block_norm(eng, n, E, gate, gate_act):
    rng = np.random.default_rng(n + E)
    for i, (ht, st, nt) in enumerate((("f32", "f32", "f32"), ("bf16", "f32", "bf16"), ("f16", "f16", "f32"),
                                      ("bf16", "bf16", "bf16"))):
        print(f"block_norm {n} x {E} gate {gate} {gate_act} {ht} {st} {nt}", flush=True)
        norm_case(eng, rng, n, E, ht, st, nt, gate, gate_act, post=i != 2, weights=i != 1, pad=(0, 3, 8, 1)[i],
                  shift=(0, 1, 0, 3)[i])


def test_block_norm_in_place(eng):
    for t in ("f32", "bf16"):
        norm_case(eng, np.random.default_rng(8), 6, 1000, t, t, t, "token", "none", True, True, 0, in_place=True)


def test_block_norm_parts(eng):
    """Without h the stream passes; out and normed are each optional; n = 0 does nothing."""
    x = torch.randn(5, 640, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    out, normed = torch.zeros_like(x), torch.zeros_like(x)
    eng.block_norm(None, x, out, normed, stream=stream())
    assert torch.equal(out, x)
    v, z, _ = ref.block_norm(None, x.cpu(), False, None, 0, None, None, 1, None, 1e-6)
    assert ((normed.cpu().double() - z).abs() <= 64 * ULP * z.abs()).all()
    h = torch.randn_like(x)
    both, alone = [torch.zeros_like(x) for _ in range(2)], [torch.zeros_like(x) for _ in range(2)]
    eng.block_norm(h, x, *both, post=True, stream=stream())
    eng.block_norm(h, x, alone[0], None, post=True, stream=stream())
    eng.block_norm(h, x, None, alone[1], post=True, stream=stream())
    assert torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])
    eng.block_norm(h[:0], x[:0], out[:0], None, stream=stream())


def test_block_norm_zero_rows(eng):
    """Rows of zeros stay zeros (eps keeps the root from zero)."""
    x = torch.zeros(3, 512, device="cuda")
    out, normed = torch.ones_like(x), torch.ones_like(x)
    eng.block_norm(x, x, out, normed, post=True, stream=stream())
    assert (out == 0).all() and (normed == 0).all()


def test_block_norm_many_rows(eng):
    """More rows than one grid dimension holds."""
    n = 65535 + 70
    x = torch.randn(n, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    normed = torch.zeros_like(x)
    eng.block_norm(None, x, None, normed, stream=stream())
    _, z, _ = ref.block_norm(None, x.cpu(), False, None, 0, None, None, 1, None, 1e-6)
    assert ((normed.cpu().double() - z).abs() <= 64 * ULP * z.abs()).all()


# ---- log probabilities -------------------------------------------------------------------------------

def logprobs_case(eng, x, tokens, top, scale=1.0, pad=0, shift=0, int64=True, entropy=True):
    """x: the rows on the CPU in their type."""
    n, V = x.shape
    xd, _ = ref.wide_rows(x, x.dtype, pad=pad, shift=shift, fill=float("nan"))
    td = None if tokens is None else tokens.to(torch.int64 if int64 else torch.int32).cuda()
    lp = None if tokens is None else torch.full(tokens.shape, 77.0, device="cuda")
    H = torch.full((n,), 77.0, device="cuda") if entropy else None
    ids = torch.full((n, top), -5, dtype=torch.int32, device="cuda") if top else None
    tl = torch.full((n, top), 77.0, device="cuda") if top else None
    ws = torch.full((eng.logprobs_workspace(n, V, top),), 0xA5, dtype=torch.uint8, device="cuda")
    eng.logprobs(xd, ws, tokens=td, logprob=lp, entropy=H, top_ids=ids, top_logprobs=tl, scale=scale, stream=stream())
    torch.cuda.synchronize()
    given, want_H, all_lp, m, logs, ts = ref.logprobs(x, tokens, scale)
    z = x.double() * scale
    m0 = torch.where(torch.isfinite(m), m, 0.0)
    sum_err = (V / 256 + 32) * ULP + 4 * ULP * (1 + ts.abs().nan_to_num(0))
    tol = 2 * ULP * (z.abs().nan_to_num(0, 0, 0) + 2 * m0.abs() + logs.abs().nan_to_num(0) + 1) + sum_err

    def same(got, want, tol):
        got, want = got.cpu().double(), want.float().double()  # past the largest fp32: -infinity
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        fine = torch.isfinite(want)
        assert torch.equal(got[~fine].nan_to_num(1.0), want[~fine].nan_to_num(1.0))
        assert ((got - want).abs()[fine] <= tol.expand_as(want)[fine]).all(), float(((got - want).abs() / tol)[fine].max())

    if tokens is not None:
        inside = torch.where((tokens >= 0) & (tokens < V), tokens, 0).long()
        same(lp, given, tol.gather(1, inside))
    if entropy:
        same(H, want_H, (sum_err * (2 + ts.abs().nan_to_num(0)) + 4 * ULP * (logs.abs().nan_to_num(0) + 1))[:, 0])
    if top:
        want = ref.order(x)[:, :top]
        assert torch.equal(ids.cpu().long(), want)
        same(tl, all_lp.gather(1, want), tol.gather(1, want))


def random_logits(rng, n, V, dtype):
    x = rng.standard_normal((n, V)) * 2.5
    x[np.arange(n), rng.integers(0, V, n)] += 8
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,V,top,given", [(1, 1, 1, 1), (2, 3, 3, 2), (3, 63, 20, 1), (1, 64, 64, 0), (5, 1000, 5, 3),
                                           (4, 2049, 64, 1), (2, 32768, 20, 1), (1, 100003, 50, 64), (7, 65537, 1, 1),
                                           (300, 517, 8, 1), (1, 131072, 0, 1), (520, 4099, 3, 1)])
def test_logprobs(eng, dtype, n, V, top, given):
    rng = np.random.default_rng(V + n)
    print(f"logprobs {n} x {V} {dtype} top {top} given {given}", flush=True)
    x = random_logits(rng, n, V, ref.DTYPES[dtype])
    tokens = torch.from_numpy(rng.integers(0, V, (n, given))) if given else None
    logprobs_case(eng, x, tokens, top, scale=1.0 if n % 2 else 0.75, int64=V % 2 == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shift,pad", [(1, 0), (2, 3), (5, 7), (7, 0), (0, 1)])
def test_logprobs_alignment(eng, dtype, shift, pad):
    rng = np.random.default_rng(shift * 10 + pad)
    for V in (5, 8, 17, 1023, 4101):
        x = random_logits(rng, 3, V, ref.DTYPES[dtype])
        logprobs_case(eng, x, torch.from_numpy(rng.integers(0, V, (3, 1))), min(V, 6), pad=pad, shift=shift)


@pytest.mark.parametrize("V", [7, 1500, 9000, 70000])
def test_logprobs_masked_rows(eng, V):
    """Banned tokens, rows of nothing but -infinity, of the type's lowest value, with one token left, NaN, +infinity."""
    rng = np.random.default_rng(V)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        print(f"masked rows V {V} {dtype}", flush=True)
        x = random_logits(rng, 10, V, dtype)
        x[0] = float("-inf")
        x[1] = torch.finfo(dtype).min
        x[2, :] = float("-inf")
        x[2, V // 2] = 1.5
        x[3, ::2] = float("-inf")
        x[4, ::3] = torch.finfo(dtype).min
        x[5, V // 3] = float("nan")
        x[6, V - 1] = float("inf")
        x[7, 1:] = float("-inf")
        x[8] = float("nan")
        tokens = torch.from_numpy(rng.integers(0, V, (10, 2)))
        tokens[2, 0] = V // 2
        for scale in (1.0, 2.0):
            logprobs_case(eng, x, tokens, min(V, 20), scale=scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [130, 4096, 50001])
def test_logprobs_ties_and_orders(eng, dtype, V):
    """Equal logits, signed zeros, rising and falling rows, all the largest in one place."""
    rows = [torch.zeros(V), torch.full((V,), -3.5), torch.arange(V) % 3 - 1.0, torch.linspace(-8, 8, V),
            torch.linspace(8, -8, V), torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0),
            torch.where(torch.arange(V) % 256 < 4, 5.0, -1.0), torch.where(torch.arange(V) > V - 100, 9.0, 0.0),
            torch.where(torch.arange(V) % 64 == 3, torch.arange(V) * 1e-3, -2.0)]
    x = torch.stack(rows).to(dtype)
    for top in (1, 20, 64):
        logprobs_case(eng, x, torch.full((len(rows), 1), V - 1), top)


def test_logprobs_tokens_outside(eng):
    x = random_logits(np.random.default_rng(0), 2, 300, torch.float32)
    for int64 in (True, False):
        logprobs_case(eng, x, torch.tensor([[0, -1, 300, 299], [-100, 2 ** 31 - 1, 5, 5]]), 0, int64=int64)


def test_logprobs_many_rows(eng):
    """More rows than one grid dimension holds; only the entropy, only the top."""
    x = random_logits(np.random.default_rng(1), 65535 + 9, 12, torch.float32)
    logprobs_case(eng, x, None, 2)
    logprobs_case(eng, x[:70], None, 0)
    logprobs_case(eng, x[:70], None, 3, entropy=False)


# ---- streams, graphs, a run together ---------------------------------------------------------------

class Chain:
    """A decode step's tail: norms, a gated 4-bit feed-forward, norms, the 4-bit head, log probabilities."""
    E, F, V, TOP = 512, 640, 5003, 10

    def __init__(self, eng, n, seed):
        rng = np.random.default_rng(seed)
        self.eng, self.n = eng, n
        self.ff, self.ffm = add(eng, rng, "q4", self.F, self.E, 64, True, True, False)
        self.down, self.downm = add(eng, rng, "q4_0", self.E, self.F, 32, False, False, False)
        self.head, self.headm = add(eng, rng, "q4_1", self.V, self.E, 32, True, False, False)
        z = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        self.h, self.x, self.normed = z(n, self.E), z(n, self.E), z(n, self.E)
        self.act, self.y, self.last = z(n, self.F), z(n, self.E), z(n, self.E)
        self.logits, self.lp, self.H = z(n, self.V), z(n, 1), z(n)
        self.ids, self.tl = z(n, self.TOP, t=torch.int32), z(n, self.TOP)
        self.tokens = z(n, 1, t=torch.int64)
        self.ws = z(max(1, eng.logprobs_workspace(n, self.V, self.TOP)), t=torch.uint8)
        self.w = torch.from_numpy(1 + 0.1 * rng.standard_normal(self.E)).float().cuda()
        self.gate = torch.from_numpy(rng.standard_normal((1, self.E))).float().cuda()

    def set(self, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        self.h.copy_(torch.randn(self.n, self.E, device="cuda", generator=g))
        self.x.copy_(torch.randn(self.n, self.E, device="cuda", generator=g))
        self.tokens.copy_(torch.randint(0, self.V, (self.n, 1), device="cuda", generator=g))

    def run(self):
        e, s = self.eng, stream()
        e.block_norm(self.h, self.x, self.x, self.normed, pre_weight=self.w, stream=s)
        e.linear(self.ff, self.normed, self.act, stream=s)
        e.linear(self.down, self.act, self.y, stream=s)
        e.block_norm(self.y, self.x, self.x, self.last, post=True, post_weight=self.w, gate=self.gate,
                     gate_act="sigmoid", scale=0.5, pre_weight=self.w, stream=s)
        e.linear(self.head, self.last, self.logits, stream=s)
        e.logprobs(self.logits, self.ws, tokens=self.tokens, logprob=self.lp, entropy=self.H, top_ids=self.ids,
                   top_logprobs=self.tl, scale=0.8, stream=s)

    def outputs(self):
        return [t.clone() for t in (self.x, self.last, self.logits, self.lp, self.H, self.ids, self.tl)]

    def plain(self):
        c = lambda t: t.cpu().double()  # noqa: E731
        v, z, _ = ref.block_norm(c(self.h), c(self.x), False, None, 0, None, None, 1.0, c(self.w), 1e-6)
        a = ref.silu(z @ self.ffm[0][1].T) * (z @ self.ffm[1][1].T)
        v, z, _ = ref.block_norm(a @ self.downm[0][1].T, v, True, c(self.w), 1e-6, c(self.gate), "sigmoid", 0.5, c(self.w), 1e-6)
        logits = z @ self.headm[0][1].T
        lp, H, *_ = ref.logprobs(logits, self.tokens.cpu(), 0.8)
        return v, z, logits, lp, H

    def release(self):
        for m in (self.ff, self.down, self.head):
            self.eng.release_matrix(m)


@pytest.mark.parametrize("n", [1, 8, 70])
def test_run_together(eng, n):
    """The whole tail against 64 bits: each step adds at most a few 1e-6 of its output's norm, which the norms
    between them pass on at about one to one."""
    c = Chain(eng, n, 11)
    c.set(1)
    want = c.plain()
    c.run()
    for got, w in zip((c.x, c.last, c.logits, c.lp, c.H), want):
        assert (got.cpu().double() - w).norm() <= 1e-5 * w.norm()
    lp = torch.log_softmax(0.8 * c.logits.cpu().double(), -1)
    assert torch.equal(c.ids.cpu().long(), ref.order(c.logits.cpu())[:, :c.TOP])
    assert ((c.tl.cpu().double() - lp.gather(1, c.ids.cpu().long())).abs() <= 1e-5).all()
    c.release()


def test_side_stream_and_graphs(eng):
    """Two captured graphs, each with its workspace, replayed several times with eager work between them and against
    each other on two streams: every replay equals the eager result."""
    side = torch.cuda.Stream()
    chains = [Chain(eng, n, 21 + n) for n in (2, 5)]
    eng.load_operators()
    wants = []
    for c in chains:
        c.set(5)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            c.run()
        torch.cuda.synchronize()
        wants.append(c.outputs())
    graphs = []
    for c in chains:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    for turn in range(4):
        for c in chains:
            c.set(5)
        torch.cuda.synchronize()
        if turn % 2:
            other = torch.cuda.Stream()
            with torch.cuda.stream(side):
                graphs[0].replay()
            with torch.cuda.stream(other):
                graphs[1].replay()
        else:
            graphs[0].replay()
            chains[0].set(5)
            torch.cuda.synchronize()
            chains[0].run()
            graphs[1].replay()
        torch.cuda.synchronize()
        for c, want in zip(chains, wants):
            for got, w in zip(c.outputs(), want):
                assert torch.equal(got, w)
    for c in chains:
        c.release()


def test_default_stream_order(eng):
    """Work on torch's default stream (handle 0) and the operators' are in order without waits between them."""
    rng = np.random.default_rng(9)
    index, ((_, W, _, _),) = add(eng, rng, "q4_0", 64, 128, 32, False, False, True)
    x, y = torch.zeros(2, 128, device="cuda"), torch.zeros(2, 64, device="cuda")
    total, want = torch.zeros(2, 64, device="cuda"), torch.zeros(2, 64, dtype=torch.float64)
    for i in range(50):
        xs = torch.full((2, 128), float(i % 5 - 2))
        x.fill_(float(i % 5 - 2))
        eng.linear(index, x, y)
        total += y
        want += xs.double() @ W.T
    assert torch.equal(total.cpu().double(), want)
    eng.release_matrix(index)


def test_capture_needs_loaded_kernels():
    """A first call inside a capture is refused before anything is queued; after load_operators it is taken."""
    e = Engine(max_tok=1)
    try:
        x = torch.randn(2, 64, device="cuda")
        normed = torch.zeros_like(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.add_(0.0)
            with pytest.raises(RuntimeError, match="not loaded"):
                e.block_norm(None, x, None, normed, stream=stream())
        e.load_operators()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            e.block_norm(None, x, None, normed, stream=stream())
        g.replay()
        torch.cuda.synchronize()
        _, z, _ = ref.block_norm(None, x.cpu(), False, None, 0, None, None, 1, None, 1e-6)
        assert ((normed.cpu().double() - z).abs() <= 64 * ULP * z.abs()).all()
    finally:
        e.close()
