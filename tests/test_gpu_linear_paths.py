"""4-bit products where the shapes of the other tests do not go: second runs of rows in the few-token kernel, activations
that need every part they are cut into, the gated epilogue's scale and accumulation.

Exact cases: small whole activations, scales that are powers of two from 1/4 to 2 and integer minima give partial sums that are
multiples of 1/4 below 2^22."""
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


def half_step(t):
    return 0.0 if t == torch.float32 else ref.half_step(t)


def gated(g, u, scale=1.0):
    """(scale silu(g) u, its error) of exact g and u: the exponential of a value whose product with log2 e rounds has a relative
    error of |g| log2(e) 2^-24 ln 2 = |g| 2^-24 beside its own, the division and three products, 16 roundings at most. Past
    g = -87 the exponential or its reciprocal leaves fp32's normal range, and less than 88 e^-87 < 1e-35 |u| is lost."""
    part = scale * ref.silu(g) * u
    return part, (16 + g.abs()) * ULP * part.abs() + 1e-35 * (scale * u).abs()


@pytest.mark.parametrize("case", ref.SECOND_RUNS, ids=str)
def test_second_runs(eng, case):
    """Rows repeat a matrix of 4001, which shares no period with the runs (test_operator_calls.py: runs > groups)."""
    rows, cols, fmt, group, mins, pair, x, n, _ = case
    print(f"second runs {case}", flush=True)
    rng = np.random.default_rng(rows + cols)
    mats = [ref.random_matrix(rng, fmt, 4001, cols, group, mins, True) for _ in range(2 if pair else 1)]
    data = [ref.repeated(m[0], -(-rows // 4001), rows) for m in mats]
    index = eng.add_matrix(fmt, rows, cols, data[0], up=data[1] if pair else None, group=group)
    xs = torch.from_numpy(rng.integers(-3, 4, (n, cols)).astype(np.float64))
    xd, _ = ref.wide_rows(xs, ref.DTYPES[x], pad=5)
    yd, buf = ref.wide_rows(torch.zeros(n, rows), torch.float32, pad=3, shift=1, fill=7.0)
    eng.linear(index, xd, yd, stream=stream())
    torch.cuda.synchronize()
    want = [(xs @ m[1].T).repeat(1, -(-rows // 4001))[:, :rows] for m in mats]
    if pair:
        y, tol = gated(*want)
        assert ((yd.cpu().double() - y).abs() <= tol).all()
    else:
        assert torch.equal(yd.cpu().double(), want[0])
    assert ref.untouched(buf, yd, 7.0)
    eng.release_matrix(index)


def full_mantissas(n, cols, x):
    """One activation a token, everywhere in turn, whose mantissa is all ones: 24 bits of fp32, 11 of binary16, 8 of bf16."""
    bits = {"f32": 24, "f16": 11, "bf16": 8}[x]
    xs = torch.zeros(n, cols, dtype=torch.float64)
    t = torch.arange(n)
    xs[t, t * 37 % cols] = (2.0 - 2.0 ** (1 - bits)) * (1.0 - 2.0 * (t % 2)).double() * torch.exp2((t % 5 - 2).double())
    return xs


@pytest.mark.parametrize("fmt,group,mins", [("q4_0", 32, False), ("q4_1", 32, True), ("q4", 64, True), ("q4", 128, False)])
@pytest.mark.parametrize("x", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n", [(300, 5), (2000, 16), (40003, 40)])
def test_every_part_counts(eng, rows, n, x, fmt, group, mins):
    """With one activation a token a result is one product. The few-token kernel gives each part's exactly (8 bits by at most 8)
    and adds them smallest first: exact up to the last sum, which rounds once. The many-token one adds an fp32
    activation's three parts times 16 + q to what the 16 (or 24) is too much: six sums, each within 2^-23 of 31 |s x|, then at
    most three roundings of sums below 70 |s| |x| + |m x|. A part left out would be 2^-17 |W x| or more."""
    print(f"every part {rows} x 256, {n} tokens, {fmt} {group} {mins} {x}", flush=True)
    rng = np.random.default_rng(rows + group)
    data, W, s, m = ref.random_matrix(rng, fmt, rows, 256, group, mins, True)
    index = eng.add_matrix(fmt, rows, 256, data, group=group)
    xs = full_mantissas(n, 256, x)
    xd, yd = xs.to(ref.DTYPES[x]).cuda(), torch.zeros(n, rows, device="cuda")
    assert torch.equal(xd.cpu().double(), xs)
    eng.linear(index, xd, yd, stream=stream())
    got, want = yd.cpu(), xs @ W.T
    if x == "f32" and rows == 40003:
        bound = ULP * (12 * 31 * (xs.abs() @ s.T) + 3 * (xs.abs() @ (70 * s + (m if mins else 0)).T))
        assert ((got.double() - want).abs() <= bound).all()
        # On the whole far nearer: a part of 8 bits left out (half a unit of the 16th bit on average) would show in this.
        assert (got.double() - want).norm() <= 2.0 ** -19 * want.norm()
    else:
        assert torch.equal(got, want.float())
    eng.release_matrix(index)


@pytest.mark.parametrize("rows,n", [(130, 4), (130, 16), (20003, 40)])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("yt", ["f32", "bf16", "f16"])
def test_gated_epilogue(eng, yt, accumulate, rows, n):
    """scale silu(G x) (U x), added to what y holds or not, in both kernels."""
    print(f"gated epilogue {rows} rows, {n} tokens, {yt}, accumulate {accumulate}", flush=True)
    rng = np.random.default_rng(rows + n)
    mats = [ref.random_matrix(rng, "q4_0", rows, 64, 32, False, True) for _ in range(2)]
    index = eng.add_matrix("q4_0", rows, 64, mats[0][0], up=mats[1][0])
    xs = torch.from_numpy(rng.integers(-1, 2, (n, 64)).astype(np.float64)) / 16
    for scale in (0.375, -2.0):
        yd, buf = ref.wide_rows(torch.from_numpy(rng.standard_normal((n, rows))), ref.DTYPES[yt], pad=1, shift=1, fill=2.0)
        held = yd.cpu().double()
        eng.linear(index, xs.bfloat16().cuda(), yd, accumulate=accumulate, scale=scale, stream=stream())
        want, tol = gated(xs @ mats[0][1].T, xs @ mats[1][1].T, scale)
        if accumulate:
            want = want + held
            tol = tol + ULP * want.abs()
        tol = tol + half_step(ref.DTYPES[yt]) * (want.abs() + tol) + 2.0 ** -25 * (yt == "f16")
        assert ((yd.cpu().double() - want).abs() <= tol).all()
        assert ref.untouched(buf, yd, 2.0)
    eng.release_matrix(index)


@pytest.mark.parametrize("act", ["none", "silu", "sigmoid"])
@pytest.mark.parametrize("yt", ["bf16", "f16"])
def test_few_token_epilogue_in_16_bits(eng, yt, act):
    """The few-token kernel's sum with 16-bit outputs, rows apart and at odd addresses."""
    print(f"few-token epilogue {yt} {act}", flush=True)
    rng = np.random.default_rng(3)
    data, W, _, _ = ref.random_matrix(rng, "q4_1", 131, 96, 32, True, True)
    index = eng.add_matrix("q4_1", 131, 96, data)
    xs = torch.from_numpy(rng.integers(-3, 4, (3, 96)).astype(np.float64))
    yd, buf = ref.wide_rows(torch.from_numpy(rng.standard_normal((3, 131))), ref.DTYPES[yt], pad=2, shift=1, fill=2.0)
    held = yd.cpu().double()
    eng.linear(index, xs.float().cuda(), yd, act=act, accumulate=True, scale=0.03125, stream=stream())
    z = 0.03125 * (xs @ W.T)
    part = {"none": z, "silu": ref.silu(z), "sigmoid": torch.sigmoid(z)}[act]
    want = part + held
    tol = 8 * ULP * (part.abs() + want.abs() + 1e-20)
    assert ((yd.cpu().double() - want).abs() <= tol + half_step(ref.DTYPES[yt]) * (want.abs() + tol) + 2.0 ** -25 * (yt == "f16")).all()
    assert ref.untouched(buf, yd, 2.0)
    eng.release_matrix(index)


@pytest.mark.parametrize("n,rows", [(4, 64), (50, 20000)])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("size", [1e-31, 1e-34, 1e-36])
def test_smallest_activations(eng, size, mins, n, rows):
    """Of an fp32 activation below 2^-103 what is below 2^-126 counts as zero, and no more: 2^-126 sum |W| beside the roundings of
    (76 + groups) 2^-23 of 55 |s| sum |x| + |m| sum |x|; the minimum and the 16 that go through other sums may keep it, 2^-126
    of the sum of both at most."""
    rng = np.random.default_rng(9)
    data, W, s, m = ref.random_matrix(rng, "q4", rows, 256, 64, mins, True)
    index = eng.add_matrix("q4", rows, 256, data, group=64)
    x = torch.from_numpy(rng.standard_normal((n, 256)) * size).float()
    yd = torch.zeros(n, rows, device="cuda")
    eng.linear(index, x.cuda(), yd, stream=stream())
    x = x.double()
    bound = (76 + 4) * 2 * ULP * (x.abs() @ (55 * s + m).T) + 2.0 ** -126 * (16 * s + m + W.abs()).sum(1)
    assert ((yd.cpu().double() - x @ W.T).abs() <= bound).all()
    eng.release_matrix(index)
