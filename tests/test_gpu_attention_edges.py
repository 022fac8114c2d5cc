"""Attention where its arithmetic and its bounds end, against 64-bit forms."""
import math
from fractions import Fraction

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import Batch, eng, reach, stream  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu
HALF = ref.half_step(torch.float16)


def test_more_tokens_than_the_bound(eng):  # noqa: F811
    """Of a sequence of more than `longest` tokens the first `longest` are computed, and all of the others' that keep to it; with
    more tiles of rows than a group finds by itself, and with fewer."""
    for sequences, longest, counts in ((1100, 1, {40: 4000}), (1100, 3, {0: 3000, 7: 500}), (700, 2, {699: 5000}), (30, 40, {3: 900})):
        print(f"{sequences} sequences, longest {longest}, {counts}", flush=True)
        of = [counts.get(b, 1 + b % longest) for b in range(sequences)]
        b = Batch(eng, "bf16", 32, 1, 16, 16, of, [n + 20 for n in of], seed=41)
        b.out.fill_(7.0)
        eng.attention(b.q, b.kc, b.vc, b.table, b.lengths, b.out, b.ws, starts=b.starts, longest=longest, stream=stream())
        torch.cuda.synchronize()
        first = torch.cat([b.starts[i] + torch.arange(min(n, longest), device="cuda") for i, n in enumerate(of)])
        # A token by itself: its sequence's keys up to its own.
        at = torch.cat([21 + torch.arange(min(n, longest)) for n in of])
        of_token = torch.cat([torch.full((min(n, longest),), i) for i, n in enumerate(of)]).cuda()
        want, bound, _ = ref.attention(b.q[first], b.kc, b.vc, b.table[of_token], at, [1] * len(at), 32, 0.25, True, 0)
        got = b.out[first].cpu().double()
        assert ((got - want).abs() <= bound + ref.half_step(torch.bfloat16) * (want.abs() + bound)).all()
        assert (b.out[b.n:] == 7).all()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sign,ones", [(-1, 64), (1, 64), (-1, 57), (1, 57)])
def test_scores_of_any_size(eng, type, sign, ones):  # noqa: F811
    """Finite scores count, whatever their size: the largest, which several keys share to the last bit, and no other. Weights are
    one and zero then: the result is the mean of the values, off by the sum's roundings and its own."""
    for counts, lengths in (([1, 3], [700, 90]), ([1], [9000]), ([150], [400]), ([18], [6000])):
        for scale in (2.0 ** 105, 1.1e32, 1e20, 3e9, 2.0 ** 26, 5e4):
            b = Batch(eng, type, 4, 2, 64, 16, counts, lengths, seed=42)
            g = torch.Generator().manual_seed(43)
            size = 2.0 ** torch.randint(0, 3, b.kc.shape[:3], generator=g)  # a key's values: 1, 2 or 4
            b.kc.copy_(sign * size[..., None].expand_as(b.kc))
            b.q.zero_()
            for head in range(4):
                b.q[:, 64 * head:64 * head + ones] = 1
            b.out.fill_(7.0)
            print(f"scores of {sign * ones} {scale:.1e} {type} {counts} {lengths}", flush=True)
            b.run(scale=scale)
            torch.cuda.synchronize()
            table, vc, row = b.table.cpu().long(), b.vc.cpu().double(), 0
            for s, (count, length) in enumerate(zip(counts, lengths)):
                j = torch.arange(length)
                page = table[s, j // 16]
                keys, v = size[page, :, j % 16] * sign, vc[page, :, j % 16]  # [length, kv], [length, kv, dim]
                for i in range(count):
                    seen = length - count + i + 1
                    for head in range(4):
                        k, x = keys[:seen, head // 2], v[:seen, head // 2]
                        top = x[k == k.max()]
                        want, room = top.mean(0), top.abs().mean(0) * (len(top) / 4 + 130) * ref.ULP
                        got = b.out[row, head * 64:(head + 1) * 64].cpu().double()
                        least = 2.0 ** -25 if type == "f16" else 0
                        assert ((got - want).abs() <= room + ref.half_step(b.dtype) * (want.abs() + room) + least).all(), (s, i, head)
                    row += 1


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [0, 70])
def test_scores_of_any_size_side_by_side(eng, type, window):  # noqa: F811
    """Rows whose scores are of every size, in one tile: the ordinary ones lose nothing by the others, of which the first
    begin with small scores and grow, and none is NaN."""
    for counts, lengths in (([5, 3], [700, 90]), ([2], [9000]), ([150, 40], [400, 300]), ([18], [6000])):
        b = Batch(eng, type, 4, 2, 64, 16, counts, lengths, seed=49)
        b.q[0::3] *= 200
        b.q[1::9] *= 60
        b.kc[:, :, 5::8] *= 100
        for scale in (0.125, 300.0):
            b.out.fill_(7.0)
            print(f"side by side {type} {counts} {lengths} {scale}", flush=True)
            b.run(scale=scale, window=window)
            b.check(scale=scale, window=window, norm=False)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("counts,lengths", [([1, 2], [4000, 300]), ([40], [4000])], ids=["few", "many"])
@pytest.mark.parametrize("below", [13, 17, 19, 21])
def test_small_weights(eng, below, counts, lengths):  # noqa: F811
    """Binary16 rows behind one key that takes nearly all weight and whose value is zero: the others' weights, e^-below of it, are
    all that there is. A weight is rounded by half a step of the type or by 2^-36 of the largest (by 2^-25,
    where the largest is 2^11 or more), whichever is more."""
    b = Batch(eng, "f16", 4, 2, 64, 16, counts, lengths, seed=44)
    b.q.fill_(1)
    b.kc.zero_()
    b.vc.add_(4).mul_(500)
    for s in range(len(counts)):
        b.kc[int(b.table[s, 0]), :, 3] = below / 8  # 64 / 8 of it, in nats
        b.vc[int(b.table[s, 0]), :, 3] = 0
    b.out.fill_(7.0)
    print(f"weights {below} below, {counts}", flush=True)
    b.run()
    torch.cuda.synchronize()
    want, bound, _ = ref.attention(b.q, b.kc, b.vc, b.table, b.lengths, counts, 4, 0.125, True, 0)
    rounded = want.abs() * 2.0 ** -36 * math.exp(below)
    err = (b.out[:b.n].cpu().double() - want).abs()
    limit = bound + rounded + HALF * (want.abs() + bound + rounded) + 2.0 ** -25
    print(f"  err / want {float((err / want.abs()).max()):.2e}, limit {float((limit / want.abs()).max()):.2e}", flush=True)
    assert (err <= limit).all()


@pytest.mark.parametrize("type", ["bf16", "f16"])
def test_whole_weight_beside_infinity(eng, type):  # noqa: F811
    """A key with one value that is not finite gives its others the whole weight, as rows of few tokens give every key's."""
    heads, dim = 64, 64
    b = Batch(eng, type, heads, heads, dim, 16, [1], [9], seed=45)
    b.q.fill_(1)
    b.kc.zero_()
    page = int(b.table[0, 0])
    b.kc[page, :, 2] = torch.linspace(-0.4, -0.01, heads)[:, None].to(b.kc)  # one key a little below the eight others
    b.vc.zero_()
    b.vc[page, :, 2] = 1 + 2.0 ** -6
    b.vc[page, :, 2, 5] = float("inf")
    b.run()
    torch.cuda.synchronize()
    k = b.kc[page, :, 2, 0].cpu().double()
    w = torch.exp(8 * k) / (8 + torch.exp(8 * k))
    got = b.out[0].cpu().double().reshape(heads, dim)
    assert torch.isinf(got[:, 5]).all()
    got = got[:, [d for d in range(dim) if d != 5]]
    want = (w * (1 + 2.0 ** -6))[:, None]
    # Two parts of a weight hold 16 bits or more; scores and sums as in attention_reference.
    room = want * (2.0 ** -16 + (2 * (2 * dim + 6) * 3.2 + 140) * ref.ULP)
    err = (got - want).abs()
    print(f"  {type}: err / half a step {float((err / (ref.half_step(b.dtype) * want)).max()):.3f}", flush=True)
    assert (err <= room + ref.half_step(b.dtype) * (want + room)).all()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("by", [1, 2], ids=["one", "two"])
@pytest.mark.parametrize("counts,lengths", [([1, 3], [700, 90]), ([150, 20], [400, 90]), ([18], [5000])], ids=["few", "many", "split"])
@pytest.mark.parametrize("dim", [64, 136])
def test_caches_aligned_to_their_type(eng, type, by, counts, lengths, dim):  # noqa: F811
    """k, v and every stride off 16 bytes by one value, or by two; values that are not finite among them."""
    b = Batch(eng, type, 8, 2, dim, 16, counts, lengths, pad=by, shift=by, seed=46)
    pages = b.kc.shape[0]
    token = dim + by
    head = 16 * token + by
    page = 2 * head + by
    for name, shift in (("kc", by), ("vc", 3 * by)):
        flat = torch.full((pages * page + 16,), float("nan"), dtype=b.dtype, device="cuda")
        cache = flat.as_strided((pages, 2, 16, dim), (page, head, token, 1), shift)
        cache.copy_(getattr(b, name))
        setattr(b, name, cache)
    for kw in (dict(), dict(window=50), dict(causal=False)):
        print(f"aligned to {by} {type} {counts} {dim} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)
    for s, length in enumerate(lengths):
        at = lambda j: (int(b.table[s, j // 16]), slice(None), j % 16)  # noqa: E731
        b.vc[at(length // 2)][0, dim - 1] = float("inf")
        b.vc[at(length - 1)][1, 0] = float("nan")
        b.kc[at(length - 1)][0, dim - 1] = float("nan")
    b.out.fill_(7.0)
    b.run()
    b.check()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("by", [1, 2], ids=["one", "two"])
@pytest.mark.parametrize("counts", [[3, 1], [40, 1]], ids=["few", "many"])
def test_wide_caches_aligned_to_their_type(eng, by, counts):  # noqa: F811
    """The same in caches that 32 bits do not span."""
    size, dim, kv, pages = 16, 128, 2, 7
    stride = (1 << 29) + 4096 + by
    b = Batch(eng, "bf16", 4, kv, dim, size, counts, [75, 30], seed=47, spare=0)
    flat = torch.zeros(stride * pages, dtype=torch.bfloat16, device="cuda")
    for name, shift in (("kc", by), ("vc", size * kv * (dim + by) + 3 * by)):
        cache = flat.as_strided((pages, kv, size, dim), (stride, size * (dim + by), dim + by, 1), shift)
        cache.copy_(getattr(b, name))
        setattr(b, name, cache)
    b.vc[int(b.table[0, 2]), 1, 3, 5] = float("nan")
    for kw in (dict(), dict(window=20), dict(causal=False)):
        print(f"wide cache aligned to {by} {counts} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)


def test_rotary_of_many_turns(eng):  # noqa: F811
    """Angles of frequencies that are many turns a position, far out."""
    f = [1.0, 100.0, 12345.678, 1e6, 1e9, 2.0 ** 31 - 1, -3e8, 6.283185307179586]
    index = eng.add_rotary(f)
    positions = torch.cat([(1 << 36) - torch.arange(1, 33), torch.arange(4)]).cuda()
    x = torch.randn(len(positions), 16, generator=torch.Generator().manual_seed(48)).cuda()
    y = torch.empty_like(x)
    eng.rotary(index, x, positions, y, heads=1, stream=stream())
    torch.cuda.synchronize()
    eng.release_rotary(index)
    turn = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    angle = [[float(Fraction(v) * int(p) / turn % 1) * 2 * math.pi for v in f] for p in positions]
    c, s = torch.tensor(angle, dtype=torch.float64).cos(), torch.tensor(angle, dtype=torch.float64).sin()
    a, b = x[:, :8].cpu().double(), x[:, 8:].cpu().double()
    want, size = torch.cat([a * c - b * s, a * s + b * c], 1), (a.abs() + b.abs()).repeat(1, 2)
    # As in attention_reference, and 2^-29 of a turn (2 pi 2^-29 in a sine or cosine) for the position times the table's rounding.
    bound = ref.rotary_bound(want, size, torch.float32) + 2 * math.pi * 2.0 ** -29 * size
    assert ((y.cpu().double() - want).abs() <= bound).all()
