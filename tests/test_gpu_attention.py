"""Rotary positions, the paged cache's appending and attention on the GPU against plain forms in 64 bits: types, layouts, one
token to hundreds, odd sizes, strides and alignments, pages that end inside a tile, tokens that a mask leaves nothing, NaNs and
infinities in masked places, pages and slots outside the cache, captured graphs, two streams, offsets past 32 bits.

Tolerances are derived in attention_reference.py. Beyond those bounds, the error of random rows as a whole is that of their
roundings: the softmax's weights and the result round once each, either by at most half a step and both ways alike, so the
errors' norm stays below half a step (of 1 / sqrt(3) of it at most each) of the result's."""
import numpy as np
import pytest
import torch

import attention_reference as ref
import op_reference
from gyrodx.engine import Engine
from gyrodx.rotary import frequencies

pytestmark = pytest.mark.gpu
DTYPES = ref.DTYPES


@pytest.fixture(scope="module")
def eng():
    e = Engine(max_tok=8)
    e.load_operators()
    yield e
    e.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- rotary positions ------------------------------------------------------------------------------

def positions_of(g, n, kind):
    far = torch.randint(0, 1 << 20, (n,), generator=g)
    if kind == "wide":  # negative ones and ones of 36 bits among them
        far[::3] = -torch.randint(0, 1 << 36, far[::3].shape, generator=g)
    return far if kind == "wide" else far.int()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "bf16")])
def test_rotary(eng, layout, x, y):
    for n, H, D, R, pad, shift in ((1, 1, 2, 2, 0, 0), (1, 32, 128, 128, 0, 0), (5, 3, 80, 20, 2, 1), (3, 7, 57, 40, 5, 3), (64, 8, 64, 6, 8, 0),
                                   (257, 40, 128, 64, 0, 0), (2, 1, 1024, 1024, 0, 0), (7, 2, 33, 2, 1, 1), (33, 5, 96, 94, 0, 8)):
        print(f"rotary {layout} {x} -> {y}: {n} tokens, {H} heads of {D}, {R} turned", flush=True)
        g = torch.Generator().manual_seed(n + D)
        f, scale = frequencies(R, base=5e5, scaling="bands", factor=8.0)
        index = eng.add_rotary(f, layout=layout, scale=scale)
        xd, _ = op_reference.wide_rows(torch.randn(n, H * D, generator=g) * 3, DTYPES[x], pad=pad, shift=shift)
        p = positions_of(g, n, "wide" if n != 5 else "near").cuda()
        yd, buf = op_reference.wide_rows(torch.zeros(n, H * D), DTYPES[y], pad=pad, shift=shift, fill=7.0)
        eng.rotary(index, xd, p, yd, heads=H, stream=stream())
        torch.cuda.synchronize()
        want, size = ref.rotary(xd, H, p, f, layout, np.float32(scale).astype(np.float64))
        err = (yd.cpu().double() - want).abs()
        assert (err <= ref.rotary_bound(want, size, DTYPES[y])).all(), float(err.max())
        assert op_reference.untouched(buf, yd, 7.0)
        if x == y:  # in place
            eng.rotary(index, xd, p, xd, heads=H, stream=stream())
            torch.cuda.synchronize()
            assert torch.equal(xd, yd)
        eng.release_rotary(index)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_rotary_parts(eng, layout, type):
    """Heads whose pairs, or what is behind them, are no whole eights; in place and apart alike."""
    for n, H, D, R in ((3, 3, 20, 16), (6, 5, 24, 18), (2, 64, 8, 2), (9, 4, 72, 36), (40, 9, 200, 198), (1, 3, 9, 8), (5, 2, 1023, 1022),
                       (70, 30, 250, 90), (2, 600, 120, 58), (11, 1, 16, 14),
                       (30, 2, 64, 14), (2051, 2, 64, 2), (2050, 5, 72, 36), (3001, 1, 128, 128), (2100, 16, 128, 64), (2100, 17, 128, 64)):
        print(f"rotary parts {layout} {type}: {n} tokens, {H} heads of {D}, {R} turned", flush=True)
        g = torch.Generator().manual_seed(n * D)
        f, _ = frequencies(R)
        index = eng.add_rotary(f, layout=layout)
        x, _ = op_reference.wide_rows(torch.randn(n, H * D, generator=g), DTYPES[type], pad=1, shift=1)
        p = positions_of(g, n, "near").cuda()
        y, buf = op_reference.wide_rows(torch.zeros(n, H * D), DTYPES[type], pad=3, fill=7.0)
        eng.rotary(index, x, p, y, heads=H, stream=stream())
        torch.cuda.synchronize()
        want, size = ref.rotary(x, H, p, f, layout, 1.0)
        assert ((y.cpu().double() - want).abs() <= ref.rotary_bound(want, size, DTYPES[type])).all()
        assert op_reference.untouched(buf, y, 7.0)
        eng.rotary(index, x, p, x, heads=H, stream=stream())
        torch.cuda.synchronize()
        assert torch.equal(x, y)
        eng.release_rotary(index)


def test_rotary_far(eng):
    """Neighbouring positions far out turn by their distance: fp32 angles would not tell them apart."""
    f, _ = frequencies(64)
    index = eng.add_rotary(f)
    p = (1 << 36) - torch.arange(1, 33, device="cuda")
    x = torch.zeros(32, 64, device="cuda")
    x[:, :32] = 1
    y = torch.empty_like(x)
    eng.rotary(index, x, p, y, heads=1)
    torch.cuda.synchronize()
    want, size = ref.rotary(x, 1, p, f, "half", 1.0)
    assert ((y.cpu().double() - want).abs() <= ref.rotary_bound(want, size, torch.float32)).all()
    assert (y[1:, :4] - y[:-1, :4]).abs().amax(0).min() > 0.1
    eng.release_rotary(index)


# ---- appending -----------------------------------------------------------------------------------

@pytest.mark.parametrize("order", ["head", "token"])
@pytest.mark.parametrize("x,cache,wide", [("f32", "bf16", True), ("bf16", "bf16", False), ("f16", "f32", True), ("f32", "f16", False), ("f32", "f32", True)])
@pytest.mark.parametrize("layout", ["half", "interleaved", None])
def test_append(eng, order, x, cache, wide, layout):
    for n, H, KVH, D, R, size, pad in ((1, 8, 2, 128, 128, 16, 0), (1, 0, 1, 64, 64, 1, 0), (37, 6, 3, 80, 20, 8, 2), (64, 0, 8, 128, 64, 100, 0),
                                       (300, 20, 4, 57, 18, 32, 3), (33, 4, 2, 1024, 512, 7, 8)):
        print(f"append {order} {x} -> {cache}, {layout}: {n} tokens, {H} and {KVH} heads of {D}, {R} turned, pages of {size}", flush=True)
        g = torch.Generator().manual_seed(n + D)
        pages = -(-n // size) + 3
        kc, vc = ref.make_cache(pages, KVH, size, D, DTYPES[cache], order, seed=n)
        before = kc.clone(), vc.clone()
        rows = lambda heads: op_reference.wide_rows(torch.randn(n, heads * D, generator=g), DTYPES[x], pad=pad, shift=pad % 2)[0]  # noqa: E731
        k, v, q = rows(KVH), rows(KVH), rows(H) if H else None
        q_out, buf = op_reference.wide_rows(torch.zeros(n, H * D), DTYPES[cache], pad=1, fill=3.0) if H else (None, None)
        slots = torch.randperm(pages * size, generator=g)[:n]
        slots[::5] = torch.tensor([-1, -(1 << 31), pages * size, (1 << 31) - 1])[torch.arange(len(slots[::5])) % 4]  # outside: skipped
        if wide and n > 10:
            slots[5], slots[10] = 1 << 40, -(1 << 62)
        slots = slots if wide else slots.int()
        positions = positions_of(g, n, "wide" if wide else "near")
        f, scale = frequencies(R, scaling="linear", factor=3.0)
        index = eng.add_rotary(f, layout=layout or "half", scale=0.75) if layout else None
        eng.cache_append(k, v, kc, vc, slots.cuda(), rotary=index, positions=positions.cuda() if layout else None, q=q, q_out=q_out,
                         stream=stream())
        torch.cuda.synchronize()

        def turned(rows, heads):
            if layout is None:
                return rows.cpu().double(), torch.zeros(n, heads * D, dtype=torch.float64)
            return ref.rotary(rows, heads, positions, f, layout, 0.75)

        wk, size_k = turned(k, KVH)
        bound_k = ref.rotary_bound(wk, size_k, DTYPES[cache])
        kept = [(t, int(s) // size, int(s) % size) for t, s in enumerate(slots) if 0 <= int(s) < pages * size]
        assert kept and len(kept) < n or n == 1
        for t, page, at in kept:
            got = kc[page, :, at].reshape(-1).cpu().double()
            assert ((got - wk[t]).abs() <= bound_k[t]).all()
            assert torch.equal(vc[page, :, at].reshape(-1), v[t].to(DTYPES[cache]))
            for c, b in zip((kc, vc), before):
                c[page, :, at] = b[page, :, at]
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])  # nothing else was written
        if H:
            want, size_q = turned(q, H)
            assert ((q_out.cpu().double() - want).abs() <= ref.rotary_bound(want, size_q, DTYPES[cache])).all()
            assert op_reference.untouched(buf, q_out, 3.0)
            if x == cache:
                eng.cache_append(k, v, kc, vc, slots.cuda(), rotary=index, positions=positions.cuda() if layout else None, q=q, q_out=q)
                torch.cuda.synchronize()
                assert torch.equal(q, q_out)
        if index is not None:
            eng.release_rotary(index)


@pytest.mark.parametrize("n,H,KVH,D,R", [(2101, 0, 8, 128, 128), (2102, 2, 3, 80, 20), (4099, 1, 1, 256, 256), (2103, 12, 4, 64, 62)])
def test_append_many(eng, n, H, KVH, D, R):
    """More tokens than groups; of few heads and many."""
    print(f"append many {n} {H} {KVH} {D} {R}", flush=True)
    g = torch.Generator().manual_seed(n)
    kc, vc = (torch.zeros(n // 16 + 3, KVH, 16, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k, v, q = (torch.randn(n, heads * D, generator=g).bfloat16().cuda() for heads in (KVH, KVH, H))
    slots = torch.randperm(kc.shape[0] * 16, generator=g)[:n]
    slots[::7] = -1
    p = positions_of(g, n, "near")
    f, _ = frequencies(R)
    index = eng.add_rotary(f)
    q_out = torch.zeros_like(q)
    eng.cache_append(k, v, kc, vc, slots.cuda(), rotary=index, positions=p.cuda(), q=q if H else None, q_out=q_out if H else None)
    torch.cuda.synchronize()
    kept = slots >= 0
    flat = lambda c: c.permute(0, 2, 1, 3).reshape(-1, KVH * D).cpu()  # noqa: E731
    want, size = ref.rotary(k, KVH, p, f, "half", 1.0)
    assert ((flat(kc)[slots[kept]].double() - want[kept]).abs() <= ref.rotary_bound(want, size, torch.bfloat16)[kept]).all()
    assert torch.equal(flat(vc)[slots[kept]], v.cpu()[kept])
    others = torch.ones(kc.shape[0] * 16, dtype=torch.bool)
    others[slots[kept]] = False
    assert (flat(kc)[others] == 0).all() and (flat(vc)[others] == 0).all()
    if H:
        want, size = ref.rotary(q, H, p, f, "half", 1.0)
        assert ((q_out.cpu().double() - want).abs() <= ref.rotary_bound(want, size, torch.bfloat16)).all()
    eng.release_rotary(index)


def test_append_no_tokens(eng):
    kc, vc = ref.make_cache(2, 1, 4, 8, torch.float32)
    empty = torch.zeros(0, 8, device="cuda")
    eng.cache_append(empty, empty, kc, vc, torch.zeros(0, dtype=torch.int64, device="cuda"))
    index = eng.add_rotary([1.0])
    eng.rotary(index, empty, torch.zeros(0, dtype=torch.int64, device="cuda"), empty, heads=1)
    eng.release_rotary(index)
    eng.attention(empty, kc, vc, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), empty)


# ---- attention -----------------------------------------------------------------------------------

class Batch:
    """Sequences of counts[b] tokens over lengths[b] cached ones, on pages in any order. The table spans `reach` keys at least:
    calls choose their kernels by that."""

    reach = 0

    def __init__(self, eng, dtype, heads, kv_heads, dim, size, counts, lengths, order="head", pad=0, shift=0, seed=0, spare=2, big=1.0):
        g = torch.Generator().manual_seed(seed + 17)
        self.eng, self.dtype, self.heads, self.counts = eng, DTYPES[dtype], heads, counts
        per = [-(-max(l, 0) // size) for l in lengths]
        width, pages = max(1, *per, -(-self.reach // size)) + 1, max(1, sum(per)) + spare
        self.kc, self.vc = ref.make_cache(pages, kv_heads, size, dim, self.dtype, order, seed=seed)
        self.kc *= big
        table = torch.randint(0, pages, (len(counts), width), generator=g, dtype=torch.int32)
        order = torch.randperm(pages, generator=g).int()
        at = 0
        for b, c in enumerate(per):
            table[b, :c] = order[at:at + c]
            at += c
        wide = torch.zeros(len(counts), width + 3, dtype=torch.int32)
        wide[:, :width] = table
        self.table = wide.cuda()[:, :width]
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.starts = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32, device="cuda")
        self.n = sum(counts)
        self.q, _ = op_reference.wide_rows(torch.randn(self.n + 3, heads * dim, generator=g) * 1.5, self.dtype, pad=pad, shift=shift)
        self.out, self.buf = op_reference.wide_rows(torch.zeros(self.n + 3, heads * dim), self.dtype, pad=pad, shift=shift, fill=7.0)
        self.out.fill_(7.0)
        self.ws = torch.full((eng.attention_workspace(heads, kv_heads, dim),), 255, dtype=torch.uint8, device="cuda")  # NaNs, and -1

    def run(self, ragged=True, out=None, **kw):
        rows = self.n + 3 if ragged else self.n
        self.eng.attention(self.q[:rows], self.kc, self.vc, self.table, self.lengths, (self.out if out is None else out)[:rows], self.ws,
                           starts=self.starts if ragged else None, longest=max(1, *self.counts) if ragged else None, stream=stream(), **kw)

    def check(self, scale=None, causal=True, window=0, norm=True):
        torch.cuda.synchronize()
        dim = self.kc.shape[3]
        want, bound, sees = ref.attention(self.q, self.kc, self.vc, self.table, self.lengths, self.counts, self.heads,
                                          np.float64(np.float32(dim ** -0.5 if scale is None else scale)), causal, window)
        got = self.out[:self.n].cpu().double()
        half = ref.half_step(self.dtype)
        finite = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
        err = torch.where(finite, got - want, 0.0).abs()
        limit = bound + half * (want.abs() + bound) + (2.0 ** -24 if self.dtype == torch.float16 else 0)
        print(f"  err / bound {float((err / limit.clamp_min(1e-300))[finite].max()) if finite.any() else 0:.4f}, "
              f"rel rms {float(err.norm() / want[finite].norm().clamp_min(1e-300)):.2e}", flush=True)
        assert (err <= limit)[finite].all()
        none = ~sees[:, :, None].expand(-1, -1, dim).reshape(self.n, -1)
        assert (got[none] == 0).all()
        if norm and self.dtype != torch.float32 and finite.all():
            assert err.norm() <= half * want.norm() + 1e-12
        assert (self.out[self.n:] == 7).all()  # rows behind the last sequence
        assert op_reference.untouched(self.buf, self.out, 7.0)


@pytest.fixture(params=[0, 1 << 18], ids=["narrow", "wide"])
def reach(request):
    Batch.reach = request.param
    yield
    Batch.reach = 0


SHAPES = [  # heads, kv_heads, dim, page, counts, lengths
    (4, 4, 64, 16, [1], [1]),
    (8, 2, 128, 16, [1, 1, 1], [777, 31, 33]),
    (16, 2, 256, 64, [1], [2000]),
    (6, 2, 72, 7, [3, 1, 5], [40, 129, 5]),
    (24, 8, 96, 32, [2, 7], [300, 64]),
    (1, 1, 8, 1, [4], [70]),
    (5, 1, 80, 100, [33, 2], [333, 2]),
    (2, 1, 128, 16, [130], [130]),
    (4, 1, 200, 48, [70, 1], [513, 1025]),
    (16, 1, 64, 256, [40], [290]),
]


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("order", ["head", "token"])
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_attention(eng, shape, type, order):
    heads, kv, dim, size, counts, lengths = shape
    pad, shift = ((0, 0), (8, 0), (3, 1))[(dim // 8) % 3]
    b = Batch(eng, type, heads, kv, dim, size, counts, lengths, order, pad, shift, seed=dim)
    for kw in (dict(), dict(window=9), dict(window=100, scale=0.3), dict(causal=False)):
        print(f"attention {type} {order} {shape} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)
        if len(set(counts)) == 1:
            b.out.fill_(7.0)
            b.run(ragged=False, **kw)
            b.check(**kw)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
def test_attention_empty_rows(eng, type):
    """Sequences without tokens, without keys, with fewer keys than tokens, lengths below zero and past the table."""
    Batch.reach = min(Batch.reach, 1 << 13)
    b = Batch(eng, type, 4, 2, 64, 16, [3, 0, 5, 2, 1, 40], [0, 50, 2, 37, 90, 17], seed=3)
    b.lengths[3] = -4
    b.lengths[4] = 1 << 30
    for kw in (dict(), dict(causal=False), dict(window=1), dict(window=3)):
        print(f"empty rows {type} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("counts,lengths", [([6, 1, 20], [200, 97, 20]), ([150], [400])])
def test_attention_not_finite(eng, type, counts, lengths):
    """NaNs and infinities where nothing looks change nothing; where a token sees them, they show in its row and no other."""
    b = Batch(eng, type, 4, 2, 96, 16, counts, lengths, seed=5)
    for s, length in enumerate(lengths):  # behind each sequence's end, on the same page
        for j in range(length, -(-length // 16) * 16):
            page = int(b.table[s, j // 16])
            b.kc[page, :, j % 16] = float("nan")
            b.vc[page, :, j % 16] = float("inf") if j % 2 else float("nan")
    for kw in (dict(), dict(window=5), dict(causal=False)):
        print(f"not finite behind the end {type} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)
    # The last token's key and value, and a value in the middle of the new tokens: earlier tokens do not see them.
    for s, (count, length) in enumerate(zip(counts, lengths)):
        at = lambda j: (int(b.table[s, j // 16]), slice(None), j % 16)  # noqa: E731
        b.kc[at(length - 1)][0, 3] = float("nan")
        if count > 3:
            b.vc[at(length - 2)][1, 5] = float("inf")
            b.vc[at(length - 3)][0, 7] = float("nan")
            b.vc[at(length - count // 2)][1, 9] = float("-inf")
    for kw in (dict(), dict(window=2), dict(window=64), dict(causal=False)):
        print(f"not finite among the tokens {type} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)
    # Queries of one token; scores of -infinity.
    b.q[0] = float("nan")
    b.kc[int(b.table[0, 0]), 0, 0, :] = float("-inf")
    b.q[1].abs_()
    b.out.fill_(7.0)
    b.run()
    b.check()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_attention_only_minus_infinity(eng, type):
    """Scores of -infinity alone leave zeros, like no keys."""
    b = Batch(eng, type, 2, 1, 64, 16, [1, 3], [40, 3], seed=8)
    b.kc.fill_(float("-inf"))
    b.q.abs_()
    b.run()
    b.check()
    assert (b.out[:b.n] == 0).all()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("counts,lengths", [([1, 4], [300, 90]), ([100], [260])])
def test_attention_bad_pages(eng, type, counts, lengths):
    """Keys on pages outside the cache are not seen."""
    b = Batch(eng, type, 4, 1, 64, 16, counts, lengths, seed=9)
    pages = b.kc.shape[0]
    b.table[0, 1], b.table[0, 4], b.table[0, 7] = -1, pages, -(1 << 31)
    for kw in (dict(), dict(window=30), dict(causal=False)):
        print(f"bad pages {type} {counts} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)
    b.table.fill_(pages + 5)
    b.out.fill_(7.0)
    b.run()
    b.check()
    assert (b.out[:b.n] == 0).all()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16", "f32"])
def test_attention_large_scores(eng, type):
    """Scores of hundreds, whose weights fall to one key, rise late and fall again."""
    b = Batch(eng, type, 4, 2, 128, 32, [1, 9, 140], [900, 300, 200], seed=11, big=20.0)
    print(f"large scores {type}", flush=True)
    b.run(scale=1.0)
    b.check(scale=1.0, norm=False)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f32"])
def test_attention_in_place(eng, type):
    """out at q's rows; the same results as apart."""
    for counts, lengths in (([1, 1], [4000, 50]), ([5, 130], [600, 140])):
        b = Batch(eng, type, 8, 2, 64, 16, counts, lengths, seed=12)
        print(f"in place {type} {counts}", flush=True)
        b.run()
        want = b.out[:b.n].clone()
        b.run(out=b.q)
        torch.cuda.synchronize()
        assert torch.equal(b.q[:b.n], want)


def test_attention_long(eng):
    """One token over many parts, and the same token over the same keys in another table: bit for bit alike."""
    for type, size, length in (("bf16", 16, 30011), ("f16", 100, 9973), ("f32", 64, 5003)):
        print(f"long {type} {length}", flush=True)
        b = Batch(eng, type, 4, 1, 128, size, [1], [length], seed=13)
        b.run(ragged=False)
        b.check()
        first = b.out[:1].clone()
        again = [b.run(ragged=False) or b.out[:1].clone() for _ in range(3)]
        torch.cuda.synchronize()
        assert all(torch.equal(first, x) for x in again)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type,dim", [("bf16", 128), ("f16", 64), ("bf16", 256), ("f16", 200)])
def test_attention_split_tiles(eng, type, dim):
    """Rows of one or a few tiles whose keys many groups share, beside sequences of few rows; the same results every time."""
    for counts, lengths, kw in (([20], [9001], {}), ([50, 1, 5, 40], [4000, 5000, 77, 30], dict(window=1000)), ([70, 17], [1500, 3000], dict(causal=False))):
        print(f"split tiles {type} {dim} {counts} {kw}", flush=True)
        b = Batch(eng, type, 2, 1, dim, 16, counts, lengths, seed=16)
        b.run(**kw)
        b.check(**kw)
        first = b.out.clone()
        for _ in range(3):
            b.run(**kw)
        torch.cuda.synchronize()
        assert torch.equal(first, b.out)


@pytest.mark.parametrize("counts", [[700, 300, 20, 3, 40, 0, 130, 1, 90], [3, 200] * 20, [40] * 170 + [400]], ids=["mixed", "alternating", "even"])
def test_attention_many_split_tiles(eng, counts):
    """Split tiles among those that every wave of a group looks at, in every order; the same results every time."""
    rng = np.random.default_rng(63)
    lengths = [int(rng.integers(max(1, n), 3001)) for n in counts]
    print(f"many split tiles {counts[:4]}", flush=True)
    b = Batch(eng, "bf16", 5, 1, 16, 100, counts, lengths, seed=19)
    b.out.fill_(7.0)
    b.run()
    b.check()
    first = b.out.clone()
    for _ in range(5):
        b.out.fill_(7.0)
        b.run()
        torch.cuda.synchronize()
        assert torch.equal(first, b.out)


def test_attention_most_parts(eng):
    """One cache head's keys in as many parts as there are: of 16 rows, and of 128."""
    for type, counts, length in (("f16", [2], 140001), ("bf16", [17], 200003)):
        print(f"most parts {type} {counts} {length}", flush=True)
        b = Batch(eng, type, 1, 1, 16, 256, counts, [length], seed=18)
        b.run()
        b.check()


def test_attention_many_sequences(eng):
    """More sequences than the plan looks at in one go, of few rows, many, none."""
    rng = np.random.default_rng(61)
    counts = [int(c) for c in rng.choice([0, 1, 2, 9, 20, 40, 150], 1300, p=[0.1, 0.3, 0.2, 0.2, 0.1, 0.09, 0.01])]
    lengths = [c + int(rng.integers(0, 30)) for c in counts]
    b = Batch(eng, "bf16", 2, 1, 64, 16, counts, lengths, seed=17)
    print(f"{len(counts)} sequences, {b.n} tokens", flush=True)
    b.run()
    b.check()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f16"])
@pytest.mark.parametrize("counts", [[1, 1], [40, 1]])
def test_offsets_past_32_bits(eng, type, counts):
    """Pages that start more than 2^32 bytes into the cache, and appended tokens there."""
    size, dim, kv, pages = 16, 128, 2, 5
    dtype = DTYPES[type]
    stride = (1 << 30) + 4096  # values between pages
    k_all = torch.zeros(stride * pages, dtype=dtype, device="cuda")
    kc = k_all.as_strided((pages, kv, size, dim), (stride, size * dim, dim, 1))
    vc = k_all[size * kv * dim:].as_strided((pages, kv, size, dim), (stride, size * dim, dim, 1))
    b = Batch(eng, type, 4, kv, dim, size, counts, [60, 10], seed=14, spare=0)
    print(f"past 32 bits {type} {counts}", flush=True)
    kc.copy_(b.kc)
    vc.copy_(b.vc)
    b.kc, b.vc = kc, vc
    b.run()
    b.check()
    k, v = torch.randn(1, kv * dim, device="cuda").to(dtype), torch.randn(1, kv * dim, device="cuda").to(dtype)
    eng.cache_append(k, v, kc, vc, torch.tensor([4 * size + 3], device="cuda"))
    torch.cuda.synchronize()
    assert torch.equal(kc[4, :, 3].reshape(1, -1), k) and torch.equal(vc[4, :, 3].reshape(1, -1), v)
    b.run()
    b.check()


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("counts", [[40, 1], [3, 20]], ids=str)
def test_wide_cache_faults(eng, counts):
    """Pages outside the cache, and keys and values that are not finite, in a cache that 32 bits do not span."""
    size, dim, kv, pages = 16, 128, 2, 7
    stride = (1 << 29) + 4096
    k_all = torch.zeros(stride * pages, dtype=torch.bfloat16, device="cuda")
    kc = k_all.as_strided((pages, kv, size, dim), (stride, size * dim, dim, 1))
    vc = k_all[size * kv * dim:].as_strided((pages, kv, size, dim), (stride, size * dim, dim, 1))
    b = Batch(eng, "bf16", 4, kv, dim, size, counts, [75, 30], seed=25, spare=0)
    kc.copy_(b.kc)
    vc.copy_(b.vc)
    b.kc, b.vc = kc, vc
    b.table[0, 1] = pages
    vc[int(b.table[0, 2]), 1, 3, 5] = float("nan")
    vc[int(b.table[1, 1]), 0, 13, 100] = float("-inf")  # the last token's
    kc[int(b.table[1, 1]), 1, 13, 9] = float("nan")
    for kw in (dict(), dict(window=20), dict(causal=False)):
        print(f"wide cache {counts} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("dim", [8, 64, 136, 256])
@pytest.mark.parametrize("counts,lengths", [([150, 70], [400, 1300]), ([20, 2], [65, 64])])
def test_not_finite_in_tiles(eng, dim, counts, lengths):
    """Values that are not finite in tiles that all rows see whole, in split ones, and next to the mask's edge."""
    b = Batch(eng, "f16", 4, 2, dim, 48, counts, lengths, seed=26)
    for s, length in enumerate(lengths):
        at = lambda j: (int(b.table[s, j // 48]), slice(None), j % 48)  # noqa: E731
        b.vc[at(length // 3)][0, dim - 1] = float("inf")
        b.vc[at(length - counts[s])][1, 0] = float("nan")
        b.vc[at(length - 1)][1, dim // 2] = float("-inf")
    for kw in (dict(), dict(window=30), dict(causal=False)):
        print(f"not finite in tiles {dim} {counts} {kw}", flush=True)
        b.out.fill_(7.0)
        b.run(**kw)
        b.check(**kw)


@pytest.mark.usefixtures("reach")
@pytest.mark.parametrize("type", ["bf16", "f32"])
@pytest.mark.parametrize("group,counts", [(1, [16, 1, 15]), (1, [17, 16, 2]), (4, [4, 3]), (4, [5, 4]), (3, [43, 42]), (16, [8, 1]), (20, [1, 2])])
def test_attention_around_tiles(eng, type, group, counts):
    """Rows and keys around the sizes of tiles and around what a single launch takes."""
    for first in (63, 64, 65, 255, 257, 1023, 1025, 2049):
        lengths = [first] + [max(n, first // 2) for n in counts[1:]]
        print(f"around {type} {group} {counts} {lengths}", flush=True)
        b = Batch(eng, type, group, 1, 32, 64, counts, lengths, seed=first)
        b.run()
        b.check()


@pytest.mark.parametrize("sequences", [512, 1024, 1025])
def test_attention_entries(eng, sequences):
    """As many tiles of rows as a group finds by itself, and one more; sequences of few rows among them."""
    rng = np.random.default_rng(67)
    counts = [int(n) for n in rng.choice([0, 1, 2, 9, 33], sequences)]
    lengths = [int(rng.integers(max(1, n), 200)) for n in counts]
    b = Batch(eng, "bf16", 2, 1, 16, 16, counts, lengths, seed=27)
    print(f"entries {sequences}", flush=True)
    b.run()
    b.check()


def test_graphs_of_tiles(eng):
    """Captured calls of split tiles and of a list of units, one workspace; lengths change between replays."""
    batches = [Batch(eng, "bf16", 8, 2, 64, 16, [90, 1, 20], [3000, 2000, 100], seed=28),
               Batch(eng, "bf16", 8, 2, 64, 16, [18] * 520 + [0] * 520, [40] * 520 + [9] * 520, seed=29)]
    batches[1].ws = batches[0].ws
    graphs = []
    for b in batches:
        b.run()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            b.run()
    for turn in range(3):
        print(f"turn {turn}", flush=True)
        for b, g in zip(batches, graphs):
            b.out.fill_(7.0)
            b.q.mul_(-1)
            b.lengths.sub_(turn)
            g.replay()
        for b in batches:
            b.check()


# ---- together -------------------------------------------------------------------------------------

class Decoder:
    """A block's attention half as a served model has it: the norm, the 4-bit product to queries, keys and values, the cache,
    the attention, the 4-bit product back and the residual step; every call on the current stream."""

    H, KVH, D, E, SIZE, WIDTH, S = 8, 2, 64, 256, 16, 6, 3

    def __init__(self, eng):
        rng = np.random.default_rng(51)
        self.eng, H, KVH, D, E = eng, self.H, self.KVH, self.D, self.E
        self.width = (H + 2 * KVH) * D
        data, self.W, _, _ = op_reference.random_matrix(rng, "q4_0", self.width, E, 32, False)
        self.qkv = eng.add_matrix("q4_0", self.width, E, data)
        data, self.O, _, _ = op_reference.random_matrix(rng, "q4_0", E, H * D, 32, False)
        self.back = eng.add_matrix("q4_0", E, H * D, data)
        self.f, _ = frequencies(D)
        self.rotary = eng.add_rotary(self.f)
        dev = dict(device="cuda")
        pages = self.S * self.WIDTH
        self.kc, self.vc = (torch.zeros(pages, KVH, self.SIZE, D, dtype=torch.bfloat16, **dev) for _ in range(2))
        self.table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().view(self.S, self.WIDTH).cuda()
        self.ws = torch.empty(eng.attention_workspace(H, KVH, D), dtype=torch.uint8, **dev)

    def buffers(self, n):
        z = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda", dtype=t)  # noqa: E731
        return dict(x=z(n, self.E), normed=z(n, self.E), rows=z(n, self.width), q=z(n, self.H * self.D, t=torch.bfloat16),
                    a=z(n, self.H * self.D, t=torch.bfloat16), h=z(n, self.E), out=z(n, self.E), slots=z(n, t=torch.int64),
                    positions=z(n, t=torch.int32), lengths=z(self.S, t=torch.int32), starts=z(self.S + 1, t=torch.int32))

    def set(self, d, firsts, counts, seed):
        """Tokens firsts[b] .. firsts[b] + counts[b] - 1 of each sequence."""
        at = torch.cat([torch.arange(f, f + c) for f, c in zip(firsts, counts)])
        seq = torch.cat([torch.full((c,), b) for b, c in enumerate(counts)])
        d["x"].copy_(torch.randn(len(at), self.E, generator=torch.Generator().manual_seed(seed)))
        d["positions"].copy_(at)
        d["slots"].copy_(self.table.cpu()[seq, at // self.SIZE].long() * self.SIZE + at % self.SIZE)
        d["lengths"].copy_(torch.tensor([f + c for f, c in zip(firsts, counts)]))
        d["starts"].copy_(torch.tensor([0, *np.cumsum(counts)]))

    def run(self, d, longest=None):
        e, s, hd, kd = self.eng, stream(), self.H * self.D, self.KVH * self.D
        e.block_norm(None, d["x"], None, d["normed"], stream=s)
        e.linear(self.qkv, d["normed"], d["rows"], stream=s)
        e.cache_append(d["rows"][:, hd:hd + kd], d["rows"][:, hd + kd:], self.kc, self.vc, d["slots"], rotary=self.rotary,
                       positions=d["positions"], q=d["rows"][:, :hd], q_out=d["q"], stream=s)
        e.attention(d["q"], self.kc, self.vc, self.table, d["lengths"], d["a"], self.ws, starts=d["starts"] if longest else None,
                    longest=longest, stream=s)
        e.linear(self.back, d["a"], d["h"], stream=s)
        e.block_norm(d["h"], d["x"], d["out"], None, stream=s)

    def check(self, d, counts):
        """Each operator against 64 bits on what it was given."""
        torch.cuda.synchronize()
        c, hd, kd = (lambda t: t.cpu().double()), self.H * self.D, self.KVH * self.D
        rows = c(d["normed"]) @ self.W.T
        assert (c(d["rows"]) - rows).norm() <= 1e-5 * rows.norm()
        want, size = ref.rotary(d["rows"][:, :hd], self.H, d["positions"], self.f, "half", 1.0)
        assert ((c(d["q"]) - want).abs() <= ref.rotary_bound(want, size, torch.bfloat16)).all()
        want, size = ref.rotary(d["rows"][:, hd:hd + kd], self.KVH, d["positions"], self.f, "half", 1.0)
        slots = d["slots"].cpu()
        got = c(self.kc)[slots // self.SIZE, :, slots % self.SIZE].reshape(len(slots), -1)
        assert ((got - want).abs() <= ref.rotary_bound(want, size, torch.bfloat16)).all()
        got = self.vc[slots // self.SIZE, :, slots % self.SIZE].reshape(len(slots), -1)
        assert torch.equal(got, d["rows"][:, hd + kd:].bfloat16())
        want, bound, _ = ref.attention(d["q"], self.kc, self.vc, self.table, d["lengths"], counts, self.H, self.D ** -0.5, True, 0)
        assert ((c(d["a"]) - want).abs() <= bound + ref.half_step(torch.bfloat16) * (want.abs() + bound)).all()
        h = c(d["a"]) @ self.O.T
        assert (c(d["h"]) - h).norm() <= 1e-5 * h.norm()
        assert torch.equal(d["out"], d["x"] + d["h"])


def test_decoder(eng):
    """Prompts, then a token a step, eager on a side stream and replayed from a graph, each step checked and both alike."""
    m, side = Decoder(eng), torch.cuda.Stream()
    counts = [33, 1, 20]
    prompt, step = m.buffers(sum(counts)), m.buffers(m.S)
    m.set(prompt, [0, 0, 0], counts, 1)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        m.run(prompt, longest=33)
    side.synchronize()
    m.check(prompt, counts)
    print("prompts done", flush=True)
    at = list(counts)
    for turn in range(3):
        m.set(step, at, [1] * m.S, 10 + turn)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            m.run(step)
        side.synchronize()
        m.check(step, [1] * m.S)
        at = [v + 1 for v in at]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m.run(step)
    for turn in range(5):
        print(f"replay {turn}", flush=True)
        m.set(step, at, [1] * m.S, 20 + turn)
        graph.replay()
        m.check(step, [1] * m.S)
        replayed = [t.clone() for t in (step["q"], step["a"], step["out"], m.kc, m.vc)]
        m.run(step)  # the same token again, eagerly
        m.check(step, [1] * m.S)
        assert all(torch.equal(x, y) for x, y in zip(replayed, (step["q"], step["a"], step["out"], m.kc, m.vc)))
        at = [v + 1 for v in at]
    del graph
    eng.release_matrix(m.qkv)
    eng.release_matrix(m.back)
    eng.release_rotary(m.rotary)


def test_two_streams(eng):
    """Calls on two streams at once, a workspace each."""
    batches = [Batch(eng, "bf16", 8, 2, 128, 16, [1, 1, 1], [5000, 3000, 70], seed=21),
               Batch(eng, "bf16", 8, 2, 128, 16, [300, 1, 40], [5000, 3000, 70], seed=22)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(4):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                b.run()
    torch.cuda.synchronize()
    for b in batches:
        b.check()


def test_two_graphs_share_a_workspace(eng):
    """Graphs whose replays follow one another may share one."""
    batches = [Batch(eng, "bf16", 8, 2, 128, 16, [1, 1], [5000, 300], seed=s) for s in (23, 24)]
    batches[1].ws = batches[0].ws
    graphs = []
    for b in batches:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            b.run()
    for turn in range(3):
        for b, g in zip(batches, graphs):
            b.out.fill_(7.0)
            b.q.mul_(-1)
            g.replay()
        for b in batches:
            b.check()
        print(f"turn {turn}", flush=True)


def test_capture_needs_loaded_kernels():
    """A capture refuses a kernel that is not loaded, and the engine goes on."""
    e = Engine(max_tok=8)
    try:
        b = Batch(e, "f16", 4, 1, 64, 16, [1], [40], seed=31)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="not loaded"):
            with torch.cuda.graph(graph):
                b.run()
        b.run()
        b.check()
    finally:
        e.close()
