"""What a served model does between a block's QKV product and its output product, as measurable cases.

  rotary   rows of heads turned by their positions (Engine.add_rotary once, Engine.rotary per call)
  append   new tokens' keys and values into the pages of a cache, the keys (and the queries beside them) turned on the way
           (Engine.cache_append)
  attend   the new tokens' attention over the paged cache: single tokens, drafts, chunks of prompts, ragged batches, and,
           without the causal mask, an encoder's states (Engine.attention)

Each runs between device tensors on the current stream. `own` false computes the same with elementary torch operations, in
32 bits and the angles in 64. Hidden sizes 2048, 2560 and 4096, batches 1, 8, 64, 777, 1023 and 4096 are this
repository's own or multiples of it; head sizes and counts, pages and lengths are generic.
"""
import math
import random
import sys
import weakref
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# rot: values of a head that turn. scaling: of the frequencies, for contexts `factor` times the one trained on.
ROTARY = dict(op="rotary", D=128, rot=128, layout="half", scaling="none", factor=1.0, base=10000.0, far=8192, x="bf16",
              y="bf16", pad=0)
# H: queries' heads turned in the same call (0: none). each: tokens of a sequence. skip: padded tokens among them.
APPEND = dict(ROTARY, op="append", H=0, KVH=8, page=16, each=1, cache="bf16", order="head", skip=False)
# tokens, kv: the longest sequence's new tokens and its cached ones, the new among them; ragged: the others' are shorter.
ATTEND = dict(op="attend", seqs=1, ragged=False, H=32, KVH=8, D=128, page=16, type="bf16", causal=True, window=0, order="head",
              pad=0)


def listed():
    return [
        # One token's queries, as the product gave them, on their way to attention in 16 bits.
        dict(ROTARY, name="rotary_token", n=1, H=32, x="f32"),
        # A prompt's chunk, half of every head turned, neighbours paired, for a context 16 times the one trained on.
        dict(ROTARY, name="rotary_chunk_1023", n=1023, H=40, rot=64, layout="interleaved", scaling="bands", factor=16.0,
             far=131072),
        # What a decode step of one sequence does before its attention.
        dict(APPEND, name="append_token", n=1, H=32, x="f32"),
        # A batch of sequences, some places of it empty, odd heads a quarter of which turns, a cache in token order.
        dict(APPEND, name="append_batch_64", n=64, H=20, KVH=4, D=80, rot=20, x="f32", y="f16", cache="f16", order="token",
             skip=True, far=131072, scaling="linear", factor=8.0),
        # A whole prompt's keys and values.
        dict(APPEND, name="append_prompt_4096", n=4096, each=4096, H=32),
        # One token of a short conversation: latency.
        dict(ATTEND, name="attend_token", tokens=1, kv=777, H=16, KVH=2),
        # A batch of decoding sequences of very different lengths.
        dict(ATTEND, name="attend_batch_64", seqs=64, tokens=1, kv=8192, ragged=True),
        # One token at the end of a long document, large heads.
        dict(ATTEND, name="attend_long_131072", tokens=1, kv=131072, H=16, KVH=2, D=256, page=64),
        # Drafted tokens of eight sequences being checked, within a window, three queries' heads to one of the cache's.
        dict(ATTEND, name="attend_drafts_8", seqs=8, tokens=5, kv=4100, H=24, KVH=8, D=96, page=64, type="f16", window=1024,
             order="token"),
        # A whole prompt.
        dict(ATTEND, name="attend_prompt_4096", tokens=4096, kv=4096),
        # A serving step's mix: chunks of prompts and single tokens over contexts of all lengths, pages of an odd size.
        dict(ATTEND, name="attend_mixed_1023", seqs=9, tokens=1023, kv=16384, ragged=True, H=20, KVH=4, page=100, pad=64),
        # A decoder's tokens over an encoder's states, in 32 bits.
        dict(ATTEND, name="attend_states_1500", seqs=3, tokens=37, kv=1500, H=16, KVH=16, D=64, type="f32", causal=False, page=50),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))

    def rotary(D):
        scaling = rng.choice(["none", "linear", "base", "bands"])
        return dict(D=D, rot=D if rng.random() < 0.5 else 2 * rng.randint(1, D // 2), layout=rng.choice(["half", "interleaved"]),
                    scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0, 40.0]),
                    base=rng.choice([10000.0, 500000.0, 1e6]), far=log_int(64, 1 << 20), x=rng.choice(["f32", "bf16", "f16"]),
                    y=rng.choice(["f32", "bf16", "f16"]), pad=rng.choice([0, 0, 2, 8]))

    op = rng.choice(["rotary", "append", "attend", "attend"])
    D = rng.choice([64, 128, 8 * rng.randint(2, 32)])
    if op == "rotary":
        H = log_int(1, 64)
        return dict(ROTARY, **rotary(D), H=H, n=log_int(1, min(8192, (1 << 24) // (H * D))))
    if op == "append":
        KVH = rng.choice([1, 2, 3, 4, 8, 16])
        H = KVH * rng.choice([0, 1, 3, 4, 8])
        n = log_int(1, min(4096, (1 << 24) // ((H + 2 * KVH) * D)))
        each = n if rng.random() < 0.5 else rng.choice([d for d in range(1, min(n, 64) + 1) if n % d == 0])
        return dict(APPEND, **rotary(D), H=H, KVH=KVH, n=n, each=each, page=rng.choice([1, 8, 16, 32, 100, 256]),
                    cache=rng.choice(["f32", "bf16", "f16"]), order=rng.choice(["head", "token"]), skip=rng.random() < 0.3)
    KVH = rng.choice([1, 2, 3, 4, 8])
    c = dict(ATTEND, KVH=KVH, H=KVH * rng.choice([1, 2, 3, 4, 5, 8, 16]), D=D, page=rng.choice([1, 8, 16, 32, 64, 100, 256]),
             type=rng.choice(["f32", "bf16", "bf16", "f16"]), ragged=rng.random() < 0.5, order=rng.choice(["head", "token"]),
             pad=rng.choice([0, 0, 8, 24]))
    kind = rng.choice(["token", "token", "drafts", "chunk", "chunk", "states"])
    most = (1 << 29) // (KVH * D * 2 * BYTES[c["type"]])  # cached tokens of all sequences
    c["seqs"] = log_int(1, 64 if kind in ("token", "drafts") else 8)
    c["kv"] = log_int(1, min(131072, most // c["seqs"]))
    pairs = min(1 << 29, (1 << 36) // (4 * D)) // (c["H"] * c["seqs"])  # scores of a head and sequence
    if c["type"] == "f32":
        pairs //= 4
    c["kv"] = max(1, min(c["kv"], pairs))
    limit = max(1, pairs // c["kv"])
    c["tokens"] = 1 if kind == "token" else log_int(1, min(8, limit)) if kind == "drafts" else log_int(1, min(4096, limit))
    if kind == "states":
        c["causal"] = False
    else:
        c["tokens"] = min(c["tokens"], c["kv"])
        c["window"] = log_int(16, 4096) if rng.random() < 0.25 else 0
    return c


# ---- inputs ------------------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1009 + stream)
    return g


def _normal(shape, seed, stream, scale=1.0):
    return torch.randn(shape, device="cuda", generator=_gen(seed, stream)) * scale


def _rows(values, dtype, pad):
    """`values` as rows of `dtype`, each `pad` elements further apart than it is long."""
    wide = torch.zeros(values.shape[0], values.shape[1] + pad, device="cuda", dtype=DTYPE[dtype])
    view = wide[:, :values.shape[1]]
    view.copy_(values)
    return view


def _heads(n, H, D, seed, stream, scale=1.0):
    """Rows of H heads, a few channels of each much larger than the rest."""
    x = _normal((n, H, D), seed, stream, scale)
    x[:, :, 3::29] *= 4
    return x.view(n, H * D)


def _paged(values, order):
    """Pages [pages, KVH, page, D] as the cache's owner lays them out: by heads, or by tokens."""
    return values if order == "head" else values.transpose(1, 2).contiguous().transpose(1, 2)


def _positions(c, seed):
    """Each sequence's tokens follow one another from somewhere in the context on."""
    each = c.get("each", c["n"])
    first = torch.randint(0, max(1, c["far"] - each), (c["n"] // each, 1), device="cuda", generator=_gen(seed, 11))
    return (first + torch.arange(each, device="cuda")).view(-1)


def _frequencies64(c):
    """The angle by which a position turns each pair, and what the turned values are scaled by, from the definitions."""
    R, s = c["rot"], c["factor"]
    base = c["base"] * s ** (R / (R - 2)) if c["scaling"] == "base" and R > 2 else c["base"]
    f = [base ** (-2.0 * j / R) for j in range(R // 2)]
    if c["scaling"] == "linear":
        f = [v / s for v in f]
    if c["scaling"] != "bands":
        return f, 1.0
    # Of a context of 4096: pairs that turn 32 times or more stay, those that turn once or less are slowed down by s.
    keep = [min(1.0, max(0.0, (4096 * v / (2 * math.pi) - 1) / 31)) for v in f]
    return [v * (k + (1 - k) / s) for v, k in zip(f, keep)], 0.1 * math.log(s) + 1


def _rotary_inputs(c, seed):
    return _rows(_heads(c["n"], c["H"], c["D"], seed, 1), c["x"], c["pad"]), _positions(c, seed)


def _append_inputs(c, seed):
    n, KVH, D, page, each = c["n"], c["KVH"], c["D"], c["page"], c["each"]
    d = dict(k=_rows(_heads(n, KVH, D, seed, 1), c["x"], c["pad"]), v=_rows(_heads(n, KVH, D, seed, 2), c["x"], c["pad"]),
             q=_rows(_heads(n, c["H"], D, seed, 3), c["x"], c["pad"]) if c["H"] else None, positions=_positions(c, seed))
    per = -(-each // page) + 1
    pages = n // each * per + 3
    for name, stream in (("k_cache", 4), ("v_cache", 5)):
        d[name] = _paged(_normal((pages, KVH, page, D), seed, stream).to(DTYPE[c["cache"]]), c["order"])
    # The pages of a sequence lie anywhere; its first new token anywhere in the first of them.
    table = torch.randperm(pages, device="cuda", generator=_gen(seed, 6))[:n // each * per].view(-1, per)
    at = torch.randint(0, page, (n // each, 1), device="cuda", generator=_gen(seed, 7)) + torch.arange(each, device="cuda")
    slots = table.gather(1, at // page) * page + at % page
    if c["skip"]:
        slots[torch.rand(slots.shape, device="cuda", generator=_gen(seed, 8)) < 0.2] = -1
    d["slots"] = slots.view(-1)
    return d


def _lengths(c):
    """(new tokens, cached tokens) of each sequence."""
    r = random.Random(f"{c['seqs']} {c['tokens']} {c['kv']}")
    q, kv = [c["tokens"]] * c["seqs"], [c["kv"]] * c["seqs"]
    if c["ragged"]:
        for i in range(1, c["seqs"]):
            q[i] = round(c["tokens"] ** r.random())
            kv[i] = round(c["kv"] ** r.uniform(0.5, 1.0))
            if c["causal"]:
                kv[i] = max(kv[i], q[i])
    return q, kv


def _attend_inputs(c, seed):
    q, kv = _lengths(c)
    n, S, KVH, D, page = sum(q), c["seqs"], c["KVH"], c["D"], c["page"]
    per = [-(-length // page) for length in kv]
    wide = max(per)
    pages = sum(per) + 2
    d = dict(q=_rows(_heads(n, c["H"], D, seed, 1, 1.5), c["type"], c["pad"]))
    for name, stream in (("k_cache", 2), ("v_cache", 3)):
        x = _normal((pages, KVH, page, D), seed, stream)
        x[..., 5::31] *= 3
        d[name] = _paged(x.to(DTYPE[c["type"]]), c["order"])
    # Pages anywhere in the pool; the table's places behind a sequence's last page name any page.
    order = torch.randperm(pages, device="cuda", generator=_gen(seed, 4)).to(torch.int32)
    table = torch.zeros(S, wide, device="cuda", dtype=torch.int32)
    at = 0
    for i, count in enumerate(per):
        table[i, :count] = order[at:at + count]
        at += count
    d["table"] = table
    d["lengths"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
    starts = [0]
    for length in q:
        starts.append(starts[-1] + length)
    d["starts"] = torch.tensor(starts, device="cuda", dtype=torch.int32)
    return d


# ---- the engine, once per process ----------------------------------------------------------------

_engines = []


def _engine():
    if not _engines:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gyro-dx_amd"))
        from gyrodx.engine import Engine
        _engines.append(Engine(max_tok=8))
    return _engines[0]


class _Rotary:
    """The engine's frequencies for a case, released with the state that holds them."""

    def __init__(self, c):
        from gyrodx.rotary import frequencies
        f, scale = frequencies(c["rot"], base=c["base"], scaling=c["scaling"], factor=c["factor"], context=4096)
        eng = _engine()
        self.index = eng.add_rotary(f, layout=c["layout"], scale=scale)
        weakref.finalize(self, eng.release_rotary, self.index)


def prepare(case, seed):
    c = case
    s = dict(case=dict(c))
    if c["op"] == "rotary":
        s["x"], s["positions"] = _rotary_inputs(c, seed)
        s["y"] = torch.empty(c["n"], c["H"] * c["D"], device="cuda", dtype=DTYPE[c["y"]])
    elif c["op"] == "append":
        s.update(_append_inputs(c, seed))
        s["y"] = torch.empty(c["n"], c["H"] * c["D"], device="cuda", dtype=DTYPE[c["y"]]) if c["H"] else None
    else:
        s.update(_attend_inputs(c, seed))
        s["out"] = torch.empty(s["q"].shape[0], c["H"] * c["D"], device="cuda", dtype=DTYPE[c["type"]])
    if own:
        eng = _engine()
        if c["op"] == "attend":
            s["workspace"] = torch.empty(eng.attention_workspace(c["H"], c["KVH"], c["D"]), device="cuda", dtype=torch.uint8)
        else:
            s["rotary"] = _Rotary(c)
    return s


# ---- one pass --------------------------------------------------------------------------------------

def _run_own(s):
    c, eng = s["case"], _engine()
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "rotary":
        eng.rotary(s["rotary"].index, s["x"], s["positions"], s["y"], heads=c["H"], stream=stream)
        return s["y"]
    if c["op"] == "append":
        eng.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], rotary=s["rotary"].index,
                         positions=s["positions"], q=s["q"], q_out=s["y"], stream=stream)
        return (s["k_cache"], s["v_cache"], s["y"]) if c["H"] else (s["k_cache"], s["v_cache"])
    same = not c["ragged"] or c["tokens"] == 1
    eng.attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"], s["workspace"],
                  starts=None if same else s["starts"], longest=None if same else c["tokens"], causal=c["causal"],
                  window=c["window"], stream=stream)
    return s["out"]


def _turned(c, x, H, positions):
    """Rows of H heads turned by their positions, in 32 bits; the angles in 64."""
    f, scale = _frequencies64(c)
    R, n = c["rot"], x.shape[0]
    x = x.float().reshape(n, H, c["D"])
    angle = positions.double()[:, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    cos, sin = (torch.cos(angle) * scale).float()[:, None], (torch.sin(angle) * scale).float()[:, None]
    turned = x[..., :R]
    if c["layout"] == "half":
        a, b = turned[..., :R // 2], turned[..., R // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(n, H, R)
    return torch.cat([turned, x[..., R:]], -1).reshape(n, H * c["D"])


def _plain_append(c, s):
    n, KVH, D = c["n"], c["KVH"], c["D"]
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    page, at = s["slots"][kept] // c["page"], s["slots"][kept] % c["page"]
    k = _turned(c, s["k"], KVH, s["positions"]).view(n, KVH, D)
    s["k_cache"][page, :, at] = k[kept].to(DTYPE[c["cache"]])
    s["v_cache"][page, :, at] = s["v"].reshape(n, KVH, D)[kept].to(DTYPE[c["cache"]])
    if not c["H"]:
        return s["k_cache"], s["v_cache"]
    return s["k_cache"], s["v_cache"], _turned(c, s["q"], c["H"], s["positions"]).to(DTYPE[c["y"]])


def _plain_attend(c, s):
    """All sequences side by side, padded to the longest."""
    S, H, KVH, D, T = c["seqs"], c["H"], c["KVH"], c["D"], c["tokens"]
    n, L, G = s["q"].shape[0], c["kv"], H // KVH
    lengths, starts = s["lengths"].long(), s["starts"].long()
    j, i = torch.arange(L, device="cuda"), torch.arange(T, device="cuda")
    page = s["table"].long()[:, j // c["page"]]
    k = s["k_cache"][page, :, j % c["page"]].float().permute(0, 2, 1, 3)  # S, KVH, L, D
    v = s["v_cache"][page, :, j % c["page"]].float().permute(0, 2, 1, 3)
    counts = starts[1:] - starts[:-1]
    rows = (starts[:-1, None] + i).clamp(max=n - 1)
    q = s["q"].float().reshape(n, KVH, G, D)[rows].permute(0, 2, 3, 1, 4).reshape(S, KVH, G * T, D)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(S, KVH, G, T, L)
    last = (lengths - counts)[:, None] + i if c["causal"] else (lengths - 1)[:, None].expand(S, T)
    seen = (j <= last[..., None]) & (j < lengths[:, None, None])
    if c["window"]:
        seen &= j > last[..., None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(S, KVH, G * T, L), v).view(S, KVH, G, T, D) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, T, H * D)
    return out[i < counts[:, None]].to(DTYPE[c["type"]])


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["op"] == "rotary":
        return _turned(c, state["x"], c["H"], state["positions"]).to(DTYPE[c["y"]])
    return _plain_append(c, state) if c["op"] == "append" else _plain_attend(c, state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "rotary":
        return {"bytes": c["n"] * (c["H"] * c["D"] * (BYTES[c["x"]] + BYTES[c["y"]]) + 8), "flops": 3 * c["n"] * c["H"] * c["rot"]}
    if c["op"] == "append":
        n, D = c["n"], c["D"]
        values = 2 * c["KVH"] * D * (BYTES[c["x"]] + BYTES[c["cache"]]) + c["H"] * D * (BYTES[c["x"]] + BYTES[c["y"]])
        return {"bytes": n * (values + 16), "flops": 3 * n * (c["H"] + c["KVH"]) * c["rot"]}
    keys, pairs, new = 0, 0, 0
    for q, kv in zip(*_lengths(c)):
        new += q
        if not c["causal"]:
            keys, pairs = keys + kv, pairs + q * kv
            continue
        w = c["window"] or kv
        keys += kv - max(0, kv - q + 1 - w)
        full = min(q, max(0, kv - w))  # the last tokens, which see a whole window
        pairs += full * w + sum(range(kv - q + 1, kv - full + 1))
    size = BYTES[c["type"]]
    return {"bytes": size * c["D"] * (2 * keys * c["KVH"] + 2 * new * c["H"]) + 4 * (keys // c["page"] + 2 * c["seqs"]),
            "flops": 4 * c["D"] * c["H"] * pairs}


# ---- the same in 64 bits --------------------------------------------------------------------------

def _turned64(c, x, H, positions):
    """Each pair as a complex number, times scale e^(i angle)."""
    f, scale = _frequencies64(c)
    R, n = c["rot"], x.shape[0]
    x = x.double().reshape(n, H, c["D"]).clone()
    angle = positions.double()[:, None, None] * torch.tensor(f, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.full_like(angle, scale), angle)
    first, second = (slice(0, R // 2), slice(R // 2, R)) if c["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x.reshape(n, H * c["D"])


def exact(case, seed):
    c = case
    if c["op"] == "rotary":
        x, positions = _rotary_inputs(c, seed)
        return _turned64(c, x, c["H"], positions)
    if c["op"] == "append":
        d = _append_inputs(c, seed)
        n, KVH, D = c["n"], c["KVH"], c["D"]
        out = []
        for rows, cache in ((_turned64(c, d["k"], KVH, d["positions"]), d["k_cache"]), (d["v"].double(), d["v_cache"])):
            pool = cache.double().transpose(1, 2).reshape(-1, KVH, D)  # slot by slot
            kept = d["slots"] >= 0
            pool[d["slots"][kept]] = rows.reshape(n, KVH, D)[kept]
            out.append(pool.view(-1, c["page"], KVH, D).transpose(1, 2).contiguous())
        return (*out, _turned64(c, d["q"], c["H"], d["positions"])) if c["H"] else tuple(out)
    d = _attend_inputs(c, seed)
    q, kv = _lengths(c)
    H, KVH, D = c["H"], c["KVH"], c["D"]
    out = torch.zeros(d["q"].shape[0], H, D, device="cuda", dtype=torch.float64)
    row = 0
    for b in range(c["seqs"]):
        used = d["table"][b, :-(-kv[b] // c["page"])].long()
        at = torch.arange(q[b], device="cuda")[:, None] + (kv[b] - q[b])
        j = torch.arange(kv[b], device="cuda")
        hidden = (j > at) | (j <= at - (c["window"] or kv[b] + 1)) if c["causal"] else torch.zeros_like(j > at)
        for g in range(KVH):
            k, v = (d[name][used, g].double().reshape(-1, D)[:kv[b]] for name in ("k_cache", "v_cache"))
            for h in range(g * (H // KVH), (g + 1) * (H // KVH)):
                z = d["q"][row:row + q[b], h * D:(h + 1) * D].double() @ k.t().contiguous() / math.sqrt(D)
                z[hidden] = -torch.inf
                out[row:row + q[b], h] = torch.nan_to_num(torch.softmax(z, -1)) @ v
        row += q[b]
    return out.view(-1, H * D)
