"""The operators between a served model's MoE layers and its answers, as measurable cases.

  linear    a batch of tokens through a 4-bit matrix with group scales, or through a gated pair of them
            (Engine.add_matrix once, Engine.linear per call): a dense feed-forward's halves, the output head
  norm      the step between two blocks: the block's output normalised, gated, scaled and added to the residual
            stream, and the next block's normalised input from it (Engine.block_norm)
  logprobs  rows of logits to the log probabilities of given tokens, the entropy and the top alternatives
            (Engine.logprobs)

Each runs between device tensors on the current stream. `own` false computes the same with elementary torch
operations in 32 bits. Hidden sizes 2048 and 2560, feed-forward widths 512 and 1024 and batches 1, 8, 37, 64, 777, 1023
and 4096 are this repository's own; vocabularies are generic, one of them odd.
"""
import sys
import weakref
from pathlib import Path

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

LINEAR = dict(op="linear", fmt="q4_0", group=32, mins=False, gated=False, x="f32", y="f32", pad=0)
NORM = dict(op="norm", h="f32", stream="f32", next="f32", gate="none", gate_type="f32", sigmoid=False, post=True, pad=0)
LOGPROBS = dict(op="logprobs", x="f32", given=1, top=0, banned=False, scale=1.0, pad=0)


def listed():
    return [
        # One token through a shared expert's down projection: the smallest product a decode step makes.
        dict(LINEAR, name="linear_token", rows=2048, cols=512, n=1),
        # Three sequences' tokens through a feed-forward's first half, rows with minima.
        dict(LINEAR, name="linear_gated_3", rows=1024, cols=2048, n=3, fmt="q4_1", mins=True, gated=True),
        # The output head for one generated token.
        dict(LINEAR, name="linear_head_1", rows=131072, cols=2048, n=1),
        # The output head of an odd vocabulary for an odd batch of sequences, scales shared by 128 values, the
        # tokens' rows a slice of wider ones.
        dict(LINEAR, name="linear_head_37", rows=100003, cols=2560, n=37, fmt="q4", group=128, x="bf16", pad=8),
        # A prompt through a dense feed-forward's first half.
        dict(LINEAR, name="linear_gated_1023", rows=4096, cols=2048, n=1023, fmt="q4", group=64, mins=True, gated=True,
             x="f16", y="f16"),
        # The step between two blocks of one token's decode.
        dict(NORM, name="norm_token", n=1, E=2048),
        # A batch whose block output a gate per token weighs.
        dict(NORM, name="norm_gate_64", n=64, E=2560, h="bf16", next="bf16", gate="token", sigmoid=True),
        # A prompt chunk, everything but the stream in 16 bits, a learned gate per channel.
        dict(NORM, name="norm_prompt_4096", n=4096, E=2048, h="bf16", next="bf16", gate="channel"),
        # Odd rows with a gate of their own for every value, all in binary16.
        dict(NORM, name="norm_odd_777", n=777, E=2047, h="f16", stream="f16", next="f16", gate="value",
             gate_type="f16", sigmoid=True, pad=3),
        # A generated token's log probability with the twenty alternatives that an answer may list.
        dict(LOGPROBS, name="logprobs_token", n=1, V=131072, top=20),
        # A batch at a temperature, with banned tokens, over an odd vocabulary in 16 bits.
        dict(LOGPROBS, name="logprobs_64", n=64, V=100003, x="bf16", top=5, banned=True, scale=1.25),
        # A prompt scored token by token.
        dict(LOGPROBS, name="logprobs_prompt_1023", n=1023, V=131072, top=1),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))

    op = rng.choice(["linear", "linear", "norm", "logprobs"])
    if op == "linear":
        fmt = rng.choice(["q4_0", "q4_1", "q4", "q4"])
        group = rng.choice([32, 64, 128]) if fmt == "q4" else 32
        c = dict(LINEAR, fmt=fmt, group=group, mins=fmt == "q4_1" or (fmt == "q4" and rng.random() < 0.5),
                 gated=rng.random() < 0.4, x=rng.choice(["f32", "bf16", "f16"]), y=rng.choice(["f32", "f32", "bf16", "f16"]),
                 pad=rng.choice([0, 0, 1, 8]))
        c["cols"] = group * max(1, log_int(256, 8192) // group)
        c["rows"] = log_int(64, min(131072, 2 ** 28 // c["cols"])) // (2 if c["gated"] else 1)
        c["n"] = log_int(1, min(1023, max(1, 2 ** 34 // (c["rows"] * c["cols"] * (2 if c["gated"] else 1)))))
        return c
    if op == "norm":
        t = rng.choice(["f32", "bf16", "f16"])
        return dict(NORM, n=log_int(1, 4096), E=log_int(64, 8192) if rng.random() < 0.5 else 8 * log_int(8, 512),
                    h=t, stream=rng.choice(["f32", t]), next=t, gate=rng.choice(["none", "token", "channel", "value"]),
                    gate_type=rng.choice(["f32", t]), sigmoid=rng.random() < 0.5, post=rng.random() < 0.8,
                    pad=rng.choice([0, 0, 5, 8]))
    V = log_int(2000, 131072)
    return dict(LOGPROBS, V=V, n=log_int(1, min(1023, 2 ** 27 // V)), x=rng.choice(["f32", "bf16", "f16"]),
                given=rng.choice([1, 1, 1, 3]), top=rng.choice([0, 1, 5, 20, 50]), banned=rng.random() < 0.3,
                scale=rng.choice([1.0, 1.0, 0.7, 1.6]), pad=rng.choice([0, 0, 1, 64]))


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


def _quantised(c, seed, stream):
    """N(0, 0.02) weights in the case's 4-bit format: the GGUF rows, or (quants, scales, mins or None)."""
    rows, cols, group = c["rows"], c["cols"], c["group"]
    w = _normal((rows, cols // group, group), seed, stream, 0.02)
    if c["mins"]:
        lo, hi = w.amin(-1, keepdim=True), w.amax(-1, keepdim=True)
        s = ((hi - lo) / 15).half()
        m = lo.half()
        q = ((w - m.float()) / s.float().clamp_min(1e-7)).round_().clamp_(0, 15).to(torch.uint8)
    else:  # the value of largest magnitude takes q = 0
        far = w.gather(-1, w.abs().argmax(-1, keepdim=True))
        s, m = (far / -8).half(), None
        q = (w / torch.where(s == 0, 1e-7, s.float())).round_().add_(8).clamp_(0, 15).to(torch.uint8)
    if c["fmt"] == "q4":  # value 2 i in the low bits of byte i
        q = q.view(rows, cols // 2, 2)
        return (q[..., 0] | (q[..., 1] << 4)).contiguous(), s.view(rows, -1), None if m is None else m.view(rows, -1)
    packed = q[..., :16] | (q[..., 16:] << 4)  # value i in the low bits of byte i, value 16 + i in its high bits
    head = [s.view(torch.uint8)] + ([m.view(torch.uint8)] if c["mins"] else [])
    return torch.cat(head + [packed], -1).reshape(rows, -1).contiguous()


def _linear_inputs(c, seed):
    w = [_quantised(c, seed, 1)] + ([_quantised(c, seed, 2)] if c["gated"] else [])
    x = _normal((c["n"], c["cols"]), seed, 3)
    x[:, ::97] *= 8  # a few channels of a model's activations are much larger than the rest
    return w, _rows(x, c["x"], c["pad"])


def _norm_inputs(c, seed):
    n, E = c["n"], c["E"]
    d = dict(h=_rows(_normal((n, E), seed, 1, 0.3), c["h"], c["pad"]),
             x=_rows(_normal((n, E), seed, 2, 2.0), c["stream"], c["pad"]),
             pre=1 + _normal((E,), seed, 3, 0.1), post=1 + _normal((E,), seed, 4, 0.1) if c["post"] else None)
    shape = {"none": None, "token": (n, 1), "channel": (1, E), "value": (n, E)}[c["gate"]]
    d["gate"] = None if shape is None else _normal(shape, seed, 5).to(DTYPE[c["gate_type"]])
    return d


def _logprobs_inputs(c, seed):
    x = _normal((c["n"], c["V"]), seed, 1, 2.5)
    at = torch.randint(0, c["V"], (c["n"], 16), device="cuda", generator=_gen(seed, 2))
    x.scatter_add_(1, at, 6 + _normal((c["n"], 16), seed, 3, 3.0))  # a few tokens that the model deems likely
    if c["banned"]:
        x[:, ::11] = float("-inf")
    other = torch.randint(0, c["V"], (c["n"], c["given"]), device="cuda", generator=_gen(seed, 4))
    likely = torch.rand((c["n"], c["given"]), device="cuda", generator=_gen(seed, 5)) < 0.7
    tokens = torch.where(likely, at[:, :c["given"]], other)
    return _rows(x, c["x"], c["pad"]), tokens


# ---- the engine, once per process ----------------------------------------------------------------

_engines = []


def _engine():
    if not _engines:
        sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "gyro-dx_amd"))
        from gyrodx.engine import Engine
        _engines.append(Engine(max_tok=8))
    return _engines[0]


class _Matrix:
    """A matrix of the engine, released with the state that holds it."""

    def __init__(self, c, w):
        host = [tuple(None if t is None else t.cpu().numpy() for t in m) if c["fmt"] == "q4" else m.cpu().numpy() for m in w]
        eng = _engine()
        self.index = eng.add_matrix(c["fmt"], c["rows"], c["cols"], host[0], up=host[1] if c["gated"] else None, group=c["group"])
        weakref.finalize(self, eng.release_matrix, self.index)


def prepare(case, seed):
    c = case
    s = dict(case=dict(c))
    if c["op"] == "linear":
        w, x = _linear_inputs(c, seed)
        s.update(w=w, x=x, y=torch.empty(c["n"], c["rows"], device="cuda", dtype=DTYPE[c["y"]]))
        if own:
            s["matrix"] = _Matrix(c, w)
    elif c["op"] == "norm":
        s.update(_norm_inputs(c, seed))
        s.update(out=torch.empty(c["n"], c["E"], device="cuda", dtype=DTYPE[c["stream"]]),
                 next=torch.empty(c["n"], c["E"], device="cuda", dtype=DTYPE[c["next"]]))
    else:
        x, tokens = _logprobs_inputs(c, seed)
        n, k = c["n"], c["top"]
        s.update(x=x, tokens=tokens, logprob=torch.empty(n, c["given"], device="cuda"), entropy=torch.empty(n, device="cuda"),
                 ids=torch.empty(n, k, device="cuda", dtype=torch.int32), top=torch.empty(n, k, device="cuda"))
        if own:
            s["workspace"] = torch.empty(_engine().logprobs_workspace(n, c["V"], k), device="cuda", dtype=torch.uint8)
    return s


# ---- one pass --------------------------------------------------------------------------------------

EPS = 1e-6


def _run_own(s):
    c, eng = s["case"], _engine()
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "linear":
        eng.linear(s["matrix"].index, s["x"], s["y"], stream=stream)
        return s["y"]
    if c["op"] == "norm":
        eng.block_norm(s["h"], s["x"], s["out"], s["next"], post=c["post"], post_weight=s["post"], post_eps=EPS,
                       gate=s["gate"], gate_act="sigmoid" if c["sigmoid"] else "none", scale=0.5, pre_weight=s["pre"],
                       pre_eps=EPS, stream=stream)
        return s["out"], s["next"]
    eng.logprobs(s["x"], s["workspace"], tokens=s["tokens"], logprob=s["logprob"], entropy=s["entropy"],
                 top_ids=s["ids"] if c["top"] else None, top_logprobs=s["top"] if c["top"] else None, scale=c["scale"],
                 stream=stream)
    return (s["logprob"], s["entropy"], s["ids"], s["top"]) if c["top"] else (s["logprob"], s["entropy"])


def _weights(c, raw):
    rows, cols, group = c["rows"], c["cols"], c["group"]
    if c["fmt"] == "q4":
        quants, s, m = raw
        q = torch.stack([quants & 15, quants >> 4], -1).view(rows, cols // group, group).float()
    else:
        blocks = raw.view(rows, cols // 32, -1)
        head = 4 if c["mins"] else 2
        half = blocks[..., :head].contiguous().view(torch.float16)
        s, m = half[..., 0], half[..., 1] if c["mins"] else None
        q = torch.cat([blocks[..., head:] & 15, blocks[..., head:] >> 4], -1).float()
    q = q - 8 if m is None else q
    q = q * s.float().unsqueeze(-1)
    if m is not None:
        q = q + m.float().unsqueeze(-1)
    return q.view(rows, cols)


def _plain_linear(c, s):
    x = s["x"].float()
    y = x @ _weights(c, s["w"][0]).T
    if c["gated"]:
        y = y / (1 + torch.exp(-y)) * (x @ _weights(c, s["w"][1]).T)
    return y.to(DTYPE[c["y"]])


def _plain_norm(c, s):
    a = s["h"].float()
    if c["post"]:
        a = a / torch.sqrt((a * a).mean(-1, keepdim=True) + EPS) * s["post"]
    if s["gate"] is not None:
        g = s["gate"].float()
        a = a * (1 / (1 + torch.exp(-g)) if c["sigmoid"] else g)
    v = s["x"].float() + 0.5 * a
    z = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["pre"]
    return v.to(DTYPE[c["stream"]]), z.to(DTYPE[c["next"]])


def _plain_logprobs(c, s):
    z = s["x"].float() * c["scale"]
    d = z - z.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1)
    logs = torch.log(total)
    logprob = d.gather(1, s["tokens"]) - logs[:, None]
    entropy = logs - torch.where(e > 0, e * d, 0.0).sum(-1) / total
    if not c["top"]:
        return logprob, entropy
    # By the logits themselves, which the scale's rounding cannot make equal; equal ones: the lower id first.
    ids = torch.sort(s["x"].float(), dim=-1, descending=True, stable=True).indices[:, :c["top"]]
    return logprob, entropy, ids.to(torch.int32), d.gather(1, ids) - logs[:, None]


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    return {"linear": _plain_linear, "norm": _plain_norm, "logprobs": _plain_logprobs}[c["op"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "linear":
        halves = 2 if c["gated"] else 1
        weights = c["rows"] * c["cols"] * halves
        scales = weights // c["group"] * (4 if c["mins"] else 2)
        ends = c["n"] * (c["cols"] * BYTES[c["x"]] + c["rows"] * BYTES[c["y"]])
        return {"bytes": weights // 2 + scales + ends, "flops": 2 * c["n"] * weights}
    if c["op"] == "norm":
        n, E = c["n"], c["E"]
        gate = {"none": 0, "token": n, "channel": E, "value": n * E}[c["gate"]] * BYTES[c["gate_type"]]
        weights = 4 * E * (2 if c["post"] else 1)
        return {"bytes": n * E * (BYTES[c["h"]] + 2 * BYTES[c["stream"]] + BYTES[c["next"]]) + gate + weights,
                "flops": 12 * n * E}
    return {"bytes": c["n"] * (c["V"] * BYTES[c["x"]] + c["given"] * 12 + 4 + 8 * c["top"]), "flops": 6 * c["n"] * c["V"]}


# ---- the same in 64 bits --------------------------------------------------------------------------

def _nibbles64(packed):
    """Low and high four bits of every byte, as float64 [..., 2]."""
    table = torch.tensor([[b % 16, b // 16] for b in range(256)], dtype=torch.float64, device=packed.device)
    return table[packed.long()]


def _product64(c, raw, x):
    """x W^T from the definition W = s q + m, a slab of rows at a time."""
    group, out = c["group"], []
    for r in range(0, c["rows"], 16384):
        end = min(c["rows"], r + 16384)
        if c["fmt"] == "q4":
            q = _nibbles64(raw[0][r:end]).reshape(end - r, -1, group)
            s = raw[1][r:end].double()
            m = -8 * s if raw[2] is None else raw[2][r:end].double()
        else:
            block = raw[r:end].reshape(end - r, -1, 20 if c["mins"] else 18)
            s = block[..., 0:2].contiguous().view(torch.float16).double()[..., 0]
            m = block[..., 2:4].contiguous().view(torch.float16).double()[..., 0] if c["mins"] else -8 * s
            q = _nibbles64(block[..., -16:]).transpose(-1, -2).reshape(end - r, -1, group)
        w = q.mul_(s[..., None]).add_(m[..., None]).reshape(end - r, c["cols"])
        out.append(torch.mm(x, w.T.contiguous()))
    return torch.cat(out, 1)


def exact(case, seed):
    c = case
    if c["op"] == "linear":
        w, x = _linear_inputs(c, seed)
        x = x.double().contiguous()
        y = _product64(c, w[0], x)
        return y * torch.sigmoid(y) * _product64(c, w[1], x) if c["gated"] else y
    if c["op"] == "norm":
        d = {k: None if t is None else t.double() for k, t in _norm_inputs(c, seed).items()}
        a = d["h"]
        if c["post"]:
            a = a * d["post"] * (a.square().sum(-1, keepdim=True) / c["E"] + EPS).rsqrt()
        if d["gate"] is not None:
            a = a * (torch.sigmoid(d["gate"]) if c["sigmoid"] else d["gate"])
        v = torch.add(d["x"], a, alpha=0.5)
        return v, v * d["pre"] * (v.square().sum(-1, keepdim=True) / c["E"] + EPS).rsqrt()
    x, tokens = _logprobs_inputs(c, seed)
    logprob, entropy, ids, top = [], [], [], []
    for r in range(c["n"]):
        z = x[r].double() * c["scale"]
        lse = torch.logsumexp(z, 0)
        p = torch.exp(z - lse)
        logprob.append(z[tokens[r]] - lse)
        entropy.append(lse - (p * z.clamp_min(-1e300)).sum())
        if c["top"]:
            # The top values by magnitude, then among equals the lower id: a key of (value, -id).
            few = (z >= torch.topk(z, c["top"]).values[-1]).nonzero()[:, 0]
            best = few[torch.sort(-z[few], stable=True).indices[:c["top"]]]
            ids.append(best)
            top.append(z[best] - lse)
    if not c["top"]:
        return torch.stack(logprob), torch.stack(entropy)
    return torch.stack(logprob), torch.stack(entropy), torch.stack(ids).to(torch.int32), torch.stack(top)
