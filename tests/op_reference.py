"""Plain 64-bit forms of the operators around the MoE layers, and the inputs of their tests."""
import numpy as np
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    """The largest relative error of one rounding to dtype t."""
    return torch.finfo(t).eps / 2


def wide_rows(values, dtype, pad=0, shift=0, device="cuda", fill=0.0):
    """`values` as rows of dtype, `pad` values apart and `shift` values into a buffer of `fill`; (rows, buffer)."""
    n, cols = values.shape
    buf = torch.full((n * (cols + pad) + shift + 16,), fill, dtype=dtype, device=device)
    rows = buf[shift:shift + n * (cols + pad)].view(n, cols + pad)[:, :cols] if n else buf[:0].view(0, cols)
    rows.copy_(values)
    return rows, buf


def untouched(buf, rows, fill):
    """Whether everything of buf but the rows still holds `fill`."""
    left = buf.clone()
    at = (rows.data_ptr() - buf.data_ptr()) // buf.element_size()
    if rows.shape[0]:
        left.as_strided(rows.shape, rows.stride(), at).fill_(fill)
    return bool((left == fill).all())


# ---- 4-bit matrices ------------------------------------------------------------------------------

def random_matrix(rng, fmt, rows, cols, group, mins, exact=False):
    """(engine data, W in float64, |s| and |m| per value): scales powers of two and integer minima with `exact`."""
    G = cols // group
    q = rng.integers(0, 16, (rows, cols), dtype=np.uint8)
    if exact:
        s = (np.exp2(rng.integers(-2, 2, (rows, G))) * rng.choice([-1, 1], (rows, G))).astype(np.float16)
        m = rng.integers(-8, 9, (rows, G)).astype(np.float16)
    else:
        s = (rng.standard_normal((rows, G)) * 0.01).astype(np.float16)
        m = (rng.standard_normal((rows, G)) * 0.05).astype(np.float16)
    s64 = np.repeat(s.astype(np.float64), group, 1)
    m64 = np.repeat(m.astype(np.float64), group, 1) if mins else -8 * s64
    W = s64 * q + m64
    if fmt == "q4":
        data = (q[:, 0::2] | (q[:, 1::2] << 4), s, m if mins else None)
    else:
        b = q.reshape(rows, G, 32)
        parts = [s[..., None].view(np.uint8)] + ([m[..., None].view(np.uint8)] if mins else [])
        data = np.concatenate(parts + [b[..., :16] | (b[..., 16:] << 4)], -1).reshape(rows, -1)
    return data, torch.from_numpy(W), torch.from_numpy(np.abs(s64)), torch.from_numpy(np.abs(m64))


def silu(v):
    return v / (1 + torch.exp(-v))


# ---- the residual step -----------------------------------------------------------------------------

def block_norm(h, x, post, post_weight, post_eps, gate, gate_act, scale, pre_weight, pre_eps):
    """(v, normed, scale gate a) in 64 bits."""
    d = lambda t: None if t is None else t.double()  # noqa: E731
    v, part = d(x), torch.zeros_like(d(x))
    if h is not None:
        a = d(h)
        if post:
            a = a / torch.sqrt((a * a).mean(-1, keepdim=True) + post_eps)
            a = a * d(post_weight) if post_weight is not None else a
        if gate is not None:
            a = a * (torch.sigmoid(d(gate)) if gate_act == "sigmoid" else d(gate))
        part = scale * a
        v = v + part
    z = v / torch.sqrt((v * v).mean(-1, keepdim=True) + pre_eps)
    return v, z * d(pre_weight) if pre_weight is not None else z, part


# ---- log probabilities -----------------------------------------------------------------------------

def order(x):
    """Ids of each row by falling value, NaNs first, equal values by id."""
    x = torch.where(torch.isnan(x), float("inf"), x.double().clamp(-1e308, 1e308))
    return torch.sort(-x, dim=-1, stable=True).indices


def logprobs(x, tokens, scale):
    """(log p of the tokens, entropy, log p of everything, max, log S, T / S) in 64 bits."""
    z = x.double() * scale
    none = (z == -np.inf).all(-1, keepdim=True)
    m = torch.where(none, 0.0, z.amax(-1, keepdim=True))
    d = z - m
    e = torch.exp(d)
    S = e.sum(-1, keepdim=True)
    T = torch.where(e == 0, 0.0, e * d).sum(-1, keepdim=True)
    logs = torch.where(none, 0.0, torch.log(S))
    bad = torch.isnan(S) | (z == np.inf).any(-1, keepdim=True)
    lp = torch.where(bad, np.nan, torch.where(none, -np.inf, d - logs))
    H = torch.where(bad, np.nan, torch.where(none, 0.0, logs - T / torch.where(none, 1.0, S)))[:, 0]
    if tokens is None:
        return None, H, lp, m, logs, T / S
    inside = (tokens >= 0) & (tokens < x.shape[1])
    given = lp.gather(1, torch.where(inside, tokens, 0).long())
    given = torch.where(inside, given, torch.where(tokens < 0, 0.0, np.nan))
    return given, H, lp, m, logs, T / S


# Products for which a group of the few-token kernel takes a second run of rows: (rows, cols, fmt, group, mins, gated, x,
# tokens, whether its LDS holds all columns of the tokens).
SECOND_RUNS = [
    (66001, 256, "q4_0", 32, False, False, "f32", 1, True), (66001, 256, "q4", 64, True, False, "f32", 5, True),
    (100003, 384, "q4_1", 32, True, False, "bf16", 16, True), (66001, 256, "q4", 128, False, False, "f16", 8, True),
    (40009, 256, "q4_0", 32, False, True, "f32", 3, True), (40009, 256, "q4", 64, True, True, "bf16", 1, True),
    (132001, 96, "q4_0", 32, False, False, "f32", 1, True),
    (66001, 2304, "q4_0", 32, False, False, "bf16", 16, False), (66001, 2400, "q4_1", 32, True, False, "f32", 5, False),
    (33001, 2304, "q4", 128, True, True, "f16", 8, False)]


def repeated(data, times, rows):
    """A matrix's data (random_matrix) repeated and cut to `rows` rows."""
    cut = lambda a: None if a is None else np.tile(a, (times, 1))[:rows]  # noqa: E731
    return tuple(cut(a) for a in data) if isinstance(data, tuple) else cut(data)
