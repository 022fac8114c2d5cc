"""Plain 64-bit forms of rotary positions, the paged cache and attention, and the inputs of their tests."""
import numpy as np
import torch

from op_reference import DTYPES, half_step  # noqa: F401

ULP = 2.0 ** -24


def rotary(x, heads, positions, frequencies, layout, scale):
    """Rows of heads turned by their positions, in 64 bits; the angles in 80. (turned, what errors are relative to)"""
    n, R = x.shape[0], 2 * len(frequencies)
    x = x.double().cpu().reshape(n, heads, -1).clone()
    angle = positions.cpu().numpy().astype(np.longdouble)[:, None] * np.asarray(frequencies, np.longdouble)
    turns = angle / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    angle = ((turns - np.floor(turns)) * 2 * np.longdouble("3.14159265358979323846264338327950288")).astype(np.float64)
    c, s = (torch.from_numpy(scale * f(angle))[:, None] for f in (np.cos, np.sin))
    a, b = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    x1, x2 = x[..., a].clone(), x[..., b].clone()
    size = torch.zeros_like(x)
    size[..., a] = size[..., b] = abs(scale) * (x1.abs() + x2.abs())
    x[..., a], x[..., b] = x1 * c - x2 * s, x1 * s + x2 * c
    return x.reshape(n, -1), size.reshape(n, -1)


def rotary_bound(want, size, dtype):
    """A sine or cosine is within 8 units of fp32's last place (the angle's three roundings, the series' four, the scale), a
    product and the sum within three; then one rounding to the type, of binary16's subnormals half of 2^-24."""
    err = 12 * ULP * size
    return err + half_step(dtype) * (want.abs() + err) + (2.0 ** -25 if dtype == torch.float16 else 0)


def make_cache(pages, heads, size, dim, dtype, order="head", device="cuda", seed=0, fill=None):
    """(k, v) caches [pages, heads, size, dim], laid out by heads or by tokens, random or filled."""
    out = []
    for i in range(2):
        shape = (pages, heads, size, dim) if order == "head" else (pages, size, heads, dim)
        g = torch.Generator().manual_seed(2 * seed + i)
        x = torch.randn(shape, generator=g) if fill is None else torch.full(shape, float(fill))
        x = x.to(device, dtype)
        out.append(x if order == "head" else x.transpose(1, 2))
    return out


def keys_of(cache, table, length, head):
    """The first `length` rows of a sequence's pages, in 64 bits; rows of pages outside the cache are NaN."""
    size = cache.shape[2]
    rows = torch.full((max(length, 0), cache.shape[3]), float("nan"), dtype=torch.float64)
    for j in range(length):
        page = int(table[j // size])
        if 0 <= page < cache.shape[0]:
            rows[j] = cache[page, head, j % size].double().cpu()
    return rows


def attention(q, kc, vc, table, lengths, counts, heads, scale, causal, window, rounding=True):
    """(out, bound of the error before out's own rounding, whether a row sees anything) for tokens side by side.

    A score sums head_dim exact products in fp32, one unit of its last place a term at most (2^-23), then the scale and the
    maximum's difference, three more of its size; a weight takes the score's error, two units for the exponential and one
    rounding to the type; the softmax's sum and the second product's sums, a rounding for every eight keys in a lane and 64 across
    lanes, waves and parts, each rescaled as often."""
    dtype, kvh, dim = q.dtype, kc.shape[1], kc.shape[3]
    n = sum(counts)
    group = heads // kvh
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    bound, sees = torch.zeros_like(out), torch.zeros(n, heads, dtype=torch.bool)
    q = q[:n].double().cpu().reshape(n, heads, dim)
    kc, vc, table = kc.cpu(), vc.cpu(), table.cpu()
    capacity = table.shape[1] * kc.shape[2]
    weight = half_step(dtype) if rounding and dtype != torch.float32 else 0.0
    t0 = 0
    for b, count in enumerate(counts):
        length = min(max(int(lengths[b]), 0), capacity)
        j = torch.arange(length)
        p = length - count + torch.arange(count)[:, None] if causal else torch.full((count, 1), length - 1)
        seen = j <= p
        if window:
            seen &= j > p - window
        held = torch.tensor([0 <= int(table[b, i // kc.shape[2]]) < kc.shape[0] for i in range(length)], dtype=torch.bool)
        seen = seen & held
        for g in range(kvh):
            k, v = keys_of(kc, table[b], length, g), keys_of(vc, table[b], length, g)
            for h in range(g * group, (g + 1) * group):
                x = q[t0:t0 + count, h]
                z = scale * (x @ k.T)
                size = scale * (torch.nan_to_num(x, 0, 0, 0).abs() @ torch.nan_to_num(k, 0, 0, 0).abs().T)
                z = torch.where(seen, z, -float("inf"))
                m = z.amax(-1, keepdim=True) if length else torch.zeros(count, 0)
                none = (~seen).all(-1) if length else torch.ones(count, dtype=torch.bool)
                if length:
                    none = none | (torch.where(seen, z, -float("inf")) == -float("inf")).all(-1)
                    e = torch.exp(z - torch.where(none[:, None], 0.0, m))
                    w = e / torch.where(none[:, None], 1.0, e.sum(-1, keepdim=True))
                    for i in range(count):
                        at = seen[i]
                        if none[i]:
                            continue
                        out[t0 + i, h] = w[i, at] @ v[at]
                        score = (2 * dim + 6) * ULP * size[i, at].max() if at.any() else 0.0
                        rel = 2 * score + 4 * ULP + weight + (length / 4 + 128) * ULP
                        bound[t0 + i, h] = rel * (w[i, at] @ torch.nan_to_num(v[at], 0, 0, 0).abs())
                sees[t0:t0 + count, h] = ~none
        t0 += count
    return out.reshape(n, -1), bound.reshape(n, -1), sees
