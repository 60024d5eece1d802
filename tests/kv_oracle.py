"""Plain float64 / float32 NumPy statement of the paged 8-bit cache, for the tests."""
import numpy as np
import torch

EPS = np.float32(2.0 ** -23)
LARGEST = {"int8": np.float32(127.0), "e4m3": np.float32(448.0)}


def to_bytes(x, fmt):
    """float32 -> grid, ties to even, as int8 bytes."""
    if fmt == "int8":
        return np.clip(np.rint(np.nan_to_num(x)), -127, 127).astype(np.int8)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).view(torch.int8).numpy()


def from_bytes(q, fmt):
    if fmt == "int8":
        return q.astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(q)).view(torch.float8_e4m3fn).float().numpy()


def write(data, scale, x, table, lens, starts, fmt):
    """In place on data [pages, heads, page, dim] int8 and scale [pages, heads]; x [tokens, heads, dim] float32."""
    page = data.shape[2]
    for b in range(len(lens)):
        n = starts[b + 1] - starts[b]
        base = lens[b] - n
        for nth in range(max(base, 0) // page, -(-lens[b] // page)):
            at, stop = max(base, nth * page, 0), min(lens[b], nth * page + page)
            p, held = table[b][nth], at - nth * page
            for h in range(data.shape[1]):
                values = x[starts[b] + at - base:starts[b] + stop - base, h]
                top = np.abs(values).max()
                s = np.maximum(top, EPS) / LARGEST[fmt]
                old = scale[p, h]
                if not np.isfinite(top) or (held and np.isnan(old)):
                    s = np.float32(np.nan)
                elif held:
                    s = np.maximum(s, old)
                with np.errstate(invalid="ignore"):
                    if held and not s == old:
                        data[p, h, :held] = to_bytes(from_bytes(data[p, h, :held], fmt) * np.float32(old / s), fmt)
                    data[p, h, held:held + stop - at] = to_bytes(values / s, fmt)
                scale[p, h] = s


def tokens_of(data, scale, table, b, first, end, fmt):
    """float32 [end - first, heads, dim] of one sequence."""
    page = data.shape[2]
    rows = [from_bytes(data[table[b][t // page], :, t % page], fmt) * scale[table[b][t // page]][:, None]
            for t in range(first, end)]
    return np.stack(rows) if rows else np.zeros((0, data.shape[1], data.shape[3]), np.float32)


def attention(q, keys, values, total, *, scale, causal=True, window=0):
    """q [n, heads, dim] at the last positions of `total`; keys, values [total, kv_heads, dim].
    Returns (out, lse, weight of |v|, largest sum of |q k| scale) in float64."""
    n, heads, dim = q.shape
    group = heads // keys.shape[1]
    out = np.zeros((n, heads, dim))
    spread = np.zeros((n, heads, dim))
    lse = np.full((n, heads), -np.inf)
    loud = np.zeros((n, heads))
    keys, values, q = keys.astype(np.float64), values.astype(np.float64), q.astype(np.float64)
    for i in range(n):
        position = total - n + i
        last = (position + 1 if causal else total) if position >= 0 else 0
        first = max(0, position - window + 1) if window else 0
        if last <= first:
            continue
        for h in range(heads):
            k, v = keys[first:last, h // group], values[first:last, h // group]
            s = k @ q[i, h] * scale
            top = s.max()
            p = np.exp(s - top)
            out[i, h] = p @ v / p.sum()
            spread[i, h] = p @ np.abs(v) / p.sum()
            lse[i, h] = top + np.log(p.sum())
            loud[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() * abs(scale)
    return out, lse, spread, loud
