"""The operators of the 4-bit cache in 64-bit numpy, one value at a time where that is clearest."""
import numpy as np


def scale_of(block):
    """d of 32 values: -1/8 of the value of the largest magnitude (the positive one of two), to 8 significant bits, as f16."""
    high, low = block.max(), block.min()
    m = (high if high >= -low else low) / -8.0
    if m == 0.0:
        return np.float16(0.0)
    mantissa, exponent = np.frexp(m)
    m = np.ldexp(np.round(mantissa * 256.0), exponent - 8)
    return np.float16(np.clip(m, -65280.0, 65280.0))


def quantise(rows):
    """[..., dim] -> bytes [..., dim / 2], scales [..., dim / 32]."""
    x = np.nan_to_num(np.asarray(rows, np.float64), nan=0.0, posinf=3e38, neginf=-3e38).clip(-3e38, 3e38)
    blocks = x.reshape(-1, 32)
    d = np.array([scale_of(b) for b in blocks], np.float16)
    wide = d.astype(np.float64)[:, None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(wide == 0, 8.0, np.clip(np.floor(blocks / wide + 8.5), 0, 15)).astype(np.uint8)
    quants = n[:, :16] | (n[:, 16:] << 4)
    return quants.reshape(*x.shape[:-1], x.shape[-1] // 2), d.reshape(*x.shape[:-1], x.shape[-1] // 32)


def values(quants, scales):
    q = quants.reshape(*scales.shape, 16)
    n = np.concatenate((q & 15, q >> 4), -1).astype(np.float64) - 8.0
    return (n * scales.astype(np.float64)[..., None]).reshape(*quants.shape[:-1], -1)


def rotated(x, position, bias=None, norm=None, eps=0.0, turns=None, adjacent=False, attn_factor=1.0):
    """x [rows, heads, dim] + bias, over its root mean square times norm, pairs turned by position * turns."""
    x = np.array(x, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64).reshape(x.shape[1:])
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    if turns is None:
        return x
    width = 2 * len(turns)
    angle = 2.0 * np.pi * np.asarray(position, np.float64)[:, None, None] * turns
    c, s = np.cos(angle) * attn_factor, np.sin(angle) * attn_factor
    first = slice(0, width, 2) if adjacent else slice(0, width // 2)
    second = slice(1, width, 2) if adjacent else slice(width // 2, width)
    a, b, y = x[..., first], x[..., second], x.copy()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def attention(q, k, v, context, scale, window=0):
    """q [tokens, heads, dim] at positions context, context + 1, ...; k, v [positions, kv heads, dim] as values."""
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    out = np.zeros((tokens, heads, dim))
    for h in range(heads):
        s = q[:, h].astype(np.float64) @ k[:, h // group].T * scale
        seen = (context + np.arange(tokens))[:, None] - np.arange(len(k))
        hidden = (seen < 0) | (seen >= (window or 1 << 40))
        s[hidden] = -np.inf
        rows = ~hidden.all(1)
        if rows.any():
            p = np.exp(s[rows] - s[rows].max(1, keepdims=True))
            out[rows, h] = p @ v[:, h // group] / p.sum(1, keepdims=True)
    return out
