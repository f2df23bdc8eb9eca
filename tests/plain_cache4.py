"""The 4-bit cache, the attention over it and the norm and rotation of heads in 64 bits, written from their definitions."""
import numpy as np

PAGE, GROUP = 64, 32
SCALES = np.array([(8 + b % 8) * 2.0 ** (b // 8 - 23) for b in range(255)])


def held(x):
    """What rows of numbers are held as: [..., dim], dim a multiple of 32."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    bad = ~np.isfinite(g).all(-1)
    top = np.where(bad, 0.0, np.abs(np.where(np.isfinite(g), g, 0.0)).max(-1))
    s = SCALES[np.minimum(np.searchsorted(7.0 * SCALES, top), 254)][..., None]
    with np.errstate(invalid="ignore"):
        y = np.clip(np.rint(np.where(np.isfinite(g), g, 0.0) / s), -7, 7) * s
    return np.where(bad[..., None], np.nan, y).reshape(x.shape)


def record(k, v):
    """The bytes of one page of one key head that is given 64 rows (k, v: [64, dim]; held values would not do: the largest of a group
    may have the code 6, and a smaller scale would then do for it)."""
    parts = []
    for x in (k, v):
        g = np.asarray(x, dtype=np.float64).reshape(PAGE, -1, GROUP)
        bad = ~np.isfinite(g).all(-1)
        g = np.where(bad[..., None], 0.0, g)
        top = np.abs(g).max(-1)
        byte = np.minimum(np.searchsorted(7.0 * SCALES, top), 254)
        code = (np.clip(np.rint(g / SCALES[byte][..., None]), -7, 7) + 8).astype(np.uint8).reshape(PAGE, -1)
        parts.append((code[:, 0::2] | code[:, 1::2] << 4, np.where(bad, 255, byte).astype(np.uint8)))
    return np.concatenate([parts[0][0].ravel(), parts[1][0].ravel(), parts[0][1].ravel(), parts[1][1].ravel()])


def attention(q, k, v, past, scale, window=0, keep_first=0):
    """q [new, heads, dim]; k, v [positions, kv_heads, dim].  Returns the result, the same sums over |v|, the largest
    scale * sum |q k| of a visible key and the number of visible keys, each per (query, head)."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    new, heads, dim = q.shape
    group = heads // k.shape[1]
    pos = past + np.arange(new)[:, None]
    key = np.arange(k.shape[0])[None]
    seen = key <= pos
    if window:
        seen &= (key > pos - window) | (key < keep_first)
    y, size, reach = np.empty_like(q), np.empty_like(q), np.empty((new, heads))
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = np.where(seen, q[:, h] @ np.where(seen.any(0)[:, None], kh, 0.0).T * scale, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        vh = np.where(seen.any(0)[:, None], vh, 0.0)
        y[:, h], size[:, h] = p @ vh, p @ np.abs(vh)
        reach[:, h] = np.where(seen, np.abs(q[:, h]) @ np.abs(np.where(seen.any(0)[:, None], kh, 0.0)).T * abs(scale), 0.0).max(-1)
    return y, size, reach, seen.sum(-1)


def allowed(dtype_bits, y, size, reach, count, dim):
    """How far a result may be from `y`: products and sums in 32 bits, and for 8-bit significands (bfloat16) the weights and the result
    each rounded once.  A weight below 2^-126 of the largest has no normal 32-bit number and may be 0: that much of a value, which is 25,088 at
    most, for each key."""
    exact = count[:, None, None] * 2.0 ** -126 * 25088 + size * 2.0 ** -24 * (2 * (dim + 8) * reach + 2 * count[:, None] + 64)[..., None]
    if dtype_bits == 8:
        return 2.0 ** -8 * (1 + 2.0 ** -7) * (np.abs(y) + size) + exact
    return exact + 2.0 ** -24 * np.abs(y)


def norm_rotary(x, positions, freq, rot, weight=None, eps=0.0, interleaved=False, size=1.0):
    """x [tokens, heads, dim] -> the result and, per channel, the sizes of what was added up for it."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    angle = np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(freq, dtype=np.float64)
    c, s = size * np.cos(angle)[:, None], size * np.sin(angle)[:, None]
    y, mass = x.copy(), np.abs(x)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    mass[..., a] = mass[..., b] = size * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, mass
