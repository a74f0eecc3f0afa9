"""The operators that serve prompts and tokens together (ops 315-319) from their definition in 64 bits, on numpy arrays: what the tests
hold the oracle and the device to, with bounds that count the roundings of a 32-bit evaluation."""
import numpy as np

U = 2.0 ** -24                       # half a step of f32, relative


def half_step(dtype):
    return 2.0 ** -8 if dtype == 'bf16' else 2.0 ** -24


def shaped(x, pro, x2=None, gamma=None, eps=0.0):
    """What rows_q8 brings to 8 bits, as f32 rounds it (SwiGLU: in 64 bits)."""
    x = x.astype(np.float32)
    if pro == 1:
        rstd = np.float32(1) * (1 / np.sqrt((x.astype(np.float64) ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))).astype(np.float32)
        return ((x * rstd).astype(np.float32) * gamma.astype(np.float32)).astype(np.float32)
    if pro == 2:
        y = x.astype(np.float64)
        return y / (1 + np.exp(-y)) * x2.astype(np.float64)
    return x


def quantise(v):
    """(bytes, scales) of the rows of v."""
    with np.errstate(invalid='ignore', over='ignore'):
        big = np.abs(v.astype(np.float32)).max(1, keepdims=True)
        scale = (big * np.float32(1 / 127)).astype(np.float32)
        scale = np.where(scale < np.float32(1.17549435e-38), np.float32(0), scale)
        fine = np.isfinite(v).all(1, keepdims=True)
        q = np.where(fine & (scale > 0), np.rint(v.astype(np.float64) / np.where(scale > 0, scale, 1).astype(np.float64)), 0)
    return np.clip(q, -127, 127).astype(np.int8), np.where(fine, scale, np.float32(np.nan))[:, 0].astype(np.float32)


def product(a, sa, w, sw, bias=None, res=None):
    """(result, bound of an f32 evaluation before the store): the sum is exact, then its conversion, two products and two sums."""
    s = a.astype(np.int64) @ w.astype(np.int64).T
    y = s * sa[:, None].astype(np.float64) * sw[None].astype(np.float64)
    mag = 3 * np.abs(y)
    if bias is not None:
        y = y + bias[None].astype(np.float64)
        mag = mag + np.abs(y)
    if res is not None:
        y = y + res.astype(np.float64)
        mag = mag + np.abs(y)
    return y, mag * U * 1.01


def near(have, want, bound, dtype):
    """|have - want| within `bound` and the roundings of the store: to f32, and from there to the buffer's type."""
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(have), nan)
    far = np.abs(have.astype(np.float64) - want)
    allow = bound + (half_step(dtype) + U) * (np.abs(want) + bound) + 2.0 ** -140
    worst = np.where(nan, 0, far / allow).max(initial=0)
    assert worst <= 1, f'{worst} times what the roundings allow, at {np.unravel_index(np.argmax(np.where(nan, 0, far / allow)), far.shape)}'


def turned(x, gamma, eps, theta, pos):
    """[rows, heads, hd] normalised per head and rotated, in 64 bits."""
    x = x.astype(np.float64)
    hd = x.shape[-1]
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * gamma.astype(np.float64)
    if theta:
        ang = pos.astype(np.float64)[:, None] * np.float64(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
        co, si = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        x = np.concatenate([a * co - b * si, a * si + b * co], -1)
    return x


def owners(cu, rows):
    """(row, sequence, number in the sequence) of every row with a token."""
    r = np.arange(cu[0], cu[-1])
    b = np.searchsorted(cu[1:], r, side='right')
    return r, b, r - cu[b]


def append(kc, vc, table, lens, cu, q, k, v, page, qgamma, kgamma, eps, theta):
    """kc, vc [pages, Hkv, page, hd] and the queries [rows, H, hd] after the call, rows without a token NaN."""
    kc, vc = kc.astype(np.float64), vc.astype(np.float64)
    r, b, i = owners(cu, len(k))
    pos = lens[b] + i
    where, at = table[b, pos // page], pos % page
    kc[where, :, at] = turned(k[r], kgamma, eps, theta, pos)
    vc[where, :, at] = v[r]
    out = np.full(q.shape, np.nan) if q is not None else None
    if q is not None:
        out[r] = turned(q[r], qgamma, eps, theta, pos)
    return kc, vc, out


def attend(q, kc, vc, table, lens, cu, page, scale):
    """([rows, H, hd], sum of weights times magnitudes of the values): rows without a token NaN. Keys past a row's position do not count."""
    H, hd, Hkv = q.shape[1], q.shape[2], kc.shape[1]
    out, mag = np.full(q.shape, np.nan), np.zeros(q.shape)
    for r, b, i in zip(*owners(cu, len(q))):
        n = lens[b] + i + 1
        t = np.arange(n)
        for h in range(H):
            k, v = (x[table[b, t // page], h * Hkv // H, t % page].astype(np.float64) for x in (kc, vc))
            s = k @ q[r, h].astype(np.float64) * np.float64(np.float32(scale))
            with np.errstate(invalid='ignore'):
                p = np.exp(s - s.max())
                p /= p.sum()
                out[r, h], mag[r, h] = p @ v, p @ np.abs(v)
    return out, mag
