"""The serving operators (ops 312-314) from their definition in 64 bits, on numpy arrays: what the tests hold the oracle and the
GPU to. Caches are dicts of kq, vq (int8 [pairs, nblk, blk, hd] and [pairs, nblk, hd, blk]), ks, vs [pairs, nblk], kt, vt
[pairs, blk, hd]."""
import numpy as np

from kvm_amd import bundle as bl

FLT_MIN = np.float32(1.17549435e-38)


def turned(x, gamma, eps, theta, t):
    """[.., hd] at positions t [..]: RMS-normalised per head, then rotated (halves together)."""
    x = np.asarray(x, np.float64)
    hd = x.shape[-1]
    if gamma is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gamma, np.float64)
    if theta > 0:
        a = np.asarray(t, np.float64)[..., None] * float(theta) ** (-2.0 * np.arange(hd // 2) / hd)
        u, v = x[..., :hd // 2], x[..., hd // 2:]
        x = np.concatenate([u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a)], -1)
    return x


def empty_cache(pairs, nblk, blk, hd):
    z = np.zeros
    return {'kq': z((pairs, nblk, blk, hd), np.int8), 'vq': z((pairs, nblk, hd, blk), np.int8), 'ks': z((pairs, nblk), np.float32),
            'vs': z((pairs, nblk), np.float32), 'kt': z((pairs, blk, hd), np.float32), 'vt': z((pairs, blk, hd), np.float32)}


def quantise(x):
    """[.., blk, hd] f32 -> (int8, scale f32), a scale per block."""
    flat = x.reshape(*x.shape[:-2], -1)
    fine = np.isfinite(flat).all(-1)
    amax = np.where(fine, np.abs(np.where(np.isfinite(flat), flat, 0)).max(-1), 0).astype(np.float32)
    s = amax * np.float32(1 / 127)
    s = np.where(s < FLT_MIN, np.float32(0), s)
    d = np.where(s > 0, s, 1).astype(np.float64)[..., None, None]
    q = np.where((fine & (s > 0))[..., None, None], np.rint(np.where(np.isfinite(x), x, 0) / d), 0)
    return np.clip(q, -127, 127).astype(np.int8), np.where(fine, s, np.float32(np.nan)).astype(np.float32)


def append(c, knew, vnew, lens, hkv, n_new, bf16, gamma=None, eps=0.0, theta=0.0):
    """c after the append of knew, vnew [B * n_new, >= hkv * hd]; token after token."""
    c = {k: v.copy() for k, v in c.items()}
    _, nblk, blk, hd = c['kq'].shape
    for b, L in enumerate(lens):
        if L < 0:
            continue
        for h in range(hkv):
            p = b * hkv + h
            for x, new in (('k', knew), ('v', vnew)):
                rows = np.asarray(new[b * n_new:(b + 1) * n_new, h * hd:(h + 1) * hd], np.float64)
                if x == 'k':
                    rows = turned(rows, gamma, eps, theta, L + np.arange(n_new))
                rows = rows.astype(np.float32)
                rows = bl.bf16_round(rows) if bf16 else rows
                tail = c[x + 't'][p].copy()
                start = tail.copy()
                for i in range(n_new):
                    t = L + i
                    tail[t % blk] = rows[i]
                    if t % blk == blk - 1:
                        q, s = quantise(tail[None])
                        c[x + 'q'][p, t // blk] = q[0] if x == 'k' else q[0].T
                        c[x + 's'][p, t // blk] = s[0]
                        tail = start.copy()                         # rows of a finished block do not stay in the tail
                c[x + 't'][p] = tail
    return c


def held(c, x, p, n):
    """[n, hd] values of pair p that the cache holds."""
    _, nblk, blk, hd = c['kq'].shape
    w = n // blk
    q = c[x + 'q'][p, :w].astype(np.float64)
    q = (q if x == 'k' else q.transpose(0, 2, 1)) * c[x + 's'][p, :w, None, None].astype(np.float64)
    return np.concatenate([q.reshape(-1, hd), c[x + 't'][p, :n - w * blk].astype(np.float64)])


def attend(c, q, lens, hkv, heads, n_new, scale, gamma=None, eps=0.0, theta=0.0):
    """(o, bound): the attention, and what it may be off in 32 bits: a score is a sum of hd products of 22 bits and more
    (relative to the sum of their magnitudes, (hd + 8) 2^-24), an exponential off by that and a step carries it into numerator and
    denominator, their sums add a few steps more (n / 2 + 64 of 2^-24 relative to the largest value)."""
    hd, G = c['kq'].shape[3], heads // hkv
    o, bound = np.zeros((len(lens) * n_new, heads * hd)), np.zeros((len(lens) * n_new, heads * hd))
    for b, L in enumerate(lens):
        if L < 0:
            continue
        for h in range(heads):
            k, v = held(c, 'k', b * hkv + h // G, L + n_new), held(c, 'v', b * hkv + h // G, L + n_new)
            for i in range(n_new):
                x = turned(q[b * n_new + i, h * hd:(h + 1) * hd], gamma, eps, theta, L + i)
                n = L + i + 1
                with np.errstate(invalid='ignore', over='ignore'):
                    s = k[:n] @ x * scale
                    w = np.exp(s - s.max())
                    r = (w[:, None] * v[:n]).sum(0) / w.sum()
                    size = (np.abs(k[:n]) @ np.abs(x)).max() * abs(scale)
                    e = (2 * (hd + 8) * size + n / 2 + 64) * 2.0 ** -24 * np.abs(v[:n]).max()
                o[b * n_new + i, h * hd:(h + 1) * hd], bound[b * n_new + i, h * hd:(h + 1) * hd] = r, e
    return o, bound


def adjust(x, par, hist=None, plen=None, hlen=None, last=None, bidx=None, bval=None, mask=None, mrow=None):
    """(out, hist, bound): bound counts five roundings to f32 of what is added up."""
    x = np.asarray(x, np.float64)
    R, V = x.shape
    out, size, hist = x.copy(), np.abs(x), None if hist is None else hist.copy()
    for r in range(R):
        rep, freq, pres = (float(p) for p in par[r, :3])
        if hist is not None:
            said = list(hist[r, :hlen[r]]) + ([last[r]] if last is not None else [])
            gen = np.bincount([t for t in said[plen[r]:] if 0 <= t < V], minlength=V)
            seen = np.bincount([t for t in said if 0 <= t < V], minlength=V) > 0
            with np.errstate(invalid='ignore', over='ignore'):
                y = np.where(x[r] > 0, x[r] / rep, x[r] * rep)
                out[r] = np.where(gen > 0, np.where(seen, y, x[r]) - freq * gen - pres, np.where(seen, y, x[r]))
            size[r] = np.abs(x[r]) * max(rep, 1 / rep) + abs(freq) * gen + abs(pres)
            if last is not None:
                hist[r, hlen[r]] = last[r]
        if bidx is not None:
            for v, a in zip(bidx[r], bval[r]):
                if 0 <= v < V:
                    out[r, v] += float(a)
                    size[r, v] += abs(float(a))
        m = r if mrow is None else mrow[r]
        if mask is not None and m >= 0:
            bits = (mask[m].view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            out[r] = np.where(bits.reshape(-1)[:V] > 0, out[r], -np.inf)
    return out, hist, 5 * 2.0 ** -24 * size
