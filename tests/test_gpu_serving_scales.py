"""Attention over the 8-bit cache where a block's value scale is far above that of the blocks which carry the weight: the result
is held to the weighted magnitudes, not to the largest value met."""
import numpy as np
import pytest

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu

SCALE = 0.5


def _cache(rng, nblk, blk, hd, heavy, big, ratio):
    """One pair: the first byte of a key is 100 in the blocks `heavy` and 20 elsewhere, and a query holds that dim alone, so scores are
    50 and 10 and a light token weighs e^-40 (2^-58) of a heavy one; the blocks `big` have values 2^ratio larger than the others."""
    c = f64.empty_cache(1, nblk, blk, hd)
    c['kq'][:] = rng.integers(-127, 128, c['kq'].shape)
    c['vq'][:] = rng.integers(-127, 128, c['vq'].shape)
    c['kq'][..., 0] = 20
    c['kq'][:, heavy, :, 0] = 100
    c['ks'][:], c['vs'][:] = 1, 1
    c['vs'][:, big] = 2.0 ** ratio
    for x in ('kt', 'vt'):
        c[x][:] = rng.standard_normal(c[x].shape)
    c['kt'][..., 0] = 20
    return c


def _want(c, q, lens, n_new, heads):
    """(o, bound). Scores are products of one number: off by 9 steps of 2^-24 of the largest, which every weight carries into
    numerator and denominator; an exponential and the sums add n / 2 + 64 steps, all of sum p |v|. A weight times its block's scale is
    held to 2^-22 (4 steps), and no closer than 2^-36 of the largest such product, times the bytes. A weight below 2^-126 may be 0."""
    hd = c['kq'].shape[3]
    o, bound = np.zeros((len(lens) * n_new, heads * hd)), np.zeros((len(lens) * n_new, heads * hd))
    for b, L in enumerate(lens):
        k, v = f64.held(c, 'k', b, L + n_new), f64.held(c, 'v', b, L + n_new)
        blk = c['kq'].shape[2]
        whole = (L + n_new) // blk * blk
        s8 = np.repeat(c['vs'][b, :whole // blk].astype(np.float64), blk)
        for h in range(heads):
            for i in range(n_new):
                n = L + i + 1
                x = q[b * n_new + i, h * hd:(h + 1) * hd].astype(np.float64)
                s = k[:n] @ x * SCALE
                p = np.exp(s - s.max())
                p /= p.sum()
                a = np.abs(v[:n])
                m = min(n, whole)
                low = (p[:m] * s8[:m]).max() * 2.0 ** -36 * (a[:m] / s8[:m, None]).sum(0)
                size = (p[:, None] * a).sum(0)
                at = slice(h * hd, (h + 1) * hd)
                o[b * n_new + i, at] = p @ v[:n]
                bound[b * n_new + i, at] = (2 * 9 * np.abs(s).max() + n / 2 + 68) * 2.0 ** -24 * size + low + (np.minimum(p, 2.0 ** -126)[:, None] * a).sum(0)
    return o, bound


@pytest.mark.parametrize('tasks', [1, 256])
@pytest.mark.parametrize('ratio', [20, 28, 36, 50, 100])
@pytest.mark.parametrize('blk,hd,heads,n_new', [(64, 128, 1, 1), (16, 64, 4, 1), (64, 128, 16, 2), (128, 64, 1, 20)])
def test_a_large_scale_with_little_weight(blk, hd, heads, n_new, ratio, tasks):
    print(f'scales blk {blk} hd {hd} heads {heads} n_new {n_new} ratio {ratio} tasks {tasks}', flush=True)
    rng = np.random.default_rng(11)
    nblk = 2048 // blk
    for heavy, big in ((nblk // 2, 1), (1, nblk // 2), (nblk - 3, slice(nblk - 2, nblk - 1)), (slice(0, 1), slice(1, nblk - 1))):
        c = _cache(rng, nblk, blk, hd, heavy, big, ratio)
        lens = [blk * (nblk - 1) - n_new + 5]
        q = np.zeros((n_new, heads * hd), np.float32)
        q[:, ::hd] = 1 + np.arange(n_new * heads).reshape(n_new, heads) / 256
        lb, init = sg.attend_graph(c, q, lens, 1, heads, n_new, SCALE, 'f32', 'f32', tasks=tasks)
        ex = Executor.from_bundle(lb, buffers=init, path=PATH_STATIC if tasks == 1 else PATH_DYNAMIC)
        ex.run()
        got = ex.read('o')
        ex.close()
        want, bound = _want(c, q, lens, n_new, heads)
        sg.near(got, want, bound, 'f32')


@pytest.mark.parametrize('hd', [64, 128])
def test_a_large_scale_out_of_sight(hd):
    """A block that only later drafted tokens may see has values 2^60 times larger: the earlier ones do not notice."""
    print(f'out of sight {hd}', flush=True)
    rng = np.random.default_rng(12)
    blk, n_new = 16, 20
    c = _cache(rng, 68, blk, hd, slice(0, 4), 64, 60)
    c['kq'][:, 64, :, 0] = 100
    lens = [65 * blk - n_new]                                          # block 64 ends with the last new token
    q = np.zeros((n_new, hd), np.float32)
    q[:, 0] = 1
    lb, init = sg.attend_graph(c, q, lens, 1, 1, n_new, SCALE, 'f32', 'f32', tasks=1)
    ex = Executor.from_bundle(lb, buffers=init)
    ex.run()
    got = ex.read('o')
    ex.close()
    want, bound = _want(c, q, lens, n_new, 1)
    assert np.abs(want[:4]).max() < 200 < 2.0 ** 40 < np.abs(want[4:]).max()
    sg.near(got, want, bound, 'f32')
