"""Tiles of the attention over a paged cache (op 319) that are cut into pieces: a piece without weight that holds a NaN, more pieces than the merge's
table of weights holds, pieces whose places fill more than one part of the list in LDS."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu


def _run(lb, init, shape, path=PATH_DYNAMIC):
    ex = Executor.from_bundle(lb, buffers=init, path=path)
    ex.run()
    o, cnt = ex.read('o').reshape(shape), ex.read('o.cnt')
    ex.close()
    assert not cnt.any()
    return o


# few rows, many, f32, the general form, more pieces times rows than the table holds
NANS = [(64, 128, 1, 4, 'bf16', [6000], [1]), (64, 128, 1, 8, 'bf16', [6000], [5]), (16, 64, 1, 2, 'f32', [6000], [1]), (64, 100, 1, 8, 'f32', [6000], [4]),
        (16, 64, 1, 16, 'bf16', [45000], [8])]


@pytest.mark.parametrize('what', ['key', 'value', 'infinite value'])
@pytest.mark.parametrize('tasks', [1, 256])
@pytest.mark.parametrize('case', NANS, ids=str)
def test_nan_in_a_piece_without_weight(case, tasks, what):
    """The first 1,000 keys score 400 below the others, so that all of their piece weighs e^-400 (0 in 32 bits): what is not finite among them, and seen, is
    not lost with it."""
    print(f'nan {case} {tasks} {what}', flush=True)
    page, hd, hkv, heads, dt, lens, new = case
    rng = np.random.default_rng(3)

    def kv(kc, vc, table):
        t = np.arange(lens[0] + new[0])
        kc[table[0, t // page], :, t % page, 0] = np.where(t < 1000, 0, 400)[:, None]
        if what == 'key':
            kc[table[0, 100 // page], :, 100 % page, 1] = np.nan
        else:
            vc[table[0, 100 // page], :, 100 % page, 1] = np.nan if what == 'value' else np.inf
        return kc, vc

    def q(rows):
        x = 0.1 * rng.standard_normal((rows, heads, hd))
        x[..., 0] = 1
        return mg.bf(x, dt)
    (lb, init), pg, qs = mg.attend_graph(case, rng, tasks=tasks, kv=kv, q=q, scale=1.0)
    o = _run(lb, init, qs.shape)[:new[0]]
    if what == 'key':
        assert np.isnan(o).all()
    else:
        assert not np.isfinite(o[..., 1]).any() and np.isfinite(np.delete(o, 1, -1)).all()


@pytest.mark.parametrize('tasks', [1, 3, 256])
@pytest.mark.parametrize('case', [(16, 64, 1, 16, 'bf16', [45000], [8]), (16, 128, 1, 8, 'bf16', [70001], [5])], ids=str)
def test_long_tiles(case, tasks):
    """Many rows over many pages of 16 tokens: in one piece (places of 2,048 pages at a time), in few, in more than 64 (weights as the merge goes)."""
    print(f'long tiles {case} {tasks}', flush=True)
    page, hd, hkv, heads, dt, lens, new = case
    (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(4), tasks=tasks)
    o = _run(lb, init, q.shape, PATH_STATIC if tasks == 3 else PATH_DYNAMIC)
    want, mag = f64.attend(q, *pg, page, 1 / np.sqrt(hd))
    sabs = np.abs(q).sum(-1).max() * np.nanmax(np.abs(pg[0])) / np.sqrt(hd)
    on = ~np.isnan(want)
    f64.near(o[on], want[on], (mg.attend_bound(case, mag, sabs, True) + 2.0 ** -16 * mag)[on], dt)
    assert (o[~on] == 7).all()
