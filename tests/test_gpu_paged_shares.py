"""How the tasks of an attention over a paged cache (op 319) share its tiles where there is a task for each: one to a task, none idle beside one with two."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import serving_graphs as sg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('path', [PATH_STATIC, PATH_DYNAMIC])
@pytest.mark.parametrize('lens,new', [([3750], [1024]), ([1500, 1400], [512, 512])], ids=str)
def test_a_tile_to_a_task(lens, new, path):
    """256 tiles of 128 rows for 256 tasks: a task without one ends after some microseconds, where a tile takes a hundred and more."""
    print(f'shares {lens} {new} path {path}', flush=True)
    b, rng = sg.Builder(0), np.random.default_rng(1)
    page, hd, hkv, heads, rows = 64, 128, 8, 32, sum(new)
    width = -(-(max(lens) + max(new)) // page)
    data = {}
    c = sg.serving.paged_buffers(b, '', len(lens) * width, hkv, hd, page)
    sg.add(b, data, 'table', rng.permutation(len(lens) * width).reshape(len(lens), width).astype(np.int32))
    sg.add(b, data, 'lens', np.array(lens, np.int32)[:, None]), sg.add(b, data, 'cu', np.cumsum([0] + new).astype(np.int32)[:, None])
    b.fill('q', rows, heads * hd, 'bf16', value=0.1), b.fill('o', rows, heads * hd, 'bf16')
    sg.serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', heads)
    lb, init = sg.compiled(b, data)
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=True)
    for _ in range(3):
        ex.relaunch()
        assert ex.finish()['done'] == lb.ntasks
    t = ex.trace()
    ex.close()
    took = (t['end'] - t['start']).astype(float)
    assert took.min() > 0.3 * np.median(took), (took.min(), np.median(took), took.max())


# fewer tiles than tasks, as many, sequences without a token between; head sizes and storages of every form
@pytest.mark.parametrize('tasks', [6, 8, 13, 256])
@pytest.mark.parametrize('case', [(16, 64, 2, 2, 'bf16', [100, 0, 130, 90], [1, 0, 1, 1]), (32, 128, 1, 4, 'bf16', [300, 0, 200], [70, 0, 64]), (16, 64, 2, 4, 'f32', [60, 80], [33, 17]),
                                  (64, 100, 1, 3, 'f32', [200, 0, 9, 0], [30, 0, 0, 11])], ids=str)
def test_whole_tiles(case, tasks):
    print(f'whole tiles {case} {tasks}', flush=True)
    page, hd, hkv, heads, dt, lens, new = case
    (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(2), tasks=tasks)
    ex = Executor.from_bundle(lb, buffers=init)
    for _ in range(2):
        ex.relaunch()
        ex.finish()
    o = ex.read('o').reshape(q.shape)
    ex.close()
    want, mag = f64.attend(q, *pg, page, 1 / np.sqrt(hd))
    sabs = np.abs(q).sum(-1).max() * np.nanmax(np.abs(pg[0])) / np.sqrt(hd)
    on = ~np.isnan(want)
    f64.near(o[on], want[on], (mg.attend_bound(case, mag, sabs, True) + 2.0 ** -16 * mag)[on], dt)
    assert (o[~on] == 7).all()
