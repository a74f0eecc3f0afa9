"""The workspace that linear_q8 finds in its graph, and rows that a caller has in 8 bits already, hold what the call needs, or it is refused where the
graph is built."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import oracle
import serving_graphs as sg
from kvm_amd.workloads import Builder, serving


def _builder(M=64, K=256):
    b = Builder(0)
    b.fill('x', M, K), b.fill('wide', M, 2 * K), b.fill('o', M, 40)
    return b, serving.weight_q8_buffers(b, 'w', 40, K), serving.weight_q8_buffers(b, 'w2', 40, 2 * K)


@pytest.mark.parametrize('M,x,what', [(64, 'x', '8 rows of 256 bytes: 64 rows of 256'), (8, 'wide', '8 rows of 256 bytes: 8 rows of 512')])
def test_a_workspace_of_the_graph_that_is_too_small(M, x, what):
    b, w, w2 = _builder()
    at = serving.linear_q8(b, 'x', w, 'o', 8)
    with pytest.raises(ValueError, match=what):
        serving.linear_q8(b, x, w if x == 'x' else w2, 'o', M, after=at)


def test_scales_of_the_workspace_that_are_too_few():
    b, w, _ = _builder()
    b.fill('o.x', 64, 64, 'i32'), b.fill('o.xs', 8)
    with pytest.raises(ValueError, match='8 rows of 256 bytes: 64 rows'):
        serving.linear_q8(b, 'x', w, 'o', 64)


def test_rows_in_8_bits_that_are_too_few():
    b, w, _ = _builder()
    y = serving.rows_q8_buffers(b, 'y', 8, 256)
    with pytest.raises(ValueError, match='8 rows'):
        serving.linear_q8(b, y, w, 'o', 9)


def test_a_larger_workspace_is_used_again():
    """Calls of fewer rows and of a smaller K after a larger one, in the same workspace."""
    rng = np.random.default_rng(1)
    b, data = Builder(0), {}
    sg.add(b, data, 'x', rng.standard_normal((20, 300)).astype(np.float32)), sg.add(b, data, 'y', rng.standard_normal((5, 77)).astype(np.float32))
    b.fill('o', 20, 40)
    want, at = {}, ()
    for n, x, M in (('w', 'x', 20), ('v', 'y', 5)):
        raw = rng.standard_normal((40, data[x].shape[1])).astype(np.float32)
        w = serving.weight_q8_buffers(b, n, *raw.shape)
        q, s = f64.quantise(raw)
        data[n], data[n + 's'] = mg.words(q, b.buffers[-2]['cols']), s[:, None]
        at = serving.linear_q8(b, x, w, 'o', M, after=at)
        want[x] = f64.product(*f64.quantise(data[x]), q, s)
    assert sum(d['name'] == 'o.x' for d in b.buffers) == 1
    lb, init = sg.compiled(b, data)
    o = oracle.run(lb, init)['buffers'][sg.names(lb).index('o')].reshape(20, 40)
    f64.near(o[:5], *want['y'], 'f32')
    f64.near(o[5:], want['x'][0][5:], want['x'][1][5:], 'f32')
