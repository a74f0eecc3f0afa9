"""Ops 315 and 319 where a looser test would pass a wrong rounding: rows in 8 bits past 4 GiB, byte by byte; every output of an attention whose scores
are in the thousands."""
import numpy as np
import pytest
import torch

import mixed_fp64 as f64
import mixed_graphs as mg
from kvm_amd import bundle as bl
from kvm_amd import compiler, executor
from kvm_amd.executor import Executor
from kvm_amd.workloads import Builder, serving

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 1: torch.int32, 2: torch.bfloat16}


def test_rows_past_4_gib():
    """f32 rows in front of, around and behind the 2^32nd byte, with the norm: bytes and scales as the definition has them."""
    print('rows past 4 GiB', flush=True)
    K, M = 12296, 100000
    rng = np.random.default_rng(14)
    b = Builder(0)
    b.fill('x', M, K), b.fill('g', 1, K)
    y = serving.rows_q8_buffers(b, 'y', M, K)
    serving.rows_q8(b, 'x', y, M, gamma='g', eps=1e-6)
    lb = bl.load(compiler.compile_spec(b.spec()))
    t = {m['name']: torch.zeros((m['rows'], m['cols']), dtype=TORCH[m['dtype']], device='cuda') for m in lb.metadata['buffers']}
    edge = (1 << 32) // (4 * K)
    rows = np.r_[0:3, edge - 10:edge + 10, M - 20:M]
    assert M * K < 1 << 31 and M * K * 4 > 1 << 32 and rows[-21] * K * 4 > 1 << 32 > edge * K * 4
    x, g = rng.standard_normal((len(rows), K)).astype(np.float32), (rng.random(K) + 0.5).astype(np.float32)
    t['x'][torch.from_numpy(rows).cuda()], t['g'][0] = torch.from_numpy(x).cuda(), torch.from_numpy(g).cuda()
    torch.cuda.synchronize()
    res, _ = executor.run_noalloc(lb, [t[m['name']].data_ptr() for m in lb.metadata['buffers']], [0])
    assert res['rc'] == 0 and res['err_code'] == 0, res
    q, s = f64.quantise(f64.shaped(x, 1, None, g, 1e-6))
    at = torch.from_numpy(rows).cuda()
    np.testing.assert_array_equal(t['ys'][at, 0].cpu().numpy(), s)
    np.testing.assert_array_equal(t['y'][at].cpu().numpy().view(np.int8)[:, :K], q)
    other = torch.ones(M, dtype=torch.bool, device='cuda')
    other[at] = False
    assert not t['y'][other].any() and not t['ys'][other].any()


@pytest.mark.parametrize('tasks', [1, 5, 64])
@pytest.mark.parametrize('case', [mg.ATTENDS[i] for i in (1, 2, 3, 5, 7, 9)], ids=str)
def test_attend_large_scores(case, tasks):
    """A score is off by d = 2 (hd + 4) steps of the sum of its products' magnitudes, a weight against the largest one's by a factor within
    e^(4 d) at most, which moves a result by that much of the others' weights times the values' distance; where one weight is all, it is that value."""
    print(f'large scores {case} {tasks}', flush=True)
    page, hd, hkv, heads, dt = case[:5]
    scale = 50.0
    (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(6), scale=scale, tasks=tasks)
    ex = Executor.from_bundle(lb, buffers=init)
    ex.run()
    got = ex.read('o').reshape(q.shape)
    ex.close()
    kc, vc, table, lens, cu = pg
    want, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for r, b, i in zip(*f64.owners(cu, len(q))):
        t = np.arange(lens[b] + i + 1)
        for h in range(heads):
            k, v = (x[table[b, t // page], h * hkv // heads, t % page].astype(np.float64) for x in (kc, vc))
            x = q[r, h].astype(np.float64)
            s = k @ x * scale
            d = 2 * (hd + 4) * f64.U * (np.abs(k) @ np.abs(x)).max() * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            top = p.argmax()
            want[r, h] = p @ v
            others = np.delete(p, top) @ np.abs(np.delete(v, top, 0) - v[top])
            bound[r, h] = np.expm1(4 * d) * others + (2.0 ** -16 + (len(t) + 64) * 2 * f64.U) * (p @ np.abs(v))
    on = ~np.isnan(want)
    f64.near(got[on], want[on], bound[on], dt)
    # most rows are decided: one weight is all but 1, and its value comes out as the buffer's type has it
    sure = on & (bound < 1e-3 * np.abs(want))
    assert sure.mean() > 0.3
