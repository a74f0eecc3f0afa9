"""The weights of the attention over a paged bf16 cache (op 319): results differ from their definition in 64 bits by the rounding of the store and
what an f32 evaluation is off by, also where values cancel."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu


def _bound(q, pg, page, scale, mag):
    """A score is off by a step for each of its hd + 4 products, sums and factors, twice (the matrix units round sums towards zero), of the sum
    of its products' magnitudes; its weight by that, relatively, in numerator and denominator. A weight is held to 2^-16 (8 bits of bf16, then the
    nearest of what they leave), sums over n keys and the merge are off by 2 (n + 64) steps."""
    kc, _, table, lens, cu = pg
    H, hd, Hkv = q.shape[1], q.shape[2], kc.shape[1]
    rel = np.zeros((len(q), H, 1))
    for r, b, i in zip(*f64.owners(cu, len(q))):
        n = lens[b] + i + 1
        t = np.arange(n)
        for h in range(H):
            k = np.abs(kc[table[b, t // page], h * Hkv // H, t % page].astype(np.float64))
            sabs = (k @ np.abs(q[r, h].astype(np.float64))).max() * scale
            rel[r, h] = 2 * (hd + 4) * 2 * f64.U * sabs + 2.0 ** -16 + (n + 64) * 2 * f64.U
    return mag * rel


# single tokens, up to 32 rows, longer tiles (whole blocks of 64 keys and the edge), cut ones; (page, hd, kv heads, heads, lengths, new tokens)
CASES = [(16, 64, 2, 4, [19, 40], [1, 1]), (16, 64, 1, 4, [3, 20], [6, 1]), (32, 128, 1, 4, [5], [60]), (64, 64, 2, 2, [0, 9], [70, 40]), (16, 128, 2, 16, [12, 33], [1, 2]),
         (64, 128, 1, 8, [4000], [1]), (32, 64, 1, 2, [3000], [80])]


@pytest.mark.parametrize('tasks', [1, 64])
@pytest.mark.parametrize('case', CASES, ids=str)
def test_weights_are_not_rounded_to_bf16(case, tasks):
    print(f'weights {case} {tasks}', flush=True)
    page, hd, hkv, heads, lens, new = case
    rng = np.random.default_rng(5)
    (lb, init), pg, q = mg.attend_graph((page, hd, hkv, heads, 'bf16', lens, new), rng, tasks=tasks, n_max=max(new),
                                        q=lambda rows: mg.bf(0.5 * rng.standard_normal((rows, heads, hd)), 'bf16'))
    ex = Executor.from_bundle(lb, buffers=init, path=PATH_STATIC if tasks == 1 else PATH_DYNAMIC)
    ex.run()
    got = ex.read('o').reshape(q.shape)
    ex.close()
    want, mag = f64.attend(q, *pg, page, 1 / np.sqrt(hd))
    on = ~np.isnan(want)
    f64.near(got[on], want[on], _bound(q, pg, page, 1 / np.sqrt(hd), mag)[on], 'bf16')
    assert (got[~on] == 7).all()
