"""Rows of op 317 that do not fit into LDS are taken in the fewest parts of K that do: the rule, compiled alone, and products over K whose number of
steps has no divisors, bit for bit those of the tiles."""
import subprocess

import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import serving_graphs as sg
from kvm_amd import build as kb


def test_fewest_parts(tmp_path):
    """All parts fit, one part fewer would not, no part is behind K."""
    (tmp_path / 'a.cpp').write_text('''#include "gemv_q8_geo.h"
#include <cstdio>
int main() {
  for (int steps = 1; steps <= 256; ++steps)
    for (int bytes = 512; bytes <= 16 * 512; bytes += 512)
      for (int room = 16 * 512; room <= 131072; room += 1234) {
        const int c = kvm::gq_part_steps(steps, bytes, room), parts = (steps + c - 1) / c;
        const bool alone = parts == 1 || (long)((steps + parts - 2) / (parts - 1)) * bytes > room;
        if (c < 1 || c > steps || (long)c * bytes > room || !alone || c * parts - steps >= parts) { std::printf("%d %d %d: %d\\n", steps, bytes, room, c); return 1; }
      }
  return 0;
}''')
    subprocess.run([kb.CXX, '-std=c++17', '-O1', f'-I{kb.CSRC}', str(tmp_path / 'a.cpp'), '-o', str(tmp_path / 'a')], check=True)
    r = subprocess.run([str(tmp_path / 'a')], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


# as mixed_graphs.GEMVS: (M, N, K, words of a weight row, dtype, pro, bias, res, columns of x); 17, 13, 23, 37, 19 and 41 steps of 512 bytes
CASES = [(16, 40, 8704, 2176, 'bf16', 2, False, True, 8704), (16, 150, 6201, 1552, 'bf16', 0, True, False, 6208), (4, 50, 11776, 2944, 'f32', 1, False, False, 11776),
         (8, 37, 18943, 4740, 'bf16', 1, False, False, 18944), (13, 20, 9728, 2433, 'f32', 0, False, False, 9728), (9, 33, 20740, 5188, 'bf16', 0, False, False, 20744)]


@pytest.mark.gpu
@pytest.mark.parametrize('case', CASES, ids=str)
def test_uneven_parts(case):
    print(f'gemv parts {case}', flush=True)
    from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
    args = mg.gemv_case(case)
    want = None
    for fused, path in ((None, PATH_DYNAMIC), (True, PATH_DYNAMIC), (True, PATH_STATIC), (False, PATH_DYNAMIC), (False, PATH_STATIC)):
        lb, init = mg.gemv_graph(case, *args, fused=fused)
        ex = Executor.from_bundle(lb, buffers=init, path=path, trace=False)
        for _ in range(2):
            ex.relaunch()
            ex.finish()
        got = {n: ex.read(n) for n in sg.names(lb)}
        ex.close()
        if want is None:
            want = got['out']
            exact, bound = f64.product(got['y'].view(np.int8).reshape(case[0], -1)[:, :case[2]], got['ys'], *args[3:])
            f64.near(want.reshape(exact.shape), exact, bound, case[4])
        np.testing.assert_array_equal(got['out'], want, err_msg=f'{fused} {path}')
