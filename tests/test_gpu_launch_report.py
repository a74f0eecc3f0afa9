"""Untraced static launches, which report themselves: results, counts, times and errors of launches one after the other, collected
one by one or several at once, and with traced launches between."""
import numpy as np
import pytest

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd import executor
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import Builder

pytestmark = pytest.mark.gpu


def _graph():
    rng = np.random.default_rng(1)
    c = f64.empty_cache(6, 2, 64, 128)
    k, v = (rng.standard_normal((3, 256)).astype(np.float32) for _ in range(2))
    lb, init = sg.append_graph(c, k, v, [0, 1, 2], 2, 1, 'f32', 'f32')
    return c, k, v, lb, init


@pytest.mark.parametrize('trace', [False, True])
def test_an_error_between_launches(trace):
    """A launch that fails says which task and why; the next one starts clean."""
    print(f'report trace {trace}', flush=True)
    c, k, v, lb, init = _graph()
    ex = Executor.from_bundle(lb, buffers=init, path=PATH_STATIC, trace=trace)
    want = c
    for step in range(4):
        lens = [5 * step, 1 + step, 2]
        for bad in (None, 128, None):
            ex.write('lens', np.array([lens[0], bad or lens[1], lens[2]], np.int32))
            ex.relaunch()
            res = ex.finish(check=False)
            if bad:
                assert res['err'] == 'OP_KVLEN' and (res['err_a'], res['err_b']) == (1, 128)
                assert 0 <= res['err_slot'] < lb.ntasks and res['done'] <= lb.ntasks
            else:
                assert res['err_code'] == 0 and res['done'] == lb.ntasks and 0 < res['kernel_ms'] < 50
        want = f64.append(want, k, v, lens, 2, 1, False)
    got = sg.cache_of(ex.read, c)
    for n in sg.CACHE:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    ex.close()


def test_launches_collected_at_once_and_traced_between():
    print('report several', flush=True)
    c, k, v, lb, init = _graph()
    ex = Executor.from_bundle(lb, buffers=init, path=PATH_STATIC, trace=True)
    for traced, launches in ((False, 5), (True, 1), (False, 1), (False, 3), (True, 2), (False, 2)):
        ex.set_trace(traced)
        for _ in range(launches):
            ex.relaunch()
        res = ex.finish()
        assert res['done'] == lb.ntasks and res['kernel_ms'] > 0
        assert ex.finish() == res                                   # collected again: the same
        if traced:
            assert (ex.trace()['exec_count'] == 1).all()
    assert ex.run_timed(7) > 0 and ex.finish()['done'] == lb.ntasks
    want = f64.append(c, k, v, [0, 1, 2], 2, 1, False)
    got = sg.cache_of(ex.read, c)
    for n in sg.CACHE:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)
    ex.close()


@pytest.mark.parametrize('trace', [False, True])
def test_the_time_of_a_launch(trace):
    """A launch whose only task waits for 20 ms: its time is that, by the report's clock and by events."""
    print(f'report time trace {trace}', flush=True)
    b = Builder(0)
    b.task('spin', us=20000)
    lb, init = sg.compiled(b, {})
    ex = Executor.from_bundle(lb, buffers=init, path=PATH_STATIC, trace=trace)
    ex.run()
    for _ in range(3):
        ex.relaunch()
        assert 20 <= ex.finish()['kernel_ms'] < 25
    ex.close()


@pytest.mark.parametrize('path,trace', [(PATH_STATIC, False), (PATH_STATIC, True), (PATH_DYNAMIC, False)])
def test_an_error_of_another_call_is_not_the_launchs(path, trace):
    """A HIP call of the program that fails between a launch and its collection (a device number that is not there) leaves its error with
    the thread; the launch is collected all the same."""
    print(f'report foreign error path {path} trace {trace}', flush=True)
    c, k, v, lb, init = _graph()
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=trace)
    L = executor.lib()
    ex.relaunch()
    assert L.hipSetDevice(1 << 20) != 0
    res = ex.finish(check=False)
    assert res['err_code'] == 0 and res['done'] == lb.ntasks
    L.hipGetLastError()                                                # the program takes its error
    ex.relaunch()
    assert ex.finish()['done'] == lb.ntasks
    ex.close()


@pytest.mark.parametrize('path,trace', [(PATH_STATIC, True), (PATH_DYNAMIC, False)])
def test_every_launch_between_events_has_a_time(path, trace):
    print(f'report event times path {path} trace {trace}', flush=True)
    c, k, v, lb, init = _graph()
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=trace)
    ex.run()
    for _ in range(500):
        ex.relaunch()
        assert 0 < ex.finish()['kernel_ms'] < 50
    ms = ex.run_timed(20)                                              # its events hold 20 launches
    assert ms > 0 and abs(ex.finish()['kernel_ms'] - ms) < 1e-3
    ex.close()
