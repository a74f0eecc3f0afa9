"""A launch that an error stops in the middle of an attention whose pieces count themselves (ops 310, 313): the next launch counts
from 0 and gives what a fresh executor gives."""
import numpy as np
import pytest

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import executor
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import Builder, serving

pytestmark = pytest.mark.gpu


def _stopper(b, data, after):
    """A task that fails when the length in `stop` is out of range (an append to a cache of its own)."""
    c = sg.random_cache(np.random.default_rng(4), 1, 1, 16, 64, False)
    cache = serving.kv_q8_buffers(b, 'own.', 1, 1, 64, 16, 16, 'f32')
    for n in sg.CACHE:
        x = np.ascontiguousarray(c[n])
        data['own.' + n] = x.view(np.int32) if n[1] == 'q' else x
    sg.add(b, data, 'row', np.ones((1, 64), np.float32))
    sg.add(b, data, 'stop', np.zeros((1, 1), np.int32))
    return serving.kv_append_q8(b, cache, 'row', 'row', 'stop', after=after, tasks=1)


def _q8(first):
    """Two heads over 6,000 tokens in 16 tasks, about eight pieces each; `first` tasks, the stopper, then the others."""
    rng = np.random.default_rng(2)
    c = sg.random_cache(rng, 2, 95, 64, 128, False)
    b, data = Builder(0), {}
    cache = sg.add_cache(b, data, c, 2, 'f32')
    sg.add(b, data, 'q', rng.standard_normal((1, 4 * 128)).astype(np.float32))
    sg.add(b, data, 'lens', np.array([[6000]], np.int32))
    b.fill('o', 1, 4 * 128), b.fill('part', 2 * 16 * 2, 130), b.fill('cnt', 2, 1, 'i32')
    kw = dict(q='q', lens='lens', o='o', cnt='cnt', part='part', qgamma=None, b0=0, b1=1, S=16, n_new=1, H=4, scale=0.1, theta=0.0, eps=0.0, **cache.args())
    before = [b.task('attn_decode_q8', s=s, **kw) for s in range(first)]
    stop = _stopper(b, data, before)
    for s in range(first, 16):
        b.task('attn_decode_q8', after=stop, s=s, **kw)
    return sg.compiled(b, data)


def _merge(first):
    """Op 310: two kv heads of two query heads each, five splits."""
    rng = np.random.default_rng(3)
    B, Hkv, H, hd, S, T = 1, 2, 4, 128, 5, 701
    b, data = Builder(0), {}
    for n, shape, dt in (('q', (1, H * hd), 'f32'), ('kc', (Hkv * T, hd), 'bf16'), ('vc', (Hkv * T, hd), 'bf16'), ('kn', (1, Hkv * hd), 'f32'),
                         ('vn', (1, Hkv * hd), 'f32'), ('qg', (1, hd), 'f32'), ('kg', (1, hd), 'f32')):
        x = rng.standard_normal(shape).astype(np.float32)
        sg.add(b, data, n, bl.bf16_round(x) if dt == 'bf16' else x, dt)
    sg.add(b, data, 'lens', np.array([[700]], np.int32))
    b.fill('o', 1, H * hd), b.fill('part', S * H, hd + 2), b.fill('cnt', Hkv, 1, 'i32')
    kw = dict(q='q', kc='kc', vc='vc', lens='lens', part='part', knew='kn', vnew='vn', b=0, S=S, H=H, Hkv=Hkv, hd=hd, Tmax=T, scale=0.1, theta=1e6, flags=1,
              qgamma='qg', kgamma='kg', eps=0.25, o='o', cnt='cnt')
    before = [b.task('attn_decode_part_merge', kvh=h, s=s, **kw) for h in range(Hkv) for s in range(first)]
    stop = _stopper(b, data, before)
    for h in range(Hkv):
        for s in range(first, S):
            b.task('attn_decode_part_merge', after=stop, kvh=h, s=s, **kw)
    return sg.compiled(b, data)


def _fresh(lb, init, q):
    ex = Executor.from_bundle(lb, buffers=init)
    ex.write('q', q)
    ex.run()
    o = ex.read('o')
    ex.close()
    return o


@pytest.mark.parametrize('collect', [True, False])
@pytest.mark.parametrize('path,trace', [(PATH_STATIC, False), (PATH_STATIC, True), (PATH_DYNAMIC, False)])
@pytest.mark.parametrize('make,first', [(_q8, 1), (_q8, 9), (_merge, 3)])
def test_after_a_stopped_launch(make, first, path, trace, collect):
    print(f'stopped {make.__name__} {first} path {path} trace {trace} collect {collect}', flush=True)
    lb, init = make(first)
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=trace)
    ex.run()
    assert not ex.read('cnt').any()
    rng = np.random.default_rng(8)
    for _ in range(3):
        ex.write('stop', np.array([99], np.int32))
        ex.relaunch()
        if collect:
            assert ex.finish(check=False)['err'] == 'OP_KVLEN'
        q = rng.standard_normal(4 * 128).astype(np.float32)
        ex.write('stop', np.array([0], np.int32)), ex.write('q', q)
        want = _fresh(lb, init, q)
        for _ in range(2):
            ex.relaunch()
            assert ex.finish()['done'] == lb.ntasks
            np.testing.assert_array_equal(ex.read('o'), want)
            assert not ex.read('cnt').any()
    ex.close()


@pytest.mark.parametrize('make,first', [(_q8, 9), (_merge, 3)])
def test_after_a_stopped_call_on_own_buffers(make, first):
    print(f'stopped noalloc {make.__name__}', flush=True)
    lb, init = make(first)
    ex = Executor.from_bundle(lb, buffers=init, trace=False)
    ptrs = [ex.device_ptr(n) for n in sg.names(lb)]
    rng = np.random.default_rng(8)
    for bad in (99, 0, 99, 0, 0):
        q = rng.standard_normal(4 * 128).astype(np.float32)
        ex.write('stop', np.array([bad], np.int32)), ex.write('q', q)
        res, _ = executor.run_noalloc(lb, ptrs, [0])
        assert (res['rc'] != 0) == bool(bad), res
        assert not ex.read('cnt').any()
        if not bad:
            np.testing.assert_array_equal(ex.read('o'), _fresh(lb, init, q))
    ex.close()
