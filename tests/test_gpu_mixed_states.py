"""The operators 315-319 where a launch or a size is out of the ordinary: launches that an error stopped in the middle of an attention, buffers
of the caller's, byte offsets past 32 bits, as many sequences as a call takes."""
import numpy as np
import pytest
import torch

import mixed_fp64 as f64
import mixed_graphs as mg
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import compiler, executor
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import Builder, serving

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 1: torch.int32, 2: torch.bfloat16}


def _stopped(first, new, S=16):
    """An attention over 6,000 tokens in `S` tasks: `first` of them, then an append that fails if its length (`stop`) is past its
    table, then the others."""
    rng = np.random.default_rng(2)
    pg = mg.paged(rng, [6000 + new], [0], 64, 2, 128, 'bf16')
    b, data = Builder(0), {}
    c = mg.add_paged(b, data, *pg[:3], np.array([6000], np.int32), np.array([0, new], np.int32), 64, 'bf16')
    sg.add(b, data, 'q', mg.bf(rng.standard_normal((new, 4 * 128)), 'bf16'), 'bf16')
    b.fill('o', new, 4 * 128, 'bf16')
    sg.add(b, data, 'stop', np.zeros((1, 1), np.int32)), sg.add(b, data, 'own.cu', np.array([[0], [1]], np.int32)), sg.add(b, data, 'own.table', np.zeros((1, 1), np.int32))
    own = serving.paged_buffers(b, 'own.', 1, 1, 64, 16, 'f32')
    b.fill('row', 1, 64)
    serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', 4, tasks=S)
    tasks, b.tasks = b.tasks, []
    before = [b.task(t['op'], **t['args']) for t in tasks[:first]]
    stop = serving.qkv_append_paged(b, own, 'row', 'row', 'own.table', 'stop', 'own.cu', after=before)
    for t in tasks[first:]:
        b.task(t['op'], after=stop, **t['args'])
    return sg.compiled(b, data)


def _fresh(lb, init, q):
    ex = Executor.from_bundle(lb, buffers=init)
    ex.write('q', q)
    ex.run()
    o = ex.read('o')
    ex.close()
    return o


@pytest.mark.parametrize('path,trace', [(PATH_STATIC, False), (PATH_STATIC, True), (PATH_DYNAMIC, False)])
@pytest.mark.parametrize('first,new', [(1, 1), (9, 1), (5, 60)])
def test_after_a_stopped_launch(first, new, path, trace):
    print(f'stopped {first} {new} path {path} trace {trace}', flush=True)
    lb, init = _stopped(first, new)
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=trace)
    ex.run()
    assert not ex.read('o.cnt').any()
    rng = np.random.default_rng(8)
    for collect in (True, False, True):
        ex.write('stop', np.array([99], np.int32))
        ex.relaunch()
        if collect:
            assert ex.finish(check=False)['err'] == 'OP_KVLEN'
        q = mg.bf(rng.standard_normal(new * 4 * 128), 'bf16')
        ex.write('stop', np.array([0], np.int32)), ex.write('q', q)
        want = _fresh(lb, init, q)
        for _ in range(2):
            ex.relaunch()
            assert ex.finish()['done'] == lb.ntasks
            np.testing.assert_array_equal(ex.read('o'), want)
            assert not ex.read('o.cnt').any()
    ex.close()


def test_after_a_stopped_call_on_own_buffers():
    print('stopped noalloc', flush=True)
    lb, init = _stopped(9, 1)
    ex = Executor.from_bundle(lb, buffers=init, trace=False)
    ptrs = [ex.device_ptr(n) for n in sg.names(lb)]
    rng = np.random.default_rng(8)
    for bad in (99, 0, 99, 0, 0):
        q = mg.bf(rng.standard_normal(4 * 128), 'bf16')
        ex.write('stop', np.array([bad], np.int32)), ex.write('q', q)
        res, _ = executor.run_noalloc(lb, ptrs, [0])
        assert (res['rc'] != 0) == bool(bad), res
        assert not ex.read('o.cnt').any()
        if not bad:
            np.testing.assert_array_equal(ex.read('o'), _fresh(lb, init, q))
    ex.close()


@pytest.mark.parametrize('path', [PATH_STATIC, PATH_DYNAMIC])
@pytest.mark.parametrize('M', [1, 5, 40])
def test_weights_of_the_same_graph(M, path):
    """Weights that a task in front brings to 8 bits are not read before it has, launch after launch."""
    print(f'weights of the same graph {M} path {path}', flush=True)
    N, K = 500, 1040
    rng = np.random.default_rng(6)
    b, data = Builder(0), {}
    sg.add(b, data, 'x', rng.standard_normal((M, K)).astype(np.float32)), sg.add(b, data, 'raw', np.zeros((N, K), np.float32))
    w = serving.weight_q8_buffers(b, 'w', N, K)
    b.fill('out', M, N)
    serving.linear_q8(b, 'x', w, 'out', M, after=serving.rows_q8(b, 'raw', w, N))
    lb, init = sg.compiled(b, data)
    ex = Executor.from_bundle(lb, buffers=init, path=path)
    x = f64.quantise(data['x'])
    for _ in range(4):
        raw = rng.standard_normal((N, K)).astype(np.float32)
        ex.write('raw', raw)
        ex.relaunch()
        ex.finish()
        want, bound = f64.product(*x, *f64.quantise(raw))
        f64.near(ex.read('out').reshape(M, N), want, bound, 'f32')
    ex.close()


def _buffers(b):
    lb = bl.load(compiler.compile_spec(b.spec()))
    return lb, {m['name']: torch.zeros((m['rows'], m['cols']), dtype=TORCH[m['dtype']], device='cuda') for m in lb.metadata['buffers']}


def _run(lb, t):
    torch.cuda.synchronize()
    res, _ = executor.run_noalloc(lb, [t[m['name']].data_ptr() for m in lb.metadata['buffers']], [0])
    assert res['rc'] == 0 and res['err_code'] == 0, res


@pytest.mark.parametrize('page,hd,hkv,heads,dt,new', [(128, 128, 8, 16, 'bf16', 3), (128, 128, 8, 8, 'bf16', 130), (64, 64, 8, 16, 'f32', 3), (128, 100, 8, 8, 'f32', 2)])
def test_large_caches(page, hd, hkv, heads, dt, new):
    """The last pages of a cache, tokens appended over two of them, then attended to: more than 4 GiB of f32, and the most elements that a
    buffer has (below 2^31) of bf16."""
    print(f'large cache {page} {hd} {dt} {new}', flush=True)
    size = hkv * page * hd * (2 if dt == 'bf16' else 4)
    pages, had = ((1 << 32) // size + 40 if dt == 'f32' else ((1 << 31) - 1) // (size // 2)), 2 * page - 1
    rng = np.random.default_rng(11)
    b = Builder(0)
    c = serving.paged_buffers(b, '', pages, hkv, hd, page, dt)
    for n, h in (('k', hkv), ('v', hkv), ('q', heads), ('o', heads)):
        b.fill(n, new, h * hd, dt)
    b.fill('table', 1, 8, 'i32'), b.fill('lens', 1, 1, 'i32'), b.fill('cu', 2, 1, 'i32')
    ap = serving.qkv_append_paged(b, c, 'k', 'v', 'table', 'lens', 'cu')
    serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', heads, after=ap)
    lb, t = _buffers(b)
    assert t['kc'].numel() * t['kc'].element_size() > (1 << 32 if dt == 'f32' else 4 * (1 << 30) - (1 << 21))
    k, v, q = (mg.bf(rng.standard_normal((new, h, hd)), dt) for h in (hkv, hkv, heads))
    table = (pages - 1 - rng.permutation(8)).astype(np.int32)[None]
    old = [mg.bf(rng.standard_normal((8, hkv, page, hd)), dt) for _ in range(2)]
    at = lambda n: t[n].view(pages, hkv, page, hd)[pages - 8:]          # noqa: E731
    for n, x in zip(('kc', 'vc'), old):
        at(n)[:] = torch.from_numpy(x).cuda()
    for n, x in (('k', k), ('v', v), ('q', q)):
        t[n][:] = torch.from_numpy(x.reshape(new, -1)).cuda()
    t['table'][:] = torch.from_numpy(table).cuda()
    t['lens'][:], t['cu'][1] = had, new
    _run(lb, t)
    lens, cu, near = np.array([had]), np.array([0, new]), table - (pages - 8)
    kc, vc, _ = f64.append(*old, near, lens, cu, None, k, v, page, None, None, 0, 0)
    for n, x in (('kc', kc), ('vc', vc)):
        np.testing.assert_array_equal(at(n).float().cpu().numpy(), x)
        assert not t[n].view(pages, hkv, page, hd)[:pages - 8].any()
    want, mag = f64.attend(q, kc, vc, near, lens, cu, page, 1 / np.sqrt(hd))
    big = np.abs(q).sum(-1).max() * np.abs(kc).max()
    bound = mg.attend_bound((page, hd, hkv, heads, dt, lens, [new]), mag, big / np.sqrt(hd), dt == 'f32')
    f64.near(t['o'].float().cpu().numpy().reshape(want.shape), want, bound, dt)


@pytest.mark.parametrize('M', [1, 9, 100])
def test_weights_of_more_than_4_gib(M):
    """Outputs of the last rows of weights whose bytes lie past 4 GiB, and of ones that lie in front."""
    print(f'large weights {M}', flush=True)
    N, K = (1 << 32) // 4096 + 200, 4096
    rng = np.random.default_rng(13)
    b = Builder(0)
    b.fill('x', M, K, 'bf16'), b.fill('out', M, N)
    w = serving.weight_q8_buffers(b, 'w', N, K)
    serving.linear_q8(b, 'x', w, 'out', M, tasks=256)
    lb, t = _buffers(b)
    x = mg.bf(rng.standard_normal((M, K)), 'bf16')
    t['x'][:] = torch.from_numpy(x).cuda()
    rows = np.r_[0:50, N - 333:N]
    q, s = rng.integers(-127, 128, (len(rows), K)).astype(np.int8), rng.random(len(rows)).astype(np.float32)
    t['w'][torch.from_numpy(rows).cuda()], t['ws'][torch.from_numpy(rows).cuda(), 0] = torch.from_numpy(q.view(np.int32)).cuda(), torch.from_numpy(s).cuda()
    _run(lb, t)
    want, bound = f64.product(*f64.quantise(x), q, s)
    f64.near(t['out'][:, torch.from_numpy(rows).cuda()].cpu().numpy(), want, bound, 'f32')
    assert not t['out'][:, 50:N - 333].any()


def test_rows_of_more_than_4_gib():
    print('large rows', flush=True)
    K, M = 12296, 174600
    rng = np.random.default_rng(14)
    b = Builder(0)
    b.fill('x', M, K, 'bf16'), b.fill('g', 1, K), b.fill('out', M, 64)
    y = serving.rows_q8_buffers(b, 'y', M, K)
    w = serving.weight_q8_buffers(b, 'w', 64, K)
    at = serving.rows_q8(b, 'x', y, M, gamma='g', eps=1e-6)
    b.task('matmul_q8', after=at, a='y', sa='ys', w='w', sw='ws', out='out', bias=None, res=None, m0=M - 64, n0=0, M=M, N=64, K=K, tile=2)
    lb, t = _buffers(b)
    assert t['x'].numel() * 2 > (1 << 32) - (1 << 21)
    x, g = mg.bf(rng.standard_normal((40, K)), 'bf16'), (rng.random(K) + 0.5).astype(np.float32)
    wq, ws = rng.integers(-127, 128, (64, K)).astype(np.int8), rng.random(64).astype(np.float32)
    t['x'][-40:], t['g'][0] = torch.from_numpy(x).cuda(), torch.from_numpy(g).cuda()
    t['w'][:], t['ws'][:, 0] = torch.from_numpy(np.pad(wq, ((0, 0), (0, -K % 16))).view(np.int32)).cuda(), torch.from_numpy(ws).cuda()
    _run(lb, t)
    q, s = f64.quantise(f64.shaped(x, 1, None, g, 1e-6))
    have = t['y'][-40:].cpu().numpy().view(np.int8)[:, :K], t['ys'][-40:, 0].cpu().numpy()
    assert np.abs(have[0].astype(int) - q).max() <= 1 and (np.abs(have[1] - s) <= 2.0 ** -21 * s).all()
    want, bound = f64.product(*have, wq, ws)
    f64.near(t['out'][-40:].cpu().numpy(), want, bound, 'f32')
    assert not t['out'][:-40].any()


@pytest.mark.parametrize('tasks', [3, 256])
def test_1024_sequences(tasks):
    """As many sequences as a call takes, many of them without a token or with their first one."""
    print(f'1024 sequences {tasks}', flush=True)
    lens, new = [(53 * i) % 300 for i in range(1024)], [(0, 1, 1, 3)[i % 4] for i in range(1024)]
    for i in range(0, 1024, 5):
        lens[i] = 0
    case = (16, 64, 1, 2, 'bf16', lens, new)
    (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(3), tasks=tasks)
    want, mag = f64.attend(q, *pg, 16, 1 / np.sqrt(64))
    on = ~np.isnan(want)
    bound = mg.attend_bound(case, mag, np.abs(q).sum(-1).max() * np.nanmax(np.abs(pg[0])) / 8, False)
    ex = Executor.from_bundle(lb, buffers=init)
    for _ in range(3):
        ex.relaunch()
        ex.finish()
    o = ex.read('o').reshape(want.shape)
    f64.near(o[on], want[on], bound[on], 'bf16')
    assert (o[~on] == 7).all()
    ex.close()
