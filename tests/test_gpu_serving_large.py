"""The serving operators at sizes whose byte offsets pass 32 bits, and with more sequences than one call of the
attention takes: buffers of the caller's on the GPU, compared where the large offsets lie."""
import numpy as np
import pytest
import torch

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import compiler, executor
from kvm_amd.workloads import Builder, serving

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 1: torch.int32, 2: torch.bfloat16}


def _buffers(b):
    lb = bl.load(compiler.compile_spec(b.spec()))
    return lb, {m['name']: torch.zeros((m['rows'], m['cols']), dtype=TORCH[m['dtype']], device='cuda') for m in lb.metadata['buffers']}


def _run(lb, t):
    torch.cuda.synchronize()
    res, _ = executor.run_noalloc(lb, [t[m['name']].data_ptr() for m in lb.metadata['buffers']], [0])
    assert res['rc'] == 0 and res['err_code'] == 0, res


@pytest.mark.parametrize('hd,kv,batch', [(128, 8, 5), (64, 16, 5), (100, 9, 5)])
def test_caches_of_more_than_4_gib(hd, kv, batch):
    """The last sequence of a cache with room for a million tokens a head: tokens appended over two blocks, then attended to."""
    print(f'large cache {hd} {kv} {batch}', flush=True)
    blk, tmax, L, n_new = 64, 1 << 20, 40, 5 if hd == 100 else 2
    steps = 100                                                        # appended as a prompt first
    rng = np.random.default_rng(11)
    b = Builder(0)
    c = serving.kv_q8_buffers(b, '', batch, kv, hd, tmax, blk, 'f32')
    b.fill('k', batch * steps, kv * hd), b.fill('v', batch * steps, kv * hd)
    b.fill('lens', batch, 1, 'i32'), b.fill('after', batch, 1, 'i32')
    b.fill('q', batch * n_new, 2 * kv * hd), b.fill('o', batch * n_new, 2 * kv * hd)
    ap = serving.kv_append_q8(b, c, 'k', 'v', 'lens', steps)
    serving.attn_decode_q8(b, c, 'q', 'o', 'after', 2 * kv, n_new, after=ap)
    lb, t = _buffers(b)
    assert t['kq'].numel() * 4 > 1 << 32 and batch * kv * tmax < 1 << 31
    k, v = (rng.standard_normal((steps, kv * hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((n_new, 2 * kv * hd)).astype(np.float32)
    tails = [rng.standard_normal((kv, blk, hd)).astype(np.float32) for _ in range(2)]
    t['lens'][:], t['after'][:] = -1, -1
    t['lens'][-1], t['after'][-1] = L, L + steps - n_new
    for n, x in (('k', k), ('v', v), ('q', q)):
        t[n][-len(x):] = torch.from_numpy(x).cuda()
    for n, x in (('kt', tails[0]), ('vt', tails[1])):
        t[n][-kv * blk:] = torch.from_numpy(x.reshape(-1, hd)).cuda()
    _run(lb, t)
    nblk = -(-(L + steps) // blk)
    start = f64.empty_cache(kv, nblk, blk, hd)
    start['kt'], start['vt'] = tails
    want = f64.append(start, k, v, [L], kv, steps, False)
    have = {}
    for x in 'kv':
        bytes_ = t[x + 'q'].view(torch.int8).reshape(batch * kv, tmax * hd)[-kv:, :nblk * blk * hd].cpu().numpy()
        have[x + 'q'] = bytes_.reshape(want[x + 'q'].shape)
        have[x + 's'] = t[x + 's'][-kv:, :nblk].cpu().numpy()
        have[x + 't'] = t[x + 't'][-kv * blk:].cpu().numpy().reshape(kv, blk, hd)
    for n in sg.CACHE:
        np.testing.assert_array_equal(have[n], want[n], err_msg=n)
    o, bound = f64.attend(want, q, [L + steps - n_new], kv, 2 * kv, n_new, np.float32(1 / np.sqrt(hd)))
    sg.near(t['o'][-n_new:].cpu().numpy(), o, bound, 'f32')
    assert not t['o'][:-n_new].any() and not t['kq'][:(batch - 1) * kv * tmax].any()


def test_logits_of_more_than_4_gib():
    print('large logits', flush=True)
    V, rows, H = 151936, 14134, 50
    rng = np.random.default_rng(12)
    b = Builder(0)
    b.fill('logits', rows, V), b.fill('out', rows, V), b.fill('par', rows, 3), b.fill('hist', rows, H, 'i32')
    b.fill('plen', rows, 1, 'i32'), b.fill('hlen', rows, 1, 'i32'), b.fill('last', rows, 1, 'i32')
    serving.logits_adjust(b, 'logits', 'out', 'par', rows, V, hist='hist', plen='plen', hlen='hlen', last='last')
    lb, t = _buffers(b)
    assert t['out'].numel() * 4 > 1 << 32
    x = rng.standard_normal((3, V)).astype(np.float32)
    g = dict(hist=rng.integers(0, V, (3, H)).astype(np.int32), plen=np.array([10, 0, 30], np.int32), hlen=np.array([40, 0, 49], np.int32),
             last=np.array([7, 150000, -1], np.int32))
    par = (rng.random((3, 3)) + 0.5).astype(np.float32)
    t['par'][:] = 1
    for n, y in (('logits', x), ('par', par), *((n, y.reshape(3, -1)) for n, y in g.items())):
        t[n][-3:] = torch.from_numpy(y).to(t[n].dtype).cuda()
    _run(lb, t)
    want, hist, bound = f64.adjust(x, par, **g)
    sg.near(t['out'][-3:].cpu().numpy(), want, bound, 'f32')
    np.testing.assert_array_equal(t['hist'][-3:].cpu().numpy(), hist)


def test_more_sequences_than_a_call():
    """1,500 sequences in two calls of the attention, which share counts but no partials."""
    print('1500 sequences', flush=True)
    case = (16, 64, 1, 2, 'f32', 1, [(53 * i) % 300 - 1 for i in range(1500)])
    blk, hd, kv, heads, dt, n_new, lens = case
    c, q = sg.attend_case(case)
    for tasks in (3, 200):
        lb, init = sg.attend_graph(c, q, lens, kv, heads, n_new, 0.1, dt, dt, tasks=tasks)
        ex = executor.Executor.from_bundle(lb, buffers=init)
        for _ in range(3):
            ex.relaunch()
            ex.finish()
        want, bound = f64.attend(c, q, lens, kv, heads, n_new, np.float32(0.1))
        sg.near(ex.read('o'), want, bound, dt)
        ex.close()
