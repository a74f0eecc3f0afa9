"""Ops 315-319 with operands of different storage in one call: SwiGLU rows of two types, residuals of another type than the outputs, new tokens of another type
than the cache, keys and values of two. Held to the definitions in 64 bits as where all are of one type."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import serving_graphs as sg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import Builder, serving

pytestmark = pytest.mark.gpu

TWO = [('bf16', 'f32'), ('f32', 'bf16')]


def _run(lb, init, path=PATH_DYNAMIC):
    ex = Executor.from_bundle(lb, buffers=init, path=path)
    for _ in range(2):
        ex.relaunch()
        ex.finish()
    got = {n: ex.read(n) for n in sg.names(lb)}
    ex.close()
    return got


# (rows, K): fewer than a vector, ragged, a row of the form in registers, a longer one, one that the one-type forms read three times
@pytest.mark.parametrize('types', TWO, ids=str)
@pytest.mark.parametrize('M,K', [(1, 5), (3, 777), (9, 4096), (2, 12288), (2, 20001)])
def test_swiglu_rows(M, K, types):
    """v is off by some steps of 2^-24 (an exponential, a reciprocal, two products: below 2^-20 of it), its byte by that and a half."""
    print(f'rows {M} {K} {types}', flush=True)
    rng = np.random.default_rng([M, K])
    x, x2 = (mg.bf(rng.standard_normal((M, K)), t) for t in types)
    b, data = Builder(0), {}
    sg.add(b, data, 'x', x, types[0]), sg.add(b, data, 'x2', x2, types[1])
    y = serving.rows_q8_buffers(b, 'y', M, K)
    serving.rows_q8(b, 'x', y, M, x2='x2')
    got = _run(*sg.compiled(b, data))
    v = f64.shaped(x, 2, x2)
    _, s = f64.quantise(v)
    q = got['y'].view(np.int8).reshape(M, -1)
    assert (np.abs(got['ys'] - s) <= 2.0 ** -20 * s).all()
    assert (np.abs(q[:, :K] - v / got['ys'][:, None]) <= 0.5 + 127 * 2.0 ** -19).all()
    assert not q[:, K:].any()


@pytest.mark.parametrize('types', TWO, ids=str)
@pytest.mark.parametrize('M,N,K', [(1, 40, 777), (5, 70, 4096), (16, 33, 12288), (3, 20, 20001)])
def test_swiglu_inside_the_product(M, N, K, types):
    """Bit for bit rows_q8 and the tiles, on both paths, with a residual of the other type than the outputs."""
    print(f'gemv {M} {N} {K} {types}', flush=True)
    rng = np.random.default_rng([M, N, K])
    x, x2, res = mg.bf(rng.standard_normal((M, K)), types[0]), mg.bf(rng.standard_normal((M, K)), types[1]), mg.bf(rng.standard_normal((M, N)), types[1])
    w, sw = rng.integers(-127, 128, (N, K)).astype(np.int8), (rng.random(N) - 0.5).astype(np.float32) / K
    b, data = Builder(0), {}
    for n, y, t in (('x', x, types[0]), ('x2', x2, types[1]), ('res', res, types[1]), ('w', mg.words(w, 4 * -(-K // 16)), None), ('sw', sw[:, None], None)):
        sg.add(b, data, n, y, t)
    b.fill('one', M, N, types[0]), b.fill('two', M, N, types[0])
    b.task('gemv_q8', x='x', x2='x2', gamma=None, w='w', sw='sw', out='one', bias=None, res='res', sx=None, n0=0, n1=N, K=K, M=M, pro=2, eps=0.0)
    y = serving.rows_q8_buffers(b, 'y', M, K)
    t = serving.rows_q8(b, 'x', y, M, x2='x2')
    for n0 in range(0, N, 64):
        b.task('matmul_q8', after=t, a='y', sa='ys', w='w', sw='sw', out='two', bias=None, res='res', m0=0, n0=n0, M=M, N=N, K=K, tile=2)
    lb, init = sg.compiled(b, data)
    for path in (PATH_DYNAMIC, PATH_STATIC):
        got = _run(lb, init, path)
        np.testing.assert_array_equal(got['one'], got['two'])
        want, bound = f64.product(got['y'].view(np.int8).reshape(M, -1)[:, :K], got['ys'], w, sw, None, res)
        f64.near(got['one'].reshape(M, N), want, bound, types[0])


@pytest.mark.parametrize('tile', [0, 1, 2])
@pytest.mark.parametrize('types', TWO, ids=str)
@pytest.mark.parametrize('M,N', [(130, 256), (65, 70)])                # whole vectors and elements on the way out
def test_residuals_of_another_type(M, N, types, tile):
    print(f'product {M} {N} {types} {tile}', flush=True)
    case = (M, N, 200, 52, types[0], True, True)
    a, sa, w, sw, bias, _ = mg.product_case(case)
    res = mg.bf(np.random.default_rng(M).standard_normal((M, N)), types[1])
    b, data = Builder(0), {}
    for n, x, t in (('a', mg.words(a, 52), None), ('sa', sa[:, None], None), ('w', mg.words(w, 52), None), ('sw', sw[:, None], None), ('bias', bias[None], None), ('res', res, types[1])):
        sg.add(b, data, n, x, t)
    b.fill('out', M, N, types[0])
    tm, tn = ((128, 256), (128, 128), (64, 64))[tile]
    for m0 in range(0, M, tm):
        for n0 in range(0, N, tn):
            b.task('matmul_q8', a='a', sa='sa', w='w', sw='sw', out='out', bias='bias', res='res', m0=m0, n0=n0, M=M, N=N, K=200, tile=tile)
    want, bound = f64.product(a, sa, w, sw, bias, res)
    f64.near(_run(*sg.compiled(b, data))['out'].reshape(M, N), want, bound, types[0])


# types of (queries, keys and values that come, cache of keys, of values)
MIXES = [('f32', 'f32', 'bf16', 'bf16'), ('bf16', 'bf16', 'f32', 'f32'), ('f32', 'bf16', 'bf16', 'bf16'), ('bf16', 'f32', 'f32', 'bf16'), ('bf16', 'bf16', 'bf16', 'f32')]


def _cache(b, data, pg, page, ktype, vtype):
    kc, vc, table, lens, cu = pg
    pages, hkv, _, hd = kc.shape
    c = serving.paged_buffers(b, '', pages, hkv, hd, page, ktype)
    next(d for d in b.buffers if d['name'] == 'vc')['dtype'] = vtype
    data['kc'], data['vc'] = kc.reshape(-1, hd), vc.reshape(-1, hd)
    sg.add(b, data, 'table', table), sg.add(b, data, 'lens', lens[:, None]), sg.add(b, data, 'cu', cu[:, None])
    return c


@pytest.mark.parametrize('types', MIXES, ids=str)
@pytest.mark.parametrize('page,hd,hkv,heads,lens,new', [(16, 64, 2, 4, [0, 15, 100], [1, 40, 3]), (64, 128, 1, 3, [63, 200], [70, 2]), (32, 100, 2, 2, [31], [40])], ids=str)
def test_append_to_a_cache_of_another_type(page, hd, hkv, heads, lens, new, types):
    """A key is off by some steps of 2^-24 of its magnitudes (norm: 4, angle: pi 2^-24 absolute and 1, products: 2, below 2^-20 with the other
    half's part), then rounded to what holds it."""
    print(f'append {page} {hd} {types}', flush=True)
    qt, nt, kt, vt = types
    rng = np.random.default_rng([page, hd])
    pg = mg.paged(rng, lens, new, page, hkv, hd, 'bf16', unseen=7.0)
    rows = int(pg[4][-1]) + 2
    q, k, v = (mg.bf(rng.standard_normal((rows, h, hd)), t) for h, t in ((heads, qt), (hkv, nt), (hkv, nt)))
    gs = [(rng.random(hd) + 0.5).astype(np.float32) for _ in range(2)]
    b, data = Builder(0), {}
    c = _cache(b, data, pg, page, kt, vt)
    for n, x, t in (('q', q, qt), ('k', k, nt), ('v', v, nt)):
        sg.add(b, data, n, x.reshape(rows, -1), t)
    sg.add(b, data, 'qg', gs[0][None]), sg.add(b, data, 'kg', gs[1][None])
    b.fill('qo', rows, heads * hd, kt, value=7.0)
    serving.qkv_append_paged(b, c, 'k', 'v', 'table', 'lens', 'cu', q='q', qo='qo', heads=heads, qgamma='qg', kgamma='kg', theta=1e6, eps=1e-6)
    got = _run(*sg.compiled(b, data))
    want = f64.append(*pg, q, k, v, page, *gs, 1e-6, 1e6)
    big = max(np.abs(x[np.isfinite(x)]).max() for x in want)
    f64.near(got['kc'].reshape(want[0].shape), want[0], 2.0 ** -20 * big, kt)
    f64.near(got['vc'].reshape(want[1].shape), want[1], 0, vt)
    on, o = ~np.isnan(want[2]), got['qo'].reshape(want[2].shape)
    f64.near(o[on], want[2][on], 2.0 ** -20 * big, kt)
    assert (o[~on] == 7).all()


@pytest.mark.parametrize('tasks', [1, 64])
@pytest.mark.parametrize('types', [('f32', 'bf16', 'bf16'), ('bf16', 'f32', 'f32'), ('bf16', 'bf16', 'f32'), ('f32', 'f32', 'bf16')], ids=str)
@pytest.mark.parametrize('page,hd,hkv,heads,lens,new', [(16, 64, 2, 4, [0, 15, 2500], [1, 40, 3]), (64, 128, 1, 8, [63, 700], [1, 2]), (32, 100, 1, 2, [31], [40])], ids=str)
def test_attend_over_a_cache_of_another_type(page, hd, hkv, heads, lens, new, types, tasks):
    """Weights stay in 32 bits here: the bound of f32 storage, rounded to the outputs' type."""
    print(f'attend {page} {hd} {types} {tasks}', flush=True)
    qt, kt, vt = types
    rng = np.random.default_rng([page, hd])
    pg = mg.paged(rng, np.asarray(lens) + np.asarray(new), np.zeros(len(new), int), page, hkv, hd, 'bf16')
    pg = (*pg[:3], np.asarray(lens, np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    rows = int(pg[4][-1]) + 2
    q = mg.bf(rng.standard_normal((rows, heads, hd)), qt)
    b, data = Builder(0), {}
    c = _cache(b, data, pg, page, kt, vt)
    sg.add(b, data, 'q', q.reshape(rows, -1), qt)
    b.fill('o', rows, heads * hd, qt, value=7.0)
    serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', heads, tasks=tasks)
    o = _run(*sg.compiled(b, data))['o'].reshape(q.shape)
    want, mag = f64.attend(q, *pg, page, 1 / np.sqrt(hd))
    sabs = np.abs(q).sum(-1).max() * np.nanmax(np.abs(pg[0])) / np.sqrt(hd)
    on = ~np.isnan(want)
    f64.near(o[on], want[on], mg.attend_bound((page, hd, hkv, heads, qt, lens, new), mag, sabs, True)[on], qt)
    assert (o[~on] == 7).all()
