"""The operators that serve prompts and tokens together (ops 315-319) on the GPU against their definition in 64 bits: bytes and scales
exactly, products bit for bit between their forms, caches and attention within bounds that count roundings (mixed_fp64)."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import serving_graphs as sg
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu


def _run(lb, init, path=PATH_DYNAMIC, times=1):
    ex = Executor.from_bundle(lb, buffers=init, path=path, trace=False)
    for _ in range(times):
        ex.relaunch()
        ex.finish()
    got = {n: ex.read(n) for n in sg.names(lb)}
    ex.close()
    return got


def _error(lb, init):
    ex = Executor.from_bundle(lb, buffers=init)
    ex.start()
    res = ex.finish(check=False)
    got = {n: ex.read(n) for n in sg.names(lb)}
    ex.close()
    return res['err'], got


@pytest.mark.parametrize('tasks', [1, 256])
@pytest.mark.parametrize('case', mg.ROWS, ids=str)
def test_rows(case, tasks):
    """SwiGLU's v is off by some steps of 2^-24 of it (an exponential, a reciprocal, two products: below 2^-20), its byte by that and a half."""
    print(f'rows {case} tasks {tasks}', flush=True)
    M, K, pro, dt, cols = case
    x, x2, g = mg.rows_case(case)
    lb, init = mg.rows_graph(x, x2, g, dt, cols, K, tasks=tasks)
    got = _run(lb, init, PATH_STATIC if tasks == 1 else PATH_DYNAMIC)
    v = f64.shaped(x, pro, x2, g, 1e-6)
    q, s = f64.quantise(v)
    y = got['y'].view(np.int8).reshape(M, -1)
    if pro == 2:
        assert (np.abs(got['ys'] - s) <= 2.0 ** -20 * s).all()
        assert (np.abs(y[:, :K] - v / got['ys'][:, None]) <= 0.5 + 127 * 2.0 ** -19).all()
    else:
        np.testing.assert_array_equal(got['ys'], s)
        np.testing.assert_array_equal(y[:, :K], q)
    assert not y[:, K:].any()


@pytest.mark.parametrize('K,dtype', [(40, 'f32'), (41, 'f32'), (5000, 'bf16')])
def test_rows_that_are_not_finite_or_tiny(K, dtype):
    """NaN and infinities, zeros, magnitudes whose scale falls below the normal numbers, the largest ones; ties between two bytes. Narrow rows keep
    the words behind them."""
    print(f'rows special {K} {dtype}', flush=True)
    x = np.zeros((8, K), np.float32)
    x[1, 3] = np.nan
    x[2, K - 1], x[2, 0] = -np.inf, 5
    x[3, 7] = 1e-37
    x[4] = np.float32(3e38)
    x[5] = np.arange(K) % 255 - 127 + 0.5
    x[5, 0] = 127
    x[6] = -(np.arange(K) % 127) / 2
    x[6, 0] = 63.5
    x[7, 1] = 1e-30
    x = mg.bf(x, dtype)
    lb, init = mg.rows_graph(x, None, None, dtype, K, K)
    got = _run(lb, init)
    q, s = f64.quantise(x)
    np.testing.assert_array_equal(got['ys'], s)
    np.testing.assert_array_equal(got['y'].view(np.int8).reshape(8, -1)[:, :K], q)
    kw = -(-K // 4)
    lb, init = mg.rows_graph(x, None, None, dtype, K, K, width=kw + 9)
    y = _run(lb, init)['y'].view(np.int8).reshape(8, -1)
    np.testing.assert_array_equal(y[:, :K], q)
    end = min(4 * (kw + 9), -(-K // 16) * 16)
    assert not y[:, K:end].any() and (y[:, end:] == 0x4d).all()


@pytest.mark.parametrize('tile', [0, 1, 2])
@pytest.mark.parametrize('case', mg.PRODUCTS, ids=str)
def test_product(case, tile):
    print(f'product {case} tile {tile}', flush=True)
    args = mg.product_case(case)
    want, bound = f64.product(*args)
    lb, init = mg.product_graph(case, *args, tile)
    got = _run(lb, init)['out']
    f64.near(got.reshape(want.shape), want, bound, case[4])
    if args[-1] is not None:                                           # the residual in place
        lb, init = mg.product_graph(case, *args, tile, inplace=True)
        np.testing.assert_array_equal(_run(lb, init, PATH_STATIC)['res'], got)


@pytest.mark.parametrize('case', mg.GEMVS, ids=str)
def test_gemv_is_rows_then_product(case):
    """The same bits from the fused form (its first weights requested before the task waits, on the static path), from rows brought to 8 bits
    before, from tiles; within bounds of the definition."""
    print(f'gemv {case}', flush=True)
    args = mg.gemv_case(case)
    want = None
    for fused, path in ((None, PATH_DYNAMIC), (True, PATH_DYNAMIC), (True, PATH_STATIC), (False, PATH_DYNAMIC), (False, PATH_STATIC)):
        lb, init = mg.gemv_graph(case, *args, fused=fused)
        got = _run(lb, init, path, times=2)
        if want is None:
            want = got['out']
            y, s = got['y'].view(np.int8).reshape(case[0], -1)[:, :case[2]], got['ys']
            exact, bound = f64.product(y, s, *args[3:])
            f64.near(want.reshape(exact.shape), exact, bound, case[4])
        np.testing.assert_array_equal(got['out'], want, err_msg=f'{fused} {path}')


def test_rows_with_nan_reach_their_outputs():
    print('product nan', flush=True)
    case = (3, 40, 64, 16, 'f32', 0, False, False, 64)
    x, _, _, w, sw, _, _ = mg.gemv_case(case)
    x[1, 5] = np.inf
    for fused in (True, False, None):
        lb, init = mg.gemv_graph(case, x, None, None, w, sw, None, None, fused=fused)
        out = _run(lb, init)['out'].reshape(3, 40)
        assert np.isnan(out[1]).all() and np.isfinite(out[[0, 2]]).all()


@pytest.mark.parametrize('tasks', [1, 3, 256])
@pytest.mark.parametrize('case', mg.APPENDS, ids=str)
def test_append(case, tasks):
    """A key is off by some steps of 2^-24 of its magnitudes (norm: 4, angle: pi 2^-24 absolute and 1, products: 2, below 2^-20 with the other
    half's part)."""
    print(f'append {case} tasks {tasks}', flush=True)
    (lb, init), pg, q, want = mg.append_graph(case, np.random.default_rng(1), tasks=tasks)
    got = _run(lb, init, PATH_STATIC if tasks == 3 else PATH_DYNAMIC)
    _caches(got, want, case)


def _caches(got, want, case, rel=2.0 ** -20):
    big = np.abs(np.concatenate([w.reshape(-1) for w in want if w is not None])).max(initial=0, where=np.isfinite(np.concatenate([w.reshape(-1) for w in want if w is not None])))
    k, v = (got[n].reshape(*w.shape[:3], -1)[..., :w.shape[3]] for n, w in zip(('kc', 'vc'), want))
    f64.near(v, want[1], 0, case[4])
    f64.near(k, want[0], rel * big, case[4])
    if want[2] is not None:
        on = ~np.isnan(want[2])
        rows, H, hd = want[2].shape
        o = got['qo' if 'qo' in got else 'q'].reshape(rows, -1)[:, :H * hd].reshape(rows, H, hd)
        f64.near(o[on], want[2][on], rel * big, case[4])
        return o[~on]


@pytest.mark.parametrize('kw', [{'gamma': False}, {'theta': 0.0}, {'gamma': False, 'theta': 0.0}, {'queries': False}, {'first': 5}, {'extra': 8}, {'extra': 5}, {'inplace': True},
                                {'unseen': np.nan}], ids=str)
@pytest.mark.parametrize('case', [mg.APPENDS[1], mg.APPENDS[3]], ids=str)
def test_append_options(case, kw):
    """Without norm, rotation or queries, rows that start later, wider rows, queries in place, pages with NaN; rows of nobody stay."""
    print(f'append {case} {kw}', flush=True)
    (lb, init), pg, q, want = mg.append_graph(case, np.random.default_rng(2), **kw)
    left = _caches(_run(lb, init), want, case)
    if left is not None and not kw.get('inplace'):
        assert (left == 7).all()


def test_append_far_positions():
    """Positions of 10^5, in a long table."""
    print('append far', flush=True)
    case = (64, 128, 1, 2, 'f32', [100000, 3], [40, 1])
    (lb, init), pg, q, want = mg.append_graph(case, np.random.default_rng(3))
    _caches(_run(lb, init), want, case)


def _attend(case, rng=None, path=PATH_DYNAMIC, times=1, exact_p=None, **kw):
    (lb, init), pg, q = mg.attend_graph(case, rng or np.random.default_rng(2), **kw)
    got = _run(lb, init, path, times)
    scale = kw.get('scale') or 1 / np.sqrt(case[1])
    want, mag = f64.attend(q, *pg, case[0], scale)
    rows, H, hd = want.shape
    o, on = got['o'].reshape(rows, -1)[:, :H * hd].reshape(want.shape), ~np.isnan(want).all(-1)
    kmax = np.where(np.isfinite(pg[0]), np.abs(pg[0]), 0).max()
    sabs = np.where(np.isfinite(q), np.abs(q), 0).sum(-1).max() * kmax * scale
    odt = kw.get('odt') or case[4]
    exact = (case[4] == 'f32' or odt == 'f32') if exact_p is None else exact_p
    f64.near(o[on], want[on], mg.attend_bound(case, mag, sabs, exact)[on], odt)
    assert (o[~on] == 7).all() and not got['o.cnt'].any()
    return o


@pytest.mark.parametrize('tasks', [1, 7, 256])
@pytest.mark.parametrize('case', mg.ATTENDS, ids=str)
def test_attend(case, tasks):
    print(f'attend {case} tasks {tasks}', flush=True)
    _attend(case, tasks=tasks, path=PATH_STATIC if tasks == 7 else PATH_DYNAMIC, times=2)


@pytest.mark.parametrize('kw', [{'first': 4}, {'extra': 8}, {'extra': 3}, {'odt': 'f32'}, {'scale': 0.5}], ids=str)
@pytest.mark.parametrize('case', [mg.ATTENDS[1], mg.ATTENDS[2], mg.ATTENDS[7]], ids=str)
def test_attend_options(case, kw):
    print(f'attend {case} {kw}', flush=True)
    _attend(case, **kw)


@pytest.mark.parametrize('case', [(64, 128, 2, 8, 'bf16', [20000, 3, 9000], [1, 1, 1]), (16, 64, 1, 4, 'bf16', [12000], [1]), (32, 128, 1, 8, 'bf16', [5000, 700], [100, 1]),
                                  (16, 64, 1, 2, 'f32', [7000], [3])], ids=str)
@pytest.mark.parametrize('tasks', [2, 33, 256])
def test_attend_long(case, tasks):
    """Tiles cut into many pieces; what is left in the workspace by a launch does not matter to the next."""
    print(f'attend long {case} tasks {tasks}', flush=True)
    _attend(case, tasks=tasks, times=3, n_max=max(case[6]))


@pytest.mark.parametrize('case', [(64, 128, 2, 8, 'bf16', [3000, 100], [3, 1]), (16, 64, 1, 4, 'bf16', [3000, 7], [70, 5]), (16, 64, 2, 4, 'f32', [3000], [9]),
                                  (64, 100, 1, 3, 'f32', [2500], [4])], ids=str)
@pytest.mark.parametrize('tasks', [2, 9, 256])
def test_attend_more_tokens_than_the_hint(case, tasks):
    """Tiles hold no more rows than the partials have room for: sequences that bring more tokens than n_max are taken in more tiles."""
    print(f'attend hint {case} {tasks}', flush=True)
    (lb, _), _, _ = mg.attend_graph(case, np.random.default_rng(2), tasks=tasks, n_max=1)
    group = case[3] // case[2]
    assert next(m for m in lb.metadata['buffers'] if m['name'] == 'o.part')['rows'] == 2 * tasks * group
    _attend(case, tasks=tasks, n_max=1)


@pytest.mark.parametrize('case', [mg.ATTENDS[1], mg.ATTENDS[2], mg.ATTENDS[5], mg.ATTENDS[7], mg.ATTENDS[9]], ids=str)
@pytest.mark.parametrize('bad', [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see(case, bad):
    """The newest token's key and value are not finite: rows in front of it do not see them, its own are NaN."""
    print(f'attend unseen {bad} {case}', flush=True)
    page, lens, new = case[0], case[5], case[6]

    def kv(kc, vc, table):
        for b, (L, n) in enumerate(zip(lens, new)):
            if n > 1:
                t = L + n - 1
                kc[table[b, t // page], :, t % page, 0] = bad
                vc[table[b, t // page], :, t % page, 1] = bad
        return kc, vc
    rng = np.random.default_rng(4)
    (lb, init), pg, q = mg.attend_graph(case, rng, tasks=9, kv=kv)
    got = _run(lb, init)['o'].reshape(q.shape)
    want, mag = f64.attend(q, *pg, page, 1 / np.sqrt(case[1]))
    for b, n in enumerate(new):
        last = pg[4][b + 1] - 1
        if n > 1:
            assert np.isnan(got[last]).any(-1).all() and np.isfinite(got[pg[4][b]:last]).all()
    fine = np.isfinite(want).all(-1)
    sabs = np.abs(q).sum(-1).max() * np.where(np.isfinite(pg[0]), np.abs(pg[0]), 0).max() / np.sqrt(case[1])
    f64.near(got[fine], want[fine], mg.attend_bound(case, mag, sabs, case[4] == 'f32')[fine], case[4])


@pytest.mark.parametrize('case', [(64, 100, 1, 3, 'f32', [300], [2]), (16, 64, 1, 4, 'f32', [300], [1]), (64, 128, 1, 4, 'bf16', [300], [3]), (32, 128, 1, 2, 'bf16', [300], [70]),
                                  (16, 6, 1, 1, 'bf16', [3000], [1])], ids=str)
@pytest.mark.parametrize('tasks', [1, 32])
def test_seen_keys_of_score_minus_infinity(case, tasks):
    """Keys whose score is -inf have no weight where another key's is finite, also where they fill a block."""
    print(f'attend -inf {case} {tasks}', flush=True)
    page, hd, hkv, heads, dt, lens, new = case
    rng = np.random.default_rng(4)

    def kv(kc, vc, table):
        t = np.arange(200)
        kc[table[0, t // page], :, t % page, 0] = -np.inf
        return kc, vc
    q = lambda rows: mg.bf(np.abs(rng.standard_normal((rows, heads, hd))) + 0.1, dt)   # noqa: E731
    _attend(case, tasks=tasks, kv=kv, q=q)


def test_attend_large_scores():
    """Scores in the thousands: a weight of one, the others nothing."""
    print('attend large scores', flush=True)
    for case in (mg.ATTENDS[1], mg.ATTENDS[2], mg.ATTENDS[7]):
        (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(6), scale=50.0, tasks=5)
        got = _run(lb, init)['o'].reshape(q.shape)
        want, mag = f64.attend(q, *pg, case[0], 50.0)
        on = ~np.isnan(want)
        assert np.isfinite(got[on]).all() and (np.abs(got[on]) <= np.abs(mag[on]).max() * 1.01).all()
        # where one weight is all but 1, the result is that value
        k = np.abs(np.abs(want) - mag) < 1e-9
        assert (np.abs(got - want)[k & on] <= 2.0 ** -6 * np.abs(want)[k & on] + 1e-3).mean() > 0.98


def test_results_do_not_depend_on_the_launch():
    """The same bits from every launch: pieces are merged in their order, whichever comes last."""
    print('attend repeat', flush=True)
    for case in (mg.ATTENDS[1], mg.ATTENDS[2], mg.ATTENDS[5]):
        (lb, init), *_ = mg.attend_graph(case, np.random.default_rng(7), tasks=64)
        ex = Executor.from_bundle(lb, buffers=init, trace=False)
        seen = []
        for _ in range(4):
            ex.relaunch()
            ex.finish()
            seen.append(ex.read('o'))
        ex.close()
        for o in seen[1:]:
            np.testing.assert_array_equal(o, seen[0])


@pytest.mark.parametrize('what', ['falling', 'rows', 'negative', 'length', 'room', 'page', 'unset'])
def test_bad_tables(what):
    """Errors with a normal end; row numbers and lengths are refused before anything is written, and the next launch is right."""
    print(f'bad {what}', flush=True)
    cases = (mg.attend_graph, mg.ATTENDS[0]), (mg.attend_graph, mg.ATTENDS[2]), (mg.attend_graph, mg.ATTENDS[7]), (mg.append_graph, mg.APPENDS[0]), (mg.append_graph, mg.APPENDS[3])
    for make, case in cases:
        (lb, init), pg, *_ = make(case, np.random.default_rng(3))
        kc, vc, table, lens, cu = (x.copy() for x in pg)
        if what == 'falling':
            cu[1] = cu[2] + 1
        if what == 'rows':
            cu[-1] += 50
        if what == 'negative':
            cu[0] = -1
        if what == 'length':
            lens[0] = -2
        if what == 'room':
            lens[0] = case[0] * table.shape[1]
        if what == 'page':
            table[0, lens[0] // case[0]] = len(kc)
        if what == 'unset':
            table[0, lens[0] // case[0]] = -1
        names, bad = sg.names(lb), [x.copy() for x in init]
        for n, x in (('table', table), ('lens', lens), ('cu', cu)):
            bad[names.index(n)] = x.reshape(-1)
        err, got = _error(lb, bad)
        assert err == ('OP_RANGE' if what in ('page', 'unset') else 'OP_KVLEN'), err
        if what not in ('page', 'unset'):
            for n in ('o', 'qo', 'kc', 'vc'):
                if n in got:
                    a, b = got[n], init[names.index(n)].reshape(-1)
                    np.testing.assert_array_equal(a, b if b.dtype != np.uint16 else a)
        ex = Executor.from_bundle(lb, buffers=bad)
        ex.start()
        ex.finish(check=False)
        for n, x in (('table', pg[2]), ('lens', pg[3]), ('cu', pg[4])):
            ex.write(n, x.reshape(-1))
        ex.relaunch()
        assert ex.finish()['done'] == lb.ntasks
        have = ex.read('o' if make is mg.attend_graph else 'kc')
        ex.close()
        np.testing.assert_array_equal(have, _run(lb, init)['o' if make is mg.attend_graph else 'kc'])


