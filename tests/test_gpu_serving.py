"""The serving operators on the GPU against their definition in 64 bits: bytes, scales and tails of an append exactly, attention
and logits within bounds that count roundings (serving_fp64), and steps that use them together."""
import numpy as np
import pytest

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import executor
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor

pytestmark = pytest.mark.gpu


def _run(lb, init, path=PATH_DYNAMIC, times=1):
    """Runs the graph and returns (read, executor closed after the reads: all buffers as arrays)."""
    ex = Executor.from_bundle(lb, buffers=init, path=path)
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


def _same(got, want, c):
    got = sg.cache_of(lambda n: got[n], c)
    for n in sg.CACHE:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)


@pytest.mark.parametrize('tasks', [1, 256])
@pytest.mark.parametrize('case', sg.APPENDS, ids=str)
def test_append(case, tasks):
    print(f'append {case} tasks {tasks}', flush=True)
    blk, hd, hkv, dt, n_new, lens = case
    c, k, v = sg.append_case(case)
    lb, init = sg.append_graph(c, k, v, lens, hkv, n_new, dt, dt, tasks=tasks)
    _same(_run(lb, init, PATH_STATIC if tasks == 1 else PATH_DYNAMIC), f64.append(c, k, v, lens, hkv, n_new, dt == 'bf16'), c)


@pytest.mark.parametrize('new,tail', [('f32', 'bf16'), ('bf16', 'f32')])
def test_append_mixed_types(new, tail):
    """The tail's type rounds; new tokens of another type, in rows wider than the heads."""
    print(f'append mixed {new} {tail}', flush=True)
    case = (32, 64, 2, new, 45, [0, 20, 31])
    c, k, v = sg.append_case(case)
    for x in 'kv':
        c[x + 't'] = bl.bf16_round(c[x + 't'])
    wide = [np.concatenate([x, x[:, :5]], 1) for x in (k, v)]
    lb, init = sg.append_graph(c, *wide, case[5], 2, 45, tail, new)
    _same(_run(lb, init), f64.append(c, k, v, case[5], 2, 45, tail == 'bf16'), c)


@pytest.mark.parametrize('hd,tail', [(128, 'bf16'), (64, 'f32'), (100, 'f32')])
def test_append_normed_and_rotated(hd, tail):
    """Keys through head norm and rotation, at positions up to 10^5. In 32 bits a key is off by some steps of 2^-24 of its
    magnitudes (norm: 4, angle: pi 2^-24 absolute and 1, products: 2, below 2^-20 with the other half's part), then by one
    rounding; a byte by that over the scale and a half step."""
    print(f'append rope {hd} {tail}', flush=True)
    lens, n_new, blk = [0, 100000 // 16 * 16 + 9], 23, 16
    rng = np.random.default_rng(3)
    c = sg.random_cache(rng, 4, -(-(max(lens) + n_new) // blk), blk, hd, tail == 'bf16')
    k, v = (rng.standard_normal((2 * n_new, 2 * hd)).astype(np.float32) for _ in range(2))
    g = (rng.random(hd) + 0.5).astype(np.float32)
    lb, init = sg.append_graph(c, k, v, lens, 2, n_new, tail, 'f32', gamma=g, theta=1e6, eps=1e-6)
    got = sg.cache_of(_run(lb, init).__getitem__, c)
    want = f64.append(c, k, v, lens, 2, n_new, tail == 'bf16', g, np.float32(1e-6), 1e6)
    for n in ('vq', 'vs', 'vt'):
        np.testing.assert_array_equal(got[n], want[n])
    rel = (2 * sg.step('bf16') if tail == 'bf16' else 0) + 2.0 ** -20        # two neighbours of bf16 are a whole step apart
    big = np.abs(want['kt']).max()
    assert np.abs(got['kt'] - want['kt']).max() <= rel * big
    assert (np.abs(got['ks'] - want['ks']) <= (rel + 2.0 ** -24) * want['ks']).all()
    off = np.abs(got['kq'].astype(int) - want['kq'])
    assert off.max() <= 1 + int(127 * 2 * rel) and (off != 0).mean() < 0.02


def test_append_blocks_that_are_not_finite():
    print('append nonfinite', flush=True)
    for blk, hd in ((16, 64), (16, 4)):
        x = np.zeros((5, blk, hd), np.float32)
        x[1, 3, 2] = 1e-37
        x[2, 0, 0], x[2, 5, 1] = np.nan, 3
        x[3, 7, 3] = -np.inf
        x[4] = np.float32(3e38)
        c = f64.empty_cache(5, 1, blk, hd)
        flat = x.reshape(-1, hd)
        lb, init = sg.append_graph(c, flat, flat, [0] * 5, 1, blk, 'f32', 'f32')
        _same(_run(lb, init), f64.append(c, flat, flat, [0] * 5, 1, blk, False), c)


def test_append_token_by_token():
    """A prompt at once, in pieces, and token by token: the same cache."""
    print('append token by token', flush=True)
    rng = np.random.default_rng(5)
    c = f64.empty_cache(2, 3, 32, 64)
    k, v = (bl.bf16_round(rng.standard_normal((75, 128)).astype(np.float32)) for _ in range(2))
    want = f64.append(c, k, v, [0], 2, 75, True)
    for cuts in ([0, 75], [0, 31, 32, 33, 70, 75], list(range(76))):
        have = c
        for a, e in zip(cuts, cuts[1:]):
            lb, init = sg.append_graph(have, k[a:e], v[a:e], [a], 2, e - a)
            have = sg.cache_of(_run(lb, init).__getitem__, c)
        for x in 'kv':
            np.testing.assert_array_equal(have[x + 'q'], want[x + 'q'])
            np.testing.assert_array_equal(have[x + 's'], want[x + 's'])
            np.testing.assert_array_equal(have[x + 't'][:, :75 % 32], want[x + 't'][:, :75 % 32])


@pytest.mark.parametrize('hd', [128, 100])
@pytest.mark.parametrize('first,drafted,kept', [(10, 7, 0), (10, 21, 5), (0, 31, 30), (32, 31, 0), (30, 2, 2), (20, 44, 44), (20, 12, 12), (25, 20, 7)], ids=str)
def test_lengths_set_back(first, drafted, kept, hd):
    """Drafted tokens are appended, attended to and all but `kept` taken back (to within the unfinished block, or to where a block
    starts); the tokens and the attention that follow are as if only the kept ones had been there."""
    print(f'set back {first} {drafted} {kept} hd {hd}', flush=True)
    rng = np.random.default_rng(6)
    have = f64.empty_cache(2, 3, 32, hd)
    rows = lambda n: tuple(bl.bf16_round(rng.standard_normal((n, 2 * hd)).astype(np.float32)) for _ in range(2))   # noqa: E731
    step = lambda c, x, at: sg.cache_of(_run(*sg.append_graph(c, *x, [at], 2, len(x[0]))).__getitem__, c)   # noqa: E731
    begin, draft, after = rows(first), rows(drafted), rows(9)
    if first:
        have = step(have, begin, 0)
    have = step(have, draft, first)
    L = first + kept
    have = step(have, after, L)
    k, v = (np.concatenate([begin[i], draft[i][:kept], after[i]]) for i in range(2))
    want = f64.append(f64.empty_cache(2, 3, 32, hd), k, v, [0], 2, L + 9, True)
    n = L + 9
    for x in 'kv':
        np.testing.assert_array_equal(have[x + 'q'][:, :n // 32], want[x + 'q'][:, :n // 32])
        np.testing.assert_array_equal(have[x + 's'][:, :n // 32], want[x + 's'][:, :n // 32])
        np.testing.assert_array_equal(have[x + 't'][:, :n % 32], want[x + 't'][:, :n % 32])
    q = bl.bf16_round(rng.standard_normal((1, 4 * hd)).astype(np.float32))
    o, bound = f64.attend(want, q, [n - 1], 2, 4, 1, np.float32(0.1))
    sg.near(_run(*sg.attend_graph(have, q, [n - 1], 2, 4, 1, 0.1))['o'], o, bound, 'bf16')


@pytest.mark.parametrize('rope', [False, True])
@pytest.mark.parametrize('tasks', [1, 7, 256])
@pytest.mark.parametrize('case', sg.ATTENDS, ids=lambda c: str(c)[:60])
def test_attend(case, tasks, rope):
    print(f'attend {case} tasks {tasks} rope {rope}', flush=True)
    blk, hd, hkv, heads, dt, n_new, lens = case
    c, q = sg.attend_case(case)
    g = np.random.default_rng(1).random(hd).astype(np.float32) + 0.5
    kw = dict(gamma=g, theta=1e6, eps=1e-6) if rope else {}
    lb, init = sg.attend_graph(c, q, lens, hkv, heads, n_new, 0.1, dt, dt, tasks=tasks, extra=3 if tasks == 7 else 0, **kw)
    got = _run(lb, init, PATH_STATIC if tasks == 256 else PATH_DYNAMIC, times=2)
    want, bound = f64.attend(c, q, lens, hkv, heads, n_new, np.float32(0.1), *((g, np.float32(1e-6), 1e6) if rope else ()))
    o = got['o'].reshape(len(q), -1)
    sg.near(o[:, :heads * hd], want, bound, dt)
    assert (o[:, heads * hd:] == 7).all()                            # columns behind the heads stay
    assert not got['o.cnt'].any()


def test_attend_long_f32_error():
    """A long context in f32 output, the error of the whole against 64 bits: sums of n terms, each addition off by a step of 2^-24
    in either direction, and 64 steps for scores and exponentials."""
    print('attend long', flush=True)
    case = (64, 128, 1, 4, 'f32', 1, [30000])
    c, q = sg.attend_case(case)
    for tasks in (1, 16):
        lb, init = sg.attend_graph(c, q, case[6], 1, 4, 1, 1 / np.sqrt(128), 'f32', 'f32', tasks=tasks)
        want, _ = f64.attend(c, q, case[6], 1, 4, 1, np.float32(1 / np.sqrt(128)))
        got = _run(lb, init)['o'].astype(np.float64)
        assert np.linalg.norm(got - want.ravel()) <= (np.sqrt(30000) + 64) * 2.0 ** -24 * np.linalg.norm(want)


def test_attend_values_of_any_size():
    """Blocks whose scales differ by many orders, among them zero and NaN; a query of zeros, of large and of small numbers; a token
    that a query may not see does not reach it, whatever its block holds."""
    print('attend scales', flush=True)
    rng = np.random.default_rng(7)
    for hd in (128, 100):
        c = sg.random_cache(rng, 2, 8, 16, hd, False)
        c['vs'][0] = [1e-30, 1e30, 0, 1, 1e-10, 1e10, 1e-35, 2]
        c['ks'][0] *= [0, 1, 1e-3, 1, 1, 1e-20, 1, 1]
        q = rng.standard_normal((6, hd)).astype(np.float32)
        q[0], q[1], q[2] = 0, q[1] * 1e3, q[2] * 1e-20
        c['ks'][1, 1], c['vs'][1, 1] = np.nan, np.nan               # tokens 16 .. 31 of the second sequence
        many = rng.standard_normal((40, hd)).astype(np.float32)       # tokens 12 .. 31: the first four may not see the NaN block
        for heads, n_new, lens, x in ((3, 1, [127, -1], q.reshape(2, -1)), (1, 3, [124, 13], q), (1, 20, [100, 12], many)):
            lb, init = sg.attend_graph(c, x, lens, 1, heads, n_new, 0.3, 'f32', 'f32')
            got = _run(lb, init)['o']
            want, bound = f64.attend(c, x, lens, 1, heads, n_new, np.float32(0.3))
            sg.near(got, want, bound, 'f32')
            if n_new == 20:
                assert np.isfinite(got.reshape(40, -1)[20:24]).all() and np.isnan(got.reshape(40, -1)[24:]).all()


@pytest.mark.parametrize('tasks', [1, 256])
@pytest.mark.parametrize('case', sg.ADJUSTS, ids=str)
def test_adjust(case, tasks):
    print(f'adjust {case} tasks {tasks}', flush=True)
    x, par, g = sg.adjust_case(case)
    want, hist, bound = f64.adjust(x, par, **g)
    lb, init = sg.adjust_graph(x, par, case[2], case[3], tasks=tasks, **g)
    got = _run(lb, init, times=2)
    sg.near(got['out'], want, bound, case[3])
    np.testing.assert_array_equal(got['logits'], np.asarray(x, np.float32).ravel())
    lb, init = sg.adjust_graph(x, par, case[2], inplace=True, tasks=tasks, **g)
    got = _run(lb, init, PATH_STATIC)
    sg.near(got['logits'], want, bound, case[2])
    if hist is not None:
        np.testing.assert_array_equal(got['hist'].reshape(hist.shape), hist)


def test_adjust_values_that_are_not_finite():
    """NaN and infinities pass through, and are -inf where the mask says so; the lowest f32 under a penalty is -inf."""
    print('adjust nonfinite', flush=True)
    x = np.zeros((1, 70), np.float32)
    x[0, :8] = [np.nan, np.inf, -np.inf, np.nan, np.inf, -np.inf, np.finfo(np.float32).min, 5]
    par = np.array([[1.5, 0.5, 0.25]], np.float32)
    mask = np.array([[~0b111000, -1, -1]], np.int32)
    hist = np.array([[0, 1, 2, 6, 7, 7]], np.int32)
    lb, init = sg.adjust_graph(x, par, hist=hist, hlen=np.array([6], np.int32), plen=np.array([4], np.int32), mask=mask)
    got = _run(lb, init)['out']
    assert np.isnan(got[0]) and got[1] == np.inf and (got[2:7] == -np.inf).all()
    assert got[7] == np.float32(5 / np.float32(1.5)) - 1.25 or abs(got[7] - (5 / 1.5 - 1.25)) <= 4 * 2.0 ** -24 * 5
    assert not got[8:].any()


@pytest.mark.parametrize('make', ['append', 'attend', 'adjust'])
def test_bad_lengths_are_refused_whole(make):
    """Lengths that no cache holds, rows of a mask or a history that are not there: an error, and nothing is written."""
    print(f'refused {make}', flush=True)
    if make == 'adjust':
        x, par, g = sg.adjust_case(sg.ADJUSTS[3])
        for bad in ({'hlen': 701}, {'plen': -1}, {'mrow': 4}, {'mrow': -2}):
            k, value = next(iter(bad.items()))
            edit = {n: v.copy() for n, v in g.items()}
            edit[k][3] = value
            lb, init = sg.adjust_graph(x, par, 'f32', tasks=1, **edit)
            err, got = _error(lb, init)
            assert err == 'OP_RANGE' and not got['out'].any()
        return
    c = f64.empty_cache(6, 2, 64, 128)
    x = np.ones((3, 256), np.float32)
    for bad in (-2, 128, 2 ** 31 - 1):
        lens = np.array([5, bad, -1], np.int64).astype(np.int32)
        lb, init = (sg.append_graph(c, x, x, lens, 2, 1, tasks=1) if make == 'append' else sg.attend_graph(c, x[[1]].repeat(3, 0), lens, 2, 2, 1, 1.0))
        err, got = _error(lb, init)
        assert err == 'OP_KVLEN'
        if make == 'append':
            assert not any(got[n].any() for n in sg.CACHE)


@pytest.mark.parametrize('hd', [128, 64, 100])
@pytest.mark.parametrize('batch', [3, 100])
def test_attention_with_a_bad_length_writes_nothing(hd, batch):
    """In the form of whole vectors and in the general one: the tasks of a call check every length before they write."""
    print(f'attention refused hd {hd} batch {batch}', flush=True)
    c = f64.empty_cache(2 * batch, 2, 64, hd)
    x = np.ones((batch, 2 * hd), np.float32)
    for bad in (-2, 128, 2 ** 31 - 1):
        for tasks in (1, 16):
            lens = np.full(batch, 70, np.int64)
            lens[0], lens[-1] = -1, bad
            lb, init = sg.attend_graph(c, x, lens.astype(np.int32), 2, 2, 1, 1.0, tasks=tasks)
            err, got = _error(lb, init)
            assert err == 'OP_KVLEN' and (got['o'] == 7).all() and not got['o.cnt'].any()


def _shifted(lb, init, skip):
    """The graph on buffers that begin `skip` elements into an allocation of the caller's; returns all contents."""
    meta = lb.metadata['buffers']
    ex = Executor(trace=False)
    size = {0: 4, 1: 4, 2: 2}
    for m, x in zip(meta, init):
        pad = np.concatenate([np.zeros(skip, x.dtype), x.reshape(-1), np.zeros(64, x.dtype)])
        ex.add_buffer(m['name'], 1, pad.size, m['dtype'], data=pad)
    ptrs = [ex.device_ptr(m['name']) + skip * size[m['dtype']] for m in meta]
    res, _ = executor.run_noalloc(lb, ptrs, [0])
    assert res['rc'] == 0 and res['err_code'] == 0, res
    got = {m['name']: ex.read(m['name'])[skip:skip + m['rows'] * m['cols']] for m in meta}
    for m in meta:
        edge = ex.read(m['name'])
        assert not edge[:skip].any() and not edge[skip + m['rows'] * m['cols']:].any(), m['name']   # nothing outside
    ex.close()
    return got


@pytest.mark.parametrize('skip', [1, 2, 3, 4])
def test_buffers_at_any_element(skip):
    print(f'unaligned {skip}', flush=True)
    for case in (sg.APPENDS[2], sg.APPENDS[3]):
        blk, hd, hkv, dt, n_new, lens = case
        c, k, v = sg.append_case(case)
        lb, init = sg.append_graph(c, k, v, lens, hkv, n_new, dt, dt)
        _same(_shifted(lb, init, skip), f64.append(c, k, v, lens, hkv, n_new, dt == 'bf16'), c)
    for case in (sg.ATTENDS[2], sg.ATTENDS[5]):
        blk, hd, hkv, heads, dt, n_new, lens = case
        c, q = sg.attend_case(case)
        lb, init = sg.attend_graph(c, q, lens, hkv, heads, n_new, 0.1, dt, dt)
        want, bound = f64.attend(c, q, lens, hkv, heads, n_new, np.float32(0.1))
        sg.near(_shifted(lb, init, skip)['o'], want, bound, dt)
    for case in sg.ADJUSTS[3:5]:
        x, par, g = sg.adjust_case(case)
        want, hist, bound = f64.adjust(x, par, **g)
        lb, init = sg.adjust_graph(x, par, case[2], case[3], **g)
        sg.near(_shifted(lb, init, skip)['out'], want, bound, case[3])
