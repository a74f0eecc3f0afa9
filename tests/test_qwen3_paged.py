"""Qwen3 steps that take prompts and single tokens together, over paged caches with 8-bit weights: the framework's own model on the
operators 315-319 in a row."""
import numpy as np
import pytest

import mixed_fp64 as f64
import oracle
import qwen3_paged_steps as steps
import serving_graphs as sg
from kvm_amd import executor
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import qwen3, serving

# (batch, rows, further options, new tokens of every step): prompts, prompts beside single tokens, sequences that bring none, rows left over
MIXED = [(3, 32, {}, [[9, 0, 20], [1, 14, 1], [1, 1, 1], [0, 0, 0]]), (2, 70, {'layers': 2, 'page': 32}, [[70, 0], [1, 69]]), (1, 1, {'ctx': 15}, [[1], [1], [0]]),
         (4, 12, {'ctx': 0, 'layers': 2, 'heads': 6, 'head_dim': 64, 'hidden': 192, 'ffn': 400}, [[3, 3, 0, 2], [1, 1, 9, 1]])]
TOKENS = [(1, {}), (3, {'ctx': 30}), (20, {'ctx': 3, 'layers': 2, 'head_dim': 64})]


def _run(c, step, given, lens, many):
    """`step` (what to write -> all buffers after it) over the plan of a run; each step's choice goes on where the next has one token."""
    rng, now = np.random.default_rng(5), {**given}
    for new in many:
        now.update(steps.plan(c, lens, new, rng))
        after = step({n: now[n] for n in steps.TABLES})
        steps.check(c, now, after)
        now, lens = after, lens + np.asarray(new)


@pytest.mark.parametrize('batch,rows,kw,many', MIXED, ids=str)
def test_mixed_oracle(batch, rows, kw, many):
    c, lb, given = steps.case(batch, rows, **kw)
    assert executor.validate(lb) is None
    bufs = steps.loaded(lb, given)

    def step(tables):
        for n, x in tables.items():
            bufs[sg.names(lb).index(n)] = np.ascontiguousarray(x).reshape(-1)
        bufs[:] = [np.ascontiguousarray(x) for x in oracle.run(lb, [x.copy() for x in bufs])['buffers']]
        return dict(zip(sg.names(lb), bufs))
    _run(c, step, dict(zip(sg.names(lb), bufs)), np.full(batch, c.ctx), many)


@pytest.mark.parametrize('batch,kw', TOKENS, ids=str)
def test_tokens_oracle(batch, kw):
    """Decode steps, each from what the one before left."""
    c, lb, given = steps.case(batch, **kw)
    bufs = steps.loaded(lb, given)
    for _ in range(3):
        after = oracle.run(lb, [x.copy() for x in bufs])['buffers']
        steps.check(c, dict(zip(sg.names(lb), bufs)), dict(zip(sg.names(lb), after)))
        bufs = [np.ascontiguousarray(x) for x in after]


@pytest.mark.parametrize('shape', [(1, 1), (3, 7), (5, 1000)])
def test_quantise_rows(shape):
    """Weights as the host prepares them are what the operator makes of them."""
    x = np.random.default_rng(3).standard_normal(shape).astype(np.float32)
    x[-1] = 0
    if shape[0] > 2:
        x[1, 0] = np.inf
    q, s = serving.quantise_rows(x)
    want, scale = f64.quantise(x)
    np.testing.assert_array_equal(q.view(np.int8)[:, :shape[1]], want)
    np.testing.assert_array_equal(s, scale)
    assert q.shape[1] % 4 == 0 and not q.view(np.int8)[:, shape[1]:].any()


def test_other_caches_keep_their_graphs():
    ops = {t['op'] for t in qwen3.build(qwen3.Qwen3Config.tiny()).spec['graphs'][0]['tasks']}
    assert not ops & {'rows_q8', 'matmul_q8', 'gemv_q8', 'qkv_append_paged', 'attn_paged'}
    ops = [{t['op'] for t in qwen3.build(qwen3.Qwen3Config.tiny(batch=b, cache='paged', rows=r)).spec['graphs'][0]['tasks']} for b, r in ((1, 0), (2, 40))]
    assert {'gemv_q8', 'qkv_append_paged', 'attn_paged'} <= ops[0] and 'rows_q8' not in ops[0]
    assert {'rows_q8', 'matmul_q8', 'qkv_append_paged', 'attn_paged'} <= ops[1]


@pytest.mark.parametrize('kw', [{'cache': 'paged', 'page': 48}, {'cache': 'paged', 'rows': -1}, {'cache': 'paged', 'presence': 0.1}, {'rows': 4}, {'pages': 9},
                                {'cache': 'paged', 'pages': 1, 'ctx': 100}, {'cache': 'paged', 'head_dim': 258}, {'cache': 'paged', 'heads': 3}, {'cache': 'paged', 'batch': 1025}], ids=str)
def test_refusals(kw):
    with pytest.raises(ValueError):
        qwen3.build(qwen3.Qwen3Config.tiny(**kw))


def _open(lb, given, path):
    return Executor.from_bundle(lb, buffers=[x.copy() for x in steps.loaded(lb, given)], path=path)


@pytest.mark.gpu
@pytest.mark.parametrize('path', [PATH_DYNAMIC, PATH_STATIC])
@pytest.mark.parametrize('batch,rows,kw,many', MIXED, ids=str)
def test_mixed(batch, rows, kw, many, path):
    print(f'qwen3 paged {batch} {rows} {kw} path {path}', flush=True)
    c, lb, given = steps.case(batch, rows, **kw)
    ex = _open(lb, given, path)

    def step(tables):
        for n, x in tables.items():
            ex.write(n, x)
        ex.relaunch()
        assert ex.finish()['done'] == lb.ntasks
        return {n: ex.read(n) for n in sg.names(lb)}
    _run(c, step, {n: ex.read(n) for n in sg.names(lb)}, np.full(batch, c.ctx), many)
    ex.close()


@pytest.mark.gpu
@pytest.mark.parametrize('path', [PATH_DYNAMIC, PATH_STATIC])
@pytest.mark.parametrize('batch,kw', TOKENS, ids=str)
def test_tokens(batch, kw, path):
    print(f'qwen3 paged tokens {batch} {kw} path {path}', flush=True)
    c, lb, given = steps.case(batch, **kw)
    ex = _open(lb, given, path)
    before = {n: ex.read(n) for n in sg.names(lb)}
    for _ in range(6):
        ex.relaunch()
        ex.finish()
        after = {n: ex.read(n) for n in sg.names(lb)}
        steps.check(c, before, after)
        before = after
    ex.close()


@pytest.mark.gpu
def test_same_steps_again():
    """Two executors of the same steps, one read in between, leave the same buffers bit for bit (the merges' order does not show)."""
    print('qwen3 paged twice', flush=True)
    c, lb, given = steps.case(5, layers=2, ctx=200, tasks_per_phase=64)
    left = []
    for reads in (True, False):
        ex = _open(lb, given, PATH_STATIC)
        for _ in range(5):
            ex.relaunch()
            ex.finish()
            if reads:
                [ex.read(n) for n in sg.names(lb)]
        left.append({n: ex.read(n) for n in sg.names(lb) if n != 'att.part'})
        ex.close()
    for n in left[0]:
        np.testing.assert_array_equal(left[0][n], left[1][n], err_msg=n)
