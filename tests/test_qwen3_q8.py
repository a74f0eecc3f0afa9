"""The Qwen3 decode step over the 8-bit cache with penalties: the framework's own model on the serving operators together."""
import numpy as np
import pytest

import oracle
import qwen3_q8_steps as steps
from kvm_amd import bundle as bl
from kvm_amd import compiler
from kvm_amd.executor import PATH_DYNAMIC, PATH_STATIC, Executor
from kvm_amd.workloads import qwen3


def _loaded(w, given):
    lb = bl.load(compiler.compile_spec(w.spec))
    init = [np.ascontiguousarray(given[m['name']]).reshape(-1) if m['name'] in given
            else bl.materialize({**m, 'init': w.init_override.get(m['name'], m['init'])}) for m in lb.metadata['buffers']]
    return lb, [m['name'] for m in lb.metadata['buffers']], init


@pytest.mark.parametrize('batch,kw', [(1, {}), (3, {'block': 32}), (2, {'head_dim': 64, 'ctx': 15})])
def test_steps_oracle(batch, kw):
    """Steps over a block's end, each from what the one before left."""
    c, w, given = steps.case(batch, **kw)
    lb, names, bufs = _loaded(w, given)
    for _ in range(4):
        after = oracle.run(lb, [x.copy() for x in bufs])['buffers']
        steps.check(c, dict(zip(names, bufs)), dict(zip(names, after)))
        bufs = [np.ascontiguousarray(x) for x in after]


def test_neutral_penalties_leave_the_graph():
    """Without the options the graph is the one over the bf16 cache, without a task of theirs."""
    ops = {t['op'] for t in qwen3.build(qwen3.Qwen3Config.tiny()).spec['graphs'][0]['tasks']}
    assert not ops & {'kv_append_q8', 'attn_decode_q8', 'logits_adjust'}
    ops = {t['op'] for t in qwen3.build(qwen3.Qwen3Config.tiny(cache='q8', presence=0.5)).spec['graphs'][0]['tasks']}
    assert {'kv_append_q8', 'attn_decode_q8', 'logits_adjust'} <= ops and not any(o.startswith('attn_decode_part') for o in ops)


@pytest.mark.parametrize('kw', [{'cache': 'fp4'}, {'cache': 'q8', 'kv_block': 48}, {'cache': 'q8', 'head_dim': 256}, {'repetition': 0.0},
                                {'cache': 'q8', 'heads': 66}])
def test_refusals(kw):
    with pytest.raises(ValueError):
        qwen3.build(qwen3.Qwen3Config.tiny(**kw))


@pytest.mark.gpu
@pytest.mark.parametrize('path', [PATH_DYNAMIC, PATH_STATIC])
@pytest.mark.parametrize('batch,kw', [(1, {}), (3, {'block': 32}), (8, {'block': 64}), (2, {'head_dim': 64, 'ctx': 15})])
def test_steps(batch, kw, path):
    """Six launches of one executor, every step held to the definitions, up to the cache's and the history's last token."""
    print(f'qwen3 q8 steps batch {batch} {kw} path {path}', flush=True)
    c, w, given = steps.case(batch, **kw)
    lb, names, init = _loaded(w, given)
    ex = Executor.from_bundle(lb, buffers=init, path=path)
    before = {n: ex.read(n) for n in names}
    for _ in range(c.max_new):
        ex.relaunch()
        ex.finish()
        after = {n: ex.read(n) for n in names}
        steps.check(c, before, after)
        before = after
    ex.close()


@pytest.mark.gpu
def test_steps_without_reads_between():
    """The same launches one behind the other leave the same buffers."""
    print('qwen3 q8 steps back to back', flush=True)
    c, w, given = steps.case(3)
    lb, names, init = _loaded(w, given)
    left = []
    for reads in (True, False):
        ex = Executor.from_bundle(lb, buffers=[x.copy() for x in init], path=PATH_STATIC)
        for _ in range(5):
            ex.relaunch()
            ex.finish()
            if reads:
                [ex.read(n) for n in names]
        left.append({n: ex.read(n) for n in names if n != 'part'})
        ex.close()
    for n in left[0]:
        np.testing.assert_array_equal(left[0][n], left[1][n], err_msg=n)
