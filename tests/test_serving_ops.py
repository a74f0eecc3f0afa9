"""The serving operators without a GPU: the CPU oracle against the definition in 64 bits, the host's refusals, the task builders
and the operators' order in a graph."""
import numpy as np
import pytest

import oracle
import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import executor
from kvm_amd.workloads import Builder, serving


def _run(lb, init):
    ref = oracle.run(lb, [x.copy() for x in init])
    at = {n: i for i, n in enumerate(sg.names(lb))}
    return lambda n: ref['buffers'][at[n]]


@pytest.mark.parametrize('case', sg.APPENDS, ids=str)
@pytest.mark.parametrize('tasks', [1, 256])
def test_append_oracle(case, tasks):
    blk, hd, hkv, dt, n_new, lens = case
    c, k, v = sg.append_case(case)
    lb, init = sg.append_graph(c, k, v, lens, hkv, n_new, dt, dt, tasks=tasks)
    assert executor.validate(lb) is None
    got, want = sg.cache_of(_run(lb, init), c), f64.append(c, k, v, lens, hkv, n_new, dt == 'bf16')
    for n in sg.CACHE:
        np.testing.assert_array_equal(got[n], want[n], err_msg=n)


@pytest.mark.parametrize('case', sg.ATTENDS, ids=lambda c: str(c)[:60])
def test_attend_oracle(case):
    blk, hd, hkv, heads, dt, n_new, lens = case
    c, q = sg.attend_case(case)
    g = np.random.default_rng(1).random(hd).astype(np.float32) + 0.5
    lb, init = sg.attend_graph(c, q, lens, hkv, heads, n_new, 0.1, dt, dt, gamma=g, theta=1e4, eps=1e-6)
    assert executor.validate(lb) is None
    want, _ = f64.attend(c, q, lens, hkv, heads, n_new, np.float32(0.1), g, np.float32(1e-6), 1e4)
    sg.near(_run(lb, init)('o'), want, 1e-12 * np.abs(want).max(), dt)


@pytest.mark.parametrize('case', sg.ADJUSTS, ids=str)
def test_adjust_oracle(case):
    x, par, g = sg.adjust_case(case)
    lb, init = sg.adjust_graph(x, par, case[2], case[3], **g)
    assert executor.validate(lb) is None
    want, hist, _ = f64.adjust(x, par, **g)
    read = _run(lb, init)
    sg.near(read('out'), want, 1e-14 * np.abs(np.where(np.isfinite(want), want, 0)), case[3])
    if hist is not None:
        np.testing.assert_array_equal(read('hist').reshape(hist.shape), hist)


def test_blocks_that_are_not_finite_or_empty():
    """Zeros and magnitudes whose scale is below the normal numbers give zero bytes; a block with NaN or infinity the scale NaN."""
    x = np.zeros((5, 16, 4), np.float32)
    x[1, 3, 2] = 1e-37
    x[2, 0, 0], x[2, 5, 1] = np.nan, 3
    x[3, 7, 3] = -np.inf
    x[4] = np.float32(3e38)
    q, s = f64.quantise(x)
    assert not q[:4].any() and (q[4] == 127).all()
    assert s[0] == s[1] == 0 and np.isnan(s[2]) and np.isnan(s[3]) and np.isfinite(s[4])
    c = f64.empty_cache(5, 1, 16, 4)
    flat = x.reshape(80, 4)
    lb, init = sg.append_graph(c, flat, flat, [0] * 5, 1, 16, 'f32', 'f32')
    got = sg.cache_of(_run(lb, init), c)
    np.testing.assert_array_equal(got['kq'][:, 0], q)
    np.testing.assert_array_equal(got['ks'][:, 0], s)
    np.testing.assert_array_equal(got['vq'][:, 0], q.transpose(0, 2, 1))


def test_ties_go_to_even():
    """Magnitudes k + 1/2 of a block whose scale is a power of two."""
    x = np.zeros((16, 4), np.float32)
    x.flat[:8] = [254, 1, 3, 5, -1, -3, 251, 253]                        # over 2: 127, .5, 1.5, 2.5, ..
    q, s = f64.quantise(x[None])
    assert s[0] == 2 and q.ravel()[:8].tolist() == [127, 0, 2, 2, 0, -2, 126, 126]


# ------------------------------------------------------------------------------------------------ refusals

def _words(lb, op):
    """{argument: [position in lb.args of every task's word]} of operator `op`."""
    from kvm_amd import abi
    o = abi.load_ops()[op]
    rows = [t for t in lb.tasks if t[0] == o.id]
    return {a.name: [int(t[6]) + i for t in rows] for i, a in enumerate(o.args)}


def _refused(make, op, change, what):
    lb, _ = make()
    assert executor.validate(lb) is None
    w, at = _words(lb, op), {n: i for i, n in enumerate(sg.names(lb))}
    for arg, value in change.items():
        if arg in w:
            word = np.float32(value).view(np.int32) if isinstance(value, float) else at[value] if isinstance(value, str) else value
            for i in w[arg]:
                lb.args[i] = word
        else:
            name, _, key = arg.rpartition('.')
            lb.metadata['buffers'][at[name]][key] = value
    why = executor.validate(lb)
    assert why is not None and what in why, why


def _append():
    case = sg.APPENDS[0]
    c, k, v = sg.append_case(case)
    return sg.append_graph(c, k, v, case[5], case[2], case[4])


def _attend():
    case = sg.ATTENDS[2]
    c, q = sg.attend_case(case)
    return sg.attend_graph(c, q, case[6], case[2], case[3], case[5], 0.1, 'f32', 'f32', tasks=2, gamma=np.ones(case[1], np.float32))


def _adjust():
    x, par, g = sg.adjust_case(sg.ADJUSTS[3])
    return sg.adjust_graph(x, par, **g)


@pytest.mark.parametrize('change,what', [
    ({'blk': 48}, 'blk must be'), ({'blk': 128}, 'too small'), ({'hd': 130}, 'hd must be'), ({'hd': 64}, 'hd / 4 columns'), ({'n_new': 0}, 'n_new'),
    ({'b1': 9}, 'too small'), ({'b0': -1}, 'range'), ({'h1': 3}, 'h0/h1'), ({'p': 1}, 'p/P'), ({'theta': -1.0}, 'theta'), ({'eps': float('nan')}, 'eps'),
    ({'vq': 'kq'}, 'of their own'), ({'vt': 'kt'}, 'of their own'), ({'lens': 'ks'}, 'i32'), ({'kq': 'kt'}, 'i32'), ({'ks': 'kt'}, 'f32'),
    ({'kgamma': 'ks', 'hd': 128}, 'too small'), ({'vs.cols': 3}, 'same columns'), ({'knew.rows': 6}, 'too small'), ({'vnew.cols': 255}, 'too small'),
    ({'kq.rows': 1}, 'too small'), ({'vt.rows': 100}, 'too small')], ids=str)
def test_append_refusals(change, what):
    _refused(_append, 'kv_append_q8', change, what)


@pytest.mark.parametrize('change,what', [
    ({'n_new': 17}, '1 .. 32'), ({'n_new': 0}, '1 .. 32'), ({'H': 5}, 'H/Hkv'), ({'Hkv': 0}, 's/S'), ({'s': 2}, 's/S'), ({'s': -1}, 's/S'),
    ({'b1': 6}, 'too small'), ({'b0': -1}, 'range'), ({'b1': 1030}, '1024'), ({'S': 4}, 'too small'), ({'o': 'q'}, 'o must not be q'), ({'scale': float('inf')}, 'scale'), ({'theta': -2.0}, 'theta'),
    ({'cnt': 'q'}, 'i32'), ({'q': 'lens'}, 'f32 or bf16'), ({'qgamma': 'lens'}, 'f32'), ({'o.part.cols': 129}, 'too small'), ({'blk': 0}, 'blk')], ids=str)
def test_attend_refusals(change, what):
    _refused(_attend, 'attn_decode_q8', change, what)


@pytest.mark.parametrize('change,what', [
    ({'v1': 5000}, 'v0/v1/V'), ({'v0': -1}, 'v0/v1/V'), ({'V': 5000}, 'too small'), ({'r1': 6}, 'too small'), ({'plen': -1}, 'go together'),
    ({'hist': -1}, 'go together'), ({'bval': -1}, 'go together'), ({'mask': -1}, 'mrow needs mask'), ({'bidx.cols': 2048}, '2047'),
    ({'par.cols': 2}, 'too small'), ({'mask.cols': 100}, 'too small'), ({'hist.cols': 1 << 20}, '2^20'), ({'logits': 'hist'}, 'f32 or bf16'),
    ({'last': 'par'}, 'i32')], ids=str)
def test_adjust_refusals(change, what):
    _refused(_adjust, 'logits_adjust', change, what)


def test_builder_refusals():
    with pytest.raises(ValueError, match='blk'):
        serving.kv_q8_buffers(Builder(0), 'x', 1, 1, 128, 64, blk=48)
    with pytest.raises(ValueError, match='hd'):
        serving.kv_q8_buffers(Builder(0), 'x', 1, 1, 129, 64)
    b = Builder(0)
    c = serving.kv_q8_buffers(b, 'x', 1, 1, 128, 65)
    assert c.tmax == 128
    with pytest.raises(ValueError, match='at most 32'):
        serving.attn_decode_q8(b, c, 'q', 'o', 'lens', 16, n_new=3)


@pytest.mark.parametrize('make,op,change', [
    (_append, 'kv_append_q8', {'knew': 'kt', 'kt.cols': 256}), (_append, 'kv_append_q8', {'vnew': 'vt', 'vt.cols': 256}),
    (_attend, 'attn_decode_q8', {'o': 'kt', 'kt.cols': 4096, 'kt.rows': 99999}), (_attend, 'attn_decode_q8', {'o': 'o.part', 'o.part.cols': 4096}),
    (_attend, 'attn_decode_q8', {'q': 'o.part', 'o.part.cols': 4096}), (_attend, 'attn_decode_q8', {'cnt': 'lens', 'lens.rows': 4096}),
    (_adjust, 'logits_adjust', {'hist': 'bidx'}), (_adjust, 'logits_adjust', {'mask': 'hist'}), (_adjust, 'logits_adjust', {'out': 'par', 'par.cols': 9999})],
    ids=str)
def test_written_buffers_are_no_inputs(make, op, change):
    _refused(make, op, change, 'a buffer of its own')


@pytest.mark.parametrize('theta', [0.5, 1e-30, float('inf')])
def test_rotation_bases_below_one(theta):
    _refused(_append, 'kv_append_q8', {'theta': theta}, 'theta')
    _refused(_attend, 'attn_decode_q8', {'theta': theta}, 'theta')


def test_more_sequences_than_a_call():
    """Two layers of 1,500 sequences share a workspace: two calls each, with a part each."""
    b = Builder(0)
    c = serving.kv_q8_buffers(b, 'c', 1500, 1, 64, 64)
    b.fill('q', 1500, 64), b.fill('o', 1500, 64), b.fill('lens', 1500, 1, 'i32'), b.fill('p', 8, 66), b.fill('n', 1500, 1, 'i32')
    for _ in range(2):
        ids = serving.attn_decode_q8(b, c, 'q', 'o', 'lens', 1, part='p', cnt='n', tasks=4)
    tasks = [t['args'] for t in b.spec()['graphs'][0]['tasks']]
    assert len(ids) == 8 and sorted({(t['b0'], t['b1'], t['part']) for t in tasks}) == [(0, 1024, 'p'), (1024, 1500, 'p.1')]
    lb, _ = sg.compiled(b, {})
    assert executor.validate(lb) is None


@pytest.mark.parametrize('lens', [[63 - 64 * 2], [-2], [128]])
def test_lengths_out_of_range(lens):
    case = sg.APPENDS[0]
    c = f64.empty_cache(2, 2, 64, 128)
    x = np.zeros((1, 256), np.float32)
    for lb, init in (sg.append_graph(c, x, x, lens, 2, 1), sg.attend_graph(c, x, lens, 2, 2, 1, 1.0)):
        with pytest.raises(oracle.OracleError, match='length'):
            oracle.run(lb, init)
    assert case
