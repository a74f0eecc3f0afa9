"""The operators that serve prompts and tokens together (ops 315-319) without a GPU: the CPU oracle against the definition in 64 bits, the
host's refusals, what the task builders lay out."""
import numpy as np
import pytest

import mixed_fp64 as f64
import mixed_graphs as mg
import oracle
import serving_graphs as sg
from kvm_amd import executor
from kvm_amd.workloads import Builder, serving


def _run(lb, init):
    ref = oracle.run(lb, [x.copy() for x in init])
    return {n: ref['buffers'][i] for i, n in enumerate(sg.names(lb))}


@pytest.mark.parametrize('case', mg.ROWS, ids=str)
def test_rows_oracle(case):
    M, K, pro, dt, cols = case
    x, x2, g = mg.rows_case(case)
    lb, init = mg.rows_graph(x, x2, g, dt, cols, K)
    assert executor.validate(lb) is None
    got = _run(lb, init)
    v = f64.shaped(x, pro, x2, g, 1e-6)
    q, s = f64.quantise(v)
    y = got['y'].view(np.int8).reshape(M, -1)
    if pro == 2:                                                       # the definition's v is exact there, the oracle's its f32
        assert (np.abs(y[:, :K] - v / s[:, None]) <= 0.5 + 1e-4).all()
    else:
        np.testing.assert_array_equal(y[:, :K], q)
    np.testing.assert_array_equal(got['ys'], s)
    assert not y[:, K:].any() and y.shape[1] == -(-K // 16) * 16


@pytest.mark.parametrize('case', mg.PRODUCTS, ids=str)
@pytest.mark.parametrize('tile', [0, 1, 2])
def test_product_oracle(case, tile):
    args = mg.product_case(case)
    lb, init = mg.product_graph(case, *args, tile)
    assert executor.validate(lb) is None
    want, bound = f64.product(*args)
    f64.near(_run(lb, init)['out'].reshape(want.shape), want, bound, case[4])


@pytest.mark.parametrize('case', mg.GEMVS, ids=str)
def test_gemv_oracle_is_rows_then_product(case):
    args = mg.gemv_case(case)
    got = []
    for fused in (True, False, None):
        lb, init = mg.gemv_graph(case, *args, fused=fused)
        assert executor.validate(lb) is None
        got.append(_run(lb, init)['out'])
    np.testing.assert_array_equal(got[0], got[1])
    np.testing.assert_array_equal(got[0], got[2])


@pytest.mark.parametrize('case', mg.APPENDS, ids=str)
def test_append_oracle(case):
    (lb, init), pg, q, want = mg.append_graph(case, np.random.default_rng(1))
    assert executor.validate(lb) is None
    got = _run(lb, init)
    for n, w in zip(('kc', 'vc'), want):
        f64.near(got[n].reshape(w.shape), w, 1e-12, case[4])
    on = ~np.isnan(want[2])
    o = got['qo'].reshape(want[2].shape)
    f64.near(o[on], want[2][on], 1e-12, case[4])
    assert (o[~on] == 7).all()


@pytest.mark.parametrize('case', mg.ATTENDS, ids=str)
def test_attend_oracle(case):
    (lb, init), pg, q = mg.attend_graph(case, np.random.default_rng(2), tasks=3)
    assert executor.validate(lb) is None
    want, mag = f64.attend(q, *pg, case[0], 1 / np.sqrt(case[1]))
    o, on = _run(lb, init)['o'].reshape(want.shape), ~np.isnan(want)
    f64.near(o[on], want[on], 1e-6 * mag[on], case[4])
    assert (o[~on] == 7).all()


# ------------------------------------------------------------------------------------------------ refusals

def _refused(lb, op, change, what):
    """The bundle with an argument of `op`, or a buffer's rows or cols, changed is refused with `what`."""
    at = {n: i for i, n in enumerate(sg.names(lb))}
    sig = [a.split(':')[0] for a in next(o for o in _signatures() if o[0] == op)[1].split(',')]
    for arg, value in change.items():
        if '.' in arg:
            name, _, key = arg.rpartition('.')
            lb.metadata['buffers'][at[name]][key] = value
            continue
        word = at[value] if isinstance(value, str) else np.float32(value).view(np.int32) if isinstance(value, float) else value
        ids = {o[0]: o[2] for o in _signatures()}
        for t in lb.tasks.reshape(-1, 16):
            if t[0] == ids[op]:
                lb.args[t[6] + sig.index(arg)] = word
    why = executor.validate(lb)
    assert why is not None and what in why, why


def _signatures():
    import re
    from kvm_amd.executor import HEADER
    text = (HEADER.parent / 'mvm_ops_kvm.def').read_text()
    return [(m[1], m[3], int(m[2])) for m in re.finditer(r'^X\((\w+),\s*(\d+), "([^"]*)"\)', text, re.M)]


def _rows(i=4):
    x, x2, g = mg.rows_case(mg.ROWS[i])
    return mg.rows_graph(x, x2, g, *mg.ROWS[i][3:], mg.ROWS[i][1])[0]


@pytest.mark.parametrize('change,what', [
    ({'K': 0}, 'K must be'), ({'K': 131072}, 'K must be'), ({'K': 1009}, 'too small'), ({'pro': 3}, 'pro must be'), ({'pro': 0}, 'gamma goes'), ({'pro': 2}, 'gamma goes'), ({'gamma': -1}, 'gamma goes'),
    ({'r1': 7}, 'too small'), ({'r0': -1}, 'range'), ({'eps': float('nan')}, 'eps'), ({'eps': -1.0}, 'eps'), ({'y.cols': 250}, 'too small'), ({'ys.rows': 1}, 'too small'),
    ({'q': 'x'}, 'i32'), ({'qs': 'y'}, 'f32'), ({'qs': 'g', 'r1': 1}, 'of its own'), ({'gamma': 'x'}, 'f32'), ({'x': 'y'}, 'f32 or bf16')], ids=str)
def test_rows_refusals(change, what):
    _refused(_rows(), 'rows_q8', change, what)


def _product(i=3):
    return mg.product_graph(mg.PRODUCTS[i], *mg.product_case(mg.PRODUCTS[i]), 2)[0]


@pytest.mark.parametrize('change,what', [
    ({'M': 66}, 'too small'), ({'N': 131}, 'too small'), ({'K': 209}, 'too small'), ({'K': 0}, 'K must be'), ({'K': 200000}, 'K must be'), ({'tile': 3}, 'tile'), ({'tile': -1}, 'tile'),
    ({'m0': 65}, 'm0/n0'), ({'n0': -64}, 'm0/n0'), ({'M': 0}, 'm0/n0'), ({'a': 'sa'}, 'i32'), ({'sw': 'a'}, 'f32'), ({'out': 'a'}, 'f32 or bf16'), ({'bias': 'res'}, 'f32'),
    ({'sa.rows': 64}, 'too small'), ({'bias.cols': 129}, 'too small'), ({'res.rows': 64}, 'too small'), ({'out.cols': 129}, 'too small'),
    ({'sa': 'out', 'out.dtype': 0}, 'of its own')], ids=str)
def test_product_refusals(change, what):
    _refused(_product(), 'matmul_q8', change, what)


def _gemv(i=4):
    return mg.gemv_graph(mg.GEMVS[i], *mg.gemv_case(mg.GEMVS[i]))[0]


@pytest.mark.parametrize('change,what', [
    ({'M': 17}, 'M must be'), ({'M': 0}, 'M must be'), ({'pro': 4}, 'pro 0 .. 3'), ({'pro': 3}, 'x must be i32'), ({'pro': 1}, 'gamma goes'), ({'x': 'w'}, 'x must be i32'), ({'sx': 'sw'}, 'sx goes'),
    ({'K': 0}, 'K must be'), ({'K': 785}, 'too small'), ({'n0': -1}, 'range'), ({'n1': 51}, 'too small'), ({'w': 'x'}, 'i32'), ({'sw': 'x'}, 'f32'), ({'w.cols': 194}, 'too small'),
    ({'out': 'x'}, 'of its own'), ({'x2': 'out', 'out.cols': 784}, 'of its own'), ({'bias.cols': 49}, 'too small'), ({'eps': float('inf')}, 'eps')], ids=str)
def test_gemv_refusals(change, what):
    _refused(_gemv(), 'gemv_q8', change, what)


@pytest.mark.parametrize('change,what', [
    ({'page': 48}, 'page must be'), ({'page': 0}, 'page must be'), ({'hd': 127}, 'hd must be'), ({'hd': 258}, 'hd must be'), ({'hd': 256}, 'too small'), ({'B': 0}, 'B must be'), ({'B': 1025}, 'B must be'),
    ({'B': 5}, 'too small'), ({'Hkv': 0}, 'B must be'), ({'Hkv': 4096}, 'a page at least'), ({'H': 0}, 'go together'), ({'q': -1}, 'go together'), ({'qo': -1}, 'go together'), ({'q': -1, 'qo': -1}, 'qgamma needs'),
    ({'r0': -1}, 'range'), ({'r1': 400}, 'too small'), ({'theta': 0.5}, 'theta'), ({'eps': -1.0}, 'eps'), ({'kc': 'k'}, 'same rows'), ({'kc': 'vc'}, 'of its own'), ({'qo': 'k', 'k.cols': 4096}, 'of its own'),
    ({'table': 'k'}, 'i32'), ({'cu': 'qg'}, 'i32'), ({'kgamma': 'k'}, 'f32'), ({'vc.rows': 1}, 'same rows'), ({'table.cols': 1 << 26}, 'table must have'), ({'kc.cols': 100}, 'too small')], ids=str)
def test_append_refusals(change, what):
    (lb, _), *_ = mg.append_graph(mg.APPENDS[2], np.random.default_rng(0))
    _refused(lb, 'qkv_append_paged', change, what)


@pytest.mark.parametrize('change,what', [
    ({'page': 24}, 'page must be'), ({'hd': 0}, 'hd must be'), ({'B': 0}, 'B must be'), ({'H': 7}, 's/S/H/Hkv'), ({'Hkv': 0}, 'B must be'), ({'s': 256}, 's/S/H/Hkv'), ({'s': -1}, 's/S/H/Hkv'),
    ({'S': 70000}, 's/S/H/Hkv'), ({'S': 300}, 'too small'), ({'tile': 3}, 'tile must be'), ({'tile': 129}, 'tile must be'), ({'scale': 0.0}, 'scale'), ({'scale': -1.0}, 'scale'),
    ({'scale': float('nan')}, 'scale'), ({'o': 'q'}, 'of its own'), ({'o': 'kc'}, 'too small'), ({'part': 'q'}, 'f32'), ({'cnt': 'lens', 'lens.rows': 512}, 'of its own'), ({'o.rows': 5}, 'same rows'),
    ({'o.part.cols': 129}, 'too small'), ({'o.cnt.rows': 255}, 'too small'), ({'q': 'lens'}, 'f32 or bf16'), ({'q.cols': 1023}, 'too small'), ({'kc.rows': 31, 'vc.rows': 31}, 'a page at least')], ids=str)
def test_attend_refusals(change, what):
    (lb, _), *_ = mg.attend_graph(mg.ATTENDS[1], np.random.default_rng(0))
    _refused(lb, 'attn_paged', change, what)


@pytest.mark.parametrize('change', [{'H': 65537}, {'Hkv': 65537}], ids=str)
def test_more_heads_than_row_counts_hold(change):
    _refused(mg.append_graph(mg.APPENDS[2], np.random.default_rng(0))[0][0], 'qkv_append_paged', change, 'at most 65536')
    _refused(mg.attend_graph(mg.ATTENDS[1], np.random.default_rng(0))[0][0], 'attn_paged', change, 'at most 65536')


def test_builder_refusals():
    b = Builder(0)
    with pytest.raises(ValueError, match='page'):
        serving.paged_buffers(b, 'x', 4, 1, 128, page=8)
    with pytest.raises(ValueError, match='hd'):
        serving.paged_buffers(b, 'x', 4, 1, 257)
    c = serving.paged_buffers(b, 'c', 4, 2, 64)
    for n, r, k in (('q', 9, 256), ('o', 9, 256), ('k', 9, 128), ('v', 9, 128)):
        b.fill(n, r, k, 'bf16')
    b.fill('cu', 1026, 1, 'i32'), b.fill('lens', 1025, 1, 'i32'), b.fill('table', 1025, 4, 'i32')
    with pytest.raises(ValueError, match='1024'):
        serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', 4)
    with pytest.raises(ValueError, match='1024'):
        serving.qkv_append_paged(b, c, 'k', 'v', 'table', 'lens', 'cu')
    b.fill('cu2', 3, 1, 'i32')
    with pytest.raises(ValueError, match='heads'):
        serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu2', 5)
    with pytest.raises(ValueError, match='exclude'):
        serving.rows_q8(b, 'q', serving.rows_q8_buffers(b, 'y', 9, 256), 9, x2='o', gamma='k')
    w = serving.weight_q8_buffers(b, 'w', 40, 128)
    with pytest.raises(ValueError, match='with the K'):
        serving.linear_q8(b, serving.RowsQ8('y', 'ys', 9, 256), w, 'o', 9)
    with pytest.raises(ValueError, match='workspace'):
        serving.linear_q8(b, 'k', w, 'o', 9, rows=serving.RowsQ8('y', 'ys', 9, 256))


@pytest.mark.parametrize('what', ['falling', 'rows', 'negative', 'length', 'room', 'page', 'unset'])
def test_bad_tables(what):
    """Row numbers that fall or end behind the buffers, lengths below zero or past the table, pages that are none: errors, nothing written."""
    def spoil(x):
        x = [y.copy() for y in x]
        kc, vc, table, lens, cu = x
        if what == 'falling':
            cu[1] = cu[2] + 1
        if what == 'rows':
            cu[-1] += 5
        if what == 'negative':
            cu[0] = -1
        if what == 'length':
            lens[0] = -2
        if what == 'room':
            lens[0] = 16 * table.shape[1]
        if what == 'page':
            table[0, 0] = len(kc)
        if what == 'unset':
            table[0, 0] = -1
        return x
    case = mg.ATTENDS[0]
    for make in (mg.attend_graph, mg.append_graph):
        (lb, init), pg, *_ = make(case[:6] + (case[6],) if make is mg.attend_graph else mg.APPENDS[0], np.random.default_rng(3))
        names = sg.names(lb)
        for n, x in zip(('kc', 'vc', 'table', 'lens', 'cu'), spoil(pg)):
            if n not in ('kc', 'vc'):
                init[names.index(n)] = x.reshape(-1)
        with pytest.raises(oracle.OracleError):
            oracle.run(lb, [x.copy() for x in init])


def test_forms_by_rows():
    """One row is quantised in the product's own tasks; more go through rows_q8; above 16 the product is tiles."""
    for M, ops in ((1, {'gemv_q8'}), (2, {'rows_q8', 'gemv_q8', 'noop'}), (16, {'rows_q8', 'gemv_q8', 'noop'}), (17, {'rows_q8', 'matmul_q8', 'noop'})):
        b = Builder(0)
        b.fill('x', M, 64), b.fill('o', M, 4096)
        serving.linear_q8(b, 'x', serving.weight_q8_buffers(b, 'w', 4096, 64), 'o', M)
        assert {t['op'] for t in b.spec()['graphs'][0]['tasks']} | {'noop'} == ops | {'noop'}
