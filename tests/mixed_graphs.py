"""Graphs and cases of the operators that serve prompts and tokens together (ops 315-319), for the oracle and for the GPU."""
import numpy as np

import mixed_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd.workloads import Builder, serving


def bf(x, dtype):
    return bl.bf16_round(x.astype(np.float32)) if dtype == 'bf16' else x.astype(np.float32)


def words(q, width):
    """Rows of bytes as rows of `width` i32 words, 77s behind their end."""
    out = np.full((q.shape[0], 4 * width), 77, np.int8)
    out[:, :q.shape[1]] = q
    return out.view(np.int32)


# ------------------------------------------------------------------------------------------------ rows and products

# (rows, K, pro, dtype, columns of x): one value, ragged and whole rows, every form of the kernel (4,096 and 16,384 values a row, longer, unaligned)
ROWS = [(1, 1, 0, 'f32', 1), (5, 7, 1, 'bf16', 8), (3, 60, 2, 'bf16', 64), (9, 1001, 0, 'f32', 1001), (6, 1001, 1, 'bf16', 1008), (7, 4096, 1, 'bf16', 4096),
        (3, 4099, 1, 'f32', 4100), (2, 12288, 2, 'bf16', 12288), (3, 16384, 1, 'f32', 16384), (2, 16390, 1, 'bf16', 16392), (2, 20001, 2, 'f32', 20001),
        (21, 1001, 1, 'bf16', 1001), (5, 777, 2, 'bf16', 777), (3, 5003, 1, 'bf16', 5003), (2, 16401, 2, 'bf16', 16401), (9, 1002, 0, 'bf16', 1002), (4, 12288, 2, 'f32', 12288)]


def rows_case(case, seed=0):
    M, K, pro, dt, cols = case
    rng = np.random.default_rng([seed, M, K, pro])
    x = bf(rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1))), dt)
    x2 = bf(rng.standard_normal((M, K)), dt) if pro == 2 else None
    g = (rng.random(K) + 0.5).astype(np.float32) if pro == 1 else None
    return x, x2, g


def add_rows(b, data, x, x2, g, dt, cols):
    wide = lambda a: np.pad(a, ((0, 0), (0, cols - a.shape[1])), constant_values=9)   # noqa: E731
    sg.add(b, data, 'x', wide(x), dt)
    if x2 is not None:
        sg.add(b, data, 'x2', wide(x2), dt)
    if g is not None:
        sg.add(b, data, 'g', g[None])
    return dict(x2='x2' if x2 is not None else None, gamma='g' if g is not None else None)


def rows_graph(x, x2, g, dt, cols, K, eps=1e-6, width=None, tasks=256):
    b, data = Builder(0), {}
    kw = add_rows(b, data, x, x2, g, dt, cols)
    y = serving.rows_q8_buffers(b, 'y', len(x), K)
    if width:
        b.buffers[-2]['cols'] = width
    data['y'] = np.full((len(x), b.buffers[-2]['cols']), 0x4d4d4d4d, np.int32)
    serving.rows_q8(b, 'x', y, len(x), eps=eps, tasks=tasks, **kw)
    return sg.compiled(b, data)


# (M, N, K, words of a row, dtype of out, bias, res): every tile, sizes around them, rows that are no whole vectors, K from one byte on
PRODUCTS = [(1, 1, 1, 1, 'f32', False, False), (17, 70, 5, 4, 'bf16', True, False), (64, 64, 64, 16, 'f32', False, True), (65, 130, 200, 52, 'bf16', True, True),
            (130, 257, 1001, 252, 'f32', True, False), (128, 256, 127, 32, 'bf16', False, True), (200, 300, 333, 85, 'f32', False, False), (33, 19, 4100, 1028, 'bf16', False, False),
            (129, 513, 640, 160, 'bf16', False, True)]


def product_case(case, seed=0):
    M, N, K, width, dt, bias, res = case
    rng = np.random.default_rng([seed, M, N, K])
    a, w = (rng.integers(-127, 128, (r, K)).astype(np.int8) for r in (M, N))
    if K > 4:
        a[0], w[0] = 127, 127
        w[-1] = -128                                                   # a caller's own weights may hold it
    return (a, rng.random(M).astype(np.float32), w, (rng.random(N) - 0.5).astype(np.float32), rng.standard_normal(N).astype(np.float32) if bias else None,
            bf(rng.standard_normal((M, N)), dt) if res else None)


def product_graph(case, a, sa, w, sw, bias, res, tile, inplace=False):
    M, N, K, width, dt, *_ = case
    b, data = Builder(0), {}
    for n, x in (('a', words(a, width)), ('sa', sa[:, None]), ('w', words(w, width)), ('sw', sw[:, None])):
        sg.add(b, data, n, x)
    if bias is not None:
        sg.add(b, data, 'bias', bias[None])
    if res is not None:
        sg.add(b, data, 'res', res, dt)
    out = 'res' if inplace else b.fill('out', M, N, dt, value=7.0)
    tm, tn = ((128, 256), (128, 128), (64, 64))[tile]
    for m0 in range(0, M, tm):
        for n0 in range(0, N, tn):
            b.task('matmul_q8', a='a', sa='sa', w='w', sw='sw', out=out, bias='bias' if bias is not None else None, res='res' if res is not None else None, m0=m0, n0=n0,
                   M=M, N=N, K=K, tile=tile)
    return sg.compiled(b, data)


# (M, N, K, words of a weight row, dtype, pro, bias, res, columns of x): gemv forms of every K, chunks of K (many rows of it), unaligned weights
GEMVS = [(1, 1, 1, 1, 'f32', 0, False, False, 1), (1, 40, 512, 128, 'bf16', 1, False, True, 512), (1, 333, 4096, 1024, 'bf16', 1, True, False, 4096),
         (3, 64, 1000, 252, 'f32', 0, False, False, 1000), (16, 50, 777, 196, 'bf16', 2, True, True, 784), (8, 37, 12288, 3076, 'bf16', 2, False, False, 12288),
         (2, 20, 5001, 1251, 'f32', 1, False, False, 5001), (16, 130, 6145, 1540, 'bf16', 1, False, True, 6152), (1, 300, 20480, 5120, 'bf16', 1, False, False, 20480)]


def gemv_graph(case, x, x2, g, w, sw, bias, res, fused=True, parts=3, eps=1e-6, after_rows=False):
    """The product of rows that the tasks quantise themselves (fused), or that rows_q8 does in front of them (pro 3), or as tiles (fused None)."""
    M, N, K, width, dt, pro, _, _, cols = case
    b, data = Builder(0), {}
    kw = add_rows(b, data, x, x2, g, dt, cols)
    sg.add(b, data, 'w', words(w, width)), sg.add(b, data, 'sw', sw[:, None])
    if bias is not None:
        sg.add(b, data, 'bias', bias[None])
    if res is not None:
        sg.add(b, data, 'res', res, dt)
    b.fill('out', M, N, dt, value=7.0)
    common = dict(w='w', sw='sw', out='out', bias='bias' if bias is not None else None, res='res' if res is not None else None, K=K, M=M)
    cuts = sorted({0, N} | {N * i // parts for i in range(parts)})
    if fused:
        for n0, n1 in zip(cuts, cuts[1:]):
            b.task('gemv_q8', x='x', sx=None, n0=n0, n1=n1, pro=pro, eps=eps, **kw, **common)
        return sg.compiled(b, data)
    y = serving.rows_q8_buffers(b, 'y', M, K)
    t = serving.rows_q8(b, 'x', y, M, eps=eps, **kw)
    if fused is None:
        for m0 in range(0, M, 64):
            for n0 in range(0, N, 64):
                b.task('matmul_q8', after=t, a='y', sa='ys', m0=m0, n0=n0, N=N, tile=2, **common)
    else:
        for n0, n1 in zip(cuts, cuts[1:]):
            b.task('gemv_q8', after=t, x='y', sx='ys', x2=None, gamma=None, n0=n0, n1=n1, pro=3, eps=0.0, **common)
    return sg.compiled(b, data)


def gemv_case(case, seed=0):
    M, N, K, width, dt, pro, bias, res, cols = case
    x, x2, g = rows_case((M, K, pro, dt, cols), seed)
    rng = np.random.default_rng([seed, M, N, K, 7])
    return (x, x2, g, rng.integers(-127, 128, (N, K)).astype(np.int8), (rng.random(N) - 0.5).astype(np.float32) / K, rng.standard_normal(N).astype(np.float32) if bias else None,
            bf(rng.standard_normal((M, N)), dt) if res else None)


# ------------------------------------------------------------------------------------------------ paged cache

def paged(rng, lens, new, page, hkv, hd, dtype, spare=2, first=0, unseen=np.nan):
    """A cache with the sequences' pages in no order, tokens that no sequence has `unseen`, and its tables: (kc, vc, table, lens, cu)."""
    lens, new = np.asarray(lens), np.asarray(new)
    used = -(-(lens + new) // page)
    width, pages = max(1, used.max()), used.sum() + spare
    order = iter(rng.permutation(pages))
    table = np.full((len(lens), width), -1, np.int32)
    kc, vc = (np.full((pages, hkv, page, hd), unseen, np.float32) for _ in range(2))
    for b, n in enumerate(used):
        table[b, :n] = [next(order) for _ in range(n)]
        t = np.arange(lens[b])
        for x in (kc, vc):
            x[table[b, t // page], :, t % page] = bf(rng.standard_normal((lens[b], hkv, hd)), dtype)
    return kc, vc, table, lens.astype(np.int32), (first + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)


def add_paged(b, data, kc, vc, table, lens, cu, page, dtype, extra=0):
    pages, hkv, _, hd = kc.shape
    c = serving.paged_buffers(b, '', pages, hkv, hd, page, dtype)
    for n, x in (('kc', kc), ('vc', vc)):
        data[n] = np.pad(x.reshape(-1, hd), ((0, 0), (0, extra)), constant_values=5).astype(np.float32)
    for m in b.buffers[-2:]:
        m['cols'] += extra
    sg.add(b, data, 'table', table), sg.add(b, data, 'lens', lens[:, None]), sg.add(b, data, 'cu', cu[:, None])
    return c


# (page, hd, kv heads, heads, dtype, lengths, new tokens): pages that end inside tiles, first tokens, sequences that bring none, prompts and tokens together
APPENDS = [(16, 64, 2, 4, 'bf16', [0, 15, 16, 100], [1, 1, 1, 1]), (64, 128, 1, 3, 'f32', [0, 63, 200], [70, 2, 0]), (128, 128, 2, 16, 'bf16', [5, 0, 0, 127], [0, 300, 0, 3]),
           (32, 100, 2, 2, 'f32', [0, 31], [40, 1]), (16, 6, 3, 6, 'bf16', [9], [33]), (16, 256, 1, 2, 'bf16', [30, 0], [2, 1])]


def append_graph(case, rng, gamma=True, theta=1e6, queries=True, first=0, behind=3, extra=0, tasks=256, inplace=False, unseen=7.0):
    page, hd, hkv, heads, dt, lens, new = case
    pg = paged(rng, lens, new, page, hkv, hd, dt, first=first, unseen=unseen)
    rows = int(pg[4][-1]) + behind
    q, k, v = (bf(rng.standard_normal((rows, h, hd)), dt) for h in (heads, hkv, hkv))
    gs = [(rng.random(hd) + 0.5).astype(np.float32) if gamma else None for _ in range(2)]
    b, data = Builder(0), {}
    c = add_paged(b, data, *pg, page, dt, extra)
    for n, x in (('q', q), ('k', k), ('v', v)):
        sg.add(b, data, n, np.pad(x.reshape(rows, -1), ((0, 0), (0, extra)), constant_values=3), dt)
    if queries and not inplace:
        b.fill('qo', rows, heads * hd + extra, dt, value=7.0)
    for n, g in zip(('qg', 'kg'), gs):
        if g is not None:
            sg.add(b, data, n, g[None])
    names = dict(q='q', qo='q' if inplace else 'qo', heads=heads, qgamma='qg' if gamma else None) if queries else {}
    serving.qkv_append_paged(b, c, 'k', 'v', 'table', 'lens', 'cu', kgamma='kg' if gamma else None, theta=theta, eps=1e-6, tasks=tasks, **names)
    want = f64.append(*pg, q if queries else None, k, v, page, *gs, 1e-6, theta)
    return sg.compiled(b, data), pg, q, want


# (page, hd, kv heads, heads, dtype, lengths, new tokens, tile or 0): tiles of every kind (up to 32 rows, more), long and cut ones, groups of 1 to 24,
# head sizes of the matrix units and others, sequences that bring nothing, first tokens
ATTENDS = [
    (16, 64, 2, 2, 'bf16', [0, 15, 16, 100, 31], [1, 1, 1, 1, 0]),
    (64, 128, 2, 8, 'bf16', [0, 63, 64, 700, 1500], [1, 1, 1, 1, 1]),
    (32, 128, 1, 4, 'bf16', [0, 0, 500, 77], [300, 1, 70, 0]),
    (16, 128, 2, 10, 'bf16', [33, 1], [40, 6]),
    (128, 64, 1, 8, 'bf16', [900, 127], [4, 200]),
    (64, 64, 2, 6, 'bf16', [10, 2500], [129, 9]),
    (16, 128, 1, 24, 'bf16', [64, 300], [1, 5]),
    (16, 64, 2, 4, 'f32', [0, 100, 40], [33, 1, 0]),
    (32, 128, 1, 1, 'f32', [70], [45]),
    (64, 100, 2, 6, 'bf16', [130, 5], [3, 20]),
    (16, 6, 1, 3, 'f32', [50], [7]),
    (128, 256, 1, 2, 'f32', [200], [19]),
    (16, 128, 1, 48, 'f32', [20, 3], [2, 1]),
]


def attend_graph(case, rng, tasks=256, first=0, behind=3, extra=0, n_max=0, q=None, kv=None, odt=None, scale=None, table=None):
    page, hd, hkv, heads, dt, lens, new = case
    pg = paged(rng, np.asarray(lens) + np.asarray(new), np.zeros(len(new), int), page, hkv, hd, dt, first=first)
    kc, vc, tb = pg[:3]
    if kv is not None:
        kc, vc = kv(kc, vc, tb)
    pg = (kc, vc, tb if table is None else table(tb), np.asarray(lens, np.int32), (first + np.concatenate([[0], np.cumsum(new)])).astype(np.int32))
    rows = int(pg[4][-1]) + behind
    q = bf(2 * rng.standard_normal((rows, heads, hd)), dt) if q is None else q(rows)
    b, data = Builder(0), {}
    c = add_paged(b, data, *pg, page, dt, extra)
    sg.add(b, data, 'q', np.pad(q.reshape(rows, -1), ((0, 0), (0, extra)), constant_values=3), dt)
    b.fill('o', rows, heads * hd + extra, odt or dt, value=7.0)
    serving.attn_paged(b, c, 'q', 'o', 'table', 'lens', 'cu', heads, n_max=n_max, tasks=tasks, scale=scale)
    return sg.compiled(b, data), pg, q


def attend_bound(case, mag, sabs, exact_p):
    """What 32-bit evaluation may be off by, relative to the weighted magnitudes `mag` of the values: a score by a step for each of its hd + 4
    products, sums and factors (twice: the matrix units round sums towards zero) times the largest sum of magnitudes `sabs`, which is what its
    weight is off by, relatively, twice over (the weight and the sum of weights); sums of up to n terms and the merge; bf16 weights by half a step."""
    n = max(np.asarray(case[5]) + np.asarray(case[6]))
    delta = (case[1] + 4) * 2 * f64.U * sabs
    return mag * (2 * delta + (n + 64) * 2 * f64.U + (0 if exact_p else 2.0 ** -8))
