"""Graphs of the serving operators for the tests: one call of an operator with given contents, on the oracle or on the GPU."""
import numpy as np

from kvm_amd import bundle as bl
from kvm_amd import compiler
from kvm_amd.workloads import Builder, serving

CACHE = ('kq', 'ks', 'vq', 'vs', 'kt', 'vt')


def add(b, data, name, x, dtype=None):
    """A buffer of array x (2-d) with x as its contents."""
    x = np.asarray(x)
    dtype = dtype or {'i': 'i32', 'f': 'f32'}[x.dtype.kind]
    data[name] = x.astype(np.int32 if dtype == 'i32' else np.float32)
    return b.fill(name, *x.shape, dtype)


def add_cache(b, data, c, hkv, dtype):
    pairs, nblk, blk, hd = c['kq'].shape
    cache = serving.kv_q8_buffers(b, '', pairs // hkv, hkv, hd, nblk * blk, blk, dtype)
    for n in CACHE:
        x = np.ascontiguousarray(c[n])
        data[n] = x.view(np.int32) if n[1] == 'q' else x
    return cache


def compiled(b, data):
    """(bundle, contents of its buffers): data by name, the others as the graph initialises them."""
    lb = bl.load(compiler.compile_spec(b.spec()))
    return lb, [np.ascontiguousarray(data[m['name']]).reshape(-1) if m['name'] in data else bl.materialize(m) for m in lb.metadata['buffers']]


def cache_of(read, c):
    """The cache as `read` (name -> flat array) has it, in the shapes of c."""
    return {n: (read(n).view(np.int8) if n[1] == 'q' else read(n)).reshape(c[n].shape) for n in CACHE}


def names(lb):
    return [m['name'] for m in lb.metadata['buffers']]


def random_cache(rng, pairs, nblk, blk, hd, bf16):
    from serving_fp64 import empty_cache, quantise
    c = empty_cache(pairs, nblk, blk, hd)
    for x in 'kv':
        q, s = quantise((rng.standard_normal((pairs, nblk, blk, hd)) * np.exp(0.5 * rng.standard_normal((pairs, nblk, 1, 1)))).astype(np.float32))
        c[x + 'q'], c[x + 's'] = np.ascontiguousarray(q if x == 'k' else q.transpose(0, 1, 3, 2)), s
        t = rng.standard_normal((pairs, blk, hd)).astype(np.float32)
        c[x + 't'] = bl.bf16_round(t) if bf16 else t
    return c


def append_graph(c, knew, vnew, lens, hkv, n_new, tail='bf16', new='bf16', tasks=256, gamma=None, theta=0.0, eps=0.0, cut=None):
    b, data = Builder(0), {}
    cache = add_cache(b, data, c, hkv, tail)
    add(b, data, 'knew', knew, new), add(b, data, 'vnew', vnew, new)
    add(b, data, 'lens', np.asarray(lens, np.int32)[:, None])
    if gamma is not None:
        add(b, data, 'kgamma', gamma[None])
    serving.kv_append_q8(b, cache, 'knew', 'vnew', 'lens', n_new, kgamma=None if gamma is None else 'kgamma', theta=theta, eps=eps, tasks=tasks)
    return compiled(b, data)


def attend_graph(c, q, lens, hkv, heads, n_new, scale, tail='bf16', qdt='bf16', odt=None, tasks=256, gamma=None, theta=0.0, eps=0.0, extra=0):
    b, data = Builder(0), {}
    cache = add_cache(b, data, c, hkv, tail)
    add(b, data, 'q', np.pad(q, ((0, 0), (0, extra))), qdt)
    add(b, data, 'o', np.full((q.shape[0], q.shape[1] + extra), 7.0, np.float32), odt or qdt)
    add(b, data, 'lens', np.asarray(lens, np.int32)[:, None])
    if gamma is not None:
        add(b, data, 'qgamma', gamma[None])
    serving.attn_decode_q8(b, cache, 'q', 'o', 'lens', heads, n_new, scale, qgamma=None if gamma is None else 'qgamma', theta=theta, eps=eps, tasks=tasks)
    return compiled(b, data)


def adjust_graph(x, par, dtype='f32', odt='f32', inplace=False, tasks=256, **given):
    b, data = Builder(0), {}
    add(b, data, 'logits', x, dtype), add(b, data, 'par', par)
    if not inplace:
        add(b, data, 'out', np.zeros(x.shape, np.float32), odt)
    for n, v in given.items():
        if v is not None:
            add(b, data, n, v if np.asarray(v).ndim == 2 else np.asarray(v)[:, None])
    serving.logits_adjust(b, 'logits', 'logits' if inplace else 'out', 'par', *x.shape, tasks=tasks, **{n: n for n, v in given.items() if v is not None})
    return compiled(b, data)


# ------------------------------------------------------------------------------------------------ cases of both test files

# (blk, hd, kv heads, tail and input type, n_new, lengths): empty and full blocks, one token and many, a slot without a sequence,
# a cache filled to its last token, head sizes of the vector form and others
APPENDS = [
    (64, 128, 2, 'bf16', 1, [0, 63, 64, 100, -1, 127, 1]),
    (16, 64, 1, 'f32', 1, [15, 14, 31]),
    (32, 128, 3, 'bf16', 5, [0, 27, 28, 31, -1]),
    (16, 128, 2, 'f32', 70, [0, 9, 16, 26]),
    (64, 64, 2, 'bf16', 200, [0, 55, 56]),
    (128, 128, 1, 'bf16', 300, [0, 84, 127]),
    (128, 64, 1, 'f32', 1, [127, 126]),
    (32, 32, 2, 'bf16', 33, [0, 31]),
    (16, 100, 2, 'f32', 18, [0, 13, 14]),
    (16, 4, 1, 'bf16', 16, [0, 16, 1]),
]


def append_case(case, seed=0):
    blk, hd, hkv, dt, n_new, lens = case
    rng = np.random.default_rng(seed)
    nblk = -(-(max(lens) + n_new) // blk)
    c = random_cache(rng, len(lens) * hkv, nblk, blk, hd, dt == 'bf16')
    new = [rng.standard_normal((len(lens) * n_new, hkv * hd)).astype(np.float32) for _ in range(2)]
    return c, *(bl.bf16_round(x) if dt == 'bf16' else x for x in new)


# (blk, hd, kv heads, heads, type, n_new, lengths): one token to many blocks, unfinished blocks of every kind, query rows of one
# tile and of two, slots without a sequence
ATTENDS = [
    (64, 128, 2, 8, 'f32', 1, [0, 1, 62, 63, 64, 127, 200, -1]),
    (64, 128, 1, 1, 'f32', 1, [700, 5]),
    (16, 128, 2, 4, 'f32', 3, [0, 14, 13, 100, 333]),
    (32, 64, 2, 16, 'f32', 4, [0, 28, 29, 31, 500, -1]),
    (128, 64, 1, 2, 'f32', 5, [122, 123, 124, 1000]),
    (128, 128, 2, 32, 'bf16', 2, [126, 127, 600]),
    (64, 128, 1, 8, 'bf16', 1, [2047, 2048, 3000]),
    (16, 64, 3, 3, 'bf16', 32, [0, 1, 200]),
    (32, 32, 2, 4, 'f32', 2, [0, 62, 300]),
    (16, 100, 1, 3, 'f32', 1, [15, 16, 77]),
    (16, 4, 1, 2, 'f32', 1, [40]),
    (64, 128, 2, 8, 'f32', 1, [5000, 3, -1, 1800, 9000]),            # pairs that are shared out over tasks, among short ones
    (16, 64, 1, 8, 'f32', 4, [3000, 100]),
    (128, 128, 1, 16, 'bf16', 2, [8190, 70]),
    (16, 64, 1, 1, 'f32', 1, [(37 * i) % 190 - 1 for i in range(300)]),   # sequences of several rounds of the search
]


def attend_case(case, seed=0):
    blk, hd, hkv, heads, dt, n_new, lens = case
    rng = np.random.default_rng(seed)
    c = random_cache(rng, len(lens) * hkv, -(-(max(lens) + n_new) // blk), blk, hd, dt == 'bf16')
    q = (2 * rng.standard_normal((len(lens) * n_new, heads * hd))).astype(np.float32)
    return c, bl.bf16_round(q) if dt == 'bf16' else q


# (rows, V, type, type of out, history columns, bias entries, mask rows, mrow, last)
ADJUSTS = [
    (1, 1, 'f32', 'f32', 3, 0, 0, False, True),
    (3, 33, 'f32', 'f32', 40, 9, 0, False, True),
    (2, 1000, 'f32', 'bf16', 0, 0, 2, False, False),
    (5, 4097, 'bf16', 'f32', 700, 30, 4, True, True),
    (2, 32000, 'f32', 'f32', 5000, 300, 1, True, False),
    (2, 53300, 'bf16', 'bf16', 100, 2047, 2, False, True),      # more than two chunks, the largest list of biases
    (300, 257, 'f32', 'f32', 17, 3, 3, True, True),
    (2, 50001, 'f32', 'f32', 6001, 143, 2, True, True),          # a long range: as many named tokens as the table takes, one more
    (2, 50001, 'f32', 'f32', 6002, 143, 2, True, True),
    (1, 45057, 'bf16', 'bf16', 9000, 5, 0, False, True),
]


def adjust_case(case, seed=0):
    R, V, dt, odt, H, nb, M, has_row, has_last = case
    rng = np.random.default_rng(seed)
    x = (4 * rng.standard_normal((R, V))).astype(np.float32)
    par = np.stack([1 + rng.random(R), rng.random(R) - 0.3, rng.random(R) - 0.2], 1).astype(np.float32)
    g = {}
    if H:
        g['hist'] = rng.integers(-2, V + 2, (R, H), dtype=np.int32)         # some that count nowhere
        g['hist'][:, ::3] = rng.integers(0, min(V, 5), g['hist'][:, ::3].shape)
        g['hlen'] = rng.integers(0, H + (0 if has_last else 1), R, dtype=np.int32)
        g['hlen'][0] = H - 1 if has_last else H
        g['plen'] = (g['hlen'] * rng.random(R)).astype(np.int32)
        if has_last:
            g['last'] = rng.integers(-1, V, R, dtype=np.int32)
    if nb:
        g['bidx'] = rng.integers(-3, V + 3, (R, nb), dtype=np.int32)
        g['bidx'][:, 1::4] = g['bidx'][:, ::4][:, :g['bidx'][:, 1::4].shape[1]]   # one token several times
        g['bval'] = rng.standard_normal((R, nb)).astype(np.float32)
    if M:
        g['mask'] = rng.integers(-2 ** 31, 2 ** 31, (M if has_row else R, -(-V // 32)), dtype=np.int64).astype(np.int32)
        g['mask'][0] = 0                                                    # nothing allowed
        if has_row:
            g['mrow'] = rng.integers(-1, M, R, dtype=np.int32)
            g['mrow'][0] = 0
    return bl.bf16_round(x) if dt == 'bf16' else x, par, g


def step(dtype):
    """What one rounding to storage `dtype` is off by, relative to the value."""
    return {'f32': 2.0 ** -24, 'bf16': 2.0 ** -8}[dtype]


def near(got, want, bound, dtype):
    """Every value within its bound and one rounding to its storage; what is not finite is the same."""
    got, want = np.asarray(got, np.float64).ravel(), np.asarray(want, np.float64).ravel()
    bound = np.broadcast_to(np.asarray(bound, np.float64).ravel(), want.shape)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine], want[~fine])
    off = np.abs(got[fine] - want[fine]) - bound[fine] - step(dtype) * (np.abs(want[fine]) + bound[fine])
    assert not (off > 0).any(), (off.max(), int((off > 0).sum()), fine.sum())
    assert np.isfinite(got[fine]).all()
