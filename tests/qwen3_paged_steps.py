"""Steps of the Qwen3 shape over paged caches with 8-bit weights: what a step's operators were given, as read back around the step, goes
through their definitions in 64 bits (mixed_fp64)."""
import numpy as np

import mixed_fp64 as f64
import serving_graphs as sg
from kvm_amd import bundle as bl
from kvm_amd import compiler
from kvm_amd.workloads import qwen3, serving

TABLES = ('tok', 'cu', 'last', 'lens', 'table')


def case(batch, rows=0, layers=1, page=16, ctx=20, seed=0, **kw):
    """(config, bundle, contents): weights of the model in 8 bits, a cache of `ctx` tokens a sequence whose other tokens are NaN."""
    c = qwen3.Qwen3Config.tiny(batch=batch, rows=rows, layers=layers, cache='paged', page=page, ctx=ctx, max_new=40, theta=1e4, **kw)
    w = qwen3.build(c)
    lb = bl.load(compiler.compile_spec(w.spec))
    rng = np.random.default_rng([seed, batch, rows])
    init = {m['name']: bl.materialize({**m, 'init': w.init_override.get(m['name'], m['init'])}) for m in lb.metadata['buffers']}
    for n, k in shapes(c).items():
        x = rng.standard_normal(k).astype(np.float32) * np.float32(k[1] ** -0.5)
        init[n], init[n + 's'] = (y.reshape(-1) for y in serving.quantise_rows(x))
    width = init['table'].size // batch
    pages = len(init['cache0.kc']) // (c.kv_heads * page * c.head_dim)
    init['table'] = rng.permutation(pages)[:batch * width].astype(np.int32)
    for l in range(c.layers):
        for n in ('qn', 'kn'):
            init[f'{n}.{l}'] = (rng.random(c.head_dim) + 0.5).astype(np.float32)
        for n in ('ln1', 'ln2'):
            init[f'{n}.{l}'] = (rng.random(c.hidden) + 0.5).astype(np.float32)
        for n in ('kc', 'vc'):
            x = np.full((pages, c.kv_heads, page, c.head_dim), np.nan, np.float32)
            for s in range(batch):
                t = np.arange(ctx)
                x[init['table'].reshape(batch, -1)[s, t // page], :, t % page] = bl.bf16_round(rng.standard_normal((ctx, c.kv_heads, c.head_dim)).astype(np.float32))
            init[f'cache{l}.{n}'] = x.reshape(-1)
    return c, lb, init


def shapes(c):
    D, hq, hkv, F = c.hidden, c.heads * c.head_dim, c.kv_heads * c.head_dim, c.ffn
    per = {'q': (hq, D), 'k': (hkv, D), 'v': (hkv, D), 'o': (D, hq), 'g': (F, D), 'u': (F, D), 'd': (D, F)}
    return {**{f'w{n}.{l}': k for l in range(c.layers) for n, k in per.items()}, 'whead': (c.vocab, D)}


def loaded(lb, init):
    return [np.ascontiguousarray(init[n]).reshape(-1) for n in sg.names(lb)]


def plan(c, lens, new, rng):
    """What the caller writes in front of a step that brings new[s] tokens of each sequence."""
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    R = c.rows or c.batch
    return {'tok': rng.integers(0, c.vocab, R).astype(np.int32), 'cu': cu, 'last': np.maximum(cu[1:] - 1, 0).astype(np.int32), 'lens': np.asarray(lens, np.int32)}


def linear(x, w, sw, pro=0, x2=None, gamma=None, eps=0.0, res=None, off=0.0):
    """(result, bound) of the product with rows brought to 8 bits. A row's values are known to 2^-20 of themselves (f32 norm, silu; the scale) and
    to `off`; where that reaches a tie, the byte may be the other one."""
    v = f64.shaped(x, pro, x2, gamma, eps)
    q, s = f64.quantise(v)
    y, bound = f64.product(q, s, w, sw, None, res)
    step = np.where(s > 0, s, 1)[:, None].astype(np.float64)
    u = np.abs(v.astype(np.float64)) / step
    slack = 127 * 2.0 ** -20 + off / step
    flips = np.where(slack < 0.5, np.abs(u - np.floor(u) - 0.5) <= slack, np.ceil(slack)) * (s > 0)[:, None]
    grow = 2.0 ** -20 + (off / step / 127).max() if np.ndim(off) else 2.0 ** -20
    back = y - (res if res is not None else 0)
    return y, bound + np.abs(back) * grow + s[:, None] * (flips @ np.abs(w.astype(np.float64)).T) * np.abs(sw.astype(np.float64))


def check(c, before, after):
    """The last layer's append and attention, the head and the choice; of a model of one layer every product as well."""
    l, B, R, hd = c.layers - 1, c.batch, c.rows or c.batch, c.head_dim
    eps = np.float32(c.eps)
    cu, lens, table = before['cu'], before['lens'], before['table'].reshape(B, -1)
    rows = lambda n: after[n].reshape(R, -1)                            # noqa: E731
    weight = lambda n: (after[n].view(np.int8).reshape(len(after[n + 's']), -1)[:, :shapes(c)[n][1]], after[n + 's'])     # noqa: E731
    at = lambda bufs, n: bufs[f'cache{l}.{n}'].reshape(-1, c.kv_heads, c.page, hd)    # noqa: E731
    heads = lambda n: rows(n).reshape(R, -1, hd)                        # noqa: E731
    # the cache: the new tokens from k and v, every other one as it was
    kc, vc, _ = f64.append(at(before, 'kc'), at(before, 'vc'), table, lens, cu, None, heads('k'), heads('v'), c.page, None, before[f'kn.{l}'], eps, c.theta)
    np.testing.assert_array_equal(at(after, 'vc'), vc)
    f64.near(at(after, 'kc'), kc, 2.0 ** -20 * np.abs(kc).max(-1, keepdims=True), 'bf16')
    want, mag = f64.attend(heads('q'), at(after, 'kc'), at(after, 'vc'), table, lens, cu, c.page, 1 / np.sqrt(hd))
    on = np.arange(R) < cu[B]
    have = heads('att')
    big = np.abs(heads('q')[on]).max(initial=0) * np.nanmax(np.abs(at(after, 'kc')))       # a score's terms, each off by two steps, hd + 4 of them
    slack = 2 * (hd + 4) * 2 * f64.U * hd * big / np.sqrt(hd) + (int(lens.max()) + R + 64) * 2 * f64.U + 2.0 ** -8
    f64.near(have[on], want[on], slack * mag[on], 'bf16')
    np.testing.assert_array_equal(have[~on], before['att'].reshape(R, -1, hd)[~on])
    if c.layers == 1:
        x0 = before['wte'].reshape(c.vocab, -1)[before['tok']]
        for n in 'kv':
            y, bound = linear(x0, *weight(f'w{n}.0'), 1, gamma=before['ln1.0'], eps=eps)
            f64.near(rows(n), y, bound, 'bf16')
        q, bound = linear(x0, *weight('wq.0'), 1, gamma=before['ln1.0'], eps=eps)           # q is turned in place, from bf16
        r, b, i = f64.owners(cu, R)
        turned = f64.turned(q[r].reshape(len(r), c.heads, hd), before['qn.0'], eps, c.theta, lens[b] + i)
        loose = (2.0 ** -8 * np.abs(q[r]) + bound[r]).reshape(len(r), c.heads, hd).max(-1) / np.sqrt((q[r].reshape(len(r), c.heads, hd) ** 2).mean(-1))
        # each value is off by at most `loose` of the root mean square, so is the mean; a rotation adds two values' errors
        f64.near(heads('q')[r], turned, (3 * loose * before['qn.0'].max())[..., None] * (1 + np.abs(turned).max(-1, keepdims=True)), 'bf16')
        x1, off = linear(rows('att'), *weight('wo.0'), res=x0)
        for n in 'gu':
            y, bound = linear(x1.astype(np.float32), *weight(f'w{n}.0'), 1, gamma=before['ln2.0'], eps=eps, off=normed(x1, off, before['ln2.0']))
            f64.near(rows(n), y, bound, 'bf16')
        y, bound = linear(rows('g'), *weight('wd.0'), 2, x2=rows('u'), res=x1)
        f64.near(rows('x'), y, bound + off, 'f32')
    np.testing.assert_array_equal(after['xl'].reshape(B, -1), rows('x')[before['last']])
    y, bound = linear(after['xl'].reshape(B, -1), *weight('whead'), 1, gamma=before['lnf'], eps=eps)
    logits = after['logits'].reshape(B, -1)
    f64.near(logits, y, bound, 'f32')
    np.testing.assert_array_equal(after['next' if c.rows else 'tok'], logits.argmax(1))
    np.testing.assert_array_equal(after['lens'], lens + (0 if c.rows else 1))
    for n in ('cu', 'last', 'table') + (('tok',) if c.rows else ()):
        np.testing.assert_array_equal(after[n], before[n])
    assert not after['att.cnt'].any()


def normed(x, off, gamma):
    """How far the norm of x may be off where x is off by `off` (and by its own rounding to f32): itself, and by its part of the mean square."""
    off = off + f64.U * np.abs(x)
    rms = np.sqrt((x * x).mean(1, keepdims=True))
    return (off + np.abs(x) * np.sqrt((off * off).mean(1, keepdims=True)) / rms) / rms * gamma * 1.01
