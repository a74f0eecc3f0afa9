"""Decode steps of the Qwen3 shape over the 8-bit cache with penalties, one operator at a time: what a step's operators were given,
as read back around the step, goes through their definitions in 64 bits (serving_fp64)."""
import numpy as np

import serving_fp64 as f64
import serving_graphs as sg
from kvm_amd.workloads import qwen3


def case(batch, ctx=61, head_dim=128, block=16, seed=0, **kw):
    """(config, workload, contents of its cache, prompt and norms): two layers, lengths around a block's end."""
    c = qwen3.Qwen3Config.tiny(batch=batch, ctx=ctx, head_dim=head_dim, cache='q8', kv_block=block, max_new=6, repetition=1.3, frequency=0.2,
                               presence=0.1, theta=1e4, **kw)
    w = qwen3.build(c)
    rng = np.random.default_rng(seed)
    given = {'hist': rng.integers(0, c.vocab, (batch, c.ctx + c.max_new)).astype(np.int32)}
    for l in range(c.layers):
        x = sg.random_cache(rng, batch * c.kv_heads, -(-(c.ctx + c.max_new) // block), block, head_dim, True)
        given.update({f'cache{l}.{n}': np.ascontiguousarray(v).view(np.int32) if n[1] == 'q' else v for n, v in x.items()})
        given.update({f'{n}.{l}': (rng.random(head_dim) + 0.5).astype(np.float32) for n in ('qn', 'kn')})
    return c, w, given


def cache(c, bufs, l):
    blk, pairs = c.kv_block, c.batch * c.kv_heads
    nblk = -(-(c.ctx + c.max_new) // blk)
    shape = {'kq': (pairs, nblk, blk, c.head_dim), 'vq': (pairs, nblk, c.head_dim, blk), 'ks': (pairs, nblk), 'vs': (pairs, nblk),
             'kt': (pairs, blk, c.head_dim), 'vt': (pairs, blk, c.head_dim)}
    return {n: (bufs[f'cache{l}.{n}'].view(np.int8) if n[1] == 'q' else bufs[f'cache{l}.{n}']).reshape(s) for n, s in shape.items()}


def check(c, before, after):
    """The last layer's append and attention (its q, k, v are still there), the logits, the history and the token. A key is off by
    steps of 2^-24 of its magnitudes in norm and rotation (below 2^-20 together, positions below 100), then by its rounding to
    bf16, whose neighbours are 2^-7 apart; a byte by that and a half step over the scale."""
    l, B, hd = c.layers - 1, c.batch, c.head_dim
    lens = before['lens'].tolist()
    kw = dict(eps=np.float32(c.eps), theta=c.theta)
    have = cache(c, after, l)
    want = f64.append(cache(c, before, l), after['k'].reshape(B, -1), after['v'].reshape(B, -1), lens, c.kv_heads, 1, True, before[f'kn.{l}'], **kw)
    for n in ('vq', 'vs', 'vt'):
        np.testing.assert_array_equal(have[n], want[n], err_msg=n)
    rel = 2.0 ** -7 + 2.0 ** -20
    assert np.abs(have['kt'] - want['kt']).max() <= rel * np.abs(want['kt']).max()
    assert (np.abs(have['ks'] - want['ks']) <= (rel + 2.0 ** -24) * want['ks']).all()
    assert np.abs(have['kq'].astype(int) - want['kq']).max() <= 1 + int(127 * 2 * rel)
    o, bound = f64.attend(have, after['q'].reshape(B, -1), lens, c.kv_heads, c.heads, 1, np.float32(1 / np.sqrt(hd)), before[f'qn.{l}'], **kw)
    sg.near(after['att'], o, bound, 'bf16' if B > 1 else 'f32')
    adj, hist, bound = f64.adjust(after['logits'].reshape(B, -1), before['par'].reshape(B, 3), before['hist'].reshape(B, -1), before['plen'], before['hlen'],
                                  before['tok'])
    sg.near(after['adj'], adj, bound, 'f32')
    np.testing.assert_array_equal(after['hist'].reshape(hist.shape), hist)
    np.testing.assert_array_equal(after['tok'], after['adj'].reshape(B, -1).argmax(1))
    np.testing.assert_array_equal(after['lens'], before['lens'] + 1)
    np.testing.assert_array_equal(after['hlen'], before['hlen'] + 1)
    assert not after['acnt'].any()
