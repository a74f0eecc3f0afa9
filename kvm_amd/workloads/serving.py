"""Task builders for the serving operators of a decode step: the 8-bit KV cache (kv_append_q8, attn_decode_q8) and adjusted
logits (logits_adjust). Each lays out one call of an operator as tasks of a `Builder` graph and returns their ids; buffers are
the graph's, by name. What the operators compute and refuse is in include/mvm_ops_kvm.def.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

from . import Builder, split


@dataclass
class CacheQ8:
    """The buffers of one layer's cache for `batch` sequences of up to `tmax` tokens (whole blocks of `blk`)."""
    kq: str
    ks: str
    vq: str
    vs: str
    kt: str
    vt: str
    batch: int
    kv_heads: int
    hd: int
    tmax: int
    blk: int

    def args(self) -> dict:
        return dict(kq=self.kq, ks=self.ks, vq=self.vq, vs=self.vs, kt=self.kt, vt=self.vt, Hkv=self.kv_heads, hd=self.hd, blk=self.blk)


def kv_q8_buffers(b: Builder, name: str, batch: int, kv_heads: int, hd: int, tmax: int, blk: int = 64, dtype: str = 'bf16') -> CacheQ8:
    """Declares an empty cache: buffers name + kq, ks, vq, vs, kt, vt, the tail in `dtype`. tmax is rounded up to whole blocks."""
    if blk not in (16, 32, 64, 128) or hd % 4 or not 0 < hd <= 128:
        raise ValueError(f'blk must be 16, 32, 64 or 128 and hd a multiple of 4 up to 128: blk {blk}, hd {hd}')
    pairs, tmax = batch * kv_heads, -(-tmax // blk) * blk
    for x in 'kv':
        b.fill(f'{name}{x}q', pairs * tmax, hd // 4, 'i32')
        b.fill(f'{name}{x}s', pairs, tmax // blk)
        b.fill(f'{name}{x}t', pairs * blk, hd, dtype)
    return CacheQ8(*(name + n for n in ('kq', 'ks', 'vq', 'vs', 'kt', 'vt')), batch, kv_heads, hd, tmax, blk)


def kv_append_q8(b: Builder, c: CacheQ8, knew: str, vnew: str, lens: str, n_new: int = 1, after=(), kgamma: str | None = None, theta: float = 0.0,
                 eps: float = 0.0, tasks: int = 256) -> list[str]:
    """Appends n_new tokens to every sequence in about `tasks` tasks: (sequence, head) pairs, and with fewer pairs than tasks
    also shares of a long n_new. Tokens that may be taken back (drafted ones) must not finish a block: a length can be set back
    within the unfinished block or to where a block starts, not into a block that has become full."""
    pairs = c.batch * c.kv_heads
    P = max(1, min(tasks // pairs, n_new // c.blk))
    kw = dict(knew=knew, vnew=vnew, lens=lens, kgamma=kgamma, theta=theta, eps=eps, n_new=n_new, P=P, **c.args())
    seqs = split(c.batch, tasks // P)
    heads = split(c.kv_heads, tasks // (len(seqs) * P))
    return [b.task('kv_append_q8', after=after, b0=b0, b1=b1, h0=h0, h1=h1, p=p, **kw) for b0, b1 in seqs for h0, h1 in heads for p in range(P)]


def attn_decode_q8(b: Builder, c: CacheQ8, q: str, o: str, lens: str, heads: int, n_new: int = 1, scale: float | None = None, after=(),
                   qgamma: str | None = None, theta: float = 0.0, eps: float = 0.0, part: str | None = None, cnt: str | None = None,
                   tasks: int = 256) -> list[str]:
    """Attention of the n_new newest tokens of every sequence over the cache, in `tasks` tasks that share the work evenly (a call of the
    operator for every 1,024 sequences, with parts of their own: `part` + '.1' and so on). `part`, `cnt`: the workspace, declared here
    (o + '.part', o + '.cnt') when absent; calls that follow each other (the layers of a model) may share one, calls that may run
    side by side not."""
    rows = n_new * (heads // c.kv_heads)
    if rows > 32:
        raise ValueError(f'n_new * heads / kv_heads must be at most 32: {n_new} * {heads} / {c.kv_heads}')
    calls = [(b0, min(c.batch, b0 + 1024)) for b0 in range(0, c.batch, 1024)]
    part = part or b.fill(o + '.part', 2 * tasks * rows, c.hd + 2)
    parts = [part] + [f'{part}.{i}' for i in range(1, len(calls))]
    for x in parts[1:]:
        if not b.has(x):
            b.fill(x, 2 * tasks * rows, c.hd + 2)
    cnt = cnt or b.fill(o + '.cnt', c.batch * c.kv_heads, 1, 'i32')
    kw = dict(q=q, lens=lens, o=o, cnt=cnt, qgamma=qgamma, S=tasks, n_new=n_new, H=heads, scale=1 / math.sqrt(c.hd) if scale is None else scale,
              theta=theta, eps=eps, **c.args())
    return [b.task('attn_decode_q8', after=after, b0=b0, b1=b1, s=s, part=p, **kw) for (b0, b1), p in zip(calls, parts) for s in range(tasks)]


def logits_adjust(b: Builder, logits: str, out: str, par: str, rows: int, V: int, after=(), hist: str | None = None, plen: str | None = None,
                  hlen: str | None = None, last: str | None = None, bidx: str | None = None, bval: str | None = None, mask: str | None = None,
                  mrow: str | None = None, tasks: int = 256) -> list[str]:
    """Adjusts `rows` rows of logits in about `tasks` tasks, ranges of at least 1,024 logits."""
    kw = dict(logits=logits, out=out, par=par, hist=hist, plen=plen, hlen=hlen, last=last, bidx=bidx, bval=bval, mask=mask, mrow=mrow, V=V)
    per_row = max(1, min(tasks // rows, V // 1024))
    words = -(-V // 32)
    return [b.task('logits_adjust', after=after, r0=r0, r1=r1, v0=32 * w0, v1=min(V, 32 * w1), **kw)
            for r0, r1 in split(rows, max(1, tasks // per_row)) for w0, w1 in split(words, per_row)]
