"""Task builders for the serving operators: of a decode step the 8-bit KV cache (kv_append_q8, attn_decode_q8) and adjusted logits
(logits_adjust); of a step that brings prompts and tokens together the products in 8-bit integers (rows_q8, linear_q8) and the paged
KV cache (qkv_append_paged, attn_paged). Each lays out one call of an operator as tasks of a `Builder` graph and returns their ids; buffers are
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


# ------------------------------------------------------------------------------------------------ products in 8-bit integers

@dataclass
class RowsQ8:
    """Rows of K signed bytes in i32 words, and a scale for each."""
    q: str
    s: str
    rows: int
    K: int


def rows_q8_buffers(b: Builder, name: str, rows: int, K: int) -> RowsQ8:
    """Declares rows of K bytes: buffers `name` (whole 16-byte vectors) and name + 's'. Weights, [N, K], are declared the same way."""
    b.fill(name, rows, 4 * -(-K // 16), 'i32')
    b.fill(name + 's', rows)
    return RowsQ8(name, name + 's', rows, K)


weight_q8_buffers = rows_q8_buffers


EDGES = 4096


def after_all(b: Builder, preds: list[str], n: int) -> list[str]:
    """What `n` tasks that need all of `preds` wait for: these, where that is few edges, else one task between (a hop of its own)."""
    return preds if len(preds) * n <= EDGES else b.join(preds, n)


def quantise_rows(x) -> tuple:
    """(words, scales) of an array [rows, K], what the operator rows_q8 makes of it: the contents of weight_q8_buffers."""
    import numpy as np
    x = np.asarray(x, np.float32)
    with np.errstate(invalid='ignore', over='ignore'):
        scale = (np.abs(x).max(1, keepdims=True) * np.float32(1 / 127)).astype(np.float32)
        scale[scale < np.finfo(np.float32).tiny] = 0
        fine = np.isfinite(x).all(1, keepdims=True)
        q = np.where(fine & (scale > 0), np.rint(x.astype(np.float64) / np.where(scale > 0, scale, 1).astype(np.float64)), 0)
    words = np.zeros((x.shape[0], 16 * -(-x.shape[1] // 16)), np.int8)
    words[:, :x.shape[1]] = q
    return words.view(np.int32), np.where(fine, scale, np.float32(np.nan))[:, 0]


def _pro(gamma, x2) -> int:
    if gamma and x2:
        raise ValueError('gamma (RMSNorm) and x2 (SwiGLU) exclude each other')
    return 1 if gamma else 2 if x2 else 0


def rows_q8(b: Builder, x: str, out: RowsQ8, M: int, after=(), x2: str | None = None, gamma: str | None = None, eps: float = 0.0, tasks: int = 256) -> list[str]:
    """The first M rows of x in 8 bits, in up to `tasks` tasks: as they are, RMS-normalised (gamma), or silu(x) * x2."""
    return [b.task('rows_q8', after=after, x=x, x2=x2, gamma=gamma, q=out.q, qs=out.s, r0=r0, r1=r1, K=out.K, pro=_pro(gamma, x2), eps=eps)
            for r0, r1 in split(M, tasks)]


def _workspace(b: Builder, out: str, K: int) -> RowsQ8:
    """The buffers of an earlier call's workspace, as what they hold: as many rows as both have, of K bytes or of fewer if they are narrower."""
    (rows, words), (r, c) = _shape(b, out + '.x'), _shape(b, out + '.xs')
    return RowsQ8(out + '.x', out + '.xs', min(rows, r * c), min(K, 4 * words))


def matmul_q8_tile(M: int, N: int, tasks: int = 256) -> tuple[int, int, int]:
    """(tile, rows, columns): the largest tile of which there are about as many as workers. Fewer and larger ones lose (333 x 2,777, K 1,001:
    46 us with 66 tiles of 128 x 128, 40 with 264 of 64 x 64, though those take two rounds)."""
    for tile, tm, tn in ((0, 128, 256), (1, 128, 128)):
        if -(-M // tm) * -(-N // tn) >= 0.7 * tasks:
            return tile, tm, tn
    return 2, 64, 64


def linear_q8(b: Builder, x: str, w: RowsQ8, out: str, M: int, after=(), x2: str | None = None, gamma: str | None = None, bias: str | None = None,
              res: str | None = None, eps: float = 0.0, tasks: int = 256, rows: RowsQ8 | None = None) -> list[str]:
    """out = x' w^T (+ bias) (+ res), the first M rows of x (x' as in rows_q8) and w [N, K] in 8 bits. One row is quantised inside the tasks
    of the product (gemv_q8), more in a phase of their own, into the workspace `rows` (declared here as out + '.x' when absent, or that of an
    earlier call with this `out` if it is large enough; layers that follow each other may share one of the same K). `x` may be rows that are in 8 bits
    already (RowsQ8)."""
    N, K = w.rows, w.K
    if isinstance(x, RowsQ8):
        if gamma or x2 or x.K != K:
            raise ValueError(f'rows in 8 bits go in as they are, with the K of the weights: K {x.K} and {K}')
        if x.rows < M:
            raise ValueError(f'{M} rows of {x.q} wanted, which holds {x.rows} rows')
        rows = x
    elif M > 1:
        if rows is None:
            rows = _workspace(b, out, K) if b.has(out + '.x') and b.has(out + '.xs') else rows_q8_buffers(b, out + '.x', M, K)
        if rows.K != K or rows.rows < M:
            raise ValueError(f'the workspace holds {rows.rows} rows of {rows.K} bytes: {M} rows of {K} needed')
        after = after_all(b, rows_q8(b, x, rows, M, after, x2, gamma, eps, tasks), tasks)
    kw = dict(w=w.q, sw=w.s, out=out, bias=bias, res=res, K=K)
    if M <= 16:
        if rows is None:
            kw.update(x=x, x2=x2, gamma=gamma, sx=None, pro=_pro(gamma, x2), eps=eps)
        else:
            kw.update(x=rows.q, x2=None, gamma=None, sx=rows.s, pro=3, eps=0.0)
        return [b.task('gemv_q8', after=after, n0=16 * lo, n1=min(N, 16 * hi), M=M, **kw) for lo, hi in split(-(-N // 16), tasks)]
    tile, tm, tn = matmul_q8_tile(M, N, tasks)
    return [b.task('matmul_q8', after=after, a=rows.q, sa=rows.s, m0=m0, n0=n0, M=M, N=N, tile=tile, **kw)
            for m0 in range(0, M, tm) for n0 in range(0, N, tn)]


# ------------------------------------------------------------------------------------------------ paged KV cache

@dataclass
class CachePaged:
    """The buffers of one layer's cache in pages of `page` tokens."""
    kc: str
    vc: str
    pages: int
    kv_heads: int
    hd: int
    page: int

    def args(self) -> dict:
        return dict(kc=self.kc, vc=self.vc, Hkv=self.kv_heads, hd=self.hd, page=self.page)


def paged_buffers(b: Builder, name: str, pages: int, kv_heads: int, hd: int, page: int = 64, dtype: str = 'bf16') -> CachePaged:
    """Declares a cache of `pages` pages: buffers name + 'kc' and name + 'vc'. Which page holds what is the caller's table."""
    if page not in (16, 32, 64, 128) or hd % 2 or not 0 < hd <= 256:
        raise ValueError(f'page must be 16, 32, 64 or 128 and hd even, up to 256: page {page}, hd {hd}')
    for x in 'kv':
        b.fill(f'{name}{x}c', pages * kv_heads * page, hd, dtype)
    return CachePaged(name + 'kc', name + 'vc', pages, kv_heads, hd, page)


def _shape(b: Builder, name: str) -> tuple[int, int]:
    return next((d['rows'], d['cols']) for d in b.buffers if d['name'] == name)


def _sequences(b: Builder, cu: str) -> int:
    rows, cols = _shape(b, cu)
    if not 2 <= rows * cols <= 1025:
        raise ValueError(f'cu holds batch + 1 row numbers, batch 1 .. 1024: {rows} x {cols}')
    return rows * cols - 1


def qkv_append_paged(b: Builder, c: CachePaged, k: str, v: str, table: str, lens: str, cu: str, q: str | None = None, qo: str | None = None, heads: int = 0,
                     qgamma: str | None = None, kgamma: str | None = None, theta: float = 0.0, eps: float = 0.0, after=(), tasks: int = 256) -> list[str]:
    """Puts the new tokens' keys and values into their pages, keys and queries normalised and rotated on the way, in up to `tasks` tasks.
    The batch is what cu holds rows for; any of k's rows may have a token."""
    kw = dict(q=q, k=k, v=v, qo=qo if qo or not q else q, table=table, lens=lens, cu=cu, qgamma=qgamma, kgamma=kgamma, B=_sequences(b, cu), H=heads,
              theta=theta, eps=eps, **c.args())
    return [b.task('qkv_append_paged', after=after, r0=r0, r1=r1, **kw) for r0, r1 in split(_shape(b, k)[0], tasks)]


def attn_paged(b: Builder, c: CachePaged, q: str, o: str, table: str, lens: str, cu: str, heads: int, n_max: int = 0, scale: float | None = None, after=(),
               part: str | None = None, cnt: str | None = None, tasks: int = 256) -> list[str]:
    """Attention of the new tokens over the pages, in `tasks` tasks that share the work evenly by the lengths that they read. n_max: the most
    new tokens of a sequence, where that is known (1 for a decode step: a smaller workspace); 0: any. `part`, `cnt`: the workspace, declared
    here (o + '.part', o + '.cnt') when absent; calls that follow each other (the layers of a model) may share one, calls that may run
    side by side not."""
    group = heads // c.kv_heads
    if heads % c.kv_heads or not 1 <= group <= 128:
        raise ValueError(f'heads must be 1 to 128 times kv_heads: {heads}, {c.kv_heads}')
    rows = group * (n_max or _shape(b, q)[0])
    tile = max(group, min(128, rows))
    part = part or b.fill(o + '.part', 2 * tasks * tile, c.hd + 2)
    cnt = cnt or b.fill(o + '.cnt', tasks, 1, 'i32')
    kw = dict(q=q, o=o, table=table, lens=lens, cu=cu, part=part, cnt=cnt, S=tasks, B=_sequences(b, cu), H=heads, tile=tile,
              scale=1 / math.sqrt(c.hd) if scale is None else scale, **c.args())
    return [b.task('attn_paged', after=after, s=s, **kw) for s in range(tasks)]
