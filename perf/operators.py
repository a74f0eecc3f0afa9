"""Measured cases of the serving operators of a decode step: the append to a key / value cache held in 8 bits, the decode
attention over that cache, and the adjustment of logits before a token is chosen.

`own` chooses what a pass runs: the plain forms below (elementary torch operations in 32 bits, in 64 where a rounding
decides), or the framework's operators, as tasks of a graph that a program submits once and launches for every step. The
buffers live on the GPU for as long as the program does; outputs are those buffers.

Layouts (registry operators kv_append_q8, attn_decode_q8, logits_adjust):
  kq     [batch * kv heads * tmax, hd] bytes: the keys of finished blocks of `blk` tokens, whole numbers of -127 .. 127
  vq     the same size: a block's values stand transposed, [hd][blk]
  ks, vs [batch * kv heads, tmax / blk] f32: the blocks' scales, a value is byte * scale
  kt, vt [batch * kv heads * blk, hd]: the tokens of the unfinished block, in the model's type
  lens   [batch]: tokens of a sequence before the step, -1 for a slot that serves none
"""
from __future__ import annotations

import math

import torch

own = False

DEV = 'cuda'


def listed():
    return [
        # one user's next token: a launch and two rows
        dict(name='append_one', op='append', dtype='bf16', batch=1, n_new=1, kv=8, hd=128, blk=64, ctx=700, ragged=False),
        # a served batch, every sequence at a length of its own; one in `blk` of them finishes a block
        dict(name='append_batch', op='append', dtype='bf16', batch=96, n_new=1, kv=8, hd=128, blk=64, ctx=1000, ragged=True),
        # a prompt of any length
        dict(name='append_prompt', op='append', dtype='bf16', batch=1, n_new=4001, kv=8, hd=128, blk=64, ctx=0, ragged=False),
        # prompts of a small f32 model, behind what a shared beginning has filled
        dict(name='append_prompts_f32', op='append', dtype='f32', batch=8, n_new=777, kv=4, hd=64, blk=32, ctx=256, ragged=False),
        # the first tokens of a conversation: latency
        dict(name='attend_short', op='attend', dtype='bf16', batch=1, n_new=1, heads=32, kv=8, hd=128, blk=64, ctx=100, ragged=False, rope=True),
        # one user with a long document
        dict(name='attend_long', op='attend', dtype='bf16', batch=1, n_new=1, heads=32, kv=8, hd=128, blk=64, ctx=32000, ragged=False, rope=True),
        # drafted tokens of a few sequences checked at once, an f32 model of small heads
        dict(name='attend_draft', op='attend', dtype='f32', batch=6, n_new=4, heads=16, kv=4, hd=64, blk=32, ctx=1531, ragged=True, rope=True),
        # a served batch at the benchmark's context
        dict(name='attend_batch', op='attend', dtype='bf16', batch=24, n_new=1, heads=32, kv=8, hd=128, blk=64, ctx=4096, ragged=True, rope=True),
        # a full card
        dict(name='attend_large', op='attend', dtype='bf16', batch=128, n_new=1, heads=32, kv=8, hd=128, blk=64, ctx=8000, ragged=False, rope=False),
        # one user's repetition penalty
        dict(name='adjust_one', op='adjust', dtype='f32', rows=1, vocab=32000, hist=500, bias=0, mask=False, last=True),
        # a served batch with everything on
        dict(name='adjust_batch', op='adjust', dtype='f32', rows=24, vocab=151936, hist=4096, bias=300, mask=True, last=True),
        # many rows of bf16 logits with a vocabulary that is no multiple of a vector, under a grammar
        dict(name='adjust_rows_bf16', op='adjust', dtype='bf16', rows=256, vocab=50257, hist=777, bias=7, mask=True, last=False),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['append', 'attend', 'attend', 'adjust'])
    if op == 'adjust':
        rows = _log(rng, 1, 256)
        hist = rng.choice([0, _log(rng, 1, 8192), _log(rng, 1, 8192)])
        return dict(op=op, dtype=rng.choice(['f32', 'bf16']), rows=rows, vocab=_log(rng, 900, min(151936, 12_000_000 // rows)), hist=hist,
                    bias=rng.choice([0, _log(rng, 1, 500)]), mask=hist == 0 or rng.random() < 0.6, last=rng.random() < 0.7)
    dtype, blk, hd = rng.choice(['bf16', 'bf16', 'f32']), rng.choice([16, 32, 64, 64, 128]), rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == 'append':
        if rng.random() < 0.5:
            return dict(op=op, dtype=dtype, batch=_log(rng, 1, 192), n_new=1, kv=kv, hd=hd, blk=blk, ctx=_log(rng, 1, 2000), ragged=True)
        batch = _log(rng, 1, 8)          # a prompt begins where a block does: at the start, or behind whole blocks of a shared beginning
        return dict(op=op, dtype=dtype, batch=batch, n_new=_log(rng, 2, 6000 // batch), kv=kv, hd=hd, blk=blk, ctx=blk * rng.randint(0, 8), ragged=False)
    group = rng.choice([1, 2, 4, 8, 16] if kv < 8 else [1, 2, 4, 8])
    n_new = rng.choice([n for n in (1, 1, 1, 2, 3, 4, 5) if n * group <= 32])
    batch = _log(rng, 1, 128)
    return dict(op=op, dtype=dtype, batch=batch, n_new=n_new, heads=kv * group, kv=kv, hd=hd, blk=blk,
                ctx=_log(rng, 1, min(40000, 8_000_000 // (batch * kv))), ragged=rng.random() < 0.7, rope=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------ inputs

THETA, EPS = 1e6, 1e-6


def _tmax(case):
    """Room for the context, the step and some more, in whole blocks."""
    return -(-(case['ctx'] + case['n_new'] + 64) // case['blk']) * case['blk']


def _blocks(g, shape, blk):
    """Blocks of 8-bit numbers with a scale each, as a cache that has been written holds them: [..., tmax, hd] and
    [..., tmax / blk], the largest magnitude of each block 127."""
    *lead, t, hd = shape
    x = torch.randn(*lead, t // blk, blk * hd, generator=g, device=DEV)
    big = x.abs().amax(-1, keepdim=True)
    scale = torch.exp(0.4 * torch.randn(*lead, t // blk, generator=g, device=DEV)) / 32
    return torch.round(x * (127 / big)).to(torch.int8).view(*shape), scale


def _inputs(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    dt = torch.bfloat16 if c['dtype'] == 'bf16' else torch.float32
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)   # noqa: E731
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV, dtype=torch.int32)   # noqa: E731
    if c['op'] == 'adjust':
        R, V, n = c['rows'], c['vocab'], max(1, c['hist'])
        s = {'logits': (3 * randn(R, V)).to(dt)}
        s['par'] = torch.stack([1 + 0.4 * torch.rand(R, generator=g, device=DEV), 0.3 * randn(R).abs(), 0.5 * randn(R).abs()], 1)
        if c['hist']:
            # tokens as text has them, a few of them often; room for the one that the last step chose
            s['hist'] = (V * torch.rand(R, n + 1, generator=g, device=DEV) ** 3).to(torch.int32).clamp_(max=V - 1)
            s['hlen'] = ints(n // 2, n + 1, R, 1)
            s['plen'] = (s['hlen'] * torch.rand(R, 1, generator=g, device=DEV)).to(torch.int32)
            if c['last']:
                s['last'] = ints(0, V, R, 1)
        if c['bias']:
            s['bidx'], s['bval'] = ints(-V // 16, V, R, c['bias']), 2 * randn(R, c['bias'])      # below zero: no entry
        if c['mask']:
            M = 3                                                     # states of the grammar
            s['mask'] = ints(-2 ** 31, 2 ** 31 - 1, M, -(-V // 32))
            s['mrow'] = ints(-1, M, R, 1)
        return s
    B, Hkv, hd, blk, n, T = c['batch'], c['kv'], c['hd'], c['blk'], c['n_new'], _tmax(c)
    lens = torch.full((B, 1), c['ctx'], dtype=torch.int32, device=DEV)
    if c['ragged']:
        lens = ints(c['ctx'] // 4, c['ctx'] + 1, B, 1)
        if B > 4:
            lens[B // 3] = -1                                         # a slot that serves no sequence
    s = {'lens': lens}
    s['kq'], s['ks'] = _blocks(g, (B, Hkv, T, hd), blk)
    s['vq'], s['vs'] = _blocks(g, (B, Hkv, T, hd), blk)
    s['kt'], s['vt'] = randn(B, Hkv, blk, hd).to(dt), randn(B, Hkv, blk, hd).to(dt)
    if c['op'] == 'append':
        for name in ('knew', 'vnew'):                                 # a few channels far larger than the others, as keys have them
            s[name] = (randn(B, n, Hkv, hd) * torch.exp(0.7 * randn(Hkv, hd))).to(dt).view(B * n, Hkv * hd)
        return s
    s['q'] = (2 * randn(B * n, c['heads'] * hd)).to(dt)
    if c['rope']:
        s['qgamma'] = 2 + 0.2 * randn(1, hd)
    return s


def _scale(case):
    return 1 / math.sqrt(case['hd'])


def _graph(case, s):
    """The step's graph, as a serving program lays it out with the task builders of kvm_amd.workloads.serving."""
    from kvm_amd.workloads import Builder, serving
    c, b, kind = case, Builder(0), {torch.float32: 'f32', torch.int32: 'i32', torch.bfloat16: 'bf16'}
    add = lambda name: b.fill(name, *s[name].shape, dtype=kind[s[name].dtype])   # noqa: E731
    if c['op'] == 'adjust':
        for name in s:
            add(name)
        b.fill('out', c['rows'], c['vocab'])
        has = lambda name: name if name in s else None   # noqa: E731
        serving.logits_adjust(b, 'logits', 'out', 'par', c['rows'], c['vocab'], **{k: has(k) for k in ('hist', 'plen', 'hlen', 'last', 'bidx', 'bval', 'mask', 'mrow')})
        return b
    cache = serving.kv_q8_buffers(b, '', c['batch'], c['kv'], c['hd'], _tmax(c), c['blk'], c['dtype'])
    add('lens')
    if c['op'] == 'append':
        add('knew'), add('vnew')
        serving.kv_append_q8(b, cache, 'knew', 'vnew', 'lens', n_new=c['n_new'])
        return b
    add('q'), b.fill('o', *s['q'].shape, dtype=c['dtype'])
    if c['rope']:
        add('qgamma')
    serving.attn_decode_q8(b, cache, 'q', 'o', 'lens', c['heads'], n_new=c['n_new'], scale=_scale(c),
                           **(dict(qgamma='qgamma', theta=THETA, eps=EPS) if c['rope'] else {}))
    return b


class _View:
    """A device buffer of an executor in the form that torch takes; keeps the executor while a tensor is alive."""

    def __init__(self, ex, name, shape, kind):
        self.ex = ex
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, data=(ex.device_ptr(name), False), version=2)


def _tensor(ex, m, like):
    """The buffer of metadata entry m as a tensor of `like`'s type and shape."""
    t = torch.as_tensor(_View(ex, m['name'], (m['rows'], m['cols']), {0: '<f4', 1: '<i4', 2: '<i2'}[m['dtype']]), device=DEV)
    return t.view(like.dtype).view(like.shape)


def prepare(case, seed):
    """The inputs, and with `own` the executor that holds them in its buffers, its graph submitted."""
    s = _inputs(case, seed)
    if not own:
        return {'case': case, **s}
    from kvm_amd import bundle as bl
    from kvm_amd import compiler
    from kvm_amd.executor import PATH_AUTO, Executor
    lb = bl.load(compiler.compile_spec(_graph(case, s).spec()))
    ex = Executor.from_bundle(lb, trace=False, timeout_s=60.0, path=PATH_AUTO)
    torch.cuda.synchronize()                                          # the executor's own initialisation is on its own stream
    by = {m['name']: m for m in lb.metadata['buffers']}
    views = {name: _tensor(ex, by[name], x).copy_(x) for name, x in s.items()}
    if case['op'] == 'adjust':
        views['out'] = _tensor(ex, by['out'], s['logits'].float())
    if case['op'] == 'attend':
        views['o'] = _tensor(ex, by['o'], s['q'])
    torch.cuda.synchronize()
    return {'case': case, 'ex': ex, **views}


def run(state):
    c = state['case']
    if own:
        state['ex'].relaunch()
        state['ex'].finish()
        out = state
    else:
        out = {**state, **{'append': _append, 'attend': _attend, 'adjust': _adjust}[c['op']](c, state)}
    return [out[k] for k in _outputs(c)]


def _outputs(case):
    """The 8-bit numbers of an append are compared as the whole numbers that they are, next to their scales."""
    if case['op'] == 'append':
        return ['kq', 'ks', 'vq', 'vs', 'kt', 'vt']
    return ['o'] if case['op'] == 'attend' else ['out', 'hist'] if case['hist'] and case['last'] else ['out']


# ------------------------------------------------------------------------------------------------ plain forms

def _append(c, s):
    """The blocks that the step touches, in one window per sequence: what the unfinished block held, then the new tokens.
    Finished blocks are written in 8 bits; the tokens of the last, unfinished one stay in the model's type."""
    B, n, Hkv, hd, blk, T = c['batch'], c['n_new'], c['kv'], c['hd'], c['blk'], _tmax(c)
    on = s['lens'][:, 0] >= 0
    L = s['lens'][:, 0].clamp(min=0).long()
    first = L // blk                                                  # the block that the first new token falls into
    nb = (n + 2 * blk - 2) // blk
    pos = first[:, None] * blk + torch.arange(nb * blk, device=DEV)   # [B, W]
    old, new = pos < L[:, None], (pos - L[:, None]).clamp(0, n - 1)
    done = (first[:, None] + torch.arange(1, nb + 1, device=DEV)) * blk <= (L + n)[:, None]
    done &= on[:, None]
    b_at, j_at = done.nonzero(as_tuple=True)
    last = (L + n) // blk * blk                                       # where the block left unfinished starts
    row = last[:, None] + torch.arange(blk, device=DEV)
    fresh = (row >= L[:, None]) & (row < (L + n)[:, None]) & on[:, None]
    r = {}
    for x in 'kv':
        tail, got = s[x + 't'], s[x + 'new'].view(B, n, Hkv, hd)
        window = torch.where(old[:, :, None, None], tail.transpose(1, 2).repeat(1, nb, 1, 1),
                             torch.gather(got, 1, new[:, :, None, None].expand(-1, -1, Hkv, hd)))
        blocks = window.view(B, nb, blk, Hkv, hd)[b_at, j_at].transpose(1, 2).float()     # [blocks, kv, blk, hd]
        scale = blocks.abs().amax((2, 3)) / 127
        q = torch.round(blocks.double() / scale.double()[:, :, None, None].clamp(min=1e-300)).clamp(-127, 127).to(torch.int8)
        q = q if x == 'k' else q.transpose(2, 3)
        s[x + 'q'].view(B, Hkv, T // blk, *q.shape[2:])[b_at, :, first[b_at] + j_at] = q
        s[x + 's'][b_at, :, first[b_at] + j_at] = scale
        put = torch.gather(got, 1, (row - L[:, None]).clamp(0, n - 1)[:, :, None, None].expand(-1, -1, Hkv, hd)).transpose(1, 2)
        tail.copy_(torch.where(fresh[:, None, :, None], put, tail))
        r.update({x + y: s[x + y] for y in 'qst'})
    return r


def _turned(c, q, gamma, pos):
    """[B, n, heads, hd] normalised per head and rotated to positions [B, n] (halves rotated together)."""
    hd = c['hd']
    q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * gamma.view(-1)
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    ang = (pos.double()[..., None] * inv)[:, :, None, :]
    co, si = ang.cos().float(), ang.sin().float()
    a, b = q[..., :hd // 2], q[..., hd // 2:]
    return torch.cat([a * co - b * si, a * si + b * co], -1)


def _attend(c, s):
    B, n, H, Hkv, hd, blk, T = c['batch'], c['n_new'], c['heads'], c['kv'], c['hd'], c['blk'], _tmax(c)
    L = s['lens'][:, 0].long()
    pos = torch.arange(T, device=DEV)
    whole = ((L + n) // blk * blk).view(B, 1, 1, 1) > pos[:, None]    # tokens held in 8 bits
    k = (s['kq'].view(B, Hkv, T // blk, -1).float() * s['ks'][..., None]).view(B, Hkv, T, hd)
    v = (s['vq'].view(B, Hkv, T // blk, -1).float() * s['vs'][..., None]).view(B, Hkv, T // blk, hd, blk).transpose(3, 4).reshape(B, Hkv, T, hd)
    k = torch.where(whole, k, s['kt'].float().repeat(1, 1, T // blk, 1))
    v = torch.where(whole, v, s['vt'].float().repeat(1, 1, T // blk, 1))
    at = L[:, None] + torch.arange(n, device=DEV)                     # the queries' positions
    q = s['q'].float().view(B, n, H, hd)
    if c['rope']:
        q = _turned(c, q, s['qgamma'], at.clamp(min=0))
    q = q.view(B, n, Hkv, H // Hkv, hd).transpose(1, 2).reshape(B, Hkv, -1, hd)
    p = (q @ k.transpose(2, 3) * _scale(c)).view(B, Hkv, n, H // Hkv, T)
    p = p.masked_fill((pos > at[:, :, None])[:, None, :, None, :], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-1e30))
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).view(B, Hkv, -1, T)
    o = (p @ v).view(B, Hkv, n, H // Hkv, hd).transpose(1, 2).reshape(B, -1)
    return {'o': torch.where(L[:, None] >= 0, o, 0.0).view(B * n, H * hd).to(s['q'].dtype)}


def _adjust(c, s):
    R, V = c['rows'], c['vocab']
    x = s['logits'].float()
    rep, freq, pres = s['par'][:, 0:1], s['par'][:, 1:2], s['par'][:, 2:3]
    r = {}
    if c['hist']:
        h, at = s['hist'].long(), torch.arange(s['hist'].shape[1], device=DEV)
        said, mine = at < s['hlen'], at >= s['plen']
        count = torch.zeros(R, V, device=DEV).scatter_add_(1, h, (said & mine).float())
        before = torch.zeros(R, V, device=DEV).scatter_add_(1, h, (said & ~mine).float())
        if c['last']:
            count.scatter_add_(1, s['last'].long(), torch.ones(R, 1, device=DEV))
            r['hist'] = s['hist'].scatter_(1, s['hlen'].long(), s['last'])
        x = torch.where((count > 0) | (before > 0), torch.where(x > 0, x / rep, x * rep), x)
        x = x - freq * count - pres * (count > 0)
    if c['bias']:
        x = x + torch.zeros(R, V, device=DEV).scatter_add_(1, s['bidx'].clamp(min=0).long(), torch.where(s['bidx'] >= 0, s['bval'], 0.0))
    if c['mask']:
        v = torch.arange(V, device=DEV)
        ok = (s['mask'][:, v // 32] >> (v % 32)) & 1
        ok = torch.cat([ok, torch.ones(1, V, dtype=ok.dtype, device=DEV)])                 # row -1: everything
        x = x.masked_fill(ok[s['mrow'][:, 0].long()] == 0, -math.inf)
    return {'out': x, **r}


# ------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    """Bytes: inputs and state that a pass reads, and what it writes, once each; flops of the products."""
    c = case
    if c['op'] == 'adjust':
        R, V, e = c['rows'], c['vocab'], 2 if c['dtype'] == 'bf16' else 4
        return {'bytes': R * (V * (e + 4) + 4 * c['hist'] + 8 * c['bias']) + (3 * V // 8 if c['mask'] else 0), 'flops': R * V}
    e, ctx = 2 if c['dtype'] == 'bf16' else 4, c['ctx'] * (0.625 if c['ragged'] else 1)
    if c['op'] == 'append':       # new rows are read, then written in 8 bits or to the unfinished block
        rows = 2 * c['batch'] * c['kv'] * c['n_new']
        return {'bytes': rows * c['hd'] * (e + 1), 'flops': 2 * rows * c['hd']}
    pairs = c['batch'] * c['kv'] * (ctx + c['n_new'])
    return {'bytes': 2 * pairs * c['hd'] + 2 * e * c['batch'] * c['n_new'] * c['heads'] * c['hd'],
            'flops': 4 * pairs * c['hd'] * c['n_new'] * c['heads'] // c['kv']}


# ------------------------------------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {'append': _append64, 'attend': _attend64, 'adjust': _adjust64}[case['op']](case, s)


def _append64(c, s):
    """Sequence by sequence, token after token of a block: the scale is the largest magnitude over 127, kept in f32."""
    blk, n, T, hd = c['blk'], c['n_new'], _tmax(c), c['hd']
    for b, L in enumerate(s['lens'][:, 0].tolist()):
        if L < 0:
            continue
        for x in 'kv':
            tail = s[x + 't'][b]
            rows = torch.cat([tail[:, :L % blk], s[x + 'new'].view(c['batch'], n, c['kv'], hd)[b].transpose(0, 1)], 1)
            full = rows.shape[1] // blk
            a = rows[:, :full * blk].double().reshape(c['kv'], full, blk, hd)
            scale = (a.abs().amax((2, 3)) / 127).float()
            q = torch.where(scale[..., None, None] > 0, a / scale.double()[..., None, None], 0.0).round().to(torch.int8)
            j = L // blk
            s[x + 's'][b, :, j:j + full] = scale
            s[x + 'q'][b].view(c['kv'], T // blk, blk * hd)[:, j:j + full] = (q if x == 'k' else q.transpose(2, 3)).reshape(c['kv'], full, blk * hd)
            left = rows.shape[1] - full * blk
            had = L % blk if full == 0 else 0                        # rows of the unfinished block that were there before
            tail[:, had:left] = rows[:, full * blk + had:]
    return [s[k] for k in _outputs(c)]


def _attend64(c, s):
    B, n, H, Hkv, hd, blk = c['batch'], c['n_new'], c['heads'], c['kv'], c['hd'], c['blk']
    G, out = H // Hkv, torch.zeros(B, n, H, hd, dtype=torch.float64, device=DEV)
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    for b, L in enumerate(s['lens'][:, 0].tolist()):
        if L < 0:
            continue
        full = (L + n) // blk
        kv = []
        for x in 'kv':
            a = s[x + 'q'][b].reshape(Hkv, -1)[:, :full * blk * hd].double().view(Hkv, full, *((blk, hd) if x == 'k' else (hd, blk)))
            a = (a if x == 'k' else a.transpose(2, 3)) * s[x + 's'][b, :, :full, None, None].double()
            kv.append(torch.cat([a.reshape(Hkv, -1, hd), s[x + 't'][b, :, :L + n - full * blk].double()], 1))
        for i in range(n):
            q = s['q'].view(B, n, H, hd)[b, i].double()
            if c['rope']:
                q = q / (q.square().mean(-1, keepdim=True) + EPS).sqrt() * s['qgamma'].view(-1).double()
                z = torch.complex(q[:, :hd // 2], q[:, hd // 2:]) * torch.polar(torch.ones_like(inv), (L + i) * inv)
                q = torch.cat([z.real, z.imag], -1)
            w = torch.softmax(q.view(Hkv, G, hd) @ kv[0][:, :L + i + 1].transpose(1, 2) * _scale(c), -1)
            out[b, i] = (w @ kv[1][:, :L + i + 1]).view(H, hd)
    return [out.view(B * n, H * hd)]


def _adjust64(c, s):
    V, out = c['vocab'], s['logits'].double()
    for r in range(c['rows']):
        x = out[r]
        rep, freq, pres = s['par'][r].double().tolist()
        if c['hist']:
            total, prompt = int(s['hlen'][r]), int(s['plen'][r])
            if c['last']:
                s['hist'][r, total] = s['last'][r, 0]
                total += 1
            said = s['hist'][r, :total].long()
            times = torch.bincount(said[prompt:], minlength=V).double()
            seen = torch.bincount(said, minlength=V) > 0
            x = torch.where(seen & (x > 0), x / rep, torch.where(seen, x * rep, x)) - freq * times - pres * (times > 0).double()
        if c['bias']:
            entry = s['bidx'][r] >= 0
            x = x + torch.bincount(s['bidx'][r][entry].long(), s['bval'][r][entry].double(), minlength=V)
        if c['mask'] and int(s['mrow'][r]) >= 0:
            bits = (s['mask'][int(s['mrow'][r])][:, None].long() >> torch.arange(32, device=DEV)) & 1
            x = torch.where(bits.view(-1)[:V] > 0, x, -math.inf)
        out[r] = x
    return [out, s['hist']] if len(_outputs(c)) == 2 else [out]
