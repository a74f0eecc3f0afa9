"""Measured cases of the operators that serve prompts and tokens together: products in 8-bit integers with the quantisation of their
rows, the append to a paged key / value cache, and the attention of new tokens over it.

`own` chooses what a pass runs: the plain forms below (elementary torch operations in 32 bits, in 64 where a rounding decides), or the
framework's operators, as tasks of a graph that a program submits once and launches for every step. The buffers live on the GPU for as
long as the program does; outputs are those buffers.

Layouts (registry operators rows_q8, matmul_q8, gemv_q8, qkv_append_paged, attn_paged):
  w, ws  [N, K] bytes (rows padded with zeros to 16 bytes) and [N, 1] f32: a weight is byte * scale of its row
  kc, vc [pages * kv heads * page, hd]: a page holds `page` tokens of every kv head, head by head
  table  [batch, pages of a sequence]: which page holds tokens j * page .. of a sequence; -1 where none is given yet
  lens   [batch]: tokens of a sequence that the cache holds before the step
  cu     [batch + 1]: the new tokens of sequence b are the rows cu[b] .. cu[b + 1] - 1; rows behind cu[batch] belong to nobody
"""
from __future__ import annotations

import math

import torch

own = False

DEV = 'cuda'


def listed():
    return [
        # a prompt's rows in front of a layer's projections: RMSNorm, then 8 bits
        dict(name='quant_prompt', op='quant', dtype='bf16', M=4001, K=4096, pro='norm'),
        # rows of a small f32 model, no multiple of a vector
        dict(name='quant_rows_f32', op='quant', dtype='f32', M=640, K=1001, pro='none'),
        # one user's next token: a feed-forward projection, bound by its weights
        dict(name='linear_token', op='linear', dtype='bf16', M=1, K=4096, N=12288, pro='norm', bias=False, res=False),
        # a served batch through the down projection, SwiGLU in front and the residual behind
        dict(name='linear_batch', op='linear', dtype='bf16', M=8, K=12288, N=4096, pro='swiglu', bias=False, res=True),
        # a chunk of a prompt in a small f32 model with biases, ragged in every direction
        dict(name='linear_chunk_f32', op='linear', dtype='f32', M=333, K=1001, N=2777, pro='none', bias=True, res=False),
        # a whole prompt through a feed-forward projection
        dict(name='linear_prompt', op='linear', dtype='bf16', M=4001, K=4096, N=12288, pro='norm', bias=False, res=False),
        # a served batch's next tokens: norm and rotation of queries and keys, keys and values to their pages
        dict(name='append_batch', op='append', dtype='bf16', batch=96, new=1, kind='all', heads=32, kv=8, hd=128, page=64, ctx=1000),
        # prompts of a small f32 model behind shared beginnings, no length like another
        dict(name='append_prompts_f32', op='append', dtype='f32', batch=5, new=777, kind='ragged', heads=16, kv=4, hd=64, page=16, ctx=256),
        # one user with a long document
        dict(name='attend_token', op='attend', dtype='bf16', batch=1, new=1, kind='all', heads=32, kv=8, hd=128, page=64, ctx=32000),
        # a served batch's next tokens
        dict(name='attend_batch', op='attend', dtype='bf16', batch=48, new=1, kind='all', heads=32, kv=8, hd=128, page=64, ctx=8000),
        # a chunk of a long prompt beside the next tokens of other users
        dict(name='attend_chunk', op='attend', dtype='bf16', batch=9, new=1000, kind='mixed', heads=32, kv=8, hd=128, page=32, ctx=6000),
        # a small f32 model: prompts' ends and slots without a new token
        dict(name='attend_ragged_f32', op='attend', dtype='f32', batch=6, new=33, kind='ragged', heads=16, kv=4, hd=64, page=16, ctx=1531),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['quant', 'linear', 'linear', 'append', 'attend', 'attend', 'attend'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    if op == 'quant':
        K = _log(rng, 60, 12288)
        return dict(op=op, dtype=dtype, M=_log(rng, 1, min(8000, 20_000_000 // K)), K=K, pro=rng.choice(['none', 'norm']))
    if op == 'linear':
        K, N = rng.choice([_log(rng, 60, 12288), 16 * _log(rng, 4, 768)]), _log(rng, 60, 12288)
        M = rng.choice([1, _log(rng, 1, 16), _log(rng, 16, 4000)])
        while M * K * N > 190_000_000_000:
            M //= 2
        return dict(op=op, dtype=dtype, M=M, K=K, N=N, pro=rng.choice(['none', 'norm', 'swiglu'] if dtype == 'bf16' else ['none']), bias=rng.random() < 0.3,
                    res=rng.random() < 0.3)
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 4, 6, 8])
    c = dict(op=op, dtype=dtype, heads=kv * group, kv=kv, hd=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 64, 128]))
    if op == 'append':
        new = rng.choice([1, 1, _log(rng, 2, 2000)])
        return dict(c, batch=_log(rng, 1, min(128, 1 + 4000 // new)), new=new, kind='all' if new == 1 else rng.choice(['all', 'ragged', 'mixed']), ctx=_log(rng, 1, 2000))
    small = dtype == 'f32'                                             # small models: fewer and shorter sequences
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 200 if small else 1000)])
    batch = _log(rng, 1, min(64, 1 + (1500 if small else 4000) // new))
    kind = 'all' if new == 1 else 'mixed' if batch * new > (400 if small else 1000) else rng.choice(['all', 'ragged', 'mixed'])
    room = (400_000 if small else 3_000_000) // (batch * kv)           # tokens of a sequence, by the cache and by the scores of a padded batch
    return dict(c, batch=batch, new=new, kind=kind, ctx=_log(rng, 1, max(1, min(40000, room, 1_500_000_000 // (batch * new * c['heads']) - new))))


# ------------------------------------------------------------------------------------------------ inputs

THETA, EPS = 1e6, 1e-6


def _pages(case):
    """Pages of a sequence, with room for the step."""
    return -(-(case['ctx'] + case['new']) // case['page']) + 1


def _inputs(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    dt = torch.bfloat16 if c['dtype'] == 'bf16' else torch.float32
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)   # noqa: E731
    ints = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV, dtype=torch.int32)   # noqa: E731
    if c['op'] in ('quant', 'linear'):
        M, K = c['M'], c['K']
        s = {'x': (randn(M, K) * torch.exp(0.5 * randn(1, K))).to(dt)}           # a few channels far larger than the others
        if c['pro'] == 'norm':
            s['gamma'] = 1 + 0.2 * randn(1, K)
        if c['pro'] == 'swiglu':
            s['x2'] = randn(M, K).to(dt)
        if c['op'] == 'linear':
            s['w'] = torch.zeros(c['N'], -(-K // 16) * 16, dtype=torch.int8, device=DEV)
            s['w'][:, :K] = (32 * randn(c['N'], K)).round().clamp(-127, 127)
            s['ws'] = torch.exp(0.3 * randn(c['N'], 1)) / (32 * math.sqrt(K))
            if c['bias']:
                s['bias'] = randn(1, c['N'])
            if c['res']:
                s['res'] = randn(M, c['N']).to(dt)
        return s
    B, n, Hkv, hd, page, P = c['batch'], c['new'], c['kv'], c['hd'], c['page'], _pages(c)
    lens = ints(c['ctx'] // 4, c['ctx'] + 1, B) if B > 1 else torch.full((1,), c['ctx'], dtype=torch.int32, device=DEV)
    new = torch.full((B,), n, dtype=torch.int32, device=DEV)
    if c['kind'] == 'ragged':                                          # any number of new tokens, none too
        new = ints(0, n + 1, B)
    if c['kind'] == 'mixed':                                           # one prompt's chunk, next tokens of the others
        new = torch.where(torch.arange(B, device=DEV) == B // 2, n, 1).int()
    s = {'lens': lens[:, None].contiguous(), 'cu': torch.cat([new.new_zeros(1), new.cumsum(0).int()])[:, None].contiguous()}
    used = (lens + new + page - 1) // page
    table = torch.randperm(B * P, generator=g, device=DEV).int().view(B, P)
    s['table'] = torch.where(torch.arange(P, device=DEV) < used[:, None], table, -1).int()
    s['kc'], s['vc'] = randn(B * P * Hkv * page, hd).to(dt), randn(B * P * Hkv * page, hd).to(dt)
    R = _rows(c)
    s['q'] = randn(R, c['heads'] * hd).to(dt)
    if c['op'] == 'append':
        s['k'], s['v'] = (randn(R, Hkv, hd) * torch.exp(0.5 * randn(Hkv, hd))).to(dt).view(R, -1), randn(R, Hkv * hd).to(dt)
        s['qgamma'], s['kgamma'] = 1 + 0.2 * randn(1, hd), 1 + 0.2 * randn(1, hd)
    return s


def _rows(case):
    """Rows of a step's buffers: the most that it brings."""
    return case['new'] + case['batch'] - 1 if case['kind'] == 'mixed' else case['batch'] * case['new']


def _graph(case, s):
    """The step's graph, as a serving program lays it out with the task builders of kvm_amd.workloads.serving."""
    from kvm_amd.workloads import Builder, serving
    c, b, kind = case, Builder(0), {torch.float32: 'f32', torch.int32: 'i32', torch.bfloat16: 'bf16'}
    add = lambda name: b.fill(name, *s[name].shape, dtype=kind[s[name].dtype])   # noqa: E731
    has = lambda name: add(name) if name in s else None   # noqa: E731
    if c['op'] == 'quant':
        serving.rows_q8(b, add('x'), serving.rows_q8_buffers(b, 'y', c['M'], c['K']), c['M'], gamma=has('gamma'), eps=EPS)
        return b
    if c['op'] == 'linear':
        w = serving.weight_q8_buffers(b, 'w', c['N'], c['K'])
        b.fill('out', c['M'], c['N'], dtype=c['dtype'])
        serving.linear_q8(b, add('x'), w, 'out', c['M'], x2=has('x2'), gamma=has('gamma'), bias=has('bias'), res=has('res'), eps=EPS)
        return b
    cache = serving.paged_buffers(b, '', c['batch'] * _pages(c), c['kv'], c['hd'], c['page'], c['dtype'])
    add('lens'), add('cu'), add('table'), add('q')
    b.fill('o', *s['q'].shape, dtype=c['dtype'])
    if c['op'] == 'append':
        serving.qkv_append_paged(b, cache, add('k'), add('v'), 'table', 'lens', 'cu', q='q', qo='o', heads=c['heads'], qgamma=add('qgamma'), kgamma=add('kgamma'),
                                 theta=THETA, eps=EPS)
    else:
        serving.attn_paged(b, cache, 'q', 'o', 'table', 'lens', 'cu', c['heads'])
    return b


class _View:
    """A device buffer of an executor in the form that torch takes; keeps the executor while a tensor is alive."""

    def __init__(self, ex, name, shape, kind):
        self.ex = ex
        self.__cuda_array_interface__ = dict(shape=shape, typestr=kind, data=(ex.device_ptr(name), False), version=2)


def _tensor(ex, m):
    """The buffer of metadata entry m as a tensor."""
    t = torch.as_tensor(_View(ex, m['name'], (m['rows'], m['cols']), {0: '<f4', 1: '<i4', 2: '<i2'}[m['dtype']]), device=DEV)
    return t.view(torch.bfloat16) if m['dtype'] == 2 else t


def prepare(case, seed):
    """The inputs, and with `own` the executor that holds them in its buffers, its graph submitted."""
    s = _inputs(case, seed)
    if case['op'] in ('append', 'attend'):
        s['o'] = torch.zeros_like(s['q'])                              # rows behind the last sequence stay as they are
    if not own:
        return {'case': case, **s}
    from kvm_amd import bundle as bl
    from kvm_amd import compiler
    from kvm_amd.executor import PATH_AUTO, Executor
    lb = bl.load(compiler.compile_spec(_graph(case, s).spec()))
    ex = Executor.from_bundle(lb, trace=False, timeout_s=60.0, path=PATH_AUTO)
    torch.cuda.synchronize()                                          # the executor's own initialisation is on its own stream
    t = {m['name']: _tensor(ex, m) for m in lb.metadata['buffers']}
    for name, x in s.items():
        t[name].copy_(x.view(torch.int32) if x.dtype == torch.int8 else x)
    torch.cuda.synchronize()
    if case['op'] == 'quant':
        t['y'], t['ys'] = t['y'].view(torch.int8)[:, :case['K']], t['ys']
    return {'case': case, 'ex': ex, **t}


def run(state):
    c = state['case']
    if own:
        state['ex'].relaunch()
        state['ex'].finish()
        out = state
    else:
        out = {**state, **{'quant': _quant, 'linear': _linear, 'append': _append, 'attend': _attend}[c['op']](c, state)}
    return [out[k] for k in {'quant': ['y', 'ys'], 'linear': ['out'], 'append': ['kc', 'vc', 'o'], 'attend': ['o']}[c['op']]]


# ------------------------------------------------------------------------------------------------ plain forms

def _quant(c, s):
    """A row is what stands in front of it (RMSNorm; silu(x) * x2), over its largest magnitude / 127, rounded to whole numbers."""
    x = s['x'].float()
    if c['pro'] == 'norm':
        rstd = (1 / (s['x'].double().square().mean(1, keepdim=True) + EPS).sqrt()).float()
        x = x * rstd * s['gamma']
    if c['pro'] == 'swiglu':
        x = x / (1 + torch.exp(-x)) * s['x2'].float()
    scale = x.abs().amax(1, keepdim=True) * torch.tensor(1 / 127, device=DEV)
    q = torch.round(x.double() / scale.double().clamp(min=1e-300)).clamp(-127, 127)
    return {'y': q.to(torch.int8), 'ys': scale}


def _linear(c, s):
    q = _quant(c, s)
    y = (q['y'].float() @ s['w'][:, :c['K']].float().t()) * q['ys'] * s['ws'].t()
    if c['bias']:
        y = y + s['bias']
    if c['res']:
        y = y + s['res'].float()
    return {'out': y.to(s['x'].dtype)}


def _owners(s, R):
    """Of every row: its sequence, its number among the sequence's new tokens, and whether it has one."""
    row, cu = torch.arange(R, device=DEV, dtype=torch.int32), s['cu'][:, 0]
    b = torch.searchsorted(cu[1:].contiguous(), row, right=True).clamp(max=len(cu) - 2)
    return b, row - cu[b], row < cu[-1]


def _turned(c, x, gamma, pos):
    """[rows, heads, hd] normalised per head and rotated to positions [rows] (halves rotated together)."""
    hd = c['hd']
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.view(-1)
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    ang = (pos.double()[:, None] * inv)[:, None, :]
    co, si = ang.cos().float(), ang.sin().float()
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([a * co - b * si, a * si + b * co], -1)


def _append(c, s):
    R, Hkv, hd, page, dt = s['q'].shape[0], c['kv'], c['hd'], c['page'], s['q'].dtype
    b, i, on = _owners(s, R)
    pos = torch.where(on, s['lens'][b, 0] + i, 0)
    q = _turned(c, s['q'].float().view(R, -1, hd), s['qgamma'], pos).to(dt)
    k = _turned(c, s['k'].float().view(R, Hkv, hd), s['kgamma'], pos).to(dt)
    where, at = s['table'][b, (pos // page).long()].long()[on], (pos % page).long()[on]
    for name, x in (('kc', k), ('vc', s['v'].view(R, Hkv, hd))):
        s[name].view(-1, Hkv, page, hd)[where, :, at] = x[on]
    s['o'][on] = q.view(R, -1)[on]
    return {}


def _attend(c, s):
    B, n, H, Hkv, hd, page, P = c['batch'], c['new'], c['heads'], c['kv'], c['hd'], c['page'], _pages(c)
    T, at, cu, L = P * page, s['table'].long().clamp(min=0), s['cu'][:, 0].long(), s['lens'][:, 0].long()
    k = s['kc'].view(-1, Hkv, page, hd)[at].transpose(1, 2).reshape(B, Hkv, T, hd).float()
    v = s['vc'].view(-1, Hkv, page, hd)[at].transpose(1, 2).reshape(B, Hkv, T, hd).float()
    i = torch.arange(n, device=DEV)
    on = i < (cu[1:] - cu[:-1])[:, None]                               # [B, n]
    row = (cu[:-1, None] + i).clamp(max=s['q'].shape[0] - 1)
    q = s['q'][row].float().view(B, n, Hkv, H // Hkv, hd).transpose(1, 2).reshape(B, Hkv, -1, hd)
    p = (q @ k.transpose(2, 3)).mul_(1 / math.sqrt(hd)).view(B, Hkv, n, H // Hkv, T)
    p.masked_fill_((torch.arange(T, device=DEV) > (L[:, None] + i)[:, :, None])[:, None, :, None, :], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, Hkv, -1, T)
    o = (p @ v).view(B, Hkv, n, H // Hkv, hd).transpose(1, 2).reshape(B, n, H * hd)
    s['o'][row[on]] = o[on].to(s['o'].dtype)
    return {}


# ------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    """Bytes: inputs and state that a pass reads, and what it writes, once each; flops of the products."""
    c, e = case, 2 if case['dtype'] == 'bf16' else 4
    if c['op'] in ('quant', 'linear'):
        M, K = c['M'], c['K']
        x = M * K * e * (2 if c['pro'] == 'swiglu' else 1) + (4 * K if c['pro'] == 'norm' else 0)
        if c['op'] == 'quant':
            return {'bytes': x + M * K + 4 * M, 'flops': 4 * M * K}
        N = c['N']
        return {'bytes': x + N * K + 4 * N + e * M * N * (2 if c['res'] else 1), 'flops': 2 * M * N * K}
    B, n, H, Hkv, hd = c['batch'], c['new'], c['heads'], c['kv'], c['hd']
    rows = _rows(c) * (0.5 if c['kind'] == 'ragged' else 1)
    if c['op'] == 'append':
        return {'bytes': int(2 * rows * (H + 2 * Hkv) * hd * e), 'flops': int(8 * rows * (H + Hkv) * hd)}
    ctx = c['ctx'] * (0.625 if B > 1 else 1)
    pairs = rows * ctx + ((n * n + B) / 2 if c['kind'] == 'mixed' else B * n * n / (6 if c['kind'] == 'ragged' else 2))
    return {'bytes': int(2 * B * (ctx + rows / B) * Hkv * hd * e + 2 * rows * H * hd * e), 'flops': int(4 * pairs * H * hd)}


# ------------------------------------------------------------------------------------------------ the same in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    return {'quant': _quant64, 'linear': _linear64, 'append': _append64, 'attend': _attend64}[case['op']](case, s)


def _quant64(c, s):
    x = s['x'].double()
    if c['pro'] == 'norm':
        x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * s['gamma'].double()
    if c['pro'] == 'swiglu':
        x = x * torch.sigmoid(x) * s['x2'].double()
    scale = x.abs().amax(1, keepdim=True) / 127
    return [(x / scale).round().to(torch.int8), scale]


def _linear64(c, s):
    q, scale = _quant64(c, s)
    y = (q.double() @ s['w'][:, :c['K']].double().t()) * scale * s['ws'].double().t()
    return [y + (s['bias'].double() if c['bias'] else 0) + (s['res'].double() if c['res'] else 0)]


def _append64(c, s):
    """Sequence by sequence, a token at a time in the page that its position names."""
    hd, page, Hkv, out = c['hd'], c['page'], c['kv'], torch.zeros_like(s['q'], dtype=torch.float64)
    inv = THETA ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEV) / hd)
    kc, vc = (s[x].double().view(-1, Hkv, page, hd) for x in ('kc', 'vc'))
    cu = s['cu'][:, 0].tolist()
    for b, L in enumerate(s['lens'][:, 0].tolist()):
        pos = torch.arange(L, L + cu[b + 1] - cu[b], device=DEV)
        turned = []
        for x in 'qk':
            y = s[x][cu[b]:cu[b + 1]].double().view(len(pos), c['heads'] if x == 'q' else Hkv, hd)
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * s[x + 'gamma'].view(-1).double()
            z = torch.complex(y[..., :hd // 2], y[..., hd // 2:]) * torch.polar(torch.ones(len(pos), 1, hd // 2, dtype=torch.float64, device=DEV), (pos[:, None] * inv)[:, None])
            turned.append(torch.cat([z.real, z.imag], -1))
        out[cu[b]:cu[b + 1]] = turned[0].flatten(1)
        where = s['table'][b].long()[pos // page]
        kc[where, :, pos % page] = turned[1]
        vc[where, :, pos % page] = s['v'][cu[b]:cu[b + 1]].double().view(len(pos), Hkv, hd)
    return [kc.view(-1, hd), vc.view(-1, hd), out]


def _attend64(c, s):
    H, Hkv, hd, out = c['heads'], c['kv'], c['hd'], torch.zeros_like(s['q'], dtype=torch.float64)
    cu, kc, vc = s['cu'][:, 0].tolist(), s['kc'].view(-1, Hkv, c['page'], hd), s['vc'].view(-1, Hkv, c['page'], hd)
    for b, L in enumerate(s['lens'][:, 0].tolist()):
        n = cu[b + 1] - cu[b]
        pages = s['table'][b, :-(-(L + n) // c['page'])].long()
        keep = torch.arange(L + n, device=DEV) <= L + torch.arange(n, device=DEV)[:, None]
        for h in range(H):
            k, v = (x[pages, h * Hkv // H].reshape(-1, hd)[:L + n].double() for x in (kc, vc))
            p = s['q'][cu[b]:cu[b + 1], h * hd:(h + 1) * hd].double() @ k.t() / math.sqrt(hd)
            out[cu[b]:cu[b + 1], h * hd:(h + 1) * hd] = torch.softmax(p.masked_fill(~keep, -math.inf), -1) @ v
    return [out]
