"""The calls whose time the training side of the scene path is judged by: the gradient of the varlen attention, the
gradient of the RMSNorm + RoPE of queries and keys, and the linear layer with bias, activation, gate and residual in its
epilogue with its gradient. Sizes are those of the repository's own workloads (HunyuanVideo-1.5 480p: 1590 tokens a frame,
16 heads x 128, width 2048; Wan2.2 704x1280: 880 tokens a frame) and ragged ones around them.

listed() names the cases, draw(rng) gives more of the same ranges; prepare makes what a program has in hand before the
call, run is one pass (in plain torch, or with `own` through the framework's entry points), exact restates it in 64 bits,
work says what a pass cannot do without. A case is a dict of plain values; lists of lengths are comma-separated text.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = 'cuda'


def listed():
    return [
        # unit-sized models, smoke runs, a prompt's refinement: one query, odd lengths, all launches and latency
        dict(name='attn-bwd-tiny', kind='attn', q='1,77,33', k='64,77,0', start='0,64,141', heads=2, dim=64),
        # fine-tuning a Wan block at 704x1280: 3 scenes x 11 latent frames, each scene reads 2 frames of the next one, so
        # rows of k and v get their gradients from two scenes
        dict(name='attn-bwd-scenes', kind='attn', q='9680,9680,9680', k='11440,11440,9680', start='0,9680,19360',
             heads=16, dim=128),
        # the cross-attention of the same block: every scene's tokens to its own 128-token sentence
        dict(name='attn-bwd-cross', kind='attn', q='9680,9680,9680', k='128,128,128', start='0,128,256', heads=16, dim=128),
        # text and image-prompt encoders on a batch of short ragged sequences
        dict(name='attn-bwd-packed', kind='attn', q='1,77,256,33,410,128,699,5,300,64,512,190',
             k='128,77,300,65,410,1,899,640,33,257,512,31', start='', heads=16, dim=128),
        # CogVideoX-like heads of 64: two videos of one thumbnail each, dense attention
        dict(name='attn-bwd-64', kind='attn', q='3001,3001', k='3001,3001', start='', heads=16, dim=64),
        # a few query tokens against a long video's keys (pooling heads, learned queries)
        dict(name='attn-bwd-few-queries', kind='attn', q='64', k='12720', start='', heads=16, dim=128),
        # the gradient of q and k of one scene layer, 480p x 8 frames
        dict(name='norm-bwd-scene', kind='norm', rows=12720, heads=16, dim=128, rope=True),
        # the key norm of a cross-attention over one odd-sized prompt
        dict(name='norm-bwd-text', kind='norm', rows=77, heads=8, dim=64, rope=False),
        # the feed forward's first product over one scene, the pre-activation kept for the backward pass
        dict(name='linear-ffn', kind='linear', rows=12720, n_in=2048, n_out=8192, act='gelu_tanh', bias=True, gate=False,
             residual=False, keep=True),
        # the time embedding's projection to the six modulation vectors, one row
        dict(name='linear-one-row', kind='linear', rows=1, n_in=2048, n_out=12288, act='silu', bias=True, gate=False,
             residual=False, keep=False),
        # the feed forward's last product and gated residual add, gradients of everything
        dict(name='linear-bwd-ffn', kind='linear_bwd', rows=12720, n_in=8192, n_out=2048, act='', bias=True, gate=True),
        # a projection with an activation over a batch of prompts, odd row count
        dict(name='linear-bwd-text', kind='linear_bwd', rows=333, n_in=1000, n_out=2048, act='gelu_tanh', bias=True,
             gate=False),
    ]


# the largest listed case bounds every drawn one
_MAX_FLOPS, _MAX_BYTES = 6.5e12, 6.0e8


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w['flops'] <= _MAX_FLOPS and w['bytes'] <= _MAX_BYTES:
            return case


def _span(rng, lo, hi):
    """an integer of [lo, hi], spread over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _text(xs):
    return ','.join(str(x) for x in xs)


def _ints(text):
    return [int(x) for x in text.split(',')] if text else []


def _draw(rng):
    kind = rng.choice(['attn', 'attn', 'norm', 'linear', 'linear_bwd'])
    heads, dim = rng.choice([1, 2, 3, 8, 16, 24]), rng.choice([64, 128, 128])
    if kind == 'attn':
        n = _span(rng, 1, 24)
        q = [_span(rng, 1, 12720) for _ in range(n)]
        form = rng.choice(['self', 'cross', 'ranges'])
        # against one key alone the gradients of q and k are zero, and what is computed for them is rounding: such segments
        # come beside others
        least = 2 if n < 4 else 1
        k = [max(x, least) for x in q] if form == 'self' else [_span(rng, least, 12720) for _ in range(n)]
        q = list(k) if form == 'self' else q
        start = []
        if form == 'ranges':
            start = [rng.randrange(0, max(k)) for _ in range(n)]
        elif rng.random() < 0.3:
            k[rng.randrange(n)] = 0
        return dict(kind=kind, q=_text(q), k=_text(k), start=_text(start), heads=heads, dim=dim)
    if kind == 'norm':
        width = rng.choice([512, 1024, 2048, 4096])
        return dict(kind=kind, rows=_span(rng, 1, 24000), heads=width // dim, dim=dim, rope=rng.random() < 0.7)
    rows, n_in, n_out = _span(rng, 1, 16000), 8 * _span(rng, 8, 1024), 8 * _span(rng, 8, 1024)
    act = rng.choice(['', 'gelu_tanh', 'silu'])
    case = dict(kind=kind, rows=rows, n_in=n_in, n_out=n_out, act=act, bias=rng.random() < 0.7, gate=rng.random() < 0.5)
    if kind == 'linear':
        case.update(residual=rng.random() < 0.5, keep=rng.random() < 0.3)
    return case


def work(case):
    if case['kind'] == 'attn':
        q, k = _ints(case['q']), _ints(case['k'])
        width = case['heads'] * case['dim']
        n_k = _key_rows(case)
        # q, o, do in and dq out; k, v in and dk, dv out; one lse a row and head
        return dict(bytes=2 * width * (4 * sum(q) + 4 * n_k) + 4 * case['heads'] * sum(q),
                    flops=10 * width * sum(a * b for a, b in zip(q, k)))
    if case['kind'] == 'norm':
        n, both = case['rows'] * case['heads'] * case['dim'], 2 if case['rope'] else 1
        return dict(bytes=both * 6 * n + (8 * case['rows'] * case['dim'] if case['rope'] else 0), flops=both * 14 * n)
    m, k, n = case['rows'], case['n_in'], case['n_out']
    if case['kind'] == 'linear':
        return dict(bytes=2 * (m * k + n * k + m * n * (1 + case['residual'] + case['keep'])), flops=2 * m * n * k)
    kept = 1 if case['act'] or case['gate'] else 0
    return dict(bytes=2 * (2 * m * k + 2 * n * k + m * n * (1 + kept)), flops=4 * m * n * k)


def _key_rows(case):
    q, k, start = _ints(case['q']), _ints(case['k']), _ints(case['start'])
    return max(a + b for a, b in zip(start, k)) if start else sum(k)


def _cumulated(lengths):
    out = [0]
    out += [sum(lengths[:i + 1]) for i in range(len(lengths))]
    return out


def _key_ranges(case):
    k, start = _ints(case['k']), _ints(case['start'])
    start = start or _cumulated(k)[:-1]
    return [(a, a + n) for a, n in zip(start, k)]


def _query_ranges(case):
    at = _cumulated(_ints(case['q']))
    return list(zip(at, at[1:]))


# ------------------------------------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)
    s = dict(case=case)
    if case['kind'] == 'attn':
        H, D, n_q, n_k = case['heads'], case['dim'], sum(_ints(case['q'])), _key_rows(case)
        # queries and keys as they leave a norm with learned weights: a scale for every dim; the gradient of the output as
        # small as it is behind a mean over a video
        scales = 0.6 + 0.8 * torch.rand(2, 1, 1, D, generator=g, device=DEV)
        s['q'], s['k'] = (randn(n_q, H, D) * scales[0]).bfloat16(), (randn(n_k, H, D) * scales[1]).bfloat16()
        s['v'], s['do'] = randn(n_k, H, D).bfloat16(), (randn(n_q, H, D) / 64).bfloat16()
        s['q_ranges'], s['k_ranges'] = _query_ranges(case), _key_ranges(case)
        # the forward pass's outputs, which a training step has kept
        s['o'], s['lse'] = _attention(s)
        if not case['start']:
            s['cu_q'], s['cu_k'] = (torch.tensor(_cumulated(_ints(case[n])), dtype=torch.int32, device=DEV) for n in 'qk')
            s['max_q'], s['max_k'] = max(_ints(case['q'])), max(_ints(case['k']))
    elif case['kind'] == 'norm':
        S, H, D = case['rows'], case['heads'], case['dim']
        C = H * D
        s['x'] = [(randn(S, C) * 1.5).bfloat16() for _ in range(2)]
        s['w'] = [(1 + 0.1 * randn(C)).bfloat16() for _ in range(2)]
        s['dy'] = [(randn(S, C) / 64).bfloat16() for _ in range(2)]
        angle = torch.rand(S, D // 2, generator=g, device=DEV, dtype=torch.float64) * 2 * math.pi
        s['cos'], s['sin'] = (t.float().repeat_interleave(2, 1) for t in (angle.cos(), angle.sin()))
    else:
        M, K, N = case['rows'], case['n_in'], case['n_out']
        s['x'], s['w'] = randn(M, K).bfloat16(), (randn(N, K) * K ** -0.5).bfloat16()
        s['b'] = (0.1 * randn(N)).bfloat16() if case['bias'] else None
        s['gate'] = 0.5 + 0.5 * randn(N) if case['gate'] else None
        if case['kind'] == 'linear':
            s['residual'] = randn(M, N).bfloat16() if case['residual'] else None
        else:
            s['dy'] = (randn(M, N) / 64).bfloat16()
            # the pre-activation that the forward pass kept
            kept = case['act'] or case['gate']
            s['z'] = _product(s['x'].float(), s['w'].float(), s['b']).bfloat16() if kept else None
    return s


def _product(x, w, b):
    z = x @ w.t()
    return z if b is None else z + b.to(z.dtype)


def _heads_first(x, lo, hi):
    return x[lo:hi].transpose(0, 1).contiguous().float()


def _attention(s):
    parts = [_attend(*(_heads_first(t, *r) for t, r in ((s['q'], a), (s['k'], b), (s['v'], b))))
             for a, b in zip(s['q_ranges'], s['k_ranges'])]
    return torch.cat([o for o, _ in parts], 1).transpose(0, 1).contiguous().bfloat16(), torch.cat([l for _, l in parts], 1)


def _attend(q, k, v):
    if k.shape[1] == 0:
        return torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, device=q.device)
    scores = (q @ k.transpose(1, 2).contiguous()).mul_(q.shape[2] ** -0.5)
    lse = torch.logsumexp(scores, 2)
    return scores.sub_(lse[:, :, None]).exp_() @ v, lse


# ------------------------------------------------------------------------------------------------------------------------
# one pass

def run(s):
    if own:
        return _run_own(s)
    kind = s['case']['kind']
    return _attention_grads(s) if kind == 'attn' else _norm_grads(s) if kind == 'norm' else \
        _linear(s) if kind == 'linear' else _linear_grads(s)


def _run_own(s):
    case = s['case']
    if case['kind'] == 'attn':
        from onereel_amd import attention as A
        if case['start']:
            return A.overlapping_ranges_backward(s['do'], s['q'], s['k'], s['v'], s['o'], s['lse'], s['q_ranges'],
                                                 s['k_ranges'])
        return A.varlen_backward(s['do'], s['q'], s['k'], s['v'], s['o'], s['lse'], s['cu_q'], s['cu_k'], s['max_q'],
                                 s['max_k'], check=False)
    if case['kind'] == 'norm':
        from onereel_amd import wan
        if case['rope']:
            return wan.qk_backward(*s['dy'], *s['x'], *s['w'], 1e-6, s['cos'], s['sin'], case['heads'])
        return wan.rms_norm_backward(s['dy'][0], s['x'][0], s['w'][0], 1e-6)
    from onereel_amd import linear as F
    if case['kind'] == 'linear':
        return F.linear(s['x'], s['w'], s['b'], activation=case['act'] or None, gate=s['gate'], residual=s['residual'],
                        keep_preactivation=case['keep'])
    grads = F.linear_backward(s['dy'], s['x'], s['w'], bias=case['bias'], activation=case['act'] or None, gate=s['gate'],
                              preactivation=s['z'])
    return [t for t in grads if t is not None]


def _attention_grads(s):
    parts = [_attend_grads(_heads_first(s['do'], *a), _heads_first(s['q'], *a), _heads_first(s['k'], *b),
                           _heads_first(s['v'], *b), _heads_first(s['o'], *a), s['lse'][:, a[0]:a[1]])
             for a, b in zip(s['q_ranges'], s['k_ranges'])]
    dq = torch.cat([p[0] for p in parts], 1).transpose(0, 1)
    H, D = s['k'].shape[1:]
    dk, dv = torch.zeros(2, H, s['k'].shape[0], D, device=DEV)
    _ = [(dk[:, a:b].add_(p[1]), dv[:, a:b].add_(p[2])) for p, (a, b) in zip(parts, s['k_ranges'])]
    return tuple(t.to(torch.bfloat16, memory_format=torch.contiguous_format).contiguous()
                 for t in (dq, dk.transpose(0, 1), dv.transpose(0, 1)))


def _attend_grads(do, q, k, v, o, lse):
    if k.shape[1] == 0:
        return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    scale = q.shape[2] ** -0.5
    p = (q @ k.transpose(1, 2).contiguous()).mul_(scale).sub_(lse[:, :, None]).exp_()
    dv = p.transpose(1, 2).contiguous() @ do
    ds = (do @ v.transpose(1, 2).contiguous()).sub_((do * o).sum(2, keepdim=True)).mul_(p)
    return ds @ k * scale, ds.transpose(1, 2).contiguous() @ q * scale, dv


def _norm_grads(s):
    both = 2 if s['case']['rope'] else 1
    done = [_one_norm_grad(s['dy'][i], s['x'][i], s['w'][i], s) for i in range(both)]
    return tuple(d[0] for d in done) + tuple(d[1] for d in done)


def _one_norm_grad(dy, x, w, s):
    g, x, w = dy.float(), x.float(), w.float()
    if s['case']['rope']:
        S, C = g.shape
        c, t = s['cos'][:, None, 0::2], s['sin'][:, None, 1::2]
        g = g.view(S, s['case']['heads'], -1)
        a, b = g[..., 0::2], g[..., 1::2]
        g = torch.stack([a * c + b * t, b * c - a * t], 3).view(S, C)
    inv = (x.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    n = x * inv
    t = g * w
    dx = inv * (t - n * (t * n).mean(1, keepdim=True))
    return dx.bfloat16(), (g * n).sum(0)


def _act(z, name):
    if name == 'silu':
        return z / (1 + torch.exp(-z))
    if name == 'gelu_tanh':
        return 0.5 * z * (1 + torch.tanh(_SQRT * (z + _CUBE * z ** 3)))
    return z


_SQRT, _CUBE = math.sqrt(2 / math.pi), 0.044715


def _act_grad(z, name):
    if name == 'silu':
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == 'gelu_tanh':
        t = torch.tanh(_SQRT * (z + _CUBE * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _SQRT * (1 + 3 * _CUBE * z * z)
    return torch.ones_like(z)


def _linear(s):
    z = _product(s['x'].float(), s['w'].float(), s['b'])
    y = _act(z, s['case']['act'])
    if s['gate'] is not None:
        y = y * s['gate']
    if s['residual'] is not None:
        y = y + s['residual'].float()
    y = y.bfloat16()
    return (y, z.bfloat16()) if s['case']['keep'] else y


def _linear_grads(s):
    case, dy = s['case'], s['dy'].float()
    z = None if s['z'] is None else s['z'].float()
    dz = dy if s['gate'] is None else dy * s['gate']
    if case['act']:
        dz = dz * _act_grad(z, case['act'])
    out = [(dz @ s['w'].float()).bfloat16(), (dz.t() @ s['x'].float()).bfloat16()]
    if case['bias']:
        out.append(dz.sum(0))
    if case['gate']:
        out.append((dy * _act(z, case['act'])).sum(0))
    return out


# ------------------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions: gradients by torch's differentiation of the forward formula where it is one

def exact(case, seed):
    s = prepare(case, seed)
    return {'attn': _attention_exact, 'norm': _norm_exact, 'linear': _linear_exact,
            'linear_bwd': _linear_bwd_exact}[case['kind']](s)


def _attention_exact(s):
    q, k, v, o, do = (s[n].double() for n in ('q', 'k', 'v', 'o', 'do'))
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    scale = q.shape[2] ** -0.5
    for (a, b), (c, d) in zip(s['q_ranges'], s['k_ranges']):
        for h in range(q.shape[1]) if d > c else ():
            qh, kh, vh, doh = q[a:b, h], k[c:d, h], v[c:d, h], do[a:b, h]
            prob = torch.exp(qh @ kh.T * scale - s['lse'][h, a:b, None].double())
            dscore = prob * (doh @ vh.T - (doh * o[a:b, h]).sum(1)[:, None])
            dv[c:d, h] += prob.T @ doh
            dq[a:b, h] = scale * (dscore @ kh)
            dk[c:d, h] += scale * (dscore.T @ qh)
    return dq, dk, dv


def _norm_exact(s):
    case, grads = s['case'], [[], []]
    for i in range(2 if case['rope'] else 1):
        x = s['x'][i].double().requires_grad_()
        w = s['w'][i].double().requires_grad_()
        y = x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + 1e-6) * w
        if case['rope']:
            y = y.view(x.shape[0], case['heads'], case['dim'])
            c, t = s['cos'].double()[:, None, 0::2], s['sin'].double()[:, None, 1::2]
            even, odd = y[..., 0::2], y[..., 1::2]
            y = torch.stack([even * c - odd * t, even * t + odd * c], 3).reshape(x.shape)
        for to, grad in zip(grads, torch.autograd.grad(y, (x, w), s['dy'][i].double())):
            to.append(grad)
    return tuple(grads[0]) + tuple(grads[1])


def _act_exact(z, name):
    if name == 'silu':
        return z * torch.sigmoid(z)
    return torch.nn.functional.gelu(z, approximate='tanh') if name else z


def _linear_exact(s):
    case = s['case']
    z = s['x'].double() @ s['w'].double().T
    if case['bias']:
        z = z + s['b'].double()
    y = _act_exact(z, case['act'])
    if case['gate']:
        y = s['gate'].double() * y
    if case['residual']:
        y = s['residual'].double() + y
    return (y, z) if case['keep'] else y


def _linear_bwd_exact(s):
    case, dy = s['case'], s['dy'].double()
    if s['z'] is None:
        dz, dgate = dy, None
    else:
        z = s['z'].double().requires_grad_()
        gate = (torch.ones(z.shape[1], device=DEV) if s['gate'] is None else s['gate']).double().requires_grad_()
        dz, dgate = torch.autograd.grad(_act_exact(z, case['act']) * gate, (z, gate), dy)
    out = [dz @ s['w'].double(), dz.T @ s['x'].double()]
    if case['bias']:
        out.append(dz.sum(0))
    if case['gate']:
        out.append(dgate)
    return out
