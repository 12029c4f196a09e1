"""The operators of a language model's step that surround its matrix products:
embedding lookup and its gradient, the root-mean-square norm (with the
residual's addition, in 8 bits, and its gradient), log probabilities of given
tokens with their gradient, and the clipping of gradients by their global norm.

``own = False`` computes them with elementary torch operations, ``own = True``
calls the package's functions on the same memory.
"""
import math

import torch

own = False

_F = {'f16': torch.float16, 'f32': torch.float32}
_SIZE = {'f16': 2, 'f32': 4}
_EPS = 1e-6


# -- the cases ------------------------------------------------------------------------

def listed():
    return [
        # the lookup of one decoding step for a small batch
        {'name': 'lookup, one step', 'op': 'embed', 'tokens': 8, 'rows': 32768, 'width': 4096,
         'type': 'f16', 'scale': 1.0},
        # the lookup of a batch of prompts, embeddings scaled by sqrt(width)
        {'name': 'lookup, prompts', 'op': 'embed', 'tokens': 16384, 'rows': 50257, 'width': 2048,
         'type': 'f32', 'scale': 45.25},
        # gradient of a table of a large vocabulary: few of its rows are met
        {'name': 'table gradient, large', 'op': 'embed_grad', 'tokens': 16384, 'rows': 131072,
         'width': 2048, 'type': 'f16', 'out': 'f16', 'scale': 1.0},
        # a small model in float32, a width that fills no whole vectors
        {'name': 'table gradient, odd', 'op': 'embed_grad', 'tokens': 4001, 'rows': 8191,
         'width': 509, 'type': 'f32', 'out': 'f32', 'scale': 1.0},
        # decoding: a handful of rows between two layers
        {'name': 'norm, one step', 'op': 'norm', 'tokens': 8, 'width': 8192, 'type': 'f16'},
        # a prompt, activations handed on in 8 bits
        {'name': 'norm to int8, prompt', 'op': 'norm_int8', 'tokens': 4096, 'width': 8192,
         'type': 'f16'},
        # float32 training with a ragged batch
        {'name': 'norm, odd', 'op': 'norm', 'tokens': 9001, 'width': 2047, 'type': 'f32'},
        # the backward pass of one norm in training
        {'name': 'norm gradient', 'op': 'norm_grad', 'tokens': 16384, 'width': 4096, 'type': 'f16'},
        # scoring while decoding: entropy and 20 alternatives for each sequence
        {'name': 'log probs, one step', 'op': 'log_prob', 'tokens': 8, 'vocab': 131072,
         'type': 'f32', 'entropy': True, 'top': 20, 'masked': True},
        # the loss of a training step over a batch of packed sequences
        {'name': 'log probs, training', 'op': 'log_prob', 'tokens': 8192, 'vocab': 50257,
         'type': 'f16', 'entropy': True, 'top': 0, 'masked': False},
        # ... and its gradient, with a bonus for entropy
        {'name': 'log probs, gradient', 'op': 'log_prob_grad', 'tokens': 8192, 'vocab': 50257,
         'type': 'f16', 'entropy': True},
        # gradients of a model's many matrices and vectors
        {'name': 'clipping, many tensors', 'op': 'clip', 'layers': 24, 'width': 1024,
         'type': 'f16', 'share': 0.5},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['embed', 'embed_grad', 'norm', 'norm_int8', 'norm_grad', 'log_prob',
                     'log_prob_grad', 'clip'])
    kind = rng.choice(['f16', 'f32'])
    if op == 'embed':
        rows, width = _log_int(rng, 1000, 131072), _log_int(rng, 64, 8192)
        rows = min(rows, (1 << 29) // (width * 4))
        tokens = min(_log_int(rng, 1, 32768), (1 << 26) // width)
        return {'op': op, 'tokens': tokens, 'rows': rows, 'width': width, 'type': kind,
                'scale': rng.choice([1.0, round(math.sqrt(width), 3)])}
    if op == 'embed_grad':
        rows, width = _log_int(rng, 1000, 131072), _log_int(rng, 64, 4096)
        rows = min(rows, (1 << 27) // width)
        tokens = min(_log_int(rng, 16, 32768), (1 << 26) // width)
        return {'op': op, 'tokens': tokens, 'rows': rows, 'width': width, 'type': kind,
                'out': rng.choice([kind, 'f32']), 'scale': rng.choice([1.0, round(math.sqrt(width), 3)])}
    if op in ('norm', 'norm_int8', 'norm_grad'):
        width = _log_int(rng, 64, 16384)
        return {'op': op, 'tokens': min(_log_int(rng, 1, 65536), (1 << 26) // width),
                'width': width, 'type': kind}
    if op == 'log_prob':
        vocab = _log_int(rng, 1000, 200000)
        top = rng.choice([0, 0, 1, 5, 20])
        most = min(1 << 25 if top else 1 << 28, (1 << 29) // _SIZE[kind]) // vocab
        return {'op': op, 'tokens': min(_log_int(rng, 1, 16384), most), 'vocab': vocab,
                'type': kind, 'entropy': rng.random() < 0.5, 'top': top,
                'masked': rng.random() < 0.5}
    if op == 'log_prob_grad':
        vocab = _log_int(rng, 1000, 200000)
        most = (1 << 29) // _SIZE[kind] // vocab
        return {'op': op, 'tokens': min(_log_int(rng, 1, 16384), most), 'vocab': vocab,
                'type': kind, 'entropy': rng.random() < 0.5}
    width = _log_int(rng, 64, 1024)
    layers = min(rng.randint(1, 24), (1 << 29) // _SIZE[kind] // (12 * width * width))
    return {'op': op, 'layers': layers, 'width': width, 'type': kind,
            'share': rng.choice([0.01, 0.5, 2.0])}


# -- inputs ---------------------------------------------------------------------------

def _tokens(g, n, rows):
    """Tokens as texts have them: the r-th most frequent about 1/r of the time,
    frequent ones anywhere in the table."""
    u = torch.rand(n, generator=g, device='cuda', dtype=torch.float64)
    rank = (torch.exp(u * math.log(rows)) - 1).long().clamp_(0, rows - 1)
    return (rank * 7919 + 13) % rows if rows % 7919 else rank


def _normal(g, shape, kind, spread=1.0):
    return (torch.randn(shape, generator=g, device='cuda') * spread).to(_F[kind])


def _shapes(case):
    """The tensors of a model: per layer two norms, the fused projections of
    attention and the feed-forward matrices of four times the width."""
    d = case['width']
    layer = [(d,), (3 * d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)]
    return layer * case['layers'] + [(d,)]


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    op, kind = case['op'], case.get('type')
    dev = {'device': 'cuda'}
    s = {'case': case}
    if op == 'embed':
        s['table'] = _normal(g, (case['rows'], case['width']), kind, 0.02)
        s['ids'] = _tokens(g, case['tokens'], case['rows'])
        o = {'out': torch.empty((case['tokens'], case['width']), dtype=_F[kind], **dev)}
    elif op == 'embed_grad':
        s['grad'] = _normal(g, (case['tokens'], case['width']), kind, 0.1)
        s['ids'] = _tokens(g, case['tokens'], case['rows'])
        s['ids'][::17] = -1    # positions of padding
        o = {'out': torch.empty((case['rows'], case['width']), dtype=_F[case['out']], **dev)}
    elif op in ('norm', 'norm_int8', 'norm_grad'):
        shape = (case['tokens'], case['width'])
        s['x'] = _normal(g, shape, kind, 0.5)
        s['other'] = _normal(g, shape, kind, 2.0)    # the residual, or its gradient
        s['weight'] = (1 + 0.1 * torch.randn(case['width'], generator=g, device='cuda')).to(_F[kind])
        o = {'sum': torch.empty(shape, dtype=_F[kind], **dev)}
        if op == 'norm':
            o['out'] = torch.empty(shape, dtype=_F[kind], **dev)
        elif op == 'norm_int8':
            o['out'] = torch.empty(shape, dtype=torch.int8, **dev)
            o['scale'] = torch.empty(shape[:1], dtype=torch.float32, **dev)
            o['values'] = torch.empty(shape, dtype=torch.float16, **dev)
        else:
            s['grad'] = _normal(g, shape, kind, 0.1)
            o['weight'] = torch.empty(shape[1:], dtype=_F[kind], **dev)
    elif op in ('log_prob', 'log_prob_grad'):
        n, v = case['tokens'], case['vocab']
        s['logits'] = _normal(g, (n, v), kind, 2.5)
        s['tokens'] = torch.randint(0, v, (n,), generator=g, device='cuda')
        # half of the tokens are likely ones, as a model's own answers are
        s['logits'][torch.arange(0, n, 2, device='cuda'), s['tokens'][::2]] = 9.0
        f32 = {'dtype': torch.float32, **dev}
        if op == 'log_prob':
            if case['masked']:    # words that a grammar rules out here
                s['logits'][:, 5::7] = -math.inf
                s['tokens'] = torch.where(s['tokens'] % 7 == 5, s['tokens'] - 1, s['tokens'])
            o = {'log_prob': torch.empty(n, **f32), 'lse': torch.empty(n, **f32)}
            if case['entropy']:
                o['entropy'] = torch.empty(n, **f32)
            if case['top']:
                o['top'] = torch.empty((n, case['top']), **f32)
                o['index'] = torch.empty((n, case['top']), dtype=torch.int64, **dev)
        else:
            s['tokens'][::13] = -1    # positions without a target
            # advantages under a loss scale
            s['grad'] = 128.0 * torch.randn(n, generator=g, **f32)
            x = s['logits'].double()
            lse = torch.logsumexp(x, -1)
            s['lse'] = lse.float()
            if case['entropy']:
                p = torch.exp(x - lse[:, None])
                s['entropy'] = (lse - (p * x).sum(-1)).float()
                s['entropy_grad'] = torch.full((n,), 12.8, **f32)
            del x
            o = {'out': torch.empty((n, v), dtype=_F[kind], **dev)}
    else:
        shapes = _shapes(case)
        sizes = [math.prod(t) for t in shapes]
        s['arrays'] = [_normal(g, t, kind, 0.01) for t in shapes]
        s['max_norm'] = 0.01 * math.sqrt(sum(sizes)) * case['share']
        o = {'flat': torch.empty(sum(sizes), dtype=_F[kind], **dev),
             'norm': torch.empty((), dtype=torch.float32, **dev)}
        s['views'] = [p.view(t) for p, t in zip(o['flat'].split(sizes), shapes)]
    s['o'] = o
    if own:
        # a program of this package holds these as its own arrays (views of the same memory)
        import cupy_amd
        wrap = cupy_amd.asarray
        s['c'] = {k: wrap(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        s['r'] = {k: wrap(v) for k, v in o.items()}
        for k in ('arrays', 'views'):
            if k in s:
                s['c'][k] = [wrap(v) for v in s[k]]
        if op == 'norm_int8':
            s['r']['column'] = s['r']['scale'].reshape(-1, 1)
        if op == 'log_prob':
            r = s['r']
            s['r'] = cupy_amd.TokenLogProb(r['log_prob'], r['lse'], r.get('entropy'),
                                           r.get('top'), r.get('index'))
    return s


# -- one pass -------------------------------------------------------------------------

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import cupy_amd as cupy
    case, c, r, o = s['case'], s['c'], s['r'], s['o']
    op = case['op']
    if op == 'embed':
        cupy.embedding(c['table'], c['ids'], case['scale'], out=r['out'])
        return o['out']
    if op == 'embed_grad':
        cupy.embedding_grad(c['grad'], c['ids'], case['rows'], case['scale'], out=r['out'])
        return o['out']
    if op == 'norm':
        cupy.rms_norm(c['x'], c['weight'], c['other'], _EPS, out=r['out'], residual_out=r['sum'])
        return o['out'], o['sum']
    if op == 'norm_int8':
        cupy.rms_norm_int8(c['x'], c['weight'], c['other'], _EPS, out=r['out'],
                           scale_out=r['scale'], residual_out=r['sum'])
        cupy.multiply(r['out'], r['column'], r['values'], casting='same_kind')
        return o['values'], o['scale'], o['sum']
    if op == 'norm_grad':
        cupy.rms_norm_grad(c['grad'], c['x'], c['weight'], _EPS, residual_grad=c['other'],
                           out=r['sum'], weight_out=r['weight'])
        return o['sum'], o['weight']
    if op == 'log_prob':
        cupy.token_log_prob(c['logits'], c['tokens'], entropy=case['entropy'], top=case['top'], out=r)
        return o
    if op == 'log_prob_grad':
        cupy.token_log_prob_grad(c['grad'], c['logits'], c['tokens'], c['lse'],
                                 entropy=c.get('entropy'), entropy_grad=c.get('entropy_grad'),
                                 out=r['out'])
        return o['out']
    cupy.clip_by_global_norm(c['arrays'], s['max_norm'], out=c['views'], norm_out=r['norm'])
    return o['flat'], o['norm']


def _plain(s):
    case = s['case']
    op = case['op']
    if op == 'embed':
        t, ids = s['table'], s['ids']
        met = (ids >= 0) & (ids < t.shape[0])
        rows = t[ids.clamp(0, t.shape[0] - 1)].float() * case['scale']
        return torch.where(met[:, None], rows, 0.0).to(t.dtype)
    if op == 'embed_grad':
        ids = s['ids']
        met = (ids >= 0) & (ids < case['rows'])
        acc = torch.zeros((case['rows'], case['width']), device='cuda')
        rows = torch.where(met[:, None], s['grad'].float(), 0.0)
        acc.index_add_(0, ids.clamp(0, case['rows'] - 1), rows)
        return (acc * case['scale']).to(_F[case['out']])
    if op in ('norm', 'norm_int8'):
        kind = s['x'].dtype
        h = s['x'].float() + s['other'].float()
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * s['weight'].float()
        if op == 'norm':
            return y.to(kind), h.to(kind)
        scale = y.abs().amax(-1, keepdim=True) / 127
        q = torch.where(scale > 0, y / scale, 0.0).round().clamp(-127, 127).to(torch.int8)
        return (q.float() * scale).half(), scale[:, 0], h.to(kind)
    if op == 'norm_grad':
        kind = s['x'].dtype
        x, g = s['x'].float(), s['grad'].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        n = x * r
        a = g * s['weight'].float()
        dx = r * (a - n * (a * n).mean(-1, keepdim=True)) + s['other'].float()
        return dx.to(kind), (g * n).sum(0).to(kind)
    if op == 'log_prob':
        x, tokens = s['logits'].float(), s['tokens']
        m = x.amax(-1, keepdim=True)
        lse = m + torch.exp(x - m).sum(-1, keepdim=True).log()
        met = (tokens >= 0) & (tokens < x.shape[1])
        at = x.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None]) - lse
        out = {'log_prob': torch.where(met, at[:, 0], 0.0), 'lse': lse[:, 0]}
        if case['entropy']:
            log_p = x - lse
            out['entropy'] = -torch.where(log_p > -math.inf, log_p.exp() * log_p, 0.0).sum(-1)
        if case['top']:
            best, index = torch.sort(x, dim=-1, descending=True, stable=True)
            out['top'] = best[:, :case['top']] - lse
            out['index'] = index[:, :case['top']].contiguous()
        return out
    if op == 'log_prob_grad':
        x, tokens, g = s['logits'].float(), s['tokens'], s['grad']
        log_p = x - s['lse'][:, None]
        p = torch.exp(log_p)
        met = (tokens >= 0) & (tokens < x.shape[1])
        g = torch.where(met, g, 0.0)[:, None]
        d = -g * p
        d.scatter_add_(1, tokens.clamp(0, x.shape[1] - 1)[:, None], g)
        if case['entropy']:
            d = d - torch.where(p > 0, s['entropy_grad'][:, None] * p
                                * (log_p + s['entropy'][:, None]), 0.0)
        return d.to(s['logits'].dtype)
    total = torch.stack([a.double().square().sum() for a in s['arrays']]).sum().sqrt()
    coef = (s['max_norm'] / (total + 1e-6)).clamp(max=1.0).float()
    flat = torch.cat([(a.float() * coef).to(a.dtype).reshape(-1) for a in s['arrays']])
    return flat, total.float()


# -- the definition in 64 bits ----------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'embed':
        return s['table'].double()[s['ids']] * case['scale']
    if op == 'embed_grad':
        order = torch.argsort(s['ids'], stable=True)
        order = order[s['ids'][order] >= 0]
        out = torch.zeros((case['rows'], case['width']), device='cuda', dtype=torch.float64)
        return out.index_add_(0, s['ids'][order], s['grad'].double()[order] * case['scale'])
    if op in ('norm', 'norm_int8'):
        h = s['x'].double() + s['other'].double()
        y = s['weight'].double() * h / torch.sqrt(h.pow(2).sum(-1, keepdim=True) / case['width'] + _EPS)
        if op == 'norm':
            return y, h
        top = torch.maximum(y.amax(-1), -y.amin(-1))
        step = top / 127.0
        return torch.round(y / step[:, None]) * step[:, None], step, h
    if op == 'norm_grad':
        x = s['x'].double().requires_grad_()
        w = s['weight'].double().requires_grad_()
        y = w * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case['width'] + _EPS)
        dx, dw = torch.autograd.grad(y, (x, w), s['grad'].double())
        return dx + s['other'].double(), dw
    if op == 'log_prob':
        x = s['logits'].double()
        log_p = torch.log_softmax(x, -1)
        rows = torch.arange(case['tokens'], device='cuda')
        out = {'log_prob': log_p[rows, s['tokens']], 'lse': torch.logsumexp(x, -1)}
        if case['entropy']:
            out['entropy'] = torch.special.entr(torch.exp(log_p)).sum(-1)
        if case['top']:
            out['top'] = torch.topk(log_p, case['top'], dim=-1)[0]
            out['index'] = None
        return out
    if op == 'log_prob_grad':
        # from the given statistics, as the operator is defined on them
        x = s['logits'].double()
        p = torch.exp(x - s['lse'].double()[:, None])
        valid = s['tokens'] >= 0
        g = s['grad'].double() * valid
        d = p * -g[:, None]
        rows = torch.nonzero(valid)[:, 0]
        d[rows, s['tokens'][rows]] += g[rows]
        if case['entropy']:
            d -= s['entropy_grad'].double()[:, None] * p * (
                x - s['lse'].double()[:, None] + s['entropy'].double()[:, None])
        return d
    flat = torch.cat([a.reshape(-1) for a in s['arrays']]).double()
    norm = torch.linalg.vector_norm(flat)
    return flat * min(1.0, s['max_norm'] / (float(norm) + 1e-6)), norm


# -- what a pass cannot do without ------------------------------------------------------

def work(case):
    op, b = case['op'], _SIZE[case['type']]
    if op == 'embed':
        n = case['tokens'] * case['width']
        met = min(case['tokens'], case['rows'])
        return {'bytes': met * case['width'] * b + n * b + 8 * case['tokens'], 'flops': n}
    if op == 'embed_grad':
        n = case['tokens'] * case['width']
        return {'bytes': n * b + case['rows'] * case['width'] * _SIZE[case['out']]
                + 8 * case['tokens'], 'flops': 2 * n}
    if op in ('norm', 'norm_int8', 'norm_grad'):
        n, d = case['tokens'] * case['width'], case['width'] * b
        if op == 'norm':
            return {'bytes': 4 * n * b + d, 'flops': 5 * n}
        if op == 'norm_int8':
            # the sum and its norm, the values that the 8 bits stand for
            return {'bytes': 3 * n * b + n + 4 * case['tokens'] + d + n + 2 * n, 'flops': 8 * n}
        return {'bytes': 4 * n * b + 2 * d, 'flops': 12 * n}
    if op == 'log_prob':
        n = case['tokens'] * case['vocab']
        out = 4 * (2 + case['entropy']) + 12 * case['top'] + 8
        return {'bytes': n * b + case['tokens'] * out, 'flops': (6 if case['entropy'] else 4) * n}
    if op == 'log_prob_grad':
        n = case['tokens'] * case['vocab']
        return {'bytes': 2 * n * b + case['tokens'] * (24 if case['entropy'] else 16),
                'flops': (7 if case['entropy'] else 4) * n}
    n = sum(math.prod(t) for t in _shapes(case))
    return {'bytes': 2 * n * b + 4, 'flops': 3 * n}
