"""The token-side operators of training and search, as a user calls them, over the sizes they meet.

* the embedding lookup with scaling and ReLU, and its gradient by sorted tokens (`ops.embedding`);
* the global gradient norm over many tensors, and clipping into a flat buffer (`optim.clip_grads`);
* beam search's selection over beams and vocabulary (`ops.beam_select`) with the reordering of the beams' states
  (`ops.reorder_rows`).

`listed()` / `draw()` give the cases, `prepare()` a case's inputs on the GPU, `run()` one pass, `work()` the bytes and operations
one pass cannot do without and `exact()` its outputs in 64 bits.  With `own` false `run` computes the plain form from
elementary torch operations; with `own` true it calls the framework.
"""
import math
import random

import numpy as np
import torch

own = False          # True: run() calls the framework's operators; False: the plain forms

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BYTES = {'float32': 4, 'bfloat16': 2, 'float16': 2}
ZIPF = 1.0           # word frequencies fall like 1 / rank
GRAD_STD = {'float32': 1e-2, 'bfloat16': 1.0, 'float16': 1.0}      # (16-bit gradients carry a loss scale of 1024)


# ----------------------------------------------------------------------------------------------------------------- cases
def _embed(name, n, vocab, width, dtype, train, relu, scale, pad):
    return dict(name=name, op='embed', n=n, vocab=vocab, width=width, dtype=dtype, train=train, relu=relu, scale=scale, pad=pad)


def _clip(name, tensors, total, dtype, part):
    return dict(name=name, op='clip', tensors=tensors, total=total, dtype=dtype, part=part)


def _beam(name, batch, beams, vocab, dtype, states, outer, width, state_dtype, done, banned):
    return dict(name=name, op='beam', batch=batch, beams=beams, vocab=vocab, dtype=dtype, states=states, outer=outer,
                width=width, state_dtype=state_dtype, done=done, banned=banned)


def listed():
    return [
        # one decode step of beam search: the next word of each of five beams
        _embed('embed_beam_rows', 5, 5000, 512, 'float32', False, True, 1.0, 0.0),
        # teacher-forced captions, 64 segments of 20 words, almost half of them padding (word 0)
        _embed('embed_train_captions', 64 * 20, 5000, 512, 'float32', True, True, 1.0, 0.45),
        # a small table of odd width: few rows that many words share
        _embed('embed_train_classes', 2049, 432, 301, 'float16', True, False, math.sqrt(301), 0.1),
        # long texts over a sub-word vocabulary of odd size, scaled by the root of the width
        _embed('embed_train_long', 32768, 50257, 1024, 'bfloat16', True, False, 32.0, 0.0),
        # the largest: a big batch of long texts over a big vocabulary
        _embed('embed_train_large', 131072, 131072, 2048, 'bfloat16', True, False, 1.0, 0.02),
        # the gradients of a captioning model: some 80 tensors, a few of them large
        _clip('clip_captioner', 81, 40000000, 'float32', 0.5),
        # many small tensors of odd sizes in two types
        _clip('clip_many_mixed', 400, 3000001, 'mixed', 0.5),
        # a large model's 16-bit gradients, unscaled into the 32-bit master gradients; the norm stays under the limit
        _clip('clip_large', 200, 500000000, 'bfloat16', 2.0),
        # one segment, five beams, four recurrent states
        _beam('beam_one', 1, 5, 5000, 'float32', 1, 4, 1024, 'float32', 0.0, 0.0),
        # a batch of segments, some beams ended
        _beam('beam_captions', 64, 5, 5000, 'float32', 1, 4, 1024, 'float32', 0.2, 0.0),
        # wide beams over a vocabulary of odd size with banned words, 16-bit logits, histories of 8-byte entries besides
        _beam('beam_wide_odd', 15, 12, 32003, 'float16', 2, 20, 1, 'int64', 0.1, 0.05),
        # a big vocabulary, and states that hold a long cache for each beam
        _beam('beam_large', 32, 8, 131072, 'bfloat16', 2, 1, 512 * 1024, 'bfloat16', 0.1, 0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['embed', 'clip', 'beam'])
    dtype = rng.choice(['float32', 'bfloat16', 'float16'])
    if op == 'embed':
        n, vocab, width = _log_int(rng, 1, 131072), _log_int(rng, 100, 131072), _log_int(rng, 32, 2048)
        if rng.random() < 0.6:
            width = max(32, width // 32 * 32)
        c = _embed('', n, vocab, width, dtype, rng.random() < 0.75, rng.random() < 0.5,
                   rng.choice([1.0, 0.5, math.sqrt(width)]), rng.choice([0.0, 0.1, 0.5]))
    elif op == 'clip':
        tensors = _log_int(rng, 1, 400)
        c = _clip('', tensors, max(tensors, _log_int(rng, 1000, 250000000)), rng.choice(['float32', 'bfloat16', 'float16', 'mixed']),
                  rng.choice([0.01, 0.5, 2.0]))
    else:
        beams = rng.randint(1, 16)
        vocab = _log_int(rng, 200, 131072)
        batch = min(_log_int(rng, 1, 256), max(1, 32 * 8 * 65536 // (beams * vocab)))
        sd = rng.choice(['float32', 'bfloat16', 'int64'])
        rows = batch * beams
        width = 1 if sd == 'int64' else min(_log_int(rng, 64, 262144), max(64, 32000000 // rows))
        c = _beam('', batch, beams, vocab, dtype, rng.randint(1, 4), rng.randint(1, 8) if width < 4096 else 1, width, sd,
                  rng.choice([0.0, 0.3]), rng.choice([0.0, 0.05]))
    del c['name']
    return c


def _sizes(case):
    """The tensors' sizes: their logarithms spread over some five factors of e, odd ones among them; the last one takes the rest."""
    k, total = case['tensors'], case['total']
    rng = random.Random(k * 1000003 + total)
    w = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(k)]
    s = sum(w)
    sizes = [max(1, int((total - k) * x / s)) for x in w[:-1]]
    return sizes + [total - sum(sizes)]


def _grad_types(case):
    d = case['dtype']
    return [('bfloat16', 'float32')[i % 2] if d == 'mixed' else d for i in range(case['tensors'])]


def _word_odds(case):
    """Odds of each word: `pad` of all is word 0, the rest falls like 1 / rank."""
    p = 1.0 / np.arange(1, case['vocab'] + 1, dtype=np.float64) ** ZIPF
    p *= (1.0 - case['pad']) / p.sum()
    p[0] += case['pad']
    return p


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(int(seed))
    dev = 'cuda'
    if case['op'] == 'embed':
        t = DTYPES[case['dtype']]
        edges = torch.from_numpy(np.cumsum(_word_odds(case))).to(dev)
        words = torch.searchsorted(edges, torch.rand(case['n'], generator=g, device=dev, dtype=torch.float64))
        words = words.clamp_(max=case['vocab'] - 1)
        table = torch.randn(case['vocab'], case['width'], generator=g, device=dev, dtype=t)
        s = dict(op='embed', words=words, table=table.requires_grad_(case['train']), scale=case['scale'], relu=case['relu'])
        if case['train']:
            s['dy'] = torch.randn(case['n'], case['width'], generator=g, device=dev, dtype=t).mul_(1e-2)
        return s
    if case['op'] == 'clip':
        sizes, types = _sizes(case), _grad_types(case)
        scaled = case['dtype'] in ('bfloat16', 'float16')          # gradients of a scaled loss
        grads = [torch.randn(n, generator=g, device=dev, dtype=DTYPES[t]).mul_(GRAD_STD[t] if scaled else 1e-2)
                 for n, t in zip(sizes, types)]
        inv = 1.0 / 1024.0 if scaled else 1.0
        std = GRAD_STD[case['dtype']] if scaled else 1e-2
        flat = torch.zeros(sum(sizes), device=dev)
        return dict(op='clip', grads=grads, flat=flat, out=list(torch.split(flat, sizes)), inv_scale=inv,
                    max_norm=case['part'] * std * inv * math.sqrt(case['total']))
    B, K, V = case['batch'], case['beams'], case['vocab']
    logits = torch.randn(B * K, V, generator=g, device=dev, dtype=torch.float32).mul_(3.0)
    if case['banned']:
        logits.masked_fill_(torch.rand(V, generator=g, device=dev) < case['banned'], float('-inf'))
    logits = logits.to(DTYPES[case['dtype']])
    scores = torch.randn(B, K, generator=g, device=dev).mul_(2.0).sub_(20.0)
    done = (torch.rand(B, K, generator=g, device=dev) < case['done']).to(torch.uint8)
    shape = (case['outer'], B * K, case['width'])
    if case['state_dtype'] == 'int64':
        states = [torch.randint(0, V, shape, generator=g, device=dev) for _ in range(case['states'])]
    else:
        states = [torch.randn(shape, generator=g, device=dev, dtype=DTYPES[case['state_dtype']]) for _ in range(case['states'])]
    return dict(op='beam', logits=logits, scores=scores, done=done, states=states)


# ------------------------------------------------------------------------------------------------------------ plain forms
def _embed_plain(s):
    table, words = s['table'].detach(), s['words']
    rows = table[words].float() * s['scale']
    out = (rows.clamp(min=0) if s['relu'] else rows).to(table.dtype)
    if 'dy' not in s:
        return {'out': out}
    up = s['dy'].float()
    if s['relu']:
        up = up * (rows > 0)
    grad = torch.zeros(table.shape, device=table.device).index_add_(0, words, up) * s['scale']
    return {'out': out, 'grad': grad.to(table.dtype)}


def _clip_plain(s):
    total = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s['grads']]).sum()
    norm = total.sqrt() * s['inv_scale']
    factor = ((s['max_norm'] / (norm + 1e-6)).clamp(max=1.0) * s['inv_scale']).float()
    return {'norm': norm.float(), 'flat': torch.cat([g.float() * factor for g in s['grads']])}


def _beam_plain(s):
    # 64 bits: two candidates of different beams may lie closer than 32 bits tell apart
    x, scores, done = s['logits'].double(), s['scores'].double(), s['done']
    B, K = scores.shape
    V = x.shape[1]
    x = x.view(B, K, V)
    top = x.max(2, keepdim=True)[0]
    lse = top + (x - top).exp().sum(2, keepdim=True).log()
    cand = scores.unsqueeze(2) + (x - lse)
    live = torch.isfinite(scores) & torch.isfinite(lse.squeeze(2))
    over = done.bool().unsqueeze(2)
    ended = torch.full_like(cand, float('-inf'))
    ended[:, :, 0] = scores
    cand = torch.where(over, ended, torch.where(live.unsqueeze(2), cand, torch.full_like(cand, float('-inf'))))
    best, at = cand.view(B, K * V).sort(dim=1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    beam, word = at // V, at % V
    parent = beam + torch.arange(B, device=x.device).unsqueeze(1) * K
    fin = done.gather(1, beam).bool() | (word == 0)
    return {'scores': best.float(), 'parent': parent, 'word': word, 'done': fin.to(torch.uint8),
            'states': [t[:, parent.view(-1)] for t in s['states']]}


# ------------------------------------------------------------------------------------------------- the framework's calls
def _embed_own(s):
    from gvd_amd import ops
    out = ops.embedding(s['words'], s['table'], scale=s['scale'], act=1 if s['relu'] else 0)
    if 'dy' not in s:
        return {'out': out}
    grad, = torch.autograd.grad(out, s['table'], s['dy'])
    return {'out': out.detach(), 'grad': grad}


def _clip_own(s):
    from gvd_amd import optim
    norm = optim.clip_grads(s['grads'], s['max_norm'], out=s['out'], inv_scale=s['inv_scale'])
    return {'norm': norm, 'flat': s['flat']}


def _beam_own(s):
    from gvd_amd import ops
    scores, parent, word, done = ops.beam_select(s['logits'], s['scores'], finished=s['done'], eos=0)
    return {'scores': scores, 'parent': parent, 'word': word, 'done': done,
            'states': ops.reorder_rows(s['states'], parent, dim=1)}


def run(state):
    if own:
        return {'embed': _embed_own, 'clip': _clip_own, 'beam': _beam_own}[state['op']](state)
    return {'embed': _embed_plain, 'clip': _clip_plain, 'beam': _beam_plain}[state['op']](state)


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    if case['op'] == 'embed':
        b, n, v, e = BYTES[case['dtype']], case['n'], case['vocab'], case['width']
        used = float((1.0 - (1.0 - _word_odds(case)) ** n).sum())          # rows of the table that are looked at
        moved = n * 8 + used * e * b + n * e * b
        flops = n * e * 2.0
        if case['train']:
            moved += n * 8 + n * e * b + v * e * b
            flops += n * e * 1.0
        return {'bytes': moved, 'flops': flops}
    if case['op'] == 'clip':
        read = sum(n * BYTES[t] for n, t in zip(_sizes(case), _grad_types(case)))
        return {'bytes': read + 4.0 * case['total'], 'flops': 3.0 * case['total']}
    rows = case['batch'] * case['beams']
    live = rows * (1.0 - case['done'])                                     # an ended beam's logits need no reading
    size = 8 if case['state_dtype'] == 'int64' else BYTES[case['state_dtype']]
    state = 2.0 * case['states'] * case['outer'] * rows * case['width'] * size
    return {'bytes': live * case['vocab'] * BYTES[case['dtype']] + rows * 34.0 + state, 'flops': live * case['vocab'] * 4.0}


# ----------------------------------------------------------------------------------------------------------------- exact
def _embed_exact(s):
    table = s['table'].detach().to(torch.float64)
    scaled = torch.mul(table, s['scale'])
    if s['relu']:
        scaled = torch.where(scaled > 0, scaled, torch.zeros_like(scaled))
    out = torch.index_select(scaled, 0, s['words'])
    if 'dy' not in s:
        return {'out': out}
    total = torch.zeros_like(table)
    total.index_put_((s['words'],), s['dy'].to(torch.float64), accumulate=True)       # one sum for each word of the table,
    slope = (scaled > 0).to(torch.float64) * s['scale'] if s['relu'] else s['scale']       # whose slope is the same everywhere
    return {'out': out, 'grad': total * slope}


def _clip_exact(s):
    squares = [float(torch.dot(g.double(), g.double())) for g in s['grads']]
    norm = math.sqrt(math.fsum(squares)) * s['inv_scale']
    by = min(1.0, s['max_norm'] / (norm + 1e-6)) * s['inv_scale']
    flat = torch.empty(s['flat'].numel(), dtype=torch.float64, device='cuda')
    at = 0
    for g in s['grads']:
        flat[at:at + g.numel()] = g.double() * by
        at += g.numel()
    return {'norm': norm, 'flat': flat}


def _beam_exact(s):
    B, K = s['scores'].shape
    scores, done = s['scores'].cpu().numpy().astype(np.float64), s['done'].cpu().numpy()
    V = s['logits'].shape[1]
    res = {'scores': np.empty((B, K)), 'parent': np.empty((B, K), np.int64), 'word': np.empty((B, K), np.int64),
           'done': np.empty((B, K), np.uint8)}
    for b in range(B):
        x = s['logits'][b * K:(b + 1) * K].cpu().to(torch.float64).numpy()
        cand = np.full((K, V), -np.inf)
        for q in range(K):
            if done[b, q]:
                cand[q, 0] = scores[b, q]
            else:
                m = x[q].max()
                cand[q] = scores[b, q] + (x[q] - (m + math.log(np.exp(x[q] - m).sum())))
        at = np.argsort(-cand.reshape(-1), kind='stable')[:K]
        res['scores'][b] = cand.reshape(-1)[at]
        res['parent'][b], res['word'][b] = at // V + b * K, at % V
        res['done'][b] = (done[b, at // V] != 0) | (at % V == 0)
    rows = torch.from_numpy(res['parent'].reshape(-1)).to('cuda')
    res['states'] = [torch.index_select(t, 1, rows).double() if t.is_floating_point() else None for t in s['states']]
    return res


def exact(case, seed):
    s = prepare(case, seed)
    return {'embed': _embed_exact, 'clip': _clip_exact, 'beam': _beam_exact}[case['op']](s)
