"""Cases of the language-model operators: rotary positions, sliding-window attention with sinks (whole sequences and single
tokens over a rolling key/value cache), and the log probabilities of given tokens.

``run`` computes a case either in a plain form (elementary tensor operations in 32 bits, 64 where far positions need them) or,
where ``own`` is true, through the framework's operators.  ``exact`` is the definition in 64 bits."""
import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # queries and keys of one layer of a training step, rotated together; forward and gradient
        dict(name='rotary_train', op='rotary', batch=8, length=2048, heads=20, dim=128, rotated=128, interleaved=False,
             dtype='bfloat16', reach=0, train=True),
        # one new token for each of 48 sequences at far positions, a quarter of each head rotated, pairs interleaved
        dict(name='rotary_token', op='rotary', batch=48, length=1, heads=12, dim=64, rotated=16, interleaved=True,
             dtype='float16', reach=1000000, train=False),
        # a training step of a layer with grouped heads, local attention and four sinks; forward and gradients
        dict(name='attention_train_window', op='attention', batch=2, length=4096, heads=16, kv_heads=4, dim=128, window=1024,
             sinks=4, dtype='bfloat16', ragged=False, train=True),
        # a training step of a small model over padded sequences, every earlier token visible
        dict(name='attention_train_causal', op='attention', batch=16, length=512, heads=12, kv_heads=12, dim=64, window=0,
             sinks=0, dtype='float16', ragged=True, train=True),
        # one long prompt
        dict(name='attention_prompt', op='attention', batch=1, length=8192, heads=32, kv_heads=8, dim=128, window=2048, sinks=4,
             dtype='bfloat16', ragged=False, train=False),
        # a short prompt, where latency counts
        dict(name='attention_short', op='attention', batch=1, length=77, heads=12, kv_heads=12, dim=64, window=32, sinks=1,
             dtype='float16', ragged=False, train=False),
        # the keys and values of a batch of prompts that are longer than the rolling cache
        dict(name='fill_prompts', op='fill', batch=16, length=6000, kv_heads=8, dim=128, capacity=4096, sinks=4,
             dtype='bfloat16', ragged=True),
        # one short prompt into an empty cache
        dict(name='fill_short', op='fill', batch=1, length=77, kv_heads=12, dim=64, capacity=512, sinks=1, dtype='float16',
             ragged=False),
        # a busy server: a token for each of 64 sequences, caches that have rolled over
        dict(name='step_batch', op='step', batch=64, heads=32, kv_heads=8, dim=128, capacity=4100, window=4096, sinks=4,
             dtype='bfloat16', reach=12000, idle=False),
        # a single conversation
        dict(name='step_single', op='step', batch=1, heads=12, kv_heads=12, dim=64, capacity=1000, window=500, sinks=3,
             dtype='float16', reach=1500, idle=False),
        # scores of the tokens of a training batch, with the gradient through log probability and entropy
        dict(name='logprobs_train', op='logprobs', rows=4096, vocab=33278, topk=0, dtype='bfloat16', masked=False, train=True),
        # the tokens that 24 sequences have drawn, with 20 alternatives each, part of the vocabulary ruled out
        dict(name='logprobs_top', op='logprobs', rows=24, vocab=131072, topk=20, dtype='float32', masked=True, train=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(['rotary', 'attention', 'attention', 'fill', 'step', 'logprobs', 'logprobs'])
    half = rng.choice(['float16', 'bfloat16'])
    if op == 'rotary':
        dim = rng.choice([64, 80, 96, 128])
        length = _log_int(rng, 1, 4096)
        batch = _log_int(rng, 1, max(1, min(64, 16384 // length)))
        return dict(op=op, batch=batch, length=length, heads=rng.randint(1, 20), dim=dim,
                    rotated=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                    dtype=rng.choice(['float32', 'float16', 'bfloat16']), reach=rng.choice([0, 4096, 1000000]),
                    train=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 128])
    if op == 'attention':
        train = rng.random() < 0.5
        length = _log_int(rng, 1, 4096)
        most = 2 * 16 * 4096 * 4096 // (length * length * heads)
        if most < 1:
            length, most = 1 + rng.randrange(1500), 4
        case = dict(op=op, batch=_log_int(rng, 1, max(1, min(24, most))), length=length, heads=heads, kv_heads=kv_heads, dim=dim,
                    window=rng.choice([0, _log_int(rng, 1, length)]), sinks=rng.choice([0, 1, 4, rng.randint(0, 150)]),
                    dtype=half, ragged=rng.random() < 0.5, train=train)
        case['batch'] = max(1, min(case['batch'], int(case['batch'] * 2e11 / work(case)['flops']) if work(case)['flops'] else 24))
        return case
    if op in ('fill', 'step'):
        sinks = rng.choice([0, 1, 4, 33])
        capacity = sinks + _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(128, 400000 // (capacity * kv_heads))))
        if op == 'fill':
            return dict(op=op, batch=batch, length=_log_int(rng, 1, 8192), kv_heads=kv_heads, dim=dim, capacity=capacity,
                        sinks=sinks, dtype=half, ragged=rng.random() < 0.5)
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, capacity=capacity,
                    window=rng.choice([0, _log_int(rng, 1, capacity)]), sinks=sinks, dtype=half,
                    reach=_log_int(rng, 1, 4 * capacity), idle=rng.random() < 0.3)
    vocab = _log_int(rng, 2, 160000)
    rows = _log_int(rng, 1, max(1, min(4096, 130000000 // vocab)))
    return dict(op=op, rows=rows, vocab=vocab, topk=rng.choice([0, 1, 5, rng.randint(1, min(32, vocab))]) if vocab >= 5 else 1,
                dtype=rng.choice(['float32', 'float16', 'bfloat16']), masked=rng.random() < 0.3, train=rng.random() < 0.5)


# --------------------------------------------------------------------------------------------------------------- inputs
def _spread(n, low, high, gen):
    """``n`` whole numbers, evenly spread over [low, high], in an order that the seed decides."""
    at = [low + int((high - low) * (i + 0.5) / n + 0.5) for i in range(n)]
    return torch.tensor(at, dtype=torch.int64)[torch.randperm(n, generator=gen)]


def _evenly(n, low, high):
    return [low + int((high - low) * (i + 0.5) / n + 0.5) for i in range(n)]


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype = DTYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)
    s = dict(case=case)
    if case['op'] == 'rotary':
        b, t, h, d = case['batch'], case['length'], case['heads'], case['dim']
        s['data'] = normal(b, t, h, d)
        if case['reach']:
            s['positions'] = torch.randint(0, case['reach'], (b, t), generator=gen, device=dev)
        else:
            s['positions'] = torch.arange(t, device=dev)
        s['inv_freq'] = (10000.0 ** (-torch.arange(0, case['rotated'], 2, dtype=torch.float64) / case['rotated'])).float().to(dev)
        if case['train']:
            s['out_grad'] = normal(b, t, h, d)
    elif case['op'] == 'attention':
        b, t, h, g, d = case['batch'], case['length'], case['heads'], case['kv_heads'], case['dim']
        s['query'], s['key'], s['value'] = normal(b, t, h, d), normal(b, t, g, d), normal(b, t, g, d)
        s['valid_length'] = _spread(b, 0, t, host).to(torch.int32).to(dev) if case['ragged'] else None
        if case['train']:
            s['out_grad'] = normal(b, t, h, d)
    elif case['op'] == 'fill':
        b, t, g, d, c = case['batch'], case['length'], case['kv_heads'], case['dim'], case['capacity']
        s['key'], s['value'] = normal(b, t, g, d), normal(b, t, g, d)
        s['key_cache'], s['value_cache'] = normal(b, c, g, d), normal(b, c, g, d)
        s['valid_length'] = _spread(b, 0, t, host).to(torch.int32).to(dev) if case['ragged'] else None
    elif case['op'] == 'step':
        b, h, g, d, c = case['batch'], case['heads'], case['kv_heads'], case['dim'], case['capacity']
        s['query'], s['key'], s['value'] = normal(b, h, d), normal(b, g, d), normal(b, g, d)
        s['key_cache'], s['value_cache'] = normal(b, c, g, d), normal(b, c, g, d)
        s['positions'] = _spread(b, -1 if case['idle'] else 0, case['reach'] - 1, host)
        if case['idle']:
            s['positions'][torch.randint(0, b, (1,), generator=host)] = -1       # a place of the batch without a sequence
        s['positions'] = s['positions'].to(dev)
    else:
        n, v = case['rows'], case['vocab']
        x = torch.randn(n, v, generator=gen, device=dev, dtype=torch.float32) * 3
        if case['masked']:
            x.masked_fill_(torch.rand(v, generator=gen, device=dev) < 0.3, -math.inf)
        s['logits'] = x.to(dtype)
        s['tokens'] = torch.randint(0, v, (n,), generator=gen, device=dev)
        if case['masked']:                                                       # a drawn token is one that was allowed
            s['tokens'] = torch.argmax(x + torch.randn(n, v, generator=gen, device=dev), dim=1)
        if case['train']:
            s['tokens'][torch.rand(n, generator=gen, device=dev) < 0.1] = -1      # padding
            s['log_prob_grad'] = torch.randn(n, generator=gen, device=dev)
            s['entropy_grad'] = torch.randn(n, generator=gen, device=dev) * 0.1
            if case['topk']:
                s['top_grad'] = torch.randn(n, case['topk'], generator=gen, device=dev) * 0.1
    return s


# ----------------------------------------------------------------------------------------------------- plain forms
def _pairs(x, rotated, interleaved):
    r = x[..., :rotated]
    return (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotated // 2], r[..., rotated // 2:])


def _joined(a, b, rest, interleaved):
    turned = torch.stack((a, b), dim=-1).flatten(-2) if interleaved else torch.cat((a, b), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _turn(x, cos, sin, rotated, interleaved):
    a, b = _pairs(x, rotated, interleaved)
    return _joined(a * cos - b * sin, b * cos + a * sin, x[..., rotated:], interleaved)


def _plain_rotary(s):
    c = s['case']
    angle = s['positions'].double()[..., None] * s['inv_freq'].double()
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    out = _turn(s['data'].float(), cos, sin, c['rotated'], c['interleaved']).to(s['data'].dtype)
    if not c['train']:
        return {'out': out}
    grad = _turn(s['out_grad'].float(), cos, -sin, c['rotated'], c['interleaved']).to(s['data'].dtype)
    return {'out': out, 'data_grad': grad}


def _visible(length, window, sinks, valid_length, batch, dev):
    """[batch or 1, length, length]: whether query i sees key j."""
    i, j = torch.arange(length, device=dev)[:, None], torch.arange(length, device=dev)[None, :]
    seen = j <= i
    if window:
        seen = seen & ((i - j < window) | (j < sinks))
    seen = seen[None]
    if valid_length is not None:
        seen = seen & (i[None] < valid_length.reshape(batch, 1, 1))
    return seen


def _plain_attention(s):
    c = s['case']
    b, t, h, g, d = c['batch'], c['length'], c['heads'], c['kv_heads'], c['dim']
    n = h // g
    scale = 1.0 / math.sqrt(d)
    q = s['query'].float().reshape(b, t, g, n, d).permute(0, 2, 3, 1, 4)          # [b, g, n, t, d]
    k = s['key'].float().permute(0, 2, 1, 3)[:, :, None]                          # [b, g, 1, t, d]
    v = s['value'].float().permute(0, 2, 1, 3)[:, :, None]
    seen = _visible(t, c['window'], c['sinks'], s['valid_length'], b, q.device)[:, None, None]
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p, v)

    def rows(x, heads):
        return x.reshape(b, heads, t, d).transpose(1, 2).contiguous().to(s['query'].dtype)
    if not c['train']:
        return {'out': rows(out, h)}
    go = s['out_grad'].float().reshape(b, t, g, n, d).permute(0, 2, 3, 1, 4)
    gv = torch.matmul(p.transpose(-1, -2), go).sum(2)
    gp = torch.matmul(go, v.transpose(-1, -2))
    gs = gp.sub_((go * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    gq = torch.matmul(gs, k)
    gk = torch.matmul(gs.transpose(-1, -2), q).sum(2)
    return {'out': rows(out, h), 'query_grad': rows(gq, h), 'key_grad': rows(gk, g), 'value_grad': rows(gv, g)}


def _slots(positions, sinks, capacity):
    """The cache row of each position: the sinks stay, the others roll over the rest."""
    return torch.where(positions < sinks, positions, sinks + (positions - sinks) % (capacity - sinks))


def _plain_fill(s):
    c = s['case']
    b, t, cap, sinks = c['batch'], c['length'], c['capacity'], c['sinks']
    dev = s['key'].device
    valid = s['valid_length'].long() if s['valid_length'] is not None else torch.full((b,), t, dtype=torch.int64, device=dev)
    at = torch.arange(t, device=dev)[None].expand(b, t)
    keep = (at < valid[:, None]) & ((at < sinks) | (at >= valid[:, None] - (cap - sinks)))
    rows, cols = keep.nonzero(as_tuple=True)
    slot = _slots(cols, sinks, cap)
    s['key_cache'][rows, slot] = s['key'][rows, cols]
    s['value_cache'][rows, slot] = s['value'][rows, cols]
    return {'key_cache': s['key_cache'], 'value_cache': s['value_cache']}


def _plain_step(s):
    c = s['case']
    b, h, g, d, cap, sinks = c['batch'], c['heads'], c['kv_heads'], c['dim'], c['capacity'], c['sinks']
    pos = s['positions']
    live = pos >= 0
    row = torch.arange(b, device=pos.device)
    slot = _slots(pos.clamp(min=0), sinks, cap)
    old_k, old_v = s['key_cache'][row, slot], s['value_cache'][row, slot]
    s['key_cache'][row, slot] = torch.where(live[:, None, None], s['key'], old_k)
    s['value_cache'][row, slot] = torch.where(live[:, None, None], s['value'], old_v)
    # the position that each cache row holds: the largest one up to the new token's that falls on the row
    at = torch.arange(cap, device=pos.device)[None]
    ring = cap - sinks
    held = torch.where(at < sinks, at, pos[:, None] - (pos[:, None] - at) % ring)
    seen = (held <= pos[:, None]) & ((at < sinks) | (held >= sinks))
    if c['window']:
        seen = seen & ((pos[:, None] - held < c['window']) | (at < sinks))
    q = s['query'].float().reshape(b, g, h // g, d)
    k, v = s['key_cache'].float().permute(0, 2, 1, 3), s['value_cache'].float().permute(0, 2, 1, 3)
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return {'out': out.reshape(b, h, d).to(s['query'].dtype), 'key_cache': s['key_cache'], 'value_cache': s['value_cache']}


def _plain_logprobs(s):
    c = s['case']
    x = s['logits'].float()
    top = x.amax(-1, keepdim=True)
    shifted = x - torch.where(top == -math.inf, 0.0, top)
    e = shifted.exp()
    # one of the largest counts 1 exactly: what the others add goes through log1p, so that a sure token keeps its digits
    first = torch.argmax(x, dim=-1, keepdim=True)
    others = e.scatter(-1, first, 0.0).sum(-1, keepdim=True)
    log_total = torch.log1p(others)
    logp = shifted - log_total
    p = e / (1.0 + others)
    entropy = log_total[:, 0] - torch.where(e > 0, p * shifted, 0.0).sum(-1)
    tok = s['tokens']
    known = tok >= 0
    chosen = torch.where(known, logp.gather(-1, tok.clamp(min=0)[:, None])[:, 0], 0.0)
    out = {'log_prob': chosen, 'entropy': entropy}
    if c['topk']:
        order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c['topk']]
        out['top_log_prob'], out['top_token'] = logp.gather(-1, order), order
    if not c['train']:
        return out
    gl = torch.where(known, s['log_prob_grad'], 0.0)
    ge = s['entropy_grad']
    total = gl + s['top_grad'].sum(-1) if c['topk'] else gl
    weight = torch.where(e > 0, total[:, None] + ge[:, None] * (logp + entropy[:, None]), 0.0)
    grad = -p * weight
    grad.scatter_add_(-1, tok.clamp(min=0)[:, None], gl[:, None])
    if c['topk']:
        grad.scatter_add_(-1, order, s['top_grad'])
    out['logits_grad'] = grad.to(s['logits'].dtype)
    return out


# ----------------------------------------------------------------------------------------------- the framework's calls
def _arrays(s, leaves):
    """The program's arrays: made of the state's tensors without a copy, the ones that are differentiated marked so."""
    from mxnet_b200 import nd
    if 'arrays' not in s:
        s['arrays'] = {k: nd.NDArray(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        for k in leaves:
            s['arrays'][k].attach_grad()
    return s['arrays']


def _own(s):
    from mxnet_b200 import autograd, nd
    c = s['case']
    train = c.get('train', False)
    if c['op'] == 'rotary':
        a = _arrays(s, ['data'] if train else [])
        if not train:
            out = nd.contrib.rotary_embedding(a['data'], a['positions'], a['inv_freq'], interleaved=c['interleaved'])
            return {'out': out._data}
        with autograd.record():
            out = nd.contrib.rotary_embedding(a['data'], a['positions'], a['inv_freq'], interleaved=c['interleaved'])
        grad = autograd.grad(out, a['data'], a['out_grad'])
        return {'out': out._data, 'data_grad': grad._data}
    if c['op'] == 'attention':
        names = ['query', 'key', 'value']
        a = _arrays(s, names if train else [])
        args = [a['query'], a['key'], a['value']] + ([a['valid_length']] if c['ragged'] else [])
        if not train:
            return {'out': nd.contrib.sldwin_attention(*args, window=c['window'], sinks=c['sinks'])._data}
        with autograd.record():
            out = nd.contrib.sldwin_attention(*args, window=c['window'], sinks=c['sinks'])
        grads = autograd.grad(out, [a[n] for n in names], a['out_grad'])
        return dict({'out': out._data}, **{n + '_grad': g._data for n, g in zip(names, grads)})
    if c['op'] == 'fill':
        a = _arrays(s, [])
        args = [a['key'], a['value'], a['key_cache'], a['value_cache']] + ([a['valid_length']] if c['ragged'] else [])
        nd.contrib.sldwin_cache_fill(*args, sinks=c['sinks'])
        return {'key_cache': a['key_cache']._data, 'value_cache': a['value_cache']._data}
    if c['op'] == 'step':
        a = _arrays(s, [])
        out = nd.contrib.sldwin_attention_step(a['query'], a['key'], a['value'], a['key_cache'], a['value_cache'],
                                               a['positions'], window=c['window'], sinks=c['sinks'])
        return {'out': out._data, 'key_cache': a['key_cache']._data, 'value_cache': a['value_cache']._data}
    a = _arrays(s, ['logits'] if train else [])
    names = ['log_prob', 'entropy'] + (['top_log_prob', 'top_token'] if c['topk'] else [])
    if not train:
        res = nd.contrib.token_log_probs(a['logits'], a['tokens'], topk=c['topk'])
        return {n: r._data for n, r in zip(names, res)}
    with autograd.record():
        res = nd.contrib.token_log_probs(a['logits'], a['tokens'], topk=c['topk'])
    heads = [a['log_prob_grad'], a['entropy_grad']] + ([a['top_grad']] if c['topk'] else [])
    grad = autograd.grad(res[:len(heads)], a['logits'], heads)
    return dict({n: r._data.detach() for n, r in zip(names, res)}, logits_grad=grad._data)


def run(state):
    if own:
        return _own(state)
    op = state['case']['op']
    return (_plain_rotary if op == 'rotary' else _plain_attention if op == 'attention' else _plain_fill if op == 'fill'
            else _plain_step if op == 'step' else _plain_logprobs)(state)


# ----------------------------------------------------------------------------------------------------------- the floor
def _seen_pairs(n, window, sinks):
    """Query-key pairs of one head over a sequence of n tokens."""
    if not window:
        return n * (n + 1) // 2
    i = torch.arange(n)
    local = torch.clamp(i + 1, max=window)
    return int((local + torch.clamp(torch.clamp(i + 1 - window, min=0), max=sinks)).sum())


def work(case):
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'rotary':
        n = case['batch'] * case['length'] * case['heads'] * case['dim']
        turned = case['batch'] * case['length'] * case['heads'] * case['rotated']
        times = 2 if case['train'] else 1
        return {'bytes': times * 2 * n * size, 'flops': times * 3 * turned}
    if case['op'] == 'attention':
        b, t, h, g, d = (case[k] for k in ('batch', 'length', 'heads', 'kv_heads', 'dim'))
        lengths = _evenly(b, 0, t) if case['ragged'] else [t] * b
        pairs = sum(_seen_pairs(n, case['window'], case['sinks']) for n in lengths) * h
        rows, used = b * t, sum(lengths)
        moved = (used * (h + 2 * g) + rows * h) * d * size
        if case['train']:
            moved += (used * h + rows * (h + 2 * g)) * d * size
        return {'bytes': moved, 'flops': pairs * d * (12 if case['train'] else 4)}
    if case['op'] == 'fill':
        lengths = _evenly(case['batch'], 0, case['length']) if case['ragged'] else [case['length']] * case['batch']
        kept = sum(min(n, case['capacity']) for n in lengths)
        return {'bytes': 4 * kept * case['kv_heads'] * case['dim'] * size, 'flops': 0}
    if case['op'] == 'step':
        b, h, g, d = (case[k] for k in ('batch', 'heads', 'kv_heads', 'dim'))
        ring = case['capacity'] - case['sinks']
        window = min(case['window'] or ring, ring)
        seen = 0
        for p in _evenly(b, -1 if case['idle'] else 0, case['reach'] - 1):
            seen += min(p + 1, case['sinks']) + max(0, min(p + 1 - case['sinks'], window))
        return {'bytes': (seen * 2 * g + 2 * b * h + 4 * b * g) * d * size, 'flops': 4 * seen * h * d}
    n = case['rows'] * case['vocab']
    return {'bytes': n * size * (2 if case['train'] else 1) + case['rows'] * (16 + 12 * case['topk']),
            'flops': n * (8 if case['train'] else 4)}


# ------------------------------------------------------------------------------------------------ the definition, 64 bits
def _exact_rotary(s):
    c = s['case']
    half = c['rotated'] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=s['data'].device),
                       s['positions'].double().unsqueeze(-1) * s['inv_freq'].double()).unsqueeze(-2)

    def rotate(x, by):
        y = x.double().clone()
        ia = torch.arange(half, device=x.device) * 2 if c['interleaved'] else torch.arange(half, device=x.device)
        ib = ia + (1 if c['interleaved'] else half)
        z = torch.complex(y[..., ia], y[..., ib]) * by
        y[..., ia], y[..., ib] = z.real, z.imag
        return y
    out = {'out': rotate(s['data'], turn)}
    if c['train']:
        out['data_grad'] = rotate(s['out_grad'], turn.conj())
    return out


def _exact_attention(s):
    c = s['case']
    b, t, h, g, d = c['batch'], c['length'], c['heads'], c['kv_heads'], c['dim']
    dev = s['query'].device
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=dev)
    gq, gk, gv = torch.zeros_like(out), torch.zeros(b, t, g, d, dtype=torch.float64, device=dev), torch.zeros(
        b, t, g, d, dtype=torch.float64, device=dev)
    lengths = s['valid_length'].tolist() if s['valid_length'] is not None else [t] * b
    for n in range(b):
        m = int(lengths[n])
        if m == 0:
            continue
        gap = torch.arange(m, device=dev)[:, None] - torch.arange(m, device=dev)[None, :]
        hide = gap < 0
        if c['window']:
            hide |= (gap >= c['window']) & (torch.arange(m, device=dev) >= c['sinks'])[None, :]
        for i in range(h):
            q, k, v = s['query'][n, :m, i].double(), s['key'][n, :m, i * g // h].double(), s['value'][n, :m, i * g // h].double()
            a = (q @ k.T / math.sqrt(d)).masked_fill(hide, -math.inf).softmax(-1)
            out[n, :m, i] = a @ v
            if c['train']:
                go = s['out_grad'][n, :m, i].double()
                gv[n, :m, i * g // h] += a.T @ go
                w = go @ v.T
                w = a * (w - (a * w).sum(-1, keepdim=True)) / math.sqrt(d)
                gq[n, :m, i] = w @ k
                gk[n, :m, i * g // h] += w.T @ q
    if not c['train']:
        return {'out': out}
    return {'out': out, 'query_grad': gq, 'key_grad': gk, 'value_grad': gv}


def _place(p, sinks, capacity):
    return p if p < sinks else sinks + (p - sinks) % (capacity - sinks)


def _exact_fill(s):
    c = s['case']
    lengths = s['valid_length'].tolist() if s['valid_length'] is not None else [c['length']] * c['batch']
    kc, vc = s['key_cache'].double(), s['value_cache'].double()
    for n, m in enumerate(lengths):
        at = [p for p in range(int(m)) if p < c['sinks'] or p >= m - (c['capacity'] - c['sinks'])]
        if at:
            to = [_place(p, c['sinks'], c['capacity']) for p in at]
            kc[n, to], vc[n, to] = s['key'][n, at].double(), s['value'][n, at].double()
    return {'key_cache': kc, 'value_cache': vc}


def _exact_step(s):
    c = s['case']
    h, g, d, cap, sinks = c['heads'], c['kv_heads'], c['dim'], c['capacity'], c['sinks']
    kc, vc = s['key_cache'].double(), s['value_cache'].double()
    out = torch.zeros(c['batch'], h, d, dtype=torch.float64, device=kc.device)
    for n, p in enumerate(s['positions'].tolist()):
        if p < 0:
            continue
        kc[n, _place(p, sinks, cap)], vc[n, _place(p, sinks, cap)] = s['key'][n].double(), s['value'][n].double()
        reach = min(c['window'] or p + 1, cap - sinks)
        at = [_place(j, sinks, cap) for j in list(range(min(sinks, p + 1))) + list(range(max(sinks, p - reach + 1), p + 1))]
        k, v = kc[n, at].repeat_interleave(h // g, 1), vc[n, at].repeat_interleave(h // g, 1)       # [keys, h, d]
        a = torch.einsum('hd,khd->hk', s['query'][n].double(), k).div(math.sqrt(d)).softmax(-1)
        out[n] = torch.einsum('hk,khd->hd', a, v)
    return {'out': out, 'key_cache': kc, 'value_cache': vc}


def _exact_logprobs(s):
    c = s['case']
    parts = {}
    for lo in range(0, c['rows'], 512):
        x = s['logits'][lo:lo + 512].double()
        tok = s['tokens'][lo:lo + 512]
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        p = logp.exp()
        plogp = torch.special.xlogy(p, p)
        picked = torch.where(tok >= 0, logp[torch.arange(len(tok), device=x.device), tok.clamp(min=0)], 0.0)
        here = {'log_prob': picked, 'entropy': -plogp.sum(-1)}
        if c['topk']:
            best = torch.argsort(-x, dim=-1, stable=True)[:, :c['topk']]
            here['top_log_prob'], here['top_token'] = torch.take_along_dim(logp, best, -1), best
        if c['train']:
            into = torch.zeros_like(x)                    # the gradient with respect to the log probabilities
            gl = torch.where(tok >= 0, s['log_prob_grad'][lo:lo + 512].double(), 0.0)
            into[torch.arange(len(tok), device=x.device), tok.clamp(min=0)] += gl
            if c['topk']:
                into.scatter_add_(-1, best, s['top_grad'][lo:lo + 512].double())
            ge = s['entropy_grad'][lo:lo + 512].double()[:, None]
            here['logits_grad'] = into - p * into.sum(-1, keepdim=True) - ge * (plogp - p * plogp.sum(-1, keepdim=True))
        for k, v in here.items():
            parts.setdefault(k, []).append(v)
    return {k: torch.cat(v) for k, v in parts.items()}


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    return (_exact_rotary if op == 'rotary' else _exact_attention if op == 'attention' else _exact_fill if op == 'fill'
            else _exact_step if op == 'step' else _exact_logprobs)(s)
