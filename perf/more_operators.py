"""Operators around the experts of a language model: the whole layer for a few tokens, the embedding in front, the norm of all gradients behind.

    listed()              the named cases
    draw(rng)             one more case from the same ranges
    prepare(case, seed)   what the program holds before the call
    run(state)            one pass: in plain torch operations, or with `own` by the framework's operators
    work(case)            bytes and operations the pass cannot do without
    exact(case, seed)     the pass's outputs in 64 bits

Kinds of case:

    layer      a mixture-of-experts layer of up to 64 tokens without gradients: router, choice, experts, weighted sum.  Returns the output, the weights of the
               chosen experts (fp32) and which they are
    embedding  rows of a table by token, times a scale; with `train` the gradient of the table too
    norm       the norm of all tensors together, as fp32
    clip       that norm, and the tensors times min(1, most / (norm + 1e-6)): to other tensors (`out`: of their own type or fp32), or where they are
"""
import math
import random

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}

# the dearest listed cases: no drawn one takes more
_MOST_WEIGHTS = 8 * 4096 * 14336 * 3
_MOST_TABLE = 100000 * 2048
_MOST_ROWS = 32768 * 2048
_MOST_ELEMENTS = 64 * 1408 * 2048 * 3
_EPS = 1e-6


def _layer(tokens, hidden, ffn, experts, top_k, gate=True, act='silu', score='softmax', bias=False, groups=1, top_groups=1, group_best=2, norm=0, scale=1.0,
           dtype='bf16'):
    return dict(kind='layer', tokens=tokens, hidden=hidden, ffn=ffn, experts=experts, top_k=top_k, gate=gate, act=act, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_best=group_best, norm=norm, scale=scale, dtype=dtype)


def _embedding(tokens, vocabulary, hidden, scale=1.0, dtype='bf16', train=False, skew=0.0, padding=0.0, wide=True):
    return dict(kind='embedding', tokens=tokens, vocabulary=vocabulary, hidden=hidden, scale=scale, dtype=dtype, train=train, skew=skew, padding=padding, wide=wide)


def _tensors(kind, tensors, elements, dtype, split, norm=2.0, most=0.0, out=''):
    return dict(kind=kind, tensors=tensors, elements=elements, dtype=dtype, split=split, norm=norm, most=most, out=out)


def listed():
    return [
        # Decoding one sequence through many small experts: the launches and their latencies.
        dict(_layer(1, 2048, 1408, 64, 6), name='layer_1_token_64e'),
        # One sequence through a few large experts: two of eight are read.
        dict(_layer(1, 4096, 14336, 8, 2, norm=1), name='layer_1_token_8e'),
        # A batch of 16 sequences, one expert each, without a gate.
        dict(_layer(16, 1024, 4096, 64, 1, gate=False, act='gelu'), name='layer_16_tokens_64e_top1'),
        # A few sequences, sizes that fill no tile, experts chosen by sigmoid scores, a bias and groups.
        dict(_layer(5, 1032, 2728, 60, 4, score='sigmoid', bias=True, groups=5, top_groups=3, norm=1, scale=2.5, dtype='fp16'), name='layer_5_tokens_odd'),
        # The largest batch: all experts are read, 16 rows each.
        dict(_layer(64, 4096, 14336, 8, 2, norm=1), name='layer_64_tokens_8e'),
        # The tokens of a decoding step.
        dict(_embedding(16, 32000, 4096), name='embedding_16_tokens'),
        # A training step of a small model, words as often as in a text.
        dict(_embedding(16384, 50000, 1024, scale=32.0, train=True, skew=1.0), name='embedding_train_text'),
        # Padded sequences: two fifths of the tokens are padding that learns nothing, odd sizes.
        dict(_embedding(32767, 100000, 2040, dtype='fp16', train=True, skew=1.1, padding=0.4, wide=False), name='embedding_train_padded'),
        # The gradients of a layer of many experts.
        dict(_tensors('norm', 4, _MOST_ELEMENTS, 'bf16', 1), name='norm_layer_64e'),
        # A small model's: many short tensors of both types, into the fp32 ones an optimizer reads.
        dict(_tensors('clip', 300, 2000003, 'mixed', 2, most=1.0, out='fp32'), name='clip_300_small'),
        # The same layer, gradients that are too long, into fp32.
        dict(_tensors('clip', 4, _MOST_ELEMENTS, 'bf16', 1, most=1.0, out='fp32'), name='clip_layer_64e'),
        # Ordinary steps, most of whose gradients are short enough: they stay as they are.
        dict(_tensors('clip', 40, _MOST_ELEMENTS // 4, 'fp32', 3, most=1e6), name='clip_in_place_short'),
    ]


def _log(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _size(rng, low, high, of):
    return max(of, int(round(_log(rng, low, high) / of)) * of)


def _draw_layer(rng):
    while True:
        of = rng.choice([8, 64, 64])
        experts = rng.choice([1, 4, 8, 12, 16, 32, 60, 64, 128, 256])
        groups = rng.choice([g for g in (1, 1, 2, 4, 5, 8) if experts % g == 0 and experts // g >= 2] or [1])
        top_groups = rng.randint(1, groups)
        top_k = rng.choice([k for k in (1, 2, 4, 6, 8) if k <= top_groups * (experts // groups)])
        c = _layer(int(_log(rng, 1, 65)), _size(rng, 256, 7168, of), _size(rng, 256, 14336, of), experts, top_k, rng.random() < 0.7,
                   rng.choice(['silu', 'silu', 'gelu']), rng.choice(['softmax', 'softmax', 'sigmoid']), rng.random() < 0.3, groups, top_groups,
                   rng.choice([1, 2]), rng.choice([0, 1, 1, 2]), rng.choice([1.0, 2.5]), rng.choice(['bf16', 'bf16', 'fp16']))
        if experts * c['hidden'] * c['ffn'] * 3 <= _MOST_WEIGHTS:
            return c


def _draw_embedding(rng):
    while True:
        train = rng.random() < 0.7
        c = _embedding(int(_log(rng, 1, 65537)), int(_log(rng, 500, 200001)), _size(rng, 64, 8192, rng.choice([1, 8, 64])), rng.choice([1.0, 1.0, 32.0]),
                       rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), train, rng.choice([0.0, 1.0, 1.2]), rng.choice([0.0, 0.0, 0.3, 0.9]), rng.random() < 0.7)
        wide = 2 if c['dtype'] == 'fp32' else 1
        if c['vocabulary'] * c['hidden'] * wide <= _MOST_TABLE and c['tokens'] * c['hidden'] * wide <= _MOST_ROWS:
            return c


def _draw_tensors(rng):
    kind = rng.choice(['norm', 'clip', 'clip'])
    tensors = int(_log(rng, 1, 401))
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32', 'mixed'])
    elements = int(_log(rng, max(tensors, 1000), _MOST_ELEMENTS // (4 if dtype in ('fp32', 'mixed') else 1)))
    out = rng.choice(['', 'same', 'fp32', 'fp32']) if kind == 'clip' else ''
    most = 1e9 if kind == 'clip' and out == '' else rng.choice([0.01, 1.0, 1e6])
    return _tensors(kind, tensors, elements, dtype, rng.randint(1, 1 << 20), rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]), most if kind == 'clip' else 0.0, out)


def draw(rng):
    return rng.choice([_draw_layer, _draw_layer, _draw_embedding, _draw_tensors])(rng)


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _sizes(case):
    """The tensors' element counts: spread over two decades, `elements` in all."""
    rng = random.Random(case['split'])
    weights = [math.exp(rng.uniform(0, math.log(100))) for _ in range(case['tensors'])]
    sizes = [max(1, int(w / sum(weights) * case['elements'])) for w in weights]
    sizes[0] += max(0, case['elements'] - sum(sizes))
    return sizes


def _types(case):
    types = ['bf16', 'fp32', 'fp16'] if case['dtype'] == 'mixed' else [case['dtype']]
    return [types[i % len(types)] for i in range(case['tensors'])]


def _places(sizes, types):
    """Where each tensor starts in its type's buffer, and the buffers' element counts: 64 elements or a multiple from one to the next."""
    starts, ends = [], {}
    for n, dtype in zip(sizes, types):
        starts.append(ends.get(dtype, 0))
        ends[dtype] = starts[-1] + -(-n // 64) * 64
    return starts, ends


def _in_buffers(sizes, types):
    """Tensors of these sizes and types as views of one buffer a type, as the gradients of a model are kept, and the buffers."""
    starts, ends = _places(sizes, types)
    buffers = {dtype: torch.zeros(n, dtype=_DTYPES[dtype], device='cuda') for dtype, n in ends.items()}
    return [buffers[dtype][at:at + n] for at, n, dtype in zip(starts, sizes, types)], buffers


def prepare(case, seed):
    g, c = _generator(seed), case
    normal = lambda *shape: torch.randn(shape, generator=g, device='cuda')
    if c['kind'] in ('norm', 'clip'):
        state = dict(case=c, out=None)
        sizes, types = _sizes(c), _types(c)
        state['tensors'], state['buffers'] = _in_buffers(sizes, types)
        for i, t in enumerate(state['tensors']):
            t.copy_(normal(t.numel()) * (0.01 * (1 + i % 3)))
        if c['out']:
            state['out'], state['buffers'] = _in_buffers(sizes, types if c['out'] == 'same' else ['fp32'] * len(sizes))
        return state
    dtype = _DTYPES[c['dtype']]
    if c['kind'] == 'embedding':
        n, v = c['tokens'], c['vocabulary']
        u = torch.rand(n, generator=g, device='cuda', dtype=torch.float64)
        if c['skew']:      # the p-th most frequent word with a probability of about p^-skew
            a = 1 - c['skew']
            ranks = torch.exp(u * math.log(v)) if abs(a) < 1e-6 else ((v ** a - 1) * u + 1) ** (1 / a)
        else:
            ranks = u * v + 1
        words = torch.randperm(v, generator=g, device='cuda')
        ids = words[(ranks.long() - 1).clamp(0, v - 1)]
        padding = None
        if c['padding']:
            padding = v // 3
            ids[torch.rand(n, generator=g, device='cuda') < c['padding']] = padding
        state = dict(case=c, ids=ids if c['wide'] else ids.int(), table=normal(v, c['hidden']).to(dtype), padding=padding)
        if c['train']:
            state['table'].requires_grad_()
            state['grad'] = normal(n, c['hidden']).to(dtype)
        return state
    e, f, h = c['experts'], c['ffn'], c['hidden']
    weights = lambda: torch.stack([(normal(f, h) * 0.02).to(dtype) for _ in range(e)])
    return dict(case=c, x=normal(c['tokens'], h).to(dtype), router=(normal(e, h) * 0.02).to(dtype), w1=weights(), v1=weights() if c['gate'] else None, w2=weights(),
                bias=torch.randint(-40, 41, (e,), generator=g, device='cuda').float() * 0.001 if c['bias'] else None)


# ---- one pass ----

def _plain_choice(s):
    """(weights in fp32, indices): in 64 bits, neighbours are often closer than 32 bits tell."""
    c = s['case']
    logits = s['x'].double() @ s['router'].double().t()
    soft = (logits - logits.max(1, keepdim=True).values).exp()
    scores = soft / soft.sum(1, keepdim=True) if c['score'] == 'softmax' else 1 / (1 + (-logits).exp())
    keys = logits if s['bias'] is None else scores + s['bias'].double()
    group_keys = scores if s['bias'] is None else keys
    if c['groups'] > 1:
        size = c['experts'] // c['groups']
        best = group_keys.view(-1, c['groups'], size).sort(dim=2, descending=True).values[:, :, :c['group_best']].sum(2)
        ranks = best.sort(dim=1, descending=True, stable=True).indices.argsort(1)
        keys = keys.masked_fill((ranks >= c['top_groups']).repeat_interleave(size, 1), -math.inf)
    indices = keys.sort(dim=1, descending=True, stable=True).indices[:, :c['top_k']]
    weights = scores.gather(1, indices)
    if c['norm']:
        weights = weights / weights.pow(c['norm']).sum(1, keepdim=True).pow(1 / c['norm'])
    return (weights * c['scale']).float(), indices


def _plain_act(c, x):
    return x / (1 + torch.exp(-x)) if c['act'] == 'silu' else 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def _plain_layer(s):
    c = s['case']
    weights, indices = _plain_choice(s)
    x, tokens, slots = s['x'].float(), c['tokens'], c['tokens'] * c['top_k']
    if slots < c['experts']:      # the chosen experts' weights, an assignment each
        chosen = indices.flatten()
        rows = x.repeat_interleave(c['top_k'], 0).unsqueeze(2)
        hidden = _plain_act(c, torch.bmm(s['w1'][chosen].float(), rows))
        if c['gate']:
            hidden = hidden * torch.bmm(s['v1'][chosen].float(), rows)
        out = torch.bmm((hidden.squeeze(2) * weights.view(-1, 1)).unsqueeze(1), s['w2'][chosen].float()).view(tokens, c['top_k'], -1).sum(1)
    else:                         # all experts for all tokens, those not chosen with a weight of zero
        columns = x.t().contiguous()
        by_expert = torch.zeros(tokens, c['experts'], device=x.device).scatter_(1, indices, weights)
        hidden = _plain_act(c, s['w1'].float().flatten(0, 1) @ columns)
        if c['gate']:
            hidden = hidden * (s['v1'].float().flatten(0, 1) @ columns)
        hidden = hidden.view(c['experts'], c['ffn'], tokens) * by_expert.t().unsqueeze(1)
        out = hidden.flatten(0, 1).t().contiguous() @ s['w2'].float().flatten(0, 1)
    return dict(out=out.to(s['x'].dtype), weights=weights, indices=indices)


def _plain_embedding(s):
    c, ids, table = s['case'], s['ids'].long(), s['table'].detach()
    out = dict(out=(table[ids].float() * c['scale']).to(table.dtype))
    if c['train']:
        grad = s['grad'].double()     # hundreds of thousands of rows may meet in one
        if s['padding'] is not None:
            grad = grad * (ids != s['padding']).unsqueeze(1)
        sums = torch.zeros(table.shape, dtype=torch.float64, device=table.device).index_add_(0, ids, grad)
        out['grad'] = (sums * c['scale']).to(table.dtype)
    return out


def _plain_norm(s):
    p = s['case']['norm']
    if p == math.inf:
        return torch.stack([t.abs().max().float() for t in s['tensors']]).max()
    parts = [t.double().abs().sum() if p == 1 else t.double().square().sum() for t in s['tensors']]     # long sums
    total = torch.stack(parts).sum()
    return (total if p == 1 else total.sqrt()).float()


def _plain_clip(s):
    norm = _plain_norm(s)
    by = (s['case']['most'] / (norm + _EPS)).clamp(max=1)
    if s['out'] is None:
        for t in s['tensors']:
            t.copy_(t.float() * by)
    else:
        for t, o in zip(s['tensors'], s['out']):
            o.copy_(t.float() * by)
    return dict(norm=norm, buffers=s['buffers'])


def _own_layer(s):
    from megablocks_amd import grouped_gemm_util as gg, ops
    c = s['case']
    out, weights, indices = ops.moe_layer(s['x'], s['router'], s['w1'], s['v1'], s['w2'], c['top_k'], gg.ACT_SILU if c['act'] == 'silu' else gg.ACT_GELU_TANH,
                                          score=c['score'], bias=s['bias'], groups=c['groups'], top_groups=c['top_groups'], group_best=c['group_best'],
                                          norm_p=c['norm'], scale=c['scale'])
    return dict(out=out, weights=weights, indices=indices)


def _own_embedding(s):
    from megablocks_amd import ops
    c = s['case']
    out = ops.embedding(s['ids'], s['table'], scale=c['scale'], padding_idx=s['padding'])
    if not c['train']:
        return dict(out=out)
    grad, = torch.autograd.grad(out, s['table'], s['grad'])
    return dict(out=out.detach(), grad=grad)


def _own_norm(s):
    from megablocks_amd import ops
    return ops.global_norm(s['tensors'], s['case']['norm'])


def _own_clip(s):
    from megablocks_amd import ops
    norm = ops.clip_by_global_norm_(s['tensors'], s['case']['most'], s['case']['norm'], out=s['out'])
    return dict(norm=norm, buffers=s['buffers'])


def run(state):
    kind = state['case']['kind']
    if own:
        return {'layer': _own_layer, 'embedding': _own_embedding, 'norm': _own_norm, 'clip': _own_clip}[kind](state)
    return {'layer': _plain_layer, 'embedding': _plain_embedding, 'norm': _plain_norm, 'clip': _plain_clip}[kind](state)


def work(case):
    c = case
    if c['kind'] in ('norm', 'clip'):
        sizes, types = _sizes(c), _types(c)
        moved = sum(n * _BYTES[t] for n, t in zip(sizes, types)) + 4
        if c['out']:
            moved += sum(n * (4 if c['out'] == 'fp32' else _BYTES[t]) for n, t in zip(sizes, types))
        return dict(bytes=moved, flops=sum(sizes) * (3 if c['out'] else 2))
    size = _BYTES[c['dtype']]
    if c['kind'] == 'embedding':
        row = c['hidden'] * size
        moved = c['tokens'] * (8 if c['wide'] else 4) + min(c['tokens'], c['vocabulary']) * row + c['tokens'] * row
        flops = c['tokens'] * c['hidden']
        if c['train']:
            moved += int(c['tokens'] * (1 - c['padding'])) * row + c['vocabulary'] * row
            flops += c['tokens'] * c['hidden']
        return dict(bytes=moved, flops=flops)
    slots, matrices = c['tokens'] * c['top_k'], 3 if c['gate'] else 2
    # experts that get a row, of as many as choose evenly
    used = min(slots, c['experts'] * (1 - (1 - c['top_k'] / c['experts']) ** c['tokens']))
    moved = used * c['hidden'] * c['ffn'] * matrices * size + c['experts'] * c['hidden'] * size + 2 * c['tokens'] * c['hidden'] * size + slots * 12
    return dict(bytes=int(moved), flops=2 * slots * c['hidden'] * c['ffn'] * matrices + 2 * c['tokens'] * c['experts'] * c['hidden'])


# ---- the same from the definitions, in 64 bits ----

def _exact_layer(s):
    c, x = s['case'], s['x'].double()
    tokens, experts = c['tokens'], c['experts']
    logits = torch.einsum('th,eh->te', x, s['router'].double())
    score = torch.softmax(logits, 1) if c['score'] == 'softmax' else torch.sigmoid(logits)
    order = logits.clone() if s['bias'] is None else score + s['bias'].double()
    if c['groups'] > 1:
        by_group = (score if s['bias'] is None else order).reshape(tokens, c['groups'], -1)
        key = torch.topk(by_group, min(c['group_best'], by_group.shape[2]), dim=2).values.sum(2)
        before = (key[:, :, None] < key[:, None, :]) | ((key[:, :, None] == key[:, None, :]) & torch.ones(c['groups'], c['groups'], device=x.device).tril(-1).bool())
        shut = before.sum(2) >= c['top_groups']
        order[shut[:, :, None].expand(by_group.shape).reshape(tokens, experts)] = -math.inf
    chosen = []
    for _ in range(c['top_k']):
        best = order.amax(1, keepdim=True)
        first = torch.where(order == best, torch.arange(experts, device=x.device), experts).amin(1, keepdim=True)
        chosen.append(first)
        order.scatter_(1, first, -math.inf)
    indices = torch.cat(chosen, 1)
    weights = score.gather(1, indices)
    if c['norm']:
        weights = weights / weights.norm(p=c['norm'], dim=1, keepdim=True)
    weights = c['scale'] * weights
    out = torch.zeros_like(x)
    for e in indices.unique().tolist():
        t, j = (indices == e).nonzero(as_tuple=True)
        a = x[t] @ s['w1'][e].double().t()
        a = torch.nn.functional.silu(a) if c['act'] == 'silu' else torch.nn.functional.gelu(a, approximate='tanh')
        if c['gate']:
            a = a * (x[t] @ s['v1'][e].double().t())
        out[t] += weights[t, j].unsqueeze(1) * (a @ s['w2'][e].double())
    return dict(out=out, weights=weights, indices=indices)


def _exact_embedding(s):
    c, ids, table = s['case'], s['ids'].long(), s['table'].detach()
    out = dict(out=torch.nn.functional.embedding(ids, table.double()) * c['scale'])
    if c['train']:
        order = ids.sort(stable=True).indices
        if s['padding'] is not None:
            order = order[ids[order] != s['padding']]
        words, counts = ids[order].unique_consecutive(return_counts=True)
        grad = torch.zeros(table.shape, dtype=torch.float64, device=table.device)
        grad[words] = torch.segment_reduce(s['grad'].double()[order], 'sum', lengths=counts, axis=0) * c['scale'] if len(order) else 0.0
        out['grad'] = grad
    return out


def _exact_norm(s):
    norms = [torch.linalg.vector_norm(t, s['case']['norm'], dtype=torch.float64) for t in s['tensors']]
    return torch.linalg.vector_norm(torch.stack(norms), s['case']['norm'])


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'layer':
        return _exact_layer(s)
    if case['kind'] == 'embedding':
        return _exact_embedding(s)
    norm = _exact_norm(s)
    if case['kind'] == 'norm':
        return norm
    by = min(1.0, case['most'] / (norm.item() + _EPS))
    sizes, types = _sizes(case), _types(case)
    types = ['fp32'] * len(sizes) if case['out'] == 'fp32' else types
    starts, ends = _places(sizes, types)
    buffers = {dtype: torch.zeros(n, dtype=torch.float64, device='cuda') for dtype, n in ends.items()}
    for at, t, dtype in zip(starts, s['tensors'], types):
        buffers[dtype][at:at + t.numel()] = t.double() * by
    return dict(norm=norm, buffers=buffers)
