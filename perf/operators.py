"""Operators of a mixture-of-experts layer: how experts are chosen and kept in balance, and experts with 4-bit weights.

    listed()              the named cases
    draw(rng)             one more case from the same ranges
    prepare(case, seed)   what the program holds before the call
    run(state)            one pass: in plain torch operations, or with `own` by the framework's operators
    work(case)            bytes and operations the pass cannot do without
    exact(case, seed)     the pass's outputs in 64 bits

Kinds of case:

    choose     the router behind its linear layer: scores, experts, weights; with `train` the gradient of the logits too
    balance    the update of the routers' balance biases from the tokens each expert got
    quantize   weights into 4 bits with group scales, and the values these stand for
    product    the experts' products with 4-bit weights: 'glu' / 'mlp' the first products with the activation, rows gathered from the
               tokens; 'down' the second product

4-bit weights W [E, n, k] as they are kept: words int32 [E, n/16, k/128, 64, 4] (sizes rounded up), scales [E, n/16, k/group, 16], zeros like the
scales or None.  Lane 16 g + f, word j holds feature 16 t + f, columns 128 u + 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), four bits each from the
lowest; a code q stands for scale (q - zero), zero 8 where there are no zeros.
"""
import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}

# the dearest listed cases: no drawn one takes more
_MOST_LOGITS = 32768 * 256
_MOST_WEIGHTS = 8 * 4096 * 14336
_MOST_MACS = 8192 * 4096 * 14336 * 2


def _choose(tokens, experts, top_k, score, bias, groups=1, top_groups=1, group_best=2, norm=1, scale=1.0, dtype='bf16', train=False, zloss=False):
    return dict(kind='choose', tokens=tokens, experts=experts, top_k=top_k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                group_best=group_best, norm=norm, scale=scale, dtype=dtype, train=train, zloss=zloss)


def _product(form, tokens, hidden, ffn, experts, top_k, group, zeros=False, dtype='bf16', skew=0.0):
    return dict(kind='product', form=form, tokens=tokens, hidden=hidden, ffn=ffn, experts=experts, top_k=top_k, group=group, zeros=zeros,
                dtype=dtype, skew=skew)


def listed():
    return [
        # Decoding a batch of 16: many experts in groups, a bias that keeps them in balance. Latency.
        dict(_choose(16, 256, 8, 'sigmoid', True, 8, 4, scale=2.5), name='choose_decode_256e'),
        # A training step's router of the same kind, with the gradient.
        dict(_choose(32768, 256, 8, 'sigmoid', True, 8, 4, scale=2.5, train=True), name='choose_train_256e'),
        # Softmax scores, experts that are no power of two, best expert of a group, z-loss.
        dict(_choose(3001, 60, 4, 'softmax', False, 5, 3, 1, dtype='fp16', train=True, zloss=True), name='choose_train_odd'),
        # The biases after a step: of one layer, of a model's.
        dict(kind='balance', layers=1, experts=64, tokens=4096, top_k=6, name='balance_1_layer'),
        dict(kind='balance', layers=32, experts=256, tokens=32768, top_k=8, name='balance_32_layers'),
        # A trained layer's second weights on their way to serving: reduction over the rows.
        dict(kind='quantize', experts=8, n=4096, k=14336, group=128, zeros=False, trans_b=False, dtype='bf16', name='quantize_8e_down'),
        # Small odd experts, zero points, fine groups.
        dict(kind='quantize', experts=12, n=2728, k=1032, group=32, zeros=True, trans_b=True, dtype='fp16', name='quantize_odd_zeros'),
        # One token: the first products of a few large experts.
        dict(_product('glu', 1, 4096, 14336, 8, 2, 128), name='glu_1_token_8e'),
        # A batch of 16 sequences, every expert has a few rows: the second product.
        dict(_product('down', 16, 4096, 14336, 8, 2, 128), name='down_16_tokens_8e'),
        # A few sequences and many small experts.
        dict(_product('glu', 5, 2048, 1408, 64, 6, 64, zeros=True), name='glu_5_tokens_64e'),
        # A short prompt through odd experts without gate, skewed.
        dict(_product('mlp', 300, 1032, 2728, 32, 2, 32, zeros=True, dtype='fp16', skew=1.0), name='mlp_300_tokens_odd'),
        # A long prompt.
        dict(_product('glu', 4096, 4096, 14336, 8, 2, 128), name='glu_4096_tokens_8e'),
    ]


def _log(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def _size(rng, low, high, of):
    return max(of, int(round(_log(rng, low, high) / of)) * of)


def _draw_choose(rng):
    experts = rng.choice([4, 8, 12, 16, 60, 64, 96, 128, 160, 256, 384, 512])
    groups = rng.choice([g for g in (1, 1, 2, 3, 4, 5, 8, 16) if experts % g == 0 and experts // g >= 2])
    top_groups = rng.randint(1, groups)
    top_k = rng.choice([k for k in (1, 2, 4, 6, 8, 10, 16) if k <= top_groups * (experts // groups)])
    tokens = int(_log(rng, 1, min(32769, _MOST_LOGITS // experts)))
    train = rng.random() < 0.5
    return _choose(tokens, experts, top_k, rng.choice(['sigmoid', 'softmax']), rng.random() < 0.6, groups, top_groups, rng.choice([1, 2]),
                   rng.choice([0, 1, 1, 2]), rng.choice([1.0, 2.5]), rng.choice(['bf16', 'bf16', 'fp16', 'fp32']), train, train and rng.random() < 0.4)


def _draw_product(rng):
    while True:
        of = rng.choice([1, 8, 64, 64])
        c = _product(rng.choice(['glu', 'glu', 'mlp', 'down', 'down']), int(_log(rng, 1, 4097)), _size(rng, 512, 4096, of), _size(rng, 704, 14336, of),
                     rng.choice([1, 4, 8, 12, 16, 32, 64]), 1, rng.choice([32, 64, 128]), rng.random() < 0.4, rng.choice(['bf16', 'fp16']),
                     rng.choice([0.0, 0.0, 1.0]))
        c['top_k'] = rng.choice([k for k in (1, 2, 4, 6) if k <= max(1, c['experts'] // 2)])
        if c['experts'] * c['hidden'] * c['ffn'] <= _MOST_WEIGHTS and work(c)['flops'] <= 2 * _MOST_MACS:
            return c


def draw(rng):
    kind = rng.choice(['choose', 'choose', 'choose', 'balance', 'quantize', 'quantize', 'product', 'product', 'product', 'product'])
    if kind == 'choose':
        return _draw_choose(rng)
    if kind == 'balance':
        return dict(kind='balance', layers=int(_log(rng, 1, 33)), experts=rng.choice([8, 12, 60, 64, 128, 256]), tokens=int(_log(rng, 1, 32769)),
                    top_k=rng.choice([1, 2, 6, 8]))
    if kind == 'product':
        return _draw_product(rng)
    while True:
        of = rng.choice([1, 8, 64])
        c = dict(kind='quantize', experts=rng.choice([1, 4, 8, 12, 64]), n=_size(rng, 512, 14336, of), k=_size(rng, 512, 14336, of),
                 group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5, trans_b=rng.random() < 0.5, dtype=rng.choice(['bf16', 'fp16', 'fp32']))
        if c['experts'] * c['n'] * c['k'] <= _MOST_WEIGHTS // (2 if c['dtype'] == 'fp32' else 1):
            return c


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _routing(tokens, experts, top_k, skew, g):
    """(indices, bin_ids, bins, tokens per expert) of tokens that choose top_k experts each, popular ones first with a skew."""
    liking = torch.randn(tokens, experts, generator=g, device='cuda') - skew * torch.log(torch.arange(1, experts + 1, device='cuda').float())
    ids = liking.topk(top_k, dim=1).indices.flatten()
    bin_ids, indices = ids.sort(stable=True)
    counts = torch.bincount(ids, minlength=experts)
    return indices.int(), bin_ids.int(), counts.cumsum(0).int(), counts.int()


def _codes(experts, n, k, group, zeros, dtype, g):
    """4-bit weights as they are kept: of normal weights with a deviation of 0.02."""
    n16, k128 = -(-n // 16), -(-k // 128)
    words = torch.zeros(experts, n16, k128, 64, 4, dtype=torch.int32, device='cuda')
    for i in range(8):
        words |= torch.randn(words.shape, generator=g, device='cuda').mul_(2.4).add_(8).round_().clamp_(0, 15).int() << (4 * i)
    shape = (experts, n16, k128 * 128 // group, 16)
    scales = ((torch.rand(shape, generator=g, device='cuda') + 0.5) * (0.02 / 2.4)).to(dtype)
    return words, scales, torch.randint(6, 11, shape, generator=g, device='cuda', dtype=torch.uint8) if zeros else None


def prepare(case, seed):
    g, c = _generator(seed), case
    if c['kind'] == 'balance':
        liking = torch.rand(c['layers'], c['experts'], generator=g, device='cuda')
        counts = (liking / liking.sum(1, keepdim=True) * (c['tokens'] * c['top_k'])).round().int()
        biases = torch.randn(c['layers'], c['experts'], generator=g, device='cuda') * 0.01
        return dict(case=c, biases=list(biases.unbind(0)), counts=list(counts.unbind(0)), rate=0.001)
    dtype = _DTYPES[c['dtype']]
    if c['kind'] == 'choose':
        shape = (c['tokens'], c['experts'])
        state = dict(case=c, logits=(torch.randn(shape, generator=g, device='cuda') * 1.5).to(dtype), bias=None)
        if c['bias']:
            state['bias'] = torch.randint(-40, 41, (c['experts'],), generator=g, device='cuda').float() * 0.001
        if c['train']:
            state['grad_weights'] = torch.randn(c['tokens'], c['top_k'], generator=g, device='cuda').to(dtype)
            state['grad_scores'] = (torch.randn(shape, generator=g, device='cuda') * 0.1).to(dtype)
            state['grad_lse'] = torch.randn(c['tokens'], generator=g, device='cuda') * 0.1
        return state
    if c['kind'] == 'quantize':
        shape = (c['experts'], c['n'], c['k']) if c['trans_b'] else (c['experts'], c['k'], c['n'])
        return dict(case=c, weights=(torch.randn(shape, generator=g, device='cuda') * 0.02).to(dtype))
    indices, bin_ids, bins, counts = _routing(c['tokens'], c['experts'], c['top_k'], c['skew'], g)
    n, k = (c['hidden'], c['ffn']) if c['form'] == 'down' else (c['ffn'], c['hidden'])
    rows = c['tokens'] * (c['top_k'] if c['form'] == 'down' else 1)
    return dict(case=c, n=n, k=k, x=torch.randn(rows, k, generator=g, device='cuda').to(dtype), indices=indices, bin_ids=bin_ids, bins=bins,
                counts=counts, most=int(counts.max()), weights=[_codes(c['experts'], n, k, c['group'], c['zeros'], dtype, g)
                                                                for _ in range(2 if c['form'] == 'glu' else 1)])


# ---- one pass ----

def _plain_choose(s):
    c, x = s['case'], s['logits']
    if c['train']:
        x = x.detach().requires_grad_()
    values = x.float()
    shifted = values - values.detach().max(1, keepdim=True).values
    total = shifted.exp().sum(1, keepdim=True)
    scores = shifted.exp() / total if c['score'] == 'softmax' else 1 / (1 + (-values).exp())
    with torch.no_grad():      # the order of the keys in 64 bits: neighbours are often closer than 32 bits tell
        wide = x.double()
        soft = (wide - wide.max(1, keepdim=True).values).exp()
        wide_scores = soft / soft.sum(1, keepdim=True) if c['score'] == 'softmax' else 1 / (1 + (-wide).exp())
        keys = wide if s['bias'] is None else wide_scores + s['bias'].double()
        group_keys = wide_scores if s['bias'] is None else keys
        if c['groups'] > 1:
            size = c['experts'] // c['groups']
            best = group_keys.view(-1, c['groups'], size).sort(dim=2, descending=True).values[:, :, :c['group_best']].sum(2)
            ranks = best.sort(dim=1, descending=True, stable=True).indices.argsort(1)
            keys = keys.masked_fill((ranks >= c['top_groups']).repeat_interleave(size, 1), -math.inf)
        indices = keys.sort(dim=1, descending=True, stable=True).indices[:, :c['top_k']]
    weights = scores.gather(1, indices)
    if c['norm']:
        weights = weights / weights.pow(c['norm']).sum(1, keepdim=True).pow(1 / c['norm'])
    weights = (weights * c['scale']).to(x.dtype)
    out = dict(scores=scores.to(x.dtype), weights=weights, indices=indices)
    if c['zloss']:
        out['lse'] = total.log().squeeze(1) + values.max(1).values.detach()
    if c['train']:
        grads = [s['grad_scores'], s['grad_weights']] + ([s['grad_lse']] if c['zloss'] else [])
        out['grad'], = torch.autograd.grad([out['scores'], weights] + ([out['lse']] if c['zloss'] else []), x, grads)
    return {key: t.detach() for key, t in out.items()}


def _plain_balance(s):
    counts = torch.stack(s['counts']).long()
    off = counts.sum(1, keepdim=True) - counts * counts.shape[1]
    return list((torch.stack(s['biases']) + s['rate'] * off.sign().float()).unbind(0))


def _plain_quantize(s):
    c = s['case']
    w = s['weights'] if c['trans_b'] else s['weights'].transpose(1, 2)
    k, group = c['k'], c['group']
    w = torch.nn.functional.pad(w, (0, -k % group)).unflatten(2, (-1, group)).float()
    if c['zeros']:
        low, high = w.amin(3, keepdim=True).clamp(max=0), w.amax(3, keepdim=True).clamp(min=0)
        scales = ((high - low) / 15).to(s['weights'].dtype)
    else:
        scales = (w.abs().amax(3, keepdim=True) / 7).to(s['weights'].dtype)
    step = torch.where(scales == 0, 1.0, scales.float()).double()     # next to a half in 32 bits a quotient may round to it
    if c['zeros']:
        zero = (-low.double() / step).round().clamp(0, 15)
        codes = ((w.double() / step).round() + zero).clamp(0, 15) - zero
    else:
        codes = (w.double() / step).round().clamp(-8, 7)
    values = (codes.float() * scales.float()).flatten(2)[:, :, :k].to(s['weights'].dtype)
    return values if c['trans_b'] else values.transpose(1, 2).contiguous(), scales.squeeze(3)


def _plain_values(weights, n, k, group):
    words, scales, zeros = weights
    experts, n16, k128 = words.shape[:3]
    codes = (words.unsqueeze(-1) >> torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)) & 15
    codes = codes.view(experts, n16, k128, 4, 16, 4, 2, 4).permute(0, 1, 4, 2, 5, 3, 7, 6)     # expert, tile, feature, block, word, part, column pair
    codes = codes.reshape(experts, n16, 16, k128 * 128 // group, group).float()
    zero = 8.0 if zeros is None else zeros.float().transpose(2, 3).unsqueeze(-1)
    values = (codes - zero) * scales.float().transpose(2, 3).unsqueeze(-1)
    return values.reshape(experts, n16 * 16, k128 * 128)[:, :n, :k]


def _plain_product(s):
    c, ids = s['case'], s['bin_ids'].long()
    rows = s['x'] if c['form'] == 'down' else s['x'][s['indices'].long() // c['top_k']]
    places = torch.arange(len(ids), device=ids.device) - (s['bins'] - s['counts'])[ids]
    stacked = torch.zeros(c['experts'], s['most'], s['k'], device=rows.device)
    stacked[ids, places] = rows.float()
    first = torch.bmm(stacked, _plain_values(s['weights'][0], s['n'], s['k'], c['group']).transpose(1, 2).contiguous())[ids, places]
    if c['form'] == 'mlp':
        first = 0.5 * first * (1 + torch.tanh(math.sqrt(2 / math.pi) * (first + 0.044715 * first ** 3)))
    elif c['form'] == 'glu':
        gate = torch.bmm(stacked, _plain_values(s['weights'][1], s['n'], s['k'], c['group']).transpose(1, 2).contiguous())[ids, places]
        first = first / (1 + torch.exp(-first)) * gate
    return first.to(s['x'].dtype)


def _own_choose(s):
    from megablocks_amd import ops
    c, x = s['case'], s['logits']
    if c['train']:
        x = x.detach().requires_grad_()
    scores, weights, indices, lse = ops.choose_experts(x, c['top_k'], score=c['score'], bias=s['bias'], groups=c['groups'], top_groups=c['top_groups'],
                                                       group_best=c['group_best'], norm_p=c['norm'], scale=c['scale'], want_lse=c['zloss'])
    out = dict(scores=scores.detach(), weights=weights.detach(), indices=indices)
    if c['zloss']:
        out['lse'] = lse.detach()
    if c['train']:
        grads = [s['grad_scores'], s['grad_weights']] + ([s['grad_lse']] if c['zloss'] else [])
        out['grad'], = torch.autograd.grad([scores, weights] + ([lse] if c['zloss'] else []), x, grads)
    return out


def _own_balance(s):
    from megablocks_amd import ops
    return ops.balance_bias(s['biases'], s['counts'], s['rate'])


def _own_quantize(s):
    from megablocks_amd import grouped_gemm_util as gg
    c = s['case']
    kept = gg.quantize_4bit(s['weights'], c['group'], trans_b=c['trans_b'], zero_points=c['zeros'])
    return kept.dequantize(), kept.group_scales()


def _own_product(s):
    from megablocks_amd import grouped_gemm_util as gg
    c = s['case']
    kept = [gg.Weights4bit(words, scales, zeros, s['n'], s['k'], c['group']) for words, scales, zeros in s['weights']]
    if c['form'] == 'down':
        return gg.gmm_4bit(s['x'], kept[0], bins=s['bins'])
    src = gg.GatheredRows(s['x'], s['indices'], s['bin_ids'], s['bins'], None, c['top_k'], s['indices'].shape[0])
    return gg.gmm_4bit_act(src, kept[0], gg.ACT_GELU_TANH) if c['form'] == 'mlp' else gg.gmm_4bit_act(src, kept[0], gg.ACT_SILU, b2=kept[1])


def run(state):
    kind = state['case']['kind']
    if own:
        return {'choose': _own_choose, 'balance': _own_balance, 'quantize': _own_quantize, 'product': _own_product}[kind](state)
    return {'choose': _plain_choose, 'balance': _plain_balance, 'quantize': _plain_quantize, 'product': _plain_product}[kind](state)


def work(case):
    c = case
    if c['kind'] == 'balance':
        return dict(bytes=12 * c['layers'] * c['experts'], flops=4 * c['layers'] * c['experts'])
    size = _BYTES[c['dtype']]
    if c['kind'] == 'choose':
        logits, chosen = c['tokens'] * c['experts'], c['tokens'] * c['top_k']
        moved = 2 * logits * size + chosen * (size + 8) + (4 * c['experts'] if c['bias'] else 0) + (4 * c['tokens'] if c['zloss'] else 0)
        if c['train']:       # the gradients of scores, weights and lse read, the logits' written
            moved += 2 * logits * size + chosen * size + (4 * c['tokens'] if c['zloss'] else 0)
        return dict(bytes=moved, flops=(12 if c['train'] else 6) * logits)
    group_bytes = (size if not c['zeros'] else size + 1) / c['group']
    if c['kind'] == 'quantize':    # to 4 bits and back
        n = c['experts'] * c['n'] * c['k']
        return dict(bytes=int(n * 2 * (size + 0.5 + group_bytes)), flops=6 * n)
    rows, matrices = c['tokens'] * c['top_k'], 2 if c['form'] == 'glu' else 1
    n, k = (c['hidden'], c['ffn']) if c['form'] == 'down' else (c['ffn'], c['hidden'])
    # experts that get a row, of as many as choose evenly
    used = min(rows, c['experts'] * (1 - (1 - c['top_k'] / c['experts']) ** c['tokens']))
    read = (rows if c['form'] == 'down' else c['tokens']) * k * size
    return dict(bytes=int(used * n * k * matrices * (0.5 + group_bytes) + read + rows * n * size), flops=2 * rows * n * k * matrices)


# ---- the same from the definitions, in 64 bits ----

def _exact_choose(s):
    c, x, bias = s['case'], s['logits'].double(), s['bias']
    tokens, experts = x.shape
    top = x.amax(1, keepdim=True)
    soft = torch.exp(x - top) / torch.exp(x - top).sum(1, keepdim=True)
    score = soft if c['score'] == 'softmax' else torch.sigmoid(x)
    order = x.clone() if bias is None else score + bias.double()
    if c['groups'] > 1:
        by_group = (score if bias is None else order).reshape(tokens, c['groups'], -1)
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
    chosen = torch.cat(chosen, 1)
    w, p = score.gather(1, chosen), c['norm']
    norm = w.norm(p=p, dim=1, keepdim=True) if p else torch.ones_like(top)
    out = dict(scores=score, weights=c['scale'] * w / norm, indices=chosen)
    if c['zloss']:
        out['lse'] = torch.logsumexp(x, 1)
    if c['train']:
        dy = c['scale'] * s['grad_weights'].double()
        dw = dy / norm - ((dy * w).sum(1, keepdim=True) / norm ** 2 * (w / norm) ** (p - 1) if p else 0)
        ds = s['grad_scores'].double().scatter_add(1, chosen, dw)
        out['grad'] = soft * (ds - (ds * soft).sum(1, keepdim=True)) if c['score'] == 'softmax' else ds * score * torch.sigmoid(-x)
        if c['zloss']:
            out['grad'] += s['grad_lse'].double()[:, None] * soft
    return out


def _exact_quantize(s):
    c, w = s['case'], s['weights']
    values, scales = torch.empty(w.shape, dtype=torch.float64, device=w.device), []
    for e in range(c['experts']):
        m = (w[e] if c['trans_b'] else w[e].t()).double()
        out, of_expert = torch.empty_like(m), []
        for first in range(0, c['k'], c['group']):
            part = m[:, first:first + c['group']]
            high = part.amax(1).clamp(min=0) if c['zeros'] else part.abs().amax(1)
            low = part.amin(1).clamp(max=0) if c['zeros'] else torch.zeros_like(high)
            scale = ((high.float() - low.float()) / (15 if c['zeros'] else 7)).to(w.dtype)     # the scale is a number of the weights' type
            one = torch.where(scale == 0, torch.ones_like(scale), scale).double()[:, None]
            if c['zeros']:
                zero = torch.clamp(torch.round(-low[:, None] / one), 0, 15)
                codes = torch.clamp(torch.round(part / one), -zero, 15 - zero)
            else:
                codes = torch.clamp(torch.round(part / one), -8, 7)
            out[:, first:first + c['group']] = codes * scale.double()[:, None]
            of_expert.append(scale.double())
        values[e] = out if c['trans_b'] else out.t()
        scales.append(torch.stack(of_expert, 1))
    return values, torch.stack(scales)


def _exact_values(words, scales, zeros, n, k, group):
    """One expert's weights [n, k], from words [n/16, k/128, 64, 4]."""
    n16, k128 = words.shape[:2]
    values = torch.empty(n16, 16, k128, 4, 4, 8, dtype=torch.float64, device=words.device)    # tile, feature, block, word, part, column
    lanes = words.reshape(n16, k128, 4, 16, 4)
    for place, column in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
        values[..., column] = ((lanes >> (4 * place)) & 15).permute(0, 3, 1, 4, 2).double()
    values = values.reshape(n16, 16, -1, group)
    values -= 8 if zeros is None else zeros.double().permute(0, 2, 1).unsqueeze(3)
    values *= scales.double().permute(0, 2, 1).unsqueeze(3)
    return values.reshape(n16 * 16, k128 * 128)[:n, :k]


def _exact_product(s):
    c, counts = s['case'], s['counts'].tolist()
    rows = (s['x'] if c['form'] == 'down' else s['x'].index_select(0, torch.div(s['indices'], c['top_k'], rounding_mode='floor'))).double()
    parts, first = [], 0
    for e, count in enumerate(counts):
        if count:
            products = [rows[first:first + count] @ _exact_values(words[e], scales[e], None if zeros is None else zeros[e], s['n'], s['k'], c['group']).t()
                        for words, scales, zeros in s['weights']]
            a = products[0]
            if c['form'] == 'mlp':
                a = torch.nn.functional.gelu(a, approximate='tanh')
            elif c['form'] == 'glu':
                a = a * torch.sigmoid(a) * products[1]
            parts.append(a)
        first += count
    return torch.cat(parts)


def exact(case, seed):
    s = prepare(case, seed)
    if case['kind'] == 'choose':
        return _exact_choose(s)
    if case['kind'] == 'balance':
        return [b.double() + s['rate'] * torch.sign(n.double().mean() - n.double()) for b, n in zip(s['biases'], s['counts'])]
    if case['kind'] == 'quantize':
        return _exact_quantize(s)
    return _exact_product(s)
