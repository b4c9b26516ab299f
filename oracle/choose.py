"""Plain restatement of the choice of experts by scores, bias and groups, its gradient and the bias's update: whole rows in float64 on the CPU,
loops instead of sorts.  The reference has no such router: parity unpinned, held to the formulas."""
import torch


def _before(a, b):
    """Whether key a comes before key b of a higher index: NaN first, then the larger."""
    return (a != a) or (b == b and a >= b)


def best(keys, count):
    """The indices of the `count` first keys of a list, in order; of equal ones the lower index first."""
    left, out = list(range(len(keys))), []
    for _ in range(count):
        first = left[0]
        for i in left[1:]:
            if not _before(keys[first], keys[i]):
                first = i
        out.append(first)
        left.remove(first)
    return out


def choose(logits, top_k, score='softmax', bias=None, groups=1, top_groups=1, group_best=2, norm_p=0, scale=1.0):
    """(scores, weights, indices, lse) in float64."""
    x = logits.detach().double().cpu()
    tokens, experts = x.shape
    s = torch.softmax(x, 1) if score == 'softmax' else torch.sigmoid(x)
    keys = x if bias is None else s + bias.double().cpu()
    group_keys = s if bias is None else keys
    size = experts // groups
    indices = torch.empty(tokens, top_k, dtype=torch.int64)
    for t in range(tokens):
        candidates = list(range(experts))
        if top_groups < groups:
            of = []
            for g in range(groups):
                row = group_keys[t, g * size:(g + 1) * size].tolist()
                of.append(sum(row[i] for i in best(row, min(group_best, size))))
            candidates = [e for g in sorted(best(of, top_groups)) for e in range(g * size, (g + 1) * size)]
        row = keys[t].tolist()
        indices[t] = torch.tensor([candidates[i] for i in best([row[e] for e in candidates], top_k)])
    w = s.gather(1, indices)
    n = w.norm(p=norm_p, dim=1, keepdim=True) if norm_p else torch.ones(tokens, 1, dtype=torch.float64)
    return s, scale * torch.where(n == 0, torch.zeros_like(w), w / n), indices, torch.logsumexp(x, 1)


def gradient(logits, indices, score, norm_p, scale, grad_scores=None, grad_weights=None, grad_lse=None):
    """(the gradient of the logits, the sum of the sizes of the terms it is made of), float64: the second is what errors are relative to."""
    x = logits.detach().double().cpu()
    soft = torch.softmax(x, 1)
    s = soft if score == 'softmax' else torch.sigmoid(x)
    slope = s if score == 'softmax' else torch.sigmoid(x) * torch.sigmoid(-x)
    ds, size = torch.zeros_like(x), torch.zeros_like(x)
    if grad_scores is not None:
        ds += grad_scores.double().cpu()
        size += grad_scores.double().cpu().abs()
    if grad_weights is not None:
        dy, w, indices = scale * grad_weights.double().cpu(), s.gather(1, indices.cpu()), indices.cpu()
        dw, terms = dy, dy.abs()
        if norm_p:
            n = w.norm(p=norm_p, dim=1, keepdim=True)
            u = w / n
            slant = torch.ones_like(u) if norm_p == 1 else u ** (norm_p - 1)
            dw = torch.where(n == 0, torch.zeros_like(w), (dy - (dy * u).sum(1, keepdim=True) * slant) / n)
            terms = torch.where(n == 0, torch.zeros_like(w), (dy.abs() + (dy.abs() * u).sum(1, keepdim=True) * slant) / n)
        ds.scatter_add_(1, indices, dw)
        size.scatter_add_(1, indices, terms)
    dx, terms = (s * (ds - (ds * s).sum(1, keepdim=True)), s * (size + (size * s).sum(1, keepdim=True))) if score == 'softmax' else (ds * slope, size * slope)
    if grad_lse is not None:
        dx = dx + grad_lse.double().cpu()[:, None] * soft
        terms = terms + grad_lse.double().cpu().abs()[:, None] * soft
    return dx, terms


def balance(bias, counts, rate):
    n = counts.cpu().long()
    n = n.sum(0) if n.ndim == 2 else n
    return bias.cpu().double() + rate * torch.sign(n.sum() - n * n.numel()).double()
