"""The choice of experts by softmax or sigmoid scores, with a balance bias and by groups, and the update of that bias.  The reference has neither (its
router is softmax and top-k, megablocks/layers/router.py:87-106)."""
import bisect
import ctypes
import math
from typing import Any, Optional

import torch

from megablocks_amd import _lib
from megablocks_amd._lib import lib

SCORES = {'softmax': 0, 'sigmoid': 1}     # mbx_score of include/mbx.h
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 512, 64, 64


def check_choice(num_experts: int, top_k: int, score: str, groups: int, top_groups: int, group_best: int, norm_p: float, scale: float):
    """ValueError for a choice that is none."""
    if score not in SCORES:
        raise ValueError(f'choose_experts: the score is one of {sorted(SCORES)}, not {score!r}')
    if groups < 1 or num_experts % groups or not 1 <= top_groups <= groups:
        raise ValueError(f'choose_experts: {num_experts} experts have no {groups} equal groups of which {top_groups} can be open')
    if group_best not in (1, 2):
        raise ValueError('choose_experts: a group goes by its best expert or its best two')
    if not 1 <= top_k <= top_groups * (num_experts // groups):
        raise ValueError(f'choose_experts: {top_groups} groups of {num_experts // groups} experts have no {top_k} to choose')
    if not 0 <= norm_p < math.inf or not math.isfinite(scale):
        raise ValueError('choose_experts: norm_p must be a number from 0 on and scale finite')
    if num_experts > MAX_EXPERTS or top_k > MAX_TOP_K or groups > MAX_GROUPS:
        raise ValueError(f'choose_experts: up to {MAX_EXPERTS} experts, {MAX_TOP_K} a token and {MAX_GROUPS} groups')


def _launch(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_int32, want_lse):
    """(scores, weights, indices, indices as int32 or None, lse or None) by `mbx_choose_experts`; logits and bias contiguous."""
    tokens, experts = logits.shape
    device, dtype = logits.device, logits.dtype
    scores = torch.empty_like(logits)
    weights = torch.empty((tokens, top_k), dtype=dtype, device=device)
    indices = torch.empty((tokens, top_k), dtype=torch.int64, device=device)
    indices32 = torch.empty((tokens, top_k), dtype=torch.int32, device=device) if want_int32 else None
    lse = torch.empty((tokens,), dtype=torch.float32, device=device) if want_lse else None
    with _lib.device_of(logits):
        rc = lib.mbx_choose_experts(logits.data_ptr(), _lib.DTYPE[dtype], tokens, experts, top_k, SCORES[score], _lib.ptr(bias), groups, top_groups, group_best,
                                    norm_p, scale, scores.data_ptr(), weights.data_ptr(), indices.data_ptr(), _lib.ptr(indices32), _lib.ptr(lse), _lib.stream())
    _lib.check(rc, 'choose_experts')
    return scores, weights, indices, indices32, lse


class ChooseExpertsOp(torch.autograd.Function):
    """`_launch` with the logits' gradient."""

    @staticmethod
    def forward(ctx: Any, logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_int32, want_lse):
        scores, weights, indices, indices32, lse = _launch(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_int32, want_lse)
        ctx.save_for_backward(logits, indices)
        ctx.choice = top_k, score, norm_p, scale
        if want_int32:
            ctx.mark_non_differentiable(indices, indices32)
        else:
            ctx.mark_non_differentiable(indices)
        ctx.set_materialize_grads(False)
        return scores, weights, indices, indices32, lse

    @staticmethod
    def backward(ctx: Any, grad_scores, grad_weights, _grad_indices, _grad_indices32, grad_lse):
        if grad_scores is None and grad_weights is None and grad_lse is None:
            return (None,) * 11
        logits, indices = ctx.saved_tensors
        # a backward that is differentiated itself (create_graph), or runs over a batch of gradients at once (is_grads_batched)
        plain = torch.is_grad_enabled() or not all(_has_memory(g) for g in (grad_scores, grad_weights, grad_lse) if g is not None)
        grad = _differentiable_gradient if plain else logits_gradient
        return (grad(logits, indices, *ctx.choice, grad_scores, grad_weights, grad_lse),) + (None,) * 10


def _has_memory(t):
    try:
        t.data_ptr()
    except RuntimeError:
        return False
    return True


def logits_gradient(logits, indices, top_k, score, norm_p, scale, grad_scores, grad_weights, grad_lse=None):
    """The gradient of the logits behind ChooseExpertsOp's outputs (`mbx_choose_experts_backward`); the outputs' may be None."""
    tokens, experts = logits.shape
    grad_logits = torch.empty_like(logits)
    plain = lambda g, dtype: None if g is None else (g if g.dtype == dtype else g.to(dtype)).contiguous()
    gs, gw, gl = plain(grad_scores, logits.dtype), plain(grad_weights, logits.dtype), plain(grad_lse, torch.float32)
    with _lib.device_of(logits):
        rc = lib.mbx_choose_experts_backward(_lib.ptr(gw), _lib.ptr(gs), _lib.ptr(gl), logits.data_ptr(), indices.data_ptr(), _lib.DTYPE[logits.dtype], tokens,
                                             experts, top_k, SCORES[score], norm_p, scale, grad_logits.data_ptr(), _lib.stream())
    _lib.check(rc, 'choose_experts_backward')
    return grad_logits


def _differentiable_gradient(logits, indices, top_k, score, norm_p, scale, grad_scores, grad_weights, grad_lse=None):
    """logits_gradient in torch's operations, which have gradients themselves."""
    x = logits.float()
    soft = torch.softmax(x, 1) if score == 'softmax' or grad_lse is not None else None
    s = soft if score == 'softmax' else torch.sigmoid(x)
    g = torch.zeros_like(x) if grad_scores is None else grad_scores.float() * s         # the gradient of log s
    if grad_weights is not None:
        dy = grad_weights.float() * scale
        if norm_p > 0:
            logs = norm_p * (torch.log_softmax(x, 1) if score == 'softmax' else torch.nn.functional.logsigmoid(x)).gather(1, indices)
            parts = torch.softmax(logs, 1)                                               # u^p
            u = ((logs - logs.logsumexp(1, keepdim=True)) / norm_p).exp()
            here = dy * u - (dy * u).sum(1, keepdim=True) * parts
            here = here.masked_fill(s.gather(1, indices).amax(1, keepdim=True) == 0, 0.)     # scores that are all zero: weights without a gradient
        else:
            here = dy * s.gather(1, indices)
        g = g.scatter_add(1, indices, here)
    dx = g - s * g.sum(1, keepdim=True) if score == 'softmax' else g * torch.sigmoid(-x)
    return (dx if grad_lse is None else dx + grad_lse.float().unsqueeze(1) * soft).to(logits.dtype)


def choose_experts(logits: torch.Tensor, top_k: int, score: str = 'softmax', bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1,
                   group_best: int = 2, norm_p: float = 0, scale: float = 1.0, want_lse: bool = False):
    """(scores, weights, indices, lse) for rows of logits [tokens, experts] (bf16, fp16 or fp32):

        scores  = softmax or sigmoid of the logits
        indices = the top_k experts of largest score + bias (bias: fp32 [experts], or None), int64, in descending order, ties to the lower index;
                  with groups (of experts / groups neighbours each) of the top_groups groups of largest key only, a group's key being the sum of
                  its group_best (1 or 2) best scores + bias
        weights = scores at the indices, without the bias, divided by their p-norm where norm_p > 0, times `scale`
        lse     = logsumexp of the logits in fp32 where want_lse, else None

    The choice is that of the exact keys.  A token whose chosen scores are all zero has weights of zero.  Gradients go to the logits from scores, weights and
    lse (in fp32 from the logits), and on to the gradients' gradients; the bias gets none (it is updated by `balance_bias`)."""
    norm_p, scale = float(norm_p or 0), float(scale)
    if logits.ndim != 2:
        raise ValueError('choose_experts: logits must be [tokens, experts]')
    if bias is not None and bias.shape != logits.shape[1:]:
        raise ValueError('choose_experts: the bias must be a vector of a number for every expert')
    check_choice(logits.shape[1], top_k, score, groups, top_groups, group_best, norm_p, scale)
    scores, weights, indices, _, lse = choose(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, False, want_lse)
    return scores, weights, indices, lse


def choose(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_int32, want_lse):
    """choose_experts of a choice that has been checked, with the indices as int32 too where want_int32: (scores, weights, indices, indices32, lse)."""
    if not logits.is_cuda or (bias is not None and not bias.is_cuda):
        raise RuntimeError('choose_experts: expected logits (and bias) on the GPU')
    if logits.dtype not in _lib.DTYPE:
        raise RuntimeError(f'choose_experts: expected bfloat16, float16 or float32 logits but got {logits.dtype}')
    if bias is not None:
        if bias.dtype != torch.float32 or bias.device != logits.device:
            raise RuntimeError(f'choose_experts: expected a float32 bias on {logits.device} but got {bias.dtype} on {bias.device}')
        bias = bias.detach().contiguous()
    logits = logits.contiguous()
    # a node of its own is 7 us of the host's time; one in forward differentiation says that it has none
    recorded = (logits.requires_grad and torch.is_grad_enabled()) or getattr(torch.autograd.forward_ad, '_current_level', 0) >= 0
    run = ChooseExpertsOp.apply if recorded else _launch
    return run(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_int32, want_lse)


_is_contiguous, _get_device, _data_ptr = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.data_ptr


def _check_outputs(outputs, biases, size):
    """ValueError where layers, which are computed side by side, have outputs that overlap, or one lies over another's bias."""
    order = sorted(outputs)
    clash = any(after - before < size for before, after in zip(order, order[1:]))
    if outputs != biases and not clash:
        for l, at in enumerate(biases):
            near = bisect.bisect_left(order, at - size + 1)
            clash = clash or any(o < at + size and (o, o) != (at, outputs[l]) for o in order[near:near + 2])
    if clash:
        raise ValueError('balance_bias: two layers have outputs, or an output and a bias, in the same place; rows of counts for one bias go into one entry')


def balance_bias(biases, tokens_per_expert, rate: float, out=None):
    """bias + rate * sign(mean - n) for every layer's bias (fp32 [experts]) and n, its tokens per expert (int32, [experts] or rows of that, which are added
    up): experts with fewer tokens than the mean are made likelier, those with more less likely.  biases, tokens_per_expert, out: lists of one tensor a
    layer, all of one number of experts; out (a list of fp32 vectors, which may be the biases themselves, else in no layer's way) or None for new ones.
    Returns the list.  One launch for up to 64 layers."""
    layers = len(biases)
    if len(tokens_per_expert) != layers or (out is not None and len(out) != layers):
        raise ValueError('balance_bias: one vector of tokens per expert, and one output, for every bias')
    if not math.isfinite(rate):
        raise ValueError('balance_bias: the rate must be finite')
    if layers == 0:
        return []
    first = biases[0]
    shape, index = first.shape, first.get_device()
    if len(shape) != 1 or shape[0] == 0:
        raise ValueError('balance_bias: a bias must be a vector of a number for every expert')
    experts = shape[0]
    # a property of all tensors at a time: 32 layers cost the host 0.2 us a step each, a layer's steps one after the other twice that
    given = (*biases, *tokens_per_expert) if out is None else (*biases, *tokens_per_expert, *out)
    shapes, rows = [t.shape for t in given], [1] * layers
    if shapes.count(shape) < len(given):
        if any(s != shape for s in shapes[:layers]):
            raise ValueError('balance_bias: all biases must be vectors of the same number of experts')
        for l, s in enumerate(shapes[layers:2 * layers]):
            if s != shape:
                if len(s) != 2 or s[1] != experts:
                    raise ValueError('balance_bias: tokens per expert must be [experts] or [rows, experts]')
                rows[l] = s[0]
        if any(s != shape for s in shapes[2 * layers:]):
            raise ValueError('balance_bias: outputs must be contiguous vectors of a number for every expert')
    contiguous = list(map(_is_contiguous, given))
    if not all(contiguous[2 * layers:]):
        raise ValueError('balance_bias: outputs must be contiguous vectors of a number for every expert')
    dtypes = [t.dtype for t in given]
    if set(map(_get_device, given)) != {index} or index < 0 or dtypes.count(torch.float32) != len(given) - layers or dtypes.count(torch.int32) != layers or \
            dtypes[layers:2 * layers].count(torch.int32) != layers:
        raise RuntimeError('balance_bias: expected float32 biases (and outputs) and int32 tokens per expert on one GPU but got '
                           f'{sorted({f"{t.dtype} on {t.device}" for t in given})}')
    if not all(contiguous):
        given = [t if c else t.detach().contiguous() for t, c in zip(given, contiguous)]       # kept until the launch is under way
    pointers = list(map(_data_ptr, given))
    b_ptrs, n_ptrs, o_ptrs = pointers[:layers], pointers[layers:2 * layers], pointers[2 * layers:]
    if out is None:
        made = torch.empty((layers, experts), dtype=torch.float32, device=first.device)
        start = made.data_ptr()
        out, o_ptrs = list(made.unbind(0)), range(start, start + 4 * layers * experts, 4 * experts)
    else:
        _check_outputs(o_ptrs, b_ptrs, 4 * experts)
        torch.autograd.graph.increment_version(out)
    addresses = ctypes.c_void_p * layers
    with _lib.device_of(first):
        rc = lib.mbx_balance_bias(addresses(*b_ptrs), addresses(*n_ptrs), (ctypes.c_int * layers)(*rows), addresses(*o_ptrs), layers, experts, float(rate), _lib.stream())
    _lib.check(rc, 'balance_bias')
    return out
