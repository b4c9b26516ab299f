"""The choice of experts by softmax or sigmoid scores, with a balance bias and by groups, and the update of that bias.  The reference has neither (its
router is softmax and top-k, megablocks/layers/router.py:87-106)."""
import ctypes
import math
from typing import Any, Optional

import torch
from torch.autograd.function import once_differentiable

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


class ChooseExpertsOp(torch.autograd.Function):
    """(scores, weights, indices, indices as int32, lse or None) of `mbx_choose_experts`."""

    @staticmethod
    def forward(ctx: Any, logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_lse):
        logits = logits.contiguous()
        bias = None if bias is None else bias.detach().contiguous()
        tokens, experts = logits.shape
        scores = torch.empty_like(logits)
        weights = torch.empty((tokens, top_k), dtype=logits.dtype, device=logits.device)
        indices = torch.empty((tokens, top_k), dtype=torch.int64, device=logits.device)
        indices32 = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
        lse = torch.empty((tokens,), dtype=torch.float32, device=logits.device) if want_lse else None
        with _lib.device_of(logits):
            _lib.check(lib.mbx_choose_experts(_lib.ptr(logits), _lib.dtype_of(logits), tokens, experts, top_k, SCORES[score], _lib.ptr(bias), groups,
                                              top_groups, group_best, norm_p, scale, _lib.ptr(scores), _lib.ptr(weights), _lib.ptr(indices),
                                              _lib.ptr(indices32), _lib.ptr(lse), _lib.stream()), 'choose_experts')
        ctx.save_for_backward(logits, indices)
        ctx.choice = top_k, score, norm_p, scale
        ctx.mark_non_differentiable(indices, indices32)
        ctx.set_materialize_grads(False)
        return scores, weights, indices, indices32, lse

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_scores, grad_weights, _grad_indices, _grad_indices32, grad_lse):
        if grad_scores is None and grad_weights is None and grad_lse is None:
            return (None,) * 10
        logits, indices = ctx.saved_tensors
        return (logits_gradient(logits, indices, *ctx.choice, grad_scores, grad_weights, grad_lse), *(None,) * 9)


def logits_gradient(logits, indices, top_k, score, norm_p, scale, grad_scores, grad_weights, grad_lse=None):
    """The gradient of the logits behind ChooseExpertsOp's outputs (`mbx_choose_experts_backward`); the outputs' may be None."""
    tokens, experts = logits.shape
    grad_logits = torch.empty_like(logits)
    gs = None if grad_scores is None else grad_scores.to(logits.dtype).contiguous()
    gw = None if grad_weights is None else grad_weights.to(logits.dtype).contiguous()
    gl = None if grad_lse is None else grad_lse.float().contiguous()
    with _lib.device_of(logits):
        _lib.check(lib.mbx_choose_experts_backward(_lib.ptr(gw), _lib.ptr(gs), _lib.ptr(gl), _lib.ptr(logits), _lib.ptr(indices), _lib.dtype_of(logits),
                                                   tokens, experts, top_k, SCORES[score], norm_p, scale, _lib.ptr(grad_logits), _lib.stream()),
                   'choose_experts_backward')
    return grad_logits


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
    lse (once: the gradient has none itself); the bias gets none (it is updated by `balance_bias`)."""
    norm_p, scale = float(norm_p or 0), float(scale)
    if logits.ndim != 2:
        raise ValueError('choose_experts: logits must be [tokens, experts]')
    if bias is not None and (bias.ndim != 1 or bias.shape[0] != logits.shape[1]):
        raise ValueError('choose_experts: the bias must be a vector of a number for every expert')
    check_choice(logits.shape[1], top_k, score, groups, top_groups, group_best, norm_p, scale)
    _lib.require_cuda(logits, bias)
    _lib.dtype_of(logits)
    if bias is not None and (bias.dtype != torch.float32 or bias.device != logits.device):
        raise RuntimeError(f'choose_experts: expected a float32 bias on {logits.device} but got {bias.dtype} on {bias.device}')
    scores, weights, indices, _, lse = ChooseExpertsOp.apply(logits, bias, top_k, score, groups, top_groups, group_best, norm_p, scale, want_lse)
    return scores, weights, indices, lse


def balance_bias(biases, tokens_per_expert, rate: float, out=None):
    """bias + rate * sign(mean - n) for every layer's bias (fp32 [experts]) and n, its tokens per expert (int32, [experts] or rows of that, which are added
    up): experts with fewer tokens than the mean are made likelier, those with more less likely.  biases, tokens_per_expert, out: lists of one tensor a
    layer, all of one number of experts; out (a list of fp32 vectors, which may be the biases themselves; no two of them the same) or None for new ones.
    Returns the list.  One launch for up to 64 layers."""
    layers = len(biases)
    if len(tokens_per_expert) != layers or (out is not None and len(out) != layers):
        raise ValueError('balance_bias: one vector of tokens per expert, and one output, for every bias')
    if not math.isfinite(rate):
        raise ValueError('balance_bias: the rate must be finite')
    if layers == 0:
        return []
    experts, device = biases[0].shape[0] if biases[0].ndim == 1 else 0, biases[0].device
    if experts == 0:
        raise ValueError('balance_bias: a bias must be a vector of a number for every expert')
    for t in (*biases, *(() if out is None else out)):
        if t.shape != (experts,):
            raise ValueError('balance_bias: all biases must be vectors of the same number of experts')
        if t.dtype != torch.float32:
            raise RuntimeError(f'balance_bias: expected float32 biases but got {t.dtype}')
    for n in tokens_per_expert:
        if n.ndim not in (1, 2) or n.shape[-1] != experts:
            raise ValueError('balance_bias: tokens per expert must be [experts] or [rows, experts]')
        if n.dtype != torch.int32:
            raise RuntimeError(f'balance_bias: expected int32 tokens per expert but got {n.dtype}')
    _lib.require_cuda(*biases, *tokens_per_expert, *(() if out is None else out))
    if any(t.device != device for t in (*biases, *tokens_per_expert, *(() if out is None else out))):
        raise RuntimeError('balance_bias: all tensors must be on one device')
    if out is None:
        out = list(torch.empty((layers, experts), dtype=torch.float32, device=device).unbind(0))
    elif any(not t.is_contiguous() for t in out):
        raise ValueError('balance_bias: outputs must be contiguous')
    elif len({t.data_ptr() for t in out}) < layers:
        raise ValueError('balance_bias: two layers have the same output; pass the rows of their tokens per expert as one')
    else:
        torch.autograd.graph.increment_version(out)
    biases = [t.detach().contiguous() for t in biases]
    counts = [n.contiguous() for n in tokens_per_expert]
    pointers = lambda tensors: (ctypes.c_void_p * layers)(*map(_lib.ptr, tensors))
    rows = (ctypes.c_int * layers)(*(1 if n.ndim == 1 else n.shape[0] for n in counts))
    with _lib.device_of(biases[0]):
        _lib.check(lib.mbx_balance_bias(pointers(biases), pointers(counts), rows, pointers(out), layers, experts, float(rate), _lib.stream()), 'balance_bias')
    return out
