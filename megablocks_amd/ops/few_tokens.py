"""A whole mixture-of-experts layer for a few tokens, without gradients: megablocks/layers/moe.py:457-475 with the dropless experts of
megablocks/layers/dmoe.py:239-280, as a decoding step runs it."""
from typing import Optional

import torch

from megablocks_amd import _lib
from megablocks_amd._lib import lib
from megablocks_amd.ops.choose import SCORES, check_choice

MAX_TOKENS, MAX_TOP_K = 64, 16


def takes(tokens: int, hidden: int, ffn: int, experts: int, top_k: int) -> bool:
    """Whether the library has the layer for these sizes (of a token or more)."""
    return lib.mbx_moe_layer_scratch_bytes(tokens, hidden, ffn, experts, top_k, 1) != 0


def check_sizes(tokens: int, hidden: int, ffn: int, experts: int, top_k: int):
    """ValueError for sizes that `moe_layer` does not take."""
    if tokens > MAX_TOKENS or top_k > MAX_TOP_K:
        raise ValueError(f'moe_layer: up to {MAX_TOKENS} tokens and {MAX_TOP_K} experts a token, not {tokens} and {top_k}')
    if hidden < 8 or ffn < 8 or hidden % 8 or ffn % 8:
        raise ValueError(f'moe_layer: the hidden and the ffn size must be multiples of 8, not {hidden} and {ffn}')
    if not takes(max(tokens, 1), hidden, ffn, experts, top_k):
        raise ValueError(f'moe_layer: experts of [{ffn}, {hidden}] are too large')


def moe_layer(x: torch.Tensor, router: torch.Tensor, w1: torch.Tensor, v1: Optional[torch.Tensor], w2: torch.Tensor, top_k: int, act: int, score: str = 'softmax',
              bias: Optional[torch.Tensor] = None, groups: int = 1, top_groups: int = 1, group_best: int = 2, norm_p: float = 0, scale: float = 1.0):
    """(out, weights, indices) of a mixture-of-experts layer for up to 64 tokens x [tokens, hidden], without gradients:

        logits  = x @ router^T, router [experts, hidden]
        weights, indices = the choice of `choose_experts` with the options of that name, [tokens, top_k], fp32 and int64; scores in 64 bits
        out[t]  = sum_j weights[t, j] (activation(x[t] @ w1[e]^T) * (x[t] @ v1[e]^T)) @ w2[e], e = indices[t, j]

    w1, v1 (None: no gate) and w2: [experts, ffn, hidden], contiguous, all of x's type, bf16 or fp16; hidden and ffn multiples of 8; up to 16 experts a token.  act: ACT_SILU or
    ACT_GELU_TANH of `grouped_gemm_util`.  Logits are sums of exact products in 64 bits and are rounded nowhere, weights to fp32, products are fp32 sums,
    and out is rounded once.  On the way the activation is kept to 2^-17 of it in bf16; in fp16 to 2^-23 of it or 2^-32, whichever is more, and it is infinite from
    about 2^20 on, where the separate operators' is from 65520 on.  (A layer called as a module rounds each of them to its type, so the two agree to a few steps of that.)"""
    from megablocks_amd import grouped_gemm_util as gg
    norm_p, scale = float(norm_p or 0), float(scale)
    if x.ndim != 2 or router.ndim != 2 or w1.ndim != 3:
        raise ValueError('moe_layer: x must be [tokens, hidden], the router [experts, hidden] and the weights [experts, ffn, hidden]')
    tokens, hidden = x.shape
    experts, ffn = w1.shape[:2]
    if router.shape != (experts, hidden) or w1.shape[2] != hidden or w2.shape != w1.shape or (v1 is not None and v1.shape != w1.shape):
        raise ValueError('moe_layer: x, the router and the weights do not match')
    if bias is not None and bias.shape != (experts,):
        raise ValueError('moe_layer: the bias must be a vector of a number for every expert')
    if act not in (gg.ACT_SILU, gg.ACT_GELU_TANH):
        raise ValueError('moe_layer: act must be ACT_SILU or ACT_GELU_TANH')
    check_choice(experts, top_k, score, groups, top_groups, group_best, norm_p, scale)
    check_sizes(tokens, hidden, ffn, experts, top_k)
    device, dtype, recorded = x.device, x.dtype, torch.is_grad_enabled()
    if not x.is_cuda or dtype not in (torch.bfloat16, torch.float16):
        raise RuntimeError(f'moe_layer: expected bfloat16 or float16 tensors on a GPU but got {dtype} on {device}')
    if getattr(torch.autograd.forward_ad, '_current_level', 0) >= 0 or (recorded and x.requires_grad):
        raise RuntimeError('moe_layer: the layer for a few tokens has no gradient; call it under torch.no_grad()')
    for w in (router, w1, w2) if v1 is None else (router, w1, v1, w2):
        if w.device != device or w.dtype != dtype:
            raise RuntimeError(f'moe_layer: expected {dtype} weights on {device}, as the tokens, but got {w.dtype} on {w.device}')
        if recorded and w.requires_grad:
            raise RuntimeError('moe_layer: the layer for a few tokens has no gradient; call it under torch.no_grad()')
        if not w.is_contiguous() or w.data_ptr() % 16:
            raise RuntimeError('moe_layer: the router and the weights must be contiguous and start at multiples of 16 bytes')
    if bias is not None and (bias.dtype != torch.float32 or bias.device != device):
        raise RuntimeError(f'moe_layer: expected a float32 bias on {device} but got {bias.dtype} on {bias.device}')
    return launch(x, router, w1, v1, w2, ffn, top_k, act, score, bias, groups, top_groups, group_best, norm_p, scale)


def launch(x, router, w1, v1, w2, ffn, top_k, act, score, bias, groups, top_groups, group_best, norm_p, scale):
    """moe_layer of operands that have been checked."""
    from megablocks_amd import grouped_gemm_util as gg
    (tokens, hidden), device, experts = x.shape, x.device, router.shape[0]
    x = gg._aligned(x)
    bias = None if bias is None else bias.contiguous()
    out = torch.empty_like(x)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=device)
    indices = torch.empty((tokens, top_k), dtype=torch.int64, device=device)
    nbytes = lib.mbx_moe_layer_scratch_bytes(tokens, hidden, ffn, experts, top_k, v1 is not None)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with _lib.device_of(x):
        counters, counter_bytes = gg._counters(device)
        _lib.check(lib.mbx_moe_layer(x.data_ptr(), tokens, hidden, _lib.DTYPE[x.dtype], router.data_ptr(), experts, top_k, SCORES[score], _lib.ptr(bias), groups, top_groups,
                                     group_best, norm_p, scale, w1.data_ptr(), _lib.ptr(v1), w2.data_ptr(), ffn, act, out.data_ptr(), weights.data_ptr(), indices.data_ptr(),
                                     scratch.data_ptr(), nbytes, counters, counter_bytes, _lib.stream()), 'moe_layer')
    return out, weights, indices
