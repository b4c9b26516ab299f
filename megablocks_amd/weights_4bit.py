"""Experts' weights in 4 bits with a scale, and if wanted a zero point, for every group of columns along the reduction.  The reference has none."""
from typing import Optional

import torch

from megablocks_amd import _lib
from megablocks_amd._lib import lib

GROUP_SIZES = (32, 64, 128)
_TILE_FEATURES, _TILE_COLUMNS = 16, 128


def _up(n, of):
    return (n + of - 1) // of


class Weights4bit:
    """Weights W [experts, n, k] in 4 bits: W[e, i, c] = scale * (code - zero), of the group of `group` columns that c is in.

        words   int32 [experts, ceil(n / 16), ceil(k / 128), 64, 4]: the codes in the order the kernels multiply them (include/mbx.h says which is where)
        scales  [experts, ceil(n / 16), ceil(k / 128) * 128 / group, 16], fp32 or of a 16-bit type
        zeros   uint8 like the scales, or None: 8 everywhere

    What lies past n and k, whole groups of scales and zeros among it, is never used and may be anything.
    trans_b: whether the weights came (and come back, `dequantize`) as [experts, n, k], else as [experts, k, n]; products are x @ W[e]^T either way."""

    def __init__(self, words: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], n: int, k: int, group: int, trans_b: bool = True):
        if group not in GROUP_SIZES:
            raise ValueError(f'4-bit weights: groups of {GROUP_SIZES} columns, not {group}')
        if n < 1 or k < 1 or words.ndim != 5 or tuple(words.shape[1:]) != (_up(n, _TILE_FEATURES), _up(k, _TILE_COLUMNS), 64, 4):
            raise ValueError(f'4-bit weights: words must be [experts, {_up(n, _TILE_FEATURES)}, {_up(k, _TILE_COLUMNS)}, 64, 4]')
        experts, tiles, blocks = words.shape[:3]
        of_groups = (experts, tiles, blocks * _TILE_COLUMNS // group, _TILE_FEATURES)
        if tuple(scales.shape) != of_groups or (zeros is not None and zeros.shape != scales.shape):
            raise ValueError(f'4-bit weights: scales (and zeros) must be {list(of_groups)}')
        if words.dtype != torch.int32 or scales.dtype not in _lib.DTYPE or (zeros is not None and zeros.dtype != torch.uint8):
            raise RuntimeError('4-bit weights: expected int32 words, bfloat16/float16/float32 scales and uint8 zeros')
        if any(t is not None and (t.device != words.device or not t.is_contiguous()) for t in (words, scales, zeros)):
            raise RuntimeError('4-bit weights: words, scales and zeros must be contiguous and on one device')
        self.words, self.scales, self.zeros = words, scales, zeros
        self.n, self.k, self.group, self.trans_b = int(n), int(k), int(group), bool(trans_b)

    @property
    def experts(self):
        return self.words.shape[0]

    @property
    def device(self):
        return self.words.device

    def group_scales(self):
        """The scales as [experts, n, groups]."""
        return self.scales.transpose(2, 3).flatten(1, 2)[:, :self.n, :_up(self.k, self.group)]

    def dequantize(self, dtype: Optional[torch.dtype] = None, trans_b: Optional[bool] = None) -> torch.Tensor:
        """The weights these stand for, rounded to `dtype` (None: the scales'), as [experts, n, k] (trans_b) or [experts, k, n]; None: as they came."""
        dtype, trans_b = dtype or self.scales.dtype, self.trans_b if trans_b is None else trans_b
        _lib.require_cuda(self.words)
        if dtype not in _lib.DTYPE:
            raise RuntimeError(f'4-bit weights: expected bfloat16, float16 or float32 but got {dtype}')
        out = torch.empty((self.experts, self.n, self.k) if trans_b else (self.experts, self.k, self.n), dtype=dtype, device=self.device)
        with _lib.device_of(out):
            _lib.check(lib.mbx_dequantize_4bit(_lib.ptr(self.words), _lib.ptr(self.scales), _lib.ptr(self.zeros), _lib.DTYPE[self.scales.dtype], self.experts,
                                               self.n, self.k, _lib.NT if trans_b else _lib.NN, self.group, _lib.ptr(out), _lib.DTYPE[dtype], _lib.stream()),
                       'dequantize_4bit')
        return out


def quantize_4bit(w: torch.Tensor, group_size: int = 128, trans_b: bool = True, zero_points: bool = False) -> Weights4bit:
    """Weights w [experts, n, k] (trans_b False: [experts, k, n]) in 4 bits, for products x @ w[e]^T (x @ w[e]), with a scale in w's type for every
    group_size (32, 64, 128) of the k columns: the largest weight of a group times 1 / 7 in fp32, or with zero_points the distance of its largest and smallest (and 0) times 1 / 15."""
    if w.ndim != 3:
        raise ValueError('quantize_4bit: w must be [experts, n, k] or [experts, k, n]')
    if group_size not in GROUP_SIZES:
        raise ValueError(f'quantize_4bit: groups of {GROUP_SIZES} columns, not {group_size}')
    if 0 in w.shape[1:]:
        raise ValueError('quantize_4bit: w has no columns or no features')
    _lib.require_cuda(w)
    _lib.dtype_of(w)
    w = w.detach().contiguous()
    experts = w.shape[0]
    n, k = w.shape[1:] if trans_b else (w.shape[2], w.shape[1])
    tiles, blocks = _up(n, _TILE_FEATURES), _up(k, _TILE_COLUMNS)
    words = torch.empty((experts, tiles, blocks, 64, 4), dtype=torch.int32, device=w.device)
    of_groups = (experts, tiles, blocks * _TILE_COLUMNS // group_size, _TILE_FEATURES)
    scales = torch.empty(of_groups, dtype=w.dtype, device=w.device)
    zeros = torch.empty(of_groups, dtype=torch.uint8, device=w.device) if zero_points else None
    with _lib.device_of(w):
        _lib.check(lib.mbx_quantize_4bit(_lib.ptr(w), _lib.dtype_of(w), experts, n, k, _lib.NT if trans_b else _lib.NN, group_size, _lib.ptr(words),
                                         _lib.ptr(scales), _lib.ptr(zeros), _lib.stream()), 'quantize_4bit')
    return Weights4bit(words, scales, zeros, n, k, group_size, trans_b)
