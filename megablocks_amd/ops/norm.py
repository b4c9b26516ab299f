"""The norm of all gradients together, and clipping by it: what a training step does between its backward and its optimizer.  The reference leaves it to the
trainer around it, whose expert weights it marks for that purpose (megablocks/layers/mpu.py)."""
import array
import math
import operator

import torch

from megablocks_amd import _lib
from megablocks_amd._lib import lib

# a property of all tensors at a time, by calls that are C throughout: for hundreds of small tensors the host's time is what a pass takes (300 and as many outputs: 393 us of it
# a tensor's properties one after the other, now 219)
_is_contiguous, _get_device, _data_ptr, _numel = torch.Tensor.is_contiguous, torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.numel
_dtype, _requires_grad = operator.attrgetter('dtype'), operator.attrgetter('requires_grad')


def _check_norm(what, norm_type):
    norm_type = float(norm_type)
    if norm_type not in (1.0, 2.0, math.inf):
        raise ValueError(f'{what}: norms are of type 1, 2 or inf, not {norm_type}')
    return norm_type


class _Operands:
    """Tensors on one GPU as the library takes them: arrays of addresses, element counts and types in host memory."""

    def __init__(self, what, tensors):
        self.tensors = tensors
        try:
            dtypes, devices = list(map(_dtype, tensors)), set(map(_get_device, tensors))
            self.numel = array.array('q', map(_numel, tensors))
            if tensors and (len(devices) > 1 or min(devices) < 0 or not _lib.DTYPE.keys() >= set(dtypes)):
                raise RuntimeError(f'{what}: expected bfloat16, float16 or float32 tensors on one GPU but got {sorted({f"{t.dtype} on {t.device}" for t in tensors})}')
            self.plain = tensors if all(map(_is_contiguous, tensors)) else [t if t.is_contiguous() else None for t in tensors]
        except (TypeError, AttributeError):
            raise RuntimeError(f'{what}: expected dense tensors') from None
        self.device, self.types = devices, array.array('i', map(_lib.DTYPE.__getitem__, dtypes))
        if getattr(torch.autograd.forward_ad, '_current_level', 0) >= 0 or (torch.is_grad_enabled() and any(map(_requires_grad, tensors))):
            raise RuntimeError(f'{what}: norms and clipping have no gradient; call them under torch.no_grad(), on gradients')

    def fill(self, make):
        """A contiguous tensor, make(t), for each t that is not."""
        if self.plain is not self.tensors:
            self.plain = [make(t) if p is None else p for t, p in zip(self.tensors, self.plain)]
        self.addresses = array.array('Q', map(_data_ptr, self.plain))


def _address(values):
    return values.buffer_info()[0]


def _results(device, n):
    scratch = torch.empty(lib.mbx_global_norm_scratch_bytes(n), dtype=torch.uint8, device=device)
    return torch.empty((), dtype=torch.float32, device=device), scratch


def global_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all values of the tensors together, as one number in fp32 on their device: (sum |x|^p)^(1/p) for p = 1 and 2, max |x| for inf.  tensors:
    bf16, fp16 and fp32 ones, mixed as they come, of any shape.  Sums are held in 64 bits and come out the same from run to run; a NaN gives NaN.  No tensor:
    0, on the CPU."""
    norm_type, tensors = _check_norm('global_norm', norm_type), list(tensors)
    given = _Operands('global_norm', tensors)
    if not tensors:
        return torch.zeros((), dtype=torch.float32)
    given.fill(torch.Tensor.contiguous)
    norm, scratch = _results(tensors[0].device, len(tensors))
    with _lib.device_of(norm):
        _lib.check(lib.mbx_global_norm(_address(given.addresses), _address(given.numel), _address(given.types), len(tensors), norm_type, norm.data_ptr(),
                                       scratch.data_ptr(), scratch.numel(), _lib.stream()), 'global_norm')
    return norm


def clip_by_global_norm_(tensors, max_norm: float, norm_type: float = 2.0, out=None) -> torch.Tensor:
    """Multiplies the tensors by min(1, max_norm / (norm + 1e-6)), norm = `global_norm` of them all, and returns the norm before that; a norm that is NaN makes all
    values NaN, an infinite one zeros and NaN.  In place, where the launches that would write do nothing if the norm is short enough, or into `out`: as many tensors of
    as many elements, in bf16, fp16 or fp32 (the fp32 gradients an optimizer reads, for instance), rounded once.  No output may lie over another, or over a tensor
    that is not its own."""
    what = 'clip_by_global_norm_'
    norm_type, max_norm, tensors = _check_norm(what, norm_type), float(max_norm), list(tensors)
    if not max_norm >= 0:
        raise ValueError(f'{what}: the largest norm must be a number from 0 on')
    given = _Operands(what, tensors)
    to = given
    if out is not None:
        to = _Operands(what, list(out))
        if to.numel != given.numel:
            raise ValueError(f'{what}: an output of as many elements for every tensor')
    if not tensors:
        return torch.zeros((), dtype=torch.float32)
    if to.device != given.device:
        raise RuntimeError(f'{what}: tensors and outputs must be on one GPU')
    outputs = to.tensors
    if to.plain is not outputs or given.plain is not tensors:      # of which the library sees others
        _refuse_overlaps(outputs, tensors)
    given.fill(torch.Tensor.contiguous)
    if to is not given:
        to.fill(lambda t: torch.empty_like(t, memory_format=torch.contiguous_format))
    norm, scratch = _results(tensors[0].device, len(tensors))
    with _lib.device_of(norm):
        rc = lib.mbx_clip_by_global_norm(_address(given.addresses), _address(to.addresses), _address(given.numel), _address(given.types), _address(to.types), len(tensors),
                                         norm_type, max_norm, norm.data_ptr(), scratch.data_ptr(), scratch.numel(), _lib.stream())
    if rc == _lib.EINVAL:
        raise ValueError(f'{what}: an output lies over another one, or over a tensor that is not its own')
    _lib.check(rc, what)
    if to.plain is not outputs:
        for o, made in zip(outputs, to.plain):
            if made is not o:
                o.copy_(made)
    try:
        torch.autograd.graph.increment_version(outputs)
    except RuntimeError:      # tensors made in inference mode have no version
        torch.autograd.graph.increment_version([o for o in outputs if not o.is_inference()])
    return norm


class _Place:
    """Where a tensor's values lie: the bytes from begin to end, and (stride in bytes, size) of the dimensions that have more than one, by stride."""

    def __init__(self, t):
        self.item, self.begin = t.element_size(), t.data_ptr()
        dims = [(stride * self.item, size) for stride, size in zip(t.stride(), t.shape) if size > 1]
        self.dims = sorted(dims)
        self.end = self.begin + self.item + sum(stride * (size - 1) for stride, size in self.dims)
        self.same = self.begin, dims, t.dtype      # value by value

    def over_itself(self):
        """Whether two values may lie over each other: one step of a dimension is within what the narrower ones reach."""
        reach = self.item
        for stride, size in self.dims:
            if stride < reach:
                return True
            reach += stride * (size - 1)
        return False

    def apart_from(self, other):
        """Whether no value lies over one of the other's: the ranges of bytes do not meet, or all values of either are in a range of their own of every period."""
        if self.end <= other.begin or other.end <= self.begin:
            return True
        for period in {stride for stride, _ in self.dims + other.dims if stride}:
            mine, its = (p.item + sum(stride * (size - 1) for stride, size in p.dims if stride % period) for p in (self, other))
            if (other.begin - self.begin) % period >= mine and (self.begin - other.begin) % period >= its:
                return True
        return False


def _refuse_overlaps(outputs, tensors):
    """The library's check of its operands, on tensors of any strides.  Layouts that no program makes of slices, steps and transposes of a tensor may be refused too."""
    outs = [_Place(o) if o.numel() else None for o in outputs]
    places = [(p.begin, p, i, True) for i, p in enumerate(outs) if p is not None]
    for i, t in enumerate(tensors):
        if t is not outputs[i] and t.numel():
            p = _Place(t)
            if p.same != outs[i].same:
                places.append((p.begin, p, i, False))
    clash = any(p.over_itself() for p in outs if p is not None)
    near = []      # those that reach past where the next one begins
    for begin, p, _, writes in sorted(places, key=operator.itemgetter(0)):
        near = [n for n in near if n[0].end > begin]
        clash = clash or any((writes or n_writes) and not p.apart_from(n) for n, n_writes in near)
        near.append((p, writes))
    if clash:
        raise ValueError('clip_by_global_norm_: an output lies over another one, over a tensor that is not its own, or over itself')


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of the parameters (or of one) in place by their global norm, as torch.nn.utils.clip_grad_norm_ does, and returns the norm.
    error_if_nonfinite waits for the GPU: RuntimeError, and gradients as they were, where the norm is not finite."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad.detach() for p in parameters if p.grad is not None]
    if error_if_nonfinite and grads:
        norm = global_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f'clip_grad_norm_: the norm of order {float(norm_type)} of the gradients is not finite, so they cannot be clipped')
    return clip_by_global_norm_(grads, max_norm, norm_type)
