"""What the norm of many tensors and clipping refuse, without a GPU."""
import ctypes
import math

import pytest
import torch

import megablocks_amd.ops as ops
from megablocks_amd import _lib


@pytest.mark.parametrize('call', [
    lambda: ops.global_norm([torch.ones(3)], 3.0), lambda: ops.global_norm([torch.ones(3)], 0.0), lambda: ops.global_norm([torch.ones(3)], -math.inf),
    lambda: ops.global_norm([torch.ones(3)], math.nan), lambda: ops.clip_by_global_norm_([torch.ones(3)], -1.0), lambda: ops.clip_by_global_norm_([torch.ones(3)], math.nan),
    lambda: ops.clip_by_global_norm_([], math.nan), lambda: ops.clip_by_global_norm_([torch.ones(3)], 1.0, 1.5), lambda: ops.clip_grad_norm_([], -1.0)])
def test_norms_that_are_none_are_refused(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize('tensors', [[torch.ones(3)], [torch.ones(3).double()], [torch.ones(3).int()], [torch.ones(3).to_sparse()], [None], [1.0]])
def test_tensors_that_are_not_on_the_gpu_are_refused(tensors):
    with pytest.raises(RuntimeError):
        ops.global_norm(tensors)
    with pytest.raises(RuntimeError):
        ops.clip_by_global_norm_(tensors, 1.0)


def test_no_tensors():
    assert ops.global_norm([]).item() == 0 and ops.clip_by_global_norm_([], 1.0).item() == 0 and ops.clip_grad_norm_([], 1.0).item() == 0
    assert ops.clip_grad_norm_([torch.nn.Parameter(torch.ones(3))], 1.0, error_if_nonfinite=True).item() == 0      # no gradients


def _clip(ranges, outs, types=None, out_types=None, most=1.0, p=2.0, scratch=None):
    """mbx_clip_by_global_norm of made-up addresses: what it refuses it refuses before it looks at them."""
    n = len(ranges)
    addresses = (ctypes.c_void_p * n)(*[r[0] for r in ranges])
    numel = (ctypes.c_int64 * n)(*[r[1] for r in ranges])
    return _lib.lib.mbx_clip_by_global_norm(addresses, (ctypes.c_void_p * n)(*outs), numel, (ctypes.c_int * n)(*(types or [0] * n)), (ctypes.c_int * n)(*(out_types or [0] * n)),
                                            n, p, most, 8, scratch, 0, None)


@pytest.mark.parametrize('ranges,outs,out_types,clash', [
    ([(1000, 100), (1200, 100)], [1000, 1200], [0, 0], False),            # in place, next to each other
    ([(1000, 100), (1198, 100)], [1000, 1198], [0, 0], True),             # an element in common
    ([(1000, 100), (1000, 100)], [1000, 1000], [0, 0], True),             # the same tensor twice
    ([(1000, 100), (1000, 100)], [5000, 6000], [0, 0], False),            # read twice, written apart
    ([(1000, 100), (2000, 100)], [5000, 5199], [0, 0], True),
    ([(1000, 100), (2000, 100)], [2000, 1000], [0, 0], True),             # over each other's inputs
    ([(1000, 100)], [1100], [0], True),                                   # over itself, shifted
    ([(1000, 100)], [1000], [2], True),                                   # in place, wider
    ([(1000, 100)], [1000], [1], True),                                   # in place, another type
    ([(1000, 100), (1200, 50)], [9000, 8000], [2, 2], False),
    ([(1000, 100), (1200, 300)], [9000, 8000], [2, 2], True),             # 300 fp32 from 8000 on reach 9200
    ([(1000, 0), (1000, 100)], [1000, 1000], [0, 0], False)])             # one without elements
def test_outputs_in_each_others_way(ranges, outs, out_types, clash):
    # without scratch the others are refused too, for that
    assert _clip(ranges, outs, out_types=out_types) == (_lib.EINVAL if clash else _lib.ESCRATCH)


def test_entry_points_refuse_without_touching_the_gpu():
    lib = _lib.lib
    assert _clip([(1000, 1)], [1000], most=-1.0) == _lib.EINVAL and _clip([(1000, 1)], [1000], most=math.nan) == _lib.EINVAL
    assert _clip([(1000, 1)], [1000], p=3.0) == _lib.EINVAL and _clip([(1000, -1)], [1000]) == _lib.EINVAL and _clip([(1000, 1)], [None]) == _lib.EINVAL
    assert _clip([(None, 1)], [1000]) == _lib.EINVAL and _clip([(1000, 1)], [1000], types=[3]) == _lib.EINVAL and _clip([(1000, 1)], [1000], out_types=[-1]) == _lib.EINVAL
    assert _clip([(1000, 1 << 60)], [1000]) == _lib.ERANGE
    assert lib.mbx_global_norm(None, None, None, -1, 2.0, 8, None, 0, None) == _lib.EINVAL
    assert lib.mbx_global_norm(None, None, None, 1, 2.0, 8, None, 0, None) == _lib.EINVAL
    assert lib.mbx_global_norm(None, None, None, 0, 2.0, None, None, 0, None) == _lib.EINVAL
    one = (ctypes.c_void_p * 1)(1000), (ctypes.c_int64 * 1)(5), (ctypes.c_int * 1)(0)
    assert lib.mbx_global_norm(*one, 1, 2.0, 8, None, 0, None) == _lib.ESCRATCH
    assert lib.mbx_global_norm(*one, 1, 2.0, 8, 8, 7, None) == _lib.ESCRATCH and lib.mbx_global_norm(*one, 1, 2.0, 8, 12, 1 << 20, None) == _lib.ESCRATCH
    assert lib.mbx_global_norm_scratch_bytes(0) == 0
    sizes = [lib.mbx_global_norm_scratch_bytes(n) for n in (1, 128, 129, 1000)]
    assert sizes == sorted(sizes) and sizes[0] >= 2048 * 8
