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


def _views():
    g = torch.zeros(64, 96)
    cube = torch.zeros(4, 6, 10)
    line = torch.zeros(100)
    return [
        # apart
        ([g[:, :48], g[:, 48:]], None, True),                                  # column halves
        ([g[:, ::2], g[:, 1::2]], None, True),                                 # every other column
        ([g.t()[:, ::2], g.t()[:, 1::2]], None, True),                         # every other row, transposed
        ([g[::2, ::2], g[1::2], g[::2, 1::2]], None, True),
        ([cube[:, :3], cube[:, 3:, :5], cube[:, 3:, 5:]], None, True),
        ([cube[..., i] for i in range(10)], None, True),
        ([line[::3], line[1::3], line[2::3]], None, True),
        ([line.as_strided((1, 5), (0, 2))], None, True),                       # one row: its step does not count
        ([line[:0], line[::2]], None, True),
        ([g[:, :48], g[:, 48:]], [line[:50].expand(64, 50)[:, :48].contiguous(), torch.zeros(64, 48)], True),
        ([line[::2]], [line[1::2]], True),                                     # between the values of its tensor
        ([line[::2]], [line[::2]], True),                                      # another view of the same values
        ([line[:50].expand(2, 50)], [torch.zeros(50, 2).t()], True),           # a tensor that repeats itself is only read
        # over each other, or itself
        ([g[:, :49], g[:, 48:]], None, False),
        ([g[:, ::2], g[:, ::3]], None, False),
        ([g[:, ::2], g[5]], None, False),
        ([line.as_strided((4, 3), (2, 1))], None, False),
        ([line[:50:2].expand(2, 25)], None, False),
        ([g[:, :48], g[:, 48:]], [g[:, 48:], g[:, :48]], False),               # over each other's
        ([line[::2]], [line[:50]], False),                                     # a contiguous output over its strided tensor
        ([torch.zeros(50), line[::2]], [line[20:70], torch.zeros(50)], False),   # over another's
        ([torch.zeros(25, 2).t()], [line.as_strided((2, 25), (1, 1))], False),
        ([g[:, :48].bfloat16()[:, ::2], g[:, :24]], [g.view(torch.bfloat16)[:, 48:96:2], torch.zeros(64, 24)], True),
        ([g[:, :48].bfloat16()[:, ::2], g[:, :24]], [g.view(torch.bfloat16)[:, 46:94:2], torch.zeros(64, 24)], False)]


@pytest.mark.parametrize('case', range(len(_views())))
def test_which_views_lie_over_each_other(case):
    from megablocks_amd.ops import norm
    tensors, out, apart = _views()[case]
    tensors = [t for t in tensors]
    if apart:
        norm._refuse_overlaps(tensors if out is None else out, tensors)
    else:
        with pytest.raises(ValueError):
            norm._refuse_overlaps(tensors if out is None else out, tensors)


def test_an_output_in_the_place_of_its_tensor_in_another_order_is_refused():
    from megablocks_amd.ops import norm
    square, line = torch.zeros(8, 8), torch.zeros(100)
    for t, o in ((square, square.t()), (square[:, ::2], square[::2].t()), (line.as_strided((3, 5), (20, 2)), line.as_strided((5, 3), (2, 20)))):
        with pytest.raises(ValueError):
            norm._refuse_overlaps([o], [t])
    norm._refuse_overlaps([square[:, ::2]], [square[:, ::2]])


def test_views_of_a_buffer_that_are_apart_are_shown_to_be():
    """Every pair of slices with steps of a small matrix: what is said to be apart has no value in common, and little that has none is refused."""
    from megablocks_amd.ops import norm
    m = torch.arange(6 * 8, dtype=torch.float32).view(6, 8)
    views = [m[a:b:s, c:d:u] for a, b, s in ((0, 6, 1), (0, 3, 1), (3, 6, 1), (0, 6, 2), (1, 6, 2), (2, 3, 1)) for c, d, u in ((0, 8, 1), (0, 4, 1), (4, 8, 1), (3, 6, 1), (0, 8, 2), (1, 8, 2), (5, 6, 1))]
    views += [v.t() for v in views]
    refused = 0
    for x in views:
        for y in views:
            apart = not set(x.flatten().tolist()) & set(y.flatten().tolist())
            said = norm._Place(x).apart_from(norm._Place(y))
            assert apart or not said
            refused += apart and not said
        assert not norm._Place(x).over_itself()
    assert refused == 0
