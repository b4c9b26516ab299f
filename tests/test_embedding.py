"""What the embedding refuses, without a GPU."""
import math

import pytest
import torch

import megablocks_amd.ops as ops
from megablocks_amd import _lib

IDS, TABLE = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)


@pytest.mark.parametrize('changed', [dict(table=torch.zeros(5)), dict(table=torch.zeros(5, 8, 1)), dict(scale=math.inf), dict(scale=math.nan), dict(padding_idx=5),
                                     dict(padding_idx=-6), dict(table=torch.zeros(0, 8), padding_idx=0)])
def test_calls_that_are_none_are_refused(changed):
    with pytest.raises(ValueError):
        ops.embedding(**(dict(ids=IDS, table=TABLE) | changed))


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError):
        ops.embedding(IDS, TABLE)


def test_entry_points_refuse_without_touching_the_gpu():
    lib = _lib.lib

    def rows(itype=2, tokens=3, dtype=0, words=5, hidden=8, ids=16, table=16, out=16):
        return lib.mbx_embedding(ids, itype, tokens, table, dtype, words, hidden, 1.0, out, None)

    def gradient(itype=2, tokens=3, dtype=0, words=5, hidden=8, grad=16, ids=16, out=16, scratch=None, nbytes=0):
        return lib.mbx_embedding_gradient(grad, ids, itype, tokens, dtype, words, hidden, -1, 1.0, out, scratch, nbytes, None)
    for call in (rows, gradient):
        for bad in (dict(itype=0), dict(itype=3), dict(tokens=-1), dict(words=-1), dict(hidden=-1), dict(dtype=3), dict(dtype=-1), dict(ids=None), dict(out=None)):
            assert call(**bad) == _lib.EINVAL
        for bad in (dict(tokens=1 << 31), dict(words=1 << 31), dict(hidden=1 << 24)):
            assert call(**bad) == _lib.ERANGE
        assert call(hidden=0) == 0
    assert rows(table=None) == _lib.EINVAL and gradient(grad=None) == _lib.EINVAL and rows(tokens=0) == 0 and gradient(words=0) == 0
    many, nbytes = dict(tokens=257), lib.mbx_embedding_gradient_scratch_bytes(257, 5, 8)      # fewer tokens need none
    assert gradient(**many) == _lib.ESCRATCH and gradient(**many, scratch=16, nbytes=nbytes - 1) == _lib.ESCRATCH and gradient(**many, scratch=8, nbytes=nbytes) == _lib.ESCRATCH
    assert lib.mbx_embedding_gradient_scratch_bytes(-1, 5, 8) == 0 and lib.mbx_embedding_gradient_scratch_bytes(256, 5, 8) == 0 and nbytes > 0


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize('padding', [-1, 2])
def test_batches_of_gradients_in_plain_operations(padding, dtype):
    """What a backward of several gradients at once computes, one gradient after the other: whole numbers, of which sums are exact."""
    from torch._vmap_internals import _vmap

    from megablocks_amd.ops import embed
    ids = torch.tensor([[1, 3, 3], [0, 2, -1], [5, 1, 2 ** 31 - 1]], dtype=torch.int32)
    grads, tables = torch.randint(-9, 10, (4, 3, 3, 8)).to(dtype), torch.randint(-9, 10, (4, 5, 8)).to(dtype)
    want = torch.zeros(4, 5, 8)
    for b in range(4):
        for i, word in enumerate(ids.flatten().tolist()):
            if 0 <= word < 5 and word != padding:
                want[b, word] += 2 * grads[b].view(9, 8)[i].float()
    got = _vmap(lambda g: embed._plain_table_gradient(g, ids, 5, 2.0, padding))(grads)
    assert got.dtype == dtype and torch.equal(got.float(), want)
    rows = _vmap(lambda t: embed._plain_rows(ids, t, 2.0))(tables)
    inside = (ids >= 0) & (ids < 5)
    assert rows.dtype == dtype and torch.equal(rows[:, inside], 2 * tables[:, ids[inside].long()]) and (rows[:, ~inside] == 0).all()
    assert embed._plain_rows(ids, tables[0, :0], 2.0).shape == (3, 3, 8) and embed._plain_table_gradient(grads[0], ids, 0, 2.0, -1).shape == (0, 8)


@pytest.mark.parametrize('scale', [1e39, -1e300, math.inf, -math.inf, math.nan])
def test_scales_that_are_not_finite_in_fp32(scale):
    """1e39 is a number as Python has it, and infinite as the library gets it: 0 times it would be none."""
    with pytest.raises(ValueError):
        ops.embedding(IDS, TABLE, scale)
    assert _lib.lib.mbx_embedding(16, 2, 3, 16, 0, 5, 8, scale, 16, None) == _lib.EINVAL
    assert _lib.lib.mbx_embedding_gradient(16, 16, 2, 3, 0, 5, 8, -1, scale, 16, None, 0, None) == _lib.EINVAL
