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
