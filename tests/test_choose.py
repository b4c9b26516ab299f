"""What the choice of experts and the update of their bias refuse, and the restatement they are held to, without a GPU."""
import pytest
import torch

import megablocks_amd.ops as ops
from megablocks_amd import _lib
from oracle import choose as oracle


@pytest.mark.parametrize('changed', [
    dict(score='tanh'), dict(groups=3), dict(groups=0), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(group_best=3), dict(top_k=0),
    dict(top_k=17), dict(groups=4, top_groups=1, top_k=5), dict(norm_p=-1), dict(norm_p=float('nan')), dict(norm_p=float('inf')), dict(scale=float('inf')),
    dict(scale=float('nan')), dict(bias=torch.zeros(15)), dict(bias=torch.zeros(1, 16)), dict(logits=torch.zeros(16)), dict(logits=torch.zeros(2, 4, 16)),
    dict(logits=torch.zeros(2, 1024)), dict(logits=torch.zeros(2, 512), top_k=65), dict(logits=torch.zeros(2, 512), groups=128, top_groups=128)])
def test_choices_that_are_none_are_refused(changed):
    call = dict(logits=torch.zeros(2, 16), top_k=2) | changed
    with pytest.raises(ValueError):
        ops.choose_experts(**call)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError):
        ops.choose_experts(torch.zeros(2, 16), 2)
    with pytest.raises(RuntimeError):
        ops.balance_bias([torch.zeros(4)], [torch.zeros(4, dtype=torch.int32)], 0.001)


@pytest.mark.parametrize('biases,counts,out', [
    ([torch.zeros(4)], [], None), ([torch.zeros(4), torch.zeros(5)], [torch.zeros(4).int(), torch.zeros(5).int()], None),
    ([torch.zeros(4)], [torch.zeros(5).int()], None), ([torch.zeros(2, 2)], [torch.zeros(4).int()], None), ([torch.zeros(4)], [torch.zeros(4).int()], []),
    ([torch.zeros(4)], [torch.zeros(2, 2, 4).int()], None), ([torch.zeros(4)], [torch.zeros(4).int()], [torch.zeros(3)])])
def test_updates_that_do_not_fit_are_refused(biases, counts, out):
    with pytest.raises(ValueError):
        ops.balance_bias(biases, counts, 0.001, out=out)


def test_updates_of_other_types_are_refused():
    with pytest.raises(RuntimeError):
        ops.balance_bias([torch.zeros(4).half()], [torch.zeros(4).int()], 0.001)
    with pytest.raises(RuntimeError):
        ops.balance_bias([torch.zeros(4)], [torch.zeros(4)], 0.001)
    with pytest.raises(ValueError):
        ops.balance_bias([torch.zeros(4)], [torch.zeros(4).int()], float('nan'))
    assert ops.balance_bias([], [], 0.001) == []


def test_entry_points_refuse_without_touching_the_gpu():
    lib = _lib.lib

    def choose(dtype=0, tokens=2, experts=16, top_k=2, score=0, groups=1, top_groups=1, best=1, p=0., scale=1., logits=None):
        return lib.mbx_choose_experts(logits, dtype, tokens, experts, top_k, score, None, groups, top_groups, best, p, scale, None, None, None, None, None, None)
    for bad in (dict(dtype=3), dict(tokens=-1), dict(experts=0), dict(top_k=0), dict(top_k=17), dict(score=2), dict(groups=3), dict(groups=4, top_groups=5),
                dict(best=0), dict(p=-1.), dict(p=float('inf')), dict(scale=float('nan')), dict(groups=8, top_groups=1, top_k=3), {}):
        assert choose(**bad) == _lib.EINVAL      # the last: no logits
    assert choose(experts=513) == _lib.EUNSUPPORTED and choose(experts=130, top_k=65) == _lib.EUNSUPPORTED
    assert choose(experts=130, groups=65, top_groups=65) == _lib.EUNSUPPORTED
    assert choose(tokens=0) == 0
    assert lib.mbx_choose_experts_backward(None, None, None, None, None, 0, 0, 16, 2, 0, 0., 1., None, None) == 0
    assert lib.mbx_choose_experts_backward(None, None, None, None, None, 0, 2, 16, 2, 0, 0., 1., None, None) == _lib.EINVAL
    assert lib.mbx_balance_bias(None, None, None, None, 0, 16, 0.1, None) == 0
    assert lib.mbx_balance_bias(None, None, None, None, 1, 16, 0.1, None) == _lib.EINVAL
    assert lib.mbx_balance_bias(None, None, None, None, 1, 0, 0.1, None) == _lib.EINVAL


def test_the_restatement_orders_and_differentiates():
    """Ties to the lower index, NaN first, and the formula's gradient against differences."""
    nan = float('nan')
    assert oracle.best([1., 3., 3., nan, 2.], 4) == [3, 1, 2, 4]
    assert oracle.best([-float('inf')] * 3, 2) == [0, 1]
    g = torch.Generator().manual_seed(3)
    x, gs, gw, gl = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 8), (3, 8), (3, 3), (3,)))
    for score in ('softmax', 'sigmoid'):
        for p in (0, 1, 2, 3):
            _, _, idx, _ = oracle.choose(x, 3, score, groups=4, top_groups=3, norm_p=p, scale=1.5)

            def loss(x):
                s, w, i, lse = oracle.choose(x, 3, score, groups=4, top_groups=3, norm_p=p, scale=1.5)
                assert torch.equal(i, idx)
                return (s * gs).sum() + (w * gw).sum() + (lse * gl).sum()
            got, _ = oracle.gradient(x, idx, score, p, 1.5, gs, gw, gl)
            for t, e in ((0, 0), (1, 5), (2, 7), (2, int(idx[2, 0]))):
                d = torch.zeros_like(x)
                d[t, e] = 1e-6
                assert abs(float((loss(x + d) - loss(x - d)) / 2e-6) - float(got[t, e])) < 1e-7


def test_outputs_of_layers_in_each_others_way():
    from megablocks_amd.ops import choose
    for outputs, biases in (([64, 128], [64, 128]), ([0, 64, 128], [256, 320, 384]), ([0], [0]), ([64, 192], [64, 128]), ([0, 64], [200, 264])):
        choose._check_outputs(outputs, biases, 64)
    for outputs, biases in (([64, 64], [64, 64]), ([64, 100], [64, 100]), ([128, 64], [64, 128]), ([0, 64], [64, 256]), ([0, 64], [256, 127]), ([32], [0]), ([0], [63])):
        with pytest.raises(ValueError):
            choose._check_outputs(outputs, biases, 64)
