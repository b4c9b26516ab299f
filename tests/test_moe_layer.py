"""What the layer for a few tokens refuses, without a GPU."""
import ctypes
import math

import pytest
import torch

import megablocks_amd.ops as ops
from megablocks_amd import _lib
from megablocks_amd.layers.arguments import Arguments
from megablocks_amd.layers.dmoe import dMoE
from megablocks_amd.ops import few_tokens

W = torch.zeros(4, 16, 8, dtype=torch.bfloat16)
CALL = dict(x=torch.zeros(2, 8, dtype=torch.bfloat16), router=torch.zeros(4, 8, dtype=torch.bfloat16), w1=W, v1=W, w2=W, top_k=2, act=0)


@pytest.mark.parametrize('changed', [
    dict(x=torch.zeros(2, 16)), dict(x=torch.zeros(8)), dict(x=torch.zeros(1, 2, 8)), dict(x=torch.zeros(65, 8)), dict(router=torch.zeros(5, 8)), dict(router=torch.zeros(4, 9)),
    dict(w1=torch.zeros(64, 8)), dict(w1=torch.zeros(4, 24, 8)), dict(v1=torch.zeros(4, 24, 8)), dict(w2=torch.zeros(4, 8, 16)), dict(act=2), dict(act=-1), dict(top_k=0), dict(top_k=5),
    dict(score='tanh'), dict(groups=3), dict(groups=4, top_groups=1), dict(group_best=3), dict(norm_p=-1), dict(norm_p=math.inf), dict(scale=math.nan), dict(bias=torch.zeros(5)),
    dict(bias=torch.zeros(1, 4)), dict(x=torch.zeros(2, 12), router=torch.zeros(4, 12), w1=torch.zeros(4, 16, 12), v1=None, w2=torch.zeros(4, 16, 12)),
    dict(w1=torch.zeros(4, 12, 8), v1=None, w2=torch.zeros(4, 12, 8)), dict(w1=torch.zeros(4, 0, 8), v1=None, w2=torch.zeros(4, 0, 8)),
    dict(x=torch.zeros(2, 8), router=torch.zeros(32, 8), w1=torch.zeros(32, 8, 8), v1=None, w2=torch.zeros(32, 8, 8), top_k=17),
    dict(router=torch.zeros(600, 8), w1=torch.zeros(600, 8, 8), v1=None, w2=torch.zeros(600, 8, 8))])
def test_calls_that_are_none_are_refused(changed):
    with pytest.raises(ValueError):
        ops.moe_layer(**(CALL | changed))


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError):
        ops.moe_layer(**CALL)


@pytest.mark.parametrize('sizes,taken', [
    ((1, 8, 8, 1, 1), True), ((64, 4096, 14336, 8, 2), True), ((65, 8, 8, 1, 1), False), ((1, 8, 8, 512, 16), True), ((1, 8, 8, 513, 1), False), ((1, 8, 8, 32, 17), False),
    ((1, 8, 8, 4, 5), False), ((1, 12, 8, 4, 1), False), ((1, 8, 12, 4, 1), False), ((1, 0, 8, 4, 1), False), ((1, 32768, 32704, 4, 1), False), ((1, 32768, 32640, 4, 1), True),
    ((1, 16, 1 << 26, 4, 1), False), ((1, 960 * 128, 64, 4, 1), True), ((1, 960 * 128 + 8, 64, 4, 1), False), ((64, 32768, 8, 16, 16), False), ((64, 8192, 8, 16, 16), True)])
def test_sizes_that_are_taken(sizes, taken):
    """Offsets that the kernels keep in 32 bits, and the counters of the workspace."""
    assert few_tokens.takes(*sizes) == taken


def test_entry_point_refuses_without_touching_the_gpu():
    lib = _lib.lib

    def call(tokens=2, hidden=8, dtype=0, experts=4, top_k=2, score=0, groups=1, top_groups=1, best=2, p=0., scale=1., ffn=16, act=0, x=16, w=16, out=16, scratch=None, nbytes=0,
             workspace=None, workspace_bytes=0):
        return lib.mbx_moe_layer(x, tokens, hidden, dtype, w, experts, top_k, score, None, groups, top_groups, best, p, scale, w, w, w, ffn, act, out, 16, 16, scratch, nbytes,
                                 workspace, workspace_bytes, None)
    for bad in (dict(tokens=-1), dict(hidden=-8), dict(ffn=-8), dict(experts=0), dict(top_k=0), dict(top_k=5), dict(score=2), dict(groups=3), dict(groups=4, top_groups=1),
                dict(groups=2, top_groups=3), dict(best=0), dict(p=-1.), dict(p=math.inf), dict(p=math.nan), dict(scale=math.inf), dict(act=2), dict(x=None), dict(w=None), dict(out=None)):
        assert call(**bad) == _lib.EINVAL
    for bad in (dict(tokens=65), dict(hidden=12), dict(ffn=12), dict(hidden=0), dict(dtype=2), dict(experts=513), dict(experts=40, top_k=17), dict(x=8), dict(w=24), dict(out=18),
                dict(experts=65, groups=65, top_groups=65)):
        assert call(**bad) == _lib.EUNSUPPORTED
    assert call(tokens=0) == 0
    nbytes = lib.mbx_moe_layer_scratch_bytes(2, 8, 16, 4, 2, 1)
    assert call() == _lib.ESCRATCH and call(scratch=16, nbytes=nbytes - 1, workspace=16, workspace_bytes=4096) == _lib.ESCRATCH
    assert call(scratch=16, nbytes=nbytes) == _lib.ESCRATCH and call(scratch=16, nbytes=nbytes, workspace=16, workspace_bytes=4095) == _lib.ESCRATCH
    assert call(scratch=8, nbytes=nbytes, workspace=16, workspace_bytes=4096) == _lib.ESCRATCH


@pytest.mark.parametrize('tokens', [-1, 65])
def test_arguments_refuse_other_numbers_of_tokens(tokens):
    with pytest.raises(ValueError):
        Arguments(device=torch.device('cpu'), moe_fused_tokens=tokens)


@pytest.mark.parametrize('sizes,taken', [((64, 8, 1 << 22, 64, 1), False), ((63, 8, 1 << 22, 64, 1), True), ((64, 8, 1 << 22, 63, 1), True), ((32, 16, 1 << 22, 128, 2), False)])
def test_a_launch_has_fewer_than_2_to_the_32_threads(sizes, taken):
    """256 of them for 16 rows of the weights of an expert that a token may choose."""
    assert few_tokens.takes(*sizes) == taken


class Known(torch.nn.Module):
    """A router's or experts' stand-in: no arguments, a result that tells it."""

    def __init__(self, result):
        super().__init__()
        self.result = result

    def forward(self, *given):
        return self.result


@pytest.mark.parametrize('recorded', [True, False])
@pytest.mark.parametrize('tokens', [0, 16])
def test_layers_whose_experts_have_no_arguments(tokens, recorded):
    layer = dMoE(Arguments(device=torch.device('cpu'), hidden_size=16, ffn_hidden_size=32, moe_num_experts=4, moe_fused_tokens=tokens, mlp_impl='grouped', bf16=False, fp16=False))
    layer.router, layer.experts = Known((None, None, torch.zeros(2, 1, dtype=torch.int64))), Known('experts')
    with torch.set_grad_enabled(recorded):
        for training in (True, False):
            layer.train(training)
            assert layer(torch.randn(2, 1, 16)) == 'experts'


def test_arguments_without_a_number_of_fused_tokens():
    class Few:
        """Some other object that holds the layer's arguments."""
    args = Arguments(device=torch.device('cpu'), hidden_size=16, ffn_hidden_size=32, moe_num_experts=4, mlp_impl='grouped', bf16=False, fp16=False)
    layer = dMoE(args).eval()
    layer.experts.args = Few()
    layer.experts.args.__dict__.update({name: value for name, value in vars(args).items() if name != 'moe_fused_tokens'})
    with torch.no_grad():
        assert layer._few_tokens(torch.randn(2, 1, 16)) is None


# Layers that are computed in every way there is, and end inside of tiles: (tokens, hidden, ffn, experts, top_k), gate -> weight fragments of a workgroup of the first product, row
# tiles, parts of the second product's reduction, whether its tiles are neighbours on an XCD
PLANS = [
    ((64, 136, 2056, 8, 2), True, (8, 2, 8, 1)), ((64, 136, 4104, 8, 2), False, (8, 2, 16, 1)), ((48, 72, 8200, 2, 1), True, (8, 4, 16, 1)), ((48, 72, 16392, 2, 1), False, (8, 4, 16, 1)),
    ((1, 4096, 8200, 3, 2), True, (4, 1, 4, 0)), ((1, 4096, 16392, 3, 2), False, (4, 1, 4, 0)), ((20, 4096, 4104, 4, 2), True, (4, 2, 2, 0)), ((20, 4096, 8200, 4, 2), False, (4, 2, 2, 0)),
    ((1, 72, 4104, 8, 4), False, (2, 1, 16, 1)), ((64, 136, 2056, 8, 2), False, (2, 2, 8, 1)), ((48, 72, 8200, 2, 1), False, (2, 4, 16, 1)),
    ((5, 1032, 1064, 60, 4), True, (2, 1, 2, 1)), ((17, 200, 520, 4, 2), True, (2, 2, 2, 0)), ((40, 200, 200, 2, 1), True, (2, 4, 1, 0)), ((33, 2056, 264, 64, 6), True, (2, 1, 1, 1)),
    ((30, 1160, 40, 64, 16), True, (2, 1, 1, 1)), ((60, 1160, 40, 64, 16), True, (2, 2, 1, 1)), ((50, 1032, 40, 32, 16), True, (2, 4, 1, 1)),
    ((2, 264, 200, 5, 2), False, (1, 1, 1, 0)), ((16, 264, 200, 5, 2), False, (1, 1, 1, 0)), ((30, 264, 200, 4, 2), False, (1, 2, 1, 0)), ((60, 264, 200, 3, 2), False, (1, 4, 1, 0))]


def plan_of(sizes, gate):
    plan = (ctypes.c_int * 4)()
    assert _lib.lib.mbx_debug_moe_layer_plan(*map(ctypes.c_int64, sizes[:3]), *sizes[3:], gate, plan) == 0
    return tuple(plan)


def test_layers_are_computed_in_every_way_there_is():
    for sizes, gate, plan in PLANS:
        assert plan_of(sizes, gate) == plan, sizes
    products = {(gate, *plan[:2]) for _, gate, plan in PLANS}
    # eight fragments are for 12 rows an expert and more, four for fewer, one for layers without a gate
    assert products == {(gate, n, r) for gate in (True, False) for n, r in ((8, 2), (8, 4), (4, 1), (4, 2), (2, 1), (2, 2), (2, 4))} | {(False, 1, r) for r in (1, 2, 4)}
    assert {plan[1:] for _, _, plan in PLANS} >= {(r, 1, x) for r in (1, 2, 4) for x in (0, 1)} | {(1, 2, 1), (2, 8, 1), (4, 16, 1), (1, 4, 0), (2, 2, 0)}


@pytest.mark.parametrize('tokens,ffn,experts,top_k,gate,fours', [(1, 8192, 4, 2, True, [4096]), (8, 2048, 32, 4, True, [4096]), (1, 16384, 4, 2, False, [4096, 8192, 16384])])
def test_rows_that_come_faster_in_fours(tokens, ffn, experts, top_k, gate, fours):
    """Measured up to 10 % shorter with two weight fragments of a workgroup for all other rows."""
    for hidden in (1024, 2048, 3584, 4032, 4096, 4160, 4608, 5120, 6144, 8192, 8256, 10240, 12288, 16384):
        assert plan_of((tokens, hidden, ffn, experts, top_k), gate)[0] == (4 if hidden in fours else 2), hidden
