"""The layers with a choice of experts by scores, bias and groups and with 4-bit experts, as far as they go without a GPU."""
import pytest
import torch

from megablocks_amd.layers import moe as moe_layers
from megablocks_amd.layers.arguments import Arguments
from megablocks_amd.layers.dmoe import ParallelDroplessMLP
from megablocks_amd.layers.router import LearnedRouter


def _args(**changed):
    return Arguments(**(dict(hidden_size=16, ffn_hidden_size=32, moe_num_experts=8, moe_top_k=2, device=torch.device('cpu'), fp16=False, bf16=True) | changed))


def test_the_defaults_are_the_router_that_was_there():
    router = LearnedRouter(_args())
    assert not router._chooses and router.balance_bias is None and list(router.state_dict()) == ['layer.weight']
    assert not LearnedRouter(_args(moe_router_groups=4, moe_router_top_groups=4))._chooses      # all groups open
    for changed in (dict(moe_router_score='sigmoid'), dict(moe_router_bias=True), dict(moe_router_groups=4, moe_router_top_groups=2), dict(moe_router_scale=2.)):
        assert LearnedRouter(_args(**changed))._chooses


@pytest.mark.parametrize('changed', [
    dict(moe_router_score='tanh'), dict(moe_router_groups=3), dict(moe_router_groups=4, moe_router_top_groups=5), dict(moe_router_bias=True, moe_router_group_best=0),
    dict(moe_router_score='sigmoid', moe_top_k=9), dict(moe_router_scale=float('nan')), dict(moe_router_groups=8, moe_router_top_groups=1)])
def test_routers_that_cannot_choose_are_refused(changed):
    with pytest.raises(ValueError):
        LearnedRouter(_args(**changed))


def test_the_balance_bias_keeps_its_type():
    router = LearnedRouter(_args(moe_router_bias=True))
    assert sorted(router.state_dict()) == ['balance_bias', 'layer.weight'] and not router.balance_bias.requires_grad
    router.balance_bias += 0.0011
    router.half()
    assert router.layer.weight.dtype == torch.float16 and router.balance_bias.dtype == torch.float32 and float(router.balance_bias[0]) == pytest.approx(0.0011)
    with pytest.raises(RuntimeError):
        router(torch.zeros(3, 1, 16).half())       # the choice has one implementation, on the GPU


def test_updates_go_by_the_bias(monkeypatch):
    calls = []
    monkeypatch.setattr(moe_layers.ops, 'balance_bias', lambda biases, loads, rate, out: calls.append((biases, loads, rate, out)))
    a, b = torch.zeros(4), torch.zeros(4)
    for bias, load in ((a, [1, 2, 3, 4]), (b, [4, 3, 2, 1]), (a, [0, 0, 0, 8])):
        moe_layers.save_expert_load(bias, torch.tensor(load, dtype=torch.int32))
    assert len(moe_layers.get_expert_loads()) == 3
    moe_layers.update_balance_biases(_args(moe_router_bias_rate=0.5))
    (biases, loads, rate, out), = calls
    assert biases[0] is a and biases[1] is b and out is biases and rate == 0.5
    assert loads[0].tolist() == [[1, 2, 3, 4], [0, 0, 0, 8]] and loads[1].tolist() == [4, 3, 2, 1]
    assert moe_layers.get_expert_loads() == []


@pytest.mark.parametrize('changed', [dict(mlp_impl='sparse'), dict(activation_fn=torch.nn.functional.relu), dict(mlp_type='glu', activation_fn=torch.nn.functional.relu)])
def test_experts_that_have_no_4_bit_form_are_refused(changed):
    with pytest.raises(ValueError):
        ParallelDroplessMLP(_args(**changed)).quantize_experts_()
    with pytest.raises(RuntimeError):
        ParallelDroplessMLP(_args()).quantize_experts_()       # on the CPU


def _made(w, group, trans_b, zero_points):
    """quantize_4bit's weights in shape, all zeros, without a GPU."""
    from megablocks_amd import grouped_gemm_util as gg
    n, k = (w.shape[1], w.shape[2]) if trans_b else (w.shape[2], w.shape[1])
    shape = (w.shape[0], -(-n // 16), -(-k // 128) * 128 // group, 16)
    return gg.Weights4bit(torch.zeros(w.shape[0], -(-n // 16), -(-k // 128), 64, 4, dtype=torch.int32), torch.ones(shape, dtype=w.dtype),
                          torch.zeros(shape, dtype=torch.uint8) if zero_points else None, n, k, group, trans_b)


@pytest.mark.parametrize('name', ['forward', 'forward_tokens'])
def test_a_replaced_method_of_the_4_bit_experts_is_called(monkeypatch, name):
    """The call that does everything behind the router at once stands aside for it."""
    from megablocks_amd import grouped_gemm_util as gg
    from megablocks_amd.layers import mlp_4bit
    monkeypatch.setattr(mlp_4bit, 'quantize_4bit', _made)
    layer = ParallelDroplessMLP(_args()).quantize_experts_(32)
    monkeypatch.setattr(gg, 'experts_forward_4bit', lambda *a: 'by one call')
    x, weights, experts = torch.zeros(3, 16, dtype=torch.bfloat16), torch.ones(6, dtype=torch.bfloat16), torch.zeros(6, dtype=torch.int32)
    with torch.no_grad():
        assert layer._one_call_forward(x, weights, experts) == 'by one call'
        setattr(layer.mlp, name, lambda *a: None)
        assert layer._one_call_forward(x, weights, experts) is None


@pytest.mark.parametrize('changed', [dict(zero_points=False), dict(zero_points=True)])
def test_4_bit_experts_go_by_the_buffers_there_are(monkeypatch, changed):
    """Buffers that a call or an assignment puts in the place of others are the ones multiplied by."""
    from megablocks_amd import grouped_gemm_util as gg
    from megablocks_amd.layers import mlp_4bit
    monkeypatch.setattr(mlp_4bit, 'quantize_4bit', _made)
    experts = ParallelDroplessMLP(_args(mlp_type='glu', activation_fn=torch.nn.functional.silu)).quantize_experts_(32, **changed).mlp
    seen = []
    monkeypatch.setattr(gg, 'gmm_4bit_act', lambda x, b, act, *sizes, b2=None: (seen.append((b, b2)), x)[1])
    monkeypatch.setattr(gg, 'gmm_4bit', lambda x, b, *sizes: (seen.append(b), x)[1])
    x, sizes = torch.zeros(2, 16, dtype=torch.bfloat16), torch.tensor([2] + [0] * 7)

    def used():
        (w1, v1), w2 = seen[-2:]
        return {f'{name}_{part}': getattr(w, part) for name, w in (('w1', w1), ('v1', v1), ('w2', w2)) for part in ('words', 'scales', 'zeros')}
    experts(x, sizes)
    first = dict(experts.named_buffers())
    assert all(t is first.get(name) for name, t in used().items())
    others = {name: t.clone() for name, t in first.items()}
    for name in others:                                    # one at a time, and all
        torch.func.functional_call(experts, {name: others[name]}, (x, sizes))
        assert all(t is (others if name == at else first).get(at) for at, t in used().items())
    torch.func.functional_call(experts, others, (x, sizes))
    assert all(t is others.get(name) for name, t in used().items())
    experts(x, sizes)
    assert all(t is first.get(name) for name, t in used().items())
    for name in others:
        setattr(experts, name, others[name])
        experts(x, sizes)
        assert used()[name] is others[name] is dict(experts.named_buffers())[name]
    experts.w1_scales = torch.ones(3, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        experts(x, sizes)                                  # that do not fit


def test_routers_made_without_the_choice_route_as_before():
    """A router of a class with an __init__ of its own, or pickled before there was a choice: softmax and top-k, casts and moves too."""
    class Own(LearnedRouter):

        def __init__(self, args):
            torch.nn.Module.__init__(self)
            self.args, self.layer = args, torch.nn.Linear(args.hidden_size, args.moe_num_experts, bias=False, dtype=torch.bfloat16)
    args = _args()
    own, plain = Own(args), LearnedRouter(args)
    x = torch.randn(5, 1, 16).bfloat16()
    with torch.no_grad():
        own.layer.weight.copy_(plain.layer.weight)
        assert all(torch.equal(a, b) for a, b in zip(own(x), plain(x)))
        assert own.float().layer.weight.dtype == torch.float32 and own(x.float())[0].shape == (5, 8)
