"""dMoE layers whose experts are chosen by scores, a balance bias and groups, in training, and with experts of 4-bit weights, in serving, against the
oracle in fp32.  Tolerance: relative Frobenius error 1e-2 for 16-bit layers, as for the others (tests/test_layers_gpu.py)."""
import copy

import pytest
import torch
import torch.nn.functional as F

import oracle
from megablocks_amd import grouped_gemm_util as gg
from megablocks_amd import ops
from megablocks_amd.layers import moe as moe_layers
from megablocks_amd.layers import router as router_layers
from megablocks_amd.layers.arguments import Arguments
from megablocks_amd.layers.dmoe import dMoE
from megablocks_amd.layers.moe import MoE

pytestmark = pytest.mark.gpu


def rel_err(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-30))


def _args(**changed):
    return Arguments(**(dict(hidden_size=256, ffn_hidden_size=512, moe_num_experts=16, moe_top_k=4, mlp_type='glu', activation_fn=F.silu, fp16=False, bf16=True,
                             bias=False, moe_loss_weight=0, moe_normalize_expert_weights=1, init_method=lambda w: torch.nn.init.normal_(w, std=0.1),
                             output_layer_init_method=lambda w: torch.nn.init.normal_(w, std=0.1)) | changed))


CHOICES = [dict(moe_router_score='sigmoid', moe_router_bias=True, moe_router_groups=4, moe_router_top_groups=2, moe_router_scale=2.5),
           dict(moe_router_groups=8, moe_router_top_groups=3, moe_router_group_best=1), dict(moe_router_score='sigmoid', moe_normalize_expert_weights=None)]


def _reference(layer, args, x, chosen):
    """The layer in fp32 on the CPU, given the experts chosen; leaves and output."""
    mlp, leaves = layer.experts.mlp, {}
    for name, t in (('x', x.view(-1, x.shape[-1])), ('router', layer.router.layer.weight), ('w1', mlp.w1), ('v1', getattr(mlp, 'v1', None)), ('w2', mlp.w2)):
        leaves[name] = None if t is None else t.detach().float().cpu().requires_grad_()
    logits = leaves['x'] @ leaves['router'].t()
    scores = torch.sigmoid(logits) if args.moe_router_score == 'sigmoid' else logits.softmax(1)
    w = scores.gather(1, chosen.cpu())
    if args.moe_normalize_expert_weights:
        w = w / w.sum(1, keepdim=True)
    out, _ = oracle.dmoe_forward(leaves['x'], w * args.moe_router_scale, chosen.cpu(), leaves['w1'], leaves['w2'], leaves['v1'], num_experts=args.moe_num_experts,
                                 top_k=args.moe_top_k, activation=args.activation_fn if leaves['v1'] is not None else None)
    return leaves, out


@pytest.mark.parametrize('choice', CHOICES)
@pytest.mark.parametrize('tokens,mlp_type,mlp_impl', [(1500, 'glu', 'grouped'), (77, 'mlp', 'grouped'), (300, 'glu', 'sparse')])
def test_training_step(tokens, mlp_type, mlp_impl, choice):
    torch.manual_seed(tokens)
    changed = dict(mlp_type=mlp_type, mlp_impl=mlp_impl, **choice) | ({} if mlp_type == 'glu' else dict(activation_fn=Arguments().activation_fn))
    args = _args(**changed)
    layer = dMoE(args)
    if args.moe_router_bias:
        layer.router.balance_bias.copy_(torch.randint(-40, 41, (16,)) * 0.01)
    x = torch.randn(tokens, 1, 256, device='cuda').bfloat16().requires_grad_()
    grad = torch.randn(tokens, 1, 256, device='cuda').bfloat16()
    moe_layers.clear_expert_loads()
    out = layer(x)
    moe_layers.clear_expert_loads()
    out.backward(grad)
    with torch.no_grad():
        logits = F.linear(x.view(tokens, 256), layer.router.layer.weight)
        scores, weights, chosen = layer.router(x)
        want = ops.choose_experts(logits, 4, score=args.moe_router_score, bias=layer.router.balance_bias, groups=args.moe_router_groups,
                                  top_groups=args.moe_router_top_groups, group_best=args.moe_router_group_best, norm_p=args.moe_normalize_expert_weights or 0,
                                  scale=args.moe_router_scale)
    if tokens > 256:      # few tokens go through a kernel that sums the logits in another order
        assert all(torch.equal(a, b) for a, b in zip((scores, weights, chosen), want))
    leaves, ref = _reference(layer, args, x, chosen)
    ref.backward(grad.view(tokens, 256).float().cpu())
    assert rel_err(out.view(tokens, 256), ref) < 1e-2
    mlp = layer.experts.mlp
    for got, name in ((x.grad.view(tokens, 256), 'x'), (mlp.w1.grad, 'w1'), (mlp.w2.grad, 'w2')):
        assert rel_err(got, leaves[name].grad) < 1e-2, name
    assert rel_err(layer.router.layer.weight.grad, leaves['router'].grad) < 5e-2     # a sum of many that nearly cancel, as in tests/test_layers_gpu.py


def test_balance_over_steps():
    """Three steps of training with accumulated gradients, two layers: every update is that of the tokens the experts got; the capacity layer too."""
    torch.manual_seed(1)
    args = _args(moe_router_score='sigmoid', moe_router_bias=True, moe_router_bias_rate=0.01, num_layers=2, moe_loss_weight=0.01, moe_lbl_in_fp32=True)
    layers = [dMoE(args), MoE(args)]
    moe_layers.clear_expert_loads()
    moe_layers.clear_load_balancing_loss()
    for step in range(3):
        counts = [torch.zeros(16, dtype=torch.int64) for _ in layers]
        before = [layer.router.balance_bias.clone() for layer in layers]
        for _ in range(2):
            x = torch.randn(200, 1, 256, device='cuda').bfloat16().requires_grad_()
            out = x
            for layer, count in zip(layers, counts):
                with torch.no_grad():
                    count += torch.bincount(layer.router(out)[2].flatten().cpu(), minlength=16)
                out = layer(out)
            (out.float().square().mean() + moe_layers.batched_load_balancing_loss(args)).backward()
            moe_layers.clear_load_balancing_loss()
        assert len(moe_layers.get_expert_loads()) == 4
        moe_layers.update_balance_biases(args)
        for layer, b, count in zip(layers, before, counts):
            want = b.cpu().double() + 0.01 * torch.sign(count.sum() - 16 * count).double()
            assert (layer.router.balance_bias.cpu().double() - want).abs().max() < 1e-8 + 2.0 ** -24
            assert not torch.equal(layer.router.balance_bias, b)
    with torch.no_grad():
        layers[0](x)
    layers[0].eval()(x)
    assert moe_layers.get_expert_loads() == []          # evaluation counts nothing


def test_layers_of_different_numbers_of_experts_are_balanced_together():
    torch.manual_seed(2)
    layers = [dMoE(_args(moe_router_score='sigmoid', moe_router_bias=True, moe_router_bias_rate=0.01, moe_num_experts=e)) for e in (16, 8, 16)]
    moe_layers.clear_expert_loads()
    out = torch.randn(100, 1, 256, device='cuda').bfloat16().requires_grad_()
    for layer in layers:
        out = layer(out)
    loads = [(b, n.clone()) for b, n in moe_layers.get_expert_loads()]
    moe_layers.update_balance_biases(layers[0].router.args)
    assert [b.numel() for b, _ in loads] == [16, 8, 16] and moe_layers.get_expert_loads() == []
    for b, n in loads:
        assert torch.allclose(b, 0.01 * torch.sign(n.sum() - n.numel() * n).float(), atol=1e-8)


def test_4_bit_experts_of_padded_rows():
    """Gathered rows that are padded for each expert, as the block-sparse layer has them: both products by the padded bins."""
    _, kept = _quantized(_args(moe_num_experts=3, moe_top_k=1), 64, False)
    mlp = kept.experts.mlp
    x = torch.randn(9, 256, device='cuda').bfloat16()
    ids = torch.tensor([2, 0, 0, 2, 2, 1, 0, 2, 2], device='cuda')
    bin_ids, indices = ids.sort(stable=True)
    bins = torch.bincount(ids, minlength=3).cumsum(0).int()
    padded = torch.tensor([16, 32, 48], dtype=torch.int32, device='cuda')
    with torch.no_grad():
        out = mlp.forward_tokens(gg.GatheredRows(x, indices.int(), bin_ids.int(), bins, padded, 1, 48), None)
        want = mlp(x[indices], torch.bincount(ids, minlength=3))
    at = torch.cat([torch.arange(3), 16 + torch.arange(1), 32 + torch.arange(5)])
    assert out.shape == (48, 256) and torch.equal(out[at.cuda()], want) and int((out != 0).any(1).sum()) == 9


def test_other_scores_leave_auxiliary_losses_and_checkpoints_alone():
    """z-loss and load-balancing loss with sigmoid scores; a copy through a state_dict routes alike."""
    torch.manual_seed(2)
    args = _args(moe_router_score='sigmoid', moe_router_bias=True, moe_loss_weight=0.01, moe_zloss_weight=0.001, moe_lbl_in_fp32=True, moe_zloss_in_fp32=True)
    layer, other = dMoE(args), dMoE(args)
    layer.router.balance_bias.uniform_(-0.1, 0.1)
    other.load_state_dict(layer.state_dict())
    x = torch.randn(400, 1, 256, device='cuda').bfloat16().requires_grad_()
    for clear in (moe_layers.clear_load_balancing_loss, router_layers.clear_router_zloss, moe_layers.clear_expert_loads):
        clear()
    out = layer(x)
    logits = F.linear(x.view(400, 256), layer.router.layer.weight).float()
    zloss = router_layers.batched_router_zloss(args).sum()
    assert abs(float(zloss.detach()) - 0.001 * float(torch.logsumexp(logits.detach(), 1).square().mean())) < 1e-5
    lbl = moe_layers.batched_load_balancing_loss(args)
    chosen = layer.router(x)[2]
    count = torch.bincount(chosen.flatten(), minlength=16).float()
    want = 16 * 0.01 / (400 * 4) * (count * torch.sigmoid(logits).mean(0)).sum()
    assert abs(float(lbl.detach()) - float(want)) < 4e-3 * float(want)      # scores are rounded to bf16
    (lbl + zloss).backward()
    assert layer.router.layer.weight.grad.isfinite().all() and layer.router.layer.weight.grad.abs().sum() > 0
    assert torch.equal(other.router(x)[2], chosen)
    for clear in (moe_layers.clear_load_balancing_loss, router_layers.clear_router_zloss, moe_layers.clear_expert_loads):
        clear()
    del out


def test_training_step_replays_from_a_captured_graph():
    torch.manual_seed(3)
    args = _args(**CHOICES[0])
    layer = dMoE(args)
    layer.router.balance_bias.uniform_(-0.1, 0.1)
    params = list(layer.parameters())
    static, grad = torch.randn(600, 1, 256, device='cuda').bfloat16().requires_grad_(), torch.randn(600, 1, 256, device='cuda').bfloat16()

    def step(x):
        out = layer(x)
        return (out.detach(), *torch.autograd.grad(out, [x, *params], grad))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    moe_layers.clear_expert_loads()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
        moe_layers.update_balance_biases(args)
    for seed in range(3):
        x = torch.randn(600, 1, 256, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        before = layer.router.balance_bias.clone()
        want = step(x.clone().requires_grad_())
        moe_layers.update_balance_biases(args)
        after = layer.router.balance_bias.clone()
        with torch.no_grad():
            static.copy_(x)
            layer.router.balance_bias.copy_(before)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)) and torch.equal(layer.router.balance_bias, after)


def _quantized(args, group, zeros, seed=5):
    torch.manual_seed(seed)
    layer = dMoE(args).eval()
    kept = copy.deepcopy(layer).quantize_experts_(group, zeros)
    with torch.no_grad():      # the reference's experts have the values the codes stand for
        for name in ('w1', 'v1', 'w2'):
            if hasattr(layer.experts.mlp, name):
                w = getattr(layer.experts.mlp, name)
                w.copy_(getattr(kept.experts.mlp, name).dequantize(torch.float32, None).view(w.shape))
    return layer, kept


@pytest.mark.parametrize('tokens', [1, 7, 60, 900, 2500])
@pytest.mark.parametrize('group,zeros', [(128, False), (32, True)])
@pytest.mark.parametrize('changed', [dict(CHOICES[0]), dict(mlp_type='mlp', activation_fn=None), dict(moe_num_experts=4, moe_top_k=1, hidden_size=136, ffn_hidden_size=200)])
def test_serving_with_4_bit_experts(monkeypatch, changed, group, zeros, tokens):
    changed = dict(changed) if changed.get('mlp_type') != 'mlp' else dict(mlp_type='mlp', activation_fn=Arguments().activation_fn)
    args = _args(**changed)
    layer, kept = _quantized(args, group, zeros)
    x = torch.randn(tokens, 1, args.hidden_size, generator=torch.Generator().manual_seed(tokens)).bfloat16().cuda()
    print(f'4-bit layer {changed} {group} {zeros} {tokens}', flush=True)
    with torch.no_grad():
        out, chosen = kept(x), kept.router(x)[2]
        _, want = _reference(layer, args, x, chosen)
        assert rel_err(out.view(tokens, -1), want) < 1e-2
        # by the separate calls: the same where those multiply the codes too
        monkeypatch.setattr(gg, 'experts_forward_4bit', lambda *a: None)
        again = kept(x)
        assert torch.equal(again, out)
        monkeypatch.setattr(gg, 'FUSED_GATHER', '0')
        assert torch.equal(kept(x), out) or tokens > 200


@pytest.mark.parametrize('tokens', [7, 900, 2500])
@pytest.mark.parametrize('changed', [CHOICES[0], dict(mlp_type='mlp', moe_num_experts=4, moe_top_k=1, hidden_size=136, ffn_hidden_size=200)])
def test_4_bit_experts_by_gathered_rows_and_by_copies_of_them(monkeypatch, changed, tokens):
    """The rows read through their assignments or from a gathered copy are the same rows, in every kernel."""
    args = _args(**changed, **(dict(activation_fn=Arguments().activation_fn) if 'mlp_type' in changed else {}))
    _, kept = _quantized(args, 32, True)
    x = torch.randn(tokens, 1, args.hidden_size, generator=torch.Generator().manual_seed(tokens)).bfloat16().cuda()
    monkeypatch.setattr(gg, 'experts_forward_4bit', lambda *a: None)
    with torch.no_grad():
        monkeypatch.setattr(gg, 'FUSED_GATHER', '1')
        want = kept(x)
        monkeypatch.setattr(gg, 'FUSED_GATHER', '0')
        assert torch.equal(kept(x), want)


def test_4_bit_experts_are_kept_moved_and_cast():
    args = _args()
    _, kept = _quantized(args, 64, True)
    x = torch.randn(9, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        want = kept(x)
        state = kept.state_dict()
        assert {'experts.mlp.w1_words', 'experts.mlp.v1_scales', 'experts.mlp.w2_zeros'} <= set(state) and not any(k.endswith('mlp.w1') for k in state)
        _, other = _quantized(args, 64, True, seed=6)
        assert not torch.equal(other(x), want)
        other.load_state_dict(state)
        assert torch.equal(other(x), want)
        _, other = _quantized(args, 64, True, seed=7)
        other.load_state_dict({k: v.clone() for k, v in state.items()}, assign=True)
        assert torch.equal(other(x), want)
        assert torch.equal(copy.deepcopy(kept)(x), want) and torch.equal(kept.cpu().cuda()(x), want)
        assert rel_err(kept.half()(x.half()), want) < 1e-2
    y = x.half().requires_grad_()
    with pytest.raises(RuntimeError):
        kept(y)                                        # no gradients
    with pytest.raises(ValueError):
        kept.quantize_experts_()                       # they are already


def test_4_bit_experts_of_fp32_weights_under_autocast():
    args = _args(fp16=False, bf16=False)
    layer, kept = _quantized(args, 128, False)
    x = torch.randn(20, 1, 256, device='cuda')
    with torch.no_grad(), torch.autocast('cuda', torch.bfloat16):
        out, chosen = kept(x), kept.router(x.bfloat16())[2]
    assert out.dtype == torch.bfloat16
    _, want = _reference(layer, args, x, chosen)
    assert rel_err(out.view(20, -1), want) < 1e-2


def test_decoding_replays_from_a_captured_graph():
    """The router's choice and the 4-bit experts of a few tokens together, captured and replayed next to eager passes."""
    args = _args(**CHOICES[0])
    _, kept = _quantized(args, 128, False)
    kept.router.balance_bias.uniform_(-0.1, 0.1)
    static = torch.randn(6, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        kept(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kept(static)
        for seed in range(4):
            x = torch.randn(6, 1, 256, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
            want = kept(x)
            static.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize('tokens', [3, 700, 2500])
@pytest.mark.parametrize('choice', [dict(), CHOICES[0]])
def test_serving_in_inference_mode(choice, tokens):
    """Tensors made in inference mode have no version by which a kept map, bins or indices are told: the layers run without, with 16 and 4 bits, by one call and by
    several, and what ordinary calls keep stays right next to it."""
    for changed in (dict(), dict(mlp_impl='sparse', mlp_type='mlp', activation_fn=Arguments().activation_fn)):
        args = _args(**choice, **changed)
        layer = dMoE(args).eval()
        layers = [layer] if changed else [layer, copy.deepcopy(layer).quantize_experts_(64, True), MoE(args).eval()]
        x = torch.randn(tokens, 1, 256, device='cuda').bfloat16()
        for layer in layers:
            with torch.no_grad():
                want = layer(x)
            with torch.inference_mode():
                got, again = layer(x), layer(x.clone())
            assert torch.equal(got, want) and torch.equal(again, want)
            with torch.no_grad():
                assert torch.equal(layer(x), want)


def test_products_and_permutation_of_inference_tensors():
    """Batch sizes and a routing made in inference mode, used there and outside."""
    kept = _quantized(_args(moe_num_experts=3, moe_top_k=2), 64, False)[1].experts.mlp
    x, ids = torch.randn(40, 256, device='cuda').bfloat16(), torch.randint(0, 3, (80,), device='cuda').int()

    def step():
        indices, bin_ids, counts, bins, _ = ops.routing.route(ids, 3, 2)
        rows = ops.gather(x, indices, bin_ids, bins, 2)
        y = kept(rows, counts)
        return ops.scatter(y, indices, bin_ids, torch.ones(80, device='cuda').bfloat16(), bins, 2), (rows, counts, indices, bin_ids, bins, y)
    with torch.no_grad():
        want, _ = step()
    with torch.inference_mode():
        got, (rows, counts, indices, bin_ids, bins, y) = step()
        counts.copy_(counts)
    assert torch.equal(got, want)
    with torch.no_grad():
        assert torch.equal(kept(rows, counts), y) and torch.equal(ops.gather(x, indices, bin_ids, bins, 2), rows)
