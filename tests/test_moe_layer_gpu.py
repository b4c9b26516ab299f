"""The layer for a few tokens, against the formulas in 64 bits.

Tolerances, from the roundings there are.  Weights are rounded to fp32 once (2^-24; the arithmetic before is in 64 bits).  An output is off by
  - the first products' sums: of n terms in fp32 at most n 2^-24 of the sum of magnitudes, through an activation of slope up to 1.13;
  - the activation: 2^-20 of itself and of its argument (an exponential and a quotient in fp32);
  - keeping it as two 16-bit numbers: the first is off by at most half its step, 2^-8 (bf16) or 2^-11 (fp16) of the value's power of two, so the second lies below that, where half a
    step is 2^-17 or 2^-23 (fp16 has no step below 2^-24: 2^-25 where the second number is that small);
  - the second product's sums, of ffn terms and top_k weighted parts, as the first's;
  - its rounding, half a step of its type.
Since roundings seldom all point one way, the norm of the error is held to a quarter more than half a step of the output's as well."""
import copy

import pytest
import torch
import torch.nn.functional as F

import megablocks_amd.ops as ops
from megablocks_amd import grouped_gemm_util as gg
from megablocks_amd.layers.arguments import DEFAULT_ACTIVATION_FN, Arguments
from megablocks_amd.layers.dmoe import dMoE
from megablocks_amd.layers.moe import clear_load_balancing_loss
from test_moe_layer import PLANS, plan_of

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
STEP = 2.0 ** -24


def make(tokens, hidden, ffn, experts, gate=True, dtype=BF16, std=0.05, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed + tokens * 7 + hidden)
    normal = lambda *shape: torch.randn(shape, generator=g, device='cuda')
    w = lambda: (normal(experts, ffn, hidden) * std).to(dtype)
    return dict(x=normal(tokens, hidden).to(dtype), router=(normal(experts, hidden) * std).to(dtype), w1=w(), v1=w() if gate else None, w2=w())


def exact_choice(o, top_k, score='softmax', bias=None, groups=1, top_groups=1, group_best=2, norm_p=0, scale=1.0):
    logits = o['x'].double() @ o['router'].double().t()
    s = logits.softmax(1) if score == 'softmax' else logits.sigmoid()
    keys = logits if bias is None else s + bias.double()
    if top_groups < groups:
        by_group = (s if bias is None else keys).view(len(s), groups, -1)
        of = by_group.topk(min(group_best, by_group.shape[2]), 2).values.sum(2)
        order = of.sort(dim=1, descending=True, stable=True).indices.argsort(1)
        keys = keys.masked_fill((order >= top_groups).repeat_interleave(by_group.shape[2], 1), -float('inf'))
    indices = keys.sort(dim=1, descending=True, stable=True).indices[:, :top_k]
    w = s.gather(1, indices)
    if norm_p:
        w = w / w.norm(p=norm_p, dim=1, keepdim=True)
    return w * scale, indices


def exact_out(o, weights, indices, act):
    """(the output in 64 bits, how far one may be off it)"""
    x, dtype = o['x'].double(), o['x'].dtype
    hidden, ffn = x.shape[1], o['w1'].shape[1]
    out, off = torch.zeros_like(x), torch.zeros_like(x)
    keep = 2.0 ** -17 if dtype == BF16 else 2.0 ** -23
    for e in indices.unique().tolist():
        t, j = (indices == e).nonzero(as_tuple=True)
        w1, w2 = o['w1'][e].double(), o['w2'][e].double()
        p, dp = x[t] @ w1.t(), hidden * STEP * (x[t].abs() @ w1.abs().t())
        a = F.silu(p) if act == gg.ACT_SILU else F.gelu(p, approximate='tanh')
        da = 1.13 * dp + 2.0 ** -20 * (a.abs() + p.abs())
        if o['v1'] is not None:
            v1 = o['v1'][e].double()
            q, dq = x[t] @ v1.t(), hidden * STEP * (x[t].abs() @ v1.abs().t())
            a, da = a * q, da * (q.abs() + dq) + a.abs() * dq + a.abs() * q.abs() * STEP
        da = da + keep * a.abs() + (2.0 ** -25 if dtype == FP16 else 0)
        w = weights[t, j].unsqueeze(1)
        out[t] += w * (a @ w2)
        off[t] += w.abs() * (da @ w2.abs() + (ffn + indices.shape[1] + 20) * STEP * (a.abs() @ w2.abs()))
    info = torch.finfo(dtype)
    return out, off + out.abs() * info.eps / 2 + info.tiny * info.eps


def check(o, top_k, act=gg.ACT_SILU, got=None, **choice):
    out, weights, indices = ops.moe_layer(**o, top_k=top_k, act=act, **choice) if got is None else got
    want_weights, want_indices = exact_choice(o, top_k, **choice)
    assert out.dtype == o['x'].dtype and weights.dtype == torch.float32 and indices.dtype == torch.int64
    assert torch.equal(indices, want_indices)
    assert ((weights.double() - want_weights).abs() <= want_weights.abs() * 1.01 * STEP + 2.0 ** -149).all()
    want, off = exact_out(o, want_weights, want_indices, act)
    error = (out.double() - want).abs()
    assert (error <= off).all()
    assert error.norm() <= 1.25 * torch.finfo(out.dtype).eps / 2 * want.norm()
    return out, weights, indices


@pytest.mark.parametrize('dtype', [BF16, FP16], ids=str)
@pytest.mark.parametrize('gate', [True, False], ids=['gated', 'plain'])
@pytest.mark.parametrize('tokens,hidden,ffn,experts,top_k', [
    (1, 8, 8, 1, 1), (1, 64, 64, 2, 1), (1, 2048, 1408, 16, 6), (1, 512, 4096, 8, 2), (2, 72, 40, 3, 3), (3, 1032, 264, 60, 4), (5, 128, 136, 130, 8), (7, 520, 1000, 512, 16),
    (8, 256, 24, 4, 1), (9, 264, 512, 8, 2), (11, 1048, 72, 29, 4), (16, 1024, 512, 64, 1), (17, 136, 200, 5, 2), (31, 512, 512, 300, 10), (33, 200, 328, 8, 2), (48, 256, 256, 2, 1),
    (63, 128, 72, 40, 16), (64, 640, 1088, 8, 2), (64, 64, 64, 1, 1)])
def test_layer(tokens, hidden, ffn, experts, top_k, gate, dtype):
    check(make(tokens, hidden, ffn, experts, gate, dtype), top_k, gg.ACT_SILU if gate else gg.ACT_GELU_TANH)


@pytest.mark.parametrize('choice', [
    dict(score='sigmoid'), dict(norm_p=1), dict(norm_p=2, scale=2.5), dict(norm_p=0.5), dict(norm_p=3, score='sigmoid'), dict(score='sigmoid', with_bias=True, norm_p=1), dict(with_bias=True),
    dict(groups=8, top_groups=3, group_best=1), dict(groups=4, top_groups=2), dict(score='sigmoid', with_bias=True, groups=8, top_groups=4, norm_p=1, scale=2.5),
    dict(groups=64, top_groups=40), dict(groups=2, top_groups=2, with_bias=True), dict(scale=-1.0), dict(scale=0.0)], ids=str)
@pytest.mark.parametrize('tokens,experts', [(1, 64), (6, 64), (20, 64), (50, 256)])
def test_choices(tokens, experts, choice):
    o = make(tokens, 256, 128, experts, std=0.1)
    choice = dict(choice)
    if choice.pop('with_bias', False):
        choice['bias'] = torch.randint(-40, 41, (experts,), device='cuda').float() * 0.001
    out, weights, indices = ops.moe_layer(**o, top_k=4, act=gg.ACT_GELU_TANH, **choice)
    if choice.get('scale') == 0.0:
        assert (out == 0).all() and (weights == 0).all()
    else:
        check(o, 4, gg.ACT_GELU_TANH, (out, weights, indices), **choice)


@pytest.mark.parametrize('tokens', [1, 15, 16, 17, 32, 33, 47, 48, 49, 64])
def test_all_tokens_on_the_same_experts(tokens):
    """A bias that nobody gets past: every row tile of two experts, the others without a row."""
    o = make(tokens, 264, 200, 9)
    bias = torch.zeros(9, device='cuda')
    bias[2], bias[7] = 9.0, 8.0
    _, _, indices = check(o, 2, bias=bias)
    assert (indices == torch.tensor([2, 7], device='cuda')).all()


def test_the_largest_matrices():
    """Experts of nearly 2 GiB a matrix, one behind the other."""
    o = make(2, 16384, 65200, 2, gate=False, std=0.01)
    _, _, indices = check(o, 1, gg.ACT_GELU_TANH, bias=torch.tensor([0.0, 9.0], device='cuda'))
    assert (indices == 1).all()


def test_equal_experts_go_to_the_lower_index():
    o = make(12, 128, 64, 100)
    for e in (10, 37, 99):
        o['router'][e] = o['router'][3]
    o['router'][50:60] = o['router'][49:50]
    check(o, 8)
    o['x'][4] = 0       # all logits zero
    _, _, indices = check(o, 8)
    assert indices[4].tolist() == list(range(8))


def test_neighbours_in_the_order_are_told_apart():
    """Logits that differ in the last of a long sum's terms: by less than fp32 sums of it are off."""
    o = make(4, 4096, 64, 8, std=0.02)
    o['router'][1:] = o['router'][:1]
    o['x'][:, -8:] = 2.0 ** -12
    for e in range(8):
        o['router'][e, -8 + e] += 2.0 ** -9 * (e + 1)
    _, _, indices = check(o, 3)
    assert (indices == torch.tensor([7, 6, 5], device='cuda')).all()


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_a_token_that_is_no_number_leaves_the_others_alone(bad):
    for tokens in (5, 40):
        o = make(tokens, 128, 72, 8)
        before = ops.moe_layer(**o, top_k=2, act=0)
        o['x'][3, 17] = bad
        out, weights, indices = ops.moe_layer(**o, top_k=2, act=0)
        rest = torch.arange(tokens, device='cuda') != 3
        # the token's rows may have gone to other experts, but rows are computed by themselves
        assert torch.equal(out[rest], before[0][rest]) and torch.equal(weights[rest], before[1][rest]) and torch.equal(indices[rest], before[2][rest])
        assert not out[3].isfinite().any() and ((indices[3] >= 0) & (indices[3] < 8)).all()
        assert indices[3, 0] != indices[3, 1]


def test_values_past_16_bits_on_the_way():
    """fp16: an activation past 65504 is infinite in 16 bits, as the separate operators have it, and shows."""
    o = make(2, 64, 8, 2, dtype=FP16, std=1.0)
    o['x'] *= 100
    out, _, _ = ops.moe_layer(**o, top_k=1, act=0)
    hidden = [F.silu(o['x'][t].double() @ o['w1'][e].double().t()) * (o['x'][t].double() @ o['v1'][e].double().t()) for t in range(2) for e in range(2)]
    assert max(h.abs().max().item() for h in hidden) > 65504 and not out.isfinite().all()


def test_experts_without_a_row_are_not_read():
    o = make(3, 128, 72, 6)
    bias = torch.zeros(6, device='cuda')
    bias[1], bias[4] = 9.0, 8.0
    out, _, _ = ops.moe_layer(**o, top_k=2, act=0, bias=bias)
    for name in ('w1', 'v1', 'w2'):
        o[name][[0, 2, 3, 5]] = float('nan')
    assert torch.equal(ops.moe_layer(**o, top_k=2, act=0, bias=bias)[0], out)


def test_operands_end_at_their_last_value():
    """Buffers whose neighbours are NaN: nothing outside is read into a result, nothing outside is written."""
    for tokens, hidden, ffn, experts in ((3, 72, 40, 5), (20, 136, 104, 3)):
        o = make(tokens, hidden, ffn, experts)
        want = ops.moe_layer(**o, top_k=2, act=0)
        padded = {}
        for name, t in o.items():
            buffer = torch.full((t.numel() + 256,), float('nan'), dtype=t.dtype, device='cuda')
            buffer[128:-128] = t.flatten()
            padded[name] = buffer[128:-128].view(t.shape)
        got = ops.moe_layer(**padded, top_k=2, act=0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layouts_and_no_tokens():
    o = make(4, 128, 72, 6)
    want = ops.moe_layer(**o, top_k=2, act=0)
    for x in (torch.cat([o['x'], o['x']], 1)[:, :128], o['x'].t().contiguous().t(), torch.cat([torch.zeros(1, device='cuda').to(BF16), o['x'].flatten()])[1:].view(4, 128)):
        assert all(torch.equal(a, b) for a, b in zip(ops.moe_layer(**(o | dict(x=x)), top_k=2, act=0), want))
    out, weights, indices = ops.moe_layer(**(o | dict(x=o['x'][:0])), top_k=2, act=0)
    assert out.shape == (0, 128) and weights.shape == (0, 2) and indices.shape == (0, 2)


def test_refusals_on_the_gpu():
    o = make(2, 64, 40, 4)
    bad = [dict(x=o['x'].float()), dict(x=o['x'].half()), dict(w2=o['w2'].float()), dict(x=o['x'].cpu()), dict(router=o['router'].cpu()), dict(w1=o['w1'].transpose(0, 1).contiguous().transpose(0, 1)),
           dict(bias=torch.zeros(4, device='cuda').half()), dict(bias=torch.zeros(4)), dict(w1=o['w1'].clone().requires_grad_()),
           dict(w2=torch.cat([torch.zeros(1, device='cuda').to(BF16), o['w2'].flatten()])[1:].view(o['w2'].shape)), {name: (None if t is None else t.float()) for name, t in o.items()}]
    for changed in bad:
        with pytest.raises(RuntimeError):
            ops.moe_layer(**(o | changed), top_k=2, act=0)
    with torch.no_grad():
        ops.moe_layer(**(o | dict(w1=o['w1'].clone().requires_grad_())), top_k=2, act=0)
    with torch.inference_mode():
        ops.moe_layer(**{name: t.clone() for name, t in o.items()}, top_k=2, act=0)


def test_the_same_from_run_to_run_and_side_by_side():
    small, large = make(3, 512, 264, 16), make(40, 1024, 520, 8, seed=1)
    want = [ops.moe_layer(**o, top_k=2, act=0) for o in (small, large)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(10):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append((s % 2, ops.moe_layer(**(small, large)[s % 2], top_k=2, act=0)))
    torch.cuda.synchronize()
    for which, result in got:
        assert all(torch.equal(a, b) for a, b in zip(result, want[which]))


def test_captured_and_replayed(monkeypatch):
    for lent in (True, False):
        monkeypatch.setattr(gg, 'GMM_WORKSPACE', lent)
        first, second = make(3, 512, 264, 16), make(20, 256, 136, 8, seed=1)
        for o in (first, second):
            ops.moe_layer(**o, top_k=2, act=0)
        graphs = []
        for o in (first, second):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, o, [ops.moe_layer(**o, top_k=2, act=0) for _ in range(2)]))
        for turn in range(3):
            for graph, o, results in (graphs if turn % 2 else reversed(graphs)):
                o['x'].copy_(torch.randn_like(o['x']))
                graph.replay()
                torch.cuda.synchronize()
                eager = ops.moe_layer(**o, top_k=2, act=0)
                for result in results:
                    assert all(torch.equal(a, b) for a, b in zip(result, eager))


# ---- in the layers ----

def make_layer(**changed):
    args = Arguments(**(dict(hidden_size=256, ffn_hidden_size=384, moe_num_experts=16, moe_top_k=4, mlp_type='glu', activation_fn=F.silu, fp16=False, bf16=True, bias=False,
                             moe_normalize_expert_weights=1, moe_fused_tokens=16, init_method=lambda w: torch.nn.init.normal_(w, std=0.1)) | changed))
    torch.manual_seed(3)
    layer = dMoE(args).eval()
    separate = copy.deepcopy(layer)
    separate.experts.args = copy.copy(args)
    separate.experts.args.moe_fused_tokens = 0
    return layer, separate


def chosen_alike(layer, x):
    """The tokens whose experts are the same whether logits are rounded to 16 bits, as the separate operators do, or not."""
    args = layer.experts.args
    _, exact = exact_choice(dict(x=x.reshape(-1, x.shape[-1]), router=layer.router.layer.weight.detach()), args.moe_top_k, args.moe_router_score, layer.router.balance_bias,
                            args.moe_router_groups, args.moe_router_top_groups, args.moe_router_group_best)
    return (layer.router(x)[2].sort(1).values == exact.sort(1).values).all(1)


def chosen_alike_plainly(layer, x):
    _, exact = exact_choice(dict(x=x.reshape(-1, x.shape[-1]), router=layer.router.layer.weight.detach()), layer.experts.args.moe_top_k)
    return (layer.router(x)[2].sort(1).values == exact.sort(1).values).all(1)


def calls(monkeypatch):
    from megablocks_amd.ops import few_tokens
    made, launch = [], few_tokens.launch
    monkeypatch.setattr(few_tokens, 'launch', lambda *args: made.append(1) or launch(*args))
    return made


@pytest.mark.parametrize('changed', [
    {}, dict(mlp_type='mlp', activation_fn=DEFAULT_ACTIVATION_FN), dict(activation_fn=DEFAULT_ACTIVATION_FN), dict(bias=True), dict(bias=True, return_bias=False), dict(fp16=True, bf16=False),
    dict(moe_router_score='sigmoid', moe_router_bias=True, moe_router_groups=4, moe_router_top_groups=2, moe_router_scale=2.5), dict(moe_top_k=1), dict(memory_optimized_mlp=True),
    dict(moe_normalize_expert_weights=None, moe_loss_weight=0)], ids=str)
def test_layer_as_a_module(changed, monkeypatch):
    layer, separate = make_layer(**changed)
    made = calls(monkeypatch)
    if layer.experts.bias is not None:
        with torch.no_grad():
            layer.experts.bias.normal_()
            separate.experts.bias.copy_(layer.experts.bias)
    x = torch.randn(2, 5, 256, device='cuda').to(next(layer.parameters()).dtype)
    with torch.no_grad():
        got, want = layer(x), separate(x)
        alike = chosen_alike(separate, x)
    assert len(made) == 1
    if layer.experts.bias is not None and layer.experts.args.return_bias:
        assert torch.equal(got[1], want[1])
        got, want = got[0], want[0]
    # the separate operators round logits, weights, both first products, the activation and the second product to 16 bits as well
    got, want = got.double().view(-1, 256)[alike], want.double().view(-1, 256)[alike]
    assert alike.sum() >= 7 and (got - want).norm() <= 1e-2 * want.norm()


def test_calls_that_stay_with_the_separate_operators(monkeypatch):
    layer, separate = make_layer()
    made = calls(monkeypatch)
    x = torch.randn(10, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        many = torch.randn(17, 1, 256, device='cuda').bfloat16()
        assert torch.equal(layer(many), separate(many))
    assert torch.equal(layer(x), separate(x))                                      # gradients are recorded
    with torch.no_grad():
        layer.train(), separate.train()
        assert torch.equal(layer(x), separate(x))
        clear_load_balancing_loss()
        layer.eval(), separate.eval()
        for module in (layer.router, layer.router.layer, layer.experts, layer.experts.mlp):
            seen = []
            handle = module.register_forward_hook(lambda *args: seen.append(1))
            layer(x)
            handle.remove()
            assert seen or module in (layer.router.layer, layer.experts.mlp)        # few rows: their weights are taken without a call
        layer.experts.forward_fn = lambda *args: (x * 2, None)
        assert torch.equal(layer(x), x * 2)
        layer.experts.forward_fn = layer.experts.forward_once
        with torch.autocast('cuda', dtype=torch.bfloat16):
            layer(x)
        quantized = copy.deepcopy(layer).quantize_experts_()
        quantized(x)
    assert not made
    with torch.no_grad():
        layer(x)
    assert len(made) == 1


@pytest.mark.parametrize('changed', [dict(moe_normalize_expert_weights=float('inf')), dict(moe_router_groups=3, moe_router_top_groups=3, moe_router_group_best=5)], ids=str)
def test_routers_that_look_at_no_options(changed, monkeypatch):
    """A router with softmax scores, no bias and all groups open takes any norm and does not look at the groups: with an infinite norm the separate operators run, as they did."""
    layer, separate = make_layer(**changed)
    made = calls(monkeypatch)
    x = torch.randn(3, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        got, want = layer(x), separate(x)
        alike = chosen_alike_plainly(separate, x)
    assert len(made) == (0 if 'moe_normalize_expert_weights' in changed else 1)
    got, want = got.double().view(-1, 256)[alike], want.double().view(-1, 256)[alike]
    assert alike.any() and (got - want).norm() <= 1e-2 * want.norm()


def test_layer_captured(monkeypatch):
    layer, _ = make_layer()
    x = torch.randn(4, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        layer(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        for _ in range(3):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer(x))


def test_a_model_trains_and_decodes():
    """Embedding, a layer, the norm of all gradients and a clipped step; then the same model a token at a time."""
    torch.manual_seed(0)
    words, hidden, tokens = 300, 256, 96
    table = torch.nn.Parameter(torch.randn(words, hidden, device='cuda').bfloat16())
    layer, _ = make_layer(moe_loss_weight=0)
    ids = torch.randint(0, words, (tokens, 1), device='cuda')
    parameters = [table, *layer.parameters()]

    layer.train()
    x = ops.embedding(ids, table, scale=0.5, padding_idx=0)
    out = layer(x) + x
    loss = (out.float() @ table.float().t()).logsumexp(-1).mean() - (out.float() * table.float()[ids]).sum(-1).mean()
    loss.backward()
    grads = [p.grad.clone() for p in parameters]
    norm = ops.clip_grad_norm_(parameters, 0.25)
    exact = torch.cat([g.double().flatten() for g in grads]).norm().item()
    assert abs(norm.item() - exact) <= exact * 1.01 * STEP
    by = min(1.0, 0.25 / (exact + 1e-6))
    for p, g in zip(parameters, grads):
        want = g.double() * by
        assert ((p.grad.double() - want).abs() <= want.abs() * (5 * STEP + 2.0 ** -8) + 2.0 ** -133).all()
    # the table's gradient through the embedding alone: that of the rows, gathered by word
    rows, = torch.autograd.grad(ops.embedding(ids, table, scale=0.5, padding_idx=0), table, torch.ones(tokens, 1, hidden, device='cuda').bfloat16())
    counts = torch.bincount(ids.flatten(), minlength=words).double()
    counts[0] = 0
    assert torch.equal(rows.double(), (counts * 0.5).unsqueeze(1).expand(words, hidden))
    with torch.no_grad():
        for p in parameters:
            p -= p.grad
        layer.eval()
        x = ops.embedding(ids, table, scale=0.5)
        whole = layer(x)                                     # 96 tokens: the separate operators
        alone = torch.cat([layer(ops.embedding(ids[t:t + 16], table, scale=0.5)) for t in range(0, tokens, 16)])
        alike = chosen_alike(layer, x)
    whole, alone = whole.double().view(-1, hidden)[alike], alone.double().view(-1, hidden)[alike]
    assert alike.sum() >= tokens * 0.8 and (whole - alone).norm() <= 1e-2 * whole.norm()


# ---- norms of scores whose powers leave every number's range ----

def exact_weights_by_logarithms(logits, indices, score, norm_p, scale=1.0):
    """scale s / ||s||_p in 64 bits, from log s: nothing is raised to a power."""
    logs = (logits.log_softmax(1) if score == 'softmax' else F.logsigmoid(logits)).gather(1, indices)
    return scale * (logs - (norm_p * logs).logsumexp(1, keepdim=True) / norm_p).exp()


@pytest.mark.parametrize('norm_p', [0.5, 2, 16, 64, 119, 120, 130, 1000, 3e38])
@pytest.mark.parametrize('score,experts,logit', [('softmax', 512, 0.0), ('softmax', 64, 3.0), ('sigmoid', 64, -50.0), ('sigmoid', 16, -600.0), ('sigmoid', 300, 5.0)])
def test_norms_of_large_order_and_small_scores(score, experts, logit, norm_p):
    """Logits around one number (softmax: flat but for a little), some of one number exactly."""
    hidden, top_k = 64, 6
    o = make(5, hidden, 72, experts, std=0.001)
    o['x'][:, 0] = 1.0
    o['router'][:, 0] = logit
    o['router'][experts // 2:, 1:] = 0
    out, weights, indices = ops.moe_layer(**o, top_k=top_k, act=gg.ACT_SILU, score=score, norm_p=norm_p, scale=1.5)
    _, want_indices = exact_choice(o, top_k, score)
    assert torch.equal(indices, want_indices)
    logits = o['x'].double() @ o['router'].double().t()
    want = exact_weights_by_logarithms(logits, indices, score, norm_p, 1.5)
    # arithmetic in 64 bits, the logarithms' too: of numbers up to 601 times p, which is 2^-43 of an exponent there, divided by p again
    assert ((weights.double() - want).abs() <= want * 1.01 * STEP + 2.0 ** -149).all()
    want_out, off = exact_out(o, want, indices, gg.ACT_SILU)
    assert ((out.double() - want_out).abs() <= off).all()


def test_norms_of_scores_that_are_zero_or_no_numbers():
    o = make(4, 64, 72, 16)
    o['x'][:, 0], o['router'][:, 0] = 1.0, 0.0
    o['x'][1, 0], o['x'][2, 3] = -30000.0, float('nan')
    o['router'][:, 0] = 1.0
    for norm_p in (1, 2, 64, 0.5):
        out, weights, _ = ops.moe_layer(**o, top_k=3, act=0, score='sigmoid', norm_p=norm_p)
        assert (weights[1] == 0).all() and (out[1] == 0).all() and weights[2].isnan().all() and out[2].isnan().all()
        rest = torch.tensor([0, 3], device='cuda')
        assert ((weights[rest].double().pow(norm_p).sum(1) - 1).abs() <= 1e-5).all()


@pytest.mark.parametrize('norm_p', [2, 130, 1000])
def test_layers_with_norms_of_large_order(norm_p, monkeypatch):
    """A dMoE's weights by either way: scores of about 1 / 512, of logits below 1, whose rounding to bf16 moves a score by 2^-9."""
    layer, separate = make_layer(moe_num_experts=512, moe_top_k=4, ffn_hidden_size=128, moe_normalize_expert_weights=norm_p, moe_router_scale=2.0)
    made = calls(monkeypatch)
    with torch.no_grad():
        for both in (layer, separate):
            both.router.layer.weight *= 0.125
        x = torch.randn(6, 1, 256, device='cuda').bfloat16()
        got, want, alike = layer(x), separate(x), chosen_alike(separate, x)
    assert len(made) == 1 and alike.any()
    got, want = got.double().view(-1, 256)[alike], want.double().view(-1, 256)[alike]
    assert want.norm() > 0 and (got - want).norm() <= 1e-2 * want.norm()


# ---- fp16: the activation in two numbers that keep their bits whatever its size ----

def exact_out_of_fp16(o, weights, indices):
    """exact_out for fp16: the activation (silu) is kept to 2^-23 of it or 2^-32."""
    x = o['x'].double()
    hidden, ffn = x.shape[1], o['w1'].shape[1]
    out, off = torch.zeros_like(x), torch.zeros_like(x)
    largest = smallest = None
    for e in indices.unique().tolist():
        t, j = (indices == e).nonzero(as_tuple=True)
        w1, w2 = o['w1'][e].double(), o['w2'][e].double()
        p, dp = x[t] @ w1.t(), hidden * STEP * (x[t].abs() @ w1.abs().t())
        a, da = F.silu(p), 1.13 * dp + 2.0 ** -20 * (F.silu(p).abs() + p.abs())
        if o['v1'] is not None:
            v1 = o['v1'][e].double()
            q, dq = x[t] @ v1.t(), hidden * STEP * (x[t].abs() @ v1.abs().t())
            a, da = a * q, da * (q.abs() + dq) + a.abs() * dq + a.abs() * q.abs() * STEP
        da = da + 2.0 ** -23 * a.abs() + 2.0 ** -32
        w = weights[t, j].unsqueeze(1)
        out[t] += w * (a @ w2)
        off[t] += w.abs() * (da @ w2.abs() + (ffn + indices.shape[1] + 20) * STEP * (a.abs() @ w2.abs()))
        largest = max(largest or 0, a.abs().max().item())
    return out, off, largest


@pytest.mark.parametrize('gate', [True, False], ids=['gated', 'plain'])
@pytest.mark.parametrize('tokens,experts', [(1, 4), (9, 4), (40, 3), (64, 2)])
@pytest.mark.parametrize('size', [2.0 ** -18, 1e-5, 1e-4, 2.0 ** -12, 1e-2, 1.0, 1e3, 3e4], ids=lambda s: f'{s:.0e}')
def test_fp16_activations_of_every_size(size, tokens, experts, gate):
    """Activations of about `size`, past 65504 too, and second weights that bring the output to about 1: its own rounding is all there is."""
    o = make(tokens, 128, 264, experts, gate, FP16, std=0.1)
    # first weights that make the gate's product (or, plain, the activation) that small or large; silu(p) is p / 2 near 0 and p far from it
    if gate:
        o['v1'] = (o['v1'].float() * min(size * 2, 1e3)).half()
        o['w1'] = (o['w1'].float() * max(1.0, size / 1e3)).half()
    else:
        o['w1'] = (o['w1'].float() * (size if size > 1 else 2 * size)).half()
    o['w2'] = (o['w2'].float() / min(max(size, 2.0 ** -9), 1e3)).half()
    if size > 1e3:
        o['w2'] = (o['w2'].float() / (size / 1e3)).half()
    out, weights, indices = ops.moe_layer(**o, top_k=2, act=gg.ACT_SILU, norm_p=1)
    want_weights, _ = exact_choice(o, 2, norm_p=1)
    want, off, largest = exact_out_of_fp16(o, want_weights, indices)
    assert largest < 2.0 ** 20 and (size < 1e4 or largest > 65504)
    error = (out.double() - want).abs()
    half = want.abs().clamp(min=2.0 ** -14) * 2.0 ** -11      # half a step, also of the numbers below the normal ones
    assert (error <= off + half).all()
    assert error.norm() <= 1.01 * half.norm()


def test_fp16_activations_past_what_two_numbers_hold_are_infinite():
    o = make(1, 64, 8, 1, gate=False, dtype=FP16)
    o['x'].fill_(0)
    o['x'][0, 0], o['w1'][0], o['w2'][0] = 32768.0, 0.0, 0.0
    o['w1'][0, 2, 0], o['w2'][0, 2, 5] = 31.0, 2.0 ** -8
    assert ops.moe_layer(**o, top_k=1, act=gg.ACT_SILU)[0][0, 5].item() == 31.0 * 2 ** 15 / 2 ** 8       # 1015808, below 2^20
    o['w1'][0, 2, 0] = 32.0
    assert ops.moe_layer(**o, top_k=1, act=gg.ACT_SILU)[0][0, 5].item() == float('inf')


# ---- every way in which the products are computed ----

@pytest.mark.parametrize('dtype', [BF16, FP16], ids=str)
@pytest.mark.parametrize('sizes,gate,plan', PLANS, ids=lambda v: '-'.join(map(str, v)) if isinstance(v, tuple) else 'gated' if v else 'plain')
def test_every_way_of_the_products(sizes, gate, plan, dtype):
    assert plan_of(sizes, gate) == plan
    tokens, hidden, ffn, experts, top_k = sizes
    o = make(tokens, hidden, ffn, experts, gate, dtype, std=min(0.1, 1.5 / hidden ** 0.5))
    check(o, top_k, gg.ACT_SILU if gate else gg.ACT_GELU_TANH)
    # all rows on the same experts: one or more rounds of row tiles, the last of which is not full
    bias = torch.zeros(experts, device='cuda')
    bias[-top_k:] = 9.0
    check(o, top_k, gg.ACT_GELU_TANH if gate else gg.ACT_SILU, score='sigmoid', bias=bias, norm_p=1)


def test_layers_with_norms_that_are_infinite_in_fp32(monkeypatch):
    """An order of 1e39 is a number to the separate operators, and none to the one for a few tokens."""
    layer, separate = make_layer(moe_normalize_expert_weights=1e39)
    made = calls(monkeypatch)
    x = torch.randn(3, 1, 256, device='cuda').bfloat16()
    with torch.no_grad():
        got, want = layer(x), separate(x)
    assert not made and torch.equal(got, want)


@pytest.mark.parametrize('score,logit', [('sigmoid', 48.0), ('sigmoid', -800.0), ('softmax', 48.0)])
@pytest.mark.parametrize('tokens,experts,groups', [(1, 32, 8), (6, 64, 4), (20, 256, 8)])
def test_groups_by_their_best_expert_where_scores_are_all_alike(tokens, experts, groups, score, logit):
    """Logits of 40 to 56, whose sigmoid scores are 1 in 64 bits, or of -800, whose are 0; groups go by the largest logit, as in choose_experts."""
    o = make(tokens, 128, 72, experts, std=0.02)
    o['x'] = (o['x'].float() * 4).bfloat16()
    o['x'][:, 0], o['router'][:, 0] = 1.0, logit
    if score == 'softmax':
        o['router'][0, 0] = 1000.0         # next to which all others have a score of 0
    logits = o['x'].double() @ o['router'].double().t()
    of = logits.view(tokens, groups, -1)
    ranks = of.amax(2).sort(dim=1, descending=True, stable=True).indices.argsort(1)
    keys = of.masked_fill((ranks >= 2).unsqueeze(2), -float('inf')).flatten(1)
    want = keys.sort(dim=1, descending=True, stable=True).indices[:, :3]
    _, _, indices = ops.moe_layer(**o, top_k=3, act=0, score=score, groups=groups, top_groups=2, group_best=1)
    assert torch.equal(indices, want)
    assert torch.equal(ops.choose_experts(logits.float(), 3, score, groups=groups, top_groups=2, group_best=1)[2], want)
