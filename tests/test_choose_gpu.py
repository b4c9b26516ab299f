"""The choice of experts by scores, bias and groups, its gradient and the update of the bias, against their restatement in float64.

Tolerances.  fp32 arithmetic: exp and reciprocal as the hardware has them are off by 2^-23 each, the exponent x - m (16 bits out: times log2 e as well) by 2^-24
of its size, sums of up to 512 positive terms by 2^-24 for each of some 16 steps: a score is off by at most (|x - m| + 24) 2^-23 of itself.  Rounding to the
output's type is half a step of it, eps / 2."""
import pytest
import torch

import megablocks_amd.ops as ops
from oracle import choose as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _spread(x):
    """How large the exponents of the scores are, per token."""
    x = x.double().cpu()
    return (x.abs().amax(1, keepdim=True) * 2).clamp(max=200.)


def _close(got, want, bound, what):
    got = got.double().cpu()
    off = (got - want).abs()
    assert bool((off <= bound).all()), (what, float((off / bound.clamp(min=1e-300)).max()))


def _tiny(dtype):
    return {BF16: 2.0 ** -126, F16: 2.0 ** -24, F32: 2.0 ** -126}[dtype]    # below the smallest normal number (fp16: its smallest step) nothing is promised


def _check(logits, top_k, dtype, **how):
    x = logits.to(dtype)
    bias = how.get('bias')
    got = ops.choose_experts(x.cuda(), top_k, want_lse=True, **{**how, 'bias': None if bias is None else bias.cuda()})
    s, w, i, lse = oracle.choose(x, top_k, **how)
    assert got[0].dtype == got[1].dtype == dtype and got[2].dtype == torch.int64 and got[3].dtype == torch.float32
    assert torch.equal(got[2].cpu(), i), (got[2].cpu() != i).nonzero()[:5]
    step, fp32 = torch.finfo(dtype).eps / 2, (_spread(x) + 24) * 2.0 ** -23
    _close(got[0], s, s * (step + fp32) + _tiny(dtype), 'scores')
    _close(got[1], w, w.abs() * (step + 4 * fp32) + _tiny(dtype), 'weights')
    _close(got[3], lse, 24 * 2.0 ** -23 * (1 + lse.abs()), 'lse')
    return x, got


SHAPES = [   # tokens, experts, top_k, groups, top_groups, group_best
    (1, 8, 2, 1, 1, 1), (7, 16, 1, 4, 2, 2), (33, 12, 2, 3, 2, 2), (17, 60, 4, 5, 3, 1), (64, 64, 6, 8, 3, 2), (50, 128, 8, 1, 1, 2), (129, 256, 8, 8, 4, 2),
    (5, 250, 16, 10, 4, 2), (40, 160, 6, 8, 3, 1), (9, 512, 10, 16, 8, 2), (6, 500, 64, 20, 10, 2), (3, 96, 17, 2, 1, 2), (2, 1, 1, 1, 1, 1), (11, 4, 4, 2, 2, 1),
    (19, 64, 64, 64, 64, 2), (13, 96, 8, 32, 9, 2), (21, 9, 2, 9, 4, 2), (8, 384, 8, 48, 5, 2), (25, 48, 4, 16, 3, 2)]


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('shape', SHAPES)
def test_choice(shape, score, dtype):
    tokens, experts, top_k, groups, top_groups, best = shape
    g = torch.Generator().manual_seed(experts * 7 + tokens)
    x = torch.randn(tokens, experts, generator=g) * 1.5
    bias = torch.randint(-40, 41, (experts,), generator=g) * 0.001
    print(f'choice {shape} {score} {dtype}', flush=True)
    for b in (None, bias, torch.zeros(experts)):
        for p, scale in ((0, 1.0), (1, 2.5)):
            _check(x, top_k, dtype, score=score, bias=b, groups=groups, top_groups=top_groups, group_best=best, norm_p=p, scale=scale)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('p', [2, 3, 0.5])
def test_norms(score, p):
    g = torch.Generator().manual_seed(5)
    _check(torch.randn(31, 24, generator=g), 5, F32, score=score, norm_p=p, scale=0.5)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('groups', [1, 8])
def test_keys_that_32_bits_do_not_tell_apart(score, groups):
    """Logits a step of fp32 apart around a value, and biases that nearly make up for the scores: the order is that of the exact keys."""
    g = torch.Generator().manual_seed(11)
    tokens, experts = 65, 64
    x = 1.25 + torch.randint(-8, 9, (tokens, experts), generator=g) * 2.0 ** -22
    bias = torch.randint(-2, 3, (experts,), generator=g) * 2.0 ** -25
    _check(x, 6, F32, score=score, bias=bias, groups=groups, top_groups=max(1, groups // 2), norm_p=1)
    _check(x, 6, F32, score=score, groups=groups, top_groups=max(1, groups // 2), norm_p=1)
    big = torch.randn(tokens, experts, generator=g) * 2 + 24      # sigmoids within 2^-24 of one
    _check(big, 6, F32, score=score, bias=bias * 0 + 0.125, groups=groups, top_groups=max(1, groups // 2))


def _border(experts, top_k, groups, score, dtype):
    """(logits, bias): top_k - 1 experts far in front; at the border two of the same logit and bias, and at a higher index one whose exact key is the larger
    and whose key in fp32 is theirs."""
    x, bias = torch.full((1, experts), -9.), torch.zeros(experts)
    x[0, :top_k - 1], bias[:top_k - 1] = 0., 2. + torch.arange(top_k - 1)
    at = experts // groups if groups > 1 else top_k - 1        # in a group of their own, the second best
    if score == 'sigmoid':
        x[0, [at, at + 1, at + 3]] = torch.tensor([20., 20., 20.125])        # 1 - 2.1e-9 and 1 - 1.8e-9
    else:
        x[0, experts - 1] = 0.
        x[0, [at, at + 1, at + 3]] = torch.tensor([-16., -16., -15.875])     # below 1.3e-7, next to a bias of one
        bias[[at, at + 1, at + 3]] = 1.
    return x.to(dtype), bias


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,top_k,groups', [(5, 1, 1), (12, 4, 1), (64, 6, 4), (256, 8, 1), (256, 8, 8), (384, 17, 4), (500, 2, 1)])
@pytest.mark.parametrize('tokens', [3, 2100])
def test_a_tie_at_the_border_hides_no_larger_key(tokens, experts, top_k, groups, score, dtype):
    """The last chosen and the first left out are made of the same logit and bias: what follows them counts all the same."""
    x, bias = _border(experts, top_k, groups, score, dtype)
    how = dict(score=score, bias=bias, groups=groups, top_groups=min(groups, 2))
    want = oracle.choose(x, top_k, **how)[2]
    assert int(want[0, -1]) == (experts // groups if groups > 1 else top_k - 1) + 3
    got = ops.choose_experts(x.repeat(tokens, 1).cuda(), top_k, **{**how, 'bias': bias.cuda()})[2].cpu()
    assert torch.equal(got, want.expand(tokens, -1))


def test_ties_at_the_border_without_a_larger_key():
    """Many of the same logit and bias, nothing behind them or only smaller keys: the lower indices."""
    for experts in (16, 40, 300):
        x, bias = torch.zeros(4, experts), torch.full((experts,), 0.25)
        x[1, experts // 2:] = -1.
        x[2, experts // 2:] = -float('inf')
        x[3, 0] = 1.
        _check(x, 3, F32, score='sigmoid', bias=bias)
        _check(x, 3, BF16, score='softmax', bias=bias, groups=2, top_groups=1)


@pytest.mark.parametrize('experts', [4, 12, 96, 128])
@pytest.mark.parametrize('size', [64., 8192., 1e6])
def test_groups_whose_keys_cancel(size, experts):
    """One expert of a group is wanted by its bias and the rest shut out by theirs: the group's key is what two large numbers leave, with their rounding."""
    g = torch.Generator().manual_seed(31)
    bias = torch.zeros(experts)
    bias[0], bias[1:experts // 2] = size, -size
    x = torch.randn(200, experts, generator=g)
    x[:, 2:experts // 2], x[:, experts // 2 + 2:] = -4., -4.
    x[:, experts // 2:experts // 2 + 2] = x[:, :2] + torch.randn(200, 2, generator=g) * 2.0 ** -10
    how = dict(score='sigmoid', bias=bias, groups=2, top_groups=1, group_best=2)
    want = oracle.choose(x, 1, **how)[2]
    assert 50 < int((want < experts // 2).sum()) < 150
    assert torch.equal(ops.choose_experts(x.cuda(), 1, **{**how, 'bias': bias.cuda()})[2].cpu(), want)


def test_groups_shut_out_by_the_lowest_number():
    """Biases of the type's lowest number or of -infinity in whole groups: their sums are none, and the open groups' experts are chosen."""
    low = torch.finfo(F32).min
    x = torch.randn(50, 32, generator=torch.Generator().manual_seed(32))
    for out in (low, -float('inf')):
        for top_groups in (1, 2):
            bias = torch.full((32,), out)
            bias[8:24] = 0.
            _check(x, 4, F32, score='sigmoid', bias=bias, groups=4, top_groups=top_groups, norm_p=1)


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('with_bias', [False, True])
def test_many_equal_logits(dtype, with_bias):
    """Ties go to the lower index, also where the bias is the same for many."""
    g = torch.Generator().manual_seed(12)
    x = torch.randint(-2, 3, (70, 96), generator=g).float()
    bias = torch.randint(0, 2, (96,), generator=g) * 0.25 if with_bias else None
    for score in ('softmax', 'sigmoid'):
        _check(x, 8, dtype, score=score, bias=bias, groups=6, top_groups=3, norm_p=1)


def test_masked_infinite_and_undefined_logits():
    inf, nan = float('inf'), float('nan')
    x = torch.zeros(6, 16)
    x[0, 3:] = -inf                 # fewer experts left than are chosen
    x[1] = -inf                     # none left
    x[2, 5] = nan
    x[3, 7] = inf
    x[4] = -200.                    # scores of zero in fp32
    x[5] = torch.arange(16) * -1.
    for bias in (None, torch.zeros(16)):
        s, w, i, lse = ops.choose_experts(x.cuda(), 4, score='sigmoid', bias=None if bias is None else bias.cuda(), norm_p=1, want_lse=True)
        i, w = i.cpu(), w.cpu()
        assert i[0].tolist() == [0, 1, 2, 3] and w[0].tolist() == pytest.approx([1 / 3, 1 / 3, 1 / 3, 0])
        assert i[1].tolist() == [0, 1, 2, 3] and w[1].tolist() == [0] * 4
        assert i[2].tolist() == [5, 0, 1, 2] and w[2].isnan().all()
        assert i[3].tolist() == [7, 0, 1, 2] and w[3].tolist() == pytest.approx([0.4, 0.2, 0.2, 0.2])
        assert i[4].tolist() == [0, 1, 2, 3] and not w[4].isnan().any()
        assert i[5].tolist() == [0, 1, 2, 3]
        assert lse.cpu()[1] == -inf and lse.cpu()[3] == inf
    # an expert that its bias shuts out, in a softmax and in groups; masked logits never bring in an expert of a closed group
    bias = torch.zeros(16)
    bias[0] = -inf
    _, _, i, _ = ops.choose_experts(x.cuda(), 4, score='sigmoid', bias=bias.cuda())
    assert i.cpu()[5].tolist() == [1, 2, 3, 4]
    y = torch.full((2, 16), -inf)
    y[:, 12] = 1.
    for best in (1, 2):
        _, _, i, _ = ops.choose_experts(y.cuda(), 4, score='sigmoid', groups=4, top_groups=1, group_best=best)
        assert i.cpu().tolist() == [[12, 13, 14, 15]] * 2
    i = ops.choose_experts(x[1:2].cuda(), 2, score='softmax', groups=4, top_groups=2)[2].cpu()   # softmax of nothing is undefined; the indices are experts
    assert ((0 <= i) & (i < 16)).all()


@pytest.mark.parametrize('experts', [5, 64, 300])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_lse_of_logits_that_are_not_numbers(score, experts):
    """A logit that is not a number makes lse none, also next to infinities; without one infinities are the sum."""
    inf, nan = float('inf'), float('nan')
    x = torch.zeros(8, experts)
    x[0] = nan
    x[1], x[1, -1] = -inf, nan
    x[2, 0], x[2, -1] = inf, nan
    x[3, 1] = nan
    x[4] = -inf
    x[5, 2] = inf
    x[6], x[6, 3] = -inf, 1.5
    for dtype in (BF16, F16, F32):
        lse = ops.choose_experts(x.to(dtype).cuda(), 2, score=score, want_lse=True)[3].cpu()
        want = torch.logsumexp(x.double(), 1)
        assert torch.equal(lse.isnan(), want.isnan()) and lse[:4].isnan().all()
        assert torch.equal(lse[4:6].double(), want[4:6]) and torch.allclose(lse[6:].double(), want[6:], rtol=24 * 2.0 ** -23, atol=0)


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('p', [0, 1, 2])
def test_gradient(shape, score, dtype, p):
    tokens, experts, top_k, groups, top_groups, best = shape
    g = torch.Generator().manual_seed(experts * 5 + tokens)
    x = (torch.randn(tokens, experts, generator=g) * 1.5).to(dtype)
    gs, gw, gl = torch.randn(tokens, experts, generator=g).to(dtype), torch.randn(tokens, top_k, generator=g).to(dtype), torch.randn(tokens, generator=g)
    print(f'gradient {shape} {score} {dtype} {p}', flush=True)
    leaf = x.cuda().requires_grad_()
    bias = (torch.randint(-40, 41, (experts,), generator=g) * 0.001).cuda()
    s, w, i, lse = ops.choose_experts(leaf, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups, group_best=best, norm_p=p, scale=2.5,
                                      want_lse=True)
    # the gradient's terms go through exp, a division and up to 512 additions in fp32, each relative to the terms' sizes
    for grads in ((gs, gw, gl), (None, gw, None), (gs, None, None), (None, None, gl)):
        outs = [(o, d.cuda()) for o, d in zip((s, w, lse), grads) if d is not None]
        got, = torch.autograd.grad([o for o, _ in outs], leaf, [d for _, d in outs], retain_graph=True)
        want, size = oracle.gradient(x, i, score, p, 2.5, *grads)
        assert got.dtype == dtype
        _close(got, want, want.abs() * torch.finfo(dtype).eps / 2 + size * (_spread(x) + 40) * 2.0 ** -22 + _tiny(dtype), 'gradient')


def test_gradient_of_scores_that_are_all_zero_and_of_masked_experts():
    x = torch.full((2, 8), -300.)
    x[1, 4:] = -float('inf')
    leaf = x.cuda().requires_grad_()
    w = ops.choose_experts(leaf, 6, score='sigmoid', norm_p=1)[1]
    grad, = torch.autograd.grad(w.sum() + (w[:, 0] * 3).sum(), leaf)
    assert (grad == 0).all()
    y = torch.zeros(1, 8)
    y[0, 4:] = -float('inf')
    leaf = y.cuda().requires_grad_()
    s, w, i, lse = ops.choose_experts(leaf, 2, score='softmax', norm_p=1, want_lse=True)
    grad, = torch.autograd.grad((w * torch.tensor([[1., 2.]]).cuda()).sum() + lse.sum(), leaf)
    want, _ = oracle.gradient(y, i, 'softmax', 1, 1.0, None, torch.tensor([[1., 2.]]), torch.ones(1))
    assert torch.allclose(grad.cpu().double(), want, atol=1e-6)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('p', [0, 1, 2])
def test_gradient_of_the_gradient(score, p):
    """A backward that is differentiated itself: against autograd's of the formula in float64.  fp32 sums of 12 terms, twice."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(5, 12, generator=g)
    gs, gw, gl, v = torch.randn(5, 12, generator=g), torch.randn(5, 3, generator=g), torch.randn(5, generator=g), torch.randn(5, 12, generator=g)
    leaf = x.cuda().requires_grad_()
    s, w, i, lse = ops.choose_experts(leaf, 3, score=score, norm_p=p, scale=1.5, want_lse=True)
    plain, = torch.autograd.grad([s, w, lse], leaf, [gs.cuda(), gw.cuda(), gl.cuda()], retain_graph=True)
    first, = torch.autograd.grad([s, w, lse], leaf, [gs.cuda(), gw.cuda(), gl.cuda()], create_graph=True)
    second, = torch.autograd.grad(first, leaf, v.cuda())
    wide = x.double().requires_grad_()
    t = torch.softmax(wide, 1) if score == 'softmax' else torch.sigmoid(wide)
    u = t.gather(1, i.cpu())
    u = 1.5 * (u / u.norm(p=p, dim=1, keepdim=True) if p else u)
    want, = torch.autograd.grad([t, u, torch.logsumexp(wide, 1)], wide, [gs.double(), gw.double(), gl.double()], create_graph=True)
    want_second, = torch.autograd.grad(want, wide, v.double())
    assert torch.allclose(plain, first, rtol=1e-5, atol=1e-5) and torch.allclose(first.cpu().double(), want, rtol=1e-5, atol=1e-5)
    assert torch.allclose(second.cpu().double(), want_second, rtol=1e-4, atol=1e-4)
    both, = torch.autograd.grad([s, w, lse], leaf, [torch.stack([t, 2 * t]).cuda() for t in (gs, gw, gl)], is_grads_batched=True)
    assert torch.allclose(both[0], plain, rtol=1e-5, atol=1e-5) and torch.allclose(both[1], 2 * plain, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('p', [1, 2, 8])
def test_norms_of_the_smallest_scores(p):
    """Sigmoid scores of 1e-26 have squares below fp32 and weights all the same: off by the exponentials (the last bits of 60 as fp32, 2^-24 60, and 2^-22 of
    their own) and the norm's powers (as much); scores of zero have weights and gradients of zero, the gradients' gradients too."""
    x = torch.tensor([[-60.5, -60., -61.25, -90.], [-200., -200., -300., -250.], [1., 2., -3., 0.]])
    leaf = x.cuda().requires_grad_()
    s, w, i, _ = ops.choose_experts(leaf, 3, score='sigmoid', norm_p=p)
    wide = x.double().requires_grad_()
    u = torch.sigmoid(wide).gather(1, i.cpu())
    most = u.detach().amax(1, keepdim=True)
    u = u / (most * ((u / most) ** p).sum(1, keepdim=True) ** (1 / p))
    real = torch.tensor([0, 2])
    assert i[0].tolist() == [1, 0, 2] and not w[1].any()
    assert torch.allclose(w[real].cpu().double(), u[real], rtol=2e-5, atol=0)
    dy, v = torch.tensor([[1., -2., .5]] * 3), torch.tensor([[.5, 1., -1., 2.]] * 3)
    plain, = torch.autograd.grad(w, leaf, dy.cuda(), retain_graph=True)
    first, = torch.autograd.grad(w, leaf, dy.cuda(), create_graph=True)
    second, = torch.autograd.grad(first, leaf, v.cuda())
    want, = torch.autograd.grad(u, wide, dy.double(), create_graph=True)
    want_second, = torch.autograd.grad(want, wide, v.double())
    for got, is_ in ((plain, want), (first, want), (second, want_second)):
        assert not got[1].any() and torch.allclose(got[real].cpu().double(), is_[real], rtol=1e-4, atol=1e-4)


def test_more_tokens_than_a_launch():
    """2^23 workgroups of 4 tokens are one launch: the last tokens of the first and those of the second, each with its own choice."""
    tokens = 2**25 + 3
    x = torch.zeros(tokens, 17, device='cuda', dtype=torch.bfloat16)
    t = torch.arange(tokens, device='cuda')
    x[t, t % 17] = 2.
    x.requires_grad_()
    _, w, i, _ = ops.choose_experts(x, 1, score='sigmoid', groups=17, top_groups=1, group_best=1)
    assert torch.equal(i[:, 0], t % 17)
    w.backward(torch.ones_like(w))
    own = x.grad[t, t % 17]
    assert bool((own == own[0]).all()) and own[0] > 0 and int((x.grad != 0).sum()) == tokens


def test_no_derivative_forward():
    x = torch.randn(3, 8, device='cuda')
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            ops.choose_experts(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), 2)
        assert torch.equal(ops.choose_experts(x, 2)[1], ops.choose_experts(x.clone(), 2)[1])


def test_strides_types_and_no_tokens():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(37, 80, generator=g)
    view = wide.cuda()[:, 3:67]                      # rows that are no whole pieces
    plain = wide[:, 3:67].contiguous()
    for a, b in zip(ops.choose_experts(view, 4, score='sigmoid'), ops.choose_experts(plain.cuda(), 4, score='sigmoid')):
        assert a is b is None or torch.equal(a, b)
    flat = torch.zeros(37 * 64 + 1, device='cuda')
    flat[1:] = plain.flatten().cuda()
    off = flat[1:].view(37, 64)                      # a base that is no whole piece
    assert torch.equal(ops.choose_experts(off, 4)[2], ops.choose_experts(plain.cuda(), 4)[2])
    s, w, i, lse = ops.choose_experts(torch.zeros(0, 8, device='cuda'), 2, want_lse=True)
    assert s.shape == (0, 8) and w.shape == i.shape == (0, 2) and lse.shape == (0,)
    bias = torch.randn(64, 2, generator=g).cuda()[:, 0]
    assert torch.equal(ops.choose_experts(plain.cuda(), 4, bias=bias)[2], ops.choose_experts(plain.cuda(), 4, bias=bias.contiguous())[2])
    with pytest.raises(RuntimeError):
        ops.choose_experts(torch.zeros(2, 8, device='cuda', dtype=torch.float64), 2)
    with pytest.raises(RuntimeError):
        ops.choose_experts(torch.zeros(2, 8, device='cuda'), 2, bias=torch.zeros(8, device='cuda').half())


def test_rows_behind_the_last_token_are_left_as_they_were():
    from megablocks_amd import _lib
    tokens, experts, top_k = 21, 16, 2
    x = torch.randn(tokens, experts, device='cuda')
    full = [torch.full((tokens + 11, n), 7, dtype=d, device='cuda') for n, d in ((experts, F32), (top_k, F32), (top_k, torch.int64), (top_k, torch.int32), (1, F32))]
    grad = torch.full((tokens + 11, experts), 7., device='cuda')
    _lib.check(_lib.lib.mbx_choose_experts(x.data_ptr(), 2, tokens, experts, top_k, 1, None, 4, 2, 2, 1., 1., *(t.data_ptr() for t in full), _lib.stream()))
    _lib.check(_lib.lib.mbx_choose_experts_backward(full[1].data_ptr(), None, None, x.data_ptr(), full[2].data_ptr(), 2, tokens, experts, top_k, 1, 1., 1.,
                                                    grad.data_ptr(), _lib.stream()))
    for t in (*full, grad):
        assert (t[tokens:] == 7).all() and not (t[:tokens] == 7).all()


def test_a_large_batch_and_a_captured_one():
    g = torch.Generator().manual_seed(21)
    x = torch.randn(70001, 16, generator=g).to(BF16)
    bias = torch.randint(-40, 41, (16,), generator=g) * 0.001
    got = ops.choose_experts(x.cuda(), 2, score='sigmoid', bias=bias.cuda(), groups=4, top_groups=2, norm_p=1)
    some = torch.cat([torch.arange(0, 50), torch.arange(65500, 65600), torch.arange(69950, 70001)])
    assert torch.equal(got[2].cpu()[some], oracle.choose(x[some], 2, 'sigmoid', bias, 4, 2, 2, 1)[2])
    static, grad = x[:300].cuda().requires_grad_(), torch.randn(300, 2, generator=g).to(BF16).cuda()

    def step(leaf):
        s, w, i, _ = ops.choose_experts(leaf, 2, score='sigmoid', bias=device_bias, norm_p=1)
        return s.detach(), w.detach(), i, torch.autograd.grad(w, leaf, grad)[0]
    device_bias = bias.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for first in (0, 1000, 40000):
        new = x[first:first + 300].cuda()
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(new.requires_grad_())):
            assert torch.equal(a, b)


@pytest.mark.parametrize('layers,experts', [(1, 1), (1, 64), (2, 12), (32, 256), (65, 300), (130, 8)])
def test_balance(layers, experts):
    g = torch.Generator().manual_seed(layers)
    biases = [torch.randn(experts, generator=g) * 0.01 for _ in range(layers)]
    counts = [torch.randint(0, 4, (experts,) if l % 3 else (3, experts), generator=g).int() for l in range(layers)]
    counts[0] = torch.full((experts,), 2 ** 31 - 1, dtype=torch.int32)     # sums pass 32 bits; all at the mean
    got = ops.balance_bias([b.cuda() for b in biases], [n.cuda() for n in counts], 0.001)
    again = [b.cuda() for b in biases]
    assert ops.balance_bias(again, [n.cuda() for n in counts], 0.001, out=again) is again
    for b, n, a, c in zip(biases, counts, got, again):
        want = oracle.balance(b, n, 0.001)
        assert (a.cpu().double() - want).abs().max() <= 2.0 ** -24 * (want.abs().max() + 0.001) and torch.equal(a, c)   # one rounding, and the rate's own
    assert torch.equal(got[0].cpu(), biases[0])


def test_balance_refuses_two_layers_with_one_output():
    b, n = torch.zeros(8, device='cuda'), torch.zeros(8, dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError):
        ops.balance_bias([b, b], [n, n], 0.001, out=[b, b])
    with pytest.raises(ValueError):
        ops.balance_bias([b], [n], 0.001, out=[torch.zeros(16, device='cuda')[::2]])
    with pytest.raises(RuntimeError):
        ops.balance_bias([b], [n.cpu()], 0.001)


@pytest.mark.parametrize('experts,spread', [(256, 0.02), (256, 0.1), (512, 0.02), (64, 0.02)])
def test_flat_scores_with_a_bias_of_zero(experts, spread):
    """Where training starts: softmax scores of many experts that are nearly alike, most tokens within what 32 bits tell apart.  With a bias of zero everywhere the
    order is that of the logits."""
    x = torch.randn(4099, experts, generator=torch.Generator().manual_seed(experts)) * spread
    for dtype in (F32, BF16):
        logits = x.to(dtype)
        want = logits.double().sort(dim=1, descending=True, stable=True).indices[:, :8]
        assert torch.equal(ops.choose_experts(logits.cuda(), 8, bias=torch.zeros(experts, device='cuda'))[2].cpu(), want)
