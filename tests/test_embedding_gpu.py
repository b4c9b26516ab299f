"""Rows of a table by token and the table's gradient, against 64 bits.

Tolerances: rows are one product in fp32 and one rounding, which torch makes alike: equal.  A gradient's row is a sum of m rows in fp32, off by at most (m - 1)
2^-24 of the sum of magnitudes whatever the order, the product with the scale and the rounding to the table's type."""
import math

import pytest
import torch

import megablocks_amd.ops as ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(tokens, words, hidden, dtype, kind='even', wide=True):
    g = torch.Generator(device='cuda').manual_seed(tokens * 31 + words)
    ids = torch.randint(0, words, (tokens,), generator=g, device='cuda')
    if kind == 'one':             # all the same word
        ids.fill_(words // 2)
    elif kind == 'half':          # one word in two tokens, in runs and alone
        ids[torch.rand(tokens, generator=g, device='cuda') < 0.5] = words - 1
    elif kind == 'few':
        ids = ids % min(words, 3)
    elif kind == 'ascending':
        ids = torch.arange(tokens, device='cuda') * words // max(tokens, 1)
    table = torch.randn(words, hidden, generator=g, device='cuda').to(dtype)
    grad = torch.randn(tokens, hidden, generator=g, device='cuda').to(dtype)
    return ids if wide else ids.int(), table, grad


def exact(ids, grad, words, scale, padding=None):
    """(the gradient in 64 bits, how far fp32 sums may be off it)"""
    ids, g = ids.flatten().long(), grad.reshape(ids.numel(), grad.shape[-1]).double()
    keep = (ids >= 0) & (ids < words)
    if padding is not None:
        keep &= ids != padding
    ids, g = ids[keep], g[keep]
    zeros = lambda: torch.zeros(words, grad.shape[-1], dtype=torch.float64, device=grad.device)
    want, size = zeros().index_add_(0, ids, g) * scale, zeros().index_add_(0, ids, g.abs()) * abs(scale)
    terms = torch.bincount(ids, minlength=words).double().unsqueeze(1)
    info = torch.finfo(grad.dtype)
    return want, size * terms * 2.0 ** -24 + want.abs() * (info.eps / 2 + 2.0 ** -23) + info.tiny * info.eps


def check(ids, table, grad, scale=1.0, padding=None):
    table = table.clone().requires_grad_()
    out = ops.embedding(ids, table, scale, padding)
    assert torch.equal(out, (table.detach()[ids.long()].float() * scale).to(table.dtype))
    out.backward(grad)
    want, off = exact(ids, grad, table.shape[0], scale, padding)
    assert table.grad.dtype == table.dtype
    assert ((table.grad.double() - want).abs() <= off).all()


@pytest.mark.parametrize('dtype', [BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize('tokens,words,hidden', [(1, 1, 8), (1, 50000, 1024), (2, 3, 1), (63, 1000, 64), (64, 70, 7), (65, 257, 513), (300, 255, 2040), (1000, 5, 1032),
                                                 (4097, 30011, 100), (3, 100000, 512), (33, 4, 4100), (20000, 1025, 72),
                                                 (256, 300, 520), (255, 5000, 2056), (257, 300, 520), (258, 70, 7), (300, 3, 1), (321, 257, 513)])
def test_rows_and_gradient(tokens, words, hidden, dtype):
    check(*make(tokens, words, hidden, dtype, wide=tokens % 2 == 0), scale=1.0)


@pytest.mark.parametrize('kind', ['one', 'half', 'few', 'ascending', 'even'])
@pytest.mark.parametrize('tokens,words,hidden', [(31, 9, 40), (32, 9, 40), (33, 9, 40), (64, 9, 40), (200, 30, 1028), (256, 700, 264), (257, 9, 40), (288, 9, 40), (289, 9, 40), (4096, 2000, 264), (9999, 300, 1030), (140000, 5000, 16)])
def test_words_that_come_often(tokens, words, hidden, kind):
    check(*make(tokens, words, hidden, BF16, kind), scale=0.5)


@pytest.mark.parametrize('padding', [0, 17, -1, 99])
@pytest.mark.parametrize('kind', ['half', 'few', 'one'])
@pytest.mark.parametrize('tokens', [3000, 150])
def test_padding_learns_nothing(tokens, kind, padding):
    ids, table, grad = make(tokens, 100, 96, FP16, kind)
    ids[::3] = padding % 100
    check(ids, table, grad, scale=32.0, padding=padding % 100)
    table.requires_grad_()
    ops.embedding(ids, table, padding_idx=padding).backward(grad)
    assert (table.grad[padding] == 0).all()


@pytest.mark.parametrize('dtype', [torch.int32, torch.int64], ids=str)
def test_ids_outside_the_table(dtype):
    ids = torch.tensor([0, -1, 4, 5, -2 ** 31, 2 ** 31 - 1, 1], device='cuda', dtype=dtype)
    if dtype == torch.int64:
        ids = torch.cat([ids, torch.tensor([2 ** 32 + 1, -2 ** 63, 2 ** 62], device='cuda')])
    table = torch.randn(5, 72, device='cuda', requires_grad=True)
    out = ops.embedding(ids, table)
    inside = (ids >= 0) & (ids < 5)
    assert (out[~inside] == 0).all() and torch.equal(out[inside], table[ids[inside].long()])
    grad = torch.randn_like(out)
    out.backward(grad)
    want, off = exact(ids, grad, 5, 1.0)
    assert ((table.grad.double() - want).abs() <= off).all()


@pytest.mark.parametrize('shape', [(), (0,), (2, 0), (3, 5), (2, 3, 4)])
def test_shapes_of_ids(shape):
    ids = torch.randint(0, 11, shape, device='cuda')
    table = torch.randn(11, 24, device='cuda', requires_grad=True)
    out = ops.embedding(ids, table, 2.0)
    assert torch.equal(out, table.detach()[ids] * 2)
    grad = torch.randn_like(out)
    out.backward(grad)
    want, off = exact(ids, grad, 11, 2.0)
    assert ((table.grad.double() - want).abs() <= off).all()


def test_a_table_without_columns_or_words():
    table = torch.empty(4, 0, device='cuda', requires_grad=True)
    out = ops.embedding(torch.zeros(3, dtype=torch.int32, device='cuda'), table)
    assert out.shape == (3, 0)
    out.sum().backward()
    assert table.grad.shape == (4, 0)
    table = torch.empty(0, 8, device='cuda', requires_grad=True)
    out = ops.embedding(torch.zeros(3, dtype=torch.int64, device='cuda'), table)
    assert out.shape == (3, 8) and (out == 0).all()
    out.sum().backward()
    assert table.grad.shape == (0, 8)


def test_layouts():
    ids = torch.randint(0, 50, (40, 30), device='cuda').t()[::2]                 # strided ids
    buffer = torch.randn(50 * 33 + 3, device='cuda').to(BF16)
    table = buffer[3:].view(50, 33)                                             # rows at odd addresses
    check(ids, table, torch.randn(15, 40, 33, device='cuda').to(BF16))
    check(ids, torch.randn(33, 50, device='cuda').t(), torch.randn(40, 15, 33, device='cuda').transpose(0, 1))
    check(ids, torch.randn(50, 66, device='cuda')[:, ::2], torch.randn(33, device='cuda').expand(15, 40, 33))


def test_a_table_of_more_than_2_to_the_31_values():
    words, hidden = (1 << 20) + 7, 2056
    table = torch.zeros(words, hidden, dtype=BF16, device='cuda')
    ids = torch.tensor([words - 1, 0, words - 2, words - 1, 1 << 20, 77], device='cuda')
    table[ids] = torch.randn(len(ids), hidden, device='cuda').bfloat16()
    grad = torch.randn(len(ids), hidden, device='cuda').bfloat16()
    table.requires_grad_()
    out = ops.embedding(ids, table)
    assert torch.equal(out, table.detach()[ids])
    got, = torch.autograd.grad(out, table, grad)
    named = ids.unique()
    assert torch.equal(got.any(1).nonzero().flatten(), named)
    want, off = exact((ids.unsqueeze(1) == named).int().argmax(1), grad, len(named), 1.0)
    assert ((got[named].double() - want).abs() <= off).all()


def test_rows_of_more_than_2_to_the_31_values():
    """Counts are exact in fp32, up to 2^24, and so are their parts."""
    tokens, hidden = (1 << 20) + 7, 2056
    ids = torch.randint(0, 3, (tokens,), device='cuda')
    table = torch.randn(3, hidden, device='cuda').bfloat16().requires_grad_()
    out = ops.embedding(ids, table)
    assert torch.equal(out, table.detach()[ids])
    grad = torch.ones_like(out)
    grad[-1, -1] = 0
    got, = torch.autograd.grad(out, table, grad)
    want = torch.bincount(ids, minlength=3).unsqueeze(1).repeat(1, hidden)
    want[ids[-1], -1] -= 1
    assert torch.equal(got, want.float().bfloat16())


def test_more_tokens_than_a_list_counts():
    """Sixteen shares of more than 2^22 tokens."""
    tokens = (1 << 26) + 12345
    ids = torch.randint(0, 13, (tokens,), device='cuda', dtype=torch.int32)
    table = torch.zeros(13, 1, device='cuda', requires_grad=True)
    grad = (torch.arange(tokens, device='cuda') % 5 == 0).float().unsqueeze(1)      # sums below 2^24
    got, = torch.autograd.grad(ops.embedding(ids, table), table, grad)
    assert torch.equal(got.flatten().long(), torch.bincount(ids[::5], minlength=13))


def test_sums_are_not_in_16_bits():
    ids = torch.zeros(40000, dtype=torch.int64, device='cuda')
    table = torch.zeros(2, 8, device='cuda', dtype=BF16, requires_grad=True)
    ops.embedding(ids, table).backward(torch.ones(40000, 8, device='cuda', dtype=BF16))
    assert (table.grad[0] == 40000 // 256 * 256).all()       # 40000 to the nearest of steps of 256


def test_the_same_from_run_to_run():
    ids, table, grad = make(30000, 500, 200, FP32, 'half')
    table.requires_grad_()
    grads = [torch.autograd.grad(ops.embedding(ids, table), table, grad)[0] for _ in range(4)]
    assert all(torch.equal(g, grads[0]) for g in grads)


def test_gradients_of_the_gradient_and_differences():
    ids = torch.tensor([[1, 3, 3], [0, 1, 4]], device='cuda')
    table = torch.randn(5, 3, device='cuda', requires_grad=True)
    x = ops.embedding(ids, table, 1.5, padding_idx=4)
    loss = (x ** 3).sum()
    g, = torch.autograd.grad(loss, table, create_graph=True)
    v = torch.randn_like(g)
    got, = torch.autograd.grad((g * v).sum(), table)
    # torch's own operations; the padding row is a constant
    leaf = table.detach().double().requires_grad_()
    fixed = torch.cat([leaf[:4], leaf[4:].detach()])
    loss = ((1.5 * fixed[ids]) ** 3).sum()
    want, = torch.autograd.grad(loss, leaf, create_graph=True)
    torch.testing.assert_close(g.double(), want, rtol=1e-5, atol=1e-5)
    want, = torch.autograd.grad((want * v.double()).sum(), leaf)
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-5)
    d = torch.randn_like(table)
    d[4] = 0
    with torch.no_grad():     # central differences of a cubic: off by h^2 times its third derivative
        f = lambda t: (ops.embedding(ids, t, 1.5).double() ** 3).sum()
        h = 2.0 ** -7
        slope = (f(table + h * d) - f(table - h * d)) / (2 * h)
    third = 18 * 1.5 ** 3 * d.abs().max() ** 3
    assert abs(slope - (g * d).sum()) <= h * h / 6 * third + 2e-3 * (g * d).abs().sum()      # fp32 rows, differences of 2^-6


def test_other_streams_and_replays():
    ids, table, grad = make(5000, 700, 264, BF16, 'half')
    table.requires_grad_()
    want_out = ops.embedding(ids, table)
    want, = torch.autograd.grad(want_out, table, grad)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got, = torch.autograd.grad(ops.embedding(ids, table), table, grad)
    stream.synchronize()
    assert torch.equal(got, want)
    del want_out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.embedding(ids, table)
        got, = torch.autograd.grad(out, table, grad)
    for turn in range(3):
        ids.copy_(ids.roll(turn * 77))
        grad.copy_(grad.roll(turn, 0))
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.embedding(ids, table)
        assert torch.equal(out, eager) and torch.equal(got, torch.autograd.grad(eager, table, grad)[0])


def test_refusals_on_the_gpu():
    ids, table = torch.zeros(3, dtype=torch.int64, device='cuda'), torch.zeros(5, 8, device='cuda')
    for bad in (dict(ids=ids.short()), dict(ids=ids.float()), dict(table=table.double()), dict(ids=ids.cpu()), dict(table=table.cpu())):
        with pytest.raises(RuntimeError):
            ops.embedding(**(dict(ids=ids, table=table) | bad))


def test_inference_mode():
    with torch.inference_mode():
        ids, table = torch.arange(4, device='cuda'), torch.randn(5, 8, device='cuda')
        assert torch.equal(ops.embedding(ids, table), table[:4])


def used_memory(*shape, **kw):
    """What a tensor of this shape is likely to be made of next: no zeros."""
    torch.full(shape, 9.0, device='cuda', **kw)


def test_rows_of_more_workgroups_than_a_launch_has_threads_for():
    """A launch has fewer than 2^32 threads, of which a token takes 64 at least."""
    tokens = (1 << 26) + 12345
    ids = torch.randint(0, 13, (tokens,), device='cuda', dtype=torch.int32)
    table = torch.arange(1.0, 14.0, device='cuda').unsqueeze(1)
    used_memory(tokens, 1)
    assert torch.equal(ops.embedding(ids, table).flatten(), ids.float() + 1)


@pytest.mark.parametrize('tokens,words', [(300, (1 << 27) + 77), (5, (1 << 28) + 77), (0, (1 << 28) + 77)])
def test_gradients_of_more_workgroups_than_a_launch_has_threads_for(tokens, words):
    """Rows of zeros too: eight words a workgroup next to the sums, sixteen where there are few tokens."""
    ids = torch.randint(words - 1000, words, (tokens,), device='cuda')
    ids[:tokens // 2] %= 1000
    table = torch.zeros(words, 1, device='cuda', dtype=BF16, requires_grad=True)
    out = ops.embedding(ids, table)
    grad = torch.randint(1, 4, out.shape, device='cuda').to(BF16)
    used_memory(words, 1, dtype=BF16)
    got, = torch.autograd.grad(out, table, grad)
    assert torch.equal(got.flatten().nonzero().flatten(), ids.unique())
    named = ids.unique()
    want, off = exact((ids.unsqueeze(1) == named).int().argmax(1) if tokens else ids, grad, len(named), 1.0)
    assert ((got[named].double() - want).abs() <= off).all()


@pytest.mark.parametrize('kind', ['one', 'half', 'few', 'even', 'text'])
@pytest.mark.parametrize('tokens,words,hidden', [(2, 3, 9), (100, 30, 1028), (256, 700, 264), (257, 9, 40), (9999, 300, 1030), (16384, 50000, 256), (40000, 5000, 128)])
def test_fp32_gradients_are_rounded_once(tokens, words, hidden, kind):
    """Sums in 64 bits, 2^-53 of the magnitudes a term, rounded to fp32 at the end: half a step of 2^-24, and what the 64 bits are off by."""
    ids, table, grad = make(tokens, words, hidden, FP32, 'even' if kind == 'text' else kind)
    if kind == 'text':       # the p-th most frequent word with a probability of about 1 / p
        ids = (torch.rand(tokens, device='cuda', dtype=torch.float64) * math.log(words + 1)).exp().long().clamp(1, words) - 1
    table.requires_grad_()
    got, = torch.autograd.grad(ops.embedding(ids, table, 3.0), table, grad)
    zeros = lambda: torch.zeros(words, hidden, dtype=torch.float64, device='cuda')
    want, size = zeros().index_add_(0, ids, grad.double()) * 3.0, zeros().index_add_(0, ids, grad.double().abs()) * 3.0
    terms = torch.bincount(ids, minlength=words).double().unsqueeze(1)
    assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -24 + 2 * (terms + 2) * 2.0 ** -53 * size).all()


@pytest.mark.parametrize('tokens', [40, 3000])
def test_several_gradients_at_once(tokens):
    ids, table, _ = make(tokens, 50, 24, FP32, 'half')
    ids[5] = -1
    table.requires_grad_()
    out = ops.embedding(ids, table, 1.5, padding_idx=3)
    grads = torch.randn(3, tokens, 24, device='cuda')
    got, = torch.autograd.grad(out, table, grads, is_grads_batched=True, retain_graph=True)
    want = torch.stack([torch.autograd.grad(out, table, g, retain_graph=True)[0] for g in grads])
    torch.testing.assert_close(got, want, rtol=2.0 ** -23, atol=1e-12)        # either is the sum in 64 bits, rounded once
    # a gradient's gradient, of several vectors at once: rows of the vectors by token, added up by word again
    first, = torch.autograd.grad((ops.embedding(ids, table, 1.5, padding_idx=3) ** 2).sum(), table, create_graph=True)
    vectors = torch.randn(2, 50, 24, device='cuda')
    got, = torch.autograd.grad(first, table, vectors, is_grads_batched=True, retain_graph=True)
    want = torch.stack([torch.autograd.grad(first, table, v, retain_graph=True)[0] for v in vectors])
    torch.testing.assert_close(got, want, rtol=2.0 ** -21, atol=1e-12)
    # and the gradients of several gradients themselves
    weights = torch.randn(tokens, 24, device='cuda', requires_grad=True)
    both, = torch.autograd.grad(ops.embedding(ids, table, 1.5, padding_idx=3), table, torch.stack([weights, 2 * weights]), is_grads_batched=True, create_graph=True)
    got, = torch.autograd.grad(both.sum(), weights)
    counts = (ids >= 0) & (ids != 3)
    torch.testing.assert_close(got, 4.5 * counts.unsqueeze(1).float().expand(tokens, 24), rtol=0, atol=0)
