"""The norm of many tensors together and clipping by it, against 64 bits.

Tolerances: a norm is a sum in 64 bits rounded to fp32 once, 2^-24 of it (and 2^-40 for the sum).  A clipped value is off by the norm's rounding, those of the
sum with 1e-6, of the quotient and of the product, 2^-24 each, and by half a step of its own type."""
import math

import pytest
import torch

import megablocks_amd.ops as ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
STEP = 2.0 ** -24


def make(sizes, dtypes, std=1.0, offset=0):
    g = torch.Generator(device='cuda').manual_seed(sum(sizes) + 7)
    made = []
    for i, n in enumerate(sizes):
        dtype = dtypes[i % len(dtypes)]
        buffer = (torch.randn(n + offset, generator=g, device='cuda') * std).to(dtype)
        made.append(buffer[offset:])
    return made


def exact_norm(tensors, p):
    if not any(t.numel() for t in tensors):
        return 0.0
    flat = torch.cat([t.detach().double().abs().flatten() for t in tensors])
    return flat.max().item() if p == math.inf else flat.sum().item() if p == 1 else flat.square().sum().sqrt().item()


def check_norm(got, want):
    assert got.dtype == FP32 and got.shape == ()
    assert abs(got.item() - want) <= want * (STEP + 2.0 ** -40) + 2.0 ** -149


def check_clipped(got, before, most, norm):
    by = min(1.0, most / (norm + 1e-6))
    for o, t in zip(got, before):
        want = t.double() * by
        info = torch.finfo(o.dtype)
        off = want.abs() * (5 * STEP + info.eps / 2) + info.tiny * info.eps
        assert ((o.double() - want).abs() <= off).all()


SIZES = [[1], [7], [8], [2047], [16384], [16385], [5 * 16384 + 3], [1, 0, 3, 70000, 1], [31] * 300, [100003, 5, 262144, 1], [3_000_001, 17], [0, 0], [1 << 24]]


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('dtypes', [(BF16,), (FP16,), (FP32,), (BF16, FP32, FP16)], ids=['bf16', 'fp16', 'fp32', 'mixed'])
@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: f'{len(s)}x{sum(s)}')
def test_norm(sizes, dtypes, p):
    tensors = make(sizes, dtypes)
    check_norm(ops.global_norm(tensors, p), exact_norm(tensors, p))


@pytest.mark.parametrize('out', ['in place', BF16, FP16, FP32], ids=str)
@pytest.mark.parametrize('dtypes', [(BF16,), (FP16,), (FP32,), (BF16, FP32, FP16)], ids=['bf16', 'fp16', 'fp32', 'mixed'])
@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: f'{len(s)}x{sum(s)}')
def test_clip(sizes, dtypes, out):
    for p, short in ((2.0, False), (2.0, True), (1.0, False), (math.inf, False)):
        tensors = make(sizes, dtypes)
        before = [t.clone() for t in tensors]
        norm = exact_norm(tensors, p)
        most = 2 * norm + 1 if short else 0.3 * norm
        outs = None if out == 'in place' else [torch.full_like(t, 9, dtype=out) for t in tensors]
        check_norm(ops.clip_by_global_norm_(tensors, most, p, out=outs), norm)
        check_clipped(tensors if outs is None else outs, before, most, norm)
        if outs is not None:
            assert all(torch.equal(t, b) for t, b in zip(tensors, before))
        if short and outs is None:
            assert all(torch.equal(t, b) for t, b in zip(tensors, before))


@pytest.mark.parametrize('offset', [1, 2, 3, 5, 7])
@pytest.mark.parametrize('dtypes', [(BF16,), (FP32,), (FP16, FP32)], ids=['bf16', 'fp32', 'mixed'])
def test_tensors_that_start_anywhere_leave_their_neighbours_alone(dtypes, offset):
    sizes = [1, 9, 16391, 40000, 255]
    tensors = make(sizes, dtypes, offset=offset)
    norm = exact_norm(tensors, 2.0)
    buffers = [torch.full((n + 16,), 7.0, device='cuda', dtype=FP32 if i % 2 else t.dtype) for i, (n, t) in enumerate(zip(sizes, tensors))]
    outs = [b[offset:offset + n] for b, n in zip(buffers, sizes)]
    check_norm(ops.clip_by_global_norm_(tensors, 0.5, out=outs), norm)
    check_clipped(outs, tensors, 0.5, norm)
    for b, n in zip(buffers, sizes):
        assert (b[:offset] == 7).all() and (b[offset + n:] == 7).all()


@pytest.mark.parametrize('dtype,value', [(FP32, 1e30), (BF16, 1e30), (FP32, 1e-30), (FP32, 2.0 ** -149), (FP16, 65504.0), (FP16, 2.0 ** -24)])
def test_large_and_small_values_are_not_lost(dtype, value):
    t = torch.full((100_000,), value, device='cuda', dtype=dtype)
    for p in (2.0, 1.0, math.inf):
        check_norm(ops.global_norm([t], p), exact_norm([t], p))


def test_many_small_values_next_to_a_large_one():
    t = torch.full((1 << 24,), 2.0 ** -13, device='cuda')
    t[12345] = 1.0      # the others' squares are below half a step of 1 in fp32, and add up to 1/4
    check_norm(ops.global_norm([t]), math.sqrt(1 + ((1 << 24) - 1) * 2.0 ** -26))


def test_a_tensor_of_more_than_2_to_the_31_values():
    n = (1 << 31) + 12345
    t = torch.ones(n, dtype=BF16, device='cuda')
    t[-3:] = 1024.0
    norm = math.sqrt(n - 3 + 3 * 2.0 ** 20)
    check_norm(ops.global_norm([t]), norm)
    check_norm(ops.clip_by_global_norm_([t], norm / 64), norm)
    # a 64th of each value, by a factor that is off by some steps of fp32 and rounds to it in 8 bits
    assert (t[-3:] == 16.0).all() and (t[:-3] == 2.0 ** -6).all()


@pytest.mark.parametrize('p', [2.0, 1.0, math.inf])
@pytest.mark.parametrize('where', [0, 16383, 99_999, -1])
def test_values_that_are_not_finite(where, p):
    for bad in (math.nan, math.inf, -math.inf):
        tensors = make([100_000, 50], (BF16,))
        tensors[0 if where >= 0 else 1][where] = bad
        norm = ops.clip_by_global_norm_(tensors, 1.0, p)
        if math.isnan(bad):
            assert norm.isnan() and all(t.isnan().all() for t in tensors)
        else:
            assert norm.item() == math.inf
            hit = torch.cat(tensors)
            assert hit.isnan().sum() == 1 and (hit[~hit.isnan()] == 0).all()


def test_as_torch_clips():
    params = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (1000, 3, 70001)]
    other = [torch.nn.Parameter(p.detach().clone()) for p in params] + [torch.nn.Parameter(torch.zeros(4, device='cuda'))]
    for p, q in zip(params, other):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_(params, 2.0)
    got = ops.clip_grad_norm_(iter(other), 2.0, error_if_nonfinite=True)      # the last one has no gradient
    torch.testing.assert_close(got, want, rtol=1e-6, atol=0)                   # torch's sums are fp32
    for p, q in zip(params, other):
        torch.testing.assert_close(q.grad, p.grad, rtol=2e-6, atol=0)
    one = torch.nn.Parameter(torch.zeros(5, device='cuda'))
    one.grad = torch.full((5,), math.nan, device='cuda')
    with pytest.raises(RuntimeError):
        ops.clip_grad_norm_(one, 1.0, error_if_nonfinite=True)
    one.grad = torch.tensor([3., 4., 0., 0., 0.], device='cuda')
    assert ops.clip_grad_norm_(one, 1.0).item() == 5.0


def test_tensors_that_are_not_contiguous():
    base = torch.randn(64, 96, device='cuda')
    tensors = [base.t()[:, ::2], torch.randn(5, 6, 7, device='cuda').permute(2, 0, 1)]
    before = [t.clone() for t in tensors]
    rest = base.t()[:, 1::2].clone()
    norm = exact_norm(tensors, 2.0)
    check_norm(ops.global_norm(tensors), norm)
    check_norm(ops.clip_by_global_norm_(tensors, 1.5), norm)
    check_clipped(tensors, before, 1.5, norm)
    assert torch.equal(base.t()[:, 1::2], rest)
    outs = [torch.empty(96, 64, device='cuda').t()[:, ::3][:48].t(), torch.empty(7, 5, 6, device='cuda', dtype=BF16)]
    tensors = [torch.randn_like(o, dtype=FP32).contiguous() for o in outs]
    norm = exact_norm(tensors, 2.0)
    ops.clip_by_global_norm_(tensors, 1.5, out=outs)
    check_clipped(outs, tensors, 1.5, norm)


def test_refusals():
    a, b = torch.ones(8, device='cuda'), torch.ones(8, device='cuda')
    for tensors, out in (([a, a], None), ([a, a[4:]], None), ([a, b], [a, a]), ([a, b], [b, a]), ([a[:4]], [a[2:6]]), ([a, b], [a]), ([a], [torch.ones(7, device='cuda')]),
                         ([torch.ones(4, 4, device='cuda')[:, ::2]] * 2, None), ([a], [torch.ones(1, device='cuda').expand(8)])):
        with pytest.raises(ValueError):
            ops.clip_by_global_norm_(tensors, 1.0, out=out)
    for tensors in ([a, torch.ones(3)], [a.double()], [a, b.int()], [torch.ones(3, device='cuda', requires_grad=True)]):
        with pytest.raises(RuntimeError):
            ops.global_norm(tensors)
        with pytest.raises(RuntimeError):
            ops.clip_by_global_norm_(tensors, 1.0)
    assert (a == 1).all() and (b == 1).all()
    with torch.no_grad():
        assert ops.global_norm([torch.full((4,), 2.0, device='cuda', requires_grad=True)]).item() == 4.0


def test_written_tensors_have_new_versions():
    a, out = torch.ones(8, device='cuda'), torch.ones(8, device='cuda')
    versions = a._version, out._version
    ops.clip_by_global_norm_([a], 1.0, out=[out])
    assert a._version == versions[0] and out._version == versions[1] + 1
    ops.clip_by_global_norm_([a], 1.0)
    assert a._version == versions[0] + 1
    with torch.inference_mode():
        t = torch.ones(4, device='cuda')
        assert ops.clip_by_global_norm_([t], 1.0).item() == 2.0 and (t - 0.5).abs().max() < 1e-6


def test_the_same_from_run_to_run_and_on_another_stream():
    tensors = make([3_000_001, 17, 70000], (BF16, FP32))
    norms = {ops.global_norm(tensors).item() for _ in range(5)}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        norms.add(ops.global_norm(tensors).item())
    assert len(norms) == 1


def test_captured_and_replayed():
    tensors = make([100_003, 5, 70000], (BF16, FP32))
    outs = [torch.empty_like(t, dtype=FP32) for t in tensors]
    ops.clip_by_global_norm_(tensors, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_by_global_norm_(tensors, 1.0, out=outs)
    for scale in (1.0, 2.0, 1e-6):
        for t in tensors:
            t.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        check_norm(norm, exact_norm(tensors, 2.0))
        check_clipped(outs, tensors, 1.0, exact_norm(tensors, 2.0))
        assert ops.global_norm(tensors).item() == norm.item()


def test_gradients_that_are_slices_of_one_buffer():
    """As torch clips them: parts of a matrix's columns, every other row, and one that is contiguous."""
    params = [torch.nn.Parameter(torch.zeros(64, 48, device='cuda')) for _ in range(2)] + [torch.nn.Parameter(torch.zeros(8, 30, device='cuda')) for _ in range(2)]
    params.append(torch.nn.Parameter(torch.zeros(1000, device='cuda')))
    columns, rows = torch.randn(64, 97, device='cuda'), torch.randn(16, 30, device='cuda')
    grads = [columns[:, :48], columns[:, 49:], rows[::2], rows[1::2], torch.randn(1000, device='cuda')]
    before, between = [g.clone() for g in grads], columns[:, 48].clone()
    for p, g in zip(params, grads):
        p.grad = g
    norm = exact_norm(grads, 2.0)
    check_norm(ops.clip_grad_norm_(params, 2.0), norm)
    check_clipped(grads, before, 2.0, norm)
    assert torch.equal(columns[:, 48], between) and all(p.grad is g for p, g in zip(params, grads))
    for p, b in zip(params, before):
        p.grad = b.clone()
    torch.nn.utils.clip_grad_norm_(params, 2.0)
    for p, g in zip(params, grads):
        torch.testing.assert_close(g, p.grad, rtol=2e-6, atol=0)


def test_outputs_over_strided_tensors_are_refused_before_anything_is_written():
    line = torch.ones(100, device='cuda')
    for tensors, out in (([line[::2]], [line[:50]]), ([torch.ones(50, device='cuda'), line[::2]], [line[20:70], torch.ones(50, device='cuda')]), ([line.as_strided((4, 3), (2, 1))], None)):
        with pytest.raises(ValueError):
            ops.clip_by_global_norm_(tensors, 0.1, out=out)
    assert (line == 1).all()
