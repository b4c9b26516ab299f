"""4-bit weights on the GPU: quantising and the values back, bit for bit; products against float64.

Tolerance of a product.  The kernels sum x (16 + q) and x over the groups in fp32 and take their difference: every x counts with up to 31 in the first
and up to 31 in the second sum, a group's sums have up to 128 terms, each addition off by 2^-24 of what has been added so far at most, and up to k / 32
groups are added up: off by at most 2^-24 (2 * 31 * 128 + 31 k / 32) of the sum of |scale x|.  The result is rounded by half a step."""
import pytest
import torch

from megablocks_amd import grouped_gemm_util as gg
from oracle import weights_4bit as oracle

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
@pytest.mark.parametrize('trans_b', [True, False])
@pytest.mark.parametrize('zero_points', [False, True])
@pytest.mark.parametrize('shape,group', [((1, 1, 1), 32), ((2, 16, 128), 128), ((3, 64, 256), 64), ((1, 72, 136), 32), ((2, 33, 129), 64), ((1, 130, 515), 128),
                                         ((5, 17, 31), 32)])
def test_quantized_weights(shape, group, zero_points, trans_b, dtype):
    g = torch.Generator().manual_seed(shape[1] + shape[2])
    w = (torch.randn(shape, generator=g) * torch.rand(shape[0], shape[1], 1, generator=g)).to(dtype)
    w[:, :, ::3] = (w[:, :, ::3] * 8).round() / 8                     # quotients half way between two codes
    w[-1, -1] = 0
    w[0, 0, :5] = torch.tensor([7., 3.5, -2.5, 0.5, 1.5][:shape[2]]).to(dtype)[:shape[2]]
    print(f'quantize {shape} {group} {zero_points} {trans_b} {dtype}', flush=True)
    kept = gg.quantize_4bit((w if trans_b else w.transpose(1, 2)).cuda(), group, trans_b, zero_points)
    codes, scales, zeros = oracle.quantize(w, group, zero_points)
    assert torch.equal(kept.group_scales().cpu(), scales)
    assert torch.equal(oracle.unpack(kept.words, *shape[1:]), codes)
    if zero_points:
        assert torch.equal(kept.zeros.cpu().transpose(2, 3).flatten(1, 2)[:, :shape[1], :scales.shape[2]].long(), zeros)
    want = oracle.values(codes, scales, zeros, group).float()         # a scale of 24 bits and four more: the product of two is rounded once
    for out in (dtype, F32):
        for layout in (True, False, None):
            got = kept.dequantize(out, layout).cpu()
            got = got if layout or (layout is None and trans_b) else got.transpose(1, 2)
            assert got.dtype == out and torch.equal(got, want.to(out))


def test_scales_next_to_a_rounding():
    """A distance whose fifteenth lies half way between two numbers of the type: by the reciprocal in fp32, as torch on the GPU divides by a number."""
    w = torch.zeros(1, 1, 32, dtype=BF16)
    w[0, 0, 3], w[0, 0, 9] = -0.033203125, 0.00124359130859375
    kept = gg.quantize_4bit(w.cuda(), 32, True, True)
    assert kept.group_scales().item() == 0.0023040771484375 == oracle.quantize(w, 32, True)[1].item()
    w = torch.zeros(1, 1, 32, dtype=F16)               # here the product in fp32 is half way itself: to even, as it is rounded twice
    w[0, 0, 3], w[0, 0, 9] = -0.03240966796875, 0.0007925033569335938
    kept = gg.quantize_4bit(w.cuda(), 32, True, True)
    assert kept.group_scales().item() == 0.0022125244140625 == oracle.quantize(w, 32, True)[1].item()
    for dtype in (BF16, F16):                          # distances of every last place
        high = (torch.arange(2 ** 11, 2 ** 12, dtype=torch.float64) / 2 ** 12).to(dtype)[:, None]
        low = -(torch.arange(1, 2 ** 8, 23, dtype=torch.float64) / 2 ** 12).to(dtype)[None]
        w = torch.zeros(1, high.numel() * low.numel(), 32, dtype=dtype)
        w[0, :, 0], w[0, :, 1] = high.expand(-1, low.numel()).flatten(), low.expand(high.numel(), -1).flatten()
        for zero_points in (True, False):
            codes, scales, _ = oracle.quantize(w, 32, zero_points)
            kept = gg.quantize_4bit(w.cuda(), 32, True, zero_points)
            assert torch.equal(kept.group_scales().cpu(), scales) and torch.equal(oracle.unpack(kept.words, w.shape[1], 32), codes)
    x = torch.rand(1 << 20, generator=torch.Generator().manual_seed(13)).cuda()
    for zero_points, by in ((True, 15), (False, 7)):
        kept = gg.quantize_4bit(torch.nn.functional.pad(x[None, :, None], (0, 31)), 32, True, zero_points)
        assert torch.equal(kept.group_scales().flatten(), x / by)


@pytest.mark.parametrize('dtype', [BF16, F16, F32])
def test_groups_that_are_not_finite_tiny_or_huge(dtype):
    w = torch.ones(1, 8, 96, dtype=dtype)
    w[0, 0, 3], w[0, 1, 40], w[0, 2, 95] = float('nan'), float('inf'), -float('inf')
    w[0, 3] = torch.finfo(dtype).smallest_normal / 4 * torch.arange(96) / 95           # not normal
    w[0, 4] = torch.finfo(dtype).max
    w[0, 5, ::2] = -torch.finfo(dtype).max
    w[0, 6] = 0.
    for zero_points in (False, True):
        if dtype != F16 and zero_points:
            w[0, 5] = 1.           # the distance of the extremes is no number of 32 bits
        kept = gg.quantize_4bit(w.cuda(), 32, True, zero_points)
        codes, scales, zeros = oracle.quantize(w, 32, zero_points)
        got = kept.group_scales().cpu()
        assert torch.equal(got.isnan(), scales.isnan()) and torch.equal(got.nan_to_num(), scales.nan_to_num())
        assert torch.equal(oracle.unpack(kept.words, 8, 96), codes)
        values = kept.dequantize(F32).cpu()
        assert values[0, 0, :32].isnan().all() and values[0, 0, 32:].isfinite().all() and values[0, 2, 64:].isnan().all() and (values[0, 6] == 0).all()


def _weights(experts, n, k, group, zeros, scale_dtype, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (experts, n, k), generator=g)
    whole = -(-k // 128) * 128
    scales = ((torch.rand(experts, n, whole // group, generator=g) + 0.2) * 0.01).to(scale_dtype)
    z = torch.randint(0, 16, scales.shape, generator=g) if zeros else None
    kept = gg.Weights4bit(oracle.pack(codes).cuda(), oracle.kept(scales).cuda(), None if z is None else oracle.kept(z).to(torch.uint8).cuda(), n, k, group)
    cut = lambda t: None if t is None else t[:, :, :-(-k // group)]
    return kept, oracle.values(codes, cut(scales), cut(z), group), scales.double().repeat_interleave(group, 2)[:, :, :k]


def _products(rows, counts, values, sizes):
    """(float64 products, what they may be off by before they are rounded)."""
    k = rows.shape[1]
    per = torch.tensor(counts)
    expert = torch.repeat_interleave(torch.arange(len(counts)), per)
    want, off = (torch.zeros(len(rows), values.shape[1], dtype=torch.float64) for _ in range(2))
    for e in range(len(counts)):
        x = rows[expert == e].double()
        want[expert == e] = x @ values[e].t()
        off[expert == e] = 2.0 ** -24 * (2 * 31 * 128 + 31 * k / 32) * (x.abs() @ sizes[e].abs().t())
    return want, off


def _close(got, want, off, dtype):
    bound = off + torch.finfo(dtype).eps / 2 * (want.abs() + off) + (2.0 ** -24 if dtype == F16 else 0)
    wrong = (got.double().cpu() - want).abs() / bound.clamp(min=1e-300)
    assert got.dtype == dtype and float(wrong.max() if wrong.numel() else 0) <= 1, float(wrong.max())


CASES = [   # counts of rows, n, k, group
    ([1], 16, 128, 128), ([0, 1, 0, 2], 48, 256, 64), ([5, 0, 16, 17], 33, 200, 32), ([1, 1, 1, 1, 1, 1], 130, 515, 128), ([40, 3], 64, 136, 64),
    ([0, 64, 65, 1], 40, 384, 32), ([130], 24, 72, 32), ([3] * 70, 17, 31, 64), ([0, 0, 0], 16, 16, 32), ([9, 200, 0, 31], 56, 1032, 128), ([2, 1], 1, 1, 32),
    ([33, 33], 8, 2048, 128), ([97], 16, 128, 128), ([120, 96], 72, 8, 32), ([300, 0, 100], 130, 520, 64), ([1000, 50], 56, 392, 128), ([63, 129], 300, 1032, 32),
    ([250], 40, 129, 128), ([100, 97, 192], 272, 1152, 64)]


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('wide', [False, True])
@pytest.mark.parametrize('case', CASES)
def test_product(case, wide, zeros, dtype):
    counts, n, k, group = case
    print(f'product {case} wide={wide} zeros={zeros} {dtype}', flush=True)
    kept, values, sizes = _weights(len(counts), n, k, group, zeros, F32 if wide else dtype, seed=n + k)
    x = torch.randn(sum(counts), k, generator=torch.Generator().manual_seed(k)).to(dtype)
    want, off = _products(x, counts, values, sizes)
    _close(gg.gmm_4bit(x.cuda(), kept, torch.tensor(counts)), want, off, dtype)
    bins = torch.tensor(counts).cumsum(0).int().cuda()
    _close(gg.gmm_4bit(x.cuda(), kept, bins=bins), want, off, dtype)
    assert torch.equal(gg.gmm_4bit(x.cuda(), kept, bins=bins), gg.gmm_4bit(x.cuda(), kept, torch.tensor(counts).cuda()))


def _routed(tokens, experts, top_k, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens * top_k,), generator=g)
    bin_ids, indices = ids.sort(stable=True)
    counts = torch.bincount(ids, minlength=experts)
    return indices.int(), bin_ids.int(), counts.cumsum(0).int(), counts.tolist()


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('act', [gg.ACT_SILU, gg.ACT_GELU_TANH])
@pytest.mark.parametrize('tokens,top_k,experts,n,k,group,zeros', [(1, 2, 8, 64, 256, 128, False), (5, 6, 64, 40, 136, 64, True), (70, 2, 3, 33, 129, 32, True),
                                                                  (300, 1, 4, 72, 384, 128, False), (16, 4, 2, 128, 1000, 32, False), (400, 2, 4, 200, 264, 64, True),
                                                                  (500, 2, 3, 70, 512, 128, False), (200, 3, 2, 33, 1000, 32, False)])
def test_first_products_of_gathered_rows(tokens, top_k, experts, n, k, group, zeros, act, gate, dtype):
    print(f'first products {tokens} {top_k} {experts} {n} {k} {group} {zeros} act={act} gate={gate} {dtype}', flush=True)
    indices, bin_ids, bins, counts = _routed(tokens, experts, top_k, tokens)
    made = [_weights(experts, n, k, group, zeros, dtype, seed) for seed in ((1, 2) if gate else (1,))]
    x = torch.randn(tokens, k, generator=torch.Generator().manual_seed(tokens)).to(dtype)
    src = gg.GatheredRows(x.cuda(), indices.cuda(), bin_ids.cuda(), bins.cuda(), None, top_k, tokens * top_k)
    got = gg.gmm_4bit_act(src, made[0][0], act, b2=made[1][0] if gate else None)
    rows = x[indices.long() // top_k]
    a, off = _products(rows, counts, *made[0][1:])
    h = a * torch.sigmoid(a) if act == gg.ACT_SILU else torch.nn.functional.gelu(a, approximate='tanh')
    # both activations rise by 1.13 at most; exp, a division and a cubic in fp32
    off = 1.13 * off + 2.0 ** -20 * (a.abs() + h.abs())
    if gate:
        b, off_b = _products(rows, counts, *made[1][1:])
        off = off * (b.abs() + off_b) + h.abs() * off_b + 2.0 ** -22 * (h * b).abs()
        h = h * b
    _close(got, h, off, dtype)
    assert torch.equal(got, gg.gmm_4bit_act(src.materialize(), made[0][0], act, bins=bins.cuda(), b2=made[1][0] if gate else None))


def test_a_row_does_not_depend_on_the_others():
    """Rows that are not finite stay by themselves, within a tile too."""
    kept, *_ = _weights(2, 32, 200, 64, False, BF16, 3)
    x = torch.randn(21, 200, generator=torch.Generator().manual_seed(4)).bfloat16()
    bins = torch.tensor([10, 21], dtype=torch.int32).cuda()
    want = gg.gmm_4bit(x.cuda(), kept, bins=bins)
    x[4], x[15, 7] = float('nan'), float('inf')
    got = gg.gmm_4bit(x.cuda(), kept, bins=bins)
    others = [r for r in range(21) if r not in (4, 15)]
    assert torch.equal(got[others], want[others]) and got[4].isnan().all() and not got[15].isfinite().any()


def test_bins_that_do_not_fit_stay_in_range_and_rows_behind_the_last_are_left():
    """Bins on the device are not checked: out of range or falling they give other values, never an access out of range; rows of no expert are not written."""
    from megablocks_amd import _lib
    kept, *_ = _weights(3, 16, 128, 128, False, BF16, 5)
    x = torch.randn(9, 128, device='cuda').bfloat16()
    right = gg.gmm_4bit(x, kept, bins=torch.tensor([2, 5, 9], dtype=torch.int32, device='cuda'))
    for bins in ([2, 5, 100], [-3, 5, 9], [9, 2, 9], [0, 0, 0], [2, 5, 7]):
        out = torch.full((9 + 8, 16), 7., device='cuda').bfloat16()
        b = torch.tensor(bins, dtype=torch.int32, device='cuda')
        _lib.check(_lib.lib.mbx_gmm_4bit(x.data_ptr(), 9, None, 1, kept.words.data_ptr(), kept.scales.data_ptr(), None, None, None, None, 0, 128, out.data_ptr(), 0,
                                         b.data_ptr(), 3, 9, 128, 16, -1, _lib.stream()))
        torch.cuda.synchronize()
        assert (out[9:] == 7).all()
        if bins == [2, 5, 7]:
            assert torch.equal(out[:7], right[:7]) and (out[7:] == 7).all()
    indices = torch.tensor([-5, 100, 3], dtype=torch.int32, device='cuda')      # assignments of no token: a token's row instead
    src = gg.GatheredRows(x[:3], indices, indices, torch.tensor([1, 2, 3], dtype=torch.int32, device='cuda'), None, 1, 3)
    assert gg.gmm_4bit(src, kept).isfinite().all()


@pytest.mark.parametrize('rows,experts', [(200, 700), (3000, 100), (20000, 130)])      # a kernel each
def test_falling_bins_of_many_experts(rows, experts):
    """More experts than lanes, every other one with all rows: the tiles there are room for are those of the first that have some, the rest is left out, as is what
    lies behind the rows."""
    from megablocks_amd import _lib
    kept, values, sizes = _weights(experts, 16, 40, 32, False, BF16, 5)
    x = torch.randn(rows, 40, device='cuda').bfloat16()
    bins = torch.tensor([rows, 0], dtype=torch.int32, device='cuda').repeat(experts // 2)
    kept.words[1:], kept.scales[1:] = kept.words[:1], kept.scales[:1]       # all alike: whichever has a row, its product is the same
    out = torch.full((rows + 64, 16), 7., device='cuda').bfloat16()
    _lib.check(_lib.lib.mbx_gmm_4bit(x.data_ptr(), rows, None, 1, kept.words.data_ptr(), kept.scales.data_ptr(), None, None, None, None, 0, 32, out.data_ptr(), 0,
                                     bins.data_ptr(), experts, rows, 40, 16, -1, _lib.stream()))
    torch.cuda.synchronize()
    assert (out[rows:] == 7).all()
    _close(out[:rows], *_products(x.cpu(), [rows], values, sizes), BF16)


def test_more_tiles_of_rows_than_a_grid():
    """65535 tiles of 64 rows are one launch: rows on either side of its end and the last ones, each a product of its own."""
    rows = 65535 * 64 + 70
    kept, values, sizes = _weights(1, 16, 8, 32, False, BF16, 11)
    x = torch.zeros(rows, 8, device='cuda').bfloat16()
    at = torch.cat([torch.arange(3), torch.arange(65535 * 64 - 3, rows)])
    x[at.cuda()] = torch.randn(len(at), 8, generator=torch.Generator().manual_seed(12)).bfloat16().cuda()
    got = gg.gmm_4bit(x, kept, bins=torch.tensor([rows], dtype=torch.int32, device='cuda'))
    want, off = _products(x[at.cuda()].cpu(), [len(at)], values, sizes)
    _close(got[at.cuda()], want, off, BF16)
    assert int((got != 0).any(1).sum()) == len(at)


@pytest.mark.parametrize('rows', [3, 40, 200])      # a kernel each
@pytest.mark.parametrize('dtype', [BF16, F16])
def test_scales_and_rows_at_odd_addresses(rows, dtype):
    kept, values, sizes = _weights(2, 80, 264, 64, True, dtype, 21)
    flat = lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)
    odd = gg.Weights4bit(kept.words, flat(kept.scales), flat(kept.zeros), kept.n, kept.k, kept.group)
    assert odd.scales.data_ptr() % 4 == 2 and odd.zeros.data_ptr() % 2 == 1
    x = torch.randn(2 * rows, 264, device='cuda').to(dtype)
    bins = torch.tensor([rows, 2 * rows], dtype=torch.int32, device='cuda')
    want = gg.gmm_4bit(x, kept, bins=bins)
    assert torch.equal(gg.gmm_4bit(x, odd, bins=bins), want) and torch.equal(gg.gmm_4bit(flat(x), odd, bins=bins), want)
    _close(want, *_products(x.cpu(), [rows, rows], values, sizes), dtype)
    assert torch.equal(odd.dequantize(), kept.dequantize())


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('wide', [False, True])
@pytest.mark.parametrize('zeros', [False, True])
@pytest.mark.parametrize('rows', [3, 40, 200])      # a kernel each
@pytest.mark.parametrize('k,group', [(8, 32), (40, 32), (96, 32), (136, 64), (264, 32), (1032, 32), (129, 64), (130, 128)])
def test_padding_is_never_used(k, group, rows, zeros, wide, dtype):
    """Codes, scales and zeros past n and k may be anything, scales that are no numbers among it: the products are those of padding of zeros."""
    n, experts = 24, 2
    g = torch.Generator().manual_seed(k)
    whole, features = -(-k // 128) * 128, -(-n // 16) * 16
    codes = torch.randint(0, 16, (experts, features, whole), generator=g)
    scales = ((torch.rand(experts, features, whole // group, generator=g) + 0.2) * 0.01).to(F32 if wide else dtype)
    offs = torch.randint(0, 16, scales.shape, generator=g)

    def made(fill_codes, fill_scales):
        c, s, z = codes.clone(), scales.clone(), offs.clone()
        for t, end, fill in ((c, k, fill_codes), (s, -(-k // group), fill_scales), (z, -(-k // group), fill_codes)):
            t[:, :, end:] = fill
            t[:, n:] = fill
        return gg.Weights4bit(oracle.pack(c).cuda(), oracle.kept(s).cuda(), oracle.kept(z).to(torch.uint8).cuda() if zeros else None, n, k, group)

    x = torch.randn(2 * rows, k, generator=g).to(dtype).cuda()
    bins = torch.tensor([rows, 2 * rows], dtype=torch.int32, device='cuda')
    plain = made(0, 0.)
    want, gated = gg.gmm_4bit(x, plain, bins=bins), gg.gmm_4bit_act(x, plain, gg.ACT_SILU, bins=bins, b2=plain)
    assert want.isfinite().all()
    for fill in (float('nan'), float('inf'), -float('inf')):
        other = made(13, fill)
        assert torch.equal(gg.gmm_4bit(x, other, bins=bins), want) and torch.equal(gg.gmm_4bit_act(x, other, gg.ACT_SILU, bins=bins, b2=other), gated)
        assert torch.equal(other.dequantize(), plain.dequantize())
    bad = made(0, 0.)
    bad.scales[0, 0, 0, 3] = float('nan')            # within k it counts
    assert gg.gmm_4bit(x, bad, bins=bins)[:rows, 3].isnan().all()


def test_what_is_refused():
    kept, *_ = _weights(2, 16, 128, 128, False, BF16, 5)
    x, bins, indices = torch.randn(4, 128, device='cuda').bfloat16(), torch.tensor([1, 4], dtype=torch.int32, device='cuda'), torch.arange(4, dtype=torch.int32, device='cuda')
    src = lambda indices, rows=4: gg.GatheredRows(x, indices, indices, bins, None, 1, rows)
    assert torch.equal(gg.gmm_4bit(src(indices), kept), gg.gmm_4bit(x, kept, bins=bins))
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(src(indices.cpu()), kept)               # assignments on the host
    for bad in (src(indices.long()), src(indices[:3]), src(indices, 5)):
        with pytest.raises(ValueError):
            gg.gmm_4bit(bad, kept)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError):
            gg.gmm_4bit(dual, kept, bins=bins)              # no derivative forward either
        assert torch.equal(gg.gmm_4bit(x, kept, bins=bins), gg.gmm_4bit(src(indices), kept))


def test_strides_streams_and_captures():
    kept, *_ = _weights(4, 48, 200, 64, True, F16, 6)
    wide = torch.randn(30, 256, device='cuda').half()
    x, bins = wide[:, 5:205], torch.tensor([3, 3, 20, 30], dtype=torch.int32, device='cuda')
    want = gg.gmm_4bit(x.contiguous(), kept, bins=bins)
    assert torch.equal(gg.gmm_4bit(x, kept, bins=bins), want)
    flat = torch.zeros(30 * 200 + 1, device='cuda').half()
    flat[1:] = x.flatten()
    assert torch.equal(gg.gmm_4bit(flat[1:].view(30, 200), kept, bins=bins), want)       # a base that is no whole piece
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = gg.gmm_4bit(x, kept, bins=bins)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    static = x.contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gg.gmm_4bit(static, kept, bins=bins)
    for scale in (1., 2., 0.5):
        static.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gg.gmm_4bit(x * scale, kept, bins=bins))
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(static.requires_grad_(), kept, bins=bins)
    with torch.no_grad():
        assert torch.equal(gg.gmm_4bit(static, kept, bins=bins), gg.gmm_4bit(static.detach(), kept, bins=bins))
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(x.float(), kept, bins=bins)
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(x.bfloat16(), kept, bins=bins)                                       # scales of another 16-bit type
    with pytest.raises(ValueError):
        gg.gmm_4bit(x, kept, bins=bins[:3])
    with pytest.raises(ValueError):
        gg.gmm_4bit(x, kept, torch.tensor([3, 0, 17, 9]))
    with pytest.raises(ValueError):
        gg.gmm_4bit(x, kept, bins=bins.long())


def test_weights_of_more_than_2_GiB():
    """Offsets past 32 bits: the last expert's weights start beyond 2 GiB of codes."""
    experts, n, k = 38, 8192, 16384
    words = torch.zeros(experts, n // 16, k // 128, 64, 4, dtype=torch.int32, device='cuda')
    scales = torch.zeros(experts, n // 16, k // 128, 16, dtype=BF16, device='cuda')
    g = torch.Generator().manual_seed(9)
    codes = torch.randint(0, 16, (1, 16, k), generator=g)
    words[-1, -1] = oracle.pack(codes)[0, 0].cuda()
    scales[-1, -1] = 0.0078125
    kept = gg.Weights4bit(words, scales, None, n, k, 128)
    x = torch.randn(2, k, generator=g).bfloat16()
    bins = torch.zeros(experts, dtype=torch.int32)
    bins[-1] = 2
    got = gg.gmm_4bit(x.cuda(), kept, bins=bins.cuda())
    values = (codes[0].double() - 8) * 0.0078125
    want, off = _products(x, [2], values[None], torch.full((1, 16, k), 0.0078125).double())
    _close(got[:, -16:], want, off, BF16)
    assert (got[:, :-16] == 0).all()
