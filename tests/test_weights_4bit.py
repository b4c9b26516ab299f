"""4-bit weights without a GPU: where a code is kept, what the restatement does, and the calls that are refused."""
import pytest
import torch

from megablocks_amd import _lib
from megablocks_amd import grouped_gemm_util as gg
from oracle import weights_4bit as oracle


def test_where_a_code_is_kept():
    """Lane 16 g + f, word j: feature f, columns 32 j + 8 g + (0, 2, 4, 6, 1, 3, 5, 7) from the lowest bits."""
    assert oracle.place(0, 0) == (0, 0, 0, 0, 0) and oracle.place(0, 1) == (0, 0, 0, 0, 16) and oracle.place(0, 2) == (0, 0, 0, 0, 4)
    assert oracle.place(17, 128 + 32 + 8 + 7) == (1, 1, 17, 1, 28) and oracle.place(15, 127) == (0, 0, 63, 3, 28)
    codes = torch.randint(0, 16, (2, 19, 150), generator=torch.Generator().manual_seed(1))
    words = oracle.pack(codes)
    assert words.shape == (2, 2, 2, 64, 4) and words.dtype == torch.int32
    assert torch.equal(oracle.unpack(words, 19, 150), codes)


def test_the_restatement_quantizes():
    w = torch.tensor([[[7., -3.5, 2.5, 0.], [15., 0., 7.4, 7.5]]])
    codes, scales, zeros = oracle.quantize(w, 32, False)
    assert scales.flatten().tolist() == pytest.approx([1., 15 / 7]) and codes[0, 0].tolist() == [15, 4, 10, 8] and (zeros == 8).all()     # halves to even
    codes, scales, zeros = oracle.quantize(w, 32, True)
    assert codes[0, 1].tolist() == [15, 0, 7, 8] and zeros[0, 1].tolist() == [0] and float(scales[0, 0]) == pytest.approx(0.7) and int(zeros[0, 0]) == 5


def weights(experts=2, n=20, k=40, group=32, zeros=False, scale_dtype=torch.bfloat16):
    shape = (experts, -(-n // 16), -(-k // 128) * 128 // group, 16)
    return gg.Weights4bit(torch.zeros(experts, -(-n // 16), -(-k // 128), 64, 4, dtype=torch.int32), torch.ones(shape, dtype=scale_dtype),
                          torch.zeros(shape, dtype=torch.uint8) if zeros else None, n, k, group)


def test_weights_that_do_not_fit_are_refused():
    good = weights()
    for group in (16, 256, 0):
        with pytest.raises(ValueError):
            gg.Weights4bit(good.words, good.scales, None, 20, 40, group)
    for n, k in ((40, 40), (20, 400), (0, 40), (20, 0)):
        with pytest.raises(ValueError):
            gg.Weights4bit(good.words, good.scales, None, n, k, 32)
    with pytest.raises(ValueError):
        gg.Weights4bit(good.words, good.scales[:, :, :1], None, 20, 40, 32)
    with pytest.raises(ValueError):
        gg.Weights4bit(good.words, good.scales, good.scales[:1].byte(), 20, 40, 32)
    for words, scales, zeros in ((good.words.long(), good.scales, None), (good.words, good.scales.double(), None), (good.words, good.scales, good.scales),
                                 (good.words, good.scales.transpose(2, 3).contiguous().transpose(2, 3), None)):
        with pytest.raises(RuntimeError):
            gg.Weights4bit(words, scales, zeros, 20, 40, 32)
    assert good.group_scales().shape == (2, 20, 2) and good.experts == 2
    with pytest.raises(RuntimeError):
        good.dequantize()                # on the CPU


@pytest.mark.parametrize('w,group,error', [
    (torch.zeros(4, 4), 32, ValueError), (torch.zeros(1, 4, 4), 48, ValueError), (torch.zeros(1, 0, 4), 32, ValueError), (torch.zeros(1, 4, 0), 32, ValueError),
    (torch.zeros(1, 4, 4), 32, RuntimeError)])
def test_quantizing_is_refused(w, group, error):
    with pytest.raises(error):
        gg.quantize_4bit(w, group)


def test_products_are_refused():
    w, sizes = weights(), torch.tensor([3, 2])
    x = torch.zeros(5, 40, dtype=torch.bfloat16)
    for call in (lambda: gg.gmm_4bit(x[:, :39], w, sizes), lambda: gg.gmm_4bit(x.view(-1), w, sizes), lambda: gg.gmm_4bit(x, w),
                 lambda: gg.gmm_4bit(x, w, sizes, bins=torch.tensor([3, 5], dtype=torch.int32)), lambda: gg.gmm_4bit_act(x, w, 2, sizes),
                 lambda: gg.gmm_4bit_act(x, w, gg.ACT_SILU, sizes, b2=weights(n=21)), lambda: gg.gmm_4bit_act(x, w, gg.ACT_SILU, sizes, b2=weights(zeros=True)),
                 lambda: gg.gmm_4bit_act(x, w, gg.ACT_SILU, sizes, b2=weights(group=64))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(x, w, sizes)         # on the CPU


def test_entry_points_refuse_without_touching_the_gpu():
    lib = _lib.lib

    def gmm(dtype=0, scale_dtype=0, group=32, groups=2, rows=5, k=40, n=20, act=-1, indices=None, top_k=1, a_rows=5, a=None, words2=None, words=None):
        return lib.mbx_gmm_4bit(a, a_rows, indices, top_k, words, None, None, words2, None, None, scale_dtype, group, None, dtype, None, groups, rows, k, n, act, None)
    for bad in (dict(dtype=4), dict(scale_dtype=3), dict(group=48), dict(groups=-1), dict(rows=-1), dict(k=-1), dict(n=-1), dict(act=2), dict(act=-2),
                dict(indices=16, top_k=0), dict(words2=16), {}):
        assert gmm(**bad) == _lib.EINVAL, bad
    for unsupported in (dict(dtype=2), dict(scale_dtype=1), dict(k=0)):
        assert gmm(**unsupported) == _lib.EUNSUPPORTED
    assert gmm(rows=0) == gmm(n=0) == gmm(groups=0) == 0 and gmm(rows=1 << 31) == _lib.ERANGE
    assert gmm(rows=(1 << 31) - 64) == gmm(n=(1 << 26) + 1) == _lib.ERANGE
    assert lib.mbx_quantize_4bit(None, 0, 1, 4, 4, _lib.TN, 32, None, None, None, None) == _lib.EINVAL
    assert lib.mbx_quantize_4bit(None, 0, 1, 4, 4, _lib.NT, 31, None, None, None, None) == _lib.EINVAL
    assert lib.mbx_quantize_4bit(None, 0, 1, 4, 4, _lib.NT, 32, None, None, None, None) == _lib.EINVAL
    assert lib.mbx_quantize_4bit(None, 0, 0, 4, 4, _lib.NT, 32, None, None, None, None) == 0
    assert lib.mbx_dequantize_4bit(None, None, None, 0, 1, 4, 4, _lib.NT, 32, None, 5, None) == _lib.EINVAL
    assert lib.mbx_dequantize_4bit(None, None, None, 0, 1, 0, 4, _lib.NT, 32, None, 0, None) == 0


def test_gathered_rows_bring_their_bins():
    """Sizes or bins next to gathered rows are refused, not passed over."""
    w, bins = weights(), torch.tensor([3, 5], dtype=torch.int32)
    indices = torch.arange(5, dtype=torch.int32)
    src = gg.GatheredRows(torch.zeros(5, 40, dtype=torch.bfloat16), indices, indices, bins, None, 1, 5)
    for given in (dict(bins=bins), dict(batch_sizes=torch.tensor([3, 2])), dict(bins=bins, batch_sizes=torch.tensor([3, 2]))):
        with pytest.raises(ValueError):
            gg.gmm_4bit(src, w, **given)
        with pytest.raises(ValueError):
            gg.gmm_4bit_act(src, w, gg.ACT_SILU, **given)
    with pytest.raises(RuntimeError):
        gg.gmm_4bit(src, w)              # on the CPU
