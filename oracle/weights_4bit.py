"""Plain restatement of 4-bit weights with group scales in float64 on the CPU: codes from weights, where each code is kept, and products.  The
reference has none: parity unpinned, held to the formulas."""
import torch


def place(feature, column):
    """(tile, block, lane, word, shift) of a code."""
    within = column % 32
    return feature // 16, column // 128, within // 8 * 16 + feature % 16, column % 128 // 32, 4 * (within % 8 // 2 + 4 * (within % 2))


def pack(codes):
    """Codes [E, n, k] in 0..15 as int32 words [E, T, B, 64, 4]; 0 past the ends."""
    experts, n, k = codes.shape
    words = torch.zeros(experts, -(-n // 16), -(-k // 128), 64, 4, dtype=torch.int64)
    at = torch.tensor([[place(i, c) for c in range(k)] for i in range(n)])
    for bits in range(0, 32, 4):
        i, c = (at[:, :, 4] == bits).nonzero(as_tuple=True)
        tile, block, lane, word, _ = at[i, c].unbind(1)
        words[:, tile, block, lane, word] |= codes[:, i, c].long() << bits
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()


def unpack(words, n, k):
    experts = words.shape[0]
    at = torch.tensor([[place(i, c) for c in range(k)] for i in range(n)]).flatten(0, 1)
    tile, block, lane, word, shift = at.unbind(1)
    return ((words.cpu().long()[:, tile, block, lane, word] >> shift) & 15).view(experts, n, k)


def quantize(w, group, zero_points):
    """(codes, scales, zeros) of w [E, n, k]: int64 codes, scales of w's type and int64 zeros [E, n, groups]."""
    experts, n, k = w.shape
    parts = torch.nn.functional.pad(w.cpu(), (0, -k % group)).view(experts, n, -1, group)
    bad = ~parts.isfinite().all(3)
    x = torch.where(bad[..., None], 0., parts.float())
    low, high = x.amin(3).clamp(max=0), x.amax(3).clamp(min=0)
    one = torch.ones((), dtype=torch.float32)      # by the reciprocal in 32 bits
    scales = ((high - low) * (one / 15) if zero_points else torch.maximum(high, -low) * (one / 7)).to(w.dtype)
    scales = torch.where(scales.float() < 2.0 ** -126, torch.zeros_like(scales), scales)
    step = torch.where(scales == 0, 1., scales.double())[..., None]
    zeros = torch.full(scales.shape, 8.).double()
    if zero_points:
        zeros = (-low.double() / step[..., 0]).round().clamp(0, 15)
    codes = ((x.double() / step).round() + zeros[..., None]).clamp(0, 15)
    if zero_points:
        zeros = torch.where((scales == 0) | bad, 0., zeros)
    codes = torch.where(((scales == 0) | bad)[..., None], zeros[..., None], codes)
    return codes.view(experts, n, -1)[:, :, :k].long(), torch.where(bad, float('nan'), scales.float()).to(w.dtype), zeros.long()


def values(codes, scales, zeros, group):
    """[E, n, k] in float64; zeros None: 8."""
    k = codes.shape[2]
    each = lambda t: t.cpu().double().repeat_interleave(group, 2)[:, :, :k]
    return (codes.double() - (8 if zeros is None else each(zeros))) * each(scales)


def kept(t):
    """Scales or zeros [E, n, groups] as they are kept, [E, T, groups of whole blocks, 16] given a number of groups that is one."""
    experts, n, groups = t.shape
    return torch.nn.functional.pad(t, (0, 0, 0, -n % 16)).view(experts, -1, 16, groups).transpose(2, 3).contiguous()
