"""Experts with 4-bit weights, for serving.  The reference has none: the layer around them is megablocks/layers/dmoe.py:239-280."""
import torch

from megablocks_amd import grouped_gemm_util as gg
from megablocks_amd.weights_4bit import Weights4bit, quantize_4bit


class Grouped4bitExperts(torch.nn.Module):
    """The experts of a GroupedMLP or GroupedGLU with their weights in 4 bits (`quantize_4bit`), w1 and v1 in groups along the hidden size, w2 along the ffn size:
    buffers w1_words, w1_scales, w1_zeros (None without zero points) and so on, which a state_dict keeps.  Without gradients."""

    def __init__(self, experts, group_size: int = 128, zero_points: bool = False):
        from megablocks_amd.layers import glu, mlp
        super().__init__()
        self.args = experts.args
        if type(experts) is mlp.GroupedMLP:
            names = ('w1', 'w2')
        elif type(experts) is glu.GroupedGLU:
            names = ('w1', 'v1', 'w2')
        else:
            raise ValueError(f'experts with 4-bit weights are made of grouped MLP or GLU experts, not of {type(experts).__name__}')
        self.act = glu._activation_code(self.args.activation_fn)
        if self.act is None:
            raise ValueError('experts with 4-bit weights have tanh-GELU or SiLU as activation')
        self._names, self._sizes = names, {}
        weights = dict(zip(names, experts._expert_views(*(getattr(experts, name) for name in names))))
        for name, w in weights.items():
            made = quantize_4bit(w, group_size, trans_b=name != 'w2', zero_points=zero_points)
            self._sizes[name] = made.n, made.k, made.group, made.trans_b
            for part in ('words', 'scales', 'zeros'):
                self.register_buffer(f'{name}_{part}', getattr(made, part))
        self._wrap()

    def _of_buffers(self, name):
        return Weights4bit(*(getattr(self, f'{name}_{part}') for part in ('words', 'scales', 'zeros')), *self._sizes[name])

    def _wrap(self):
        self._weights = {name: self._of_buffers(name) for name in self._names}

    def _kept(self, name):
        """The weights that the buffers are now: made once (5 us) while nobody puts others in their place, as an assignment and torch.func.functional_call do."""
        kept, buffers = self._weights[name], self._buffers
        if buffers.get(f'{name}_words') is kept.words and buffers.get(f'{name}_scales') is kept.scales and buffers.get(f'{name}_zeros', self) is kept.zeros:
            return kept
        return self._of_buffers(name)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        self._wrap()
        return self

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._wrap()       # load_state_dict(assign=True) replaces the buffers

    @property
    def w1(self):
        return self._kept('w1')

    @property
    def v1(self):
        return self._kept('v1') if 'v1' in self._weights else None

    @property
    def w2(self):
        return self._kept('w2')

    def forward(self, x, tokens_per_expert):
        x, = gg.autocast_operands(x)
        return gg.gmm_4bit(gg.gmm_4bit_act(x, self.w1, self.act, tokens_per_expert, b2=self.v1), self.w2, tokens_per_expert)

    def forward_tokens(self, src, tokens_per_expert):
        """forward on the rows of the tokens that `src` (a `gg.GatheredRows`) describes."""
        return gg.gmm_4bit(gg.gmm_4bit_act(src, self.w1, self.act, b2=self.v1), self.w2, bins=src.bins if src.padded_bins is None else src.padded_bins)
