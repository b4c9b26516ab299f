"""The operator surface of megablocks.ops (megablocks/ops/__init__.py:4-35), MI355X-native."""
from megablocks_amd.ops.choose import balance_bias, choose_experts
from megablocks_amd.ops.embed import embedding
from megablocks_amd.ops.few_tokens import moe_layer
from megablocks_amd.ops.norm import clip_by_global_norm_, clip_grad_norm_, global_norm
from megablocks_amd.ops.permute import (binned_gather, binned_scatter, gather, padded_gather, padded_scatter,
                                        scatter)
from megablocks_amd.ops.routing import (exclusive_cumsum, histogram, inclusive_cumsum, repeat, replicate, round_up,
                                        sort, sum, topology)

__all__ = [
    'balance_bias', 'binned_gather', 'binned_scatter', 'choose_experts', 'clip_by_global_norm_', 'clip_grad_norm_',
    'embedding', 'exclusive_cumsum', 'inclusive_cumsum', 'gather', 'global_norm', 'histogram', 'moe_layer',
    'padded_gather', 'padded_scatter', 'repeat', 'replicate', 'round_up', 'scatter', 'sort', 'sum', 'topology',
]
