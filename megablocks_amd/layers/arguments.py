"""Layer configuration: the field names and defaults of megablocks/layers/arguments.py:22-73."""
import dataclasses
from functools import partial
from typing import Any, Callable, Optional, Union

import torch
import torch.nn.functional as F

InitFn = Union[Callable[[torch.Tensor], None], partial]

DEFAULT_ACTIVATION_FN = partial(F.gelu, approximate='tanh')


def _current_device():
    return torch.cuda.current_device()


@dataclasses.dataclass
class Arguments:
    # Model.
    hidden_size: int = 1024
    ffn_hidden_size: int = 4096
    num_layers: int = 1
    bias: bool = True
    return_bias: bool = True
    activation_fn: Optional[Callable] = DEFAULT_ACTIVATION_FN

    # MoE.
    moe_num_experts: int = 1
    moe_top_k: int = 1
    moe_capacity_factor: int = 1
    moe_normalize_expert_weights: Optional[Union[int, float]] = None
    moe_loss_weight: float = 0.1
    moe_jitter_eps: Optional[float] = None
    moe_lbl_in_fp32: bool = False

    # Parallelism.  This build runs one GPU holding all experts; the fields exist so that
    # configurations written for the reference still construct.
    moe_expert_model_parallelism: bool = False
    expert_parallel_group: Optional[Any] = None
    pipeline_model_parallel_size: int = 1
    num_layers_per_virtual_pipeline_stage: Optional[int] = None

    # Compute.
    memory_optimized_mlp: bool = False
    mlp_type: str = 'mlp'
    mlp_impl: str = 'grouped'

    # Initialisation.
    fp16: bool = True
    bf16: bool = False
    device: Union[int, torch.device] = dataclasses.field(default_factory=_current_device)
    init_method: InitFn = partial(torch.nn.init.normal_, mean=0.0, std=0.02)
    output_layer_init_method: InitFn = init_method

    # Benchmarking.
    uniform_expert_assignment: bool = False

    # Shared expert (not part of the dropless path; accepted and ignored unless enabled).
    shared_expert: bool = False
    fc_cls: Any = torch.nn.Linear
    fc_kwargs: dict = dataclasses.field(default_factory=dict)
    remat_act_fn: bool = True
    shared_expert_hidden_size: Optional[int] = None
    shared_expert_weighted_sum: bool = False

    # Router z-loss.
    moe_zloss_weight: float = 0
    moe_zloss_in_fp32: bool = False

    # Choice of experts (ops.choose_experts); the defaults are the reference's router.  Scores 'softmax' or 'sigmoid'; a bias for the choice alone, which
    # layers.moe.update_balance_biases moves by moe_router_bias_rate towards equally many tokens an expert; experts in groups of which the best
    # moe_router_top_groups are open, a group going by its moe_router_group_best best experts; the weights times moe_router_scale.
    moe_router_score: str = 'softmax'
    moe_router_bias: bool = False
    moe_router_bias_rate: float = 0.001
    moe_router_groups: int = 1
    moe_router_top_groups: int = 1
    moe_router_group_best: int = 2
    moe_router_scale: float = 1.0

    # Decoding: a dropless layer in evaluation and without gradients runs up to this many tokens (64 at most; 0: none) as one operator (ops.moe_layer),
    # whose results are rounded in fewer places than the separate ones'.
    moe_fused_tokens: int = 0

    def __post_init__(self):
        if self.moe_expert_model_parallelism:
            raise NotImplementedError('expert model parallelism is not part of this single-GPU build')
        if self.shared_expert:
            raise NotImplementedError('the shared expert is not part of the dropless-MoE hot path')
        if not 0 <= self.moe_fused_tokens <= 64:
            raise ValueError(f'moe_fused_tokens must be from 0 to 64, not {self.moe_fused_tokens}')
        if self.shared_expert_hidden_size is None:
            self.shared_expert_hidden_size = self.ffn_hidden_size


def from_megatron(megatron_args: Any):
    """megablocks/layers/arguments.py:95-100."""
    args = Arguments()
    for field in dataclasses.fields(args):
        if hasattr(megatron_args, field.name):
            setattr(args, field.name, getattr(megatron_args, field.name))
    return args
