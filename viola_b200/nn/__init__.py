"""FP8 neural-network modules: Linear, gated MLP and the expert (grouped) linear with the routing around it."""

from .linear import Linear
from .mlp import MLP
from .grouped import GroupedLinear
from .experts import ExpertPlan, Routing, combine_tokens, dispatch_tokens, plan_experts, route_tokens
from .fused import activation_linear, gated_residual, norm_modulate_linear, norm_modulate_mlp
from .norms import rms_norm_modulate, rms_norm_residual

__all__ = ["Linear", "MLP", "GroupedLinear", "ExpertPlan", "Routing", "route_tokens", "plan_experts", "dispatch_tokens",
           "combine_tokens", "gated_residual", "norm_modulate_linear", "norm_modulate_mlp", "activation_linear",
           "rms_norm_modulate", "rms_norm_residual"]
