"""B200 (sm_100a) Mixture-of-Experts layer behind the reference's MoELayer interface, and what stands beside it in a training step."""
from .moe_layer import MoELayer, MoeError, launch_count  # noqa: F401
from .routing import route, route_backward  # noqa: F401
from .training import AdamW, Kept8, check_status, head_loss, head_loss_backward, keep8, residual_norm, residual_norm_backward, restore8  # noqa: F401
