"""MI355X-native attention hot path (joint-attention forward + ring LSE merge) behind
xDiT's attention call surfaces, and the operators around that call in a DiT block (modulated norms with gate and residual,
rotation by positions on several axes, block-scaled fp8 projections)."""
from .block_ops import (axes_rope, axes_rope_backward, fp8_block_matmul, fp8_block_quant, gated_norm, gated_norm_backward,  # noqa: F401
                        rope_frequencies)
from .ops import attn_fwd, attn_fwd_accumulate, fp8_quant, launch_plan, lse_merge  # noqa: F401
