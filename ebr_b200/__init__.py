"""ebr_b200: the B200 (sm_100a) rebuild of the second-order attention hot path of wwillchen/ebr.

``ebr_b200.fused_attn`` is the drop-in for the reference's ``models.fused_attn``; ``ebr_b200.energy`` is the energy
network and latent-descent caller that drives it; ``ebr_b200.runtime`` holds the data-parallel plumbing.
``ebr_b200.token_ops`` has the operators driven by integer ids (scaled embedding, expert routing, distillation from a
teacher's top logits) and ``ebr_b200.expert_net`` the network and training segment that use them.
"""

from ebr_b200.fused_attn import fused_attention, implementation

__all__ = ["fused_attention", "implementation"]
