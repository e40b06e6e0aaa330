"""A sparse energy network on the token operators, and its training by distillation.

``ExpertEnergyNet`` is ``LatentEnergyNet`` with the blocks' MLP replaced by a router and experts: each cell goes to its
``experts_per_cell`` best experts, a SwiGLU MLP each. Cells are sorted by expert into fixed-capacity buffers
(``expert_route`` / ``expert_dispatch``), the experts' products are batched library GEMMs, and ``expert_combine`` adds the
results back with the router's weights. Every step is differentiable to second order, as the descent's training needs it
(dE/dz is itself differentiated), and nothing depends on the loads on the host, so microsteps replay as CUDA graphs.

``distill_segment_loss`` trains either network on a teacher's top logits instead of labels: the board is embedded as the
network does it (``scaled_embedding`` here), the segment rolled out as in ``energy.train_segment_loss``, and the decoded
endpoint's loss is ``topk_distill_loss``. ``teacher_entries`` makes such entries from a trained network.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from ebr_b200 import layers as fl
from ebr_b200.energy import AttentionFn, LatentEnergyNet, NetShape, graphed_microstep
from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route, scaled_embedding, topk_distill_loss


@dataclass(frozen=True)
class ExpertShape(NetShape):
    """``NetShape`` and the experts: each has the MLP width of the dense network over ``experts_per_cell`` (so that a cell
    costs the same), rounded up to a multiple of 64. An expert takes ``capacity_factor`` times its even share of a batch's
    slots; later ones are dropped and their cells keep the residual alone."""

    experts: int = 8
    experts_per_cell: int = 2
    capacity_factor: float = 1.5

    @property
    def expert_width(self) -> int:
        width = -(-self.mlp_width // self.experts_per_cell)
        return (width + 63) // 64 * 64

    def capacity(self, cells: int) -> int:
        return max(1, math.ceil(self.capacity_factor * cells * self.experts_per_cell / self.experts))


class _RouterScores(torch.autograd.Function):
    """h W^T in float32, h and W as they are: scores rounded to 16 bits would leave near ties between experts to the
    rounding. The backward is a 16-bit product's, with the scores' gradient rounded as any activation's, and is
    differentiable. It makes both gradients whichever is asked for: 0.04 ms of a microstep of 768 boards, which takes 5.6.
    (Casting h and W to float32 instead took a training step of 768 boards from 24 to 26 ms.)"""

    @staticmethod
    def forward(ctx, h: Tensor, w: Tensor) -> Tensor:
        ctx.save_for_backward(h, w)
        return torch.mm(h, w.t()) if h.dtype == torch.float32 else torch.mm(h, w.t(), out_dtype=torch.float32)

    @staticmethod
    def backward(ctx, g: Tensor):
        h, w = ctx.saved_tensors
        g = g.to(h.dtype)
        return g @ w, g.t() @ h


class ExpertEnergyNet(LatentEnergyNet):
    def __init__(self, shape: ExpertShape, attention: Optional[AttentionFn] = None,
                 generator: Optional[torch.Generator] = None) -> None:  # fmt: skip
        super().__init__(shape, attention, generator)
        c, w, e = shape.hidden, shape.expert_width, shape.experts
        for blk in self.blocks:
            del blk.w_gate_up, blk.w_down
            blk.router = nn.Parameter(torch.randn(e, c, generator=generator) * c**-0.5)
            blk.expert_gate_up = nn.Parameter(torch.randn(e, 2 * w, c, generator=generator) * c**-0.5)
            blk.expert_down = nn.Parameter(torch.randn(e, c, w, generator=generator) * w**-0.5)

    def _name_map(self) -> dict[str, str]:
        raise NotImplementedError("the reference has no network with experts: its state does not translate")

    def embed(self, tokens: Tensor) -> Tensor:
        """x = sqrt(hidden) * embedding[tokens] from the float32 table with one rounding; a token outside the vocabulary
        (a cell off the board) embeds to zero."""
        return scaled_embedding(tokens, self.embedding, math.sqrt(self.shape.hidden), self.shape.dtype)

    def _experts(self, blk: nn.Module, h: Tensor) -> Tensor:
        s, dt, c = self.shape, h.dtype, h.shape[-1]
        scores = _RouterScores.apply(h.reshape(-1, c), blk.router.to(dt)).view(*h.shape[:-1], s.experts)
        best, ids = scores.topk(s.experts_per_cell, dim=-1)
        route = expert_route(ids, s.experts, s.capacity(h.numel() // c))
        rows = expert_dispatch(h, route).view(s.experts, -1, c)
        act = fl.swiglu_act(torch.bmm(rows, blk.expert_gate_up.to(dt).transpose(1, 2)))
        rows = torch.bmm(act, blk.expert_down.to(dt).transpose(1, 2))
        return expert_combine(rows.reshape(-1, c), route, best.softmax(dim=-1))

    def _block(self, blk: nn.Module, h: Tensor, graded: bool) -> Tensor:
        s, dt = self.shape, h.dtype
        folded = None if graded else blk.log_temp.detach().exp().to(dt)
        q, k, v = fl.qkv_rope_split(h, blk.w_qkv.to(dt), self.rope_cos, self.rope_sin, s.heads, folded)
        if graded:
            q = q * blk.log_temp.exp().to(dt).view(1, -1, 1, 1)
        h = fl.add_rms_norm(h, fl.o_proj(self._attend(q, k, v), blk.w_out.to(dt)), s.eps)
        return fl.add_rms_norm(h, self._experts(blk, h), s.eps)

    def _dz_fusable(self, v: Tensor) -> bool:
        return False  # the explicit backward is the dense block's


@torch.no_grad()
def teacher_entries(logits: Tensor, k: int) -> tuple[Tensor, Tensor]:
    """A teacher's ``k`` largest logits per row, as they would be stored: (ids int32, logits in the logits' type)."""
    top, ids = logits.topk(min(k, logits.shape[-1]), dim=-1)
    return ids.to(torch.int32), top


def distill_segment_loss(net: LatentEnergyNet, z: Tensor, tokens: Tensor, teacher_ids: Tensor, teacher_logits: Tensor,
                         prefix: int, graded: int, *, temperature: float = 1.0,
                         cell_weight: Optional[Tensor] = None) -> Tensor:  # fmt: skip
    """A training segment against a teacher's top logits ``[B, L, K]`` per cell: ``prefix`` microsteps without a graph,
    ``graded`` with one, and the mean distillation loss of the decoded endpoint. ``cell_weight`` [B, L]: weights of the
    cells' losses (0 leaves a given cell out). Gradients reach the embedding through every graded microstep."""
    sigma = net.shape.noise_scale
    x = net.embed(tokens)  # as in use: the dense network rounds its table before the product, the sparse one after
    with torch.no_grad():
        for _ in range(prefix):
            noise = torch.randn_like(z) * sigma if sigma else torch.zeros_like(z)
            z = graphed_microstep(net, z, x.detach(), noise)
        z = z.clone()
    for _ in range(graded):
        z, _ = net.microstep(z, x, graded=True)
    return topk_distill_loss(net.decode(z), teacher_ids, teacher_logits, temperature, row_weight=cell_weight)


__all__ = ["ExpertEnergyNet", "ExpertShape", "distill_segment_loss", "teacher_entries"]
