"""Distil a dense energy network into one with experts, on synthetic 9 x 9 boards.

    python examples/distill_experts.py [--steps 20] [--boards 64] [--experts 8] [--entries 4]

A dense ``LatentEnergyNet`` (random weights: there is nothing to download here) descends on each batch of boards and keeps
its best logits per cell; the ``ExpertEnergyNet`` student is trained on those entries alone. Prints the loss per step.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from ebr_b200.energy import LatentEnergyNet, NetShape, descend  # noqa: E402
from ebr_b200.expert_net import ExpertEnergyNet, ExpertShape, distill_segment_loss, teacher_entries  # noqa: E402


def boards(n: int, generator: torch.Generator, device: str) -> torch.Tensor:
    """Cells that are blank (0) with probability 0.7 and 1 to 9 otherwise."""
    digits = torch.randint(1, 10, (n, 81), generator=generator, device=device)
    return torch.where(torch.rand(n, 81, generator=generator, device=device) < 0.7, torch.zeros_like(digits), digits)


def run(steps: int, n: int, experts: int, entries: int, layers: int = 2, device: str = "cuda") -> list[float]:
    gen = torch.Generator(device=device).manual_seed(0)
    weights = torch.Generator().manual_seed(1)
    teacher = LatentEnergyNet(NetShape(layers=layers), generator=weights).to(device)
    student = ExpertEnergyNet(ExpertShape(layers=layers, experts=experts), generator=weights).to(device)
    optimizer = torch.optim.AdamW(student.parameters(), lr=1e-3)
    losses = []
    for _ in range(steps):
        tokens = boards(n, gen, device)
        z = teacher.fresh_states(n, gen)
        with torch.no_grad():
            end, _ = descend(teacher, z, teacher.embed(tokens), 4)
            ids, top = teacher_entries(teacher.decode(end), entries)
        loss = distill_segment_loss(student, z, tokens, ids, top, prefix=1, graded=1, temperature=2.0)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    return losses


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--boards", type=int, default=64)
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--entries", type=int, default=4)
    a = ap.parse_args()
    for i, loss in enumerate(run(a.steps, a.boards, a.experts, a.entries)):
        print(f"step {i}: distillation loss {loss:.5f}")


if __name__ == "__main__":
    main()
