"""Trains a small network end to end on synthetic positions: the feature
transformer, its epilogue, and routed layer stacks behind it.

    python examples/train_routed_stacks.py [--steps 50] [--batch 4096] [--bf16]

The target is the material balance of each position, squashed to [0, 1].
Prints the loss, the balance loss and how often each stack was chosen.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from stockfish_trainer_b200 import SparseLinearPairFunction, positions  # noqa: E402
from stockfish_trainer_b200.feature_transformer import transform_inputs  # noqa: E402
from stockfish_trainer_b200.layer_stacks import RoutedLayerStacks  # noqa: E402

FEATURES, L1, N_PSQT = "HalfKAv2_hm^", 256, 8
PIECE_VALUES = (1.0, 3.0, 3.2, 5.0, 9.0, 0.0)  # pawn .. king; boards hold type * 2 + colour, 12 = empty


def targets(boards: torch.Tensor) -> torch.Tensor:
    values = torch.tensor([v * s for v in PIECE_VALUES for s in (1.0, -1.0)] + [0.0], device=boards.device)
    return torch.sigmoid(values[boards.long()].sum(1) / 6)


def train(steps: int = 50, batch: int = 4096, dtype: torch.dtype = torch.float32, seed: int = 0,
          report=print) -> list[float]:
    """Runs the steps and returns the value loss of each."""
    dev = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(seed)
    rows = positions.feature_set_info(FEATURES)[1]
    table = torch.nn.Parameter(torch.randn(rows, L1 + N_PSQT, device=dev) * 0.05)
    bias = torch.nn.Parameter(torch.full((L1 + N_PSQT,), 0.3, device=dev))
    net = RoutedLayerStacks(l1=L1, width=64, hidden=128, blocks=2, stacks=8, k=2).to(dev, dtype)
    # a row of the table is met by few positions and has to move fast; the network, at its rate, would swing
    opt = torch.optim.Adam([{"params": [table, bias], "lr": 1e-2}, {"params": net.parameters(), "lr": 1e-3}])
    losses = []
    for step in range(steps):
        board_np, _ = positions.generate_positions(batch, seed=seed + 1 + step)
        boards = torch.from_numpy(board_np).to(dev)
        white, black = positions.encode_device(boards, FEATURES)
        out_w, out_b = SparseLinearPairFunction.apply(white, black, table, bias)
        us = torch.ones(batch, 1, device=dev)  # white to move everywhere
        pieces = (boards != 12).sum(1)
        l0, psqt = transform_inputs(out_w, out_b, us, ((pieces - 1) // 4).clamp(0, N_PSQT - 1), L1)
        value, routing = net(l0.to(dtype))
        loss = (torch.sigmoid(value + psqt[:, 0]) - targets(boards)).square().mean()
        opt.zero_grad(set_to_none=True)
        (loss + 1e-2 * routing.balance_loss).backward()
        opt.step()
        losses.append(float(loss.detach()))
        if report and (step % 10 == 0 or step == steps - 1):
            report(f"step {step:4d}  loss {losses[-1]:.5f}  balance {float(routing.balance_loss.detach()):.3f}  "
                   f"counts {routing.counts.tolist()}")
    return losses


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=50)
    parser.add_argument("--batch", type=int, default=4096)
    parser.add_argument("--bf16", action="store_true")
    args = parser.parse_args()
    train(args.steps, args.batch, torch.bfloat16 if args.bf16 else torch.float32)
