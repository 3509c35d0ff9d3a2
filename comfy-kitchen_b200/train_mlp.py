"""A small training run on the layers of ``comfy_kitchen.training``: blocks of ``x + fc2(gelu(fc1(norm(x))))`` learn a fixed random function.

    python comfy-kitchen_b200/train_mlp.py [--tokens 4608] [--features 3072] [--hidden 12288] [--blocks 2] [--steps 20]
        [--dtype bfloat16] [--dense]

Prints the loss, the time of a step and the bytes that the blocks keep for their backward pass; ``--dense`` runs the same blocks
built of torch's layers, from the same weights on the same data.  Needs the GPU.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))


def blocks_of(count: int, features: int, hidden: int, dtype, dense: bool):
    import torch
    from torch import nn

    from comfy_kitchen.training import CheckpointedMLP

    class DenseMLP(nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = nn.LayerNorm(features, device="cuda", dtype=dtype)
            self.fc1, self.fc2 = nn.Linear(features, hidden, device="cuda", dtype=dtype), nn.Linear(hidden, features, device="cuda", dtype=dtype)

        def forward(self, x):
            return x + self.fc2(nn.functional.gelu(self.fc1(self.norm(x)), approximate="tanh"))

    torch.manual_seed(0)
    return nn.Sequential(*[DenseMLP() if dense else CheckpointedMLP(features, hidden, device="cuda", dtype=dtype) for _ in range(count)])


def run(tokens: int, features: int, hidden: int, blocks: int, steps: int, dtype_name: str = "bfloat16", dense: bool = False, report=print) -> dict:
    """Losses, milliseconds of a step and bytes that are kept of the activations."""
    import torch

    dtype = getattr(torch, dtype_name)
    model = blocks_of(blocks, features, hidden, dtype, dense)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, features, generator=gen, device="cuda").to(dtype)
    target = x + torch.tanh(x.roll(1, -1)) * 0.5
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-4, fused=True)

    def step():
        loss = torch.nn.functional.mse_loss(model(x).float(), target.float())
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        return loss.detach()

    params = {p.untyped_storage().data_ptr() for p in model.parameters()}
    kept = {}

    def pack(t):
        storage = t.untyped_storage()
        if storage.data_ptr() not in params:
            kept[storage.data_ptr()] = storage.nbytes()
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = model(x)
    kept_bytes = sum(kept.values())
    del y
    losses = []
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for i in range(steps):
        if i == min(3, steps - 1):
            start.record()
        losses.append(step())
    stop.record()
    torch.cuda.synchronize()
    ms = start.elapsed_time(stop) / (steps - min(3, steps - 1))
    losses = [float(v) for v in losses]
    report(f"{'dense' if dense else 'MXFP8 checkpoints'}: loss {losses[0]:.5f} -> {losses[-1]:.5f}, {ms:.3f} ms a step, "
           f"{kept_bytes / 2**20:.1f} MiB kept for the backward pass of {blocks} blocks on {tokens} tokens")
    return {"losses": losses, "ms_per_step": ms, "kept_bytes": kept_bytes}


def main(argv=None) -> int:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("tokens", 4608), ("features", 3072), ("hidden", 12288), ("blocks", 2), ("steps", 20)):
        parser.add_argument(f"--{name}", type=int, default=default)
    parser.add_argument("--dtype", choices=["bfloat16", "float16", "float32"], default="bfloat16")
    parser.add_argument("--dense", action="store_true", help="torch's layers instead")
    args = parser.parse_args(argv)
    run(args.tokens, args.features, args.hidden, args.blocks, args.steps, args.dtype, args.dense)
    return 0


if __name__ == "__main__":
    sys.exit(main())
