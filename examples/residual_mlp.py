"""Trains a residual MLP with dropout on synthetic data, then serves single rows.

    python examples/residual_mlp.py --dtype bf16 --steps 200
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ferrograd_b200 import data, kernels  # noqa: E402
from ferrograd_b200.residual import ResidualMlp  # noqa: E402

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", choices=DTYPES, default="f32")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=256)
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--blocks", type=int, default=2)
    ap.add_argument("--p", type=float, default=0.1, help="dropout probability")
    ap.add_argument("--lr", type=float, default=0.005)
    args = ap.parse_args()

    x, t = data.mlp_batch(args.batch, 784, 10, 1, 2)
    x, t = torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()
    model = ResidualMlp(784, args.width, 4 * args.width, 10, args.blocks, p=args.p,
                        dtype=DTYPES[args.dtype])
    for step in range(args.steps):
        loss = model.train_step(x, t, args.lr)
        if step % 20 == 0 or step + 1 == args.steps:
            print(f"step {step:4d}  loss {float(loss):.4f}")
    together = model(x)
    alone = torch.cat([model(x[i:i + 1]) for i in range(8)])
    kernels.check_device_error()
    hits = (together.argmax(1) == t.argmax(1)).float().mean()
    gap = (together[:8].float() - alone.float()).abs().max()
    print(f"training accuracy {float(hits):.3f}; a row served alone differs by {float(gap):.2e}")


if __name__ == "__main__":
    main()
