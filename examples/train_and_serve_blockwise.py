"""Trains a small stack of pre-norm blocks on block-scaled float8 linears and serves it from block-scaled weights.

    python examples/train_and_serve_blockwise.py [--steps 60] [--dim 512] [--hidden 1408] [--tokens 1000] [--dtype bf16]

A training step is: layer norm and blockwise linears forward and backward, gradients clipped to a global norm, an update.  With bfloat16
parameters the optimizer keeps fp32 ones and takes the clipped gradients in fp32 straight from ``clip_grads``; with fp32 parameters
``clip_grad_norm_`` clips in place.  Then the weights are cast once and the model answers for one token and for many.
"""
import argparse
import copy
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import float8_experimental_amd as f8
from float8_experimental_amd.inference import ActivationCasting, QuantConfig, quantize_to_float8

BLOCKWISE = f8.CastConfig(scaling_type=f8.ScalingType.BLOCKWISE)
CONFIG = f8.Float8LinearConfig(cast_config_input=BLOCKWISE, cast_config_weight=BLOCKWISE, cast_config_grad_output=BLOCKWISE)


class Block(nn.Module):
    def __init__(self, dim, hidden):
        super().__init__()
        self.norm, self.up, self.down = nn.LayerNorm(dim), nn.Linear(dim, hidden, bias=False), nn.Linear(hidden, dim)

    def forward(self, x):
        return x + self.down(nn.functional.silu(self.up(self.norm(x))))


def make_model(dim, hidden, layers, dtype, device="cuda"):
    model = nn.Sequential(*[Block(dim, hidden) for _ in range(layers)], nn.LayerNorm(dim)).to(device, dtype)
    return f8.convert_layer_norms(f8.convert_to_float8_training(model, config=CONFIG))


def train_step(model, optimizer, masters, x, target, max_norm):
    """One step; returns (loss, norm of the gradients before clipping) as tensors on the GPU."""
    params = list(model.parameters())
    loss = nn.functional.mse_loss(model(x).float(), target.float())
    loss.backward()
    if masters is None:
        norm = f8.clip_grad_norm_(params, max_norm)
        optimizer.step()
    else:
        norm, grads = f8.clip_grads([p.grad for p in params], max_norm, out_dtype=torch.float32)
        for master, grad in zip(masters, grads):
            master.grad = grad
        optimizer.step()
        with torch.no_grad():
            torch._foreach_copy_(params, masters)
    model.zero_grad()
    return loss.detach(), norm


def serving_copy(model):
    """The model with its linears' weights cast once to block-scaled e4m3, for torch.no_grad()."""
    return quantize_to_float8(copy.deepcopy(model), QuantConfig(ActivationCasting.BLOCKWISE)).eval()


def run(steps=60, dim=512, hidden=1408, layers=2, tokens=1000, dtype=torch.bfloat16, max_norm=0.05, seed=0):
    """Returns the losses, the gradients' norms, the trained model and its serving copy."""
    torch.manual_seed(seed)
    model = make_model(dim, hidden, layers, dtype)
    masters = None if dtype == torch.float32 else [p.detach().float().requires_grad_() for p in model.parameters()]
    optimizer = torch.optim.AdamW(masters or model.parameters(), lr=2e-3)
    mix = torch.randn(dim, dim, device="cuda") / dim ** 0.5
    losses, norms = [], []
    for _ in range(steps):
        x = torch.randn(tokens, dim, device="cuda", dtype=dtype)
        target = torch.tanh(x.float() @ mix)
        loss, norm = train_step(model, optimizer, masters, x, target, max_norm)
        losses.append(loss)
        norms.append(norm)
    return torch.stack(losses), torch.stack(norms), model, serving_copy(model)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("steps", 60), ("dim", 512), ("hidden", 1408), ("layers", 2), ("tokens", 1000)):
        parser.add_argument(f"--{name}", type=int, default=default)
    parser.add_argument("--dtype", choices=("bf16", "fp16", "fp32"), default="bf16")
    args = vars(parser.parse_args())
    args["dtype"] = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[args["dtype"]]
    losses, norms, model, served = run(**args)
    print(f"loss {losses[0].item():.4f} -> {losses[-1].item():.4f}, norm of the gradients {norms[0].item():.4f} -> {norms[-1].item():.4f}")
    with torch.no_grad():
        for rows in (1, 300):
            x = torch.randn(rows, args["dim"], device="cuda", dtype=args["dtype"])
            y, served_y = model(x).float(), served(x).float()
            print(f"{rows} token(s): served against trained model, largest difference {(y - served_y).abs().max().item():.4g} of {y.abs().max().item():.4g}")


if __name__ == "__main__":
    main()
