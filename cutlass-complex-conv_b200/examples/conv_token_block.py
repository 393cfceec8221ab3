"""A complex convolution followed by a token-wise block, trained for a few
steps on synthetic data.

    python cutlass-complex-conv_b200/examples/conv_token_block.py [--steps 20]

``ComplexConv2d.forward_planar`` hands out the real and imaginary planes as
NHWC float32 tensors; side by side they are one row of 2 K features per pixel.
On those rows run layer norm (float32 in, bfloat16 out), the gated
feed-forward block (bfloat16) and counter-based dropout, which adds the
float32 residual in the same pass:

    t = cat(conv(x).real, conv(x).imag);   out = t + dropout(ffn(norm(t)))
"""

import argparse
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(HERE))

import torch  # noqa: E402
from torch import nn  # noqa: E402

from complex_conv2d import ComplexConv2d, Dropout, GatedFeedForward, LayerNorm  # noqa: E402


class ConvTokenBlock(nn.Module):
    """Planes ``[N, H, W, C]`` in, rows ``[N, P, Q, 2 K]`` out."""

    def __init__(self, in_channels, out_channels, hidden, kernel_size=3, p=0.1, activation="gelu",
                 device="cuda"):
        super().__init__()
        self.conv = ComplexConv2d(in_channels, out_channels, kernel_size,
                                  padding=kernel_size // 2, device=device)
        self.conv.weight_real.requires_grad_(True)
        self.conv.weight_imag.requires_grad_(True)
        self.norm = LayerNorm(2 * out_channels, out_dtype=torch.bfloat16, device=device)
        self.ffn = GatedFeedForward(2 * out_channels, hidden, activation, device=device)
        self.dropout = Dropout(p, seed=1)

    def forward(self, x_real, x_imag):
        t = torch.cat(self.conv.forward_planar(x_real, x_imag), dim=-1)
        return self.dropout(self.ffn(self.norm(t)), residual=t)


def train(steps=20, batch=8, channels=64, size=28, hidden=512, lr=0.01, device="cuda"):
    """Fits the block's first half of the features to smoothed input planes;
    returns the losses."""
    gen = torch.Generator(device=device).manual_seed(0)
    torch.manual_seed(0)
    x_real, x_imag = (torch.randn(batch, size, size, channels, generator=gen, device=device)
                      for _ in range(2))
    target = torch.tanh(torch.cat((x_real, x_imag), dim=-1))
    block = ConvTokenBlock(channels, channels, hidden, device=device)
    optimizer = torch.optim.Adam(block.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        optimizer.zero_grad(set_to_none=True)
        loss = (block(x_real, x_imag) - target).square().mean()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return [v.item() for v in losses]


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=20)
    args = ap.parse_args()
    for i, loss in enumerate(train(args.steps)):
        print(f"step {i}: loss {loss:.4f}")


if __name__ == "__main__":
    main()
