"""A residual block trained for a few steps: a convolution layer, group norm with SiLU, a 1 x 1 projection with GELU
and dropout, added to its own input.

    conv     c = conv_fprop(x, filters)                  planes, as the layer leaves them
    norm     h = silu(group_norm(c))                      written channels last
    linear   l = gelu(rows of h times weight^T + bias)    a row is a pixel
    dropout  y = dropout(l) + h

The loss is the mean squared distance to a target; every gradient comes from the library, and plain torch
operations only move the parameters.

    python examples/residual_block.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fbcuda_amd as F  # noqa: E402


def ok(code):
    if code != F.Success:
        raise RuntimeError(F.error_string(code))


class ResidualBlock:
    """Shapes, parameters, buffers and workspaces of one block, allocated once."""

    def __init__(self, batch=8, cin=16, channels=32, size=27, kernel=5, groups=4, p=0.1, seed=1, device="cuda"):
        self.groups, self.p, self.seed = groups, p, seed
        gen = torch.Generator().manual_seed(seed)
        randn = lambda *shape: torch.randn(*shape, generator=gen).to(device)  # noqa: E731
        out = size - kernel + 1
        self.params = {
            "filters": randn(channels, cin, kernel, kernel) * (cin * kernel * kernel) ** -0.5,
            "gamma": torch.ones(channels, device=device), "beta": torch.zeros(channels, device=device),
            "weight": randn(channels, channels) * channels ** -0.5, "bias": torch.zeros(channels, device=device)}
        self.grads = {k: torch.empty_like(v) for k, v in self.params.items()}
        planes = lambda: torch.empty((batch, channels, out, out), device=device)  # noqa: E731
        rows = lambda: torch.empty((batch * out * out, channels), device=device)  # noqa: E731
        self.image = lambda r: r.view(batch, out, out, channels).permute(0, 3, 1, 2)  # noqa: E731
        self.c, self.dc = planes(), planes()
        self.h, self.l, self.z, self.y, self.dl, self.dh = (rows() for _ in range(6))
        self.mean, self.rstd = (torch.empty((batch, groups), device=device) for _ in range(2))
        space = lambda size: torch.empty(size, dtype=torch.uint8, device=device)  # noqa: E731
        self.conv_space = [space(F.conv_workspace_image(q, batch, cin, channels, size, size, kernel, kernel, 0)) for q in (0, 2)]
        self.norm_space = [space(F.group_norm_workspace(q, self.c, groups)) for q in (0, 1)]
        self.linear_space = [space(F.linear_workspace(q, self.h.shape[0], channels, channels, torch.float32)) for q in (0, 1)]

    def forward(self, x, step):
        p = self.params
        ok(F.conv_fprop(x, p["filters"], self.c, 0, self.conv_space[0]))
        ok(F.group_norm_fprop(self.c, p["gamma"], p["beta"], self.image(self.h), self.groups, self.norm_space[0],
                              activation="silu", mean=self.mean, rstd=self.rstd))
        ok(F.linear_fprop(self.h, p["weight"], p["bias"], self.l, self.linear_space[0], activation="gelu",
                          preactivation=self.z))
        ok(F.dropout_fprop(self.l, self.y, self.p, self.seed, step, residual=self.h))
        return self.y

    def backward(self, x, dy, step):
        p, g = self.params, self.grads
        ok(F.dropout_bprop(dy, self.dl, self.p, self.seed, step))
        ok(F.linear_bprop(self.h, p["weight"], self.dl, self.z, self.dh, g["weight"], g["bias"], self.linear_space[1],
                          activation="gelu"))
        self.dh += dy
        ok(F.group_norm_bprop(self.c, p["gamma"], p["beta"], self.mean, self.rstd, self.image(self.dh), self.dc, g["gamma"],
                              g["beta"], self.groups, self.norm_space[1], activation="silu"))
        ok(F.conv_accgrad(x, self.dc, g["filters"], 0, self.conv_space[1]))


def train(block, x, target, steps, rate=0.5):
    """The loss of each step."""
    losses = []
    for step in range(steps):
        off = block.forward(x, step) - target
        losses.append(float(off.square().mean()))
        block.backward(x, off * (2 / off.numel()), step)
        for k, v in block.params.items():
            v -= rate * block.grads[k]
    return losses


def data(block, batch=8, cin=16, size=27, seed=2):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, cin, size, size, generator=gen).to(block.c.device)
    return x, torch.randn(*block.y.shape, generator=gen).to(block.c.device) * 0.5


def main():
    steps = int(sys.argv[1]) if len(sys.argv) > 1 else 20
    block = ResidualBlock()
    for step, loss in enumerate(train(block, *data(block), steps)):
        print("step %d: loss %.5f" % (step, loss), flush=True)


if __name__ == "__main__":
    main()
