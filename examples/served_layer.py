"""A feed-forward block trained with orthogonalised updates and then served in 4 bits.

    norm      n = layer_norm(x)
    up        h = gelu(n w1^T + b1)
    down      y = h w2^T + b2 + x

The loss is the mean squared distance to a target.  Every gradient comes from the library; the two weight matrices move by
their momentum, made nearly orthogonal, everything else by its gradient.  Then the weights go to microscaled 4-bit floating
point, and rows one by one through the block.

    python examples/served_layer.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import fbcuda_amd as F  # noqa: E402


def ok(code):
    if code != F.Success:
        raise RuntimeError(F.error_string(code))


def space(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device)


class Block:
    """Shapes, parameters, buffers and workspaces of one block, allocated once."""

    def __init__(self, rows=256, width=64, hidden=192, seed=1, dtype=torch.float32, device="cuda"):
        self.rows, self.device, self.dtype = rows, device, dtype
        gen = torch.Generator().manual_seed(seed)
        randn = lambda *shape: torch.randn(*shape, generator=gen).to(device)  # noqa: E731
        self.params = {
            "gamma": torch.ones(width, device=device), "beta": torch.zeros(width, device=device),
            "w1": (randn(hidden, width) * width ** -0.5).to(dtype), "b1": torch.zeros(hidden, device=device),
            "w2": (randn(width, hidden) * hidden ** -0.5).to(dtype), "b2": torch.zeros(width, device=device)}
        self.grads = {k: torch.empty_like(v) for k, v in self.params.items()}
        self.momentum = {k: torch.zeros_like(self.params[k]) for k in ("w1", "w2")}
        self.update = {k: torch.empty_like(self.params[k]) for k in ("w1", "w2")}
        make = lambda cols: torch.empty((rows, cols), dtype=dtype, device=device)  # noqa: E731
        self.n, self.dn, self.y, self.dx = (make(width) for _ in range(4))
        self.h, self.z, self.dh = (make(hidden) for _ in range(3))
        self.mean, self.rstd = (torch.empty(rows, device=device) for _ in range(2))
        self.norm_space = [space(F.layer_norm_workspace(q, rows, width), device) for q in (0, 1)]
        self.up_space = [space(F.linear_workspace(q, rows, width, hidden, dtype), device) for q in (0, 1)]
        self.down_space = [space(F.linear_workspace(q, rows, hidden, width, dtype), device) for q in (0, 1)]
        self.update_space = {k: space(F.orthogonalize_workspace(1, *self.params[k].shape), device) for k in self.update}

    def forward(self, x):
        p = self.params
        ok(F.layer_norm_fprop(x, p["gamma"], p["beta"], self.n, self.norm_space[0], mean=self.mean, rstd=self.rstd))
        ok(F.linear_fprop(self.n, p["w1"], p["b1"], self.h, self.up_space[0], activation="gelu", preactivation=self.z))
        ok(F.linear_fprop(self.h, p["w2"], p["b2"], self.y, self.down_space[0], residual=x))
        return self.y

    def backward(self, x, dy):
        p, g = self.params, self.grads
        ok(F.linear_bprop(self.h, p["w2"], dy, None, self.dh, g["w2"], g["b2"], self.down_space[1]))
        ok(F.linear_bprop(self.n, p["w1"], self.dh, self.z, self.dn, g["w1"], g["b1"], self.up_space[1], activation="gelu"))
        ok(F.layer_norm_bprop(x, p["gamma"], self.mean, self.rstd, self.dn, self.dx, g["gamma"], g["beta"], self.norm_space[1]))
        self.dx += dy
        return self.dx

    def step(self, rate=0.05, decay=0.9):
        for k, v in self.params.items():
            if k in self.update:
                rows, cols = v.shape
                self.momentum[k].mul_(decay).add_(self.grads[k])
                ok(F.orthogonalize(self.momentum[k], self.update[k], self.update_space[k], scale=max(1.0, rows / cols) ** 0.5))
                v -= rate * self.update[k]
            else:
                v -= rate * self.grads[k]


class Served:
    """The block for a few rows at a time, its weights in 4 bits."""

    def __init__(self, block, rows=1):
        p, d = block.params, block.device
        self.params, self.weights = p, {}
        for k in ("w1", "w2"):
            n, cols = p[k].shape
            blocks = -(-cols // 32)
            codes = torch.empty((n, 16 * blocks), dtype=torch.uint8, device=d)
            scales = torch.empty((n, blocks), dtype=torch.uint8, device=d)
            ok(F.mx4_quantize(p[k], codes, scales))
            self.weights[k] = codes, scales
        hidden, width = p["w1"].shape
        make = lambda cols: torch.empty((rows, cols), dtype=block.dtype, device=d)  # noqa: E731
        self.n, self.h, self.y = make(width), make(hidden), make(width)
        self.norm_space = space(F.layer_norm_workspace(0, rows, width), d)
        self.up_space = space(F.linear_mx4_workspace(rows, width, hidden), d)
        self.down_space = space(F.linear_mx4_workspace(rows, hidden, width), d)

    def __call__(self, x):
        p = self.params
        ok(F.layer_norm_fprop(x, p["gamma"], p["beta"], self.n, self.norm_space))
        ok(F.linear_mx4_fprop(self.n, *self.weights["w1"], p["b1"], self.h, self.up_space, activation="gelu"))
        ok(F.linear_mx4_fprop(self.h, *self.weights["w2"], p["b2"], self.y, self.down_space, residual=x))
        return self.y


def data(block, seed=2):
    gen = torch.Generator().manual_seed(seed)
    make = lambda: torch.randn(*block.y.shape, generator=gen).to(block.device).to(block.dtype)  # noqa: E731
    return make(), make()


def train(block, x, target, steps):
    """The loss of each step."""
    losses = []
    for _ in range(steps):
        off = block.forward(x) - target
        losses.append(float(off.float().square().mean()))
        block.backward(x, off * (2 / off.numel()))
        block.step()
    return losses


def main():
    steps = int(sys.argv[1]) if len(sys.argv) > 1 else 30
    block = Block()
    x, target = data(block)
    for step, loss in enumerate(train(block, x, target, steps)):
        print("step %d: loss %.5f" % (step, loss), flush=True)
    y, served = block.forward(x), Served(block)
    off = torch.cat([served(x[i:i + 1]) - y[i:i + 1] for i in range(block.rows)])
    print("served in 4 bits: %.3f of the block's own change to its rows" % float(off.norm() / (y - x).norm()))


if __name__ == "__main__":
    main()
