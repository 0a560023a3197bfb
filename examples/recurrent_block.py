"""Trains a residual recurrent block and serves it token by token.

    python examples/recurrent_block.py [--steps 200] [--batch 8] [--time 256] [--width 128]

The block mixes a sequence with a gated recurrence between two norms:

    x = u W_in                      n = layernorm(x)
    h = recurrence(n W_g + b_g, n W_i + b_i)        (sigmoid gates)
    z = layernorm(x + dropout(h W_o))               (one call)
    out = z W_head

It learns to follow running averages of its input, each with a decay of its own, from padded
sequences of different lengths. Every product is ops.linear / ops.matmul, and the gradients are
the operators' own backward calls: nothing is differentiated automatically. Afterwards the block
answers one token at a time from the recurrence's state, which gives the same outputs as the
whole sequence at once.
"""
from __future__ import annotations

import argparse
import math
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from tensorcx_b200 import ops  # noqa: E402


def linear_backward(dy, x, weight):
    """(dx, dweight, dbias) of ops.linear for x [..., in] and weight [out, in]."""
    rows = dy.reshape(-1, dy.shape[-1])
    dx = ops.matmul(rows, weight).view(*dy.shape[:-1], weight.shape[1])
    dweight = ops.matmul(rows.t().contiguous(), x.reshape(-1, x.shape[-1]))
    return dx, dweight, ops.sum(rows, axis=0)


class RecurrentBlock:
    def __init__(self, features: int, width: int, outputs: int, p: float = 0.1, seed: int = 0):
        def weight(index, out, inner):
            scale = 1.0 / math.sqrt(inner)
            return ops.rand_uniform((out, inner), -scale, scale, seed=seed * 16 + index)

        def full(value, n):
            return torch.full((n,), value, device="cuda")
        self.p, self.seed = p, seed
        self.params = dict(
            w_in=weight(1, width, features), n1_w=full(1.0, width), n1_b=full(0.0, width),
            w_gate=weight(2, width, width), b_gate=full(1.0, width), w_input=weight(3, width, width),
            b_input=full(0.0, width), w_out=weight(4, width, width), b_out=full(0.0, width),
            n2_w=full(1.0, width), n2_b=full(0.0, width), w_head=weight(5, outputs, width))

    def forward(self, u, state=None, *, lengths=None, step: int | None = None):
        """(outputs, state, what backward needs). `step` counts the training steps and places
        the dropout mask in the seed's stream; None (serving) drops nothing."""
        w, k = self.params, {}
        k["u"], k["state"], k["lengths"] = u, state, lengths
        width = w["w_in"].shape[0]
        k["p"], k["offset"] = (0.0, 0) if step is None else (self.p, step * u.shape[0] * u.shape[1] * width)
        x = ops.linear(u, w["w_in"])
        k["n"], _, k["m1"], k["r1"] = ops.layernorm_forward(x, w["n1_w"], w["n1_b"])
        k["gate"] = ops.linear(k["n"], w["w_gate"], w["b_gate"])
        k["input"] = ops.linear(k["n"], w["w_input"], w["b_input"])
        k["h"], state = ops.gated_recurrence(k["gate"], k["input"], state, form="sigmoid", lengths=lengths)
        mixed = ops.linear(k["h"], w["w_out"], w["b_out"])
        k["z"], k["total"], k["m2"], k["r2"] = ops.layernorm_forward(
            mixed, w["n2_w"], w["n2_b"], residual=x, p=k["p"], seed=self.seed, offset=k["offset"])
        k["x"] = x
        return ops.linear(k["z"], w["w_head"]), state, k

    def backward(self, dout, k):
        """The gradient of every parameter."""
        w, g = self.params, {}
        dz, g["w_head"], _ = linear_backward(dout, k["z"], w["w_head"])
        dmixed, dx, g["n2_w"], g["n2_b"] = ops.layernorm_backward(
            dz, k["total"], k["m2"], k["r2"], w["n2_w"], p=k["p"], seed=self.seed, offset=k["offset"])
        dh, g["w_out"], g["b_out"] = linear_backward(dmixed, k["h"], w["w_out"])
        dgate, dinput, _ = ops.gated_recurrence_backward(dh, k["gate"], k["input"], k["h"], k["state"], form="sigmoid",
                                                         lengths=k["lengths"])
        dn, g["w_gate"], g["b_gate"] = linear_backward(dgate, k["n"], w["w_gate"])
        dn_input, g["w_input"], g["b_input"] = linear_backward(dinput, k["n"], w["w_input"])
        dx, _, g["n1_w"], g["n1_b"] = ops.layernorm_backward(ops.add(dn, dn_input), k["x"], k["m1"], k["r1"], w["n1_w"],
                                                             dtotal=dx)
        _, g["w_in"], _ = linear_backward(dx, k["u"], w["w_in"])
        return g


class Momentum:
    def __init__(self, params, rate: float, keep: float = 0.9):
        self.rate, self.keep = (torch.tensor(v, device="cuda") for v in (rate, keep))
        self.speed = {name: torch.zeros_like(t) for name, t in params.items()}

    def step(self, params, grads):
        for name, g in grads.items():
            self.speed[name] = ops.add(ops.multiply(self.speed[name], self.keep), g)
            params[name] = ops.subtract(params[name], ops.multiply(self.speed[name], self.rate))


def batch_of(step: int, batch: int, time: int, features: int, decays):
    """Inputs, the running averages to follow and the sequences' lengths, on the device."""
    u = ops.randn((batch, time, features), seed=1234 + step)
    lengths = torch.randint(time // 2, time + 1, (batch,), dtype=torch.int32,
                            generator=torch.Generator().manual_seed(step)).cuda()
    gates = decays.expand(batch, time, features).contiguous()
    wanted, _ = ops.gated_recurrence(gates, ops.multiply(u, ops.subtract(torch.ones_like(gates), gates)))
    inside = (torch.arange(time, device="cuda")[None, :] < lengths[:, None]).float()[:, :, None].contiguous()
    return u, wanted, lengths, inside


def train(steps: int, batch: int, time: int, width: int, features: int = 16, rate: float = 0.05):
    block = RecurrentBlock(features, width, features, p=0.05, seed=7)
    decays = torch.linspace(0.5, 0.98, features, device="cuda")
    optimizer = Momentum(block.params, rate)
    losses = []
    for step in range(steps):
        u, wanted, lengths, inside = batch_of(step, batch, time, features, decays)
        out, _, kept = block.forward(u, lengths=lengths, step=step)
        off = ops.multiply(ops.subtract(out, wanted), inside)
        count = ops.sum(inside) * features
        losses.append(ops.divide(ops.sum(ops.multiply(off, off)), count))
        grads = block.backward(ops.multiply(off, 2.0 / count), kept)
        optimizer.step(block.params, grads)
    return block, [float(v) for v in losses]


def serve(block: RecurrentBlock, u):
    """Outputs of a batch of sequences, a token of each at a time."""
    state = torch.zeros(u.shape[0], block.params["w_in"].shape[0], device="cuda")
    outs = []
    for t in range(u.shape[1]):
        out, state, _ = block.forward(u[:, t:t + 1].contiguous(), state)
        outs.append(out)
    return torch.cat(outs, 1)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--time", type=int, default=256)
    ap.add_argument("--width", type=int, default=128)
    a = ap.parse_args()
    block, losses = train(a.steps, a.batch, a.time, a.width)
    for i in range(0, len(losses), max(1, len(losses) // 8)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"last       loss {losses[-1]:.5f}")
    u = ops.randn((a.batch, 64, 16), seed=99)
    whole, _, _ = block.forward(u)
    apart = serve(block, u)
    print(f"token by token against the whole sequence: largest difference {float((whole - apart).abs().max()):.2e}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
