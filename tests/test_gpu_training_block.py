"""The training operators together: the block of examples/recurrent_block.py. Its gradients
against automatic differentiation of the same block in 64 bits, its training, and its answers
token by token against the whole sequence."""
import importlib.util
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(tcx):
    path = os.path.join(ROOT, "examples", "recurrent_block.py")
    spec = importlib.util.spec_from_file_location("recurrent_block", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def block_64(w, u, keep, p, lengths):
    def norm(x, weight, bias):
        m = x.mean(-1, keepdim=True)
        return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * weight + bias
    x = u @ w["w_in"].T
    n = norm(x, w["n1_w"], w["n1_b"])
    s = torch.sigmoid(n @ w["w_gate"].T + w["b_gate"])
    inp = n @ w["w_input"].T + w["b_input"]
    state, states = torch.zeros_like(x[:, 0]), []
    for t in range(u.shape[1]):
        on = (t < lengths)[:, None]
        state = torch.where(on, s[:, t] * state + (1 - s[:, t]) * inp[:, t], state)
        states.append(state)
    mixed = torch.stack(states, 1) @ w["w_out"].T + w["b_out"]
    z = norm(x + torch.where(keep, mixed / (1 - p), 0.0), w["n2_w"], w["n2_b"])
    return z @ w["w_head"].T


@pytest.mark.parametrize("batch,time,width", [(3, 50, 64), (2, 200, 37)])
def test_gradients_of_the_block(tcx, example, batch, time, width):
    """Relative error of each parameter's gradient within 2e-5: three products of 3xTF32 or
    float32 (some 1e-6 each) and two norms lie on the longest way back."""
    p, step, features = 0.2, 3, 8
    block = example.RecurrentBlock(features, width, 5, p=p, seed=11)
    u = tcx.randn((batch, time, features), seed=5)
    lengths = torch.tensor([time, time // 3, time - 7][:batch], dtype=torch.int32, device="cuda")
    out, _, kept = block.forward(u, lengths=lengths, step=step)
    dout = tcx.randn(out.shape, seed=6)
    grads = block.backward(dout, kept)
    offset = step * batch * time * width
    keep = (tcx.rand_uniform((batch, time, width), seed=11, offset=offset) >= p).cpu()
    w = {k: v.double().cpu().requires_grad_(True) for k, v in block.params.items()}
    want = block_64(w, u.double().cpu(), keep, p, lengths.cpu())
    assert float(((out.cpu().double() - want).norm() / want.norm()).detach()) < 1e-5
    (want * dout.double().cpu()).sum().backward()
    assert set(grads) == set(w)
    for name, g in grads.items():
        exact = w[name].grad
        assert float((g.cpu().double() - exact).norm() / exact.norm()) < 2e-5, name


def test_the_block_learns_and_serves(tcx, example):
    block, losses = example.train(120, 8, 96, 64)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-10:]) < 0.3 * np.mean(losses[:3]), (losses[:3], losses[-10:])
    u = tcx.randn((4, 40, 16), seed=99)
    whole, _, _ = block.forward(u)
    apart = example.serve(block, u)
    assert float((whole - apart).abs().max()) < 1e-4 * float(whole.abs().max() + 1)


def test_a_step_replays_as_a_graph(tcx, example):
    """A captured step reads its mask's place from a counter on the device."""
    from tensorcx_b200.graphs import CapturedSequence
    x, r = tcx.randn((64, 128), seed=1), tcx.randn((64, 128), seed=2)
    w = torch.ones(128, device="cuda")
    place = torch.zeros(1, dtype=torch.int64, device="cuda")

    def body():
        y, total, mean, rstd = tcx.layernorm_forward(x, w, w, residual=r, p=0.3, seed=4, offset=place)
        grads = tcx.layernorm_backward(y, total, mean, rstd, w, p=0.3, seed=4, offset=place)
        place.add_(x.numel())
        return (total, *grads)
    seq = CapturedSequence(body)
    place.zero_()
    for i in range(3):
        got = [t.clone() for t in seq()]
        y, total, mean, rstd = tcx.layernorm_forward(x, w, w, residual=r, p=0.3, seed=4, offset=i * x.numel())
        want = (total, *tcx.layernorm_backward(y, total, mean, rstd, w, p=0.3, seed=4, offset=i * x.numel()))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
    seq.release()
    h0 = torch.zeros(2, 40, device="cuda")
    gate, inp = tcx.randn((2, 500, 40), seed=3), tcx.randn((2, 500, 40), seed=4)
    seq = CapturedSequence(lambda: tcx.gated_recurrence(gate, inp, h0, form="sigmoid"))
    want = tcx.gated_recurrence(gate, inp, h0, form="sigmoid")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(seq(), want))
    seq.release()
