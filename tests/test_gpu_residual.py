"""The residual MLP: one step's loss, gradients and update against torch's
64-bit autograd with the same dropout masks, and training in every type."""
import math

import numpy as np
import pytest
import torch

from ferrograd_b200 import data
from ferrograd_b200.residual import ResidualMlp
from layer_ref import keep_mask, threshold

pytestmark = pytest.mark.gpu


def reference(model, x, t, steps):
    """Loss and gradients in 64 bits, from the model's parameters."""
    params = [[p.detach().double().cpu().requires_grad_() for p in layer.params]
              for layer in model.layers()]
    width = 2 * len(model.blocks)

    def drop(v, layer, index):
        if layer.p == 0:
            return v
        mask = torch.from_numpy(keep_mask(*v.shape, layer.p, model.seed, steps * width + index))
        return torch.where(mask, v / (1 - threshold(layer.p) / 65536), 0.0)

    it = iter(zip(params, model.layers()))
    (w, b), _ = next(it)
    h = x.double().cpu() @ w.t() + b
    for i in range(len(model.blocks)):
        (w1, b1), up = next(it)
        (w2, b2), down = next(it)
        z = h @ w1.t() + b1
        a = {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu,
             "relu": torch.relu}[up.act](z)
        h = h + drop(drop(a, up, 2 * i) @ w2.t() + b2, down, 2 * i + 1)
    (w, b), _ = next(it)
    logits = h @ w.t() + b
    loss = -(t.double().cpu() * torch.log_softmax(logits, 1)).sum(1).mean()
    loss.backward()
    return float(loss.detach()), [[p.grad for p in pair] for pair in params]


@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_step_against_autograd(act, p):
    """f32: every sum of the step is good to 2^-20 of its terms and a chain of a
    dozen of them to 1e-4 of the largest gradient of a parameter."""
    x, t = data.mlp_batch(96, 50, 7, 1, 2)
    x, t = torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()
    model = ResidualMlp(50, 40, 136, 7, 2, act=act, p=p)
    model.train_step(x, t, 0.01)
    ref_loss, ref_grads = reference(model, x, t, 1)
    before = [[q.clone() for q in layer.params] for layer in model.layers()]
    loss = float(model.train_step(x, t, 0.01))
    assert abs(loss - ref_loss) <= 1e-5 * abs(ref_loss)
    for layer, old, grads in zip(model.layers(), before, ref_grads):
        for new, o, g in zip(layer.params, old, grads):
            got = (o - new).double().cpu() / 0.01
            # the difference of two f32 parameters, over the rate
            slack = 2.0 ** -22 * float(o.abs().max()) / 0.01
            assert float((got - g).abs().max()) <= 1e-4 * float(g.abs().max()) + slack


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_training_lowers_the_loss_and_serves(dtype):
    x, t = data.mlp_batch(128, 64, 10, 3, 4)
    x, t = torch.from_numpy(x).cuda(), torch.from_numpy(t).cuda()
    model = ResidualMlp(64, 64, 256, 10, 2, p=0.1, dtype=dtype)
    losses = [float(model.train_step(x, t, 0.02)) for _ in range(60)]
    assert all(math.isfinite(v) for v in losses)
    assert np.mean(losses[-10:]) < 0.8 * np.mean(losses[:5])
    together = model(x).float()
    alone = torch.cat([model(x[i:i + 1]) for i in range(4)]).float()
    # four layers, each rounding its output once: 4 roundings and their growth
    unit = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert float((together[:4] - alone).abs().max()) <= 16 * unit * float(together.abs().max())


def test_misuse():
    model = ResidualMlp(8, 8, 16, 3, 1)
    with pytest.raises(RuntimeError):
        model.backward(torch.zeros((2, 3), device="cuda"))
    with pytest.raises(RuntimeError):
        model.first.step(0.1)
    with pytest.raises(ValueError):
        ResidualMlp(8, 8, 16, 3, 1, act="tanh")
