"""The residual MLP's dropout draws: one for every layer and training pass."""
import pytest
import torch

from ferrograd_b200.residual import ResidualMlp

pytestmark = pytest.mark.gpu


def test_every_training_pass_draws_anew():
    x = torch.randn((64, 20), device="cuda")
    t = torch.zeros((64, 5), device="cuda")
    t[:, 2] = 1
    make = lambda: ResidualMlp(20, 32, 64, 5, 2, p=0.5, seed=9)  # noqa: E731
    model = make()
    first, second = model.forward(x, train=True), model.forward(x, train=True)
    assert not torch.equal(first, second)  # two passes within a step
    assert torch.equal(model(x), model(x))  # none without training
    again = make()
    assert torch.equal(again.forward(x, train=True), first)  # fixed by seed and count
    again(x)
    assert torch.equal(again.forward(x, train=True), second)
    # a step's pass is one of them
    third = model.forward(x, train=True)
    again.train_step(x, t, 0.0)
    assert not torch.equal(again.forward(x, train=True), third)
    assert torch.equal(model.forward(x, train=True), make_fourth(make, x))


def make_fourth(make, x):
    model = make()
    for _ in range(3):
        model.forward(x, train=True)
    return model.forward(x, train=True)
