"""Residual MLPs on the layer operators (``kernels.linear`` / ``linear_grad``).

The reference's MLP (Linear layers with ReLU between them, examples/mnist.rs)
grows here into residual blocks with dropout:

    block(x) = x + D(D(act(x w1^T + b1)) w2^T + b2)

``ResidualMlp`` puts blocks between an input and an output ``Linear``.  One
training step is forward -> cross_entropy -> backward -> Sgd as in the
reference's loop (examples/mnist.rs:90-97); bias, activation, dropout and
residual run inside the products, and no dropout mask is kept: the backward
pass recomputes it from ``(seed, offset)``.

Weights are initialised as ``Linear::new`` (src/nn.rs:77-85).  With a 16-bit
``dtype`` the layers compute in that type from f32 master weights, which
``Sgd::step`` (src/optim.rs:60-71) updates.  The loss is not scaled: in f16,
gradients below 2^-24 are lost, so bf16 is the type for large batches.
"""
from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import kernels
from .mlp import InitRng, linear_init


class Layer:
    """One ``Linear`` with activation and dropout in its epilogue: f32 master
    parameters, their copies in the compute type, and their gradients."""

    def __init__(self, in_features: int, out_features: int, rng: InitRng, device: torch.device,
                 dtype: torch.dtype, act: str = "none", p: float = 0.0):
        if act not in kernels.ACTIVATIONS:
            raise ValueError(f"unknown activation {act!r}")
        w, b = linear_init(in_features, out_features, rng)
        self.master = [torch.from_numpy(w).to(device), torch.from_numpy(b).to(device)]
        self.params = [m if dtype == torch.float32 else m.to(dtype) for m in self.master]
        self.grads: List[Optional[torch.Tensor]] = [None, None]
        self.act, self.p = act, p
        self._saved: Optional[Tuple] = None

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                drop: Optional[kernels.Dropout] = None, train: bool = False) -> torch.Tensor:
        w, b = self.params
        need_pre = train and self.act != "none"
        got = kernels.linear(x, w, b, act=self.act, residual=residual, drop=drop,
                             save_pre=need_pre)
        out, pre = got if need_pre else (got, None)
        self._saved = (x, pre, drop) if train else None
        return out

    def backward(self, dy: torch.Tensor, need_dx: bool = True,
                 dx_residual: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        if self._saved is None:
            raise RuntimeError("backward without a training forward pass")
        x, pre, drop = self._saved
        self._saved = None
        dx, dw, db = kernels.linear_grad(dy, x, self.params[0], pre=pre, act=self.act, drop=drop,
                                         need_dx=need_dx, dx_residual=dx_residual)
        self.grads = [dw, db]
        return dx

    def step(self, lr: float) -> None:
        for i, grad in enumerate(self.grads):
            if grad is None:
                raise RuntimeError("step without a backward pass")
            kernels.sgd_(self.master[i], grad.float(), lr)
            if self.params[i] is not self.master[i]:
                self.params[i].copy_(self.master[i])
        self.grads = [None, None]


class ResidualMlp:
    """``Linear(d_in, width) -> blocks -> Linear(width, classes)``; each block
    is two layers, ``width -> hidden -> width``, around a residual."""

    def __init__(self, d_in: int, width: int, hidden: int, classes: int, blocks: int, *,
                 act: str = "gelu", p: float = 0.0, dtype: torch.dtype = torch.float32,
                 seed: int = 42, device: str = "cuda"):
        dev = torch.device(device)
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        rng = InitRng(seed)
        make = lambda i, o, a="none", q=0.0: Layer(i, o, rng, dev, dtype, a, q)  # noqa: E731
        self.dtype, self.seed = dtype, seed
        self.first = make(d_in, width)
        self.blocks = [(make(width, hidden, act, p), make(hidden, width, "none", p))
                       for _ in range(blocks)]
        self.last = make(width, classes)
        self.steps = 0
        self.draws = 0  # training forward passes so far

    def layers(self) -> List[Layer]:
        return [self.first, *[layer for block in self.blocks for layer in block], self.last]

    def _drop(self, layer: Layer, index: int, train: bool) -> Optional[kernels.Dropout]:
        """The layer's draw of this pass: every layer and training pass has its own offset."""
        if not train or layer.p == 0.0:
            return None
        return kernels.Dropout(layer.p, self.seed, self.draws * 2 * len(self.blocks) + index)

    def forward(self, x: torch.Tensor, train: bool = False) -> torch.Tensor:
        """Logits [rows, classes]; a single row to serve is ``x`` of one row."""
        h = self.first.forward(x.to(self.dtype), train=train)
        for i, (up, down) in enumerate(self.blocks):
            a = up.forward(h, drop=self._drop(up, 2 * i, train), train=train)
            h = down.forward(a, residual=h, drop=self._drop(down, 2 * i + 1, train), train=train)
        if train:
            self.draws += 1
        return self.last.forward(h, train=train)

    __call__ = forward

    def backward(self, dlogits: torch.Tensor) -> None:
        """Gradients of every parameter, for the last training forward pass, into the
        layers' ``grads`` (in place of what was there)."""
        dh = self.last.backward(dlogits.to(self.dtype))
        for up, down in reversed(self.blocks):
            # the residual passes dh on unchanged, next to the block's own path
            dh = up.backward(down.backward(dh), dx_residual=dh)
        self.first.backward(dh, need_dx=False)

    def train_step(self, x: torch.Tensor, targets: torch.Tensor, lr: float) -> torch.Tensor:
        """One step on a batch with dense targets [rows, classes]; returns the
        loss (a device scalar; the mean over the rows)."""
        logits = self.forward(x, train=True)
        loss, dlogits = kernels.xent_fwd_bwd(logits.float(), targets)
        self.backward(dlogits)
        for layer in self.layers():
            layer.step(lr)
        self.steps += 1
        return loss
