"""Python entry points for the fused building blocks, on torch CUDA tensors.

torch only provides device memory and the current stream here; every call
lands in ``libferro_cuda.so``.  Each function names the reference computation
it implements.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import call


def _p(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(stream: Optional[int]) -> int:
    return torch.cuda.current_stream().cuda_stream if stream is None else stream


def _check_f32(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is None:
            continue
        if not (t.is_cuda and t.is_contiguous()):
            raise ValueError("expected a contiguous CUDA tensor")


def ew_fma_relu_scale(a, b, c, scale: float = 0.5, out=None, stream=None) -> torch.Tensor:
    """relu(a*b + c) * scale (Tensor::mul/add/relu, src/tensor.rs:471-491,519-531)."""
    _check_f32(a, b, c)
    out = torch.empty_like(a) if out is None else out
    call("fg_ew_fma_relu_scale", _p(a), _p(b), _p(c), _p(out), a.numel(), ctypes.c_float(scale),
         _stream(stream))
    return out


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return _lib.F32
    if t.dtype == torch.int32:
        return _lib.I32
    raise ValueError(f"unsupported dtype {t.dtype}")


def reduce_rows(x: torch.Tensor, op: int = _lib.REDUCE_SUM, stream=None) -> torch.Tensor:
    """Tensor::sum / Tensor::max over the last axis of a 2-D tensor (keepdim)."""
    _check_f32(x)
    rows, cols = x.shape
    out = torch.empty((rows, 1), dtype=x.dtype, device=x.device)
    call("fg_reduce_rows", _dtype_code(x), op, _p(x), _p(out), rows, cols, _stream(stream))
    return out


def reduce_cols(x: torch.Tensor, op: int = _lib.REDUCE_SUM, stream=None) -> torch.Tensor:
    """Tensor::sum / Tensor::max over axis 0 of a 2-D tensor (keepdim)."""
    _check_f32(x)
    rows, cols = x.shape
    out = torch.empty((1, cols), dtype=x.dtype, device=x.device)
    call("fg_reduce_cols", _dtype_code(x), op, _p(x), _p(out), rows, cols, _stream(stream))
    return out


def xent_fwd_bwd(logits: torch.Tensor, targets: torch.Tensor, need_grad: bool = True,
                 grad_scale: float = 1.0, stream=None):
    """Tensor::cross_entropy forward and d loss / d logits (src/tensor.rs:738-752)."""
    _check_f32(logits, targets)
    rows, cols = logits.shape
    loss = torch.empty(1, dtype=torch.float32, device=logits.device)
    dx = torch.empty_like(logits) if need_grad else None
    call("fg_xent_fwd_bwd", _p(logits), _p(targets), rows, cols, _p(loss), _p(dx),
         ctypes.c_float(grad_scale), _stream(stream))
    return loss, dx


def sgd_(param: torch.Tensor, grad: torch.Tensor, lr: float, param_lo=None, stream=None):
    """In-place Sgd::step update p <- p + (-(g*lr)) (src/optim.rs:60-71)."""
    _check_f32(param, grad)
    call("fg_sgd", _p(param), _p(grad), param.numel(), ctypes.c_float(lr), _p(param_lo),
         _stream(stream))
    return param


def split_lo(x: torch.Tensor, stream=None) -> torch.Tensor:
    """TF32 residual x - trunc_tf32(x) used by the 3xTF32 GEMM."""
    _check_f32(x)
    lo = torch.empty_like(x)
    call("fg_split_lo", _p(x), _p(lo), x.numel(), _stream(stream))
    return lo


def gemm(a, b, *, a_lo=None, b_lo=None, a_mn_major=False, b_mn_major=False, one_pass=False,
         epilogue=_lib.EPI_NONE, bias=None, mask=None, out=None, out_lo=None, stream=None):
    """C[m,n] = sum_k A(m,k) B(n,k) on the tcgen05 tensor cores (3xTF32).

    ``a`` is [M, K] (or [K, M] with ``a_mn_major``), ``b`` is [N, K] (or
    [K, N] with ``b_mn_major``).  Residuals are computed when not given.
    """
    _check_f32(a, b)
    M = a.shape[1] if a_mn_major else a.shape[0]
    K = a.shape[0] if a_mn_major else a.shape[1]
    N = b.shape[1] if b_mn_major else b.shape[0]
    if not one_pass:
        a_lo = split_lo(a, stream) if a_lo is None else a_lo
        b_lo = split_lo(b, stream) if b_lo is None else b_lo
    out = torch.empty((M, N), dtype=torch.float32, device=a.device) if out is None else out
    flags = ((_lib.GEMM_A_MN_MAJOR if a_mn_major else 0) | (_lib.GEMM_B_MN_MAJOR if b_mn_major else 0)
             | (_lib.GEMM_1XTF32 if one_pass else 0))
    call("fg_gemm_3xtf32", M, N, K, _p(a), _p(a_lo), a.stride(0), _p(b), _p(b_lo), b.stride(0),
         _p(out), _p(out_lo), out.stride(0), flags, epilogue, _p(bias), _p(mask),
         0 if mask is None else mask.stride(0), _stream(stream))
    return out


# ---- layer operators: linear + bias + activation + dropout + residual ----------
class Dropout(NamedTuple):
    """A dropout draw: probability ``p``, and the ``(seed, offset)`` that fix
    the mask.  Forward and backward calls with equal values see the same mask
    (it is recomputed, never stored); a training loop takes a new ``offset``
    for every layer and step."""

    p: float
    seed: int
    offset: int = 0


ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
               "gelu_tanh": _lib.ACT_GELU_TANH, "silu": _lib.ACT_SILU}
_NO_DROP = (0.0, 0, 0)
_layer_module = None


def _layer():
    """The binding of the layer operators (``csrc/layer_py.cpp``)."""
    global _layer_module
    if _layer_module is None:
        _lib.lib()
        try:
            from . import _layer as module
        except ImportError as e:  # pragma: no cover - build problem, fail loudly
            raise ImportError(
                "ferrograd_b200._layer is not built; run python -m ferrograd_b200.build") from e
        _layer_module = module
    return _layer_module


def _act_code(act: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"unknown activation {act!r}")
    return code


def linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           act: str = "none", residual: Optional[torch.Tensor] = None,
           drop: Optional[Dropout] = None, save_pre: bool = False,
           out: Optional[torch.Tensor] = None, stream: Optional[int] = None):
    """``residual + dropout(act(x @ w.T + bias))`` in one pass (Linear::forward,
    src/nn.rs:97-104, with its neighbours in the epilogue).

    ``x`` [M, K] and ``w`` [N, K] in f32, bf16 or f16, any strides (a weight
    kept as [K, N] is passed as its transpose); ``bias`` [N]; ``residual``
    [M, N].  ``act`` is one of ``ACTIVATIONS``.  With ``save_pre`` returns
    ``(out, pre)``, ``pre`` being the pre-activations ``linear_grad`` needs
    for an activation.  ``out`` may be the residual.  No autograd graph is
    recorded, whatever the arguments require.

    ``stream`` is a ``cudaStream_t`` as an integer (None: torch's current
    stream).  On another stream than the current one the call allocates its
    results and workspace there; what comes before and after it on other
    streams is for the caller to order (wait for an event), as in torch.  The
    same goes for ``linear_grad`` and ``dropout``.
    """
    p, seed, offset = _NO_DROP if drop is None else drop
    return _layer().linear(x, w, bias, _act_code(act), residual, p, seed, offset, save_pre, out,
                           stream)


def linear_grad(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *,
                pre: Optional[torch.Tensor] = None, act: str = "none",
                drop: Optional[Dropout] = None, need_dx: bool = True, need_dw: bool = True,
                need_db: bool = True, dx_residual: Optional[torch.Tensor] = None,
                stream: Optional[int] = None):
    """``(dx, dw, db)`` of ``linear(x, w, bias, act=act, drop=drop)`` for the
    gradient ``dy`` of its output; ``pre`` is what ``save_pre`` returned (not
    needed for ``act="none"``).  Gradients that are not wanted are ``None``.
    The residual's gradient is ``dy`` itself; ``dx_residual`` [M, K] is added to
    ``dx`` in the product's epilogue.  With 16-bit types the gradient at the
    pre-activations is rounded to that type before the two products (exact for
    ``"none"`` and ``"relu"``: dropout's scale multiplies the sums)."""
    code = _act_code(act)
    if code and pre is None:
        raise ValueError(f"the gradient of {act} needs pre (linear(..., save_pre=True))")
    p, seed, offset = _NO_DROP if drop is None else drop
    return _layer().linear_grad(dy, x, w, pre, code, p, seed, offset, need_dx, need_dw, need_db,
                                dx_residual, stream)


def dropout(x: torch.Tensor, drop: Optional[Dropout], *, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """``residual + dropout(x)`` on the last dimension's columns and the rows
    before it (a 1-D tensor is one row).  ``out`` may be ``x`` or the residual."""
    p, seed, offset = _NO_DROP if drop is None else drop
    return _layer().dropout(x, residual, p, seed, offset, out, stream)


def dropout_grad(dy: torch.Tensor, drop: Optional[Dropout], *, out: Optional[torch.Tensor] = None,
                 stream: Optional[int] = None) -> torch.Tensor:
    """d/dx of ``dropout(x, drop)``: the same mask and scale on ``dy``."""
    return dropout(dy, drop, out=out, stream=stream)


def check_device_error() -> None:
    call("fg_check_device_error")


def kernel_launches() -> int:
    return int(_lib.lib().fg_kernel_launches())
