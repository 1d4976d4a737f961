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
_LAYER_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _layer_check(name: str, t: torch.Tensor, dtype: torch.dtype, device: torch.device, shape,
                 unit_cols: bool = False) -> None:
    """``t`` is a tensor of this dtype, device and shape (with ``unit_cols``: its
    last dimension has stride 1)."""
    if t.dtype is dtype and t.device == device and t.shape == shape:
        if unit_cols and t.stride()[-1] != 1 and t.shape[-1] > 1 and t.numel():
            raise ValueError(f"{name}: expected unit stride in the last dimension")
        return
    if t.device != device:
        raise ValueError(f"{name}: expected a CUDA tensor on {device}, got {t.device}")
    if t.dtype is not dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")


def _layer_dtype(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError(f"expected a CUDA tensor, got {t.device}")
    code = _LAYER_DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype}")
    return code


def _drop_spec(spec: _lib.DropoutC, drop: Dropout) -> None:
    spec.p = drop.p
    spec.seed = drop.seed & 0xFFFFFFFFFFFFFFFF
    spec.offset = drop.offset & 0xFFFFFFFFFFFFFFFF


# Handle of the current stream without building a torch.cuda.Stream for it (3 us).
_raw_stream = torch._C._cuda_getCurrentRawStream


def _layer_run(ask, run, args, x: torch.Tensor, device: torch.device,
               stream: Optional[int]) -> None:
    """Calls ``run`` with the workspace that ``ask`` names, on ``device``."""
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _layer_run(ask, run, args, x, device, stream)
    ref = ctypes.byref(args)
    need = ctypes.c_size_t()
    code = ask(ref, ctypes.byref(need))
    if code:
        _lib.check(code)
    if need.value:
        ws = x.new_empty(need.value, dtype=torch.uint8)
        if stream is not None:  # the allocator must not hand it out before that stream is done
            ws.record_stream(torch.cuda.ExternalStream(stream, device=device))
        args.workspace = ws.data_ptr()
        args.workspace_bytes = need.value
    code = run(ref, _raw_stream(index) if stream is None else stream)
    if code:
        _lib.check(code)


def _ld(t: torch.Tensor) -> int:
    """Row pitch of a 2-D tensor with unit column stride (rows of one row, or
    of one element, may carry any stride)."""
    rows, cols = t.shape
    pitch = t.stride()[0]
    return max(pitch, cols) if rows <= 1 else pitch


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
    for an activation.  ``out`` may be the residual.
    """
    code = _layer_dtype(x)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("expected 2-D x and w")
    act_code = ACTIVATIONS.get(act)
    if act_code is None:
        raise ValueError(f"unknown activation {act!r}")
    dtype, device = x.dtype, x.device
    M, K = x.shape
    N = w.shape[0]
    _layer_check("w", w, dtype, device, (N, K))
    a = _lib.LinearArgsC(code, M, N, K, x.data_ptr(), *x.stride(), w.data_ptr(), *w.stride())
    a.act = act_code
    if bias is not None:
        _layer_check("bias", bias, dtype, device, (N,), True)
        a.bias = bias.data_ptr()
    if residual is not None:
        _layer_check("residual", residual, dtype, device, (M, N), True)
        a.residual, a.ld_residual = residual.data_ptr(), _ld(residual)
    if out is None:
        out = x.new_empty(M, N)
        a.ld_out = N
    else:
        _layer_check("out", out, dtype, device, (M, N), True)
        a.ld_out = _ld(out)
    a.out = out.data_ptr()
    pre = None
    if save_pre:
        pre = x.new_empty(M, N)
        a.pre, a.ld_pre = pre.data_ptr(), N
    if drop is not None:
        _drop_spec(a.drop, drop)
    lib = _lib.lib()
    _layer_run(lib.fg_linear_workspace, lib.fg_linear, a, x, device, stream)
    return (out, pre) if save_pre else out


def linear_grad(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *,
                pre: Optional[torch.Tensor] = None, act: str = "none",
                drop: Optional[Dropout] = None, need_dx: bool = True, need_dw: bool = True,
                need_db: bool = True, dx_residual: Optional[torch.Tensor] = None,
                stream: Optional[int] = None):
    """``(dx, dw, db)`` of ``linear(x, w, bias, act=act, drop=drop)`` for the
    gradient ``dy`` of its output; ``pre`` is what ``save_pre`` returned (not
    needed for ``act="none"``).  Gradients that are not wanted are ``None``.
    The residual's gradient is ``dy`` itself; ``dx_residual`` [M, K] is added to
    ``dx`` in the product's epilogue.  With 16-bit types the gradient
    at the pre-activations is rounded to that type before the two products."""
    code = _layer_dtype(x)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError("expected 2-D x and w")
    act_code = ACTIVATIONS.get(act)
    if act_code is None:
        raise ValueError(f"unknown activation {act!r}")
    dtype, device = x.dtype, x.device
    M, K = x.shape
    N = w.shape[0]
    _layer_check("w", w, dtype, device, (N, K))
    _layer_check("dy", dy, dtype, device, (M, N))
    a = _lib.LinearGradArgsC(code, M, N, K, dy.data_ptr(), *dy.stride(), x.data_ptr(),
                             *x.stride(), w.data_ptr(), *w.stride())
    a.act = act_code
    if act != "none":
        if pre is None:
            raise ValueError(f"the gradient of {act} needs pre (linear(..., save_pre=True))")
        _layer_check("pre", pre, dtype, device, (M, N), True)
        a.pre, a.ld_pre = pre.data_ptr(), _ld(pre)
    dx = dw = db = None
    if need_dx:
        dx = x.new_empty(M, K)
        a.dx, a.ld_dx = dx.data_ptr(), K
        if dx_residual is not None:
            _layer_check("dx_residual", dx_residual, dtype, device, (M, K), True)
            a.dx_residual, a.ld_dx_residual = dx_residual.data_ptr(), _ld(dx_residual)
    elif dx_residual is not None:
        raise ValueError("dx_residual without dx")
    if need_dw:
        dw = x.new_empty(N, K)
        a.dw, a.ld_dw = dw.data_ptr(), K
    if need_db:
        db = x.new_empty(N)
        a.db = db.data_ptr()
    if drop is not None:
        _drop_spec(a.drop, drop)
    lib = _lib.lib()
    _layer_run(lib.fg_linear_grad_workspace, lib.fg_linear_grad, a, x, device, stream)
    return dx, dw, db


def dropout(x: torch.Tensor, drop: Optional[Dropout], *, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """``residual + dropout(x)`` on the last dimension's columns and the rows
    before it (a 1-D tensor is one row).  ``out`` may be ``x`` or the residual."""
    code = _layer_dtype(x)
    shape, dtype, device = x.shape, x.dtype, x.device
    flat = len(shape) != 2  # rows are then a contiguous tensor's
    cols = shape[-1] if shape else 1
    rows = x.numel() // cols if cols else 0

    def pitched(name: str, t: torch.Tensor):
        _layer_check(name, t, dtype, device, shape, not flat)
        if not flat:
            return t.data_ptr(), _ld(t)
        if not t.is_contiguous():
            raise ValueError(f"{name}: expected a 2-D or a contiguous tensor")
        return t.data_ptr(), cols

    ptrs = pitched("x", x)
    ptrs += (None, 0) if residual is None else pitched("residual", residual)
    if out is None:
        out = x.new_empty(shape)
        ptrs += (out.data_ptr(), cols)
    else:
        ptrs += pitched("out", out)
    spec = _lib.DropoutC()
    if drop is not None:
        _drop_spec(spec, drop)
    index = device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return dropout(x, drop, residual=residual, out=out, stream=stream)
    code = _lib.lib().fg_dropout(code, rows, cols, *ptrs, ctypes.byref(spec),
                                 _raw_stream(index) if stream is None else stream)
    if code:
        _lib.check(code)
    return out


def dropout_grad(dy: torch.Tensor, drop: Optional[Dropout], *, out: Optional[torch.Tensor] = None,
                 stream: Optional[int] = None) -> torch.Tensor:
    """d/dx of ``dropout(x, drop)``: the same mask and scale on ``dy``."""
    return dropout(dy, drop, out=out, stream=stream)


def check_device_error() -> None:
    call("fg_check_device_error")


def kernel_launches() -> int:
    return int(_lib.lib().fg_kernel_launches())
