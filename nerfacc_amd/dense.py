"""A dense layer with its epilogue: the building block of a radiance field's decoder, between `sampling` and `rendering`.

No reference counterpart: the reference leaves fields to its examples (examples/radiance_fields/mlp.py:16-107, torch layers).
"""
import functools
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad
from torch import Tensor

from . import cuda as _C

_ACTIVATIONS = {None: 0, "relu": 1, "sigmoid": 2, "softplus": 3, "silu": 4, "gelu": 5, "exp": 6}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


_EXT = None                   # the torch extension, False on the ctypes face, None before the first call


def _ext():
    """the torch extension, which holds each operator as one call (refusals, autograd and launch); False on the ctypes face, where the
    same steps are Python"""
    global _EXT
    if _EXT is None:
        from .cuda import _backend

        _EXT = _backend._C if _backend.BACKEND == "ext" else False
    return _EXT


def _check_native(name: str, ref: Tensor, others) -> None:
    """the refusals that every feature operator shares; `others`: (name, tensor or None, shape, dtype)"""
    if not ref.is_cuda:
        raise RuntimeError(f"{name}: inputs must be a CUDA/HIP tensor (nerfacc_amd has no CPU kernels)")
    if ref.dtype not in _DTYPES:
        raise TypeError(f"{name}: inputs must be float32, bfloat16 or float16, got {ref.dtype}")
    for what, t, shape, dtype in others:
        if t is None:
            continue
        if not isinstance(t, Tensor):
            raise TypeError(f"{name}: {what} must be a torch.Tensor, got {type(t)}")
        if t.device != ref.device:
            raise RuntimeError(f"{name}: {what} is on {t.device}, inputs on {ref.device}")
        if t.dtype != dtype:
            raise TypeError(f"{name}: {what} must have dtype {dtype}, got {t.dtype}")
        if t.shape != torch.Size(shape):
            raise ValueError(f"{name}: {what} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _refuse_forward(name: str, *tensors) -> None:
    """a tangent would be dropped without a word"""
    if torch._C._is_fwd_grad_enabled() and any(isinstance(t, Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name}: forward mode derivatives are not implemented")


def _capturing(tensors) -> bool:
    """whether the current stream of the tensors' device is being captured into a graph"""
    with torch.cuda.device(next(t.device for t in tensors if t is not None)):
        return torch.cuda.is_current_stream_capturing()


def _records_grad(name: str, *tensors) -> bool:
    """whether autograd records the call; refuses one whose captured backward pass would end the process, or (without the extension, which
    alone can tell) might"""
    if not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)):
        return False
    if _capturing(tensors) and _C.foreign_nodes(tensors):
        raise RuntimeError(f"{name}: captured into a graph while an eager autograd graph of the same tensors lives, or may live without the torch "
                           "extension to tell (its backward pass could not be captured): drop the eager outputs first, or call under torch.no_grad()")
    return True


def _activation_id(name: str, activation: Optional[str], allowed=tuple(_ACTIVATIONS)) -> int:
    if activation not in allowed:
        raise ValueError(f"{name}: activation must be one of {', '.join(map(repr, allowed))}, got {activation!r}")
    return _ACTIVATIONS[activation]


def linear(inputs: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
           residual: Optional[Tensor] = None) -> Tensor:
    """`activation(inputs @ weight.T + bias) + residual` in one kernel, differentiable in all four tensors.

    Args:
        inputs: (..., in_features); rows may be strided (a slice of a wider tensor), float32, bfloat16 or float16; up to 2^20 features in and
            out.
        weight: (out_features, in_features), the same dtype.
        bias: (out_features,), the same dtype.
        activation: None, "relu", "sigmoid", "softplus", "silu", "gelu" (the exact form) or "exp" (a field's density).
        residual: (..., out_features), the same dtype, added behind the activation.

    Sums are held in 32 bits and the result is rounded once.  The backward pass differentiates once; its sums have a fixed order
    (the same bits every time).  Forward mode derivatives are refused, second ones raise.  All tensors have one dtype: autocast does not
    cast for it.

        >>> x = torch.tensor([[1., 2.]], device="cuda")
        >>> linear(x, torch.tensor([[1., 1.], [1., -1.]], device="cuda"), activation="relu")
        tensor([[3., 0.]], device='cuda:0')
    """
    act = _activation_id("linear", activation)
    ext = _EXT or _ext()
    if ext:
        return ext.linear(inputs, weight, bias, residual, act)
    _refuse_forward("linear", inputs, weight, bias, residual)
    if not isinstance(inputs, Tensor) or not isinstance(weight, Tensor):
        raise TypeError("linear: inputs and weight must be torch.Tensors")
    if inputs.dim() < 1 or weight.dim() != 2 or inputs.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear: inputs (..., in) and weight (out, in) expected, got {tuple(inputs.shape)} and {tuple(weight.shape)}")
    n, k = weight.shape
    if n == 0 or k == 0:
        raise ValueError("linear: in_features and out_features must be at least 1")
    if max(n, k) > 1 << 20:
        raise ValueError("linear: more than 2^20 features")
    shape = inputs.shape[:-1] + (n,)
    _check_native("linear", inputs, (("weight", weight, (n, k), inputs.dtype), ("bias", bias, (n,), inputs.dtype),
                                     ("residual", residual, shape, inputs.dtype)))
    x = inputs if inputs.dim() == 2 else inputs.reshape(-1, k)
    r = None if residual is None else (residual if residual.dim() == 2 else residual.reshape(-1, n))
    if _records_grad("linear", inputs, weight, bias, residual):
        out = _Linear.apply(x, weight, bias, r, act)
    else:
        out = _C.linear_fwd(x, weight, bias, r, act, False)[0]
    return out if inputs.dim() == 2 else out.view(shape)


class _Once(torch.autograd.Function):
    """passes gradients through; a backward pass over it is an error"""

    @staticmethod
    def forward(ctx, *grads):
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("trying to differentiate twice a function that was marked with @once_differentiable")


def _differentiates_once(depends):
    """A backward pass that differentiates once.  Under create_graph those of its results that depend on something learnt are an error in
    another backward pass (a penalty on them would have no effect otherwise): all where a gradient that came in requires one, else those
    that `depends(ctx)` names, a truth value for each."""
    def wrap(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            with torch.no_grad():
                outs = backward(ctx, *grads)
            if not torch.is_grad_enabled():
                return outs
            outer = any(g is not None and g.requires_grad for g in grads)
            names = depends(ctx)
            held = [i for i, g in enumerate(outs) if g is not None and (outer or (i < len(names) and names[i]))]
            marked = _Once.apply(*(outs[i].detach().requires_grad_(True) for i in held)) if held else ()
            return tuple(marked[held.index(i)] if i in held else g for i, g in enumerate(outs))
        return run
    return wrap


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        learns = any(ctx.needs_input_grad[:3])
        slope = learns and act > 1                          # act' depends on something learnt
        ctx.depends = (slope or ctx.needs_input_grad[1], slope or ctx.needs_input_grad[0], slope)
        out, saved = _C.linear_fwd(x, weight, bias, residual, act, learns)
        ctx.act, ctx.has_bias = act, bias is not None
        if learns:
            ctx.save_for_backward(x, weight, out if saved is None and act else saved)
        return out

    @staticmethod
    @_differentiates_once(lambda ctx: ctx.depends)
    def backward(ctx, grad):
        gx = gw = gb = None
        need = ctx.needs_input_grad
        if any(need[:3]):
            x, weight, saved = ctx.saved_tensors
            gx, gw, gb = _C.linear_bwd(grad, x, weight, saved, ctx.act, need[0], need[1], ctx.has_bias and need[2])
        return gx, gw, gb, (grad if need[3] else None), None
