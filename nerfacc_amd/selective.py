"""Learned mixing along rays: a short causal convolution and a selective state space scan over each ray's samples.

They stand beside the sums and products of `scan.py` and take the same layouts: flattened samples with `packed_info` [n_rays, 2], or
batched (n_rays, n, channels) tensors.  The recurrence h[t] = exp(step A) h[t - 1] + step B[t] u[t] is the general linear one along a
ray; front-to-back compositing is its case of one state.  No reference counterpart (the reference's scans, nerfacc/scan.py:12-294, are
sums and products of one number per sample).
"""
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import cuda as _C
from .dense import _activation_id, _check_native, _differentiates_once, _ext, _records_grad, _refuse_forward

_MAX_STATES = 256


def _check_channels(name: str, channels: int) -> None:
    if channels > 1 << 23:
        raise ValueError(f"{name}: more than 2^23 channels")


def _sequences(name: str, inputs: Tensor, packed_info: Optional[Tensor]) -> int:
    """number of rays of a batched or packed tensor"""
    if not isinstance(inputs, Tensor):
        raise TypeError(f"{name}: inputs must be a torch.Tensor, got {type(inputs)}")
    if packed_info is None:
        if inputs.dim() != 3:
            raise ValueError(f"{name}: inputs must be (n_rays, n, channels), or (n_samples, channels) with packed_info; got {tuple(inputs.shape)}")
        n_rays = inputs.shape[0]
    else:
        if inputs.dim() != 2:
            raise ValueError(f"{name}: with packed_info inputs must be (n_samples, channels), got {tuple(inputs.shape)}")
        if packed_info.dim() != 2 or packed_info.shape[1] != 2:
            raise ValueError(f"{name}: packed_info must be 2-D with shape (n_rays, 2), got {tuple(packed_info.shape)}")
        n_rays = packed_info.shape[0]
    if inputs.shape[-1] == 0:
        raise ValueError(f"{name}: at least one channel expected")
    _check_channels(name, inputs.shape[-1])
    if max(n_rays, inputs.shape[:-1].numel()) >= 2**31:
        raise ValueError(f"{name}: more than 2^31 - 1 rays or samples")
    return n_rays


def _map_of(packed_info: Optional[Tensor], x: Tensor, n_rays: int):
    """(packed_info, the ray of every row of x, its position there), None where sequences are equal"""
    rows = x.shape[0]
    if packed_info is None:
        if n_rays > 0:
            return None, None, None
        packed_info = torch.empty((0, 2), dtype=torch.int64, device=x.device)
    info = packed_info.contiguous()
    return (info, *_C.row_map(info, rows))


def _scan_map_of(packed_info: Optional[Tensor], x: Tensor, n_rays: int):
    """_map_of and the dealing order of a scan: where whole rays are a few for each wave place of the chip, their lengths decide when the
    last one ends"""
    rows = _map_of(packed_info, x, n_rays)
    return (*rows, _C.ray_order(rows[0], x.shape[0]) if packed_info is not None and 1024 <= n_rays <= 65536 else None)


def _flat(t: Optional[Tensor]) -> Optional[Tensor]:
    return t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _overlaps(s: Tensor, t: Tensor) -> bool:
    """whether two tensors share memory, by the spans between their first and last element"""
    if s.numel() == 0 or t.numel() == 0:
        return False
    span = lambda x: (x.data_ptr(), x.data_ptr() + (1 + sum((n - 1) * k for n, k in zip(x.shape, x.stride()))) * x.element_size())  # noqa: E731
    (a, b), (c, d) = span(s), span(t)
    return a < d and c < b


def _state_buffer(name: str, state: Tensor, out_state: Optional[Tensor], **inputs) -> Tensor:
    """where a step leaves its new state: `state` itself, or a buffer that shares no memory with it; nor with what the step reads beside it, in
    whatever order its workgroups run"""
    if out_state is None:
        return torch.empty_like(state, memory_format=torch.contiguous_format)
    if not out_state.is_contiguous():
        raise ValueError(f"{name}: out_state must be contiguous")
    if (out_state.data_ptr() != state.data_ptr() or not state.is_contiguous()) and _overlaps(state, out_state):
        raise ValueError(f"{name}: out_state overlaps state; pass state itself to update it in place")
    for what, t in inputs.items():
        if t is not None and _overlaps(t, out_state):
            raise ValueError(f"{name}: out_state overlaps {what}")
    return out_state


def _written(out_state: Optional[Tensor]) -> None:
    if out_state is not None and not out_state.is_inference():
        torch.autograd.graph.increment_version(out_state)


def causal_conv(inputs: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
                packed_info: Optional[Tensor] = None, initial_state: Optional[Tensor] = None,
                return_final_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Causal convolution of `width` taps along each ray, channel by channel, differentiable in inputs, weight, bias and state.

    Args:
        inputs: (n_rays, n, channels), or (n_samples, channels) with `packed_info`; float32, bfloat16 or float16; rows may be strided.
        weight: (channels, width), width 2 to 4; `weight[:, -1]` meets the sample itself.  The dtype of inputs, like all below.
        bias: (channels,).
        activation: None or "silu".
        packed_info: (n_rays, 2) int64 (start, count), in any order; rays must not overlap.  Samples of no ray get zeros.
        initial_state: (n_rays, width - 1, channels), the inputs before each ray's first, oldest first; zeros without it.
        return_final_state: also return the last width - 1 inputs of each ray (its initial state in front where it is shorter): what
            the next samples of the same rays continue from.

        >>> x = torch.tensor([[1.], [2.], [3.]], device="cuda")
        >>> causal_conv(x, torch.tensor([[1., 10.]], device="cuda"), packed_info=torch.tensor([[0, 2], [2, 1]], device="cuda"))
        tensor([[10.], [21.], [30.]], device='cuda:0')
    """
    act = _activation_id("causal_conv", activation, (None, "silu"))
    ext = _ext()
    if ext:
        out = ext.causal_conv(inputs, weight, bias, packed_info, initial_state, act, return_final_state)
        return out if return_final_state else out[0]
    _refuse_forward("causal_conv", inputs, weight, bias, initial_state)
    n_rays = _sequences("causal_conv", inputs, packed_info)
    channels, dt = inputs.shape[-1], inputs.dtype
    width = _width("causal_conv", weight, channels)
    state = (n_rays, width - 1, channels)
    _check_native("causal_conv", inputs, (("weight", weight, (channels, width), dt), ("bias", bias, (channels,), dt),
                                          ("packed_info", packed_info, (n_rays, 2), torch.int64), ("initial_state", initial_state, state, dt)))
    x = _flat(inputs)
    if _records_grad("causal_conv", inputs, weight, bias, initial_state):
        out, final = _CausalConv.apply(x, weight, bias, initial_state, _map_of(packed_info, x, n_rays), n_rays, act, return_final_state)
    else:
        out, final = _C.causal_conv_fwd(x, weight, bias, initial_state, *_map_of(packed_info, x, n_rays), n_rays, act, return_final_state)
    out = out.view(inputs.shape)
    return (out, final) if return_final_state else out


def _width(name: str, weight: Tensor, channels: int) -> int:
    if not isinstance(weight, Tensor) or weight.dim() != 2 or weight.shape[0] != channels or not 2 <= weight.shape[1] <= 4:
        got = tuple(weight.shape) if isinstance(weight, Tensor) else type(weight)
        raise ValueError(f"{name}: weight must be (channels, width) with {channels} channels and width 2, 3 or 4, got {got}")
    return weight.shape[1]


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, init, rows, n_rays, act, want_final):
        ctx.set_materialize_grads(False)
        out, final = _C.causal_conv_fwd(x, weight, bias, init, *rows, n_rays, act, want_final)
        ctx.save_for_backward(x, weight, bias, init, *rows)
        learns = ctx.needs_input_grad[:4]
        slope = act > 0 and any(learns)
        ctx.depends = (slope or learns[1], slope or learns[0] or learns[3], slope, slope or learns[1])
        ctx.n_rays, ctx.act = n_rays, act
        return out, final

    @staticmethod
    @_differentiates_once(lambda ctx: ctx.depends)
    def backward(ctx, gy, gfinal):
        x, weight, bias, init, *rows = ctx.saved_tensors
        need = ctx.needs_input_grad
        if gy is None:
            gy = torch.zeros_like(x)
        gx, gw, gb, gi = _C.causal_conv_bwd(gy, gfinal, x, weight, bias, init, *rows, ctx.n_rays, ctx.act, need[0], need[1],
                                            bias is not None and need[2], init is not None and need[3])
        return gx, gw, gb, gi, None, None, None, None


def causal_conv_step(inputs: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor] = None, activation: Optional[str] = None,
                     out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One more sample of every ray: `inputs` (n_rays, channels) and the rays' state (n_rays, width - 1, channels) -> (outputs, new
    state).  The new state goes to `out_state` if given (`out_state=state` updates it in place; it shares no memory with the other tensors).
    Not differentiable.

        >>> causal_conv_step(torch.tensor([[3.]], device="cuda"), torch.tensor([[[2.]]], device="cuda"), torch.tensor([[1., 10.]], device="cuda"))
        (tensor([[32.]], device='cuda:0'), tensor([[[3.]]], device='cuda:0'))
    """
    act = _activation_id("causal_conv_step", activation, (None, "silu"))
    ext = _ext()
    if ext:
        return ext.causal_conv_one(inputs, state, weight, bias, act, out_state)
    _refuse_forward("causal_conv_step", inputs, state, weight, bias, out_state)
    if not isinstance(inputs, Tensor) or inputs.dim() != 2 or inputs.shape[1] == 0:
        raise ValueError("causal_conv_step: inputs must be (n_rays, channels)")
    n_rays, channels = inputs.shape
    width, dt = _width("causal_conv_step", weight, channels), inputs.dtype
    _check_channels("causal_conv_step", channels)
    shape = (n_rays, width - 1, channels)
    if not isinstance(state, Tensor):
        raise TypeError("causal_conv_step: state must be a torch.Tensor")
    _check_native("causal_conv_step", inputs, (("state", state, shape, dt), ("weight", weight, (channels, width), dt),
                                               ("bias", bias, (channels,), dt), ("out_state", out_state, shape, dt)))
    _refuse_grad("causal_conv_step", "causal_conv", inputs, state, weight, bias, out_state)
    to = _state_buffer("causal_conv_step", state, out_state, inputs=inputs, weight=weight, bias=bias)
    out = _C.causal_conv_step(inputs, state, weight, bias, act, to)
    _written(out_state)
    return out, to


def _refuse_grad(name: str, other: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} is not differentiable: call it under torch.no_grad(), or use {other} with initial_state")


def selective_scan(inputs: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor] = None,
                   gate: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None, delta_softplus: bool = False,
                   packed_info: Optional[Tensor] = None, initial_state: Optional[Tensor] = None,
                   return_final_state: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Selective state space scan along each ray, differentiable in every tensor.  Per channel, with a state of `states` numbers:

        step[t] = delta[t] + delta_bias, through softplus if delta_softplus
        h[t] = exp(step[t] * A) * h[t - 1] + step[t] * B[t] * inputs[t]
        out[t] = (C[t] . h[t] + D * inputs[t]) * silu(gate[t])            (no gate: the first factor alone)

    Args:
        inputs, delta, gate: (n_rays, n, channels), or (n_samples, channels) with `packed_info`; float32, bfloat16 or float16; rows may
            be strided (slices of one projection).
        A: (channels, states) float32, 1 to 256 states; negative values decay.
        B, C: (n_rays, n, states) or (n_samples, states), shared by the channels; the dtype of inputs.
        D, delta_bias: (channels,) float32.
        packed_info: (n_rays, 2) int64 (start, count), in any order; rays must not overlap.  Samples of no ray get zeros.
        initial_state: (n_rays, channels, states) float32, h before each ray's first sample; zeros without it.
        return_final_state: also return h after each ray's last sample (its initial state where it has none).

    States and sums are held in 32 bits; the sums of the backward pass have a fixed order (the same bits every time).  It differentiates
    once (second derivatives raise, forward mode is refused) and needs as much memory again as the states kept for it, rows / 8 of them.

        >>> one = torch.ones(3, 1, device="cuda")     # running sums per ray: no decay, unit steps
        >>> selective_scan(one, one, torch.zeros(1, 1, device="cuda"), one, one, packed_info=torch.tensor([[0, 2], [2, 1]], device="cuda"))
        tensor([[1.], [2.], [1.]], device='cuda:0')
    """
    ext = _ext()
    if ext:
        out = ext.selective_scan(inputs, delta, A, B, C, D, gate, delta_bias, bool(delta_softplus), packed_info, initial_state, return_final_state)
        return out if return_final_state else out[0]
    _refuse_forward("selective_scan", inputs, delta, A, B, C, D, gate, delta_bias, initial_state)
    n_rays = _sequences("selective_scan", inputs, packed_info)
    rows, channels = inputs.shape[:-1], inputs.shape[-1]
    _check_scan("selective_scan", inputs, rows, channels, n_rays, delta, A, B, C, D, gate, delta_bias,
                (("packed_info", packed_info, (n_rays, 2), torch.int64),
                 ("initial_state", initial_state, (n_rays, channels, A.shape[-1] if isinstance(A, Tensor) and A.dim() else 0), torch.float32)))
    flat = [_flat(t) for t in (inputs, delta, gate, B, C)]
    if _records_grad("selective_scan", inputs, delta, A, B, C, D, gate, delta_bias, initial_state):
        out, final = _SelectiveScan.apply(*flat, A, D, delta_bias, initial_state, _scan_map_of(packed_info, flat[0], n_rays), n_rays,
                                          bool(delta_softplus), return_final_state)
    else:
        out, final, _ = _C.selective_scan_fwd(*flat, A, D, delta_bias, initial_state, *_scan_map_of(packed_info, flat[0], n_rays), n_rays,
                                              bool(delta_softplus), return_final_state, False)
    out = out.view(inputs.shape)
    return (out, final) if return_final_state else out


def _check_scan(name, inputs, rows, channels, n_rays, delta, A, B, C, D, gate, delta_bias, more) -> None:
    for what, t in (("delta", delta), ("A", A), ("B", B), ("C", C)):
        if not isinstance(t, Tensor):
            raise TypeError(f"{name}: {what} must be a torch.Tensor, got {type(t)}")
    if A.dim() != 2 or not 1 <= A.shape[1] <= _MAX_STATES:
        raise ValueError(f"{name}: A must be (channels, states) with 1 to {_MAX_STATES} states, got {tuple(A.shape)}")
    states, dt, f32 = A.shape[1], inputs.dtype, torch.float32
    _check_native(name, inputs, (("delta", delta, (*rows, channels), dt), ("A", A, (channels, states), f32), ("B", B, (*rows, states), dt),
                                 ("C", C, (*rows, states), dt), ("D", D, (channels,), f32), ("gate", gate, (*rows, channels), dt),
                                 ("delta_bias", delta_bias, (channels,), f32), *more))


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, gate, B, C, A, D, bias, init, rows, n_rays, softplus, want_final):
        ctx.set_materialize_grads(False)
        out, final, kept = _C.selective_scan_fwd(u, delta, gate, B, C, A, D, bias, init, *rows, n_rays, softplus, want_final, True)
        ctx.save_for_backward(u, delta, gate, B, C, A, D, bias, init, kept, *rows)
        # outputs are linear in u, B, C, D and the initial state, each by itself
        ctx.depends = tuple(any(l and (j != i or i in (1, 2, 5, 7)) for j, l in enumerate(ctx.needs_input_grad[:9])) for i in range(9))
        ctx.n_rays, ctx.softplus = n_rays, softplus
        return out, final

    @staticmethod
    @_differentiates_once(lambda ctx: ctx.depends)
    def backward(ctx, gy, gfinal):
        u, delta, gate, B, C, A, D, bias, init, kept, *rows = ctx.saved_tensors
        if gy is None:
            gy = torch.zeros_like(u)
        grads = _C.selective_scan_bwd(gy, gfinal, u, delta, gate, B, C, A, D, bias, init, kept, *rows, ctx.n_rays, ctx.softplus)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None, None, None, None)


def selective_scan_step(inputs: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, state: Tensor, D: Optional[Tensor] = None,
                        gate: Optional[Tensor] = None, delta_bias: Optional[Tensor] = None, delta_softplus: bool = False,
                        out_state: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """One more sample of every ray: inputs, delta, gate (n_rays, channels), B, C (n_rays, states) and the rays' state (n_rays, channels,
    states) float32 -> (outputs, new state), as `selective_scan` of one row each.  The new state goes to `out_state` if given
    (`out_state=state` updates it in place; it shares no memory with the other tensors).  Not differentiable."""
    ext = _ext()
    if ext:
        return ext.selective_scan_one(inputs, delta, A, B, C, state, D, gate, delta_bias, bool(delta_softplus), out_state)
    _refuse_forward("selective_scan_step", inputs, delta, A, B, C, D, gate, delta_bias, state, out_state)
    if not isinstance(inputs, Tensor) or inputs.dim() != 2 or inputs.shape[1] == 0:
        raise ValueError("selective_scan_step: inputs must be (n_rays, channels)")
    if not isinstance(state, Tensor):
        raise TypeError("selective_scan_step: state must be a torch.Tensor")
    n_rays, channels = inputs.shape
    _check_channels("selective_scan_step", channels)
    shape = (n_rays, channels, A.shape[-1] if isinstance(A, Tensor) and A.dim() else 0)
    _check_scan("selective_scan_step", inputs, (n_rays,), channels, n_rays, delta, A, B, C, D, gate, delta_bias,
                (("state", state, shape, torch.float32), ("out_state", out_state, shape, torch.float32)))
    _refuse_grad("selective_scan_step", "selective_scan", inputs, delta, A, B, C, D, gate, delta_bias, state, out_state)
    to = _state_buffer("selective_scan_step", state, out_state, inputs=inputs, delta=delta, A=A, B=B, C=C, D=D, gate=gate, delta_bias=delta_bias)
    out = _C.selective_scan_step(inputs, delta, gate, B, C, A, D, delta_bias, state, bool(delta_softplus), to)
    _written(out_state)
    return out, to
