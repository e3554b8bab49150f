"""Activations in 8 bits (``csrc/act8.cu``): what is kept between a forward and its backward pass, in half of 16 bits' room.

``pack8`` / ``unpack8``     a tensor (or the sum of two) as whole numbers from -127 to 127 times a power of two that 32 neighbours of a row share, and back.
``swiglu8``                 ``silu(gate) * up`` that keeps gate and up so, in the same pass, and takes its gradient at what was kept.
``checkpoint8``             activation checkpointing of a layer ``(delta, residual) -> (delta, residual)``: of both only their sum is kept, in 8 bits, and the
                            layer is run again on it in the backward pass (``Qwen3ForCausalLM.gradient_checkpointing_enable(activation_bits=8)``).

A value is off by at most half a step, 1 / 127 of its block's largest magnitude; forward results are not touched. Infinities and NaN come back as NaN.
The reference's scripts train with ``gradient_checkpointing=True`` (Fine-Tuning/qwen3-8b-lora-dist.py:160-161), which keeps 16 bits.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Callable, NamedTuple, Optional, Tuple

import torch
from torch.utils._python_dispatch import TorchDispatchMode

from . import _native as nv

vp, i32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
BLOCK = 32
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MOST = 2 ** 28          # columns: a row's are counted in 32 bits
_SWIGLU_FWD = [vp, i64, vp, vp, vp, i64, i32, i32, vp]
_SWIGLU_BWD = [vp, vp, vp, vp, i64, i32, i32, vp]
_PACK = [vp, i64, vp, i64, vp, vp, i64, i32, i32, vp]
_UNPACK = [vp, vp, vp, i64, i32, i32, vp]


class Packed8(NamedTuple):
    """``q`` int8 [rows, blocks * 32] (columns behind the last are zeros) and ``e`` uint8 [rows, blocks]: a value is q * 2 ** (e - 127); q = -128 is NaN."""
    q: torch.Tensor
    e: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype

    def nbytes(self) -> int:
        return self.q.numel() + self.e.numel()


def _rows_of(what, x):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MOST or x.dtype not in _TYPES:
        raise ValueError(f"{what}: needs [..., columns] in fp32, bf16 or fp16, up to {_MOST} columns, not {x.dtype} {list(x.shape)}")
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _room(x, rows, D, parts=1):
    nb = -(-D // BLOCK)
    return x.new_empty((rows, parts * nb * BLOCK), dtype=torch.int8), x.new_empty((rows, parts * nb), dtype=torch.uint8)


def pack8(x: torch.Tensor, add: Optional[torch.Tensor] = None) -> Packed8:
    """``x`` [..., columns], or ``x + add`` rounded to their type, in 8 bits. No gradient."""
    if add is not None and (add.shape != x.shape or add.dtype != x.dtype or add.device != x.device):
        raise ValueError("pack8: add must be like x in shape, type and device")
    shape, x = tuple(x.shape), _rows_of("pack8", x)
    if add is not None:
        add = _rows_of("pack8", add)
    rows, D = x.shape
    if not nv.use_native(x):
        with torch.no_grad():
            q, e = _pack_torch(x if add is None else x + add)
        return Packed8(q, e, shape, x.dtype)
    q, e = _room(x, rows, D)
    if rows:
        fn = nv.proto("b200_pack8", _PACK)
        nv.check(nv.call_on(x.device, fn, x.data_ptr(), _stride(x), nv.ptr(add), 0 if add is None else _stride(add), q.data_ptr(), e.data_ptr(), rows, D,
                            nv.dtype_code(x.dtype)), "pack8")
        nv.count_launch()
    return Packed8(q, e, shape, x.dtype)


def unpack8(p: Packed8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that ``p`` stands for, in its own type or another."""
    dtype = dtype or p.dtype
    D = p.shape[-1]
    nb = -(-D // BLOCK)
    rows = p.q.shape[0]
    if (dtype not in _TYPES or p.q.dtype != torch.int8 or p.e.dtype != torch.uint8 or p.q.shape != (rows, nb * BLOCK) or p.e.shape != (rows, nb)
            or p.q.device != p.e.device or not p.q.is_contiguous() or not p.e.is_contiguous() or rows * D != torch.Size(p.shape).numel()):
        raise ValueError("unpack8: not what pack8 gives")
    if not nv.use_native(p.q):
        return _unpack_torch(p.q, p.e, D).to(dtype).view(p.shape)
    y = torch.empty(p.shape, dtype=dtype, device=p.q.device)
    if rows:
        fn = nv.proto("b200_unpack8", _UNPACK)
        nv.check(nv.call_on(y.device, fn, p.q.data_ptr(), p.e.data_ptr(), y.data_ptr(), rows, D, nv.dtype_code(dtype)), "unpack8")
        nv.count_launch()
    return y


def _power(e):
    """2 ** (e - 127) in fp32, exactly."""
    e = e.to(torch.int32)
    return torch.where(e > 0, e << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _pack_torch(x):
    rows, D = x.shape
    top = 127 + (9 if x.dtype == torch.float16 else 121)
    nb = -(-D // BLOCK)
    b = torch.nn.functional.pad(x.float(), (0, -D % BLOCK)).view(rows, nb, BLOCK)
    finite = b.isfinite()
    part, power = torch.frexp(torch.where(finite, b, 0.0).abs().amax(2, keepdim=True))
    e = (power + 120 + (part * 128 >= 127.5).int()).clamp(0, top)
    q = torch.where(finite, torch.round(torch.where(finite, b, 0.0) * _power(254 - e)).clamp(-127, 127), -128.0)
    return q.to(torch.int8).view(rows, nb * BLOCK), e.to(torch.uint8).view(rows, nb)


def _unpack_torch(q, e, D):
    q = q.view(*e.shape, BLOCK).float()
    y = torch.where(q == -128.0, torch.full_like(q, float("nan")), q * _power(e).unsqueeze(2))
    return y.flatten(1)[:, :D]


def _first_order_only(what):
    """In a backward pass: gradients are being recorded for a second one only where it was asked for."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no second derivative (create_graph)")


def _swiglu8(gate_up, keep):
    """(y, q, e) of gate_up [..., 2F]; q and e None without ``keep``."""
    gu = _rows_of("swiglu8", gate_up)
    rows, F = gu.shape[0], gu.shape[1] // 2
    shape = (rows, F) if gate_up.dim() == 2 else (*gate_up.shape[:-1], F)
    q = e = None
    if not nv.use_native(gu):
        g, u = gu[:, :F].float(), gu[:, F:].float()
        y = (g * torch.sigmoid(g) * u).to(gu.dtype).view(shape)
        if keep:
            (gq, ge), (uq, ue) = _pack_torch(gu[:, :F]), _pack_torch(gu[:, F:])
            q, e = torch.cat([gq, uq], 1), torch.cat([ge, ue], 1)
        return y, q, e
    y = gu.new_empty(shape)
    if keep:
        q, e = _room(gu, rows, F, 2)
    if rows:
        rc = nv.call_on(gu.device, nv.proto("b200_swiglu8_fwd", _SWIGLU_FWD), gu.data_ptr(), _stride(gu), y.data_ptr(), nv.ptr(q), nv.ptr(e), rows, F,
                        nv.dtype_code(gu.dtype))
        if rc:
            nv.check(rc, "swiglu8_fwd")
        nv.count_launch()
    return y, q, e


class _SwiGLU8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate_up):
        y, q, e = _swiglu8(gate_up, True)
        ctx.save_for_backward(q, e)
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_order_only("swiglu8")
        q, e = ctx.saved_tensors
        shape, rows = dy.shape, q.shape[0]
        F = shape[-1]
        if not nv.use_native(dy):
            n = q.shape[1] // 2
            g, u, d = _unpack_torch(q[:, :n], e[:, :n // BLOCK], F), _unpack_torch(q[:, n:], e[:, n // BLOCK:], F), dy.reshape(rows, F).float()
            s = torch.sigmoid(g)
            return torch.cat([d * u * s * (1 + g * (1 - s)), d * g * s], 1).to(dy.dtype).view(*shape[:-1], 2 * F)
        dy = dy.contiguous()
        dgu = dy.new_empty((*shape[:-1], 2 * F))
        if rows:
            rc = nv.call_on(dy.device, nv.proto("b200_swiglu8_bwd", _SWIGLU_BWD), dy.data_ptr(), q.data_ptr(), e.data_ptr(), dgu.data_ptr(), rows, F,
                            nv.dtype_code(dy.dtype))
            if rc:
                nv.check(rc, "swiglu8_bwd")
            nv.count_launch()
        return dgu


def swiglu8(gate_up: torch.Tensor) -> torch.Tensor:
    """``silu(gate) * up`` for ``gate_up`` = [..., 2F] (gate in the first F columns, any F), rounded once. Where a gradient is asked for, gate and up are kept
    in 8 bits, and it is taken there."""
    n = gate_up.shape[-1] if gate_up.dim() else 0
    if n < 2 or n % 2 or gate_up.dtype not in _TYPES:
        raise ValueError(f"swiglu8: needs [..., 2F] in fp32, bf16 or fp16, not {gate_up.dtype} {list(gate_up.shape)}")
    if gate_up.requires_grad and torch.is_grad_enabled():
        return _SwiGLU8Fn.apply(gate_up)
    return _swiglu8(gate_up, False)[0]


# ------------------------------------------------------------------------------------------------
# checkpoints
# ------------------------------------------------------------------------------------------------
class _Checkpoint8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, run, delta, residual):
        ctx.run, ctx.n_in = run, 1 + (residual is not None)
        ctx.draws, ctx.autocast = _draws(delta), _autocast(delta.device.type)
        p = pack8(delta, residual)
        with torch.no_grad(), _no_draws(delta):
            out = run(delta, residual)
        if not isinstance(out, tuple) or not all(isinstance(t, torch.Tensor) for t in out):
            raise TypeError("checkpoint8: the layer must return a tuple of tensors")
        ctx.kept = p.shape, p.dtype
        ctx.save_for_backward(p.q, p.e)
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, *grads):
        _first_order_only("checkpoint8")
        x = unpack8(Packed8(*ctx.saved_tensors, *ctx.kept)).requires_grad_(True)
        now = _draws(x)
        try:                                             # dropout masks of the layer are those of its forward
            _set_draws(ctx.draws)
            with torch.enable_grad(), torch.autocast(x.device.type, **ctx.autocast), _no_draws(x):
                out = ctx.run(x, None)
        finally:
            _set_draws(now)
        pairs = [(o, g) for o, g in zip(out, grads) if g is not None and o.requires_grad]
        if pairs:
            torch.autograd.backward([o for o, _ in pairs], [g for _, g in pairs])
        return None, None, x.grad if ctx.needs_input_grad[2] else None, x.grad if ctx.n_in == 2 and ctx.needs_input_grad[3] else None


def _autocast(device):
    return {"enabled": torch.is_autocast_enabled(device), "dtype": torch.get_autocast_dtype(device), "cache_enabled": torch.is_autocast_cache_enabled()}


def _capturing(x):
    return x.is_cuda and torch.cuda.is_current_stream_capturing()


class _NoDraws(TorchDispatchMode):
    """Torch's operators that draw random numbers on a device are errors."""

    def __init__(self, device):
        super().__init__()
        self.device = device

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if torch.Tag.nondeterministic_seeded in func.tags and self._drew(func, args, kwargs or {}):
            if any(isinstance(t, torch.Tensor) and t.device == self.device for t in (out if isinstance(out, (tuple, list)) else [out])):
                raise RuntimeError(f"checkpoint8: while a graph is captured the layer may not draw from torch's generator ({func}): what its forward drew could not "
                                   "be drawn again for the gradients; ops.elementwise.dropout can")
        return out

    @staticmethod
    def _drew(func, args, kwargs):
        """Attention and recurrent layers count as drawing, whatever their dropout."""
        for i, a in enumerate(func._schema.arguments):
            if a.name in ("dropout_p", "dropout"):
                return bool(args[i] if i < len(args) else kwargs.get(a.name, a.default_value))
        return True


def _no_draws(x):
    """Torch's generator on x's device can neither be asked nor set where a capture is under way; so nothing may draw from it there."""
    return _NoDraws(x.device) if _capturing(x) else contextlib.nullcontext()


def _draws(x):
    """Where the streams of random numbers stand: the package's own, torch's on the host and on x's device (None in a capture, ``_no_draws``)."""
    from . import elementwise as ew
    cuda = torch.cuda.get_rng_state(x.device) if x.is_cuda and not _capturing(x) else None
    return dict(ew._seed_state), torch.get_rng_state(), cuda, x.device


def _set_draws(state):
    from . import elementwise as ew
    ew._seed_state.clear()
    ew._seed_state.update(state[0])
    torch.set_rng_state(state[1])
    if state[2] is not None and not torch.cuda.is_current_stream_capturing():
        torch.cuda.set_rng_state(state[2], state[3])


def checkpoint8(layer: Callable, delta: torch.Tensor, residual: Optional[torch.Tensor], *args) -> Tuple[torch.Tensor, ...]:
    """``layer(delta, residual, *args)`` -> tuple of tensors, where the layer needs its first two arguments only as ``delta + residual`` (a branch and the stream
    it is added to; ``residual`` None: delta is the stream). Keeps that sum in 8 bits and runs the layer again on it for the gradients: results are those of a
    plain call, gradients those of the layer at what was kept. ``args`` get no gradients; parameters of the layer do, in place, as by ``backward()``. In a captured step the layer
    may draw random numbers from ``ops.elementwise.dropout`` and on the host, but not from torch's generator on the device: that is an error."""
    if not torch.is_grad_enabled():
        return layer(delta, residual, *args)
    anchor = delta.new_empty(0, dtype=torch.float32).requires_grad_(True)      # so that a frozen input layer does not end the graph here
    return _Checkpoint8Fn.apply(anchor, lambda d, r: layer(d, r, *args), delta, residual)
