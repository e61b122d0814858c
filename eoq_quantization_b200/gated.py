"""The gated feed-forward block of a model whose linear layers are ``QuantizedLinear``: h = act(gate(x)) * up(x) straight from
the packed codes of both projections, with gradients for the activations and the biases (the weights are codes, and stay as they
are), the gradient that any packed weight passes on, and activations kept in 8 bits between the two passes.

torch is used for device memory, streams and the autograd graph; every computation is a call into ``libeoq_b200.so``.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules import module as _modules

from . import _lib
from .core.quantized_linear import QuantizedLinear
from .fused import _DTYPES, GRADIENT, PLAIN, WATCHED, autocast_dtype, call_kind, dequant_packed, require_cuda

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}
KEEP = {"none": 0, "full": 1, "8bit": 2}
STORE_BLOCK = 64                        # values of a row that share a scale in 8-bit storage
# torch's own operations, for calls that something watches: the activations, and their gradients (of what follows, at g)
_TORCH_BACKWARD = {0: torch.ops.aten.silu_backward, 1: torch.ops.aten.gelu_backward, 2: lambda d, g: torch.ops.aten.gelu_backward(d, g, approximate="tanh")}
_TORCH_ACTIVATIONS = {"silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda g: F.gelu(g, approximate="tanh")}


def _check_weight(packed: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, bits: int, group: int, x: torch.Tensor, what: str) -> None:
    require_cuda(packed, what)
    if not (rows > 0 and cols > 0 and group > 0 and 2 <= bits <= 8):
        raise ValueError(f"{what}: no packed weight has {rows} x {cols} codes of {bits} bits in groups of {group}")
    row_bytes = (cols + 1) // 2 if bits == 4 else (cols + 3) // 4 if bits == 2 else cols
    if packed.dtype != (torch.uint8 if bits in (2, 4) else torch.int8) or packed.numel() != rows * row_bytes:
        raise ValueError(f"{what}: expected {rows} rows of {row_bytes} {'uint8' if bits in (2, 4) else 'int8'}, got {tuple(packed.shape)} of {packed.dtype}")
    if scales.numel() < -(-rows * cols // group):
        raise ValueError(f"{what}: expected {-(-rows * cols // group)} scales, got {scales.numel()}")
    for t in (packed, scales):
        if t.device != x.device:
            raise RuntimeError(f"{what}: the activations are on {x.device} but the weight lives on {t.device}")
    if scales.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: no gradients for scales; detach them")


def _check_activations(x: torch.Tensor, cols: int, what: str) -> None:
    require_cuda(x, what)
    if x.dim() < 1 or x.shape[-1] != cols:
        raise ValueError(f"{what}: expected last dimension {cols}, got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: unsupported activation dtype {x.dtype}")


class _Unsupported(RuntimeError):
    pass


def _without_autocast():
    """A backward pass's types are its tensors'.  (Entering torch's context takes ten microseconds, so only where autocast is on.)"""
    return torch.autocast("cuda", enabled=False) if torch.is_autocast_enabled("cuda") else nullcontext()


class _Once(torch.autograd.Function):
    """A zero to be added to a gradient that depends on what it was taken at and that nobody can differentiate again: an error on the
    way to whatever `tie` is made of, instead of a gradient that is a constant."""

    @staticmethod
    def forward(ctx, tie, dtype):
        return tie.new_zeros((), dtype=dtype)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("gated_packed: differentiable once; there are no second derivatives")


class _Gated(torch.autograd.Function):
    """h, and from what the forward pass kept of gate and up the gradients of x and the biases.  Beside h an empty result, which
    ties the gradients to x and the biases without holding them."""

    @staticmethod
    def forward(ctx, x, gate_bias, up_bias, gate, gate_scales, up, up_scales, shape, activation, form):
        out = _lib.native().gated_packed(gate, gate_scales, up, up_scales, *shape, x, gate_bias, up_bias, activation, form)
        if out is None:
            raise _Unsupported("gated_packed: the call is not supported")
        ctx.shape, ctx.activation, ctx.form, ctx.x_shape = shape, activation, form, x.shape
        ctx.bias_dtypes = [None if b is None else b.dtype for b in (gate_bias, up_bias)]
        ctx.bias_shapes = [None if b is None else b.shape for b in (gate_bias, up_bias)]
        tie = torch.empty(0)
        ctx.save_for_backward(gate, gate_scales, up, up_scales, tie, *out[1:])
        ctx.set_materialize_grads(False)
        return out[0], tie

    @staticmethod
    def backward(ctx, dh, _):
        if dh is None:
            return (None,) * 10
        saved = ctx.saved_tensors                # an error if the weights have been written since
        if not torch.is_grad_enabled():
            return (*_Gated._gradients(ctx, dh, saved), *(None,) * 7)
        with torch.no_grad():                    # create_graph
            gradients = _Gated._gradients(ctx, dh, saved)
        return (*(None if v is None else v + _Once.apply(saved[4], v.dtype) for v in gradients), *(None,) * 7)

    @staticmethod
    def _gradients(ctx, dh, saved):
        gate, gate_scales, up, up_scales, _, *kept = saved
        if call_kind(dh) == WATCHED:             # several gradients at once (is_grads_batched)
            with _without_autocast():
                return _Gated._watched_gradients(ctx, dh, gate, gate_scales, up, up_scales, kept)
        if ctx.form == KEEP["full"]:
            kept += [None, None]
        types = {t for t in ctx.bias_dtypes if t is not None}          # of one type: written in it; else cast below
        bias_type = _DTYPES.get(next(iter(types)), _lib.F32) if len(types) == 1 else _lib.F32
        with _without_autocast():
            out = _lib.native().gated_grad(gate, gate_scales, up, up_scales, *ctx.shape, ctx.activation, dh, *kept, *ctx.needs_input_grad[:3], bias_type)
        if out is None:
            raise RuntimeError("gated_packed: the backward pass is not supported")
        dx, *db = out
        if dx is not None and dx.shape != ctx.x_shape:
            dx = dx.view(ctx.x_shape)
        for i, b in enumerate(db):
            if b is not None and (b.dtype != ctx.bias_dtypes[i] or b.shape != ctx.bias_shapes[i]):
                db[i] = b.to(ctx.bias_dtypes[i]).view(ctx.bias_shapes[i])
        return dx, *db

    @staticmethod
    def _watched_gradients(ctx, dh, gate, gate_scales, up, up_scales, kept):
        g, u = (v.float() for v in kept[:2])
        if ctx.form == KEEP["8bit"]:
            g, u = (v * s.repeat_interleave(STORE_BLOCK, 1)[:, :v.shape[1]] for v, s in ((g, kept[2]), (u, kept[3])))
        d = dh.reshape(g.shape).float()
        value = list(_TORCH_ACTIVATIONS.values())[ctx.activation](g)
        dg, du = _TORCH_BACKWARD[ctx.activation](d * u, g), d * value
        dx = None
        if ctx.needs_input_grad[0]:
            dx = (dg @ dequant_packed(gate, gate_scales, *ctx.shape) + du @ dequant_packed(up, up_scales, *ctx.shape)).to(dh.dtype).reshape(ctx.x_shape)
        return dx, *(v.sum(0).to(t).reshape(s) if wanted else None for v, t, s, wanted in zip((dg, du), ctx.bias_dtypes, ctx.bias_shapes, ctx.needs_input_grad[1:3]))


class _InputGradProduct(torch.autograd.Function):
    """A product with a packed weight: forward as the layer computes it, backward straight from the codes."""

    @staticmethod
    def forward(ctx, x, bias, layer, packed, scales):
        ctx.shape = (layer.out_features, layer.in_features, layer.bits, layer.block_size)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(packed, scales)
        return layer(x)

    @staticmethod
    def backward(ctx, dy):
        packed, scales = ctx.saved_tensors
        with _without_autocast():
            dx = None
            if ctx.needs_input_grad[0]:          # of several gradients at once, or to be differentiated again: torch's own product
                dx = packed_input_grad(packed, scales, *ctx.shape, dy) if call_kind(dy) == PLAIN else dy @ dequant_packed(packed, scales, *ctx.shape).to(dy.dtype)
            db = dy.reshape(-1, dy.shape[-1]).sum(0).to(ctx.bias_dtype) if ctx.needs_input_grad[1] else None
        return dx, db, None, None, None


def gated_packed(gate: torch.Tensor, gate_scales: torch.Tensor, up: torch.Tensor, up_scales: torch.Tensor, rows: int, cols: int,
                 bits: int, group: int, x: torch.Tensor, gate_bias: Optional[torch.Tensor] = None,
                 up_bias: Optional[torch.Tensor] = None, *, activation: str = "silu", saved: str = "full") -> torch.Tensor:
    """h = act(x @ Wg.T + gate_bias) * (x @ Wu.T + up_bias) in x.dtype, for x of shape (..., cols) and any number of rows of it.

    Both weights are ``QuantizedLinear`` buffers of one shape: (rows, cols) codes of `bits` bits and fp16 scales, one for `group`
    codes of the flattened matrix.  `activation`: "silu", "gelu" (exact) or "gelu_tanh".  Differentiable once with respect to x
    and the biases; `saved` says what is kept for that, both projections' results in x.dtype ("full") or in 8 bits ("8bit": as
    ``store_8bit`` keeps them, 8.5 bits a value); without gradients nothing is.  Scales that want gradients are refused.  Sums in fp32."""
    code = ACTIVATIONS.get(activation)
    if code is not None and saved in ("full", "8bit"):
        h = _lib.native().gated_packed(gate, gate_scales, up, up_scales, rows, cols, bits, group, x, gate_bias, up_bias, code, 0)
        if h is not None:
            return h
        # training: the checks below are for what this does not take
        if call_kind(x, gate_bias, up_bias) == GRADIENT and not torch.is_autocast_enabled("cuda") and not gate_scales.requires_grad and not up_scales.requires_grad:
            try:
                return _Gated.apply(x, gate_bias, up_bias, gate, gate_scales, up, up_scales, (rows, cols, bits, group), code, KEEP[saved])[0]
            except _Unsupported:
                pass
    what = "gated_packed"
    if code is None:
        raise ValueError(f"{what}: unknown activation {activation!r}; one of {', '.join(ACTIVATIONS)}")
    if saved not in ("full", "8bit"):
        raise ValueError(f"{what}: saved is 'full' or '8bit', not {saved!r}")
    _check_activations(x, cols, what)
    _check_weight(gate, gate_scales, rows, cols, bits, group, x, what)
    _check_weight(up, up_scales, rows, cols, bits, group, x, what)
    for b in (gate_bias, up_bias):
        if b is not None and (b.numel() != rows or b.device != x.device or not b.is_floating_point()):
            raise ValueError(f"{what}: a bias is {rows} floating-point values beside the activations")
    dt = autocast_dtype(x)
    if dt is not None:
        with torch.autocast("cuda", enabled=False):
            return gated_packed(gate, gate_scales, up, up_scales, rows, cols, bits, group, x.to(dt), gate_bias, up_bias, activation=activation, saved=saved)
    kind = call_kind(x, gate_bias, up_bias)
    if kind == WATCHED:                      # transforms, tangents, modes: torch's own operations on dequantised copies
        g, u = (F.linear(x, dequant_packed(w, s, rows, cols, bits, group).to(x.dtype), None if b is None else b.to(x.dtype).reshape(rows))
                for w, s, b in ((gate, gate_scales, gate_bias), (up, up_scales, up_bias)))
        return _TORCH_ACTIVATIONS[activation](g) * u
    if x.numel() == 0:                       # no rows: nothing to launch, the graph as it would be
        h = x.new_zeros(*x.shape[:-1], rows) + x.sum() * 0
        return h if kind != GRADIENT else h + sum((b.sum() * 0).to(h.dtype) for b in (gate_bias, up_bias) if b is not None)
    if kind == GRADIENT:
        return _Gated.apply(x, gate_bias, up_bias, gate, gate_scales, up, up_scales, (rows, cols, bits, group), code, KEEP[saved])[0]
    h = _lib.native().gated_packed(gate, gate_scales, up, up_scales, rows, cols, bits, group, x, gate_bias, up_bias, code, 0)
    if h is None:
        raise RuntimeError(f"{what}: the call is not supported")
    return h


def packed_input_grad(packed: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, bits: int, group: int, grad: torch.Tensor) -> torch.Tensor:
    """grad @ W in grad.dtype, for grad of shape (..., rows): the gradient with respect to its activations that a packed
    ``QuantizedLinear`` weight (rows, cols) passes on, straight from the codes, sums in fp32.  Not differentiable itself."""
    what = "packed_input_grad"
    with torch.no_grad():
        dx = _lib.native().input_grad(packed, scales, rows, cols, bits, group, grad)
        if dx is not None:
            return dx
        _check_activations(grad, rows, what)
        _check_weight(packed, scales, rows, cols, bits, group, grad, what)
        if grad.numel() == 0:
            return grad.new_zeros(*grad.shape[:-1], cols)
        with torch.autocast("cuda", enabled=False):
            dx = _lib.native().input_grad(packed, scales, rows, cols, bits, group, grad)
    if dx is None:
        raise RuntimeError(f"{what}: the call is not supported")
    return dx


class Stored8:
    """Activations in 8 bits: signed codes (..., n) and one fp32 scale for 64 of a row, (..., ceil(n / 64))."""

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype):
        self.codes, self.scales, self.dtype = codes, scales, dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def dequantize(self, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """The values that the codes stand for, in the type they were stored from or in `dtype`."""
        dtype = dtype or self.dtype
        if dtype not in _DTYPES:
            raise TypeError(f"Stored8.dequantize: unsupported dtype {dtype}")
        y = _lib.native().load_8bit(self.codes, self.scales, _DTYPES[dtype])
        if y is not None:
            return y
        require_cuda(self.codes, "Stored8.dequantize")
        blocks = -(-self.codes.shape[-1] // STORE_BLOCK)
        if self.codes.dtype != torch.int8 or self.scales.dtype != torch.float32 or self.scales.shape != (*self.codes.shape[:-1], blocks) or \
                self.scales.device != self.codes.device:
            raise ValueError("Stored8.dequantize: int8 codes (..., n) and fp32 scales (..., ceil(n / 64)) on one device")
        if self.codes.numel() == 0:
            return self.codes.new_empty(self.codes.shape, dtype=dtype)
        y = _lib.native().load_8bit(self.codes.contiguous(), self.scales.contiguous(), _DTYPES[dtype])
        if y is None:
            raise RuntimeError("Stored8.dequantize: the call is not supported")
        return y


def store_8bit(x: torch.Tensor) -> Stored8:
    """The rows of x (last dimension) in 8 bits: blocks of 64 values, code = round(127 x / largest magnitude of the block).  Off by
    at most 1/254 of the block's largest magnitude.  A block with a NaN or an infinity comes back as NaN, one that is below 1e-30
    throughout as zeros.  Outside the autograd graph."""
    with torch.no_grad():
        out = _lib.native().store_8bit(x)
        if out is None:
            require_cuda(x, "store_8bit")
            if x.dtype not in _DTYPES:
                raise TypeError(f"store_8bit: unsupported activation dtype {x.dtype}")
            if x.dim() < 1:
                raise ValueError("store_8bit: a tensor of rows is wanted, not a single value")
            if x.numel() == 0:
                return Stored8(x.new_empty(x.shape, dtype=torch.int8), x.new_empty(*x.shape[:-1], -(-x.shape[-1] // STORE_BLOCK), dtype=torch.float32), x.dtype)
            with torch.autocast("cuda", enabled=False):
                out = _lib.native().store_8bit(x.detach())
            if out is None:
                raise RuntimeError("store_8bit: the call is not supported")
    return Stored8(*out, x.dtype)


def _only_products(*layers: nn.Module) -> bool:
    """Whether calling the layers comes to their products with packed weights: nothing hooked on, put in their place or in their
    ``forward``'s."""
    if _modules._global_forward_hooks or _modules._global_forward_pre_hooks or _modules._global_backward_hooks or _modules._global_backward_pre_hooks:
        return False
    return all(type(m) is QuantizedLinear and not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks) and
               "forward" not in m.__dict__ for m in layers)


class QuantizedGatedMLP(nn.Module):
    """down(act(gate(x)) * up(x)) of three ``QuantizedLinear`` layers, gate and up in one kernel.

    With gradients, gate's and up's results are kept as `saved` says ("full" or "8bit"), and the gradients go back through the
    codes: no projection is dequantised.  Layers with hooks, or that something else has taken the place of, are called as they are, and so
    are all of them for types that the kernels do not take (fp64)."""

    def __init__(self, gate: QuantizedLinear, up: QuantizedLinear, down: QuantizedLinear, activation: str = "silu", saved: str = "full"):
        super().__init__()
        same = ("in_features", "out_features", "bits", "block_size")
        if any(getattr(gate, n) != getattr(up, n) for n in same):
            raise ValueError("QuantizedGatedMLP: gate and up differ in shape, bits or block size")
        if down.in_features != gate.out_features:
            raise ValueError(f"QuantizedGatedMLP: down takes {down.in_features} features, gate and up give {gate.out_features}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"QuantizedGatedMLP: unknown activation {activation!r}; one of {', '.join(ACTIVATIONS)}")
        if saved not in ("full", "8bit"):
            raise ValueError(f"QuantizedGatedMLP: saved is 'full' or '8bit', not {saved!r}")
        self.gate, self.up, self.down = gate, up, down
        self.activation, self.saved = activation, saved

    @classmethod
    def from_float(cls, gate: nn.Linear, up: nn.Linear, down: nn.Linear, bits: int = 4, block_size: int = 128, activation: str = "silu",
                   saved: str = "full") -> "QuantizedGatedMLP":
        """The three layers quantised as ``QuantizedLinear.from_float`` does."""
        return cls(*(QuantizedLinear.from_float(m, bits=bits, block_size=block_size) for m in (gate, up, down)), activation=activation, saved=saved)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        g, u, d = self.gate, self.up, self.down
        if _only_products(g, u) and x.dtype in _DTYPES:
            h = gated_packed(g.packed_weight, g.scales, u.packed_weight, u.scales, g.out_features, g.in_features, g.bits, g.block_size, x, g.bias_param,
                             u.bias_param, activation=self.activation, saved=self.saved)
        else:
            h = _TORCH_ACTIVATIONS[self.activation](g(x)) * u(x)
        if _only_products(d) and autocast_dtype(h) is None and h.dtype in _DTYPES and h.numel() and call_kind(h, d.bias_param) == GRADIENT:
            return _InputGradProduct.apply(h, d.bias_param, d, d.packed_weight, d.scales)
        return d(h)

    def extra_repr(self) -> str:
        return f"activation={self.activation!r}, saved={self.saved!r}"
