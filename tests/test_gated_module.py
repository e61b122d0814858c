"""``QuantizedGatedMLP`` calls its layers as modules wherever calling them does more than their product: no device is needed, the
layers and the fused operator are replaced by the same products in torch."""
import pytest
import torch
import torch.nn.functional as F

from eoq_quantization_b200 import gated
from eoq_quantization_b200.core.quantized_linear import QuantizedLinear


def _weight(layer):
    codes = layer.unpack_4bit(layer.packed_weight, layer.out_features * layer.in_features).float()
    return (codes * layer.scales.float().repeat_interleave(layer.block_size)).view(layer.out_features, layer.in_features)


@pytest.fixture
def fused(monkeypatch):
    """The calls of the fused operator and of the product with its own gradient; layers that compute on the CPU."""
    calls = []

    def block(gate, gate_scales, up, up_scales, rows, cols, bits, group, x, gate_bias=None, up_bias=None, *, activation, saved):
        calls.append("block")
        dense = lambda p, s: (QuantizedLinear.unpack_4bit(p, rows * cols).float() * s.float().repeat_interleave(group)).view(rows, cols)  # noqa: E731
        return F.silu(F.linear(x, dense(gate, gate_scales), gate_bias)) * F.linear(x, dense(up, up_scales), up_bias)

    class Product(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, bias, layer, *held):
            calls.append("product")
            ctx.layer = layer
            return layer(x)

        @staticmethod
        def backward(ctx, dy):
            return (dy @ _weight(ctx.layer), dy.sum(0), None) + (None,) * 2
    monkeypatch.setattr(QuantizedLinear, "forward", lambda self, x: F.linear(x, _weight(self), self.bias_param))
    monkeypatch.setattr(gated, "gated_packed", block)
    monkeypatch.setattr(gated, "_InputGradProduct", Product)
    monkeypatch.setattr(gated, "call_kind", lambda *t: gated.GRADIENT if any(v is not None and v.requires_grad for v in t) else 0)
    return calls


def _mlp():
    torch.manual_seed(1)
    return gated.QuantizedGatedMLP.from_float(torch.nn.Linear(128, 64), torch.nn.Linear(128, 64), torch.nn.Linear(64, 128), block_size=64)


def _same(mlp, adapters, calls, allowed):
    """Values and gradients of the block and of its layers called one after the other."""
    x = torch.randn(5, 128, generator=torch.Generator().manual_seed(2))
    got = []
    for call in (mlp, lambda t: mlp.down(F.silu(mlp.gate(t)) * mlp.up(t))):
        leaf = x.clone().requires_grad_()
        for a in adapters:
            a.zero_grad()
        if call is mlp:
            calls.clear()
        y = call(leaf)
        if call is mlp:
            assert calls == allowed
        (y * torch.linspace(-1, 1, 128)).sum().backward()
        got.append([y.detach(), leaf.grad] + [p.grad.clone() for a in adapters for p in a.parameters()])
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)


def test_nothing_registered(fused):
    _same(_mlp(), [], fused, ["block", "product"])


@pytest.mark.parametrize("where", ["gate", "up", "down"])
@pytest.mark.parametrize("kind", ["forward", "pre", "full backward", "backward pre", "forward of all modules", "pre of all modules",
                                  "full backward of all modules", "backward pre of all modules"])
def test_hooks(where, kind, fused):
    mlp = _mlp()
    layer = getattr(mlp, where)
    adapter = torch.nn.Linear(layer.in_features, layer.out_features, bias=False)
    narrow = torch.nn.Linear(layer.in_features, layer.in_features, bias=False)
    adapters = [adapter]
    allowed = ["block"] if where == "down" else ["product"]        # the other half stays
    every = torch.nn.modules.module
    if "forward" in kind:
        hook = lambda m, args, out: out + adapter(args[0]) if m is layer else None  # noqa: E731
    elif kind.startswith("pre"):
        hook, adapters = lambda m, args: (args[0] + narrow(args[0]),) if m is layer else None, [narrow]  # noqa: E731
    elif "full" in kind:
        hook, adapters = lambda m, gi, go: tuple(None if g is None else 2 * g for g in gi) if m is layer else None, []  # noqa: E731
    else:
        hook, adapters = lambda m, go: tuple(3 * g for g in go) if m is layer else None, []  # noqa: E731
    name = {"forward": "forward_hook", "pre": "forward_pre_hook", "full backward": "full_backward_hook", "backward pre": "full_backward_pre_hook"}
    if kind.endswith("of all modules"):
        handle, allowed = getattr(every, "register_module_" + name[kind[:-len(" of all modules")]])(hook), []
    else:
        handle = getattr(layer, "register_" + name[kind])(hook)
    try:
        _same(mlp, adapters, fused, allowed)
    finally:
        handle.remove()
    _same(mlp, [], fused, ["block", "product"])


@pytest.mark.parametrize("where", ["gate", "up", "down"])
def test_other_layers(where, fused):
    """A layer that something else has taken the place of, or whose forward has been replaced."""
    class Adapted(torch.nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.layer = layer
            self.adapter = torch.nn.Linear(layer.in_features, layer.out_features, bias=False)

        def forward(self, x):
            return self.layer(x) + self.adapter(x)

    allowed = ["block"] if where == "down" else ["product"]
    mlp = _mlp()
    setattr(mlp, where, Adapted(getattr(mlp, where)))
    _same(mlp, [getattr(mlp, where).adapter], fused, allowed)
    mlp = _mlp()
    layer = getattr(mlp, where)
    adapter, plain = torch.nn.Linear(layer.in_features, layer.out_features, bias=False), layer.forward
    layer.forward = lambda x: plain(x) + adapter(x)
    _same(mlp, [adapter], fused, allowed)
