"""What the gated block refuses before anything is launched: no device is needed."""
import ctypes as C

import pytest
import torch

from eoq_quantization_b200 import _lib as L
from eoq_quantization_b200 import gated
from eoq_quantization_b200.core.quantized_linear import QuantizedLinear

NULL_PTR, UNSUPPORTED, INVALID = L.EOQ_ERR_NULL_PTR, L.EOQ_ERR_UNSUPPORTED, L.EOQ_ERR_INVALID_HEADER
P = 0x1000                                     # an address that nothing reads: every call below ends in its checks


def _gated(**kw):
    w = L.Gated(P, P, P, P, None, None, 64, 128, 4, 128, 0, L.F32)
    for k, v in kw.items():
        setattr(w, k, v)
    return w


@pytest.mark.parametrize("weight,dtype,batch,kept,code", [
    (dict(gate=None), 0, 1, None, NULL_PTR), (dict(up=None), 0, 1, None, NULL_PTR), (dict(gate_scales=None), 0, 1, None, NULL_PTR),
    (dict(up_scales=None), 0, 1, None, NULL_PTR), (dict(), 3, 1, None, UNSUPPORTED), (dict(), -1, 1, None, UNSUPPORTED),
    (dict(activation=3), 0, 1, None, UNSUPPORTED), (dict(bias_dtype=3), 0, 1, None, UNSUPPORTED), (dict(activation=-1), 0, 1, None, UNSUPPORTED), (dict(bits=1), 0, 1, None, INVALID),
    (dict(bits=9), 0, 1, None, INVALID), (dict(group=0), 0, 1, None, INVALID), (dict(cols=0), 0, 1, None, INVALID),
    (dict(), 0, 1, L.Kept(3, P, P, P, P), UNSUPPORTED), (dict(), 0, 1, L.Kept(1, None, P, None, None), NULL_PTR),
    (dict(), 0, 1, L.Kept(2, P, P, P, None), NULL_PTR), (dict(), 0, 0, None, 0), (dict(rows=0), 0, 1, None, 0)])
def test_forward(weight, dtype, batch, kept, code):
    w = _gated(**weight)
    assert L.lib().eoq_b200_gated_packed(C.byref(w), P, dtype, batch, P, P, None if kept is None else C.byref(kept), None) == code


def test_forward_without_pointers():
    w = _gated()
    f = L.lib().eoq_b200_gated_packed
    assert f(None, P, 0, 1, P, P, None, None) == f(C.byref(w), None, 0, 1, P, P, None, None) == f(C.byref(w), P, 0, 1, P, None, None, None) == NULL_PTR
    assert L.lib().eoq_b200_gated_scratch(C.byref(w), None, 2, 4) and f(C.byref(w), P, 2, 4, None, P, None, None) == NULL_PTR


@pytest.mark.parametrize("weight,dtype,batch,kept,code", [
    (dict(gate=None), 0, 1, L.Kept(1, P, P, None, None), NULL_PTR), (dict(), 0, 1, None, NULL_PTR), (dict(), 0, 1, L.Kept(2, P, P, None, P), NULL_PTR),
    (dict(), 0, 1, L.Kept(0, P, P, None, None), UNSUPPORTED), (dict(), 5, 1, L.Kept(1, P, P, None, None), UNSUPPORTED),
    (dict(activation=9), 0, 1, L.Kept(1, P, P, None, None), UNSUPPORTED), (dict(group=0), 0, 1, L.Kept(1, P, P, None, None), INVALID),
    (dict(), 0, 0, L.Kept(1, P, P, None, None), 0)])
def test_backward(weight, dtype, batch, kept, code):
    w = _gated(**weight)
    assert L.lib().eoq_b200_gated_grad(C.byref(w), None if kept is None else C.byref(kept), P, dtype, batch, P, P, None, None, None) == code


def test_the_others():
    lib = L.lib()
    grad = lib.eoq_b200_packed_input_grad
    assert grad(None, P, 64, 128, 4, 128, P, 0, 1, P, P, None) == grad(P, None, 64, 128, 4, 128, P, 0, 1, P, P, None) == NULL_PTR
    assert grad(P, P, 64, 128, 4, 128, P, 0, 1, None, P, None) == NULL_PTR and grad(P, P, 64, 128, 4, 128, P, 7, 1, P, P, None) == UNSUPPORTED
    assert grad(P, P, 64, 128, 1, 128, P, 0, 1, P, P, None) == grad(P, P, 64, 128, 4, 0, P, 0, 1, P, P, None) == INVALID
    assert grad(P, P, 64, 128, 4, 128, P, 0, 0, P, P, None) == 0
    assert lib.eoq_b200_packed_input_grad_scratch(64, 128, 4, 0, 0, 1) == 0 and lib.eoq_b200_packed_input_grad_scratch(64, 128, 4, 128, 0, 1) > 0
    assert lib.eoq_b200_store_8bit(None, 0, 1, 64, P, P, None) == lib.eoq_b200_load_8bit(P, None, 1, 64, P, 0, None) == NULL_PTR
    assert lib.eoq_b200_store_8bit(P, 3, 1, 64, P, P, None) == lib.eoq_b200_load_8bit(P, P, 1, 64, P, -1, None) == UNSUPPORTED
    assert lib.eoq_b200_store_8bit(P, 0, 0, 64, P, P, None) == lib.eoq_b200_load_8bit(P, P, 1, 0, P, 0, None) == 0


def test_python_checks():
    u8, f16 = torch.zeros(64, 64, dtype=torch.uint8), torch.ones(64, dtype=torch.float16)
    x = torch.zeros(2, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        gated.gated_packed(u8, f16, u8, f16, 64, 128, 4, 128, x)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        gated.packed_input_grad(u8, f16, 64, 128, 4, 128, x[:, :64])
    with pytest.raises(RuntimeError, match="CUDA device only"):
        gated.store_8bit(x)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        gated.Stored8(u8.to(torch.int8), f16.float(), torch.float16).dequantize()
    with pytest.raises(ValueError, match="activation"):
        gated.gated_packed(u8, f16, u8, f16, 64, 128, 4, 128, x, activation="relu6")
    with pytest.raises(ValueError, match="saved"):
        gated.gated_packed(u8, f16, u8, f16, 64, 128, 4, 128, x, saved="4bit")
    with pytest.raises(TypeError):
        gated.Stored8(u8.to(torch.int8), f16.float(), torch.int8).dequantize()


def test_module_checks():
    a, b, c = QuantizedLinear(128, 64), QuantizedLinear(128, 64, bits=8), QuantizedLinear(64, 128)
    with pytest.raises(ValueError, match="differ"):
        gated.QuantizedGatedMLP(a, b, c)
    with pytest.raises(ValueError, match="features"):
        gated.QuantizedGatedMLP(a, a, QuantizedLinear(128, 64))
    with pytest.raises(ValueError, match="activation"):
        gated.QuantizedGatedMLP(a, a, c, activation="x")
    with pytest.raises(ValueError, match="saved"):
        gated.QuantizedGatedMLP(a, a, c, saved="none")
    m = gated.QuantizedGatedMLP(a, QuantizedLinear(128, 64), c)
    assert "silu" in repr(m) and sorted(m.state_dict()) == sorted(f"{p}.{n}" for p in ("gate", "up", "down") for n in ("packed_weight", "scales", "bias_param"))
