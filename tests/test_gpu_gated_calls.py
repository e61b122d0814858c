"""Calls of the gated block and of the packed gradient out of the ordinary."""
import pytest
import torch

from eoq_quantization_b200 import gated
from gated_reference import Gated, inside, weight

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _layers(n, k, bits, group, seed):
    return weight(n, k, bits, group, seed), weight(n, k, bits, group, seed + 100)


def _inputs(m, k, dtype, seed, spread=1.0):
    return (torch.randn(m, k, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype).cuda()


@pytest.mark.parametrize("m", [1, 12, 40])
@pytest.mark.parametrize("bits", [2, 4, 8])
def test_strided_codes(m, bits):
    """Copied in front of kernels that read codes early: these are launched behind the copy, and in a recording, too."""
    n, k = 2816, 4096
    (pg, sg, _), (pu, su, _) = _layers(n, k, bits, 128, 1)
    wide = lambda t: torch.stack([t, t + 1], 1)[:, 0]  # noqa: E731
    x, dh = _inputs(m, k, BF16, 2), _inputs(m, n, BF16, 3)
    want = gated.gated_packed(pg, sg, pu, su, n, k, bits, 128, x), gated.packed_input_grad(pg, sg, n, k, bits, 128, dh)
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(gated.gated_packed(pg, sg, pu, su, n, k, bits, 128, leaf), leaf, dh)
    sg_, su_ = torch.stack([sg, sg], 1)[:, 0], torch.stack([su, su], 1)[:, 0]
    pg_, pu_ = wide(pg), wide(pu)
    assert not pg_.is_contiguous() and not sg_.is_contiguous()

    def calls():
        h = gated.gated_packed(pg_, sg_, pu_, su_, n, k, bits, 128, leaf)
        return (gated.gated_packed(pg_, sg_, pu, su, n, k, bits, 128, x), gated.packed_input_grad(pg_, sg_, n, k, bits, 128, dh), h.detach(),
                torch.autograd.grad(h, leaf, dh)[0])
    for got in (calls(), calls()):
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, want[0], dx)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, (*want, want[0], dx)))


@pytest.mark.parametrize("where", ["gate", "up", "down"])
@pytest.mark.parametrize("m,dtype", [(3, F32), (40, F16)])
def test_adapters_hooked_on(where, m, dtype):
    """An adapter's output added by a hook counts, in the value, in its own gradient and in that of the activations."""
    torch.manual_seed(1)
    mlp = gated.QuantizedGatedMLP.from_float(*(torch.nn.Linear(*s).cuda() for s in ((256, 320), (256, 320), (320, 256))), block_size=64)
    layer = getattr(mlp, where)
    adapter = torch.nn.Linear(layer.in_features, layer.out_features, bias=False).cuda().to(dtype)
    handle = layer.register_forward_hook(lambda module, args, out: out + adapter(args[0]))
    x, dy = _inputs(m, 256, dtype, 2), _inputs(m, 256, dtype, 3)
    got = []
    for call in (mlp, lambda t: mlp.down(torch.nn.functional.silu(mlp.gate(t)) * mlp.up(t))):
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        got.append([y.detach(), *torch.autograd.grad(y, (leaf, adapter.weight), dy)])
    handle.remove()
    # the fused half rounds h once where the layers round gate, up, their product and h: half steps, weighed by what follows
    tol = 12 * torch.finfo(dtype).eps / 2 + 2.0 ** -10 * (dtype != F32) + 2.0 ** -16
    for a, b in zip(*got):
        assert (a - b).double().norm() <= tol * b.double().norm()
    leaf = x.clone().requires_grad_()
    y = mlp(leaf)
    assert (y.detach() - got[0][0]).double().norm() > 0.05 * y.double().norm()


def test_module_takes_what_its_layers_take():
    torch.manual_seed(1)
    mlp = gated.QuantizedGatedMLP.from_float(*(torch.nn.Linear(*s).cuda() for s in ((256, 320), (256, 320), (320, 256))), block_size=64, activation="gelu")
    x = _inputs(5, 256, F32, 2).double()
    got = []
    for call in (mlp, lambda t: mlp.down(torch.nn.functional.gelu(mlp.gate(t)) * mlp.up(t))):
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        got.append((call(x), y.detach(), *torch.autograd.grad(y, leaf, x)))
    for a, b in zip(*got):
        assert a.dtype == torch.float64 and torch.equal(a, b)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("wants", [False, True])
def test_scales_that_want_gradients(which, wants):
    """Refused, whether or not the activations want some too; without gradients the call is what it is for any scales."""
    n, k = 64, 128
    (pg, sg, _), (pu, su, _) = _layers(n, k, 4, 128, 1)
    x = _inputs(3, k, F16, 2)
    want = gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x)
    (sg, su)[which].requires_grad_()
    with pytest.raises(ValueError, match="no gradients for scales"):
        gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x.clone().requires_grad_(wants))
    with torch.no_grad():
        assert torch.equal(gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x), want)
        dx = gated.packed_input_grad(pg, sg, n, k, 4, 128, want)
    assert torch.equal(gated.packed_input_grad(pg, sg.detach(), n, k, 4, 128, want), dx)


@pytest.mark.parametrize("n", [61, 64, 8200, 16384])
@pytest.mark.parametrize("form", ["full", "8bit"])
def test_gradients_through_closed_gates(n, form):
    """A row's gradients that meet closed gates alone, from what the forward pass has kept: eleven bits of each, whatever the width.
    The slopes and values of silu down to -30 are some 2^-17 off in fp32 (the exponential 37 units, the division 2)."""
    from eoq_quantization_b200 import _lib
    k = 128
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 1)
    gates = torch.tensor([-2.0, -10.0, -15.0, -20.0, -25.0, -30.0], device="cuda")
    m = len(gates)
    u = _inputs(m, n, BF16, 2)
    dh = torch.zeros(m, n, dtype=BF16, device="cuda")
    at = torch.arange(m, device="cuda")
    dh[at, 9 * at] = torch.tensor([1.0, -3.0, 2e-3, 5.0, 100.0, 7.0], dtype=BF16, device="cuda")
    if form == "full":
        kept = (gates[:, None].to(BF16).expand(m, n).contiguous(), u, None, None)
        g, u = kept[0].double(), u.double()
    else:
        s = gated.store_8bit(u)
        scale = (gates.abs() / 127)[:, None].expand(m, -(-n // 64)).contiguous()
        kept = (torch.full((m, n), -127, dtype=torch.int8, device="cuda"), s.codes, scale, s.scales)
        g, u = (-127 * scale[:, :1]).double().expand(m, n), s.dequantize(F32).double()
    dx, dbg, dbu = _lib.native().gated_grad(pg, sg, pu, su, n, k, 4, 128, gated.ACTIVATIONS["silu"], dh, *kept, True, True, True, _lib.F32)
    d, sig = dh.double(), torch.sigmoid(g)
    dg, du = d * u * sig * (1 + g * (1 - sig)), d * g * sig
    most = torch.maximum(dg.abs(), du.abs()).amax(1, keepdim=True) * 2.0 ** -38
    eg, eu = ((2.0 ** -16 + 2.0 ** -11) * v.abs() + (d != 0) * most for v in (dg, du))
    # (a bias's gradient has one term, or one beside zeros)
    for got, v, e in ((dbg, dg, eg), (dbu, du, eu)):
        assert ((got.double() - v.sum(0)).abs() <= e.sum(0) + 2.0 ** -23 * v.abs().sum(0)).all()
    off = eg @ wg.abs() + eu @ wu.abs() + 2.0 ** -10.9 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    want = dg @ wg + du @ wu
    assert ((dx.double() - want).abs() <= off + 2.0 ** -8 * (want.abs() + off)).all()


@pytest.mark.parametrize("kind", list(gated.ACTIVATIONS))
@pytest.mark.parametrize("m,n,dtype", [(4, 64, BF16), (40, 61, BF16), (3, 64, F32)])
def test_gradients_of_huge_activations(kind, m, n, dtype):
    """Gates whose squares are beyond fp32."""
    k = 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 1)
    x, dh = _inputs(m, k, dtype, 2, 1e21).requires_grad_(), _inputs(m, n, dtype, 3, 1e-30)
    dx, = torch.autograd.grad(gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x, activation=kind), x, dh)
    (want, off), *_ = Gated(x.detach(), wg, wu, kind).gradients(dh, "full")
    assert (Gated(x.detach(), wg, wu, kind).g.abs() > 1e20).any()
    inside(dx, want, off, "dx")


def _module(saved="full"):
    torch.manual_seed(1)
    return gated.QuantizedGatedMLP.from_float(*(torch.nn.Linear(*s).cuda() for s in ((256, 320), (256, 320), (320, 256))), block_size=64, saved=saved)


def _dense(layer):
    return layer._dequantize_weight().double()


def _exact_module(mlp, x):
    """The module in 64 bits, in torch's own operations."""
    f = lambda layer, t: t @ _dense(layer).T + layer.bias_param.double()  # noqa: E731
    return f(mlp.down, torch.nn.functional.silu(f(mlp.gate, x)) * f(mlp.up, x))


@pytest.mark.parametrize("m", [1, 40])
@pytest.mark.parametrize("which", ["layer", "block"])
def test_function_transforms_and_recordings(m, which):
    """torch.func's derivatives and torch.jit.trace of the block and of a layer alone, fp32: ten roundings and sums of 320 terms at most."""
    mlp = _module()
    f, exact = (mlp, lambda t: _exact_module(mlp, t)) if which == "block" else \
        (mlp.gate, lambda t: t @ _dense(mlp.gate).T + mlp.gate.bias_param.double())
    x, v = _inputs(m, 256, F32, 2), _inputs(m, 256, F32, 3)
    near = lambda a, b: (a.double() - b).norm() <= (10 * 2.0 ** -24 + 320 * 2.0 ** -23) * b.norm()  # noqa: E731
    leaf = x.double().requires_grad_()
    want, = torch.autograd.grad(exact(leaf).square().sum(), leaf)
    assert near(torch.func.grad(lambda t: f(t).square().sum())(x), want)
    _, tangent = torch.func.jvp(f, (x,), (v,))
    assert near(tangent, torch.func.jvp(exact, (x.double(),), (v.double(),))[1])
    assert near(torch.func.jacrev(f)(x[:1]), torch.func.jacrev(exact)(x[:1].double()))
    assert near(torch.func.vmap(torch.func.grad(lambda t: f(t).square().sum()))(x), want)
    traced = torch.jit.trace(f, (x,))
    for _ in range(3):
        torch.full((320, 256), float("nan"), device="cuda")         # what memory may hold that nobody has written
        assert near(traced(v), exact(v.double()))


@pytest.mark.parametrize("kind", list(gated.ACTIVATIONS))
@pytest.mark.parametrize("saved", ["full", "8bit"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_several_gradients_at_once(kind, saved, dtype):
    """``is_grads_batched`` and what uses it: each gradient as by itself."""
    n, k, m = 130, 256, 6
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 1)
    leaves = [_inputs(m, k, dtype, 2).view(2, 3, k), _inputs(1, n, F32, 3)[0], _inputs(1, n, dtype, 4)[0]]
    want = Gated(leaves[0].view(m, k), wg, wu, kind, *leaves[1:])
    leaves = [t.requires_grad_() for t in leaves]
    h = gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, *leaves, activation=kind, saved=saved)
    dhs = torch.stack([_inputs(m, n, dtype, 5 + i).view(2, 3, n) for i in range(3)])
    got = torch.autograd.grad(h, leaves, dhs, is_grads_batched=True)
    for i, dh in enumerate(dhs):
        (v, e), *db = want.gradients(dh.view(m, n), saved)
        inside(got[0][i].reshape(m, k), v, e, f"dx {i}")
        for t, (v, e) in zip(got[1:], db):
            inside(t[i], v, e + torch.finfo(t.dtype).eps / 2 * (v.abs() + e), f"bias {i}")


def test_jacobian_of_the_module():
    mlp, x = _module(), _inputs(2, 256, F32, 2)
    whole = torch.autograd.functional.jacobian(mlp, x, vectorize=True)
    rows = torch.autograd.functional.jacobian(mlp, x)
    assert (whole - rows).norm() <= 2.0 ** -16 * rows.norm()


@pytest.mark.parametrize("bits", [3, 5, 6, 7])
@pytest.mark.parametrize("m,n,k,group,dtype", [(1, 200, 256, 32, F16), (7, 96, 384, 96, BF16), (20, 130, 512, 128, F16), (33, 65, 320, 64, BF16),
                                               (280, 200, 256, 32, F16), (5, 70, 256, 64, F32)])
def test_other_widths(bits, m, n, k, group, dtype):
    """One code a byte, at the tensor cores."""
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, bits, group, 1)
    x, dh = _inputs(m, k, dtype, 2).requires_grad_(), _inputs(m, n, dtype, 3, 1e-3)
    want = Gated(x.detach(), wg, wu, "gelu")
    h = gated.gated_packed(pg, sg, pu, su, n, k, bits, group, x, activation="gelu", saved="8bit")
    inside(h.detach(), want.h, want.h_bound(), "h")
    inside(gated.gated_packed(pg, sg, pu, su, n, k, bits, group, x.detach(), activation="gelu"), want.h, want.h_bound(), "h")
    (v, e), *_ = want.gradients(dh, "8bit")
    inside(torch.autograd.grad(h, x, dh)[0], v, e, "dx")
    d, half = dh.double(), torch.finfo(dtype).eps / 2
    off = ((0 if dtype == F32 else 2.0 ** -11) + n * 2.0 ** -23 + 2.0 ** -37) * (d.abs() @ wg.abs())
    inside(gated.packed_input_grad(pg, sg, n, k, bits, group, dh), d @ wg, off + half * ((d @ wg).abs() + off) + 2.0 ** -25, "dy W")


@pytest.mark.parametrize("what", ["block", "module"])
def test_second_derivatives_are_errors(what):
    """Also where the gradient of the result is a constant: the block's own depends on its activations."""
    n, k = 320, 256
    (pg, sg, _), (pu, su, _) = _layers(n, k, 4, 128, 1)
    call = _module() if what == "module" else lambda t: gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, t)
    x = _inputs(12, k, F32, 2).requires_grad_()
    plain, = torch.autograd.grad(call(x).sum(), x)
    for loss in (lambda y: y.sum(), lambda y: y.square().sum()):
        dx, = torch.autograd.grad(loss(call(x)), x, create_graph=True)
        assert dx.requires_grad
        with pytest.raises(RuntimeError):
            (dx.square().sum() + x.sum()).backward()
    with pytest.raises(RuntimeError, match="differentiable once"):          # (which takes what is not reached for zeros)
        torch.autograd.functional.hvp(lambda t: call(2 * t).sum(), x.detach(), x.detach())
    whole = torch.autograd.functional.jacobian(call, x[:2].detach(), create_graph=True, vectorize=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        whole.sum().backward()
    dx, = torch.autograd.grad(call(x).sum(), x, create_graph=True)
    assert torch.equal(dx.detach(), plain) and not plain.requires_grad
    x.grad = None
    call(x).sum().backward()
    assert torch.equal(x.grad, plain) and not x.grad.requires_grad


def _loud(n, k, bits, group, seed):
    """A weight a hundredth of whose groups are beyond fp16 (some of their codes)."""
    packed, scales, dense = weight(n, k, bits, group, seed)
    codes = torch.round(dense.view(-1, group) / scales.double()[:, None])
    qmax = (1 << (bits - 1)) - 1
    loud = torch.rand(len(scales), generator=torch.Generator().manual_seed(seed + 7)) < 0.01
    assert loud.any()
    scales = torch.where(loud.cuda(), torch.tensor(3 * 65504.0 / qmax if bits > 2 else 60000.0).to(F16).cuda(), scales)
    return packed, scales, (codes * scales.double()[:, None]).view(n, k)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("m,n,k,group", [(3, 130, 512, 128), (20, 130, 512, 64), (40, 130, 4096, 128), (300, 257, 320, 32), (150, 11000, 512, 64), (520, 64, 256, 128)])
def test_weights_beyond_fp16(bits, m, n, k, group):
    """Codes times scales above 65504, which bf16 and fp32 results have room for: right with any number of rows, by whichever kernel."""
    (pg, sg, wg), (pu, su, wu) = _loud(n, k, bits, group, 1), _loud(n, k, bits, group, 2)
    assert wg.abs().max() > 65504
    x, dh = _inputs(m, k, BF16, 3, 1e-4).requires_grad_(), _inputs(m, n, BF16, 4, 1e-3)
    x.data[0, 0] = float("inf")                # one row is not finite, and that stays
    rest = slice(1, m)
    for saved in ("full", "8bit"):
        want = Gated(x.detach()[rest], wg, wu, "silu")
        h = gated.gated_packed(pg, sg, pu, su, n, k, bits, group, x, saved=saved)
        dx, = torch.autograd.grad(h, x, dh)
        inside(h.detach()[rest], want.h, want.h_bound(), "h")
        (v, e), *_ = want.gradients(dh[rest], saved)
        inside(dx[rest], v, e, "dx")
        assert not h[0].isfinite().any()
    d = dh.double()
    off = (2.0 ** -11 + n * 2.0 ** -23 + 2.0 ** -37) * (d.abs() @ wg.abs())
    inside(gated.packed_input_grad(pg, sg, n, k, bits, group, dh), d @ wg, off + 2.0 ** -8 * ((d @ wg).abs() + off), "dy W")
    half = _inputs(m, n, F16, 5, 1e-5)
    want = half.double() @ wg
    off = (2.0 ** -11 + n * 2.0 ** -23 + 2.0 ** -37) * (half.double().abs() @ wg.abs())
    inside(gated.packed_input_grad(pg, sg, n, k, bits, group, half), want, off + 2.0 ** -11 * (want.abs() + off) + 2.0 ** -25, "fp16 dy W")


@pytest.mark.parametrize("shape", [(1, 130), (130, 1), (2, 65)])
@pytest.mark.parametrize("batched", [False, True])
def test_biases_of_any_shape(shape, batched):
    """A bias is as many values as the weight has rows; its gradient has its shape."""
    n, k, m = 130, 256, 5
    (pg, sg, _), (pu, su, _) = _layers(n, k, 4, 128, 1)
    x, dh = _inputs(m, k, F32, 2), _inputs(m, n, F32, 3)
    flat, shaped = ([b.view(s).requires_grad_() for b in (_inputs(1, n, F32, 4), _inputs(1, n, F32, 5))] for s in ((n,), shape))
    (h, got), (want_h, want) = ((y.detach(), torch.autograd.grad(y, b, dh[None] if batched else dh, is_grads_batched=batched)) for b in (shaped, flat)
                                for y in [gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x, *b)])
    assert torch.equal(h, want_h)
    assert all(g.shape == ((1, *shape) if batched else shape) and torch.equal(g.flatten(), w.flatten()) for g, w in zip(got, want))
    watched = torch.func.vmap(lambda t: gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, t, *(b.detach() for b in shaped)))(x)
    assert (watched - h).norm() <= 2.0 ** -16 * h.norm()


@pytest.mark.parametrize("m", [1, 8, 20, 40])
@pytest.mark.parametrize("dtype,k", [(F16, 256), (F32, 256), (BF16, 77)])
def test_nothing_is_kept_where_nothing_is_to_be(m, dtype, k):
    """The C entry with EOQ_B200_KEEP_NONE writes to none of the pointers beside it."""
    import ctypes as C
    from eoq_quantization_b200 import _lib as L
    n = 64
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 64, 1)
    x, h = _inputs(m, k, dtype, 2), torch.empty(m, n, dtype=dtype, device="cuda")
    other = [torch.full((m, n), 7.0, device="cuda") for _ in range(4)]
    w = L.Gated(pg.data_ptr(), pu.data_ptr(), sg.data_ptr(), su.data_ptr(), None, None, n, k, 4, 64, 0, L.F32)
    kept = L.Kept(0, *(t.data_ptr() for t in other))
    code = {F16: L.F16, BF16: L.BF16, F32: L.F32}[dtype]
    lib = L.lib()
    scratch = torch.empty(lib.eoq_b200_gated_scratch(C.byref(w), C.byref(kept), code, m) + 16, dtype=torch.uint8, device="cuda")
    L.check(lib.eoq_b200_gated_packed(C.byref(w), x.data_ptr(), code, m, scratch.data_ptr(), h.data_ptr(), C.byref(kept), torch.cuda.current_stream().cuda_stream), "call")
    want = Gated(x, wg, wu, "silu")
    inside(h, want.h, want.h_bound(), "h")
    assert all((t == 7).all() for t in other)


@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("m,dtype", [(1, F16), (20, BF16), (40, F16), (300, BF16), (5, F32)])
def test_any_bytes(bits, m, dtype):
    """Codes to the very ends of their bits (2, 8, -128), scales of either sign and of zero."""
    n, k, group = 130, 512, 64

    def layer(seed):
        gen = torch.Generator().manual_seed(seed)
        raw = torch.randint(0, 256, (n, k if bits == 8 else k * bits // 8), generator=gen)
        scales = (torch.randn(n * k // group, generator=gen) * 0.01).to(F16)
        scales[::7] = 0
        if bits == 8:
            packed = raw.to(torch.uint8).view(torch.int8)
            codes = packed.double()
        else:
            packed = raw.to(torch.uint8)
            codes = torch.stack([(raw >> s) & (2 ** bits - 1) for s in range(0, 8, bits)], -1).view(n, k).double() - (2 ** (bits - 1) - 1)
        return packed.cuda(), scales.cuda(), (codes * scales.double().repeat_interleave(group).view(n, k)).cuda()
    (pg, sg, wg), (pu, su, wu) = layer(1), layer(2)
    x, dh = _inputs(m, k, dtype, 3).requires_grad_(), _inputs(m, n, dtype, 4)
    want = Gated(x.detach(), wg, wu, "silu")
    h = gated.gated_packed(pg, sg, pu, su, n, k, bits, group, x)
    inside(h.detach(), want.h, want.h_bound(), "h")
    (v, e), *_ = want.gradients(dh, "full")
    inside(torch.autograd.grad(h, x, dh)[0], v, e, "dx")


def test_second_derivatives_behind_hooked_layers():
    """With gate and up called as layers, which can be differentiated again, down can, too."""
    mlp = _module()
    handle = mlp.gate.register_forward_hook(lambda module, args, out: out + 1)
    x = _inputs(6, 256, F32, 2).requires_grad_()
    got = []
    for call in (mlp, lambda t: mlp.down(torch.nn.functional.silu(mlp.gate(t)) * mlp.up(t))):
        for loss in (lambda y: y.sum(), lambda y: y.square().sum()):
            dx, = torch.autograd.grad(loss(call(x)), x, create_graph=True)
            got.append((dx.detach(), torch.autograd.grad(dx.square().sum(), x)[0]))
    handle.remove()
    for (a, b), (c, d) in zip(got[:2], got[2:]):
        assert (a - c).norm() <= 2.0 ** -16 * c.norm() and (b - d).norm() <= 2.0 ** -16 * d.norm() and d.norm() > 0
