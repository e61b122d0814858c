"""The gated block on packed weights: forward, backward, the gradient of a packed product, 8-bit storage, against 64 bits."""
import copy

import pytest
import torch

from eoq_quantization_b200 import gated
from eoq_quantization_b200.core.quantized_linear import QuantizedLinear
from gated_reference import HALF_STEP, Gated, _tiny, act, inside, weight

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _inputs(m, k, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=gen) * spread).to(dtype).cuda()


SHAPES = [
    # rows, features, columns, bits, group, type
    (1, 704, 512, 4, 128, F16), (1, 1, 128, 4, 128, BF16), (3, 37, 256, 4, 64, F16), (8, 1003, 384, 4, 32, BF16), (5, 130, 256, 8, 64, F16),
    (7, 64, 512, 8, 128, BF16), (2, 129, 512, 2, 128, F16), (8, 65, 256, 2, 64, BF16),
    (9, 64, 128, 4, 128, F16), (16, 200, 256, 4, 128, BF16), (24, 1100, 1024, 4, 128, BF16), (33, 63, 512, 4, 64, F16), (100, 513, 384, 4, 32, F16),
    (129, 320, 768, 4, 128, BF16), (257, 96, 320, 4, 64, F16), (300, 1000, 512, 4, 128, F16), (513, 65, 256, 4, 128, BF16),
    (40, 257, 384, 8, 128, F16), (70, 127, 320, 8, 32, BF16), (40, 257, 512, 2, 128, BF16), (280, 190, 256, 2, 64, F16),
    (5, 301, 512, 4, 128, F32), (40, 66, 256, 8, 64, F32),
    # several slices of activations, several tiles a CTA, groups of several units
    (32, 1201, 8192, 4, 128, F16), (19, 1190, 2816, 8, 64, BF16), (17, 130, 512, 2, 64, BF16), (30, 77, 256, 8, 32, F16), (12, 64, 768, 4, 256, F16),
    (25, 40, 1024, 2, 128, F16), (10, 200, 1536, 4, 96, BF16), (31, 9500, 256, 4, 32, BF16), (4, 70, 768, 4, 256, BF16), (1, 2500, 4096, 4, 128, BF16),
    # rows that end inside a scale group, odd columns, other widths, odd groups
    (3, 50, 200, 4, 128, F16), (20, 33, 77, 4, 16, BF16), (2, 30, 90, 2, 24, F32), (11, 45, 96, 3, 48, F16), (6, 20, 40, 6, 40, BF16),
    (17, 40, 130, 8, 130, F16),
]


def _layers(n, k, bits, group, seed):
    return weight(n, k, bits, group, seed), weight(n, k, bits, group, seed + 1)


@pytest.mark.parametrize("m,n,k,bits,group,dtype", SHAPES)
def test_forward_and_gradients(m, n, k, bits, group, dtype):
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, bits, group, m + n)
    x, dh = _inputs(m, k, dtype, 1), _inputs(m, n, dtype, 2, 1e-3)
    for kind, saved, bias in (("silu", "full", False), ("gelu", "8bit", True), ("gelu_tanh", "full", True)):
        bg, bu = (_inputs(1, n, t, s)[0] if bias else None for t, s in ((F32, 3), (dtype, 4)))
        want = Gated(x, wg, wu, kind, bg, bu)
        call = lambda *a: gated.gated_packed(pg, sg, pu, su, n, k, bits, group, *a, activation=kind, saved=saved)  # noqa: E731
        h = call(x, bg, bu)
        assert h.dtype == dtype and not h.requires_grad
        inside(h, want.h, want.h_bound(), f"h {kind}")
        leaves = [t.clone().requires_grad_() for t in (x, bg, bu) if t is not None]
        y = call(*leaves)
        inside(y.detach(), want.h, want.h_bound(), f"h for gradients {kind}")
        grads = torch.autograd.grad(y, leaves, dh)
        (dx, off), *db = want.gradients(dh, saved)
        assert [g.dtype for g in grads] == [t.dtype for t in leaves]
        inside(grads[0], dx, off, f"dx {kind} {saved}")
        for got, leaf, (v, e) in zip(grads[1:], leaves[1:], db):
            inside(got, v, e + HALF_STEP[leaf.dtype] * (v.abs() + e) + _tiny(leaf.dtype), f"bias {kind} {saved}")


@pytest.mark.parametrize("m,n,k,bits,group,dtype", SHAPES)
def test_input_grad(m, n, k, bits, group, dtype):
    packed, scales, w = weight(n, k, bits, group, 5)
    dy = _inputs(m, n, dtype, 6, 1e-3)
    got = gated.packed_input_grad(packed, scales, n, k, bits, group, dy)
    d = dy.double()
    each = (0 if dtype == F32 else 2.0 ** -11) + n * 2.0 ** -23 + 2.0 ** -37
    off = each * (d.abs() @ w.abs())
    off = off + HALF_STEP[dtype] * ((d @ w).abs() + off) + _tiny(dtype)
    assert got.dtype == dtype
    inside(got, d @ w, off, "dx")


def test_gradient_against_differences():
    m, n, k = 24, 96, 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 64, 7)
    x, dh = _inputs(m, k, F16, 8).requires_grad_(), _inputs(m, n, F16, 9)
    for kind in ("silu", "gelu", "gelu_tanh"):
        y = gated.gated_packed(pg, sg, pu, su, n, k, 4, 64, x, activation=kind)
        dx, = torch.autograd.grad(y, x, dh)
        (_, off), *_ = Gated(x.detach(), wg, wu, kind).gradients(dh, "full")
        v = _inputs(m, k, F32, 10).double()
        # a difference in 64 bits; its own error is of third order, 1e-8 of the values
        step = 1e-4
        want = (_value(x.detach().double() + step * v, wg, wu, kind, dh) - _value(x.detach().double() - step * v, wg, wu, kind, dh)) / (2 * step)
        assert abs((dx.double() * v).sum() - want) <= (off * v.abs()).sum() + 1e-5 * abs(want) + 1e-6, kind


def _value(x, wg, wu, kind, dh):
    return (act(x @ wg.T, kind)[0] * (x @ wu.T) * dh.double()).sum()


def _exact_store(x):
    """(quotients 127 x / largest in 64 bits, scales): NaN where a block is not finite, zero where it is below 1e-30."""
    m, n = x.shape
    v = torch.cat([x.double(), x.new_zeros(m, -n % 64).double()], 1).view(m, -1, 64)
    most = v.abs().amax(-1, keepdim=True)
    keep = most >= 1e-30
    q = torch.where(keep, 127 * v / torch.where(keep, most, 1.0), 0.0)
    return q.view(m, -1)[:, :n], torch.where(most.isfinite(), torch.where(keep, most / 127, 0.0), float("nan"))[..., 0].float()


def _check_stored(s, x):
    """Codes: the nearest whole number, half to even.  A quotient in fp32 is off by 2^-24 of itself at most, which decides where
    it is that near to a half (and not one)."""
    q, scale = _exact_store(x)
    fine = ~scale.isnan().repeat_interleave(64, 1)[:, :x.shape[1]]
    codes = s.codes.view(q.shape).double()
    near = ((q - q.floor() - 0.5).abs() <= 127 * 2.0 ** -23) & (q - q.floor() != 0.5)
    assert torch.equal(codes[fine & ~near], torch.round(q)[fine & ~near]) and ((codes - q).abs() <= 0.5 + 127 * 2.0 ** -23)[fine].all() and (codes[~fine] == 0).all()
    assert torch.equal(s.scales.view(scale.shape).nan_to_num(-1), scale.nan_to_num(-1))
    return (s.codes.view(q.shape).float() * scale.repeat_interleave(64, 1)[:, :x.shape[1]])


@pytest.mark.parametrize("shape", [(1, 1), (1, 64), (3, 65), (5, 1003), (2, 7, 128), (64, 4096), (130, 24), (0, 64), (3, 0)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_store_8bit(shape, dtype):
    x = _inputs(max(1, int(torch.tensor(shape[:-1]).prod())), shape[-1], dtype, 11)
    x = x[:int(torch.tensor(shape[:-1]).prod())].view(shape)
    s = gated.store_8bit(x)
    y = s.dequantize()
    assert y.shape == x.shape and y.dtype == dtype and s.codes.dtype == torch.int8 and s.scales.shape == (*shape[:-1], -(-shape[-1] // 64))
    if not x.numel():
        return
    values = _check_stored(s, x.reshape(-1, shape[-1]))
    assert torch.equal(y.view(values.shape), values.to(dtype))
    assert torch.equal(s.dequantize(F32).view(values.shape), values)
    assert (y.double() - x.double()).abs().max() <= x.abs().max().item() * (1 / 253 + HALF_STEP[dtype])


def test_store_8bit_of_what_is_not_finite():
    x = _inputs(6, 200, F32, 12)
    x[0, 3], x[1, 70], x[2, 199], x[3] = float("nan"), float("inf"), -float("inf"), 0.0
    x[4, :64] *= 1e-38
    x[5, 64:128] = 1e38 * torch.sign(x[5, 64:128])
    s = gated.store_8bit(x)
    values = _check_stored(s, x)
    y = s.dequantize()
    assert y[0, :64].isnan().all() and y[1, 64:128].isnan().all() and y[2, 192:].isnan().all() and (y[3] == 0).all() and (y[4, :64] == 0).all()
    assert y.isnan().sum() == 64 + 64 + 8 and torch.equal(y.nan_to_num(-7), values.nan_to_num(-7))


@pytest.mark.parametrize("m", [2, 40, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_that_are_not_finite(m, dtype):
    n, k = 130, 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 13)
    x = _inputs(m, k, dtype, 14)
    x[1, 5] = float("nan")
    x[0] = 0
    h = gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x)
    want = Gated(x, wg, wu, "silu")
    rest = [i for i in range(m) if i != 1]
    assert h[1].isnan().all() and (h[0] == 0).all()
    inside(h[rest], want.h[rest], want.h_bound()[rest], "the other rows")
    dh = _inputs(m, n, dtype, 15)
    dh[1, 4] = float("inf")
    dx = gated.packed_input_grad(pg, sg, n, k, 4, 128, dh)
    assert not dx[1].isfinite().any() and dx[rest].isfinite().all()


@pytest.mark.parametrize("m", [4, 50])
@pytest.mark.parametrize("spread", [2.0 ** -30, 2.0 ** 20])
def test_rows_of_any_magnitude(m, spread):
    """bf16 rows far outside fp16's range, small and large in one call."""
    n, k = 65, 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 16)
    x = _inputs(m, k, BF16, 17)
    x[::2] *= spread
    want = Gated(x, wg, wu, "gelu")
    inside(gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x, activation="gelu"), want.h, want.h_bound() + 1e-38, "h")
    dy = _inputs(m, n, BF16, 18)
    dy[::2] *= spread
    off = (2.0 ** -11 + n * 2.0 ** -23 + 2.0 ** -37) * (dy.double().abs() @ wg.abs())
    inside(gated.packed_input_grad(pg, sg, n, k, 4, 128, dy), dy.double() @ wg, off + 2.0 ** -8 * ((dy.double() @ wg).abs() + off) + 1e-38, "dx")


@pytest.mark.parametrize("how", ["strided", "transposed", "misaligned", "three dimensions", "scales cast", "weights off 16 bytes", "scales off 16 bytes", "no rows"])
@pytest.mark.parametrize("m", [4, 36])
def test_layouts(how, m):
    n, k = 96, 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 64, 19)
    x, dh = _inputs(m, k, BF16, 20), _inputs(m, n, BF16, 21)
    off = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view_as(t)  # noqa: E731
    if how == "strided":
        x, dh = torch.stack([x, x], -1)[..., 0], torch.stack([dh, dh], -1)[..., 0]
    elif how == "transposed":
        x, dh = x.T.contiguous().T, dh.T.contiguous().T
    elif how == "misaligned":
        x, dh = off(x), off(dh)
    elif how == "three dimensions":
        x, dh = x.view(2, m // 2, k), dh.view(2, m // 2, n)
    elif how == "scales cast":
        sg, su = sg.float(), su.double()
    elif how == "weights off 16 bytes":
        pg, pu, sg, su = off(pg), off(pu), off(sg), off(su)
    elif how == "scales off 16 bytes":
        sg, su = off(sg), off(su)
    elif how == "no rows":
        x, dh = x[:0], dh[:0]
    x.requires_grad_()
    h = gated.gated_packed(pg, sg, pu, su, n, k, 4, 64, x, saved="8bit")
    dx, = torch.autograd.grad(h, x, dh)
    dy = gated.packed_input_grad(pg, sg, n, k, 4, 64, dh)
    assert h.shape == (*x.shape[:-1], n) and dx.shape == x.shape and dy.shape == x.shape
    if how == "no rows":
        return
    want = Gated(x.detach().reshape(-1, k), wg, wu, "silu")
    inside(h.detach().reshape(-1, n), want.h, want.h_bound(), "h")
    (v, e), *_ = want.gradients(dh.reshape(-1, n), "8bit")
    inside(dx.reshape(-1, k), v, e, "dx")


def test_expanded_gradient_and_two_backward_passes():
    n, k = 96, 256
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 64, 22)
    x, b = _inputs(40, k, F16, 23).requires_grad_(), _inputs(1, n, F32, 24)[0].requires_grad_()
    h = gated.gated_packed(pg, sg, pu, su, n, k, 4, 64, x, b, b)         # one bias for both: its gradient is the sum
    h.sum().backward(retain_graph=True)
    first = x.grad.clone(), b.grad.clone()
    (v, e), *db = Gated(x.detach(), wg, wu, "silu", b.detach(), b.detach()).gradients(torch.ones(40, n, device="cuda", dtype=F16), "full")
    inside(first[0], v, e, "dx")
    inside(first[1], db[0][0] + db[1][0], db[0][1] + db[1][1] + 2.0 ** -23 * (db[0][0] + db[1][0]).abs(), "shared bias")
    x.grad = b.grad = None
    h.sum().backward()
    assert torch.equal(x.grad, first[0]) and torch.equal(b.grad, first[1])     # the same bits


def test_refusals():
    n, k = 64, 128
    (pg, sg, _), (pu, su, _) = _layers(n, k, 4, 128, 25)
    x = _inputs(3, k, F16, 26)
    call = gated.gated_packed
    for wrong, error in (((pg, sg, pu, su, n, k, 4, 128, x[:, :64]), ValueError), ((pg[:32], sg, pu, su, n, k, 4, 128, x), ValueError),
                         ((pg, sg[:5], pu, su, n, k, 4, 128, x), ValueError), ((pg, sg, pu.to(torch.int8), su, n, k, 4, 128, x), ValueError),
                         ((pg, sg, pu, su, n, k, 4, 0, x), ValueError), ((pg, sg, pu, su, n, k, 9, 128, x), ValueError),
                         ((pg, sg, pu, su, n, k, 4, 128, x.double()), TypeError), ((pg, sg, pu, su, n, k, 4, 128, x.cpu()), RuntimeError),
                         ((pg.cpu(), sg, pu, su, n, k, 4, 128, x), RuntimeError), ((pg, sg, pu, su, n, k, 4, 128, x, sg[:3]), ValueError),
                         ((pg, sg, pu, su, n, k, 4, 128, x, torch.zeros(n)), ValueError), ((pg, sg.requires_grad_(), pu, su, n, k, 4, 128, x.clone().requires_grad_()), ValueError)):
        with pytest.raises(error):
            call(*wrong)
    sg.requires_grad_(False)
    with pytest.raises(ValueError):
        call(pg, sg, pu, su, n, k, 4, 128, x, activation="tanh")
    with pytest.raises(ValueError):
        call(pg, sg, pu, su, n, k, 4, 128, x, saved="none")
    with pytest.raises(ValueError):
        gated.packed_input_grad(pg, sg, n, k, 4, 128, x)
    with pytest.raises(TypeError):
        gated.store_8bit(x.double())
    with pytest.raises(RuntimeError):
        gated.store_8bit(x.cpu())
    h = call(pg, sg, pu, su, n, k, 4, 128, x.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        pg += 1                              # written between the passes
        h.sum().backward()


def _mlp(bits=4, block=64, bias=True, **kw):
    torch.manual_seed(27)
    gate, up, down = torch.nn.Linear(256, 320, bias=bias), torch.nn.Linear(256, 320, bias=bias), torch.nn.Linear(320, 256, bias=bias)
    return gated.QuantizedGatedMLP.from_float(gate.cuda(), up.cuda(), down.cuda(), bits=bits, block_size=block, **kw)


@pytest.mark.parametrize("m,dtype,saved", [(1, F16, "full"), (8, BF16, "8bit"), (48, F16, "8bit"), (200, BF16, "full"), (12, F32, "full")])
def test_module_against_its_layers(m, dtype, saved):
    mlp = _mlp(saved=saved)
    x = _inputs(m, 256, dtype, 28)
    layers = lambda t: mlp.down(torch.nn.functional.silu(mlp.gate(t)) * mlp.up(t))  # noqa: E731
    # the layers round gate, up, their product and h to the type, the block h alone: four roundings, weighed by what follows
    tol = 6 * HALF_STEP[dtype] + 2.0 ** -10 * (dtype != F32) + 2.0 ** -17
    y, want = mlp(x), layers(x)
    assert y.dtype == dtype and (y - want).double().norm() <= tol * want.double().norm()
    x1, x2 = (x.clone().requires_grad_() for _ in range(2))
    dy = _inputs(m, 256, dtype, 29)
    mlp(x1).backward(dy)
    layers(x2).backward(dy)
    kept = 1 / 127 if saved == "8bit" else 0           # (of a block's largest, some three times its root mean square)
    assert (x1.grad - x2.grad).double().norm() <= (2 * tol + 3 * kept) * x2.grad.double().norm()


def test_module_as_a_program_uses_it():
    mlp = _mlp()
    x = _inputs(24, 256, F32, 30)
    with torch.autocast("cuda", torch.bfloat16):
        y = mlp(x)
    assert y.dtype == BF16
    half = copy.deepcopy(mlp).half()                   # scales and biases cast with the module
    assert half(x.half()).dtype == F16
    state = mlp.state_dict()
    other = _mlp()
    other.load_state_dict(state)
    assert torch.equal(other(x), mlp(x))
    out = torch.func.vmap(mlp)(x.view(4, 6, 256))      # function transforms: torch's own operations
    assert (out.view(24, 256) - mlp(x)).norm() <= 1e-4 * out.norm()
    p = torch.nn.Parameter(torch.zeros(24, 256, device="cuda"))
    (mlp(x + p)).square().mean().backward()
    assert p.grad.isfinite().all() and p.grad.abs().sum() > 0


def test_streams_graphs_and_two_calls_at_once():
    n, k = 320, 512
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, 4, 128, 31)
    for m in (1, 30, 280):
        xs = [_inputs(m, k, F16, 32 + i) for i in range(2)]
        call = lambda t: gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, t)  # noqa: E731
        want = [call(t) for t in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        got = []
        for s, t in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append([call(t) for _ in range(5)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
        # captured with its backward pass, while an eager graph of the same leaf is alive
        leaf = xs[0].clone().requires_grad_()
        alive = call(leaf)
        static, dh = xs[0].clone().requires_grad_(), torch.ones(m, n, device="cuda", dtype=F16)
        eager, = torch.autograd.grad(call(static), static, dh)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                torch.autograd.grad(call(static), static, dh)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(static)
            dx, = torch.autograd.grad(y, static, dh)
            dy = gated.packed_input_grad(pg, sg, n, k, 4, 128, dh)
            back = gated.store_8bit(y.detach()).dequantize()
        with torch.no_grad():
            static.copy_(xs[1])
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[1]) and torch.equal(back, gated.store_8bit(want[1]).dequantize())
        fresh = xs[1].clone().requires_grad_()
        assert torch.equal(dx, torch.autograd.grad(call(fresh), fresh, dh)[0])
        assert torch.equal(dy, gated.packed_input_grad(pg, sg, n, k, 4, 128, dh))
        assert torch.equal(eager, torch.autograd.grad(alive, leaf, dh)[0])


def test_quantized_linear_is_what_it_was():
    layer = QuantizedLinear.from_float(torch.nn.Linear(256, 320).cuda(), bits=4, block_size=64)
    x = _inputs(40, 256, BF16, 40).requires_grad_()
    dy = _inputs(40, 320, BF16, 41)
    layer(x).backward(dy)
    assert torch.equal(x.grad, dy @ layer._dequantize_weight().to(BF16))


@pytest.mark.parametrize("m,n,k,bits,group,dtype", [
    # more tiles than pairs of SMs, whose runs end inside tiles; fewer tiles, several pairs each; runs of two whole tiles
    (60, 10100, 4096, 4, 128, F16), (250, 5000, 8192, 4, 128, BF16), (1000, 2400, 4096, 2, 128, F16), (90, 4500, 2816, 8, 64, F16),
    (40, 3000, 20000, 4, 160, BF16), (150, 11000, 512, 4, 64, F16), (230, 9000, 2048, 8, 128, BF16), (200, 9000, 1024, 2, 64, F16),
])
def test_tiles_that_pairs_share(m, n, k, bits, group, dtype):
    (pg, sg, wg), (pu, su, wu) = _layers(n, k, bits, group, 7)
    x = _inputs(m, k, dtype, 1)
    want = Gated(x, wg, wu, "silu", None, None)
    inside(gated.gated_packed(pg, sg, pu, su, n, k, bits, group, x), want.h, want.h_bound(), "h")
    test_input_grad(m, n, k, bits, group, dtype)


def test_waits_that_run_out_say_so_and_leave_the_next_call_alone():
    """No patience at all, behind a kernel that waits for a peer that never sends: a call whose waits run out gives NaN and a status, once (one that started
    late enough is right); the calls after it are right."""
    import ctypes as C
    from eoq_quantization_b200 import _lib as L
    lib = L.lib()
    n, k = 700, 1024
    (pg, sg, _), (pu, su, _) = _layers(n, k, 4, 128, 3)
    handle, g = (C.c_ubyte * 64)(), C.c_void_p()
    L.check(lib.eoq_b200_gather_create(2, 0, 2, 2 * 96 * 2, C.byref(g), handle), "eoq_b200_gather_create")
    L.check(lib.eoq_b200_gather_set_timeout_ms(g, 100), "eoq_b200_gather_set_timeout_ms")
    ran_out = 0
    try:
        for m in (48, 300):
            x, dy = _inputs(m, k, F16, 1), _inputs(m, n, F16, 2)
            for call in (lambda: gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x), lambda: gated.packed_input_grad(pg, sg, n, k, 4, 128, dy)):
                want = call()
                assert want.isfinite().all() and lib.eoq_b200_linear_status() == 0
                torch.cuda.synchronize()
                assert lib.eoq_b200_tune(b"qmm_wait_us", 0) == 0
                L.check(lib.eoq_b200_gather_wait(g, 0, 96, 1, L.F16, 3, torch.cuda.current_stream().cuda_stream), "eoq_b200_gather_wait")
                late = call()
                torch.cuda.synchronize()
                assert lib.eoq_b200_tune(b"qmm_wait_us", 2000000) == 0
                assert torch.equal(call(), want)
                status = lib.eoq_b200_linear_status()
                assert lib.eoq_b200_linear_status() == 0
                assert late.isnan().any() if status else torch.equal(late, want)
                ran_out += status
                # a kernel in front that takes longer than a wait may: its time does not count
                assert lib.eoq_b200_tune(b"qmm_wait_us", 20000) == 0
                L.check(lib.eoq_b200_gather_wait(g, 0, 96, 1, L.F16, 3, torch.cuda.current_stream().cuda_stream), "eoq_b200_gather_wait")
                assert torch.equal(call(), want) and lib.eoq_b200_linear_status() == 0
                assert lib.eoq_b200_tune(b"qmm_wait_us", 2000000) == 0
        assert ran_out
    finally:
        lib.eoq_b200_tune(b"qmm_wait_us", 2000000)
        lib.eoq_b200_gather_destroy(g)
