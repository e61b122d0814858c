"""The gated block on packed weights in 64 bits, from its definition, and how far the kernels may be from it: bounds for every
element, from the roundings that the forms make (half a step each: 2^-11 fp16, 2^-8 bf16, 2^-24 fp32) and from fp32 sums of
`n` terms, of which the tensor cores cut each addition off (n 2^-23 of the sum of magnitudes)."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# largest slopes and second derivatives of the activations
SLOPE = {"silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13}
BEND = {"silu": 0.51, "gelu": 0.8, "gelu_tanh": 0.85}
FUNCTION = 2.0 ** -18      # an activation or its slope in fp32, by the approximate exponential: 2 ulp and the argument's rounding


def weight(n, k, bits, group, seed, spread=0.02):
    """(packed, fp16 scales, the weight in 64 bits) of seeded codes over the whole of their range, on the GPU."""
    gen = torch.Generator().manual_seed(seed)
    qmax = (1 << (bits - 1)) - 1
    q = torch.randint(-qmax, qmax + 1, (n, k), generator=gen)
    scales = (torch.rand(-(-n * k // group), generator=gen) * spread / qmax + 1e-4).to(torch.float16)
    dense = q.double() * scales.double().repeat_interleave(group)[:n * k].view(n, k)
    u = (q + qmax).to(torch.uint8)
    per = 8 // bits if bits in (2, 4) else 1
    if per == 1:
        packed = q.to(torch.int8)
    else:
        u = torch.cat([u, u.new_zeros(n, -k % per)], 1)
        packed = sum(u[:, j::per] << (bits * j) for j in range(per)).to(torch.uint8)
    return packed.cuda(), scales.cuda(), dense.cuda()


def act(g, kind):
    """Value and slope."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        p = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return g * 0.5 * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


class Gated:
    """Values and bounds of one call."""

    def __init__(self, x, wg, wu, kind, bg=None, bu=None):
        self.kind, self.dtype, self.x, self.wg, self.wu = kind, x.dtype, x.double(), wg, wu
        self.rounding = 0.0 if x.dtype == torch.float32 else 2.0 ** -11           # code x scale to fp16
        bg, bu = (0 if b is None else b.double() for b in (bg, bu))
        self.g, self.u = self.x @ wg.T + bg, self.x @ wu.T + bu
        self.value, self.slope = act(self.g, kind)
        self.h = self.value * self.u
        k = x.shape[-1]
        # fp32 activations go in as halves of 22 bits; bf16 ones as fp16 that keeps all within 2^-24 of the row's largest
        each = self.rounding + k * 2.0 ** -23 + 2.0 ** -21
        self.dg = (self.x.abs() @ wg.abs().T) * each + 2.0 ** -23 * self.g.abs()
        self.du = (self.x.abs() @ wu.abs().T) * each + 2.0 ** -23 * self.u.abs()

    def h_bound(self):
        d = SLOPE[self.kind] * self.dg * (self.u.abs() + self.du) + self.value.abs() * self.du
        return d + (HALF_STEP[self.dtype] + FUNCTION) * (self.h.abs() + d) + _tiny(self.dtype)

    def gradients(self, dh, saved):
        """dx and the biases' gradients with their bounds; with "8bit" of the values as they are kept, whose distance from the
        exact ones counts as the kernels'."""
        step = HALF_STEP[self.dtype]
        g, u, eg, eu = self.g, self.u, self.dg, self.du
        if saved == "8bit":
            eg, eu = (e + _block_max(v.abs() + e) / 253 for v, e in ((g, eg), (u, eu)))
        else:
            eg, eu = (e + step * (v.abs() + e) + _tiny(self.dtype) for v, e in ((g, eg), (u, eu)))
        d = dh.double()
        dg, du = d * u * self.slope, d * self.value
        slope_off = BEND[self.kind] * eg + FUNCTION
        edg = d.abs() * (eu * (self.slope.abs() + slope_off) + u.abs() * slope_off) + 2.0 ** -22 * dg.abs()
        edu = d.abs() * (SLOPE[self.kind] * eg + FUNCTION * self.value.abs()) + 2.0 ** -22 * du.abs()
        if self.rounding:                              # to fp16, times a power of two of the row
            row = torch.maximum(dg.abs().amax(-1, keepdim=True), du.abs().amax(-1, keepdim=True)) * 2.0 ** -38
            edg, edu = edg + 2.0 ** -11 * (dg.abs() + edg) + row, edu + 2.0 ** -11 * (du.abs() + edu) + row
        n, m = 2 * dg.shape[-1], dg.shape[0]
        dx = dg @ self.wg + du @ self.wu
        each = self.rounding + n * 2.0 ** -23
        off = edg @ self.wg.abs() + edu @ self.wu.abs() + each * ((dg.abs() + edg) @ self.wg.abs() + (du.abs() + edu) @ self.wu.abs())
        bias = []
        for v, e in ((dg, edg), (du, edu)):
            s = e.sum(0) + m * 2.0 ** -24 * (v.abs() + e).sum(0)
            bias.append((v.sum(0), s))
        return (dx, off + step * (dx.abs() + off) + _tiny(self.dtype)), *bias


def _tiny(dtype):
    """Half the spacing of a type's smallest numbers."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]


def _block_max(v, block=64):
    m, n = v.shape
    b = torch.cat([v, v.new_zeros(m, -n % block)], 1).view(m, -1, block)
    return b.amax(-1, keepdim=True).expand_as(b).reshape(m, -1)[:, :n]


def inside(got, want, bound, what):
    """Every element within its bound."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} of the bound, at {int((off / bound).argmax())}"
