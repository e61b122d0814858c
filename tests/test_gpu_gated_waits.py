"""Waits of the gated block's kernels that run out: NaN where a CTA has given up, a status, and the next call as if nothing had been."""
import ctypes as C

import pytest
import torch

from eoq_quantization_b200 import _lib as L
from eoq_quantization_b200 import gated
from gated_reference import weight

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture
def patience():
    """A call that sets how many microseconds a wait may take; two seconds again behind the test."""
    lib = L.lib()

    def set_us(us):
        torch.cuda.synchronize()
        assert lib.eoq_b200_tune(b"qmm_wait_us", us) == 0
    yield set_us
    set_us(2000000)
    lib.eoq_b200_linear_status()


def _runs_out(call, patience, times=30):
    """Without patience what is not there at once has run out, as codes are that come from HBM: results are right or NaN, and NaN
    at least once."""
    lib = L.lib()
    cache = torch.empty(512 << 20, dtype=torch.uint8, device="cuda")

    def late_call():
        cache.zero_()                          # more than the L2 holds
        return call()
    want = call()
    assert want.isfinite().all() and lib.eoq_b200_linear_status() == 0
    late = []
    for us in (1, 0):
        patience(us)
        late += [late_call() for _ in range(times)]
    patience(2000000)
    again = call()
    assert torch.equal(again, want)
    assert all(((y == want) | y.isnan()).all() for y in late)
    assert lib.eoq_b200_linear_status() == 1 and lib.eoq_b200_linear_status() == 0
    assert any(y.isnan().any() for y in late)


# several chunks of codes a warp beyond those of its ring; several rounds of tiles a CTA
@pytest.mark.parametrize("m,n,k,group", [(1, 11008, 4096, 128), (8, 11008, 4096, 128), (1, 5000, 20480, 32)])
def test_few_rows(m, n, k, group, patience):
    (pg, sg, _), (pu, su, _) = weight(n, k, 4, group, 1), weight(n, k, 4, group, 2)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    _runs_out(lambda: gated.gated_packed(pg, sg, pu, su, n, k, 4, group, x), patience)


# slices of activations and codes that do not come; several tiles a warp; several rounds of tiles a CTA
@pytest.mark.parametrize("m,n,k,group", [(24, 11008, 4096, 128), (32, 3000, 4096, 64), (9, 30000, 1024, 128), (17, 700, 8192, 128)])
def test_up_to_32_rows(m, n, k, group, patience):
    """A warp that gives up for want of activations has copies of codes under way, which end before the warp's ring holds its sums and
    before the CTA does."""
    test_few_rows(m, n, k, group, patience)


@pytest.mark.parametrize("m", [1, 8, 24])
def test_a_slow_kernel_in_front_does_not_count(m, patience):
    lib = L.lib()
    n, k = 700, 1024
    (pg, sg, _), (pu, su, _) = weight(n, k, 4, 128, 1), weight(n, k, 4, 128, 2)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(3)).to(F16).cuda()
    call = lambda: gated.gated_packed(pg, sg, pu, su, n, k, 4, 128, x)  # noqa: E731
    want = call()
    handle, g = (C.c_ubyte * 64)(), C.c_void_p()
    L.check(lib.eoq_b200_gather_create(2, 0, 2, 2 * 96 * 2, C.byref(g), handle), "eoq_b200_gather_create")
    try:
        L.check(lib.eoq_b200_gather_set_timeout_ms(g, 100), "eoq_b200_gather_set_timeout_ms")
        patience(20000)
        L.check(lib.eoq_b200_gather_wait(g, 0, 96, 1, L.F16, 3, torch.cuda.current_stream().cuda_stream), "eoq_b200_gather_wait")
        assert torch.equal(call(), want) and lib.eoq_b200_linear_status() == 0
    finally:
        torch.cuda.synchronize()
        lib.eoq_b200_gather_destroy(g)


def test_a_call_that_gave_up_takes_no_patience_from_later_ones(patience):
    """A product whose last sums take two milliseconds, with eight to wait for them, while the status says that another call's
    waits have run out."""
    (pg, sg, _), (pu, su, _) = weight(11008, 4096, 4, 128, 1), weight(11008, 4096, 4, 128, 2)
    few = torch.ones(1, 4096, dtype=F16, device="cuda")
    # a tile of 256 columns for each of up to 74 pairs of SMs, its sums over half a million rows
    n, k, m = 1 << 19, 74 * 256, 256
    packed = torch.randint(0, 15, (n, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.full((n,), 2.0 ** -10, dtype=F16, device="cuda")
    dy = torch.randn(m, n, device="cuda").to(F16)
    call = lambda: gated.packed_input_grad(packed, scales, n, k, 4, k, dy)  # noqa: E731
    want = call()
    assert want.isfinite().all() and L.lib().eoq_b200_linear_status() == 0
    _give_up(lambda: gated.gated_packed(pg, sg, pu, su, 11008, 4096, 4, 128, few), patience)
    patience(8000)
    assert torch.equal(call(), want) and L.lib().eoq_b200_linear_status() == 1


def _give_up(call, patience):
    """The call without patience, its codes not in the L2, and the status not asked for."""
    patience(0)
    cache = torch.empty(512 << 20, dtype=torch.uint8, device="cuda")
    for _ in range(20):
        cache.zero_()
        late = call()
    assert late.isnan().any()
