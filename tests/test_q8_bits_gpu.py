"""The 8-bit product's results do not depend on which kernel computes them: bit for bit the same for every plan and
for rows of ``x`` and ``y`` on 16 bytes and off them."""
import math

import pytest
import torch

from skyla_kernel_b200.kernels import ops
from test_q8_gpu import BF16, DEV, F32, _q8, _rand, _view
from test_q8_plans_gpu import GATED, PLAIN

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", GATED)
def test_gated_results_by_every_kernel(m, k, n):
    x = _q8(_rand(m, k, seed=m + k + n))
    w = ops.Q8Weight.quantize(_rand(2 * n, k, seed=n) * (8 / math.sqrt(k)), gated=True)
    off = ops.Q8Rows(_view(x.q, 3 if (k + 3) % 16 else 5), x.scale)  # rows off 16 bytes: the plain kernel
    y = ops.linear_q8(x, w, torch.zeros(m, n, dtype=BF16, device=DEV), ops.GATED)
    launches = dict(ops.LAUNCHES_BY_MODULE)
    plain = ops.linear_q8(off, w, torch.zeros(m, n, dtype=BF16, device=DEV), ops.GATED)
    assert m == 1 or ops.LAUNCHES_BY_MODULE["linear_q8_plain"] == launches.get("linear_q8_plain", 0) + 1
    assert torch.equal(y, plain), int((y != plain).sum())
    few = ops.linear_q8(ops.Q8Rows(x.q[:5], x.scale[:5]), w, torch.zeros(min(m, 5), n, dtype=BF16, device=DEV), ops.GATED)
    assert torch.equal(y[:5], few)
    ops.check_device_errors(DEV)


def test_gates_far_below_zero():
    """Down to -87 the exponential is a normal 32-bit number, and silu(gate) * up is what it is in 64 bits within half a
    step of bfloat16 and the exponential's 2 + 1.2 * 87 steps of 32 bits, the quotient's 2 and the products' 2 halves:
    110 * 2^-23 < 2^-16.  Beyond, the output goes to zero: at most what the true value is at -87, and never NaN."""
    gates = torch.linspace(-130, 130, 4096)
    for up in (1.0, -3.0e30):
        scale = torch.cat([gates, torch.full_like(gates, up)]).to(DEV)  # one input, ones throughout: the scales are the values
        w = ops.Q8Weight(torch.ones(2 * len(gates), 1, dtype=torch.int8, device=DEV), scale, gated=True)
        g = gates.double()
        want, near = g / (1 + torch.exp(-g)) * up, g >= -87
        for tokens in (1, 20, 200, 700):
            rows = ops.Q8Rows(ops.q8_rows(tokens, 1, DEV).q.fill_(1), torch.ones(tokens, device=DEV))
            y = ops.linear_q8(rows, w, torch.zeros(tokens, len(gates), dtype=BF16, device=DEV), ops.GATED).cpu()
            assert torch.equal(y, y[:1].expand_as(y))
            torch.testing.assert_close(y[0].double()[near], want[near], rtol=2.0 ** -8 + 2.0 ** -16, atol=2.0 ** -134)
            assert (y[0].double()[~near].abs() <= 87 * math.exp(-87) * abs(up)).all()


@pytest.mark.parametrize("m,k,n", PLAIN)
def test_values_and_sums_below_the_normal_numbers(m, k, n):
    """Products of 2^-127 and less, and sums of such numbers, keep their bits in every kernel."""
    x, w = _q8(_rand(m, k, seed=m + k + n)), ops.Q8Weight.quantize(_rand(n, k, seed=n))
    acc = (x.q.double() @ w.rows.q.double().T).float()
    small = ops.Q8Rows(x.q, torch.full((m,), 2.0 ** -75, device=DEV))
    w = ops.Q8Weight(w.rows.q, torch.full((n,), 2.0 ** -75, device=DEV))
    v = (acc * 2.0 ** -75) * 2.0 ** -75
    assert float(v.abs().max()) < 2.0 ** -126 and int((v != 0).sum()) > 0
    for gap in (0, 1):
        for dtype in (F32, BF16):
            y = _view(torch.zeros(m, n, dtype=dtype, device=DEV), gap)
            assert torch.equal(ops.linear_q8(small, w, y), v.to(dtype)), (gap, dtype)
        y = _view(_rand(m, n, seed=3) * 2.0 ** -127, gap)
        want = y + v
        assert int(((want != 0) & (want.abs() < 2.0 ** -126)).sum()) > 0
        ops.linear_q8(small, w, y, ops.ACCUMULATE)
        assert torch.equal(y, want), (gap, int((y != want).sum()))
    ops.check_device_errors(DEV)
