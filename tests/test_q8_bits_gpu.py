"""The 8-bit product's results do not depend on which kernel computes them: bit for bit the same for every plan and
for rows of ``x`` and ``y`` on 16 bytes and off them."""
import math

import pytest
import torch

from skyla_kernel_b200.kernels import ops
from test_q8_gpu import BF16, DEV, _q8, _rand, _view
from test_q8_plans_gpu import GATED

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
