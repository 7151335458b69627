"""Every kernel that ``linear_q8`` chooses among, gated and not, by a size that reaches it: results against the definition,
with rows of ``y`` on 16 bytes and off them."""
import math

import pytest
import torch

from skyla_kernel_b200.kernels import ops
from test_q8_gpu import BF16, DEV, F32, _gated_close, _q8, _rand, _values, _view

pytestmark = pytest.mark.gpu

STREAM, TILES, PAIR = "streaming, ", "tiles of ", "tiles of two SMs"
# (tokens, inputs, outputs) -> what the plan says of them (y aligned), however many clusters a B200 runs at a time
PLAIN = {
    (1, 2048, 8): STREAM + "16 K blocks stacked", (16, 256, 215): STREAM + "2 K blocks stacked", (3, 512, 203): STREAM + "4 K blocks stacked",
    (8, 1000, 24): STREAM + "K in 1", (17, 1621, 128): STREAM + "K in 2", (33, 9728, 64): STREAM + "K in 4",
    (65, 384, 512): TILES + "64 columns, K in 1", (17, 4096, 3001): TILES + "64 columns, K in 2", (300, 1621, 171): TILES + "64 columns, K in 4",
    (17, 64, 9728): TILES + "128 columns, K in 1", (65, 8863, 5000): TILES + "128 columns, K in 2", (17, 9728, 3001): TILES + "128 columns, K in 4",
    (257, 64, 9728): TILES + "256 columns, K in 1", (384, 64, 12288): TILES + "256 columns, K in 1",
    (129, 11142, 5000): TILES + "256 columns, K in 2", (300, 12288, 4096): TILES + "256 columns, K in 2",
    (129, 16384, 2560): TILES + "256 columns, K in 4", (200, 16384, 3001): TILES + "256 columns, K in 4",
    (129, 64, 9728): PAIR,
}
GATED = {
    (8, 1000, 24): STREAM + "K in 1", (20, 4096, 12288): STREAM + "K in 1", (20, 2048, 6144): TILES + "128 columns, K in 1",
    (17, 64, 8): TILES + "128 columns, K in 1", (17, 2560, 2560): TILES + "128 columns, K in 2", (257, 2560, 8): TILES + "128 columns, K in 4",
    (48, 64, 9728): TILES + "256 columns, K in 1", (65, 130, 12288): TILES + "256 columns, K in 1", (64, 4096, 12288): TILES + "256 columns, K in 1",
    (100, 4096, 12288): TILES + "256 columns, K in 1", (300, 4096, 12288): TILES + "256 columns, K in 1",
    (129, 11142, 2560): TILES + "256 columns, K in 2", (183, 16384, 1500): TILES + "256 columns, K in 4",
    (129, 64, 5000): PAIR,
}
EVERY = {TILES + f"{c} columns, K in {s}" for c in (64, 128, 256) for s in (1, 2, 4)} | {STREAM + f"K in {s}" for s in (1, 2, 4)} | {PAIR}


def test_every_plan_has_a_size():
    """A gated product has no tile of 64 columns, and its weight streams with K whole."""
    assert EVERY <= set(PLAIN.values())
    assert {p for p in EVERY if " 64 " not in p and p not in (STREAM + "K in 2", STREAM + "K in 4")} <= set(GATED.values())


@pytest.mark.parametrize("m,k,n", PLAIN)
def test_store_and_add(m, k, n):
    assert ops.linear_q8_plan(m, n, k) == PLAIN[m, k, n]
    x, w = _q8(_rand(m, k, seed=m + k + n)), ops.Q8Weight.quantize(_rand(n, k, seed=n) * 0.1)
    v = _values(x, w)
    for gap in (0, 8, 1):
        for dtype in (F32, BF16):
            y = _view(torch.zeros(m, n, dtype=dtype, device=DEV), gap)
            assert torch.equal(ops.linear_q8(x, w, y), v.to(dtype)), (gap, dtype)
        y = _view(_rand(m, n, seed=3), gap)
        want = y + v
        assert torch.equal(ops.linear_q8(x, w, y, ops.ACCUMULATE), want), gap
    ops.check_device_errors(DEV)


@pytest.mark.parametrize("m,k,n", GATED)
def test_gated(m, k, n):
    assert ops.linear_q8_plan(m, n, k, True) == GATED[m, k, n]
    x = _q8(_rand(m, k, seed=m + k + n))
    w = ops.Q8Weight.quantize(_rand(2 * n, k, seed=n) * (8 / math.sqrt(k)), gated=True)
    v = _values(x, w)
    for gap in (0, 8, 1):
        y = _view(torch.zeros(m, n, dtype=BF16, device=DEV), gap)
        ops.linear_q8(x, w, y, ops.GATED)
        _gated_close(v, n, y)
    ops.check_device_errors(DEV)
