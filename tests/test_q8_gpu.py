"""The 8-bit operators against their definitions in 64 bits."""
import math
import os

import pytest
import torch

from skyla_kernel_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = torch.bfloat16, torch.float32
FLOOR = 127 * 2.0 ** -126  # under a row's largest magnitude


def _rand(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(DEV)


def _view(t, gap):
    """The same values in rows ``gap`` elements further apart."""
    out = torch.full((t.shape[0], t.shape[1] + gap), 7.0, dtype=t.dtype, device=t.device)[:, : t.shape[1]]
    return out.copy_(t)


def _want(x):
    """(q, scale) of finite rows.  In 64 bits 127 x is exact, and a quotient that is not a half is further from
    one than the division's error."""
    most = x.double().abs().amax(1, keepdim=True).clamp_min(FLOOR)
    return torch.round(x.double() * 127 / most).to(torch.int8), (most[:, 0] / 127).float()


def _q8(x, gap=0):
    r = ops.quantize_rows(x)
    if gap:
        r = ops.Q8Rows(_view(r.q, gap), r.scale)
    return r


# ----------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,width,gap", [(1, 1, 0), (3, 7, 0), (1, 4096, 0), (5, 4096, 8), (37, 130, 5), (9, 1000, 0),
                                         (300, 64, 0), (4, 2561, 13), (2, 12288, 0), (2, 70001, 0)])
def test_quantize_rows(n, width, gap, dtype):
    x = _view((_rand(n, width, seed=n + width) * torch.exp(_rand(width, seed=1))).to(dtype), gap)
    got = ops.quantize_rows(x)
    q, scale = _want(x)
    assert torch.equal(got.q, q) and torch.equal(got.scale, scale)


def test_quotients_that_end_in_one_half():
    # with a largest value of 254 the quotients are half the values: every odd one is a tie, and goes to the even
    x = torch.arange(-254, 255, dtype=F32, device=DEV)[None, :]
    for t in (x, x.to(BF16), x * 2.0 ** -60, x * 2.0 ** 100):
        got = ops.quantize_rows(t)
        assert torch.equal(got.q, torch.round(x / 2).to(torch.int8))
    # values one step of 32 bits to either side of the halves of a largest value that 127 does not divide
    most = torch.tensor(0.7310234, device=DEV)
    near = [((k + 0.5) / 127 * most.double()).float() for k in range(127)]
    near = torch.stack([t for v in near for t in (v, torch.nextafter(v, torch.zeros_like(v)), torch.nextafter(v, torch.ones_like(v)))])
    x = torch.cat([near, -near, most[None]])[None, :]
    q, scale = _want(x)
    got = ops.quantize_rows(x)
    assert torch.equal(got.q, q) and torch.equal(got.scale, scale)


def test_every_bfloat16_value_against_every_largest():
    """Rows of all 16-bit values up to their largest, for every significand that a largest can have."""
    sig = torch.arange(128, 256, dtype=F32)                                # significands
    values = torch.cat([sig * 2.0 ** e for e in range(-10, 1)])            # nearer to 0 than A / 254 all quotients round to 0
    for lo in range(128, 256, 16):
        rows = []
        for a in range(lo, lo + 16):
            rows.append(torch.where(values <= a, values, torch.full_like(values, -a)))
            rows[-1][-1] = a
        x = torch.stack(rows).to(BF16).to(DEV)
        assert torch.equal(x.float().amax(1).cpu(), torch.arange(lo, lo + 16).float())
        for t in (x, x * 2.0 ** -100):
            q, scale = _want(t)
            got = ops.quantize_rows(t)
            assert torch.equal(got.q, q) and torch.equal(got.scale, scale)


def test_rows_of_zeros_small_numbers_and_nans():
    w = 40
    x = _rand(9, w, seed=3)
    x[1] = 0
    x[2] *= 2.0 ** -140          # no 32-bit number but a few bits of one is left: the floor under the scale
    x[3] = 0; x[3, 5] = 2.0 ** -149
    x[4, 7] = math.nan
    x[5, 0] = math.inf
    x[6, w - 1] = -math.inf
    x[7] = 0; x[7, 11] = 3.4e38
    got = ops.quantize_rows(x)
    fine = [0, 1, 2, 3, 7, 8]
    q, scale = _want(x[fine])
    assert torch.equal(got.q[fine], q) and torch.equal(got.scale[fine], scale)
    for r in (4, 5, 6):
        assert math.isnan(float(got.scale[r])) and not got.q[r].any()
    back = ops.dequantize_rows(got, torch.empty(9, w, device=DEV))
    assert not back[1].any() and torch.isnan(back[4:7]).all() and float(back[7, 11]) == pytest.approx(3.4e38, rel=2 ** -22)


def test_only_the_rows_are_written():
    out = ops.Q8Rows(torch.full((6, 48), 55, dtype=torch.int8, device=DEV), torch.full((6,), 5.0, device=DEV))
    x = _rand(3, 33, seed=4)
    ops.quantize_rows(x, ops.Q8Rows(out.q[1:4, :33], out.scale[1:4]))
    q, scale = _want(x)
    assert torch.equal(out.q[1:4, :33], q) and torch.equal(out.scale[1:4], scale)
    assert (out.q[[0, 4, 5]] == 55).all() and (out.q[:, 33:] == 55).all() and (out.scale[[0, 4, 5]] == 5).all()
    none = ops.quantize_rows(torch.empty(0, 33, device=DEV))
    assert none.q.shape == (0, 33) and none.scale.shape == (0,)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,width,gap", [(1, 1, 0), (5, 33, 0), (4, 4096, 16), (3, 1000, 7), (2, 20000, 0)])
def test_dequantize_rows(n, width, gap, dtype):
    q = torch.randint(-128, 128, (n, width), dtype=torch.int8, device=DEV)
    rows = ops.Q8Rows(_view(q, gap), torch.rand(n, device=DEV) + 0.1)
    out = _view(torch.zeros(n, width, dtype=dtype, device=DEV), gap)
    ops.dequantize_rows(rows, out)
    assert torch.equal(out, (q.float() * rows.scale[:, None]).to(dtype))  # one rounding of the product, one of the type


# ------------------------------------------------------------------------ norm
def _norm_close(x, weight, eps, got):
    """``got`` against the norm of ``x`` in 64 bits.  The kernel rounds x * weight once, the largest of them once: a
    quotient moves by at most 127 * 2^-23, so its integer is the exact one unless the exact quotient lies within that
    of a half.  The scale takes the rounding of the sum of squares (a chain of at most width / 32 + 40 additions,
    halved by the root) and of eight operations more."""
    t = x.double() * weight.double()
    most = t.abs().amax(1, keepdim=True).clamp_min(FLOOR)
    z = t * 127 / most
    off = (got.q.double() - z).abs()
    assert float(off.max()) <= 0.5 + 127 * 2.0 ** -23
    inv = 1 / torch.sqrt(x.double().square().mean(1) + eps)
    torch.testing.assert_close(got.scale.double(), most[:, 0] * inv / 127, rtol=(x.shape[1] / 64 + 28) * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("dtype,rdtype", [(F32, None), (F32, F32), (F32, BF16), (BF16, None), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("n,width,gap", [(1, 1, 0), (1, 4096, 0), (3, 80, 4), (5, 2561, 3), (64, 5120, 0), (300, 64, 0),
                                         (2, 16384, 8), (2, 40001, 0)])
def test_rmsnorm_q8(n, width, gap, dtype, rdtype):
    x = _view((_rand(n, width, seed=width) * torch.exp(0.5 * _rand(width, seed=1))).to(dtype), gap)
    weight = 1 + 0.2 * _rand(width, seed=2)
    before = x.clone()
    if rdtype is None:
        got = ops.rmsnorm_q8(x, weight, 1e-6)
        assert torch.equal(x, before)
    else:
        residual = _view((0.5 * _rand(n, width, seed=5)).to(rdtype), 2 * gap)
        got = ops.rmsnorm_q8(x, weight, 1e-6, residual=residual)
        assert torch.equal(x, (before.float() + residual.float()).to(dtype))
    _norm_close(x, weight, 1e-6, got)


def test_a_residual_row_for_all_and_x_itself():
    x, weight = _rand(4, 96, seed=1), torch.ones(96, device=DEV)
    row = _rand(1, 96, seed=2)
    want = x + row
    got = ops.rmsnorm_q8(x, weight, 1e-6, residual=row.expand(4, 96))
    assert torch.equal(x, want)
    _norm_close(x, weight, 1e-6, got)
    ops.rmsnorm_q8(x, weight, 1e-6, residual=x)
    assert torch.equal(x, 2 * want)
    both = _rand(5, 224, seed=3)                      # x and residual as columns of one buffer
    want = both[:, :96] + both[:, 128:]
    got = ops.rmsnorm_q8(both[:, :96], weight, 1e-6, residual=both[:, 128:])
    assert torch.equal(both[:, :96], want)
    _norm_close(want, weight, 1e-6, got)


def test_norm_rows_of_zeros_nans_and_overflow():
    x, weight = _rand(7, 200, seed=6), 1 + 0.1 * _rand(200, seed=7)
    x[1] = 0
    x[2, 3] = math.nan
    x[3, 9] = math.inf
    x[4] *= 1e25                 # its squares leave the 32-bit numbers
    x[5] *= 1e-30                # eps is all that is left of the mean square
    got = ops.rmsnorm_q8(x, weight, 1e-6)
    fine = [0, 1, 5, 6]
    _norm_close(x[fine], weight, 1e-6, ops.Q8Rows(got.q[fine], got.scale[fine]))
    for r in (2, 3, 4):
        assert math.isnan(float(got.scale[r])) and not got.q[r].any()
    none = ops.rmsnorm_q8(x[:2], weight, 0.0)
    assert math.isnan(float(none.scale[1])) and torch.isfinite(none.scale[0])


# --------------------------------------------------------------------- product
def _values(x, w):
    """The product's values bit for bit: whole sums (exact in 64 bits), then the two scales in 32 bits."""
    acc = x.q.double() @ w.rows.q.double().T
    return acc.float() * x.scale[:, None] * w.rows.scale


def _gated_close(v, n, y):
    """Against silu(gate) * up in 64 bits of the same values: half a step of bfloat16, and 2^-15 for the exponential
    (its error grows with its argument, up to about 60 here), the quotient and the products in 32 bits."""
    g, u = v[:, :n].double(), v[:, n:].double()
    torch.testing.assert_close(y.double(), g / (1 + torch.exp(-g)) * u, rtol=2.0 ** -8 + 2.0 ** -15, atol=1e-25)


def _check_product(m, k, n, x_gap=0, y_gap=0, seed=0):
    x = _q8(_rand(m, k, seed=seed), x_gap)
    w = ops.Q8Weight.quantize(_rand(n, k, seed=seed + 1) * 0.1)
    v = _values(x, w)
    for dtype in (F32, BF16):
        y = _view(torch.zeros(m, n, dtype=dtype, device=DEV), y_gap)
        assert ops.linear_q8(x, w, y) is y
        assert torch.equal(y, v.to(dtype))
    y = _view(_rand(m, n, seed=seed + 2), y_gap)
    want = y + v
    ops.linear_q8(x, w, y, ops.ACCUMULATE)
    assert torch.equal(y, want)
    w2 = ops.Q8Weight.quantize(_rand(2 * n, k, seed=seed + 3) * (8 / math.sqrt(k)), gated=True)
    y = _view(torch.zeros(m, n, dtype=BF16, device=DEV), y_gap)
    ops.linear_q8(x, w2, y, ops.GATED)
    _gated_close(_values(x, w2), n, y)
    if y_gap:
        assert (torch.as_strided(y, (m, y_gap), (n + y_gap, 1), n)[: m - 1] == 7).all()  # between the rows
    ops.check_device_errors(DEV)


# tokens around every tile, inputs and outputs that no tile divides
SIZES = [(1, 1, 1), (1, 16, 8), (1, 4096, 6144), (2, 130, 77), (8, 4096, 512), (15, 1000, 333),
         (16, 4096, 4096), (17, 4096, 4096), (33, 2048, 1000), (64, 12288, 256), (65, 512, 516), (100, 384, 4097),
         (128, 2560, 2560), (129, 2560, 640), (130, 100, 70), (256, 1024, 96), (300, 2561, 1111), (513, 640, 129),
         (700, 192, 2050), (20, 2048, 6144), (40, 9728, 2560), (257, 4096, 4000), (1025, 1000, 3001), (2000, 2048, 2048),
         (2100, 130, 2052), (600, 9728, 2560), (1500, 700, 5000), (27, 1621, 64), (2096, 8863, 215), (20, 11142, 171)]


@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_q8(m, k, n):
    _check_product(m, k, n, seed=m + k + n)


def test_every_kernel_is_among_the_sizes():
    """Weight streaming whole, stacked and in clusters, tiles of every width, whole and split, tiles of two SMs."""
    plans = {ops.linear_q8_plan(m, n, k, g) for m, k, n in SIZES for g in (False, True)}
    want = {"streaming, K in 1", "streaming, K in 2", "streaming, K in 4", "tiles of 64 columns, K in 1", "tiles of 64 columns, K in 2",
            "tiles of 64 columns, K in 4", "tiles of 128 columns, K in 1", "tiles of 128 columns, K in 4", "tiles of two SMs"}
    assert want <= plans and any("stacked" in p for p in plans), sorted(want - plans)


@pytest.mark.parametrize("m,k,n", [(3, 64, 40), (40, 1024, 1024), (200, 256, 300)])
@pytest.mark.parametrize("x_gap,y_gap", [(16, 4), (3, 1), (32, 8), (5, 0)])
def test_linear_q8_rows_apart(m, k, n, x_gap, y_gap):
    _check_product(m, k, n, x_gap, y_gap)


@pytest.mark.parametrize("m", [2, 40, 130])
def test_the_longest_sums_are_exact(m):
    k = ops.Q8_MAX_WIDTH
    q = torch.full((m, -(-k // 16) * 16), -128, dtype=torch.int8, device=DEV)[:, :k]
    x = ops.Q8Rows(q, torch.ones(m, device=DEV))
    w = ops.q8_rows(3, k, DEV)
    w.q.fill_(-128); w.q[1].fill_(127); w.q[2, ::2] = 127
    w.scale.fill_(1)
    w = ops.Q8Weight(*w)
    y = torch.empty(m, 3, device=DEV)
    assert torch.equal(ops.linear_q8(x, w, y), _values(x, w))
    assert float(y[0, 0]) == 2.0 ** 31 - 2.0 ** 14  # (rounded to 24 bits: it has 17 ones)


@pytest.mark.parametrize("m", [1, 8, 30, 200])
def test_a_row_without_a_scale_spoils_itself_only(m):
    raw = _rand(m, 256, seed=8)
    raw[m // 2, 100] = math.nan
    x, w = ops.quantize_rows(raw), ops.Q8Weight.quantize(_rand(64, 256, seed=9))
    y = ops.linear_q8(x, w, torch.zeros(m, 64, device=DEV))
    bad = torch.zeros(m, dtype=torch.bool, device=DEV)
    bad[m // 2] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], _values(x, w)[~bad])
    assert ops.linear_q8(ops.Q8Rows(x.q[:0], x.scale[:0]), w, y[:0]).shape == (0, 64)


@pytest.mark.parametrize("m", [1, 16, 40, 100, 129, 300])
@pytest.mark.parametrize("n", [64, 203])
def test_a_product_writes_its_rows_only(m, n):
    """y as the middle of a larger buffer: what lies before, behind and between stays."""
    x = ops.quantize_rows(_rand(m, 512, seed=1))
    for dtype, mode, gated in ((F32, ops.STORE, False), (BF16, ops.STORE, False), (F32, ops.ACCUMULATE, False), (BF16, ops.GATED, True)):
        w = ops.Q8Weight.quantize(_rand(2 * n if gated else n, 512, seed=2), gated=gated)
        whole = torch.full((m + 4, n + 13 if n % 2 else n + 16), 3.0, dtype=dtype, device=DEV)
        before = whole.clone()
        ops.linear_q8(x, w, whole[2:m + 2, :n], mode)
        assert not torch.equal(whole[2:m + 2, :n], before[2:m + 2, :n])
        whole[2:m + 2, :n] = 3
        assert torch.equal(whole, before), (dtype, mode)


def test_many_tokens_of_a_narrow_product():
    """More tiles of tokens than a launch has blocks, offsets beyond 2^31 bytes of y."""
    m, k, n = 300000, 16, 2048
    q = torch.randint(-127, 128, (m, k), dtype=torch.int8, device=DEV)
    x = ops.Q8Rows(q, torch.full((m,), 0.5, device=DEV))
    w = ops.Q8Weight(torch.randint(-127, 128, (n, k), dtype=torch.int8, device=DEV), torch.full((n,), 0.25, device=DEV))
    y = ops.linear_q8(x, w, torch.empty(m, n, device=DEV))
    for lo in (0, 149990, m - 200):
        rows = ops.Q8Rows(q[lo:lo + 200], x.scale[lo:lo + 200])
        assert torch.equal(y[lo:lo + 200], _values(rows, w))


def test_long_rows_apart_beyond_32_bits():
    """Rows 2^30 elements apart: offsets of 2^32 bytes and more."""
    apart, width = 1 << 30, 1000
    x = torch.empty(2 * apart + width, dtype=BF16, device=DEV).as_strided((3, width), (apart, 1))
    x.copy_(_rand(3, width, seed=5))
    got = ops.quantize_rows(x)
    q, scale = _want(x)
    assert torch.equal(got.q, q) and torch.equal(got.scale, scale)
    weight = torch.ones(width, device=DEV)
    got = ops.rmsnorm_q8(x, weight, 1e-6, residual=x)
    _norm_close(x, weight, 1e-6, got)


def test_a_weight_is_not_laid_out_inside_a_capture():
    w = _rand(64, 64)
    ops.Q8Weight.quantize(w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = ops.quantize_rows(w)
        with pytest.raises(ops.KernelError):
            ops.Q8Weight(*rows)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(rows.q, _want(w)[0])


def test_a_product_whose_first_call_is_captured():
    """In a process of its own: nothing of the package has run before."""
    import subprocess
    import sys
    code = """
import torch
from skyla_kernel_b200.kernels import ops
w = ops.Q8Weight.quantize(torch.ones(64, 128, device="cuda"))
x = ops.quantize_rows(torch.ones(200, 128, device="cuda"))
y = torch.zeros(200, 64, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.linear_q8(x, w, y, ops.ACCUMULATE)
ops.check_device_errors("cuda:0")
assert not y.any()
for _ in range(3):
    graph.replay()
ops.check_device_errors("cuda:0")
v = torch.full((200, 64), float(128 * 127 * 127), device="cuda") * x.scale[:, None] * w.rows.scale
assert torch.equal(y, v + v + v), (y, v)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert done.returncode == 0, done.stderr[-2000:]


def test_a_weight_of_the_first_outputs():
    x, w = ops.quantize_rows(_rand(5, 128, seed=1)), ops.Q8Weight.quantize(_rand(96, 128, seed=2))
    whole = ops.linear_q8(x, w, torch.empty(5, 96, device=DEV))
    assert torch.equal(ops.linear_q8(x, w.first_outputs(40), torch.empty(5, 40, device=DEV)), whole[:, :40])


# -------------------------------------------------------------------- together
def _layer(x, residual, norm, gate_up, down):
    """The feed-forward of a layer in 8 bits, and what it leaves on the way."""
    h = ops.rmsnorm_q8(x, norm, 1e-6, residual=residual)
    act = torch.empty(x.shape[0], gate_up.n_out, dtype=BF16, device=DEV)
    ops.linear_q8(h, gate_up, act, ops.GATED)
    a = ops.quantize_rows(act)
    ops.linear_q8(a, down, x, ops.ACCUMULATE)
    return h, act, a


@pytest.mark.parametrize("m", [1, 9, 50, 128, 260])
def test_a_run_of_the_operators(m):
    hidden, inter = 384, 1040
    x, residual = _rand(m, hidden, seed=1), _rand(m, hidden, seed=2).to(BF16)
    norm = 1 + 0.1 * _rand(hidden, seed=3)
    gate_up = ops.Q8Weight.quantize(_rand(2 * inter, hidden, seed=4) * 0.1, gated=True)
    down = ops.Q8Weight.quantize((_rand(hidden, inter, seed=5) * 0.03).to(BF16))
    kept = x + residual.float()
    start = x.clone()
    h, act, a = _layer(x, residual, norm, gate_up, down)
    _norm_close(kept, norm, 1e-6, h)
    _gated_close(_values(h, gate_up), inter, act)
    q, scale = _want(act)
    assert torch.equal(a.q, q) and torch.equal(a.scale, scale)
    assert torch.equal(x, kept + _values(a, down))

    # the same on another stream, and captured and replayed, twice over
    other, stream = start.clone(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _layer(other, residual, norm, gate_up, down)
        again = start.clone()
        graph = torch.cuda.CUDAGraph()
    stream.synchronize()
    assert torch.equal(other, x)
    with torch.cuda.graph(graph):
        _layer(again, residual, norm, gate_up, down)
    for _ in range(2):
        again.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(again, x)
    ops.check_device_errors(DEV)


def test_two_streams_at_once():
    w = ops.Q8Weight.quantize(_rand(1024, 2048, seed=1))
    xs = [ops.quantize_rows(_rand(m, 2048, seed=m)) for m in (8, 40, 129, 260, 1500)]
    want = [_values(x, w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    ys = [torch.zeros(x.q.shape[0], 1024, device=DEV) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, y, s in zip(xs, ys, streams):
            with torch.cuda.stream(s):
                ops.linear_q8(x, w, y)
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for y, v in zip(ys, want))
