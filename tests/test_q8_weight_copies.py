"""A weight in 8 bits that is copied, pickled or saved: what comes back reads its own memory."""
import copy
import io
import pickle

import pytest
import torch

from skyla_kernel_b200.kernels import ops


def _saved(w, **kw):
    f = io.BytesIO()
    torch.save(w, f)
    f.seek(0)
    return torch.load(f, **kw)


def _loaded_safely(w):
    with torch.serialization.safe_globals([ops.Q8Weight]):
        return _saved(w, weights_only=True)


WAYS = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda w: pickle.loads(pickle.dumps(w)),
        "pickle, first protocol": lambda w: pickle.loads(pickle.dumps(w, 0)),
        "save": lambda w: _saved(w, weights_only=False), "save, weights only": _loaded_safely}


def _weight(device, gated, n=6, k=33):
    rows = ops.q8_rows(n, k, device)
    rows.q.copy_(torch.arange(n * k).reshape(n, k) % 100)
    rows.scale.copy_(1 + torch.arange(n))
    return ops.Q8Weight(*rows, gated=gated)


def _same(a, b):
    return torch.equal(a.rows.q, b.rows.q) and torch.equal(a.rows.scale, b.rows.scale) and \
        (a.gated, a.n_out, a.n_in, a.bytes()) == (b.gated, b.n_out, b.n_in, b.bytes())


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("gated", [False, True])
def test_a_copy_reads_its_own_memory(way, gated):
    w = _weight("cpu", gated)
    c = WAYS[way](w)
    assert _same(w, c) and c.ld % 16 == 0 and c.ld == c.rows.q.stride(0)
    assert (c._q, c._scale) == (c.rows.q.data_ptr(), c.rows.scale.data_ptr())
    if way != "copy":  # (a shallow copy shares the tensors)
        assert c._q != w._q and c._scale != w._scale
        w.rows.q.fill_(0)
        w.rows.scale.fill_(0)
        assert _same(c, _weight("cpu", gated))


def test_parts_of_a_weight():
    """The first outputs share the whole's memory; a copy of them, made together with the whole, does too."""
    w = _weight("cpu", False)
    both = copy.deepcopy([w, w.first_outputs(4), w])
    assert both[2] is both[0] and both[1]._q == both[0]._q == both[0].rows.q.data_ptr() != w._q
    assert both[1].n_out == 4 and torch.equal(both[1].rows.q, w.rows.q[:4])


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
def test_products_with_a_copy(way):
    x = ops.quantize_rows(torch.randn(20, 33, generator=torch.Generator().manual_seed(1)).cuda())
    w = _weight("cuda:0", False)
    want = ops.linear_q8(x, w, torch.empty(20, 6, device="cuda"))
    c = WAYS[way](w)
    if way != "copy":
        w.rows.q.fill_(0)
        w.rows.scale.fill_(0)
        torch.cuda.synchronize()
    assert torch.equal(ops.linear_q8(x, c, torch.empty(20, 6, device="cuda")), want)
    ops.check_device_errors("cuda:0")
