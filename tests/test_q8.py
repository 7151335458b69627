"""What the 8-bit operators refuse, and how a weight in 8 bits is laid out, without a GPU."""
import pytest
import torch

from skyla_kernel_b200.kernels import ops


def _rows(n, k, pad=0):
    q = torch.zeros(n, k + pad, dtype=torch.int8)[:, :k]
    return ops.Q8Rows(q, torch.ones(n))


def test_rows_begin_on_multiples_of_16_bytes():
    for n, k in ((1, 1), (3, 16), (5, 17), (2, 100)):
        r = ops.q8_rows(n, k, "cpu")
        assert r.q.shape == (n, k) and r.q.stride(0) % 16 == 0 and r.q.dtype == torch.int8
        assert r.scale.shape == (n,) and r.scale.dtype == torch.float32


def test_a_weight_is_kept_or_laid_out():
    aligned = ops.q8_rows(6, 33, "cpu")
    aligned.q.copy_(torch.arange(6 * 33).reshape(6, 33) % 100)
    w = ops.Q8Weight(*aligned)
    assert w.rows.q.data_ptr() == aligned.q.data_ptr() and (w.n_out, w.n_in, w.ld) == (6, 33, 48)
    packed = aligned.q.contiguous()                      # rows of 33 bytes: copied
    v = ops.Q8Weight(packed, aligned.scale, gated=True)
    assert v.rows.q.data_ptr() != packed.data_ptr() and torch.equal(v.rows.q, packed) and v.ld % 16 == 0
    assert (v.n_out, v.gated, v.bytes()) == (3, True, 6 * 37)
    part = w.first_outputs(2)
    assert part.rows.q.data_ptr() == w.rows.q.data_ptr() and part.n_out == 2
    broadcast = ops.Q8Weight(packed[:1].expand(4, 33), torch.ones(4))  # one row for all outputs: copied as well
    assert broadcast.ld % 16 == 0 and torch.equal(broadcast.rows.q, packed[:1].expand(4, 33))


@pytest.mark.parametrize("make", [
    lambda: ops.Q8Weight(torch.zeros(4, 8, dtype=torch.uint8), torch.ones(4)),
    lambda: ops.Q8Weight(torch.zeros(4, 8, dtype=torch.int8), torch.ones(3)),
    lambda: ops.Q8Weight(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4, dtype=torch.bfloat16)),
    lambda: ops.Q8Weight(torch.zeros(3, 8, dtype=torch.int8), torch.ones(3), gated=True),
    lambda: ops.Q8Weight(torch.zeros(0, 8, dtype=torch.int8), torch.ones(0)),
    lambda: ops.Q8Weight(torch.zeros(1, ops.Q8_MAX_WIDTH + 1, dtype=torch.int8), torch.ones(1)),
    lambda: ops.Q8Weight(torch.zeros(8, 4, dtype=torch.int8).T, torch.ones(4)),
    lambda: ops.Q8Weight(*_rows(4, 16), gated=True).first_outputs(1),
    lambda: ops.Q8Weight(*_rows(4, 16)).first_outputs(5),
    # quantisation
    lambda: ops.quantize_rows(torch.zeros(2, 3, 4)),
    lambda: ops.quantize_rows(torch.zeros(2, 3, dtype=torch.float16)),
    lambda: ops.quantize_rows(torch.zeros(2, 3), _rows(2, 4)),
    lambda: ops.quantize_rows(torch.zeros(2, 3), ops.Q8Rows(torch.zeros(1, 3, dtype=torch.int8).expand(2, 3), torch.ones(2))),
    lambda: ops.dequantize_rows(_rows(2, 3), torch.zeros(2, 4)),
    lambda: ops.dequantize_rows(_rows(2, 3), torch.zeros(1, 3).expand(2, 3)),
    lambda: ops.dequantize_rows(ops.Q8Rows(torch.zeros(2, 3, dtype=torch.int8), torch.ones(4)[::2]), torch.zeros(2, 3)),
    # norm
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(7), 1e-6),
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(8, dtype=torch.bfloat16), 1e-6),
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(8), 1e-6, residual=torch.zeros(1, 8)),
    lambda: ops.rmsnorm_q8(torch.zeros(1, 8).expand(2, 8), torch.ones(8), 1e-6, residual=torch.zeros(2, 8)),
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(8), -1e-6),
    lambda: (lambda t: ops.rmsnorm_q8(t[1:], torch.ones(8), 1e-6, residual=t[:3]))(torch.zeros(4, 8)),
    lambda: (lambda t: ops.rmsnorm_q8(t[:, :8], torch.ones(8), 1e-6, residual=t[:, 4:12]))(torch.zeros(4, 16)),
    lambda: (lambda t: ops.rmsnorm_q8(t, torch.ones(8), 1e-6, residual=t[:1].expand(4, 8)))(torch.zeros(4, 8)),
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(8), float("nan")),
    # product
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 32)), torch.zeros(2, 4)),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(2, 5)),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(2, 4), ops.GATED),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16), gated=True), torch.zeros(2, 2, dtype=torch.bfloat16)),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16), gated=True), torch.zeros(2, 2), ops.GATED),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(2, 4, dtype=torch.bfloat16), ops.ACCUMULATE),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(2, 4), 7),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(1, 4).expand(2, 4)),
    # sizes that the launchers cannot count
    lambda: ops.quantize_rows(torch.empty(1, 2 ** 31, device="meta")),
    lambda: ops.quantize_rows(torch.empty(2 ** 31, 1, device="meta")),
    # all of them on the host
    lambda: ops.quantize_rows(torch.zeros(2, 3)),
    lambda: ops.rmsnorm_q8(torch.zeros(2, 8), torch.ones(8), 1e-6),
    lambda: ops.linear_q8(_rows(2, 16), ops.Q8Weight(*_rows(4, 16)), torch.zeros(2, 4)),
])
def test_refusals(make):
    with pytest.raises(ops.KernelError):
        make()


def test_what_shares_memory():
    t = torch.zeros(6, 20)
    apart = lambda a, b: ops._apart(a, a.stride(0), b, b.stride(0))  # noqa: E731
    assert apart(t[:3], t[3:]) and apart(t[3:], t[:3]) and apart(t[:, :10], t[:, 10:]) and apart(t[:, 12:], t[:, :12])
    assert not apart(t[:4], t[2:]) and not apart(t[:, :10], t[:, 9:19]) and not apart(t, t)
    assert not apart(t[:3, :10], t[::2, 10:])                     # apart, but not by one step: counted as shared
    assert not apart(t, t[:1].expand(6, 20)) and apart(t, torch.zeros(1, 20).expand(6, 20))
    assert not apart(t[:1, :10], t[:1, 5:15]) and apart(t[:1, :10], t[:1, 10:])


def test_outputs_in_the_memory_of_inputs_are_refused():
    t = torch.zeros(4, 32)
    inside = lambda n, k: ops.Q8Rows(t.view(torch.int8)[:n, 4:4 + k], torch.ones(n))  # noqa: E731
    for call in (lambda: ops.quantize_rows(t[:, :8], inside(4, 8)),
                 lambda: ops.quantize_rows(t[:1], inside(1, 32)),
                 lambda: ops.quantize_rows(t[:1].expand(4, 32), inside(4, 32)),
                 lambda: ops.rmsnorm_q8(t, torch.ones(32), 1e-6, inside(4, 32)),
                 lambda: ops.rmsnorm_q8(torch.zeros(4, 32), torch.ones(32), 1e-6, inside(4, 32), residual=t),
                 lambda: ops.dequantize_rows(inside(4, 32), t),
                 lambda: ops.linear_q8(inside(4, 16), ops.Q8Weight(*_rows(32, 16)), t)):
        with pytest.raises(ops.KernelError, match="input's memory"):
            call()
    # beside one another in one buffer they are apart: what is refused then is only that there is no GPU
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.quantize_rows(t[:, 9:], inside(4, 23))


def test_too_many_elements_are_named():
    for shape in ((1, 2 ** 31), (2 ** 31, 2)):
        with pytest.raises(ops.KernelError, match="2\\^29"):
            ops.rmsnorm_q8(torch.empty(*shape, device="meta"), torch.empty(shape[1], device="meta"), 1e-6)


def test_what_a_runtime_takes():
    from skyla_kernel_b200.parts.base import Runtime
    assert Runtime(torch.device("cpu"), "bfloat16", weights="int8").int8 and not Runtime(torch.device("cpu"), "bfloat16").int8
    with pytest.raises(ValueError):
        Runtime(torch.device("cpu"), "float32", weights="int8")
    with pytest.raises(ValueError):
        Runtime(torch.device("cpu"), "bfloat16", weights="int4")


def test_one_error_word_for_threads_that_come_first_together(monkeypatch):
    """The word that the product's kernels write is the one that ``check_device_errors`` reads."""
    import threading
    import time

    class Slow:
        def __init__(self, device):
            time.sleep(0.02)
            self.error_flag = torch.zeros(1, dtype=torch.int32)

    monkeypatch.setattr(ops, "KernelState", Slow)
    monkeypatch.setattr(ops, "_DEFAULT_STATES", {})
    monkeypatch.setattr(ops, "_FLAGS", {})
    start, got = threading.Barrier(8), []

    def ask():
        start.wait()
        got.append(ops._default_flag(0))

    threads = [threading.Thread(target=ask) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    read = ops.default_state("cuda:0").error_flag
    assert len(got) == 8 and all(flag is read for flag in [*got, ops._default_flag(0)])


def _packed(n, k, at, buf):
    """8-bit rows whose scales begin at byte ``at`` of ``buf``; the integers lie elsewhere."""
    return ops.Q8Rows(torch.zeros(n, k, dtype=torch.int8), buf.view(-1).view(torch.int8)[at:at + 4 * n].view(torch.float32))


def test_scales_in_the_memory_of_other_operands_are_refused():
    t = torch.zeros(4, 32)
    q = lambda n, k: t.view(torch.int8)[:n, :k]  # noqa: E731
    flat = t.view(-1)
    for call in (lambda: ops.quantize_rows(t, _packed(4, 32, 16, t)),
                 lambda: ops.quantize_rows(t[:, :8], _packed(4, 8, 24, t)),                    # across the end of a row
                 lambda: ops.quantize_rows(torch.zeros(4, 8), ops.Q8Rows(q(4, 8), flat[:4])),  # the rows' own scales
                 lambda: ops.dequantize_rows(_packed(4, 32, 0, t), t),
                 lambda: ops.rmsnorm_q8(t, torch.ones(32), 1e-6, _packed(4, 32, 16, t)),
                 lambda: ops.rmsnorm_q8(torch.zeros(4, 32), torch.ones(32), 1e-6, _packed(4, 32, 16, t), residual=t),
                 lambda: ops.rmsnorm_q8(torch.zeros(4, 32), flat[:32], 1e-6, _packed(4, 32, 16, t)),
                 lambda: ops.rmsnorm_q8(torch.zeros(4, 32), flat[:32], 1e-6, ops.Q8Rows(q(4, 32), torch.ones(4))),
                 lambda: ops.rmsnorm_q8(torch.zeros(4, 32), torch.ones(32), 1e-6, ops.Q8Rows(q(4, 32), flat[:4])),
                 lambda: ops.rmsnorm_q8(t, flat[32:64], 1e-6, residual=torch.zeros(4, 32)),    # the weight in rows that are written
                 lambda: ops.linear_q8(_packed(4, 16, 128, t), ops.Q8Weight(*_rows(32, 16)), t)):
        with pytest.raises(ops.KernelError, match="memory"):
            call()
    # behind the columns that are used they are apart: what is refused then is only that there is no GPU
    for call in (lambda: ops.quantize_rows(t[:, :8], _packed(4, 8, 32, t)),
                 lambda: ops.quantize_rows(t[1:], _packed(3, 32, 0, t)),
                 lambda: ops.quantize_rows(t[:3], _packed(3, 32, 4 * 96, t)),
                 lambda: ops.dequantize_rows(_packed(4, 8, 32, t), t[:, :8]),
                 lambda: ops.rmsnorm_q8(t[:, :8], flat[8:16], 1e-6, residual=torch.zeros(4, 8)),
                 lambda: ops.rmsnorm_q8(t, flat[32:64], 1e-6),
                 lambda: ops.linear_q8(_packed(4, 16, 32, t), ops.Q8Weight(*_rows(8, 16)), t[:, :8]),
                 lambda: ops.quantize_rows(torch.zeros(0, 8), ops.q8_rows(0, 8, "cpu"))):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()
