"""First calls of the 8-bit product from several threads at once, in a process of their own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PLANS = """
import threading, torch
from skyla_kernel_b200.kernels import ops
torch.zeros(1, device="cuda")
ops._fn("gemm_q8", "skyla_linear_q8_plan", [ops.c_int] * 4)        # the library is loaded, nothing has been asked
sizes = [(2048, 6144, 4096), (33, 64, 9728), (17, 128, 1621)]      # tiles of two SMs, clusters of four and of two
start, got = threading.Barrier(16), {}
def ask(i):
    start.wait()
    got[i] = [ops.linear_q8_plan(*size) for size in sizes]
threads = [threading.Thread(target=ask, args=(i,)) for i in range(16)]
for t in threads: t.start()
for t in threads: t.join()
print(sorted(set(map(tuple, got.values()))))
assert all(g == ["tiles of two SMs", "streaming, K in 4", "streaming, K in 2"] for g in got.values())
"""

PRODUCTS = """
import threading, torch
from skyla_kernel_b200.kernels import ops
sizes = [(700, 256, 4096), (33, 4096, 64), (17, 1621, 128), (8, 1024, 64), (260, 512, 640)]
work = []
for m, k, n in sizes:
    w, x = ops.Q8Weight.quantize(torch.randn(n, k, device="cuda")), ops.quantize_rows(torch.randn(m, k, device="cuda"))
    want = (x.q.double() @ w.rows.q.double().T).float() * x.scale[:, None] * w.rows.scale
    work.append((x, w, want))
torch.cuda.synchronize()
start, wrong = threading.Barrier(16), []
def run(i):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        for j in range(len(work)):
            x, w, want = work[(i + j) % len(work)]
            y = ops.linear_q8(x, w, torch.empty(want.shape, device="cuda"))
            torch.cuda.current_stream().synchronize()
            if not torch.equal(y, want): wrong.append((i, j))
def safely(i):
    try: run(i)
    except Exception as e: wrong.append((i, repr(e)))
threads = [threading.Thread(target=safely, args=(i,)) for i in range(16)]
for t in threads: t.start()
for t in threads: t.join()
assert not wrong, wrong
ops.check_device_errors("cuda:0")
"""


@pytest.mark.parametrize("code", [PLANS, PRODUCTS], ids=["plans", "products"])
def test_first_calls_at_once(code):
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]
