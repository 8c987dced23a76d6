"""gemv_w4 from two host threads: kernels whose shared memory depends on the sizes, first called with a small and a large one at
once, in a process of its own.  Each kernel is called for the first time once in a process, so every kernel takes part."""
import os
import subprocess
import sys

import pytest

CODE = """
import itertools, threading, torch
from rocwmma_b200 import api

m = 4800
def operands(n, rows, group, dtype, zeros):
    groups = -(-n // group)
    z = torch.full((m, groups), 7, dtype=torch.uint8, device="cuda") if zeros else None
    a = torch.full((m, n // 2), 0x19, dtype=torch.uint8, device="cuda")
    return (m, n, rows, a, n // 2, torch.ones(m, groups, device="cuda", dtype=dtype), groups, group,
            torch.ones(rows, n, device="cuda", dtype=dtype), n, torch.zeros(rows, m, device="cuda"), m, 1.0, 0.0), dict(zeros=z, ld_zeros=groups)

failed = []
def call(args, kw, barrier=None):
    if barrier:
        barrier.wait()
    try:
        api.gemv_w4(*args, **kw)
    except Exception as e:
        failed.append((args[1], args[2], args[7], str(args[8].dtype), kw["zeros"] is not None, str(e)))

# a vector that lies in shared memory whole (66 KB against 37), and 8 vectors against 2 in rings (49.7 KB against 25)
sizes = [((2048, 1), (16384, 1)), ((2048, 2), (2048, 8))]
for (small, large), group, dtype, zeros in itertools.product(sizes, (32, 64, 96, 128, 256), (torch.float16, torch.bfloat16), (False, True)):
    calls = [operands(n, rows, group, dtype, zeros) for n, rows in (small, large)]
    torch.cuda.synchronize()
    barrier = threading.Barrier(2)
    threads = [threading.Thread(target=call, args=(*c, barrier)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    call(*calls[1])
    torch.cuda.synchronize()
    if not failed:
        for args, kw in calls:
            n, q = args[1], (9 - 7 if zeros else -7, 1 - 7 if zeros else 1)  # nibbles 9 and 1
            assert bool((args[10] == n // 2 * (q[0] + q[1])).all()), (n, args[2], group, dtype, zeros)
assert api.device_status()[0] == 0
print(len(failed), "failed", failed[:3])
"""


@pytest.mark.gpu
def test_first_calls_of_two_threads():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CODE], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.startswith("0 failed"), done.stdout[-1500:] + done.stderr[-1500:]
