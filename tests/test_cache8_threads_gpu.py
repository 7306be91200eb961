"""First calls of a process, made by two threads at once."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import threading
import torch
from swifttransformer_b200 import ops

def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")

def case(kind, form, act, d, n):
    # one request of n keys: few of them take few warps or a small tile, many take more shared memory
    pool, scales = ops.cache8_pool(-(-n // 16), 1, 1, 16, d, form, "cuda")
    pool.view(torch.int8).random_(0, 60)
    scales.fill_(0.01)
    q = torch.randn((1, d), device="cuda").to(act)
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda").view(1, -1)
    args = (ints([n - 1]), ints([0]), ints([0]), table, 1, d ** -0.5)
    if kind == "single":
        return lambda out: ops.attention_cache8_single(q, pool, scales, 0, out, None, 1, *args, max_kv=n), q
    plan = ops.portion_plan([1], [n - 1], 1, 1)
    return lambda out: ops.attention_cache8_tiles(q, pool, scales, 0, out, plan, args[0], args[2], table, 1, d ** -0.5), q

bad = []
for act in (torch.bfloat16, torch.float32):
    for form in (torch.int8, torch.float8_e4m3fn):
        # two calls that reach the same kernel with different sizes of it
        pairs = [(("single", d, 300), ("single", d, 9000)) for d in (32, 64, 80, 96, 128)]
        pairs += [(("portion", a, 40), ("portion", b, 40)) for a, b in ((13, 61), (65, 127), (129, 255))]
        for sizes in pairs:
            calls = [case(kind, form, act, d, n) for kind, d, n in sizes]
            ready = threading.Barrier(2)
            torch.cuda.synchronize()
            def go(i):
                out = torch.empty_like(calls[i][1])
                ready.wait()
                try:
                    calls[i][0](out)
                except Exception as e:
                    bad.append((str(act), str(form), sizes[i], str(e)))
            threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
            for t in threads:
                t.start()
            for t in threads:
                t.join()
            torch.cuda.synchronize()
assert not bad, bad
print("ok")
"""


def test_first_calls_of_two_threads():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout[-2000:] + r.stderr[-2000:]
