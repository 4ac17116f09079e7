"""The attention operators' first calls in a process are recorded ones."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = r"""
import ctypes as C
import numpy as np
import torch
from peregrine_b200 import attention as at, cuda
from tests import attention_ref as ref
from tests.attention_ref import i32

assert cuda.init([0]) == 1
L, rng = cuda.lib(), np.random.default_rng(0)
n, r, H, Kv, D, cap, Tp, keep = 3, 9, 12, 2, 128, 3000, 500, 900
k, v = (ref.cache(rng, n, Kv, cap, D, "bf16") for _ in range(2))
pk, pv = (ref.cache(rng, 1, Kv, Tp, D, "bf16") for _ in range(2))
start = [t.clone() for t in (k, v)]
dk, dv = (torch.zeros((n, Kv, keep, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
pos, acc = i32(np.broadcast_to(np.arange(cap), (n, Kv, cap))), torch.zeros((n, Kv, cap), device="cuda")
dpos, dacc = i32(np.zeros((n, Kv, keep))), torch.zeros((n, Kv, keep), device="cuda")
index, new, length, base = i32(np.zeros((n, Kv, keep))), i32([0] * n), i32([1009, 73, 2001]), i32([1000, 64, 1992])
x = torch.from_numpy(rng.standard_normal((n * r, (H + 2 * Kv) * D), dtype=np.float32)).cuda()
where = i32(np.arange(n * r))
q, out = torch.zeros((n * r, H, D), dtype=torch.bfloat16, device="cuda"), torch.zeros((n * r, H, D), device="cuda")
one, out1 = torch.zeros((n, H, D), dtype=torch.bfloat16, device="cuda") + 0.5, torch.zeros((n, H, D), device="cuda")
own, pre, to = ref.view(k, v, "bf16", pos, acc), ref.view(pk, pv, "bf16"), ref.view(dk, dv, "bf16", dpos, dacc)
need = max(at.attention_workspace(0, n * r, H, own, Tp, r), at.attention_workspace(0, n, H, own, 0, 1))
work = torch.zeros(need, dtype=torch.uint8, device="cuda")
torch.cuda.synchronize()


def calls():
    at.qk_norm_rope(0, q.data_ptr(), x.data_ptr(), n * r, H, own, base.data_ptr(), where.data_ptr(), 1e4, rows_per_seq=r)
    at.attention(0, out.data_ptr(), q.data_ptr(), n * r, H, own, base.data_ptr(), 0.1, work.data_ptr(), need, rows_per_seq=r,
                 prefix=pre, prefix_len=Tp)
    at.attention(0, out1.data_ptr(), one.data_ptr(), n, H, own, base.data_ptr(), 0.1, work.data_ptr(), need)
    at.kv_evict(0, to, own, length.data_ptr(), new.data_ptr(), index.data_ptr(), keep, 4, 50)


h, got = C.c_void_p(), []
assert L.coli_cuda_graph_begin(0) == 1
calls()
assert L.coli_cuda_graph_end(0, C.byref(h)) == 1
for run in (lambda: L.coli_cuda_graph_launch(h), calls):
    k.copy_(start[0]), v.copy_(start[1]), acc.zero_()
    torch.cuda.synchronize()
    run()
    ref.done()
    got.append([t.clone() for t in (q, k, v, acc, out, out1, dk, dv, dpos, dacc, index, new)])
for a, b in zip(*got):
    assert torch.equal(a, b)
assert float(got[0][4].abs().sum()) > 0 and new.cpu().tolist() == [900, 73, 900]
assert cuda.last_device_error(0) == 0
L.coli_cuda_graph_free(h)
cuda.shutdown()
print("recorded")
"""


def test_the_first_calls_of_a_process_may_be_recorded_ones():
    done = subprocess.run([sys.executable, "-c", SCRIPT], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and "recorded" in done.stdout, done.stdout + done.stderr
