"""First calls of the windowed prefill from several threads of a fresh process."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CODE = """
import sys, threading
sys.path.insert(0, {root!r})
import torch
from infer_b200 import _lib, ops
gen = torch.Generator().manual_seed(1)
pools = [torch.randn(6, 256, 2, 128, generator=gen).bfloat16().cuda() for _ in range(2)]
q = torch.randn(3, 8, 128, generator=gen).bfloat16().cuda()
cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32).cuda() for n in (3, 1500))
table = torch.arange(6, dtype=torch.int32)[None].cuda()
pool, lib = ops.pool_of(*pools), _lib.load()
streams = [torch.cuda.Stream() for _ in range(8)]
got = [torch.zeros_like(q) for _ in range(9)]
torch.cuda.synchronize()
barrier, failed = threading.Barrier(8), []

def call(out, stream):                       # through the C entry point: ctypes lets the other threads run meanwhile
    return lib.infer_paged_prefill_window(pool.handle, out.data_ptr(), q.data_ptr(), 3, cu_q.data_ptr(), cu_k.data_ptr(),
                                          table.data_ptr(), 6, 1, 3, 1500, 8, 0.1, 1400, 4, stream.cuda_stream)

def first(i):
    torch.cuda.set_device(0)
    barrier.wait()
    rc = call(got[i], streams[i])
    if rc:
        failed.append((i, rc))

threads = [threading.Thread(target=first, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
assert call(got[8], streams[0]) == 0
torch.cuda.synchronize()
again = ops.paged_attn_prefill(q, *pools, cu_q, cu_k, 3, 1500, 0.1, table, window=1400, sinks=4)
assert bool((again != 0).any())
assert all(torch.equal(g, again) for g in got)
print("same bits from every thread")
"""


def test_first_calls_from_eight_threads():
    """Every thread gets the split over clusters that later calls get, whichever of them looks the device's counts up."""
    run = subprocess.run([sys.executable, "-c", CODE.format(root=str(ROOT))], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same bits from every thread" in run.stdout, run.stderr[-3000:]
