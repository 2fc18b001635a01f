"""The package without its host module, and with a PyTorch that was built without CUDA."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent

WITHOUT = """
import sys
sys.path.insert(0, {root!r})
sys.modules["infer_b200._host_ops"] = None                # what an import of a missing or unfitting module comes to
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if {cpu_torch} and hasattr(torch._C, name):
        delattr(torch._C, name)
from infer_b200 import BlockManager, Sequence, _lib, ops, selftest
manager, seq = BlockManager(4, 256), Sequence(list(range(300)))
manager.allocate(seq)
assert len(seq.block_table) == 2
assert _lib.load().infer_abi_version() == 1 and _lib.load().infer_paged_decode(None, *[None] * 4, 1, 1, 8, 0.1, None, 0, None) == _lib.ERR_NULL
with selftest.variant(wait_limit=10):
    pass
try:
    ops.rotary_embedding(None, None, None, None)
except ImportError as e:
    assert "_host_ops.so" in str(e) and "infer_b200.build" in str(e)
else:
    raise AssertionError("an op of the host module has to say that the module is missing")
print("fine")
"""


def _run(cpu_torch):
    run = subprocess.run([sys.executable, "-c", WITHOUT.format(root=str(ROOT), cpu_torch=cpu_torch)], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0 and "fine" in run.stdout, run.stderr[-3000:]


def test_the_older_ops_and_the_page_allocator_need_no_host_module():
    _run(False)


def test_a_pytorch_without_cuda_imports_the_package():
    _run(True)
