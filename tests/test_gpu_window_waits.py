"""Bounded waits of the windowed decode: a producer that loads nothing and a limit of a few thousand polls.  The kernels set their
status word and return, the host reads it once, and the same call is right again afterwards."""
import ctypes as C

import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import _lib, ops, selftest

pytestmark = pytest.mark.gpu


# few sequences in parts that meet, whole ones in turn, and ranges over all sequences
@pytest.mark.parametrize("lens,window,hkv", [([5200, 900], 4000, 2), ([600] * 40, 100, 8), ([300 + 90 * i for i in range(24)], 1500, 8)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3", "append"])
def test_waits_that_run_out_are_reported_once(kind, lens, window, hkv, monkeypatch):
    monkeypatch.setattr(ops, "_CHECK", False)                          # the status word is read by hand below
    gen = torch.Generator().manual_seed(len(lens))
    need = [-(-n // 256) for n in lens]
    blocks = sum(need)
    perm = torch.randperm(blocks, generator=gen).to(torch.int32)
    bt = torch.zeros(len(lens), max(need), dtype=torch.int32)
    for b, c in enumerate(need):
        bt[b, :c] = perm[sum(need[:b]):sum(need[:b]) + c]
    bt, lens = bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    if kind == "e4m3":
        (k, ks), (v, vs) = (plain64.e4m3_pool(blocks, 256, hkv, gen) for _ in range(2))
        k, v, scales = k.cuda(), v.cuda(), dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    else:
        k, v = (torch.randn(blocks, 256, hkv, 128, generator=gen).bfloat16().cuda() for _ in range(2))
        scales = {}
    q = torch.randn(len(lens), 4 * hkv, 128, generator=gen).bfloat16().cuda()
    new = torch.randn(2, len(lens), hkv, 128, generator=gen).bfloat16().cuda()
    pool, lib, stream = ops.pool_of(k, v, scales.get("k_scale"), scales.get("v_scale")), _lib.load(), torch.cuda.current_stream().cuda_stream
    ws = torch.zeros(pool.decode_workspace_bytes(len(lens), 4 * hkv), dtype=torch.uint8, device="cuda")

    def run():
        if kind == "append":
            return ops.paged_attn_decode_append(q, new[0], new[1], k, v, lens, bt, 0.1, window=window, sinks=4, workspace=ws)
        return ops.paged_attn_decode(q, k, v, lens, bt, 0.1, window=window, sinks=4, workspace=ws, **scales)

    status = lambda: lib.infer_paged_decode_status(C.c_void_p(ws.data_ptr()), stream)
    good = run()
    assert status() == _lib.OK
    with selftest.variant(wait_limit=1 << 22):                          # the routed call by itself changes nothing
        assert bits_equal(run(), good)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    with selftest.variant(wait_limit=4096, stall_producer=1):
        run()
    end.record()
    torch.cuda.synchronize()                                            # returns: nothing hangs
    assert start.elapsed_time(end) < 1000.0
    assert status() == _lib.ERR_DEVICE and status() == _lib.OK           # reported once, then cleared, the tickets with it
    assert bits_equal(run(), good) and status() == _lib.OK


def test_a_status_word_that_is_set_raises_in_the_windowed_call(monkeypatch):
    """Injected from the host: the word of a workspace is written before the call."""
    monkeypatch.setattr(ops, "_CHECK", True)
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, 256, 2, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    q = torch.randn(1, 8, 128, generator=gen).bfloat16().cuda()
    args = (q, k, v, torch.tensor([400], dtype=torch.int32).cuda(), torch.tensor([[0, 1]], dtype=torch.int32).cuda(), 0.1)
    ws = torch.zeros(ops.pool_of(k, v).decode_workspace_bytes(1, 8), dtype=torch.uint8, device="cuda")
    want = ops.paged_attn_decode(*args, window=100, sinks=4, workspace=ws)
    ws[:4].copy_(torch.tensor([0x5AFE0003], dtype=torch.int32).view(torch.uint8))
    with pytest.raises(RuntimeError, match="bounded device-side wait"):
        ops.paged_attn_decode(*args, window=100, sinks=4, workspace=ws)
    assert bits_equal(ops.paged_attn_decode(*args, window=100, sinks=4, workspace=ws), want)
