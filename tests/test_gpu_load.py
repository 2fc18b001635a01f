"""Rows of the page pools read back (``load_kvcache``)."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops

pytestmark = pytest.mark.gpu


def _pool(kind, num_blocks, block_size, hkv, gen):
    if kind == "bf16":
        mk = lambda: torch.randn(num_blocks, block_size, hkv, 128, generator=gen).bfloat16().cuda()
        return mk(), mk(), None, None
    (k, ks), (v, vs) = (plain64.e4m3_pool(num_blocks, block_size, hkv, gen) for _ in range(2))
    return k.cuda(), v.cuda(), ks.cuda(), vs.cuda()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("hkv", [1, 3, 8])
@pytest.mark.parametrize("n", [0, 1, 2, 17, 301, 2050])
def test_load(kind, hkv, n):
    gen = torch.Generator().manual_seed(100 * hkv + n)
    k, v, ks, vs = _pool(kind, 9, 256, hkv, gen)
    slots = torch.randint(0, 9 * 256, (n,), generator=gen).to(torch.int32)          # repeats among them
    if n > 4:
        slots[1], slots[3], slots[4] = -1, 9 * 256, 9 * 256 - 1                     # padding, past the pool, the last slot
    got = ops.load_kvcache(k, v, slots.cuda(), k_scale=ks, v_scale=vs)
    inside = (slots >= 0) & (slots < 9 * 256)
    idx = torch.where(inside, slots, 0).long().cuda()
    for g, cache, scale in ((got[0], k, ks), (got[1], v, vs)):
        want = cache.view(-1, hkv, 128)[idx]
        if scale is not None:
            # a product of 32-bit numbers rounded once: 4 by 24 bits, exact in 64
            want = want.view(torch.float8_e4m3fn).double() * scale.double()[idx // 256][..., None]
            want = want.float().bfloat16()
        want = torch.where(inside.cuda()[:, None, None], want, torch.zeros_like(want))
        assert g.shape == (n, hkv, 128) and torch.equal(g, want)


def test_load_into_slices_of_a_wider_row_and_large_pages():
    gen = torch.Generator().manual_seed(5)
    k, v, ks, vs = _pool("e4m3", 3, 768, 2, gen)
    slots = torch.randperm(3 * 768, generator=gen)[:100].to(torch.int32).cuda()
    want = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    wide = torch.full((100, 3 * 256), 7.0, dtype=torch.bfloat16, device="cuda")
    k_out, v_out = wide[:, 256:512].view(100, 2, 128), wide[:, 512:].view(100, 2, 128)
    got = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs, k_out=k_out, v_out=v_out)
    assert got[0] is k_out and torch.equal(k_out, want[0]) and torch.equal(v_out, want[1])
    assert bool((wide[:, :256] == 7.0).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_load_into_rows_at_sixteen_bytes(kind):
    gen = torch.Generator().manual_seed(13)
    k, v, ks, vs = _pool(kind, 3, 256, 2, gen)
    slots = torch.randperm(3 * 256, generator=gen)[:77].to(torch.int32).cuda()
    want = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    wide = torch.zeros(77, 2 * 256 + 24, dtype=torch.bfloat16, device="cuda")
    k_out, v_out = wide[:, 8:264].view(77, 2, 128), wide[:, 264:520].view(77, 2, 128)
    assert k_out.data_ptr() % 32 == 16
    ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs, k_out=k_out, v_out=v_out)
    assert torch.equal(k_out, want[0]) and torch.equal(v_out, want[1])


def test_store_then_load_round_trip():
    """bf16: the stored bits; e4m3: within half a step of the format (2^-4) of the row, or of its subnormals."""
    gen = torch.Generator().manual_seed(6)
    n, hkv = 700, 4
    key, value = (torch.randn(n, hkv, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    slots = torch.randperm(4 * 256, generator=gen)[:n].to(torch.int32).cuda()
    k, v = (torch.zeros(4, 256, hkv, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.store_kvcache(key, value, k, v, slots)
    got = ops.load_kvcache(k, v, slots)
    assert bits_equal(got[0], key) and bits_equal(got[1], value)
    k, v = (torch.zeros(4, 256, hkv, 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(4, hkv, device="cuda") for _ in range(2))
    ops.store_kvcache(key, value, k, v, slots, ks, vs)
    got = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    for g, x, s in ((got[0], key, ks), (got[1], value, vs)):
        step = s[slots.long() // 256][..., None].double()
        bound = (2.0 ** -4 * x.double().abs() + 2.0 ** -10 * step) * (1 + 2.0 ** -8) + 2.0 ** -8 * x.double().abs()
        assert bool(((g.double() - x.double()).abs() <= bound).all())


def test_load_in_a_graph_and_on_another_stream():
    gen = torch.Generator().manual_seed(7)
    k, v, ks, vs = _pool("e4m3", 4, 256, 8, gen)
    slots = torch.arange(64, dtype=torch.int32, device="cuda")
    ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    slots += 300
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_load_refusals():
    k = torch.zeros(2, 256, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="slot_mapping"):
        ops.load_kvcache(k, k, slots.long())
    with pytest.raises(RuntimeError, match="slot_mapping"):
        ops.load_kvcache(k, k, slots.cpu())
    with pytest.raises(RuntimeError, match="k_out"):
        ops.load_kvcache(k, k, slots, k_out=torch.zeros(2, 2, 128, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="v_out"):
        ops.load_kvcache(k, k, slots, v_out=torch.zeros(3, 2, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="aligned"):
        ops.load_kvcache(k, k, slots, k_out=torch.zeros(3 * 256 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(3, 2, 128))
    with pytest.raises(ValueError):
        ops.load_kvcache(k.view(torch.uint8)[..., :128].contiguous(), k.view(torch.uint8)[..., :128].contiguous(), slots)


def test_pools_released_and_made_again():
    """Handles that were given back are not used again, and pools of another type at the same addresses are others."""
    cache = torch.randn(2, 2, 256, 2, 128, device="cuda").bfloat16()
    slots = torch.tensor([3, 400, 3], dtype=torch.int32, device="cuda")
    for _ in range(2):
        k, v = ops.load_kvcache(cache[0], cache[1], slots)
        assert bits_equal(k, cache[0].view(-1, 2, 128)[slots.long()]) and bits_equal(v, cache[1].view(-1, 2, 128)[slots.long()])
        ops.release_pools()
    half = cache.view(torch.uint8).view(2, 2, 512, 2, 128)           # the same memory as e4m3 pages of 512 rows
    with pytest.raises(ValueError):
        ops.load_kvcache(half[0], half[1], slots)
    one = torch.ones(2, 2, device="cuda")
    k, _ = ops.load_kvcache(half[0], half[1], slots, one, one)
    want = half[0].view(torch.float8_e4m3fn).view(-1, 2, 128)[slots.long()].float().bfloat16()
    assert torch.equal(k.float().nan_to_num(7.0), want.float().nan_to_num(7.0))
    k, _ = ops.load_kvcache(cache[0], cache[1], slots)
    assert bits_equal(k, cache[0].view(-1, 2, 128)[slots.long()])
