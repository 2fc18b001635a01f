"""Rotary positions in general form, with and without the append (``rotary_append``, ``rotary_embedding``)."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops
from infer_b200.rotary import rotary_frequencies

pytestmark = pytest.mark.gpu


def _rows(t, hq, hkv, gen):
    """q, k, v as column slices of one fused row, as a model's projection leaves them."""
    qkv = torch.randn(t, (hq + 2 * hkv) * 128, generator=gen).bfloat16().cuda()
    return [x.view(t, -1, 128) for x in qkv.split([hq * 128, hkv * 128, hkv * 128], dim=1)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [16, 32, 48, 64, 96, 112, 128])
@pytest.mark.parametrize("t,hq,hkv", [(1, 1, 1), (5, 7, 1), (33, 16, 8), (300, 30, 3)])
def test_rotary_append(t, hq, hkv, rot, interleaved):
    gen = torch.Generator().manual_seed(rot + t)
    q, k, v = _rows(t, hq, hkv, gen)
    positions = torch.randint(0, 9000, (t,), generator=gen).cuda()
    inv_freq, _ = rotary_frequencies(rot, device="cuda")
    slots = torch.randperm(3 * 256, generator=gen)[:t].to(torch.int32)
    if t > 4:
        slots[2], slots[3] = -1, 3 * 256                                          # rows that are not stored
    pools = [torch.full((3, 256, hkv, 128), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    got = ops.rotary_append(q, k, v, positions, inv_freq, *pools, slots.cuda(), interleaved=interleaved)
    want, bound = plain64.rotary(q, positions, inv_freq, interleaved, 1.0)
    assert got.is_contiguous()
    plain64.check(got, want, bound, "q")
    kw, kb = plain64.rotary(k, positions, inv_freq, interleaved, 1.0)
    stored = (slots >= 0) & (slots < 3 * 256)
    flat = [p.view(-1, hkv, 128) for p in pools]
    at = slots[stored].long().cuda()
    plain64.check(flat[0][at], kw[stored.cuda()], kb[stored.cuda()], "k")
    assert bits_equal(flat[1][at], v[stored.cuda()])
    # dims behind rot_dim keep their bits, other slots keep what they held
    assert bits_equal(got[..., rot:], q[..., rot:]) and bits_equal(flat[0][at][..., rot:], k[stored.cuda()][..., rot:])
    rest = torch.ones(3 * 256, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((flat[0][rest] == 5.0).all()) and bool((flat[1][rest] == 5.0).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_rotary_far_positions_and_scaling(scaling, interleaved):
    """Positions up to 2^40: the angle keeps its digits (64-bit products lose 2^-53 of up to 2^40 / 2 pi turns: 2^-15 of a
    turn at the very end, below bf16's step but above the bound for sincos, so the bound is widened by it there)."""
    gen = torch.Generator().manual_seed(3)
    positions = torch.tensor([0, 1, 2, 4095, 65537, 999999, 2 ** 31 + 7, 2 ** 40 - 1, -5])
    q, k, _ = _rows(len(positions), 4, 2, gen)
    inv_freq, factor = rotary_frequencies(128, 10000.0, scaling, 4.0, 4096, device="cuda")
    got = ops.rotary_embedding(q, k, positions.cuda(), inv_freq, interleaved=interleaved, attention_factor=factor)
    for g, x in zip(got, (q, k)):
        want, bound = plain64.rotary(x, positions.cuda(), inv_freq, interleaved, factor)
        angle = positions.double().abs().cuda() * 2.0 ** -51          # two roundings of the angle on either side
        plain64.check(g, want, bound + angle[:, None, None] * factor * x.double().abs().amax(-1, keepdim=True) * 2, str(scaling))


def test_rotary_in_place_and_through_an_8_bit_cache():
    gen = torch.Generator().manual_seed(8)
    q, k, v = _rows(40, 8, 2, gen)
    positions = torch.arange(100, 140, device="cuda")
    inv_freq, _ = rotary_frequencies(64, device="cuda")
    want = ops.rotary_embedding(q, k, positions, inv_freq)
    q2, k2 = q.clone(), k.clone()
    got = ops.rotary_embedding(q2, k2, positions, inv_freq, q_out=q2, k_out=k2)
    assert got[0] is q2 and got[1] is k2 and bits_equal(q2, want[0]) and bits_equal(k2, want[1])
    # the same rows as rotary_append stores
    kc, vc = (torch.zeros(1, 256, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    got = ops.rotary_append(q, k, v, positions, inv_freq, kc, vc, slots, q_out=q)             # q is a column slice, written in place
    assert got is q and bits_equal(q.contiguous(), want[0]) and bits_equal(kc[0, :40], want[1])
    k8, v8 = (torch.zeros(1, 256, 2, 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(1, 2, device="cuda") for _ in range(2))
    with pytest.raises(ValueError):
        ops.rotary_append(q, k, v, positions, inv_freq, k8, v8, slots)                        # bf16 pools alone
    ops.store_kvcache(want[1], v.contiguous(), k8, v8, slots, ks, vs)
    back = ops.load_kvcache(k8, v8, slots, k_scale=ks, v_scale=vs)[0]
    x = want[1].double()
    assert bool(((back.double() - x).abs() <= (2.0 ** -4 + 2.0 ** -7) * x.abs() + 2.0 ** -10 * ks[0][:, None].double()).all())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_on_rows_at_sixteen_bytes(interleaved):
    """Columns and pitches that are multiples of 16 bytes but not of 32 take the narrow accesses, with the same result."""
    gen = torch.Generator().manual_seed(12)
    hq, hkv, t = 6, 2, 50
    wide = torch.randn(t, (hq + 2 * hkv) * 128 + 24, generator=gen).bfloat16().cuda()
    q, k, v = (x.view(t, -1, 128) for x in wide[:, 8:8 + (hq + 2 * hkv) * 128].split([hq * 128, hkv * 128, hkv * 128], dim=1))
    assert q.data_ptr() % 32 == 16 and q.stride(0) % 16 == 8
    positions = torch.arange(t, device="cuda") * 37
    inv_freq, _ = rotary_frequencies(96, device="cuda")
    want = ops.rotary_embedding(q.contiguous(), k.contiguous(), positions, inv_freq, interleaved=interleaved)
    got = ops.rotary_embedding(q, k, positions, inv_freq, interleaved=interleaved)
    assert bits_equal(got[0], want[0]) and bits_equal(got[1], want[1])
    kc, vc = (torch.zeros(1, 256, hkv, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(t, dtype=torch.int32, device="cuda")
    assert bits_equal(ops.rotary_append(q, k, v, positions, inv_freq, kc, vc, slots, interleaved=interleaved), want[0])
    assert bits_equal(kc[0, :t], want[1]) and bits_equal(vc[0, :t], v)


def test_rotary_in_a_graph():
    gen = torch.Generator().manual_seed(9)
    q, k, v = _rows(64, 16, 8, gen)
    positions = torch.arange(64, device="cuda")
    inv_freq, _ = rotary_frequencies(128, device="cuda")
    kc, vc = (torch.zeros(2, 256, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    slots = torch.arange(64, dtype=torch.int32, device="cuda")
    ops.rotary_append(q, k, v, positions, inv_freq, kc, vc, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rotary_append(q, k, v, positions, inv_freq, kc, vc, slots)
    positions += 1000
    slots += 70
    graph.replay()
    torch.cuda.synchronize()
    want = ops.rotary_embedding(q, k, positions, inv_freq)
    assert bits_equal(got, want[0]) and bits_equal(kc.view(-1, 8, 128)[70:134], want[1])


def test_rotary_refusals():
    gen = torch.Generator().manual_seed(1)
    q, k, v = _rows(4, 4, 2, gen)
    pos = torch.arange(4, device="cuda")
    inv_freq, _ = rotary_frequencies(64, device="cuda")
    kc = torch.zeros(1, 256, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    call = lambda **kw: ops.rotary_append(*[kw.get(n, d) for n, d in (
        ("q", q), ("k", k), ("v", v), ("positions", pos), ("inv_freq", inv_freq), ("k_cache", kc), ("v_cache", kc), ("slots", slots))])
    for bad, match in ((dict(q=q.float()), "q must be"), (dict(k=k[:3]), "rows"), (dict(v=v[:, :1]), "heads"),
                       (dict(positions=pos.int()), "positions"), (dict(positions=pos[:3]), "positions"),
                       (dict(inv_freq=inv_freq.float()), "inv_freq"), (dict(inv_freq=inv_freq[:5]), "geometry"),
                       (dict(inv_freq=torch.ones(72, dtype=torch.float64, device="cuda")), "geometry"),
                       (dict(slots=slots.long()), "slot_mapping"), (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "heads"),
                       (dict(q=q.cpu()), "q must be")):
        with pytest.raises(RuntimeError, match=match):
            call(**bad)
