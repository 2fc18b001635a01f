"""Decode over e4m3 pools with queries of any size: the products run on f16, so a row is scaled by a power of two where it has to be."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _case(hq, hkv, seed):
    gen = torch.Generator().manual_seed(seed)
    lens, tables = [700, 1, 0, 300], [[3, 1, 6], [5], [], [0, 2]]
    (k, ks), (v, vs) = (plain64.e4m3_pool(7, 256, hkv, gen, 0.5) for _ in range(2))
    return dict(q=torch.randn(4, hq, 128, generator=gen).bfloat16().cuda(), k=k.cuda(), v=v.cuda(), ks=ks.cuda(), vs=vs.cuda(),
                lens=torch.tensor(lens, dtype=torch.int32).cuda(), tables=tables,
                bt=torch.tensor([t + [-1] * (3 - len(t)) for t in tables], dtype=torch.int32).cuda())


def _run(c, window, sinks, scale):
    return ops.paged_attn_decode(c["q"], c["k"], c["v"], c["lens"], c["bt"], scale, k_scale=c["ks"], v_scale=c["vs"], window=window,
                                 sinks=sinks)


def _check(c, got, window, sinks, scale, heads=slice(None)):
    for b, n in enumerate(c["lens"].tolist()):
        if n:
            k, v = (plain64.values(c[x], c[x + "s"], c["tables"][b], n) for x in "kv")
            seen = plain64.visible(n, torch.tensor([n - 1], device="cuda"), window, sinks)
            # f16 probabilities: half a step of theirs, 2^-25 in absolute terms below 2^-14.  Queries: exact, or within 2^-22 of
            # the row's largest value, 2^-22 max|q| sum |k| in a score, twice over (its own and the sum's)
            want, bound = plain64.attention(c["q"][b:b + 1], k, v, seen, scale, plain64.E_F16, 2.0 ** -25)
            group = c["q"].shape[1] // k.shape[1]
            top = c["q"][b].double().abs().amax(-1) * k.abs().sum(-1).amax(0).repeat_interleave(group) * scale * 2.0 ** -22
            bound = bound + 2 * top[None, :, None] * v.abs().amax() * (1 + 2.0 ** -8)
            plain64.check(got[b:b + 1, heads], want[:, heads], bound[:, heads], f"sequence {b} ({n} keys)")


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4), (5000, 0)])
@pytest.mark.parametrize("hq,hkv", [(3, 1), (16, 2), (12, 4), (8, 8)])
@pytest.mark.parametrize("amplitude", [2.0 ** -124, 2.0 ** -100, 1e-6, 2.0 ** -4, 1.0, 2.0 ** 14, 65520.0, 1e6, 2.0 ** 100, 2.0 ** 124])
def test_amplitudes(amplitude, hq, hkv, window, sinks):
    c = _case(hq, hkv, 3)
    c["q"] = (c["q"].float() * amplitude).bfloat16()
    _check(c, _run(c, window, sinks, SCALE / amplitude), window, sinks, SCALE / amplitude)


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4)])
def test_heads_of_one_group_far_apart(window, sinks):
    """Every head of a group with a size of its own, a row of zeros, and large and small values within one row."""
    c = _case(16, 2, 4)
    for h, a in enumerate([1.0, 2.0 ** 20, 2.0 ** -30, 0.0, 2.0 ** 60, 1.0, 2.0 ** -100, 2.0 ** 15]):
        c["q"][:, h] = (c["q"][:, h].float() * a).bfloat16()
        c["q"][:, 8 + h] = (c["q"][:, 8 + h].float() * a).bfloat16()
    c["q"][:, 5, 7] = 65536.0
    c["q"][:, 13, 9] = -2.0 ** 40
    # a score of 2^60 and more leaves one key: the larger heads are checked where the scale brings them into range
    for h, scale in ((0, SCALE), (1, SCALE * 2.0 ** -20), (2, SCALE * 2.0 ** 30), (3, SCALE), (4, SCALE * 2.0 ** -60),
                     (5, SCALE * 2.0 ** -14), (6, SCALE * 2.0 ** 100), (7, SCALE * 2.0 ** -15), (13, SCALE * 2.0 ** -38)):
        heads = [h] if h > 7 or h == 5 else [h, 8 + h]
        _check(c, _run(c, window, sinks, scale), window, sinks, scale, heads)


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4)])
def test_rows_that_are_not_finite_stay_their_own(window, sinks):
    c = _case(16, 2, 5)
    want = _run(c, window, sinks, SCALE)
    live = c["lens"] > 0
    c["q"][0, 3, 17], c["q"][3, 9, 0] = float("nan"), float("inf")
    got = _run(c, window, sinks, SCALE)
    assert torch.isnan(got[0, 3]).all() and torch.isnan(got[3, 9]).all()
    got[0, 3], got[3, 9] = want[0, 3], want[3, 9]
    assert bits_equal(got[live], want[live])


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4)])
@pytest.mark.parametrize("amplitude", [2.0 ** -124, 2.0 ** -118, 2.0 ** -112, 1e-30, 1.0, 2.0 ** 118, 2.0 ** 125])
def test_prefill_amplitudes(amplitude, window, sinks, rows):
    """The split of a query into two e4m3 values over all of bf16's range: exact for values down to 2^-10 of the row's largest,
    off by 2^-16 of the largest below; rows under 2^-119 are lifted less, by 2^126, and off by 2^-9 (a cut, no rounding) in those units."""
    gen = torch.Generator().manual_seed(rows)
    (k, ks), (v, vs) = (plain64.e4m3_pool(3, 256, 2, gen, 0.5) for _ in range(2))
    k, v, ks, vs = k.cuda(), v.cuda(), ks.cuda(), vs.cuda()
    q = (torch.randn(rows, 8, 128, generator=gen).clamp(-4, 4) * amplitude).bfloat16().cuda()
    q[1, 3] = 0.0
    assert torch.isfinite(q).all()
    n, scale = 700, SCALE / amplitude
    cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32).cuda() for x in (rows, n))
    got = ops.paged_attn_prefill(q, k, v, cu_q, cu_k, rows, n, scale, torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda(), k_scale=ks,
                                 v_scale=vs, window=window, sinks=sinks)
    kk, vv = plain64.values(k, ks, [2, 0, 1], n), plain64.values(v, vs, [2, 0, 1], n)
    seen = plain64.visible(n, torch.arange(n - rows, n, device="cuda"), window, sinks)
    want, bound = plain64.attention(q, kk, vv, seen, scale, plain64.E_F16)
    # that in every product of a score, twice over (its own and the sum's), and the f16 probabilities' absolute step
    off = torch.maximum(q.double().abs().amax(-1) * 2.0 ** -16, torch.tensor(2.0 ** -135, dtype=torch.float64, device="cuda"))
    top = off * kk.abs().sum(-1).amax(0).repeat_interleave(4)[None] * scale
    bound = bound + (2 * top[..., None] * (1 + 2.0 ** -8) + 2.0 ** -31 * n) * vv.abs().amax()
    plain64.check(got, want, bound)
