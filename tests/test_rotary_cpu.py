"""Rotary frequencies, and what the C entry points refuse before any CUDA call."""
import ctypes as C
import math

import pytest
import torch

from infer_b200 import _lib
from infer_b200.rotary import rotary_frequencies


def test_plain_linear_and_ntk():
    f, a = rotary_frequencies(64, 500000.0)
    assert f.dtype == torch.float64 and a == 1.0
    assert torch.allclose(f, torch.tensor([500000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-15, atol=0)
    g, a = rotary_frequencies(64, 500000.0, "linear", 8.0)
    assert a == 1.0 and torch.equal(g, f / 8)
    h, a = rotary_frequencies(64, 500000.0, "ntk", 8.0)
    assert a == 1.0 and h[0] == f[0] == 1.0
    assert math.isclose(h[-1].item(), f[-1].item() / 8, rel_tol=1e-12)


def test_yarn_keeps_fast_pairs_and_slows_slow_ones():
    f, _ = rotary_frequencies(128)
    g, a = rotary_frequencies(128, scaling="yarn", factor=16.0, original_max_position=4096)
    ratio = g / f
    turns = 4096 * f / (2 * math.pi)
    assert math.isclose(a, 1 + 0.1 * math.log(16))
    assert bool((ratio[turns > 40] == 1).all()) and torch.allclose(ratio[turns < 0.9], torch.tensor(1 / 16, dtype=torch.float64))
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all())


@pytest.mark.parametrize("kw", [dict(rot_dim=20), dict(rot_dim=144), dict(rot_dim=0), dict(rot_dim=64, base=1.0),
                                dict(rot_dim=64, scaling="linear", factor=0.5), dict(rot_dim=64, scaling="cubic"),
                                dict(rot_dim=64, scaling="yarn", factor=2.0),
                                dict(rot_dim=64, scaling="yarn", factor=2.0, original_max_position=4096, fast_turns=1.0)])
def test_refusals(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)


def test_c_entry_points_check_arguments_first():
    lib = _lib.load()
    buf = C.create_string_buffer(4096 + 16)
    p = C.c_void_p((C.addressof(buf) + 15) // 16 * 16)
    odd = C.c_void_p(p.value + 2)
    embed = lambda q_out=p, k_out=p, so=256, sk=128, q=p, k=p, sq=256, pk=128, pos=p, f=p, rot=64, n=1, hq=2, hkv=1: \
        lib.infer_rotary_embed(q_out, k_out, so, sk, q, k, sq, pk, pos, f, rot, 0, 1.0, n, hq, hkv, None)
    assert embed(n=0) == _lib.OK
    assert embed(n=0, q=None) == _lib.OK                          # nothing to do: no pointer is looked at
    for bad in (dict(rot=0), dict(rot=24), dict(rot=130), dict(rot=144), dict(n=-1), dict(hq=0), dict(hkv=0)):
        assert embed(**bad) == _lib.ERR_GEOMETRY, bad
    for bad in (dict(q=None), dict(k_out=None), dict(pos=None), dict(f=None)):
        assert embed(**bad) == _lib.ERR_NULL, bad
    for bad in (dict(so=128), dict(sk=120), dict(sq=8), dict(pk=0)):
        assert embed(**bad) == _lib.ERR_STRIDE, bad
    for bad in (dict(q=odd), dict(k=odd), dict(q_out=odd), dict(k_out=odd), dict(so=260), dict(pk=129)):
        assert embed(**bad) == _lib.ERR_ALIGN, bad
    assert lib.infer_rotary_append(None, p, 256, p, p, p, 256, 128, 128, p, p, 64, 0, 1.0, p, 1, 2, None) == _lib.ERR_NULL
    assert lib.infer_kv_load(None, p, p, 128, 128, p, 1, None) == _lib.ERR_NULL


def test_window_entry_points_check_window_and_scale_first():
    lib = _lib.load()
    buf = C.create_string_buffer(64)
    p = C.cast(buf, C.c_void_p)
    for window, sinks, scale in ((0, 0, 0.1), (-1, 0, 0.1), (5, -1, 0.1), (5, 0, 0.0), (5, 0, -0.1), (5, 0, float("nan")),
                                 (5, 0, float("inf"))):
        assert lib.infer_paged_decode_window(None, p, p, p, p, 4, 1, 8, scale, window, sinks, None, 0, None) == _lib.ERR_GEOMETRY
        assert lib.infer_paged_decode_append_window(None, p, p, p, p, 128, 128, p, p, 4, 1, 8, scale, window, sinks, None, 0,
                                                    None) == _lib.ERR_GEOMETRY
    assert lib.infer_paged_decode_window(None, p, p, p, p, 4, 1, 8, 0.1, 5, 0, None, 0, None) == _lib.ERR_NULL


def _ramp(rot_dim, base, context, fast, slow):
    """How far pair i lies from the pair that makes ``fast`` turns over the context (0) to the one that makes ``slow`` (1), pairs
    counted from the fastest, both ends moved outwards to whole pairs and the first to pair 0 at least."""
    out = []
    for i in range(rot_dim // 2):
        first = max(0, math.floor(rot_dim / 2 * math.log(context / (2 * math.pi * fast), base)))
        last = math.ceil(rot_dim / 2 * math.log(context / (2 * math.pi * slow), base))
        out.append(min(1.0, max(0.0, (i - first) / (last - first))))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("rot_dim", [16, 32, 64, 96, 128])
@pytest.mark.parametrize("context", [300, 4096, 65536, 131072, 262144, 2 ** 22])
@pytest.mark.parametrize("factor", [1.0, 4.0, 32.0])
def test_yarn_at_contexts_short_and_long(context, rot_dim, base, factor):
    """Pairs above fast_turns keep their frequency, pairs below slow_turns are divided by the factor, the ramp is between, also
    where it ends behind the last pair: base 10000, 128 dims, 131072 positions, the slowest pair makes 2.41 turns."""
    f, _ = rotary_frequencies(rot_dim, base)
    g, _ = rotary_frequencies(rot_dim, base, "yarn", factor, context)
    turns, ratio = context * f / (2 * math.pi), g / f
    assert torch.allclose(ratio[turns > 32], torch.ones(1, dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.allclose(ratio[turns < 1], torch.tensor([1 / factor], dtype=torch.float64), rtol=1e-14, atol=0)
    want = 1 - (1 - 1 / factor) * _ramp(rot_dim, base, context, 32.0, 1.0)
    assert torch.allclose(ratio, want, rtol=1e-12, atol=0)
    if factor > 1:
        assert bool((ratio[turns > 1 + 1e-9] > 1 / factor).all())


def test_yarn_where_the_slowest_pair_is_on_the_ramp():
    for rot_dim, context, ratio in ((128, 65536, 0.31), (128, 131072, 0.46)):
        f, g = rotary_frequencies(rot_dim)[0], rotary_frequencies(rot_dim, scaling="yarn", factor=4.0, original_max_position=context)[0]
        assert abs((g / f)[-1].item() - ratio) < 0.005


@pytest.mark.parametrize("context", [1, 3, 6])
def test_yarn_of_a_context_of_less_than_a_turn(context):
    """No pair makes a turn: all are divided."""
    f, g = rotary_frequencies(64)[0], rotary_frequencies(64, scaling="yarn", factor=8.0, original_max_position=context)[0]
    assert torch.allclose(g, f / 8, rtol=1e-14, atol=0)


def test_prefill_window_entry_points_check_arguments_first():
    lib = _lib.load()
    buf = C.create_string_buffer(64)
    p = C.cast(buf, C.c_void_p)
    for window, sinks, scale, want in ((-1, 0, 0.1, _lib.ERR_GEOMETRY), (5, -1, 0.1, _lib.ERR_GEOMETRY), (5, 0, 0.0, _lib.ERR_GEOMETRY),
                                       (5, 0, float("nan"), _lib.ERR_GEOMETRY), (5, 0, float("inf"), _lib.ERR_GEOMETRY),
                                       (5, 4, 0.1, _lib.ERR_NULL), (0, 0, 0.1, _lib.ERR_NULL)):
        assert lib.infer_paged_prefill_window(None, p, p, 1, p, p, p, 4, 1, 1, 1, 8, scale, window, sinks, None) == want
        assert lib.infer_paged_prefill_window_columns(None, p, p, 1, p, p, p, 4, 3, 1, 1, 1, 8, scale, window, sinks, None) == want
