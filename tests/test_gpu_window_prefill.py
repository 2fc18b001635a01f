"""Paged prefill over a sliding window and sinks (bf16 and e4m3 pools), and over e4m3 pools without a window."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops, selftest

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _case(kind, chunks, hq, hkv, seed, block_size=256, spread=0.5, poison=None, extra=0, amplitude=1.0):
    """``chunks``: (keys, queries) per sequence.  ``poison`` (window, sinks): every slot that no query may see holds NaN."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // block_size) for n, _ in chunks]
    blocks = sum(need) + 2
    perm = torch.randperm(blocks, generator=gen).tolist()
    tables = [[perm.pop() for _ in range(c)] for c in need]
    total = sum(m for _, m in chunks)
    q = (torch.randn(total + extra, hq, 128, generator=gen) * amplitude).bfloat16()
    if kind == "bf16":
        k, v = (torch.randn(blocks, block_size, hkv, 128, generator=gen).bfloat16() for _ in range(2))
        ks = vs = None
    else:
        (k, ks), (v, vs) = (plain64.e4m3_pool(blocks, block_size, hkv, gen, spread) for _ in range(2))
    if poison is not None:
        window, sinks = poison
        live = torch.zeros(blocks * block_size, dtype=torch.bool)
        for (n, m), t in zip(chunks, tables):
            if m:
                seen = plain64.visible(n, torch.arange(n - m, n), window, sinks).any(0)
                at = torch.arange(n)[seen]
                live[torch.tensor(t + [0])[at // block_size] * block_size + at % block_size] = True
        for c in (k, v):
            c.view(-1, hkv, 128)[~live] = float("nan") if kind == "bf16" else 0x7f
    width = max(need) + 1
    bt = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32)
    cu = lambda x: torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32).cuda()
    cuda = lambda x: None if x is None else x.cuda()
    return dict(q=q.cuda(), k=k.cuda(), v=v.cuda(), ks=cuda(ks), vs=cuda(vs), bt=bt.cuda(), tables=tables, chunks=chunks,
                cu_q=cu([m for _, m in chunks]), cu_k=cu([n for n, _ in chunks]), max_q=max(m for _, m in chunks),
                max_k=max(n for n, _ in chunks))


def _run(c, window=None, sinks=0, scale=SCALE, **kw):
    return ops.paged_attn_prefill(c["q"], c["k"], c["v"], c["cu_q"], c["cu_k"], c["max_q"], c["max_k"], scale, c["bt"],
                                  k_scale=c["ks"], v_scale=c["vs"], window=window, sinks=sinks, **kw)


def _check(c, got, window=None, sinks=0, scale=SCALE, what=""):
    at = 0
    for b, (n, m) in enumerate(c["chunks"]):
        if m:
            k, v = (plain64.values(c[x], c[x + "s"], c["tables"][b], n) for x in "kv")
            seen = plain64.visible(n, torch.arange(n - m, n, device="cuda"), window, sinks)
            rows = c["q"][at:at + m]
            if c["ks"] is None:
                want, bound = plain64.attention(rows, k, v, seen, scale, plain64.E_BF16)
            else:
                # f16 probabilities: relative half steps, and in absolute terms 2^-25 below 2^-14 in units of
                # 2^-6 of the reference and of the largest V scale met (|v| reaches 448 scales)
                want, bound = plain64.attention(rows, k, v, seen, scale, plain64.E_F16)
                top = torch.where(seen.any(0)[:, None, None], v.abs(), 0.0).nan_to_num(0.0).amax() if n else 0.0
                bound = bound + 2.0 ** -31 * n * top
            plain64.check(got[at:at + m], want, bound, f"{what} sequence {b} ({n} keys, {m} queries)")
        at += m


EDGES = [(1, 1), (130, 1), (128, 128), (129, 129), (300, 44), (0, 0), (257, 1), (511, 300), (700, 257), (5, 5), (64, 0), (1100, 70)]


@pytest.mark.parametrize("kind,hq,hkv", [("bf16", 4, 2), ("bf16", 3, 1), ("e4m3", 4, 2), ("e4m3", 7, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 4), (64, 0), (128, 130), (129, 1), (200, 256), (255, 4), (1000, 3),
                                          (5000, 9), (2 ** 31 - 1, 0)])
def test_edges(kind, hq, hkv, window, sinks):
    """Lengths, chunks and windows around tile and page borders; every slot that no query sees holds NaN."""
    c = _case(kind, EDGES, hq, hkv, (7 * window + sinks) % 1000, poison=(window, sinks))
    _check(c, _run(c, window, sinks), window, sinks)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("sinks", [1, 15, 16, 17, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("window", [40, 128, 300])
def test_sinks_in_front_of_the_window(kind, sinks, window):
    """The window's first tile with more, as many and fewer rows in front of the window than there are sinks; the sinks' page
    also one that lies outside of the pool: rows of zeros."""
    chunks = [(window + 127 + x + 2, 2) for x in (0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 126, 127, 128, 144, 300)]
    c = _case(kind, chunks + [(1500, 600), (900, 140)], 6, 2, sinks, poison=(window, sinks))
    _check(c, _run(c, window, sinks), window, sinks)
    c = _case(kind, [(1000, 3), (1040, 70)], 6, 2, sinks)
    for b, outside in ((0, -1), (1, c["k"].shape[0])):
        c["bt"][b, 0] = outside
        c["tables"][b][0] = c["k"].shape[0]
    got = _run(c, window, sinks)
    for x in "kv":                                       # what the kernel has to take it for: one more page, of zeros
        c[x] = torch.cat([c[x], torch.zeros_like(c[x][:1])])
        c[x + "s"] = None if c[x + "s"] is None else torch.cat([c[x + "s"], torch.ones_like(c[x + "s"][:1])])
    _check(c, got, window, sinks)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 16, 128])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_groups(kind, group):
    c = _case(kind, [(333, 200), (90, 33)], 2 * group if group < 128 else 128, 2 if group < 128 else 1, group)
    _check(c, _run(c, 150, 5), 150, 5)
    if kind == "e4m3":
        _check(c, _run(c))


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 5), (6, 1)])
def test_e4m3_causal(hq, hkv):
    c = _case("e4m3", EDGES + [(2000, 900)], hq, hkv, 31, poison=(2 ** 31, 0))
    _check(c, _run(c))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_queries_without_keys_give_zeros(kind):
    """A sequence with fewer keys than queries: its first queries stand in front of key 0 and see nothing."""
    c = _case(kind, [(40, 40), (64, 64), (300, 300)], 8, 2, 41)
    want = _run(c, 20, 2)
    lens = torch.tensor([10, 0, 40], dtype=torch.int32)
    c["cu_k"] = torch.cat([torch.zeros(1, dtype=torch.int32), lens.cumsum(0).to(torch.int32)]).cuda()
    got = _run(c, 20, 2)
    assert bool((got[:30] == 0).all()) and bool((got[40:104] == 0).all()) and bool((got[104:364] == 0).all())
    assert not bool((got[30:40] == 0).all()) and torch.isfinite(got).all() and got.shape == want.shape
    c["chunks"] = [(10, 10)]
    c["q"] = c["q"][30:40].contiguous()
    _check(c, got[30:40], 20, 2)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (4000, 100), (700, 0)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1), (16, 8)])
def test_split_over_the_keys(kind, window, sinks, hq, hkv):
    """Few rows over many keys: the parts of a cluster's thread blocks joined, of 2 to 16 of them; sequences of other lengths
    beside the long ones leave some of the blocks without a key."""
    if kind == "bf16" and window is None:
        window = 10 ** 6
    for chunks in ([(9000, 1)], [(5000, 3), (4100, 40)], [(2600, 30), (3, 3), (130, 1), (0, 0)], [(1200, 130), (900, 2)]):
        c = _case(kind, chunks, hq, hkv, 43, poison=(window or 10 ** 6, sinks))
        got = _run(c, window, sinks)
        _check(c, got, window, sinks)
        assert bits_equal(_run(c, window, sinks), got)


@pytest.mark.parametrize("batch,hkv", [(14, 5), (8, 5), (6, 5), (5, 5), (3, 7), (2, 7), (11, 1), (1, 7), (1, 1)])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_every_number_of_parts(kind, batch, hkv):
    """From 70 row blocks down to one: parts of 2, 3, 4, 5 and more thread blocks, up to 16, over 20 to 24 key tiles."""
    c = _case(kind, [(2500 + 40 * b, 3 + b) for b in range(batch)], 2 * hkv, hkv, batch)
    window = None if kind == "e4m3" else 10 ** 6
    got = _run(c, window)
    _check(c, got, window)
    assert bits_equal(_run(c, window), got)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("chunks", [[(900, 300), (100, 100)], [(6000, 2), (50, 1)]])
def test_rows_behind_the_last_sequence_stay(kind, chunks):
    c = _case(kind, chunks, 8, 2, 47, extra=5)
    c["max_q"] += 5
    out = torch.full_like(c["q"], 7.0)
    got = _run(c, 800, 4, out=out)
    assert got is out
    _check(c, got, 800, 4)
    assert bool((got[-5:] == 7.0).all())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_pages_outside_of_the_window_may_be_gone(kind):
    c = _case(kind, [(2000, 100), (3000, 1)], 8, 2, 53)
    want = _run(c, 300, 4)
    for b, (n, m) in enumerate(c["chunks"]):
        c["bt"][b, 1:(n - m + 1 - 300) // 256] = -1
    assert bits_equal(_run(c, 300, 4), want)


def test_e4m3_scales_far_apart():
    """V scales from 2^-12 to 2^12 from page to page, in both orders, K scales of 0 among them, and pages of scale 0."""
    c = _case("e4m3", [(1500, 1300), (2300, 40)], 8, 2, 59)
    for b in (0, 1):
        for i, page in enumerate(c["tables"][b]):
            c["vs"][page] *= 2.0 ** [0, -12, 12, 3, -5, 0, 7, -9, 1, 2][i]
        c["vs"][c["tables"][b][4], 0] = 0
        c["v"][c["tables"][b][4], :, 0] = 0x7f                        # a scale of 0 means values of 0, whatever the bytes
        c["ks"][c["tables"][b][3], 1] = 0
    v = c["v"].clone()
    got = _run(c)
    for b in (0, 1):
        c["v"][c["tables"][b][4], :, 0] = 0
    _check(c, got)
    c["v"].copy_(v)
    got = _run(c, 600, 4)
    for b in (0, 1):
        c["v"][c["tables"][b][4], :, 0] = 0
    _check(c, got, 600, 4)


@pytest.mark.parametrize("amplitude", [2.0 ** -100, 1e-6, 1e6, 2.0 ** 100])
def test_e4m3_queries_of_any_size(amplitude):
    c = _case("e4m3", [(400, 130)], 4, 2, 61, amplitude=amplitude)
    _check(c, _run(c, scale=SCALE / amplitude), scale=SCALE / amplitude)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_large_pages_long_context_and_repeats(kind):
    """Pages of 768 tokens, a context of 20000 keys, the same bits twice and on another stream."""
    c = _case(kind, [(20000, 500), (1000, 1000)], 8, 2, 67, block_size=768)
    got = _run(c, 3000, 64)
    _check(c, got, 3000, 64)
    assert bits_equal(_run(c, 3000, 64), got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _run(c, 3000, 64)
    torch.cuda.synchronize()
    assert bits_equal(again, got)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_in_a_graph(kind):
    """Queries, cache and lengths change between replays."""
    c = _case(kind, [(4000, 8), (900, 5)], 8, 2, 71)
    _run(c, 3000, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(c, 3000, 4)
    c["q"].copy_(torch.randn_like(c["q"].float()).bfloat16())
    c["cu_k"].copy_(torch.tensor([0, 3900, 4700], dtype=torch.int32))
    c["chunks"] = [(3900, 8), (800, 5)]
    graph.replay()
    torch.cuda.synchronize()
    _check(c, out, 3000, 4)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("chunks", [[(700, 300)], [(6000, 2)]])
def test_waits_that_run_out_are_reported(kind, chunks):
    """A producer that loads nothing and a short limit: the call raises once, and the next one is right again."""
    c = _case(kind, chunks, 8, 2, 73)
    want = _run(c, 500, 4)
    with selftest.variant(wait_limit=4096, stall_producer=1):
        with pytest.raises(RuntimeError, match="bounded device-side wait"):
            _run(c, 500, 4)
    assert bits_equal(_run(c, 500, 4), want)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_pages_outside_of_the_pool_and_narrow_tables_read_as_zeros(kind):
    c = _case(kind, [(700, 130), (600, 3)], 8, 2, 83)
    clean = {x: c[x].clone() for x in "kv"}
    top = 448 * c["vs"].amax().double() if kind == "e4m3" else c["v"].abs().amax().double()
    for x in "kv":
        for b in (0, 1):
            c[x][c["tables"][b][1]] = 0
    want = _run(c, 600, 4)
    for x in "kv":
        c[x].copy_(clean[x])
    bt = c["bt"]
    for bad in (-1, bt.max().item() + 50, 2 ** 31 - 1, -2 ** 31):
        c["bt"] = bt.clone()
        c["bt"][:2, 1] = bad
        if kind == "bf16":
            assert bits_equal(_run(c, 600, 4), want)
        else:
            # a page without a place has no V scale either, so the f16 probabilities are taken in other units: half a step
            # (2^-11) of each on either side, and half a step (2^-8) of the result on either side
            plain64.check(_run(c, 600, 4), want.double(), 2.0 ** -7 * want.double().abs() + 2.0 ** -10 * top)
    # keys behind the table's columns
    c["bt"] = bt
    for x in "kv":
        for b in (0, 1):
            c[x][c["tables"][b][2]] = 0
    want = _run(c, 600, 4)
    for x in "kv":
        c[x].copy_(clean[x])
    c["bt"] = bt[:, :2].contiguous()
    got = _run(c, 600, 4)
    assert torch.isfinite(got).all()
    plain64.check(got, want.double(), 2.0 ** -7 * want.double().abs() + 2.0 ** (-10 if kind == "e4m3" else -7) * top)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_queries_that_are_not_finite_stay_their_own(kind):
    """A NaN or an infinity in one query's row gives NaN there and nowhere else, split or not."""
    for chunks in ([(700, 300)], [(4000, 5)]):
        c = _case(kind, chunks, 8, 2, 89)
        want = _run(c, 3000, 4)
        c["q"][2, 3, 17] = float("nan")
        c["q"][4, 5, 0] = float("inf")
        got = _run(c, 3000, 4)
        assert torch.isnan(got[2, 3]).all() and torch.isnan(got[4, 5]).all()
        got[2, 3], got[4, 5] = want[2, 3], want[4, 5]
        assert bits_equal(got, want)


def test_sixteen_byte_aligned_queries_and_output():
    c = _case("e4m3", [(500, 200)], 8, 2, 97)
    want = _run(c, 300, 4)
    buf = torch.zeros(2, c["q"].numel() + 8, dtype=torch.bfloat16, device="cuda")
    q, out = (b[8:].view(c["q"].shape) for b in buf)
    assert q.data_ptr() % 32 == 16
    q.copy_(c["q"])
    assert bits_equal(_run({**c, "q": q}, 300, 4, out=out), want)


def test_refusals():
    c = _case("e4m3", [(300, 10)], 8, 2, 79)
    for kw, match in ((dict(window=0), "window"), (dict(window=5, sinks=-1), "sinks"), (dict(sinks=3), "sinks"),
                      (dict(scale=0.0), "geometry"), (dict(scale=-1.0), "geometry"), (dict(scale=float("nan")), "geometry"),
                      (dict(out=torch.zeros(10, 8, 128, device="cuda")), "out"),
                      (dict(out=torch.zeros(9, 8, 128, dtype=torch.bfloat16, device="cuda")), "out")):
        with pytest.raises(RuntimeError, match=match):
            _run(c, **kw)
    for name, bad, match in (("cu_k", c["cu_k"][:1], "cu_seqlens"), ("bt", c["bt"][0], "block_table"), ("q", c["q"].float(), "bf16"),
                             ("q", c["q"].cpu(), "device"), ("bt", c["bt"].long(), "int32"), ("cu_q", c["cu_q"].cpu(), "int32")):
        with pytest.raises(RuntimeError, match=match):
            _run({**c, name: bad})
    with pytest.raises(ValueError):
        _run({**c, "ks": None})
    with pytest.raises(RuntimeError, match="geometry"):
        _run({**c, "max_q": 3})                       # fewer rows than the queries that came
