"""Paged decode over a sliding window and the first tokens (sinks), bf16 and e4m3 pools, with and without the fused append."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _case(kind, lens, hq, hkv, seed, block_size=256, spread=0.5, poison=None):
    """Pools, page lists and queries.  ``poison`` (window, sinks): every slot that no query may see holds NaN."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // block_size) for n in lens]
    blocks = sum(need) + 2
    perm = torch.randperm(blocks, generator=gen).tolist()
    tables = [[perm.pop() for _ in range(c)] for c in need]
    q = torch.randn(len(lens), hq, 128, generator=gen).bfloat16()
    if kind == "bf16":
        k, v = (torch.randn(blocks, block_size, hkv, 128, generator=gen).bfloat16() for _ in range(2))
        ks = vs = None
    else:
        (k, ks), (v, vs) = (plain64.e4m3_pool(blocks, block_size, hkv, gen, spread) for _ in range(2))
    if poison is not None:
        window, sinks = poison
        live = torch.zeros(blocks * block_size, dtype=torch.bool)
        for n, t in zip(lens, tables):
            for j in range(n):
                if j >= n - window or j < sinks:
                    live[t[j // block_size] * block_size + j % block_size] = True
        for c in (k, v):
            c.view(-1, hkv, 128)[~live] = float("nan") if kind == "bf16" else 0x7f
    width = max(need) + 1
    bt = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int32)
    cuda = lambda x: None if x is None else x.cuda()
    return dict(q=q.cuda(), k=k.cuda(), v=v.cuda(), ks=cuda(ks), vs=cuda(vs), bt=bt.cuda(), tables=tables,
                lens=torch.tensor(lens, dtype=torch.int32).cuda())


def _want(c, b, window, sinks, scale=SCALE):
    n = int(c["lens"][b])
    k, v = (plain64.values(c[x], c[x + "s"], c["tables"][b], n) for x in "kv")
    seen = plain64.visible(n, torch.tensor([n - 1], device="cuda"), window, sinks)
    # e4m3: probabilities in f16, absolute half step 2^-25 below 2^-14; sums of 32-bit partial results otherwise
    eps, lost = (plain64.E_BF16, 0.0) if c["ks"] is None else (plain64.E_F16, 2.0 ** -25)
    return plain64.attention(c["q"][b:b + 1], k, v, seen, scale, eps, lost)


def _run(c, window, sinks, scale=SCALE, **kw):
    return ops.paged_attn_decode(c["q"], c["k"], c["v"], c["lens"], c["bt"], scale, k_scale=c["ks"], v_scale=c["vs"],
                                 window=window, sinks=sinks, **kw)


def _check(c, got, window, sinks, what="", scale=SCALE):
    for b in range(len(c["tables"])):
        if int(c["lens"][b]):
            want, bound = _want(c, b, window, sinks, scale)
            plain64.check(got[b:b + 1], want, bound, f"{what} sequence {b} ({int(c['lens'][b])} keys)")


LENS = [1, 2, 15, 16, 17, 100, 127, 128, 129, 255, 256, 257, 383, 512, 700, 1025, 2600]


@pytest.mark.parametrize("kind,hkv", [("bf16", 2), ("e4m3", 1), ("e4m3", 2), ("e4m3", 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (16, 0), (64, 130), (128, 0), (129, 1), (200, 256), (255, 4),
                                          (1000, 3), (5000, 0), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_edges(kind, hkv, window, sinks):
    """Lengths and windows around tile and page borders; every slot outside of the visible keys holds NaN."""
    c = _case(kind, LENS, 4 * hkv, hkv, 7 * window % 1000 + sinks % 1000, poison=(window, sinks))
    _check(c, _run(c, window, sinks), window, sinks)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("group", [1, 2, 3, 5, 6, 7, 8])
def test_groups(kind, group):
    c = _case(kind, [900, 33, 0, 1500], 5 * group, 5, group)
    out = torch.full_like(c["q"], 7.0)
    got = _run(c, 300, 5, out=out)
    _check(c, got, 300, 5)
    assert bool((out[2] == 7.0).all()), "the row of an empty sequence was written"


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_pages_outside_of_the_window_may_be_gone(kind):
    """Entries of pages without a visible key are -1: the engine has given those pages back."""
    c = _case(kind, [2000, 1024, 3000], 8, 4, 11)
    want = _run(c, 300, 4)
    for b, n in enumerate([2000, 1024, 3000]):
        first = (n - 300) // 256
        c["bt"][b, 1:first] = -1                       # page 0 holds the sinks
    assert bits_equal(_run(c, 300, 4), want)
    for b, n in enumerate([2000, 1024, 3000]):
        c["bt"][b, 0] = -1
    assert torch.isfinite(_run(c, 300, 0)).all()


@pytest.mark.parametrize("kind,hkv", [("bf16", 10), ("e4m3", 9), ("e4m3", 10), ("e4m3", 12)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 4), (64, 130), (129, 1), (1000, 3), (2 ** 31 - 1, 0)])
def test_edges_of_more_rows_than_thread_blocks(kind, hkv, window, sinks):
    """As above, with tiles handed out in equal ranges over all sequences, of one, two and four heads in an e4m3 pool."""
    c = _case(kind, LENS, 2 * hkv, hkv, window % 1000 + sinks, poison=(window, sinks))
    _check(c, _run(c, window, sinks), window, sinks)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [100, 900, 2000, 4000])
def test_parts_of_few_sequences(kind, window):
    """One to eighteen sequences of two heads and up to 41 key tiles: one part and more, up to one per tile, some of them empty."""
    for lens in ([5200], [5200, 40, 0], [3000, 260] * 9):
        c = _case(kind, lens, 8, 2, window + len(lens), poison=(window, 5))
        got = _run(c, window, 5)
        _check(c, got, window, 5)
        rows = c["lens"] > 0                                # an empty sequence's row is left as it was
        assert bits_equal(_run(c, window, 5)[rows], got[rows])


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_window_of_everything_is_plain_decode(kind):
    c = _case(kind, [700, 130, 2048, 1], 16, 8, 13)
    plain = ops.paged_attn_decode(c["q"], c["k"], c["v"], c["lens"], c["bt"], SCALE, k_scale=c["ks"], v_scale=c["vs"])
    got = _run(c, 2048, 0)
    # the windowed call may cut the keys into other parts, whose 32-bit sums meet in another order: either is within the bound
    # of the exact value, |got - plain| <= |got - exact| + |exact - plain| <= 2 bounds
    for b in range(4):
        _, bound = _want(c, b, 2048, 0)
        plain64.check(got[b:b + 1], plain[b:b + 1].double(), 2 * bound)
    _check(c, got, 2048, 0)
    _check(c, plain, 2048, 0)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_large_pages_and_many_sequences(kind):
    c = _case(kind, [(37 * i) % 1500 for i in range(300)], 4, 2, 17, block_size=768)
    got = _run(c, 190, 20, out=torch.zeros_like(c["q"]))
    for b in range(0, 300, 7):
        if int(c["lens"][b]):
            want, bound = _want(c, b, 190, 20)
            plain64.check(got[b:b + 1], want, bound, f"sequence {b}")


def test_e4m3_pages_without_scale():
    """Pages of scale 0 (nothing but zeros stored): scores of 0 that count, values of 0."""
    c = _case("e4m3", [900, 300], 8, 4, 19)
    for x in ("k", "v"):
        page = c["tables"][0][3 if x == "k" else 2]
        c[x][page] = 0
        c[x + "s"][page] = 0
    _check(c, _run(c, 400, 4), 400, 4)


def test_fused_append_with_a_window():
    lens = [1, 2, 128, 129, 256, 257, 600, 1300, 0, 2049]
    for window, sinks in ((1, 0), (1, 4), (100, 4), (512, 0), (4000, 0)):
        c = _case("bf16", lens, 16, 8, window)
        gen = torch.Generator().manual_seed(window)
        rows = torch.randn(len(lens), 2 * 8 * 128, generator=gen).bfloat16().cuda()
        key, value = rows[:, :1024].view(-1, 8, 128), rows[:, 1024:].view(-1, 8, 128)
        slots = torch.tensor([t[(n - 1) // 256] * 256 + (n - 1) % 256 if n else -1 for t, n in zip(c["tables"], lens)],
                             dtype=torch.int32, device="cuda")
        k2, v2 = c["k"].clone(), c["v"].clone()
        ops.store_kvcache(key, value, k2, v2, slots)
        got = ops.paged_attn_decode_append(c["q"], key, value, c["k"], c["v"], c["lens"], c["bt"], SCALE, window=window, sinks=sinks,
                                           out=torch.zeros_like(c["q"]))
        assert bits_equal(c["k"], k2) and bits_equal(c["v"], v2)
        _check(c, got, window, sinks, f"window {window}")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_in_a_graph_with_growing_lengths_and_own_workspace(kind):
    c = _case(kind, [250, 500, 1000, 260], 8, 2, 23)
    pool = ops.pool_of(c["k"], c["v"], c["ks"], c["vs"])
    ws = torch.zeros(pool.decode_workspace_bytes(4, 8), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(c["q"])
    c["lens"] -= 3
    _run(c, 100, 4, workspace=ws, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(c, 100, 4, workspace=ws, out=out)
    for _ in range(3):
        c["lens"] += 1
        graph.replay()
        torch.cuda.synchronize()
        _check(c, out, 100, 4)


def test_pinned_host_queries_and_output_and_four_dims():
    for kind in ("bf16", "e4m3"):
        c = _case(kind, [700, 30], 8, 2, 31)
        want = _run(c, 100, 4)
        q, out = c["q"].cpu().pin_memory(), torch.zeros(2, 8, 128, dtype=torch.bfloat16).pin_memory()
        got = _run({**c, "q": q}, 100, 4, out=out)
        torch.cuda.synchronize()
        assert got.data_ptr() == out.data_ptr() and bits_equal(out, want)
        four = _run({**c, "q": c["q"][:, None]}, 100, 4)
        assert four.shape == (2, 1, 8, 128) and bits_equal(four[:, 0], want)


def test_refusals():
    c = _case("bf16", [100, 30], 8, 2, 29)
    with pytest.raises(RuntimeError, match="pinned"):
        _run({**c, "q": c["q"].cpu()}, 10, 0)
    with pytest.raises(RuntimeError, match="cache_seqlens"):
        _run({**c, "lens": c["lens"][:1]}, 10, 0)
    with pytest.raises(RuntimeError, match="block_table"):
        _run({**c, "bt": c["bt"].long()}, 10, 0)
    with pytest.raises(RuntimeError, match="out must"):
        _run(c, 10, 0, out=torch.zeros(2, 8, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="key must"):
        ops.paged_attn_decode_append(c["q"], c["q"], c["q"], c["k"], c["v"], c["lens"], c["bt"], SCALE, window=5)
    with pytest.raises(RuntimeError, match="window"):
        _run(c, 0, 0)
    with pytest.raises(RuntimeError, match="sinks"):
        _run(c, 10, -1)
    with pytest.raises(RuntimeError, match="sinks"):
        _run(c, None, 4)
    with pytest.raises(RuntimeError, match="geometry"):
        _run(c, 10, 0, scale=0.0)
    with pytest.raises(RuntimeError, match="workspace"):
        _run(c, 10, 0, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
