"""Block tables that are views: a single row of any stride, and columns of a wider table."""
import pytest
import torch

import plain64
from gpu_util import bits_equal
from infer_b200 import ops

pytestmark = pytest.mark.gpu
SCALE, BS, HQ, HKV, COLS = 128 ** -0.5, 256, 8, 2, 6
FORMS = [("bf16", 900, 4), ("e4m3", 900, 4), ("e4m3", None, 0)]


def _pools(kind, gen):
    blocks = 4 * COLS
    if kind == "bf16":
        return [torch.randn(blocks, BS, HKV, 128, generator=gen).bfloat16().cuda() for _ in range(2)] + [None, None]
    (k, ks), (v, vs) = (plain64.e4m3_pool(blocks, BS, HKV, gen) for _ in range(2))
    return [x.cuda() for x in (k, v, ks, vs)]


def _prefill(pools, q, keys, new, table, window, sinks):
    k, v, ks, vs = pools
    cu = lambda x: torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32).cuda()
    return ops.paged_attn_prefill(q, k, v, cu(new), cu(keys), max(new), max(keys), SCALE, table, k_scale=ks, v_scale=vs, window=window,
                                  sinks=sinks)


@pytest.mark.parametrize("kind,window,sinks", FORMS)
@pytest.mark.parametrize("new", [3, 300])
def test_prefill_with_a_single_row_of_any_stride(kind, window, sinks, new):
    """PyTorch may report any stride for a dimension of one: pages[:, None].t() is [1, n] with strides (1, 1)."""
    gen = torch.Generator().manual_seed(new)
    pools = _pools(kind, gen)
    pages = torch.randperm(4 * COLS, generator=gen)[:COLS].to(torch.int32).cuda()
    q = torch.randn(new, HQ, 128, generator=gen).bfloat16().cuda()
    keys = COLS * BS - 7
    want = _prefill(pools, q, [keys], [new], pages[None].clone(), window, sinks)
    one = pages[:, None].t()
    assert one.shape == (1, COLS) and one.stride() == (1, 1)
    assert bits_equal(_prefill(pools, q, [keys], [new], one, window, sinks), want)
    assert bits_equal(_prefill(pools, q, [keys], [new], torch.as_strided(pages, (1, COLS), (0, 1)), window, sinks), want)
    exact, bound = plain64.attention(q, *(plain64.values(pools[i], pools[i + 2], pages.tolist(), keys) for i in (0, 1)),
                                     plain64.visible(keys, torch.arange(keys - new, keys, device="cuda"), window, sinks), SCALE,
                                     plain64.E_BF16)
    plain64.check(want, exact, bound + 2.0 ** -25 * pools[1].float().abs().amax() if kind == "bf16" else
                  bound + 2.0 ** -31 * keys * 448 * pools[3].amax())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_with_a_single_row_of_any_stride(kind):
    gen = torch.Generator().manual_seed(5)
    k, v, ks, vs = _pools(kind, gen)
    pages = torch.randperm(4 * COLS, generator=gen)[:COLS].to(torch.int32).cuda()
    q = torch.randn(1, HQ, 128, generator=gen).bfloat16().cuda()
    lens = torch.tensor([COLS * BS - 7], dtype=torch.int32).cuda()
    run = lambda table: ops.paged_attn_decode(q, k, v, lens, table, SCALE, k_scale=ks, v_scale=vs, window=900, sinks=4)
    want = run(pages[None].clone())
    for one in (pages[:, None].t(), torch.as_strided(pages, (1, COLS), (0, 1))):
        assert bits_equal(run(one), want)                 # the same parts: the choice looks at the table's columns


@pytest.mark.parametrize("kind,window,sinks", FORMS)
@pytest.mark.parametrize("lo,hi", [(0, 3), (0, COLS), (2, 5), (3, COLS), (COLS - 1, COLS)])
def test_prefill_with_columns_of_a_wider_table(kind, window, sinks, lo, hi):
    """A key behind the table's columns counts as a row of zeros, although the wider table goes on; of the last row nothing
    behind the columns may be read, since the memory ends there."""
    gen = torch.Generator().manual_seed(7 * lo + hi)
    pools = _pools(kind, gen)
    wide = torch.randperm(4 * COLS, generator=gen)[:3 * COLS].to(torch.int32).view(3, COLS).cuda()
    keys, new = [COLS * BS - 9, 700, COLS * BS], [200, 3, 1]
    q = torch.randn(sum(new), HQ, 128, generator=gen).bfloat16().cuda()
    part = wide[:, lo:hi]
    assert part.stride(0) == COLS
    want = _prefill(pools, q, keys, new, part.contiguous(), window, sinks)
    got = _prefill(pools, q, keys, new, part, window, sinks)
    assert bits_equal(got, want)
    # a single row that is a column slice: its pitch is the wider table's
    one = _prefill(pools, q[:200], keys[:1], new[:1], part[:1], window, sinks)
    assert bits_equal(one, _prefill(pools, q[:200], keys[:1], new[:1], part[:1].contiguous(), window, sinks))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_with_columns_of_a_wider_table(kind):
    gen = torch.Generator().manual_seed(9)
    k, v, ks, vs = _pools(kind, gen)
    wide = torch.randperm(4 * COLS, generator=gen)[:3 * COLS].to(torch.int32).view(3, COLS).cuda()
    q = torch.randn(3, HQ, 128, generator=gen).bfloat16().cuda()
    lens = torch.tensor([700, 3 * BS, 12], dtype=torch.int32).cuda()
    tables = wide[:, 2:5]
    got = ops.paged_attn_decode(q, k, v, lens, tables, SCALE, k_scale=ks, v_scale=vs, window=600, sinks=4)
    eps, lost = (plain64.E_BF16, 0.0) if kind == "bf16" else (plain64.E_F16, 2.0 ** -25)
    for b, n in enumerate(lens.tolist()):
        kk, vv = plain64.values(k, ks, tables[b].tolist(), n), plain64.values(v, vs, tables[b].tolist(), n)
        want, bound = plain64.attention(q[b:b + 1], kk, vv, plain64.visible(n, torch.tensor([n - 1], device="cuda"), 600, 4), SCALE, eps,
                                        lost)
        plain64.check(got[b:b + 1], want, bound, f"sequence {b}")


def test_prefill_with_rows_that_overlap():
    """Rows of three columns that start one entry apart: every row is the table's own, whatever the pitch."""
    gen = torch.Generator().manual_seed(11)
    pools = _pools("bf16", gen)
    pages = torch.randperm(4 * COLS, generator=gen)[:COLS].to(torch.int32).cuda()
    keys, new = [700, 600, 650], [40, 3, 1]
    q = torch.randn(sum(new), HQ, 128, generator=gen).bfloat16().cuda()
    table = torch.as_strided(pages, (3, 3), (1, 1))
    assert bits_equal(_prefill(pools, q, keys, new, table, 300, 4), _prefill(pools, q, keys, new, table.contiguous(), 300, 4))
