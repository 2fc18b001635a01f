"""The rotary, append, windowed-attention and read-back ops as a serving loop uses them together."""
import pytest
import torch

import plain64
from infer_b200 import metadata, ops
from infer_b200.attention import Attention
from infer_b200.context import get_context, reset_context, set_context
from infer_b200.engine import AttentionLayerModel, Engine, LayerRunner, Scheduler
from infer_b200.rotary import rotary_frequencies
from infer_b200.sequence import Sequence

pytestmark = pytest.mark.gpu
BS, HQ, HKV = 256, 8, 2


def _layer(kind, blocks, window, sinks):
    attn = Attention(HQ, 128, 128 ** -0.5, HKV, window=window, sinks=sinks)
    dtype = torch.bfloat16 if kind == "bf16" else torch.uint8
    attn.k_cache, attn.v_cache = (torch.zeros(blocks, BS, HKV, 128, dtype=dtype, device="cuda") for _ in range(2))
    if kind == "e4m3":
        attn.k_scale, attn.v_scale = (torch.zeros(blocks, HKV, device="cuda") for _ in range(2))
    return attn


def _check(attn, q, o, tables, lens, new, kind, what):
    """The layer's output against 64 bits on the rows that load_kvcache reads back: what is in the cache is what it attends to.
    (Read back as bf16: an e4m3 value times its scale is rounded, 2^-8 of it, twice over in a score.)"""
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        slots = torch.tensor(metadata.chunk_slots(tables[b], 0, n, BS), dtype=torch.int32, device="cuda")
        k, v = ops.load_kvcache(attn.k_cache, attn.v_cache, slots, k_scale=attn.k_scale, v_scale=attn.v_scale)
        seen = plain64.visible(n, torch.arange(n - m, n, device="cuda"), attn.window, attn.sinks)
        want, bound = plain64.attention(q[at:at + m], k, v, seen, attn.scale, plain64.E_BF16)
        if kind == "e4m3":
            top = v.double().abs().amax()
            score = torch.einsum("qhd,khd->qhk", q[at:at + m].double().abs(),
                                 k.double().abs().repeat_interleave(HQ // HKV, 1)).amax(-1, keepdim=True) * attn.scale
            bound = bound + (2 * 2.0 ** -8 * score + 2.0 ** -8) * top
        plain64.check(o[at:at + m].view(m, HQ, 128), want, bound, f"{what} sequence {b}")
        at += m


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_prefill_in_chunks_then_decode(kind, interleaved):
    window, sinks = 200, 4
    gen = torch.Generator().manual_seed(2)
    lens, chunks = [0, 0, 0], [[130, 300], [257, 256], [1, 64]]
    tables = [[4, 1, 7], [0, 5, 2], [3, 6, 8]]
    attn = _layer(kind, 9, window, sinks)
    inv_freq, factor = rotary_frequencies(64, scaling="yarn", factor=4.0, original_max_position=1024, device="cuda")
    rnd = lambda t: torch.randn(t, (HQ + 2 * HKV) * 128, generator=gen).bfloat16().cuda()

    def split(qkv):
        return [x.view(qkv.shape[0], -1, 128) for x in qkv.split([HQ * 128, HKV * 128, HKV * 128], dim=1)]

    for step in range(2):                                                 # chunked prefill of three sequences
        new = [c[step] for c in chunks]
        positions = torch.cat([torch.arange(n, n + m) for n, m in zip(lens, new)]).cuda()
        metadata.prepare_chunk(tables, lens, new, BS, "cuda")
        q, k, v = split(rnd(sum(new)))
        q, k = ops.rotary_embedding(q, k, positions, inv_freq, interleaved=interleaved, attention_factor=factor)
        o = attn(q, k, v.contiguous())
        reset_context()
        lens = [n + m for n, m in zip(lens, new)]
        _check(attn, q, o, tables, lens, new, kind, f"chunk {step}")
    state = metadata.DecodeState(4, 3, BS, "cuda")                         # one row of padding, as in a captured batch
    seqs = []
    for t, n in zip(tables, lens):
        s = Sequence(list(range(n)))
        s.block_table = list(t)
        seqs.append(s)
    state.load(seqs)
    for step in range(5):
        state.advance()
        lens = [n + 1 for n in lens]
        q, k, v = split(rnd(4))
        pos = torch.tensor([n - 1 for n in lens] + [0]).cuda()
        if kind == "bf16" and step % 2:
            # the append inside rotary_append, the attention by itself
            q = ops.rotary_append(q, k, v, pos, inv_freq, attn.k_cache, attn.v_cache, state.slot_mapping, interleaved=interleaved,
                                  attention_factor=factor)
            o = ops.paged_attn_decode(q, attn.k_cache, attn.v_cache, state.context_lens, state.block_tables, attn.scale, window=window,
                                      sinks=sinks)
        else:
            q, k = ops.rotary_embedding(q, k, pos, inv_freq, interleaved=interleaved, attention_factor=factor)
            set_context(False, slot_mapping=state.slot_mapping, context_lens=state.context_lens, block_tables=state.block_tables)
            o = attn(q, k, v.contiguous())
        reset_context()
        _check(attn, q[:3], o[:3], tables, lens, [1, 1, 1], kind, f"step {step}")


@pytest.mark.parametrize("kv_dtype,window,eager", [("e4m3", None, False), ("e4m3", 150, False), ("bf16", 150, False), ("e4m3", 150, True)])
def test_engine_on_8_bit_pools_and_windows(kv_dtype, window, eager):
    """The engine loop with e4m3 pools and a windowed layer: every 20th step's attention against 64 bits on the pools."""
    blocks = 7
    sch = Scheduler(blocks, BS, max_num_seqs=8)
    model = AttentionLayerModel(hidden=256, n_q_heads=16, n_kv_heads=8, vocab=1000, max_position=2048, device="cuda", window=window,
                                sinks=4 if window else 0)
    runner = LayerRunner(model, blocks, BS, max_num_seqs=8, max_model_len=1024, device="cuda", enforce_eager=eager, kv_dtype=kv_dtype)
    engine = Engine(runner, sch)
    gen = torch.Generator().manual_seed(3)
    for n, more in ((300, 120), (40, 230), (1, 60)):
        engine.add_request(torch.randint(0, 1000, (n,), generator=gen).tolist(), more)
    late = False
    while not sch.is_finished():
        lens = None
        batch, is_prefill, _ = engine.step()
        ctx = get_context()
        if is_prefill or engine.steps % 20 == 0:
            if is_prefill:
                cu_q, cu_k = ctx.cu_seqlens_q.tolist(), ctx.cu_seqlens_k.tolist()
                new, lens = ([c[i + 1] - c[i] for i in range(len(batch))] for c in (cu_q, cu_k))
            else:
                new, lens = [1] * len(batch), ctx.context_lens.tolist()[:len(batch)]
            at = 0
            for b, (n, m) in enumerate(zip(lens, new)):
                q, o = (runner.last_tap[x][at:at + m].view(m, 16, 128) for x in ("q", "o"))
                table = ctx.block_tables[b].tolist()
                scales = (None, None) if kv_dtype == "bf16" else (runner.kv_scale[0], runner.kv_scale[1])
                k, v = (plain64.values(runner.kv_cache[i], scales[i], table, n) for i in (0, 1))
                seen = plain64.visible(n, torch.arange(n - m, n, device="cuda"), window, model.attn.sinks)
                want, bound = plain64.attention(q, k, v, seen, model.attn.scale, plain64.E_BF16)
                plain64.check(o, want, bound + 2.0 ** -25 * n * v.abs().amax(), f"step {engine.steps} sequence {b}")
                at += m
        reset_context()
        if not late and engine.steps > 130:                                # takes over pages of finished requests
            engine.add_request(torch.randint(0, 1000, (500,), generator=gen).tolist(), 30)
            late = True
    assert late and engine.steps > 200


def test_torch_ops_of_the_new_kernels():
    from infer_b200 import infer_ops
    gen = torch.Generator().manual_seed(4)
    (k, ks), (v, vs) = (plain64.e4m3_pool(4, BS, HKV, gen) for _ in range(2))
    k, v, ks, vs = k.cuda(), v.cuda(), ks.cuda(), vs.cuda()
    slots = torch.arange(100, 140, dtype=torch.int32, device="cuda")
    want = ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    got = [torch.zeros_like(w) for w in want]
    infer_ops.load_kvcache(*got, k, v, slots, ks, vs)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    q = torch.randn(2, HQ, 128, generator=gen).bfloat16().cuda()
    lens, bt = torch.tensor([300, 80], dtype=torch.int32).cuda(), torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    out = torch.zeros_like(q)
    infer_ops.paged_attn_decode_window(out, q, k, v, lens, bt, 0.1, 64, 2, ks, vs)
    assert torch.equal(out, ops.paged_attn_decode(q, k, v, lens, bt, 0.1, k_scale=ks, v_scale=vs, window=64, sinks=2))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    cu_k = torch.tensor([0, 300, 380], dtype=torch.int32).cuda()
    infer_ops.paged_attn_prefill_window(out, q, k, v, cu, cu_k, 1, 300, 0.1, bt, None, 0, ks, vs)
    assert torch.equal(out, ops.paged_attn_prefill(q, k, v, cu, cu_k, 1, 300, 0.1, bt, k_scale=ks, v_scale=vs))
    kc, vc = (torch.zeros(1, BS, HKV, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kv = torch.randn(2, HKV, 128, generator=gen).bfloat16().cuda()
    pos, f = torch.tensor([5, 9]).cuda(), rotary_frequencies(32, device="cuda")[0]
    infer_ops.rotary_append(out, q, kv, kv, pos, f, kc, vc, slots[:2], True, 1.0)
    want = ops.rotary_embedding(q, kv, pos, f, interleaved=True)
    assert torch.equal(out, want[0]) and torch.equal(kc[0, 100:102], want[1]) and torch.equal(vc[0, 100:102], kv)


def _against_the_pools(attn, q, o, tables, lens, new, kind, decode, what):
    """The layer's output against 64 bits on the values that the pools hold, with the bounds of the kernels' own tests: f16
    probabilities over e4m3 pools, bf16 ones over bf16 pools.  Returns how many values another window or no sinks would have put
    out of those bounds (worked out on the CPU)."""
    at, told = 0, {"a shorter window": 0, "no sinks": 0, "nothing": 0}
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = (plain64.values(c, s, tables[b], n).cpu() for c, s in ((attn.k_cache, attn.k_scale), (attn.v_cache, attn.v_scale)))
        rows, got = q[at:at + m].cpu(), o[at:at + m].view(m, HQ, 128).double().cpu()

        def exact(window, sinks):
            seen = plain64.visible(n, torch.arange(n - m, n), window, sinks)
            if kind == "bf16":
                return plain64.attention(rows, k, v, seen, attn.scale, plain64.E_BF16)
            want, bound = plain64.attention(rows, k, v, seen, attn.scale, plain64.E_F16, 2.0 ** -25 if decode else 0.0)
            return want, bound + (0.0 if decode else 2.0 ** -31 * n * v.abs().amax())

        want, bound = exact(attn.window, attn.sinks)
        plain64.check(got, want, bound, f"{what} sequence {b}")
        for name, other in (("a shorter window", exact(attn.window - 1, attn.sinks)), ("no sinks", exact(attn.window, 0)),
                            ("nothing", (torch.zeros_like(want), bound))):
            told[name] += int(((got - other[0]).abs() > other[1]).sum())
        at += m
    return told


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_chunks_then_decode_against_the_pools(kind):
    """Chunked prefill, append and windowed decode through the layer, with bounds that a wrong window or lost sinks cannot meet; what
    load_kvcache reads back is checked against the same pools by itself."""
    gen = torch.Generator().manual_seed(6)
    attn = _layer(kind, 9, 200, 4)
    lens, tables = [0, 0, 0], [[4, 1, 7], [0, 5, 2], [3, 6, 8]]
    rnd = lambda t, h: torch.randn(t, h, 128, generator=gen).bfloat16().cuda()
    for step, new in enumerate(([300, 257, 1], [130, 256, 64])):
        metadata.prepare_chunk(tables, lens, new, BS, "cuda")
        q = rnd(sum(new), HQ)
        o = attn(q, rnd(sum(new), HKV), rnd(sum(new), HKV))
        reset_context()
        lens = [n + m for n, m in zip(lens, new)]
        told = _against_the_pools(attn, q, o, tables, lens, new, kind, False, f"chunk {step}")
        assert min(told.values()) > 1000, told
    for step in range(3):
        lens = [n + 1 for n in lens]
        slots = torch.tensor([metadata.chunk_slots(t, n - 1, n, BS)[0] for t, n in zip(tables, lens)], dtype=torch.int32).cuda()
        set_context(False, slot_mapping=slots, context_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                    block_tables=torch.tensor(tables, dtype=torch.int32).cuda())
        q = rnd(3, HQ)
        o = attn(q, rnd(3, HKV), rnd(3, HKV))
        reset_context()
        told = _against_the_pools(attn, q, o, tables, lens, [1, 1, 1], kind, True, f"step {step}")
        assert min(told.values()) > 100, told
    for t, n in zip(tables, lens):
        slots = torch.tensor(metadata.chunk_slots(t, 0, n, BS), dtype=torch.int32, device="cuda")
        back = ops.load_kvcache(attn.k_cache, attn.v_cache, slots, k_scale=attn.k_scale, v_scale=attn.v_scale)
        for got, c, s in zip(back, (attn.k_cache, attn.v_cache), (attn.k_scale, attn.v_scale)):
            # a product of 4 by 24 bits: exact in 64, rounded once to 32 bits and once to bf16
            assert torch.equal(got, plain64.values(c, s, t, n).float().bfloat16())
