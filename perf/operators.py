"""What the attention, rotary and cache operators are measured on: cases, their inputs, and every operator in its plain form.

Four operators over the paged key/value cache (pools ``[num_blocks, block_size, Hkv, 128]`` in bf16, or in e4m3 bytes with one
fp32 scale per page and KV head):

* ``decode``   one query token per sequence, attention over the last ``window`` keys and the first ``sinks`` ones;
* ``prefill``  many query tokens per sequence, causal, over a bf16 or an e4m3 cache, with or without window and sinks;
* ``rotary``   rotary positions applied to q and k, k and v appended to the cache;
* ``load``     rows of the cache read back as bf16.

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits, with ``own`` true it calls the package.
"""
import math
import random

import torch

own = False

D = 128            # head dimension of the pools
PAGE = 256         # tokens of a page


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest decode call: one request with a short context and a small window, latency only
        dict(name="decode one request", op="decode", kv="bf16", batch=1, hq=16, hkv=8, lo=1000, hi=1000, window=256, sinks=4, shape=1),
        # an ordinary decode step of a batch whose contexts are partly shorter and partly longer than the window
        dict(name="decode batch 64", op="decode", kv="bf16", batch=64, hq=32, hkv=8, lo=512, hi=8192, window=4096, sinks=4, shape=2),
        # a large decode step over an 8-bit cache: long contexts, eight query heads per KV head, an odd window
        dict(name="decode e4m3 long contexts", op="decode", kv="e4m3", batch=256, hq=64, hkv=8, lo=1024, hi=32768, window=4095, sinks=16,
             shape=3),
        # chunked prefill of a model whose layers see a window and a few first tokens
        dict(name="prefill window", op="prefill", kv="bf16", batch=16, hq=16, hkv=8, prefix=4096, chunk=2048, ragged=False, window=1024,
             sinks=4, shape=4),
        # the same chunks over an 8-bit cache, full causal attention
        dict(name="prefill e4m3", op="prefill", kv="e4m3", batch=16, hq=16, hkv=8, prefix=4096, chunk=2048, ragged=False, window=0, sinks=0,
             shape=4),
        # the tail of one prompt behind a cached prefix: a handful of query rows, latency counts
        dict(name="prefill e4m3 one short chunk", op="prefill", kv="e4m3", batch=1, hq=32, hkv=8, prefix=301, chunk=45, ragged=False,
             window=0, sinks=0, shape=5),
        # a few long documents, ragged chunks, 8-bit cache, odd window, five query heads per KV head
        dict(name="prefill e4m3 long documents", op="prefill", kv="e4m3", batch=3, hq=40, hkv=8, prefix=28000, chunk=1500, ragged=True,
             window=2047, sinks=64, shape=6),
        # the rows of one decode step
        dict(name="rotary decode step", op="rotary", tokens=64, hq=32, hkv=8, rot=128, interleaved=False, scaling="none", far=8192, shape=7),
        # a large prefill batch, positions scaled for a context four times as long as the trained one
        dict(name="rotary prefill batch", op="rotary", tokens=32768, hq=32, hkv=8, rot=128, interleaved=False, scaling="yarn", far=131072,
             shape=8),
        # interleaved pairs over half of every head, odd number of rows, far positions
        dict(name="rotary interleaved, half a head", op="rotary", tokens=5001, hq=64, hkv=8, rot=64, interleaved=True, scaling="linear",
             far=1000000, shape=9),
        # a prompt's pages read back from an 8-bit cache in bulk
        dict(name="load e4m3 32768 rows", op="load", kv="e4m3", tokens=32768, hkv=8, shape=10),
        # a short prefix copied out of a bf16 cache
        dict(name="load bf16 301 rows", op="load", kv="bf16", tokens=301, hkv=8, shape=11),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "prefill", "rotary", "load"])
    shape = rng.randrange(1, 1 << 20)
    hkv = rng.choice([1, 2, 3, 4, 5, 8, 8])
    if op == "decode":
        hq = hkv * rng.randint(1, 8)
        hi = _log(rng, 1, 32768)
        batch = max(1, min(_log(rng, 1, 256), 2000000 // hi))
        return dict(op=op, kv=rng.choice(["bf16", "e4m3"]), batch=batch, hq=hq, hkv=hkv, lo=max(1, hi // rng.randint(1, 8)), hi=hi,
                    window=_log(rng, 1, 8192) if rng.random() < 0.9 else 0, sinks=rng.choice([0, 1, 4, _log(rng, 1, 512)]), shape=shape)
    if op == "prefill":
        kv = rng.choice(["bf16", "e4m3", "e4m3"])
        hq = hkv * rng.randint(1, 8)
        prefix, chunk = _log(rng, 1, 16000) - 1, _log(rng, 1, 2048)
        # at most the padded query-key pairs of the largest listed case
        batch = max(1, min(_log(rng, 1, 16), int(16 * 16 * 2048 * 6144 / (hq * chunk * (prefix + chunk)))))
        window = _log(rng, 1, 8192) if kv == "bf16" or rng.random() < 0.5 else 0
        return dict(op=op, kv=kv, batch=batch, hq=hq, hkv=hkv, prefix=prefix, chunk=chunk, ragged=rng.random() < 0.7, window=window,
                    sinks=rng.choice([0, 1, 4, _log(rng, 1, 512)]) if window else 0, shape=shape)
    if op == "rotary":
        return dict(op=op, tokens=_log(rng, 1, 32768), hq=hkv * rng.randint(1, 4), hkv=hkv, rot=16 * rng.randint(1, 8),
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "yarn"]), far=_log(rng, 64, 1000000), shape=shape)
    return dict(op=op, kv=rng.choice(["bf16", "e4m3"]), tokens=_log(rng, 1, 32768), hkv=hkv, shape=shape)


def _lengths(case):
    """(keys, new tokens) of every sequence: a matter of the case alone. Some rows of a decode batch are empty, as a captured batch's padding is."""
    rng = random.Random(case["shape"])
    if case["op"] == "decode":
        keys = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        if case["batch"] >= 16:
            keys[-1] = keys[case["batch"] // 2] = 0
        return keys, [1 if n else 0 for n in keys]
    new = [rng.randint(1, case["chunk"]) if case["ragged"] else case["chunk"] for _ in range(case["batch"])]
    return [rng.randint(case["prefix"] // 2 if case["ragged"] else 0, case["prefix"]) + n for n in new], new


def _visible(n, first, window, sinks):
    """Keys that the rows first .. n - 1 of a sequence of n keys see: (pairs of row and key, keys that any of them sees)."""
    if not window:
        return sum(range(first + 1, n + 1)), n
    pairs = sum(min(i + 1, window + min(sinks, max(0, i + 1 - window))) for i in range(first, n))
    start = max(0, first + 1 - window)
    return pairs, n - start + min(sinks, start)


def work(case):
    if case["op"] in ("decode", "prefill"):
        keys, new = _lengths(case)
        seen = [_visible(n, n - m, case["window"], case["sinks"]) for n, m in zip(keys, new) if n]
        pairs, touched = sum(p for p, _ in seen), sum(t for _, t in seen)
        elem = 1 if case["kv"] == "e4m3" else 2
        return {"bytes": touched * case["hkv"] * D * 2 * elem + 2 * sum(new) * case["hq"] * D * 2, "flops": 4 * D * case["hq"] * pairs}
    if case["op"] == "rotary":
        return {"bytes": case["tokens"] * ((2 * case["hq"] + 4 * case["hkv"]) * D * 2 + 12),
                "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rot"]}
    elem = 1 if case["kv"] == "e4m3" else 2
    return {"bytes": case["tokens"] * (case["hkv"] * D * 2 * (elem + 2) + 4), "flops": case["tokens"] * case["hkv"] * D * 2 if elem == 1 else 0}


# --------------------------------------------------------------------------- inputs
def _pool(blocks, hkv, kv, gen):
    """One pool and its scales. Every page and head has an amplitude of its own, as the layers and positions of a model do."""
    x = torch.randn(blocks, PAGE, hkv, D, generator=gen, device="cuda")
    x *= torch.exp(0.4 * torch.randn(blocks, 1, hkv, 1, generator=gen, device="cuda"))
    if kv == "bf16":
        return x.to(torch.bfloat16), None
    scale = x.abs().amax(dim=(1, 3)) / 448
    return (x / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _inverse_frequencies(rot, scaling):
    """Radians per position of every pair, in 64 bits: plain, slowed down by 4, or by 4 for the slow pairs alone with a ramp between."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-2 * i / rot)
    if scaling == "none":
        return freq, 1.0
    if scaling == "linear":
        return freq / 4, 1.0
    turns = 4096 * freq / (2 * math.pi)                     # turns of a pair over the trained context
    keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
    return freq * keep + freq / 4 * (1 - keep), 0.1 * math.log(4) + 1


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] in ("decode", "prefill"):
        keys, new = _lengths(case)
        pages = [-(-n // PAGE) for n in keys]
        blocks = sum(pages) + 2
        order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
        first = torch.tensor([sum(pages[:b]) for b in range(len(pages))], device="cuda")
        count = torch.tensor(pages, device="cuda")
        at = torch.arange(max(1, max(pages)), device="cuda")
        table = order[(first[:, None] + at).clamp(max=blocks - 1)]
        s["block_table"] = torch.where(at < count[:, None], table, -1).to(torch.int32).contiguous()
        s["k_cache"], s["k_scale"] = _pool(blocks, case["hkv"], case["kv"], gen)
        s["v_cache"], s["v_scale"] = _pool(blocks, case["hkv"], case["kv"], gen)
        s["scale"] = D ** -0.5
        s["lens"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
        if case["op"] == "decode":
            s["q"] = rnd(case["batch"], case["hq"], D).to(torch.bfloat16)
            s["out"] = torch.zeros_like(s["q"])             # rows of empty sequences stay as they are
        else:
            s["q"] = rnd(sum(new), case["hq"], D).to(torch.bfloat16)
            cu = lambda v: torch.tensor([sum(v[:b]) for b in range(len(v) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
            s["cu_q"], s["cu_k"], s["max_q"], s["max_k"] = cu(new), cu(keys), max(new), max(keys)
        return s
    t, hkv = case["tokens"], case["hkv"]
    blocks = -(-t // PAGE) + 2
    if case["op"] == "load":
        s["k_cache"], s["k_scale"] = _pool(blocks, hkv, case["kv"], gen)
        s["v_cache"], s["v_scale"] = _pool(blocks, hkv, case["kv"], gen)
        page = torch.randperm(blocks, generator=gen, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = (page[at // PAGE] * PAGE + at % PAGE).to(torch.int32)
        return s
    hq = case["hq"]
    qkv = rnd(t, (hq + 2 * hkv) * D).to(torch.bfloat16)     # the fused projection's rows; q, k and v are columns of it
    s["q"], s["k"], s["v"] = (x.view(t, -1, D) for x in qkv.split([hq * D, hkv * D, hkv * D], dim=1))
    if t > 256:                                             # chunks of consecutive positions
        start = torch.randint(0, case["far"], (-(-t // 256),), generator=gen, device="cuda")
        at = torch.arange(t, device="cuda")
        s["positions"] = start[at // 256] + at % 256
    else:                                                   # one position per sequence
        s["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
    s["slots"] = torch.randperm(blocks * PAGE, generator=gen, device="cuda")[:t].to(torch.int32)
    s["inv_freq"], s["factor"] = _inverse_frequencies(case["rot"], case["scaling"])
    s["k_cache"] = torch.zeros(blocks, PAGE, hkv, D, dtype=torch.bfloat16, device="cuda")
    s["v_cache"] = torch.zeros_like(s["k_cache"])
    return s


# --------------------------------------------------------------------------- the plain forms
def _rows(cache, scale, slots):
    """Rows of a pool by flat slot, in 32 bits."""
    flat = cache.view(-1, *cache.shape[2:])[slots.long()]
    if scale is None:
        return flat.float()
    return flat.view(torch.float8_e4m3fn).float() * scale[slots.long() // cache.shape[1]][..., None]


def _slots(table, positions):
    """Flat slots of key positions [B, n]; a position without a page reads slot 0 and is masked by the caller."""
    page = table.gather(1, (positions // PAGE).clamp(0, table.shape[1] - 1))
    return (page.clamp(min=0) * PAGE + positions % PAGE).long()


def _softmax(scores, seen):
    """Softmax over the last axis among the places that `seen` marks; 0 throughout a row that it leaves nothing of."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, 1.0, total))


def _decode(s):
    b, hq, hkv = s["batch"], s["hq"], s["hkv"]
    lens = s["lens"].long()[:, None]
    window = s["window"] or s["block_table"].shape[1] * PAGE
    sinks = s["sinks"] if s["window"] else 0
    back = lens - 1 - torch.arange(min(window, s["block_table"].shape[1] * PAGE), device="cuda")        # the window, newest key first
    head = torch.arange(sinks, device="cuda").expand(b, -1)                                            # first keys outside of it
    at = torch.cat([back, head], 1)
    seen = torch.cat([back >= 0, head < lens - window], 1)
    slots = torch.where(seen, _slots(s["block_table"].long(), at.clamp(min=0)), 0)
    k, v = _rows(s["k_cache"], s["k_scale"], slots), _rows(s["v_cache"], s["v_scale"], slots)           # [B, n, Hkv, D]
    q = s["q"].float().view(b, hkv, hq // hkv, D)
    p = _softmax(torch.einsum("bhgd,bnhd->bhgn", q, k) * s["scale"], seen[:, None, None])
    return torch.einsum("bhgn,bnhd->bhgd", p, v).reshape(b, hq, D).to(torch.bfloat16)


def _prefill(s):
    hq, hkv, most_q, most_k = s["hq"], s["hkv"], s["max_q"], s["max_k"]
    cu_q, lens = s["cu_q"].long(), s["lens"].long()
    b, new = lens.numel(), cu_q[1:] - cu_q[:-1]
    row, key = torch.arange(most_q, device="cuda"), torch.arange(most_k, device="cuda")
    alive = row < new[:, None]                                                                          # [B, rows]
    q = s["q"][(cu_q[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)].float().view(b, most_q, hkv, hq // hkv, D)
    slots = _slots(s["block_table"].long(), key.expand(b, -1))
    k, v = _rows(s["k_cache"], s["k_scale"], slots), _rows(s["v_cache"], s["v_scale"], slots)
    at = (lens - new)[:, None, None] + row[:, None]                                                     # position of a row
    seen = key <= at
    if s["window"]:
        seen = seen & ((key > at - s["window"]) | (key < s["sinks"]))
    scores = torch.einsum("bqhgd,bnhd->bhgqn", q, k).mul_(s["scale"])
    p = _softmax(scores, seen[:, None, None])
    out = torch.einsum("bhgqn,bnhd->bqhgd", p, v).reshape(b, most_q, hq, D)
    return out[alive].to(torch.bfloat16)


def _rotated(x, cos, sin, rot, interleaved):
    x = x.float()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1).to(torch.bfloat16)


def _rotary(s):
    angle = s["positions"].double()[:, None] * s["inv_freq"]              # 64 bits: a far position leaves no digits in 32
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    q, k = (_rotated(s[x], cos, sin, s["rot"], s["interleaved"]) for x in "qk")
    slots = s["slots"].long()
    s["k_cache"].view(-1, *k.shape[1:])[slots] = k
    s["v_cache"].view(-1, *k.shape[1:])[slots] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _load(s):
    return tuple(_rows(s[c], s[e], s["slots"]).to(torch.bfloat16) for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale")))


def _own(s):
    from infer_b200 import ops
    if s["op"] == "decode":
        return ops.paged_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["block_table"], s["scale"], out=s["out"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"], window=s["window"] or None,
                                     sinks=s["sinks"] if s["window"] else 0)
    if s["op"] == "prefill":
        return ops.paged_attn_prefill(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"], s["scale"],
                                      s["block_table"], k_scale=s["k_scale"], v_scale=s["v_scale"], window=s["window"] or None,
                                      sinks=s["sinks"])
    if s["op"] == "rotary":
        q = ops.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"], s["slots"],
                              interleaved=s["interleaved"], attention_factor=s["factor"])
        return q, s["k_cache"], s["v_cache"]
    return ops.load_kvcache(s["k_cache"], s["v_cache"], s["slots"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(s):
    if own:
        return _own(s)
    return {"decode": _decode, "prefill": _prefill, "rotary": _rotary, "load": _load}[s["op"]](s)


# --------------------------------------------------------------------------- the definitions in 64 bits
def _values64(cache, scale, pages):
    """Keys or values of a sequence's pages [n, Hkv, D], in 64 bits."""
    x = cache[pages]
    x = x.double() if scale is None else x.view(torch.float8_e4m3fn).double() * scale[pages].double()[:, None, :, None]
    return x.reshape(-1, *x.shape[2:])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("decode", "prefill"):
        keys, new = _lengths(case)
        group, window, sinks = case["hq"] // case["hkv"], case["window"], case["sinks"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        done = 0
        for b, (n, m) in enumerate(zip(keys, new)):
            if n:
                pages = s["block_table"][b, :-(-n // PAGE)].long()
                k, v = (_values64(s[c], s[e], pages)[:n] for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale")))
                rows = slice(b, b + 1) if case["op"] == "decode" else slice(done, done + m)
                i = torch.arange(n - m, n, device="cuda")[:, None]
                j = torch.arange(n, device="cuda")[None]
                blocked = j > i
                if window:
                    blocked |= (i - j >= window) & (j >= sinks)
                for h in range(case["hq"]):
                    x = s["q"][rows, h].double() @ k[:, h // group].T * s["scale"]
                    x[blocked] = -math.inf
                    out[rows, h] = torch.softmax(x, -1) @ v[:, h // group]
            done += m
        return out
    if case["op"] == "load":
        slots = s["slots"].long()
        got = []
        for c, e in (("k_cache", "k_scale"), ("v_cache", "v_scale")):
            x = s[c][slots // PAGE, slots % PAGE]
            got.append(x.double() if s[e] is None else x.view(torch.float8_e4m3fn).double() * s[e].double()[slots // PAGE][..., None])
        return tuple(got)
    half = case["rot"] // 2
    first, second = (range(0, case["rot"], 2), range(1, case["rot"], 2)) if case["interleaved"] else (range(half), range(half, case["rot"]))
    first, second = torch.tensor(first, device="cuda"), torch.tensor(second, device="cuda")
    turn = torch.polar(torch.full((1, 1, 1), s["factor"], dtype=torch.float64, device="cuda"),
                       (s["positions"].double()[:, None] * s["inv_freq"])[:, None])
    got = []
    for name in "qk":
        x = s[name].double()
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        got.append(x)
    slots = s["slots"].long()
    pools = []
    for name, x in (("k_cache", got[1]), ("v_cache", s["v"].double())):
        pool = s[name].double()
        pool[slots // PAGE, slots % PAGE] = x
        pools.append(pool)
    return got[0], pools[0], pools[1]
