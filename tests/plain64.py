"""Plain implementations in 64 bits of the windowed attention, rotary and read-back operators, with error bounds.

``attention`` returns, next to the result, how far a kernel's bf16 result may be off, from the roundings that the kernels
make: one of every probability (``p_eps``: half a step of its type, relative), one of the result (2^-8 for bf16), and the
error of the scores, which are sums of 128 products in 32 bits: |ds| <= 130 * 2^-24 * scale * sum |q k|, doubled because a
probability is off by the errors of its own score and of the sum.  2^-20 covers the exponential and the subtraction of the
maximum (|score| below 100 in units of log 2, each step half of 2^-23 relative).  ``p_abs``: what a probability of
magnitude 1 or less may lose in absolute terms (half a step of the smallest f16 values).
"""
import torch

E_BF16, E_F16 = 2.0 ** -8, 2.0 ** -11


def visible(n_keys, positions, window, sinks):
    """[rows, keys]: which keys the queries at ``positions`` see (window None: causal alone)."""
    i, j = positions[:, None], torch.arange(n_keys, device=positions.device)[None]
    seen = j <= i
    if window is not None:
        seen = seen & ((i - j < window) | (j < sinks))
    return seen


def attention(q, k, v, seen, scale, p_eps, p_abs=0.0):
    """q [rows, Hq, D], k, v [keys, Hkv, D] -> (out, bound), both float64 [rows, Hq, D]; rows that see nothing give zeros."""
    group = q.shape[1] // k.shape[1]
    q = q.double()
    # a key that nobody sees may hold anything, NaN included
    used = seen.any(0)[:, None, None]
    k, v = torch.where(used, k.double(), 0.0), torch.where(used, v.double(), 0.0)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    ds = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()).masked_fill(~seen, 0).amax(-1).T[..., None] * scale * 130 * 2.0 ** -24
    s = s.masked_fill(~seen, -torch.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    out = torch.einsum("hqk,khd->qhd", p, v)
    weight = torch.einsum("hqk,khd->qhd", p, v.abs())
    lost = p_abs * torch.einsum("hqk,khd->qhd", seen[None].double().expand_as(p), v.abs())
    return out, E_BF16 * out.abs() + (p_eps + 2 * ds + 2.0 ** -20) * (1 + E_BF16) * weight + lost + 1e-30


def check(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: non-finite output"
    err = (got - want.cpu()).abs()
    bad = err > bound.cpu()
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values out of bounds, first at {at}: got "
                             f"{got[tuple(at)]:.6g}, want {want[tuple(at)]:.6g} +- {bound[tuple(at)]:.3g}")


def values(cache, scale, table, n):
    """The first n cached rows of a page list, [n, Hkv, D] float64."""
    bs = cache.shape[1]
    pages = torch.as_tensor(table[:-(-n // bs)], device=cache.device).long()
    # entries of pages that nobody may look at can be -1
    x = cache[pages.clamp(min=0)]
    x = x.view(torch.float8_e4m3fn).double() * scale[pages.clamp(min=0)].double()[:, None, :, None] if scale is not None else x.double()
    return x.reshape(-1, *x.shape[2:])[:n]


def rotary(x, positions, inv_freq, interleaved, factor):
    """x [T, H, D] -> (rotated, bound): bf16 rounding of the result, and 32-bit products and sums of values with 2^-21
    relative error of cosine and sine (the angle within 2^-24 of half a turn, 1 unit for sincospi, 1 for the factor)."""
    rot = 2 * inv_freq.numel()
    t = positions.double()[:, None] * inv_freq.double()
    c, s = (t.cos() * factor)[:, None], (t.sin() * factor)[:, None]
    y = x.double().clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    u, w = x.double()[..., a], x.double()[..., b]
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    bound = torch.zeros_like(y)
    # cosine and sine are off by up to 2^-21 of the factor in absolute terms, whatever their size
    slack = 2.0 ** -21 * abs(factor) * (u.abs() + w.abs())
    bound[..., a], bound[..., b] = E_BF16 * y[..., a].abs() + slack * (1 + E_BF16), E_BF16 * y[..., b].abs() + slack * (1 + E_BF16)
    return y, bound


def e4m3_pool(num_blocks, block_size, hkv, gen, spread=1.0):
    """An e4m3 pool with an amplitude of its own for every page and head -> (bytes uint8, scale fp32), on the CPU."""
    x = torch.randn(num_blocks, block_size, hkv, 128, generator=gen)
    x = x * torch.exp(spread * torch.randn(num_blocks, 1, hkv, 1, generator=gen))
    scale = x.abs().amax(dim=(1, 3)) / 448
    return (x / scale[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8), scale
