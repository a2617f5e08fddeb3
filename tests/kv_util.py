"""Plain 64-bit forms of the 4-bit key/value cache's operators, and caches with known contents, for the GPU tests."""
import math

import torch

import mps_bitsandbytes_b200 as bnb

CODE = {"nf4": bnb.NF4_CODEBOOK, "fp4": bnb.FP4_CODEBOOK}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make_cache(pages, kv_heads, head_dim, page_size=64, blocksize=64, quant="nf4", dtype=torch.float16, layers=1, seed=0,
               k_size=1.0, v_size=1.0):
    """A cache full of random codes and positive absmax values around k_size / v_size."""
    cache = bnb.KVCache4bit(layers, pages, kv_heads, head_dim, page_size=page_size, blocksize=blocksize, quant_type=quant, dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cache.data.random_(0, 256, generator=gen)
    for t, size in ((cache.k_absmax, k_size), (cache.v_absmax, v_size)):
        t.copy_(torch.exp(0.5 * torch.randn(t.shape, generator=gen, device="cuda")) * size)
    return cache


def random_table(batch, width, pages, seed=0):
    """Every entry a page of its own."""
    gen = torch.Generator().manual_seed(seed)
    assert batch * width <= pages
    return torch.randperm(pages, generator=gen)[:batch * width].view(batch, width).to(torch.int32).cuda()


def widen(table, page):
    """The table with room for 128 K places, of entries that no key needs: prompts then go to the prompt kernel."""
    wide = torch.full((table.shape[0], max(table.shape[1], (1 << 17) // page)), -1, dtype=torch.int32, device=table.device)
    wide[:, :table.shape[1]] = table
    return wide


def rows_of(cache, layer, pages, first, last, name):
    """[last - first, kv heads, head_dim] in 64 bits: the values of places first .. last - 1."""
    place = torch.arange(first, last, device="cuda")
    page, off = pages.long()[place // cache.page_size], place % cache.page_size
    codes = getattr(cache, name + "_codes")[layer][page, :, off // 16, off % 16]
    absmax = getattr(cache, name + "_absmax")[layer][page, :, off // 16, off % 16].double()
    code = CODE[cache.quant_type].double().cuda()
    x = torch.stack((code[(codes & 15).long()], code[(codes >> 4).long()]), -1).flatten(-2)
    return x * absmax.repeat_interleave(cache.blocksize, -1)


def attention(q, cache, layer, table, lens, starts, causal=True, window=None, scale=None):
    """(out, lse, bound) in 64 bits; rows that belong to no sequence are NaN.  ``bound`` is how far the kernels may be off
    before their result is rounded to the cache's type:

    an element of K or V enters its product with two fp16 roundings at most, of its code and of code * absmax: off by 2 * 2^-11
    of itself (and, under the power of two that brings the largest absmax of a tile to 2^8, by 2^-25 of that unit: 2^-33 of the
    tile's largest).  A bf16 query is exact but for parts under 2^-14 of its row's largest, off by 2^-25 of that.  So a score is off by
    e = scale (2 * 2^-11 sum_d |q_d k_d| + 2^-25 max|q| sum_d |k_d| + 2^-33 max|k| sum_d |q_d|) and a probability by a factor within
    exp(+-2 e_max) (numerator and denominator).  A weight p * absmax, or p, is rounded to fp16: by 2^-11 of itself, or, being
    small, by 2^-25 under factors that bring the largest absmax to 16 at least and the largest p to 1 (single tokens: 2^-29 of
    their product) or the largest p to 2^7 (prompts: 2^-32, and as much again for V's own 2^-33).  fp32 sums of n terms add 2^-24
    each step at most: n * 2^-23 covers numerator and denominator, and 2^-18 the scores' sums and the last bits of the exponential.
    """
    T, H, D = q.shape
    group = H // cache.num_kv_heads
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device="cuda")
    lse = torch.full((T, H), math.nan, dtype=torch.float64, device="cuda")
    bound = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        a, e = starts[b], starts[b + 1]
        n = e - a
        k, v = (rows_of(cache, layer, table[b], 0, length, x) for x in "kv")
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        seen = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if causal:
            seen &= key <= pos
        if window:
            seen &= key > pos - window
        for h in range(H):
            kk, vv, x = k[:, h // group], v[:, h // group], q[a:e, h].double()
            s = (x @ kk.T * scale).masked_fill(~seen, -math.inf)
            m = s.amax(-1, keepdim=True) if length else torch.full((n, 1), -math.inf, device="cuda", dtype=torch.float64)
            m = torch.where(m == -math.inf, 0.0, m)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            lse[a:e, h] = torch.log(total[:, 0]) + m[:, 0]
            p = p / torch.where(total == 0, 1.0, total)
            out[a:e, h] = p @ vv
            if length == 0:
                continue
            err = abs(scale) * ((x.abs() @ kk.abs().T) * 2 * 2.0 ** -11 + x.abs().amax(-1, keepdim=True) * kk.abs().sum(-1)[None] * 2.0 ** -25
                                + kk.abs().max() * x.abs().sum(-1, keepdim=True) * 2.0 ** -33)
            err = err.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            rel = torch.expm1(2 * err) + 3 * 2.0 ** -11 + length * 2.0 ** -23 + 2.0 ** -18
            small = 2.0 ** -29 * p.amax(-1, keepdim=True) * vv.abs().max()
            bound[a:e, h] = (p @ vv.abs()) * rel + length * small
    return out, lse, bound


def check(got, want, bound, dtype):
    """Every element within its bound and half a step of its own; and the whole within what roundings that do not all
    point the same way leave: half a step of the type and three of fp16's, in the root mean square."""
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any()
    got, want, bound = (x[~torch.isnan(want)] for x in (got, want, bound))
    if want.numel() == 0:
        return
    d = (got.double() - want).abs()
    limit = bound * 1.001 + HALF_STEP[dtype] * (want.abs() + bound) + 2.0 ** -25
    worst = (d / limit).max().item()
    assert worst <= 1.0, f"off by {worst:.3f} of the bound"
    rms = (d.square().mean().sqrt() / want.square().mean().sqrt()).item()
    assert rms <= HALF_STEP[dtype] + 3 * 2.0 ** -11, f"root mean square error {rms:.2e}"
