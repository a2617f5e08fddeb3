"""Attention over the 4-bit cache where keys and values of very different magnitudes lie side by side: what a row does not
see, or gives next to no weight, must cost it nothing of its precision."""
import math

import pytest
import torch

import mps_bitsandbytes_b200 as bnb
from gpu_util import assert_device_ok

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def reference(q, cache, layer, table, length, window=None):
    """(out, limit) in 64 bits of one sequence's last rows q [n, heads, head_dim], causal.  ``limit`` counts what a row sees and
    nothing else, a = a block's absmax:

    an element of K or V goes into its product with two fp16 roundings at most, of 2^-11 of itself each, or of 2^-25 where it is
    subnormal under a power of two that brings each block's absmax to 2^-14 at least: 2^-11 a.  bf16 queries: 2^-25 of the row's largest,
    times sum |k|.  So a score is off by e = scale sum_d (|q_d| (2^-10 |k_d| + 2^-11 a) + 2^-25 max|q| |k_d|) and a probability by a factor
    within exp(+-2 max e).  A weight is off by 2^-11 of itself, or by 2^-25 (and by no more than itself) where the key's a is 2^-4 at
    least and the row's largest power of two is 1 at least: 2^-21 a of the row's largest probability.  fp32 sums: n 2^-23, and
    2^-18 for scores and powers.
    """
    import kv_util as U
    n, H, D = q.shape
    group = H // cache.num_kv_heads
    k, v = (U.rows_of(cache, layer, table, 0, length, x) for x in "kv")
    place = torch.arange(length, device="cuda")
    page = table.long()[place // cache.page_size], place % cache.page_size
    ka, va = (getattr(cache, x + "_absmax")[layer][page[0], :, page[1] // 16, page[1] % 16].double().repeat_interleave(cache.blocksize, -1) for x in "kv")
    pos = torch.arange(length - n, length, device="cuda")[:, None]
    seen = place[None] <= pos
    if window:
        seen &= place[None] > pos - window
    out, limit = torch.zeros(n, H, D, dtype=torch.float64, device="cuda"), torch.zeros(n, H, D, dtype=torch.float64, device="cuda")
    for h in range(H):
        x, g = q[:, h].double(), h // group
        s = (x @ k[:, g].T * D ** -0.5).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, -1)
        e = D ** -0.5 * (x.abs() @ (2.0 ** -10 * k[:, g].abs() + 2.0 ** -11 * ka[:, g]).T + 2.0 ** -25 * x.abs().amax(-1, keepdim=True) * k[:, g].abs().sum(-1)[None])
        # (probabilities beyond the row's own resolution do not count)
        e = e.masked_fill(~seen | (p < 2.0 ** -40), 0.0).amax(-1, keepdim=True)
        size = p @ v[:, g].abs()
        out[:, h] = p @ v[:, g]
        limit[:, h] = (size * (torch.expm1(2 * e) + 3 * 2.0 ** -11 + length * 2.0 ** -23 + 2.0 ** -18) + p @ va[:, g] * 2.0 ** -11
                       + torch.minimum(p, 2.0 ** -21 * p.amax(-1, keepdim=True)) @ va[:, g])
    return out, limit + HALF_STEP[q.dtype] * (out.abs() + limit) + 2.0 ** -25


def close(got, want, limit):
    worst = ((got.double() - want).abs() / limit).max().item()
    assert torch.isfinite(got).all() and worst <= 1.0, f"off by {worst:.3g} of the limit"


def _cache(head_dim, blocksize, dtype, length, kv_heads, gen, quant="nf4"):
    cache = bnb.KVCache4bit(1, -(-length // 32), kv_heads, head_dim, page_size=32, blocksize=blocksize, quant_type=quant, dtype=dtype)
    table = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(length)).to(torch.int32)[None].cuda()
    k, v = (torch.randn(length, kv_heads, head_dim, generator=gen, device="cuda") for _ in range(2))
    return cache, table, k, v


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("head_dim,blocksize,heads,kv_heads,new,length", [
    (128, 64, 2, 2, 4, 100), (128, 64, 8, 2, 4, 97), (64, 32, 6, 2, 8, 333), (256, 64, 2, 1, 5, 70), (256, 32, 12, 1, 5, 64), (128, 32, 16, 1, 2, 35), (64, 64, 1, 1, 3, 40)])
@pytest.mark.parametrize("dtype,large", [(BF16, 1e10), (BF16, 1e25), (F16, 6e4)])
def test_a_drafted_token_of_any_magnitude_leaves_the_rows_before_it_alone(dtype, large, head_dim, blocksize, heads, kv_heads, new, length, side):
    gen = torch.Generator(device="cuda").manual_seed(length)
    cache, table, k, v = _cache(head_dim, blocksize, dtype, length, kv_heads, gen)
    if dtype == F16:
        k, v = k * 2.0 ** -12, v * 2.0 ** -12
    x = k if side == "k" else v
    x[-1] = large * torch.sign(x[-1])
    lens = _i32([length])
    bnb.append_kv_4bit(cache, 0, k.to(dtype), v.to(dtype), table, lens)
    q = torch.randn(new, heads, head_dim, generator=gen, device="cuda").to(dtype)
    got = bnb.attention_4bit(q[None], cache, 0, table, lens)[0]
    want, limit = reference(q, cache, 0, table[0], length)
    close(got[:-1], want[:-1], limit[:-1])
    if side == "v":
        close(got, want, limit)
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,head_dim,blocksize", [(2, 2, 128, 64), (12, 1, 64, 32), (4, 1, 256, 64)])
@pytest.mark.parametrize("dtype,sizes", [(BF16, (1e10, 1.0)), (BF16, (1.0, 1e-6)), (BF16, (1e20, 1e-6)), (F16, (6e4, 1e-3))])
def test_values_of_any_magnitude_that_have_next_to_no_weight(dtype, sizes, heads, kv_heads, head_dim, blocksize):
    """Every eighth key is far larger than the others, and so far from the queries that its weight vanishes."""
    length = 200
    gen = torch.Generator(device="cuda").manual_seed(7)
    cache, table, k, v = _cache(head_dim, blocksize, dtype, length, kv_heads, gen)
    far = torch.arange(length, device="cuda") % 8 == 3
    k, v = k * 0.05, v * sizes[1]
    k[far], v[far] = -4.0, v[far] * (sizes[0] / sizes[1])
    v = v.clamp(-sizes[0], sizes[0])
    lens = _i32([length])
    bnb.append_kv_4bit(cache, 0, k.to(dtype), v.to(dtype), table, lens)
    q = (4.0 + 0.5 * torch.randn(1, heads, head_dim, generator=gen, device="cuda")).to(dtype)
    got = bnb.attention_4bit(q, cache, 0, table, lens)
    want, limit = reference(q, cache, 0, table[0], length)
    assert limit.max() < 0.1 * sizes[1]                              # (the large ones do count for nothing)
    close(got, want, limit)


@pytest.mark.parametrize("dtype,sizes", [(BF16, (1e12, 1e-6)), (F16, (6e4, 1e-4))])
@pytest.mark.parametrize("head_dim,blocksize,heads", [(128, 64, 1), (128, 32, 12), (64, 32, 3), (256, 32, 2)])
def test_blocks_of_a_row_of_any_magnitude(dtype, sizes, head_dim, blocksize, heads):
    """The last block of every value is far smaller than the first ones: its channels are as exact as theirs."""
    length = 150
    gen = torch.Generator(device="cuda").manual_seed(8)
    cache, table, k, v = _cache(head_dim, blocksize, dtype, length, 1, gen, "fp4")
    v = v.clamp(-1, 1) * sizes[0]
    v[..., -blocksize:] *= sizes[1] / sizes[0]
    v[3::5] *= 2.0 ** -3
    lens = _i32([length])
    bnb.append_kv_4bit(cache, 0, k.to(dtype), v.to(dtype), table, lens)
    q = torch.randn(1, heads, head_dim, generator=gen, device="cuda").to(dtype)
    close(bnb.attention_4bit(q, cache, 0, table, lens), *reference(q, cache, 0, table[0], length))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_blocks_of_zeros_beside_others(dtype):
    gen = torch.Generator(device="cuda").manual_seed(9)
    cache, table, k, v = _cache(128, 32, dtype, 120, 2, gen)
    k[..., 96:], v[..., 96:], k[::7], v[::5] = 0, 0, 0, 0
    lens = _i32([120])
    bnb.append_kv_4bit(cache, 0, k.to(dtype), v.to(dtype), table, lens)
    q = torch.randn(3, 8, 128, generator=gen, device="cuda").to(dtype)
    got = bnb.attention_4bit(q[None], cache, 0, table, lens)[0]
    close(got, *reference(q, cache, 0, table[0], 120))
    assert (got[..., 96:].abs() < 1e-7).all()


#  heads, kv heads, new tokens of each sequence: keys shared out; not; prompts among single tokens
PROMPTS = [(32, 8, [150, 300, 129]), (64, 16, [100, 33, 256, 64, 1, 17, 130, 70, 90] * 2), (32, 8, [1, 1, 400, 3, 1, 2, 1, 13])]


def _prompts(head_dim, blocksize, dtype, heads, kv_heads, new, before, gen, change):
    """A cache of the sequences' keys and values, change(k, v, b) made to those of each, and what an attention call takes."""
    import kv_util as U
    page = 32
    lens = [n + before for n in new]
    width = -(-max(lens) // page)
    cache = bnb.KVCache4bit(1, len(new) * width, kv_heads, head_dim, page_size=page, blocksize=blocksize, dtype=dtype)
    table = U.widen(U.random_table(len(new), width, len(new) * width), page)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = [0]
    for n in lens:
        rows.append(rows[-1] + n)
    k, v = (torch.randn(rows[-1], kv_heads, head_dim, generator=gen, device="cuda") for _ in range(2))
    for b in range(len(new)):
        change(k[rows[b]:rows[b + 1]], v[rows[b]:rows[b + 1]], b)
    bnb.append_kv_4bit(cache, 0, k.to(dtype), v.to(dtype), table, _i32(lens), _i32(rows))
    q = torch.randn(starts[-1], heads, head_dim, generator=gen, device="cuda").to(dtype)
    return cache, table, lens, starts, q


@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("heads,kv_heads,new", PROMPTS, ids=["shared out", "whole", "mixed"])
@pytest.mark.parametrize("head_dim,blocksize,dtype,large", [(128, 64, BF16, 1e10), (128, 32, F16, 6e4), (64, 64, BF16, 1e25), (256, 64, BF16, 1e10)])
def test_a_prompts_token_of_any_magnitude_leaves_the_rows_before_it_alone(head_dim, blocksize, dtype, large, heads, kv_heads, new, side):
    gen = torch.Generator(device="cuda").manual_seed(head_dim)
    at = {b: n // 2 for b, n in enumerate(new) if n > 30 and b % 4 != 1}   # (of the new tokens)

    def change(k, v, b):
        if dtype == F16:
            k.mul_(2.0 ** -12), v.mul_(2.0 ** -12)
        if b in at:
            x = (k if side == "k" else v)[20 + at[b]]
            x.copy_(large * torch.sign(x))
    cache, table, lens, starts, q = _prompts(head_dim, blocksize, dtype, heads, kv_heads, new, 20, gen, change)
    got, lse = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new), return_lse=True)
    again, lse2 = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new), return_lse=True)
    for b, n in enumerate(new):
        rows = slice(starts[b], starts[b + 1])
        want, limit = reference(q[rows], cache, 0, table[b], lens[b])
        some = at.get(b, n) if side == "k" else n                    # (scores of 1e10 know no limit)
        close(got[rows][:some], want[:some], limit[:some])
        assert torch.equal(got[rows][:some], again[rows][:some]) and torch.equal(lse[rows][:some], lse2[rows][:some]) and torch.isfinite(lse[rows][:some]).all()
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,new", PROMPTS, ids=["shared out", "whole", "mixed"])
@pytest.mark.parametrize("head_dim,blocksize,dtype,sizes", [(128, 64, F16, (6e4, 1e-4)), (128, 32, BF16, (1e12, 1e-3)), (64, 32, BF16, (1.0, 1e-7)), (256, 32, F16, (100.0, 1e-6))])
def test_prompts_with_small_values_behind_or_beside_large_ones(head_dim, blocksize, dtype, sizes, heads, kv_heads, new):
    """Where large values lie far before the small ones, among them (with a window, of rows that see the small ones alone), or in
    another block of channels; sequences of ordinary ones beside them."""
    gen = torch.Generator(device="cuda").manual_seed(3)

    def change(k, v, b):
        if b % 3 == 1:
            return
        v.clamp_(-1, 1).mul_(sizes[1])
        if b % 3 == 0:
            v[:60] *= sizes[0] / sizes[1]
        else:
            v[..., :blocksize] *= sizes[0] / sizes[1]
        v.clamp_(-sizes[0], sizes[0])
    cache, table, lens, starts, q = _prompts(head_dim, blocksize, dtype, heads, kv_heads, new, 70, gen, change)
    got = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new), window=16)
    for b, n in enumerate(new):
        rows = slice(starts[b], starts[b + 1])
        close(got[rows], *reference(q[rows], cache, 0, table[b], lens[b], 16))
    assert_device_ok()


def test_a_graph_of_prompts_follows_magnitudes():
    """Captured over ordinary values, replayed over others and back."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    cache, table, lens, starts, q = _prompts(128, 64, BF16, 32, 8, [150, 300, 129], 20, gen, lambda k, v, b: None)
    args = (q, cache, 0, table, _i32(lens), _i32(starts), 300)
    clean = bnb.attention_4bit(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bnb.attention_4bit(*args)
    before = cache.data.clone()
    for large in (False, True, False, True):
        cache.data.copy_(before)
        if large:
            page, place = table[1, 250 // 32], 250 % 32
            cache.v_absmax[0, page, :, place // 16, place % 16] = 1e12
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        if not large:
            assert torch.equal(out, clean)
        else:
            for b, n in enumerate([150, 300, 129]):
                rows = slice(starts[b], starts[b + 1])
                close(out[rows], *reference(q[rows], cache, 0, table[b], lens[b]))
            assert torch.equal(out[:150], clean[:150]) and torch.equal(out[450:], clean[450:])
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,new", [(4, 2, [1, 3])] + PROMPTS, ids=["tokens", "shared out", "whole", "mixed"])
@pytest.mark.parametrize("head_dim,dtype,size", [(128, BF16, 2.0 ** 13), (128, BF16, 2.0 ** 30), (64, BF16, 2.0 ** 45), (256, BF16, 2.0 ** 7), (128, F16, 2.0 ** 10)])
def test_scores_of_any_size(head_dim, dtype, size, heads, kv_heads, new):
    """Every score is size^2 times +-2^(0 .. 3) times head_dim ** 0.5, many of them equal: the weights are shared by the largest that a row sees."""
    gen = torch.Generator(device="cuda").manual_seed(11)

    def change(k, v, b):
        order = torch.randint(0, 4, (k.shape[0], 1, 1), generator=gen, device="cuda")
        k.copy_(size * 2.0 ** order * torch.where(torch.arange(head_dim, device="cuda") % 3 == 0, -1.0, 1.0))
    cache, table, lens, starts, q = _prompts(head_dim, 64, dtype, heads, kv_heads, new, 20, gen, change)
    signs = torch.where(torch.arange(head_dim, device="cuda") % 3 == 0, -size, size).to(dtype)
    q[:, ::2], q[:, 1::2] = signs, -signs
    got, lse = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new), return_lse=True)
    import kv_util as U
    for b, n in enumerate(new):
        k, v = (U.rows_of(cache, 0, table[b], 0, lens[b], x) for x in "kv")
        seen = torch.arange(lens[b], device="cuda")[None] <= torch.arange(lens[b] - n, lens[b], device="cuda")[:, None]
        for h in range(heads):
            g = h // (heads // kv_heads)
            s = (q[starts[b]:starts[b + 1], h].double() @ k[:, g].T * head_dim ** -0.5).masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = (s == top).double()                                  # (the others are 2^13 at least below)
            total = p.sum(-1, keepdim=True)
            p /= total
            size_v = p @ v[:, g].abs()
            want, out = p @ v[:, g], got[starts[b]:starts[b + 1], h].double()
            limit = size_v * (3 * 2.0 ** -11 + lens[b] * 2.0 ** -23 + 2.0 ** -18) + HALF_STEP[dtype] * size_v * 1.01 + 2.0 ** -25
            worst = ((out - want).abs() / limit).max().item()
            assert torch.isfinite(out).all() and worst <= 1.0, f"off by {worst:.3g} of the limit"
            want_lse = top[:, 0] + torch.log(total[:, 0])
            assert ((lse[starts[b]:starts[b + 1], h].double() - want_lse).abs() <= 2.0 ** -9 * want_lse.abs() + 1e-3).all()
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,new", [(4, 2, [1, 3, 1])] + PROMPTS, ids=["tokens", "shared out", "whole", "mixed"])
@pytest.mark.parametrize("before,size", [(20, 3e38), (2000, 3e38), (300, 1e33)])
def test_values_up_to_the_types_largest(heads, kv_heads, new, before, size):
    """Their sum over the keys leaves fp32, their mean does not."""
    gen = torch.Generator(device="cuda").manual_seed(12)

    def change(k, v, b):
        k.mul_(0.1)
        v.copy_(size * torch.where(v > 1.0, 0.5, 1.0) * torch.where(v > 1.5, -1.0, 1.0))
    cache, table, lens, starts, q = _prompts(128, 64, BF16, heads, kv_heads, new, before, gen, change)
    got = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new))
    for b, n in enumerate(new):
        rows = slice(starts[b], starts[b + 1])
        close(got[rows], *reference(q[rows], cache, 0, table[b], lens[b]))
    assert_device_ok()


def test_one_sequence_of_many_with_magnitudes_far_apart():
    """Forty prompts, two of which have a value that the others do not: theirs are done again, whichever else are with them."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    new = [40 + 7 * (b % 9) for b in range(40)]

    def change(k, v, b):
        if b in (2, 35):
            v[-20] *= 1e12
    cache, table, lens, starts, q = _prompts(64, 64, BF16, 16, 4, new, 5, gen, change)
    got = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), max(new))
    for b, n in enumerate(new):
        rows = slice(starts[b], starts[b + 1])
        close(got[rows], *reference(q[rows], cache, 0, table[b], lens[b]))
    assert_device_ok()
