"""The paged 4-bit key/value cache on the GPU: append, read back, page copies, and attention over it, each against a plain
64-bit form (kv_util) or the repository's own quantiser, and all of them together as a server would call them."""
import math

import numpy as np
import pytest
import torch

import mps_bitsandbytes_b200 as bnb
from gpu_util import assert_device_ok
from oracle import oracle_np as O

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _starts(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------- append and read back
@pytest.mark.parametrize("quant", ["nf4", "fp4"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("head_dim,blocksize,page,kv_heads", [(128, 64, 64, 2), (64, 32, 16, 3), (256, 64, 32, 1), (128, 32, 128, 5), (64, 64, 16, 1), (256, 32, 64, 2)])
def test_append_stores_what_quantize_4bit_stores(head_dim, blocksize, page, kv_heads, dtype, quant):
    import kv_util as U
    new, lens = [5, 0, 1, 37, 70], [5, 9, 40, 50, 133]
    starts = _starts(new)
    T, width = starts[-1] + 3, 133 // page + 1                      # three rows past the last sequence
    cache = U.make_cache(5 * width + 2, kv_heads, head_dim, page, blocksize, quant, dtype, layers=2)
    before = cache.data.clone()
    table = U.random_table(5, width, 5 * width + 2, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(T, kv_heads, head_dim, generator=gen, device="cuda").to(dtype)
    v = (torch.randn(T, kv_heads, head_dim, generator=gen, device="cuda") * 3e-3).to(dtype)
    k[2, 0] = 0.0                                                   # a block of zeros
    v[0, -1, :blocksize] = torch.finfo(dtype).max
    v[1, 0, ::3] = 2.0 ** -24                                       # fp16's smallest
    bnb.append_kv_4bit(cache, 1, k, v, table, _i32(lens), _i32(starts))
    assert torch.equal(cache.data[0], before[0])
    touched = torch.zeros(cache.num_pages, page, dtype=torch.bool)
    for x, name in ((k, "k"), (v, "v")):
        src = x.float().cpu().numpy().reshape(-1, head_dim)
        packed, absmax, _ = O.quantize_4bit(src, blocksize, quant)
        packed = packed.reshape(T, kv_heads, head_dim // 2)
        absmax = torch.from_numpy(absmax).to(dtype).view(T, kv_heads, -1)
        own, state = bnb.quantize_4bit(x.reshape(-1, head_dim), blocksize=blocksize, quant_type=quant)
        assert np.array_equal(own.cpu().numpy().reshape(packed.shape), packed)
        codes, scales = getattr(cache, name + "_codes")[1].cpu().numpy(), getattr(cache, name + "_absmax")[1].cpu()
        for b, (n, length) in enumerate(zip(new, lens)):
            for i in range(n):
                place = length - n + i
                pg, off = int(table[b, place // page]), place % page
                touched[pg, off] = True
                assert np.array_equal(codes[pg, :, off // 16, off % 16], packed[starts[b] + i]), (name, b, i)
                assert torch.equal(scales[pg, :, off // 16, off % 16], absmax[starts[b] + i]), (name, b, i)
    # nothing else has changed
    for name in ("k_codes", "v_codes", "k_absmax", "v_absmax"):
        now = getattr(cache, name)[1].flatten(2, 3)
        saved, cache.data = cache.data, before
        half, codes_bytes = cache.data.shape[-1] // 2, 16 * head_dim // 2
        old = cache.data[1][..., (half if name[0] == "v" else 0):][..., :half]
        old = old[..., :codes_bytes] if "codes" in name else old[..., codes_bytes:].view(dtype)
        old = old.unflatten(-1, (16, -1)).flatten(2, 3)
        cache.data = saved
        same = (now.view(torch.uint8) == old.view(torch.uint8)).all(-1)                  # pages, heads, places
        assert same.transpose(1, 2)[~touched.cuda()].all(), name
    assert_device_ok()


@pytest.mark.parametrize("dtype,head_dim,blocksize,page", [(F16, 128, 64, 64), (BF16, 64, 32, 16), (BF16, 256, 64, 128)])
def test_read_back_is_dequantize_4bit(dtype, head_dim, blocksize, page):
    import kv_util as U
    lens = [77, 0, 16, 1, 130]
    width = 160 // page + 1
    cache = U.make_cache(5 * width, 3, head_dim, page, blocksize, "nf4", dtype, layers=2, seed=4)
    table = U.random_table(5, width, 5 * width)
    k, v = bnb.dequantize_kv_4bit(cache, 1, table, _i32(lens), 130)
    assert k.shape == (5, 130, 3, head_dim) and k.dtype == dtype
    for x, name in ((k, "k"), (v, "v")):
        for b, length in enumerate(lens):
            want = U.rows_of(cache, 1, table[b], 0, length, name)
            # the product of a 24-bit code and an 11-bit absmax is rounded to 24 bits and then to the type
            assert torch.equal(x[b, :length], want.float().to(dtype))
            assert (x[b, length:] == 0).all()
    short, _ = bnb.dequantize_kv_4bit(cache, 1, table, _i32(lens), 7)
    assert torch.equal(short, k[:, :7])
    whole, _ = bnb.dequantize_kv_4bit(cache, 1, table, _i32(lens))
    assert whole.shape[1] == width * page and torch.equal(whole[:, :130], k)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_then_read_back_equals_the_roundtrip_of_quantize_4bit(dtype):
    cache = bnb.KVCache4bit(1, 6, 4, 128, dtype=dtype)
    x = torch.randn(1, 100, 4, 128, device="cuda").to(dtype)
    table, lens = _i32([[4, 1]]), _i32([100])
    bnb.append_kv_4bit(cache, 0, x, x * 0.5, table, lens)
    k, v = bnb.dequantize_kv_4bit(cache, 0, table, lens, 100)
    for got, src in ((k, x), (v, x * 0.5)):
        want = bnb.dequantize_4bit(*bnb.quantize_4bit(src.reshape(-1, 128)))
        assert torch.equal(got.reshape(-1, 128), want)


def test_append_takes_strided_rows_and_uneven_addresses():
    qkv = torch.randn(2, 9, 12, 64, device="cuda", dtype=F16)              # 8 query heads, 2 of k, 2 of v
    table, lens = _i32([[0], [1]]), _i32([9, 12])
    a, b = (bnb.KVCache4bit(1, 2, 2, 64, blocksize=32, page_size=16) for _ in range(2))
    bnb.append_kv_4bit(a, 0, qkv[:, :, 8:10], qkv[:, :, 10:], table, lens)
    bnb.append_kv_4bit(b, 0, qkv[:, :, 8:10].contiguous(), qkv[:, :, 10:].contiguous(), table, lens)
    assert torch.equal(a.data, b.data) and a.data.any()
    flat = torch.empty(2 * 9 * 2 * 64 + 1, device="cuda", dtype=F16)
    odd = flat[1:].view(2, 9, 2, 64)
    odd.copy_(qkv[:, :, 8:10])
    wide = torch.zeros(2, 9, 2, 65, device="cuda", dtype=F16)
    wide[..., :64] = qkv[:, :, 10:]
    b.data.zero_()
    bnb.append_kv_4bit(b, 0, odd, wide[..., :64], table, lens)
    assert torch.equal(a.data, b.data)


def test_non_finite_rows_poison_their_block_only():
    cache = bnb.KVCache4bit(1, 1, 1, 128, page_size=16)
    k = torch.randn(3, 1, 128, device="cuda", dtype=F16)
    k[0, 0, 3], k[1, 0, 70] = math.inf, math.nan
    table, lens = _i32([[0]]), _i32([3])
    bnb.append_kv_4bit(cache, 0, k, torch.zeros_like(k), table, lens)
    got, zero = bnb.dequantize_kv_4bit(cache, 0, table, lens, 3)
    bad = torch.isnan(got[0, :, 0])
    want = torch.zeros(3, 128, dtype=torch.bool, device="cuda")
    want[0, :64] = want[1, 64:] = True
    assert torch.equal(bad, want) and (zero == 0).all()


# ---------------------------------------------------------------------- page copies
@pytest.mark.parametrize("pages,n,layers,head_dim,page,kv_heads", [(5, 2, 3, 128, 64, 2), (80, 40, 1, 64, 16, 1), (1200, 600, 2, 64, 16, 3), (9, 1, 2, 256, 128, 8)])
def test_copy_pages(pages, n, layers, head_dim, page, kv_heads):
    cache = bnb.KVCache4bit(layers, pages, kv_heads, head_dim, page_size=page)
    cache.data.random_(0, 256)
    want = cache.data.clone()
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(pages)).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]                                                # one page to two places
    want[:, dst] = want[:, src]
    bnb.copy_kv_pages_4bit(cache, src, dst)
    assert torch.equal(cache.data, want)
    bnb.copy_kv_pages_4bit(cache, [], [])
    with pytest.raises(ValueError, match="written twice"):
        bnb.copy_kv_pages_4bit(cache, [0, 1], [2, 2])
    with pytest.raises(ValueError, match="both source and destination"):
        bnb.copy_kv_pages_4bit(cache, [0, 1], [1, 2])
    with pytest.raises(IndexError, match="outside the cache"):
        bnb.copy_kv_pages_4bit(cache, [0], [pages])
    with pytest.raises(ValueError, match="2 source pages but 1"):
        bnb.copy_kv_pages_4bit(cache, [0, 1], [2])
    assert torch.equal(cache.data, want)


# ---------------------------------------------------------------------- attention
#  head_dim, blocksize, page, quant, dtype, heads, kv heads, new, lens, causal, window
CASES = [
    (128, 64, 64, "nf4", F16, 8, 8, [1], [1], True, None),
    (128, 64, 64, "nf4", F16, 8, 1, [1, 1, 1], [17, 64, 300], True, None),
    (128, 64, 64, "fp4", BF16, 16, 2, [1] * 4, [16, 15, 129, 1000], True, None),
    (128, 64, 16, "nf4", BF16, 6, 2, [1] * 3, [5000, 3, 777], True, None),
    (64, 32, 16, "nf4", F16, 3, 3, [1] * 2, [63, 65], True, None),
    (64, 64, 32, "fp4", BF16, 12, 1, [4, 2, 3], [100, 2, 3001], True, 63),
    (64, 32, 128, "nf4", F16, 5, 1, [3], [2000], True, 1),
    (256, 64, 64, "nf4", F16, 4, 2, [1, 1], [513, 90], True, None),
    (256, 32, 32, "fp4", BF16, 16, 1, [1, 2], [700, 33], True, 100),
    (256, 32, 32, "nf4", F16, 16, 2, [1, 2], [700, 333], True, None),
    (128, 32, 64, "nf4", BF16, 24, 2, [1, 1], [400, 41], True, None),          # 12 rows a head: 16-row tiles
    (128, 64, 64, "nf4", F16, 40, 1, [1], [1500], True, None),                 # 40 rows: three tiles
    (128, 64, 64, "nf4", F16, 7, 7, [5, 1, 0, 8], [5, 33, 20, 100], True, None),
    (128, 64, 64, "nf4", F16, 8, 2, [37, 64, 1], [37, 150, 90], True, None),   # short prompts
    (64, 64, 16, "nf4", BF16, 4, 4, [33, 16], [33, 500], True, 17),
    (128, 64, 64, "fp4", F16, 8, 2, [130], [1040], False, None),
    (128, 64, 64, "nf4", BF16, 8, 2, [300, 129, 257, 2], [300, 700, 257, 900], True, None),
    (256, 64, 64, "nf4", BF16, 6, 2, [200, 140], [333, 140], True, None),
    # prompts: 16-row tiles of all sequences and heads above 700, 430, 225 for head_dim 64, 128, 256
    (128, 64, 64, "nf4", BF16, 32, 8, [300, 129, 257, 2], [300, 700, 257, 900], True, None),
    (64, 64, 64, "nf4", F16, 24, 8, [260, 513], [260, 600], True, 200),
    (256, 64, 64, "nf4", BF16, 24, 8, [200, 140], [333, 140], True, None),
    (128, 32, 16, "fp4", F16, 40, 8, [201], [444], True, None),
    (64, 32, 32, "nf4", BF16, 24, 8, [500], [500], False, None),
    (256, 32, 128, "fp4", F16, 16, 8, [257, 300], [1000, 300], True, 129),
    (128, 64, 128, "fp4", BF16, 56, 8, [37, 130, 128], [1037, 130, 1000], True, 1),
    (128, 32, 64, "nf4", BF16, 12, 4, [513, 700], [515, 1500], True, 300),
    (64, 64, 16, "fp4", BF16, 16, 16, [700, 1], [701, 5], True, None),
    (256, 32, 64, "nf4", BF16, 8, 1, [511], [900], False, None),
    (128, 64, 32, "nf4", F16, 8, 8, [900, 0, 1100], [900, 20, 1111], True, None),
    # ... and more blocks of rows than two rounds over the card
    (128, 64, 64, "nf4", BF16, 64, 16, [100, 33, 256, 64, 1, 17, 0, 130, 70, 90] * 2, [177, 33, 400, 64, 5, 99, 50, 131, 700, 90] * 2, True, None),
    (128, 32, 32, "fp4", F16, 32, 16, [140, 99] * 10, [200, 99] * 10, True, 70),
    (64, 64, 16, "nf4", F16, 32, 16, [200, 301] * 7, [200, 310] * 7, False, None),
    (64, 32, 64, "nf4", BF16, 16, 16, [513, 400, 300, 600] * 3, [513, 499, 300, 601] * 3, True, None),
    (256, 64, 64, "fp4", BF16, 32, 16, [65, 129, 64] * 4, [190, 140, 64] * 4, True, None),
    (256, 32, 16, "nf4", F16, 16, 16, [130, 260, 190, 129] * 2, [131, 300, 250, 129] * 2, True, 150),
    # an item shared by many blocks
    (128, 64, 64, "nf4", F16, 16, 1, [33], [20000], True, None),
    (256, 64, 64, "nf4", BF16, 8, 1, [16, 40], [9000, 40], True, 5000),
    (64, 32, 16, "fp4", BF16, 20, 1, [50, 1, 13], [50, 700, 8000], False, None),
    # prompts among single tokens and drafts: both kernels in a call (the first: keys shared out; the last: more pairs than that looks through)
    (128, 64, 64, "nf4", BF16, 32, 8, [1, 1, 400, 3, 1, 0, 1, 13], [700, 20, 555, 90, 1000, 40, 3, 13], True, None),
    (256, 32, 32, "fp4", F16, 8, 2, [1, 2, 1, 1, 300, 1, 1, 9, 1], [300, 20, 77, 90, 500, 1, 640, 200, 33], True, 90),
    (64, 64, 16, "nf4", F16, 48, 8, [2, 1, 1, 1, 1, 900, 14, 1, 1, 1] * 4, [70, 500, 33, 1, 90, 900, 400, 64, 65, 17] * 4, True, None),
    (128, 32, 64, "nf4", F16, 40, 4, [1] * 40 + [700, 11, 5] + [1] * 40, list(range(1, 41)) + [900, 11, 600] + list(range(40, 400, 9)), True, None),
]


def _kernel(case, sms, places):
    """Which kernel the case's shape should go to: by 16-row tiles and blocks of 256 (128) rows of all sequences and heads, and by the
    places that the table has room for."""
    head_dim, new, kv_heads, group, window = case[0], case[7], case[6], case[5] // case[6], case[10]
    rows, lists, block = -(-sum(new) * group // len(new)), len(new) * kv_heads, 128 if head_dim == 256 else 256
    blocks, tiles = lists * -(-rows // block), lists * -(-rows // 16)
    meet, sooner = {64: (4.7, 570e3), 128: (2.9, 450e3), 256: (1.5, 50e3)}[head_dim]
    split = lists * -(-max(new) * group // block) <= 2 * sms
    keys = min(places, window + max(new)) if window else places
    if rows <= 16 or keys * (tiles - meet * (blocks if split else -(-blocks // sms) * sms)) <= sooner:
        return "tokens"
    return "prompts, split" if split else "prompts"


def test_all_kernels_are_covered():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    kinds = [(_kernel(c, sms, 1 << 17), c[0], c[1]) for c in CASES] + [(_kernel(c, sms, max(c[8])), c[0], c[1]) for c in CASES]
    assert set(kinds) == {(k, d, b) for k in ("tokens", "prompts", "prompts, split") for d in (64, 128, 256) for b in (32, 64)}


def _problem(case, seed=0, k_size=1.0, v_size=1.0):
    import kv_util as U
    head_dim, blocksize, page, quant, dtype, heads, kv_heads, new, lens, causal, window = case
    width = max(-(-max(lens) // page), 1)
    cache = U.make_cache(len(lens) * width + 1, kv_heads, head_dim, page, blocksize, quant, dtype, layers=2, seed=seed, k_size=k_size, v_size=v_size)
    table = U.random_table(len(lens), width, len(lens) * width + 1, seed)
    starts = _starts(new)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(starts[-1], heads, head_dim, generator=gen, device="cuda").to(dtype)
    return cache, table, starts, q


@pytest.mark.parametrize("case", CASES, ids=[f"d{c[0]}b{c[1]}p{c[2]}-{c[3]}-{str(c[4])[6:]}-h{c[5]}of{c[6]}-{len(c[7])}x{max(c[7])}of{max(c[8])}-{'w%s' % c[10] if c[10] else 'causal' if c[9] else 'full'}" for c in CASES])
def test_attention(case):
    import kv_util as U
    cache, table, starts, q = _problem(case)
    new, lens, causal, window = case[7:]
    want, want_lse, bound = U.attention(q, cache, 1, table, lens, starts, causal, window)
    for table in (table, U.widen(table, case[2])):                   # prompts: both kernels
        got, lse = bnb.attention_4bit(q, cache, 1, table, _i32(lens), _i32(starts), max(new), causal, window, return_lse=True)
        U.check(got, want, bound, case[4])
        # scores are off by about 2^-11 of sum |q k| / sqrt(D) at most
        err = 2.0 ** -11 * 16 + 2.0 ** -20 * want_lse.abs()
        assert ((lse.double() - want_lse).abs() <= err).all()
        again = bnb.attention_4bit(q, cache, 1, table, _i32(lens), _i32(starts), max(new), causal, window)
        assert torch.equal(got, again)                               # same bits each time
        if len(set(new)) == 1:
            even = bnb.attention_4bit(q.view(len(new), new[0], *q.shape[1:]), cache, 1, table, _i32(lens), causal=causal, window=window)
            assert torch.equal(even.flatten(0, 1), got)
    assert_device_ok()


@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (128, 8, 1), (256, 4, 2), (64, 48, 8), (128, 24, 4)])
def test_many_sequences_of_all_kinds(head_dim, heads, kv_heads):
    """More blocks of rows than there are SMs, in an order that mixes sequences with one and with two row tiles, without new tokens,
    without keys, and shorter than their new tokens."""
    import random
    import kv_util as U
    rng = random.Random(head_dim)
    news = [rng.choice([0, 1, 5, 16, 30, 31, 40, 64, 70, 100, 129]) for _ in range(180)]
    lens = [rng.choice([0, n // 2, n, n, n + rng.randint(0, 60), rng.randint(0, 160)]) for n in news]
    starts = _starts(news)
    cache = U.make_cache(180 * 6, kv_heads, head_dim, 32, seed=6)
    table = U.widen(U.random_table(180, 6, 180 * 6), 32)
    q = torch.randn(starts[-1], heads, head_dim, device="cuda", dtype=F16)
    for window in (None, 23):
        want, want_lse, bound = U.attention(q, cache, 0, table, lens, starts, window=window)
        got, lse = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), 129, window=window, return_lse=True)
        U.check(got, want, bound, F16)
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,new", [(8, 2, 6), (8, 2, 200), (48, 8, 200)])
def test_rows_without_keys_are_zero_and_rows_past_the_last_sequence_stay(heads, kv_heads, new):
    import kv_util as U
    # lengths 0; shorter than the new tokens; none new; whole
    news, lens = [2, new, 0, 3, new], [0, 4, 30, 3, new + 100]
    starts = _starts(news)
    cache = U.make_cache(5 * 5, kv_heads, 128, seed=2)
    table = U.widen(U.random_table(5, 5, 25), 64)
    q = torch.randn(starts[-1] + 4, heads, 128, device="cuda", dtype=F16)
    want, want_lse, bound = U.attention(q, cache, 0, table, lens, starts)
    out = torch.full_like(q, 7.0)
    got, lse = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), new, out=out, return_lse=True)
    assert got is out and (out[starts[-1]:] == 7.0).all()
    n = starts[-1]
    U.check(got[:n], want[:n], bound[:n], F16)
    empty = torch.isinf(want_lse[:n])
    assert empty.sum() == (2 + new - 4) * heads
    assert (got[:n][empty] == 0).all() and torch.equal(torch.isinf(lse[:n]), empty) and (lse[:n][empty] < 0).all()
    fresh = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), new)
    assert (fresh[n:] == 0).all() and torch.equal(fresh[:n], got[:n])


@pytest.mark.parametrize("new,kv_heads", [(1, 2), (150, 2), (150, 8)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_what_lies_in_unseen_places_does_not_matter(dtype, new, kv_heads):
    import kv_util as U
    lens, window = [200, 333], 90
    cache = U.make_cache(13, kv_heads, 128, dtype=dtype, seed=5)
    table = U.widen(U.random_table(2, 6, 13, seed=1), 64)
    q = torch.randn(2, new, 4 * kv_heads, 128, device="cuda").to(dtype)
    clean = bnb.attention_4bit(q, cache, 0, table, _i32(lens), window=window)
    bad = torch.ones(13, 64, dtype=torch.bool, device="cuda")       # pages, places
    for b, length in enumerate(lens):
        for place in range(max(0, length - new - window + 1), length):
            bad[table[b, place // 64], place % 64] = False
    bad = bad.view(13, 4, 16)
    for t, value in ((cache.k_absmax, math.nan), (cache.v_absmax, math.inf)):
        t[0].permute(0, 2, 3, 1, 4)[bad] = value
    # entries of the table that no key needs may hold anything
    table[0, 4:], table[1, 6:] = 1 << 30, -5
    assert torch.equal(bnb.attention_4bit(q, cache, 0, table, _i32(lens), window=window), clean)
    assert_device_ok()


@pytest.mark.parametrize("new,kv_heads", [(1, 2), (130, 2), (130, 8)])
@pytest.mark.parametrize("k_size,v_size,scale", [(1e-20, 1e-30, None), (0.05, 1e30, None), (30.0, 1e-3, 0.02), (1.0, 1.0, 0.0), (1.0, 1.0, -0.1)])
def test_magnitudes_and_scales(new, kv_heads, k_size, v_size, scale):
    import kv_util as U
    case = (128, 64, 64, "nf4", BF16, 4 * kv_heads, kv_heads, [new, new], [400, 1100], True, None)
    cache, table, starts, q = _problem(case, 3, k_size, v_size)
    table = U.widen(table, 64)
    # values of very different size beside one another, the first of them the largest by far
    cache.v_absmax[:, :, :, 0, 0] *= 2.0 ** 6
    cache.v_absmax[:, :, :, 1:] *= 2.0 ** -6
    want, _, bound = U.attention(q, cache, 1, table, case[8], starts, scale=scale)
    got = bnb.attention_4bit(q, cache, 1, table, _i32(case[8]), _i32(starts), new, scale=scale)
    assert torch.isfinite(got).all()
    d = (got.double() - want).abs()
    assert (d <= bound * 1.001 + 2.0 ** -8 * (want.abs() + bound) + 1e-37).all()


# (keys of 2^20 are infinities in fp16, and every row is NaN)
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -12, 2.0 ** 14])
def test_small_and_large_fp16_queries(size):
    import kv_util as U
    case = (64, 64, 64, "fp4", F16, 4, 2, [1, 1], [100, 30], True, None)
    cache, table, starts, q = _problem(case, 3, 1 / size)
    q = (q.float() * size).to(F16)
    want, _, bound = U.attention(q, cache, 1, table, case[8], starts)
    U.check(bnb.attention_4bit(q, cache, 1, table, _i32(case[8])), want, bound, F16)


@pytest.mark.parametrize("new,kv_heads", [(1, 2), (140, 2), (140, 8)])
def test_a_page_outside_the_cache_gives_nan_and_a_status(new, kv_heads):
    import ctypes as C
    import kv_util as U
    from mps_bitsandbytes_b200 import _native as N
    cache = U.make_cache(9, kv_heads, 128)
    table = U.widen(U.random_table(3, 3, 9), 64)
    q = torch.randn(3, new, 4 * kv_heads, 128, device="cuda", dtype=F16)
    lens = _i32([150, 190, 150])
    clean = bnb.attention_4bit(q, cache, 0, table, lens)
    st = C.c_int(0)
    for value in (9, -1, 1 << 30):
        bad = table.clone()
        bad[1, 1] = value                                            # places 64 .. 127 of the second sequence
        got = bnb.attention_4bit(q, cache, 0, bad, lens)
        seen = torch.arange(190 - new, 190, device="cuda") >= 64
        assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
        assert torch.isnan(got[1][seen]).all() and torch.equal(got[1][~seen], clean[1][~seen])
        assert N.lib().mpsbnb_device_status(C.byref(st), 1) == 0 and st.value == 401
        k, v = bnb.dequantize_kv_4bit(cache, 0, bad, lens, 190)
        assert torch.isnan(k[1, 64:128]).all() and torch.isnan(v[1, 64:128]).all() and torch.isfinite(k[1, 128:]).all()
        assert N.lib().mpsbnb_device_status(C.byref(st), 1) == 0 and st.value == 401
        before = cache.data.clone()
        x = torch.randn(3, 100, kv_heads, 128, device="cuda", dtype=F16)
        bnb.append_kv_4bit(cache, 0, x, x, bad, lens)
        assert N.lib().mpsbnb_device_status(C.byref(st), 1) == 0 and st.value == 401
        assert torch.equal(cache.data[0, table[1, 1].item()], before[0, table[1, 1].item()])
        cache.data.copy_(before)
    assert_device_ok()


def test_lengths_beyond_the_table_are_cut():
    import kv_util as U
    cache = U.make_cache(4, 1, 64, 16)
    table = U.random_table(2, 2, 4)
    q = torch.randn(2, 1, 4, 64, device="cuda", dtype=F16)
    cut = bnb.attention_4bit(q, cache, 0, table, _i32([32, 7]))
    assert torch.equal(bnb.attention_4bit(q, cache, 0, table, _i32([1000, 7])), cut)
    assert (bnb.attention_4bit(q, cache, 0, table, _i32([-4, 7]))[0] == 0).all()
    assert (bnb.attention_4bit(q, cache, 0, table[:, :0], _i32([5, 7])) == 0).all()


def test_strided_queries_and_tables():
    import kv_util as U
    cache = U.make_cache(8, 2, 64)
    big = U.random_table(2, 4, 8)
    qkv = torch.randn(2, 3, 12, 64, device="cuda", dtype=F16)
    lens = _i32([60, 200])
    want = bnb.attention_4bit(qkv[:, :, :8].contiguous(), cache, 0, big, lens)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:7] = big
    assert torch.equal(bnb.attention_4bit(qkv[:, :, :8], cache, 0, wide[:, 3:7], lens), want)
    odd = torch.empty(2 * 3 * 8 * 64 + 1, device="cuda", dtype=F16)[1:].view(2, 3, 8, 64)
    odd.copy_(qkv[:, :, :8])
    assert torch.equal(bnb.attention_4bit(odd, cache, 0, big, lens), want)
    wide_rows = torch.zeros(2, 3, 8, 66, device="cuda", dtype=F16)
    wide_rows[..., :64] = qkv[:, :, :8]
    assert torch.equal(bnb.attention_4bit(wide_rows[..., :64], cache, 0, big, lens), want)


@pytest.mark.parametrize("new", [1, 70])
def test_output_over_the_queries_and_windows_of_any_size(new):
    import kv_util as U
    cache = U.make_cache(24, 2, 128, seed=4)
    table = U.widen(U.random_table(3, 8, 24), 64)
    q = torch.randn(3, new, 32, 128, device="cuda", dtype=F16)
    lens = _i32([500, 70, 333])
    want = bnb.attention_4bit(q, cache, 0, table, lens)
    for window in (1 << 20, 1 << 30, 1 << 31, (1 << 32) + 1):
        assert torch.equal(bnb.attention_4bit(q, cache, 0, table, lens, window=window), want)
    with pytest.raises(RuntimeError, match="attention_4bit failed"):
        bnb.attention_4bit(q, cache, 0, table, lens, scale=math.nan)
    for _ in range(3):
        x = q.clone()
        assert bnb.attention_4bit(x, cache, 0, table, lens, out=x) is x and torch.equal(x, want)


def test_offsets_beyond_32_bits():
    import kv_util as U
    # a page is 2 * 256 * 36 * 8 bytes (147 KB); 3 layers of 12000 pages: 5.3 GB
    cache = bnb.KVCache4bit(3, 12000, 8, 64, page_size=256, blocksize=32)
    small = U.make_cache(6, 8, 64, 256, 32)
    table = _i32([[11999, 0, 7777], [11998, 6000, 1]])
    cache.data[2, table.flatten().long()] = small.data[0]
    q = torch.randn(2, 1, 16, 64, device="cuda", dtype=F16)
    lens = _i32([700, 513])
    want = bnb.attention_4bit(q, small, 0, _i32([[0, 1, 2], [3, 4, 5]]), lens)
    assert torch.equal(bnb.attention_4bit(q, cache, 2, table, lens), want)
    q = torch.randn(2, 400, 16, 64, device="cuda", dtype=F16)         # 16 lists of 50 row tiles: the prompt kernel
    want = bnb.attention_4bit(q, small, 0, U.widen(_i32([[0, 1, 2], [3, 4, 5]]), 256), lens)
    assert torch.equal(bnb.attention_4bit(q, cache, 2, U.widen(table, 256), lens), want)
    k, _ = bnb.dequantize_kv_4bit(cache, 2, table, lens, 700)
    assert torch.equal(k, bnb.dequantize_kv_4bit(small, 0, _i32([[0, 1, 2], [3, 4, 5]]), lens, 700)[0])
    x = torch.randn(2, 9, 8, 64, device="cuda", dtype=F16)
    bnb.append_kv_4bit(cache, 2, x, x, table, lens)
    bnb.append_kv_4bit(small, 0, x, x, _i32([[0, 1, 2], [3, 4, 5]]), lens)
    assert torch.equal(cache.data[2, table.flatten().long()], small.data[0])
    bnb.copy_kv_pages_4bit(cache, [11999], [11000])
    assert torch.equal(cache.data[:, 11000], cache.data[:, 11999]) and cache.data[2, 11000].any()


@pytest.mark.parametrize("new", [1, 45, 700])                        # each kernel
def test_graph_replays_follow_lengths_and_two_graphs_do_not_share_workspaces(new):
    import kv_util as U
    cache = U.make_cache(33, 8, 128)
    table = U.widen(U.random_table(2, 16, 33), 64)
    q = [torch.randn(2, new, 64, 128, device="cuda", dtype=F16) for _ in range(2)]
    lens = [_i32([700, 40]), _i32([3, 1000])]
    eager = lambda i: bnb.attention_4bit(q[i], cache, 0, table, lens[i])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager(0), eager(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager(i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(4):
        for i in range(2):
            lens[i].copy_(_i32([100 * step + 1 + i, 1000 - 99 * step]))
            q[i].normal_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager(i))
    assert_device_ok()


@pytest.mark.parametrize("new", [1, 60, 3000])                       # each kernel
def test_calls_on_two_streams_at_once(new):
    import kv_util as U
    cache = U.make_cache(65, 4, 128)
    table = U.widen(U.random_table(1, 64, 65), 64)
    qs = [torch.randn(1, new, 32, 128, device="cuda", dtype=F16) for _ in range(2)]
    lens = [_i32([4000]), _i32([3333])]
    want = [bnb.attention_4bit(q, cache, 0, table, n) for q, n in zip(qs, lens)]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(bnb.attention_4bit(qs[i], cache, 0, table, lens[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


def test_refusals():
    cache = bnb.KVCache4bit(1, 4, 2, 128)
    table, lens = _i32([[0, 1], [2, 3]]), _i32([3, 4])
    q = torch.zeros(2, 1, 8, 128, device="cuda", dtype=F16)
    ok = lambda **kw: bnb.attention_4bit(**{**dict(q=q, cache=cache, layer=0, page_table=table, seq_lens=lens), **kw})
    ok()
    for kw, err, match in [
            (dict(q=q.cpu()), ValueError, "must be on cuda"), (dict(q=q.bfloat16()), ValueError, "cache's dtype"), (dict(q=q[..., :64]), ValueError, "must be"),
            (dict(q=q[:, :, :7]), ValueError, "do not divide"), (dict(q=q[0, 0]), ValueError, "must be"), (dict(layer=1), IndexError, "layer 1"),
            (dict(page_table=table.long()), ValueError, "int32"), (dict(page_table=table.cpu()), ValueError, "int32"), (dict(page_table=table[0]), ValueError, "int32"),
            (dict(page_table=table[:1].expand(2, 2)), ValueError, "distinct rows"), (dict(page_table=table.t()), ValueError, "contiguous"),
            (dict(seq_lens=lens[:1]), ValueError, "2 rows, seq_lens 1"), (dict(seq_lens=lens.float()), ValueError, "int32"),
            (dict(cu_seqlens=lens), ValueError, "need 3"), (dict(q=q[:1].repeat(3, 1, 1, 1)), ValueError, "cu_seqlens is needed"), (dict(max_seqlen=2), ValueError, "max_seqlen is 2"),
            (dict(window=0), ValueError, "window"), (dict(window=3, causal=False), ValueError, "window"), (dict(q=q.clone().requires_grad_()), RuntimeError, "no backward"),
            (dict(out=q[:1]), ValueError, "out must be"), (dict(out=q.float()), ValueError, "out must be"), (dict(out=torch.zeros(2, 8, 1, 128, device="cuda", dtype=F16).transpose(1, 2)), None, None)]:
        if err is None:
            continue
        with pytest.raises(err, match=match):
            ok(**kw)
    k = torch.zeros(2, 1, 2, 128, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="same shape"):
        bnb.append_kv_4bit(cache, 0, k, k[:, :0], table, lens)
    with pytest.raises(ValueError, match="with 2 heads"):
        bnb.append_kv_4bit(cache, 0, q, q, table, lens)
    with pytest.raises(ValueError, match="max_len"):
        bnb.dequantize_kv_4bit(cache, 0, table, lens, -1)
    with torch.no_grad():
        ok(q=q.clone().requires_grad_())


# ---------------------------------------------------------------------- all together
@pytest.mark.parametrize("dtype,quant", [(F16, "nf4"), (BF16, "fp4")])
def test_a_server_run(dtype, quant):
    """Prompts, tokens, a fork, drafted tokens that are dropped again, a sequence that ends, gaps that are closed: the
    outputs at each step are those of a plain cache that keeps each sequence's dequantised rows by itself."""
    import kv_util as U
    layers, H, HK, D = 2, 8, 2, 128
    cache = bnb.KVCache4bit(layers, 24, HK, D, page_size=32, quant_type=quant, dtype=dtype)
    plain = {}                                                       # sequence -> layer -> ([n, HK, D] k, v) as stored
    gen = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)

    def roundtrip(x):
        return bnb.dequantize_4bit(*bnb.quantize_4bit(x.reshape(-1, D), quant_type=quant)).view(x.shape)

    def step(ids, counts):
        cache.extend(ids, counts)
        table, lens = cache.batch(ids)
        starts = _starts(counts)
        for layer in range(layers):
            k, v, q = rand(starts[-1], HK, D), rand(starts[-1], HK, D), rand(starts[-1], H, D)
            bnb.append_kv_4bit(cache, layer, k, v, table, lens, _i32(starts))
            got = bnb.attention_4bit(q, cache, layer, table, lens, _i32(starts), max(counts))
            kd, vd = bnb.dequantize_kv_4bit(cache, layer, table, lens)
            for b, i in enumerate(ids):
                a, e = starts[b], starts[b + 1]
                old = plain.setdefault(i, {}).get(layer)
                new = (roundtrip(k[a:e]), roundtrip(v[a:e]))
                kk, vv = plain[i][layer] = new if old is None else tuple(torch.cat(p) for p in zip(old, new))
                n = kk.shape[0]
                assert n == cache.length(i) and torch.equal(kd[b, :n], kk) and torch.equal(vd[b, :n], vv)
            want, _, bound = U.attention(q, cache, layer, table, lens.tolist(), starts)
            U.check(got, want, bound, dtype)

    a, b, e = (cache.new_sequence() for _ in range(3))
    step([a, b, e], [70, 33, 40])                                    # pages 0 - 2, 3 - 4 and 5 - 6
    step([a, b], [1, 1])
    c = cache.fork(a)
    plain[c] = {layer: rows for layer, rows in plain[a].items()}
    step([a, c, b], [1, 1, 1])                                       # a and c part: their last page is copied
    step([c], [5])                                                   # drafted
    cache.truncate(c, cache.length(c) - 4)
    plain[c] = {layer: tuple(x[:-4] for x in rows) for layer, rows in plain[c].items()}
    step([c, a], [1, 2])
    step([c, b], [60, 1])                                            # pages behind those of a and e
    for gone in (a, e):
        cache.free(gone)
        del plain[gone]
    assert cache.compact() > 0
    d = cache.new_sequence()
    step([b, d, c], [1, 150, 1])
    step([b, d, c], [1, 1, 1])
    assert cache.num_free_pages == cache.num_pages - len({p for i in (b, c, d) for p in cache.pages(i)})
    assert_device_ok()
