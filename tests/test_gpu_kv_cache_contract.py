"""The 4-bit key/value cache's operators on calls at the edge of what is documented, on the GPU: pages outside the cache that some rows see,
bounds that do not hold, and the sizes at which the kernels change their course."""
import ctypes as C
import math

import pytest
import torch

import mps_bitsandbytes_b200 as bnb
from gpu_util import assert_device_ok
from mps_bitsandbytes_b200 import _native as N

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _status():
    st = C.c_int(0)
    assert N.lib().mpsbnb_device_status(C.byref(st), 1) == 0
    return st.value


@pytest.mark.parametrize("head_dim,blocksize", [(128, 64), (64, 32), (256, 64)])
def test_a_page_outside_the_cache_is_no_matter_of_the_rows_that_do_not_see_it(head_dim, blocksize):
    """Drafts of five tokens with a window: the first two rows see the end of a page that is not there, the others do not.  What the
    kernel has in that page's place - the other heads' values, fetched before - must not show."""
    import kv_util as U
    from test_gpu_kv_cache_ranges import close, reference
    batch, kv_heads, new, length, window = 64, 8, 5, 258, 224        # rows see places from 30, 31, 32 ... on; 16 to 31 are outside
    width = -(-length // 16)
    cache = U.make_cache(batch * width, kv_heads, head_dim, 16, blocksize, "nf4", BF16, seed=1)
    table = U.random_table(batch, width, batch * width)
    q = torch.randn(batch, new, kv_heads, head_dim, device="cuda").to(BF16)
    bad = table.clone()
    bad[:, 1] = -1
    outs = []
    for size in (1.0, 1e30, math.inf):
        cache.v_absmax[0, :, 1::2] = size                            # the odd heads'
        outs.append(bnb.attention_4bit(q, cache, 0, bad, _i32([length] * batch), window=window)[:, :, ::2])
        assert _status() == 401
    assert all(torch.isnan(got[:, :2]).all() and torch.equal(got[:, 2:], outs[0][:, 2:]) for got in outs)
    cache.v_absmax[0, :, 1::2] = 1.0
    for b in range(0, batch, 9):
        want, limit = reference(q[b], cache, 0, table[b], length, window)
        close(outs[2][b, 2:], want[2:, ::2], limit[2:, ::2])


@pytest.mark.parametrize("head_dim,heads,kv_heads,new,lens", [
    (128, 8, 2, [3, 1, 9, 2], [40, 1, 77, 30]), (128, 32, 8, [300, 129, 1, 200], [400, 129, 30, 700]), (256, 16, 8, [257, 300], [500, 300]),
    (64, 64, 16, [100, 33, 256, 64, 1, 17, 130] * 3, [177, 33, 400, 64, 5, 99, 131] * 3)])
def test_max_seqlen_guides_the_choice_of_kernels_and_nothing_else(head_dim, heads, kv_heads, new, lens):
    import kv_util as U
    width = -(-max(lens) // 32)
    cache = U.make_cache(len(new) * width, kv_heads, head_dim, 32, seed=3)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    narrow = U.random_table(len(new), width, len(new) * width)
    q = torch.randn(starts[-1], heads, head_dim, device="cuda", dtype=F16)
    want, _, bound = U.attention(q, cache, 0, narrow, lens, starts)
    for table in (narrow, U.widen(narrow, 32)):
        for longest in (0, 1, max(new) // 2, max(new), starts[-1], None):
            U.check(bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), longest), want, bound, F16)
    assert_device_ok()


def test_append_stores_every_row_whatever_the_longest_is_said_to_be():
    cache, other = (bnb.KVCache4bit(1, 8, 2, 64, page_size=16) for _ in range(2))
    k, v = (torch.randn(20, 2, 64, device="cuda", dtype=F16) for _ in range(2))
    table, lens, starts = _i32([[0, 1], [2, 3]]), _i32([17, 20]), _i32([0, 7, 20])
    bnb.append_kv_4bit(other, 0, k, v, table, lens, starts)
    for longest in (0, 3, 13, 20):
        cache.data.zero_()
        sq = N.Kv4Seqs(table.data_ptr(), 2, lens.data_ptr(), starts.data_ptr(), 20, 2, 2, longest)
        assert N.lib().mpsbnb_kv4_append(cache._ref, 0, sq, k.data_ptr(), 128, 64, v.data_ptr(), 128, 64, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(cache.data, other.data) and cache.data.any()


def test_the_attention_tests_reach_all_kernels():
    """By the library's own choice, over the cases of the attention test (with the table's own width and widened)."""
    from test_gpu_kv_cache import CASES
    kinds = set()
    for head_dim, blocksize, page, _, dtype, heads, kv_heads, new, lens, _, window in CASES:
        cache = bnb.KVCache4bit(1, 1, kv_heads, head_dim, page, blocksize, dtype=dtype)
        for width in (max(-(-max(lens) // page), 1), (1 << 17) // page):
            sq = N.Kv4Seqs(1 << 21, width, 1 << 22, 1 << 23, sum(new), width, len(new), max(new))
            kinds.add((N.lib().mpsbnb_attention_4bit_kernels(cache._ref, sq, heads, window or 0), head_dim, blocksize))
    assert kinds >= {(k, d, b) for k in (1, 2, 6) for d in (64, 128, 256) for b in (32, 64)}
    assert {(3, d) for d in (64, 128)} <= {(k, d) for k, d, _ in kinds}   # single tokens and prompts in a call; the others below


@pytest.mark.parametrize("head_dim,blocksize,dtype,window,heads,kv_heads,kinds", [
    (64, 64, F16, None, 8, 2, 7), (128, 64, BF16, None, 8, 2, 7), (128, 32, F16, 150, 8, 2, 7), (256, 64, F16, None, 4, 1, 7), (256, 32, BF16, None, 32, 8, 3)])
def test_prompts_among_single_tokens(head_dim, blocksize, dtype, window, heads, kv_heads, kinds):
    import kv_util as U
    new, lens = [1, 2, 1, 400, 1, 1, 0, 5], [30, 500, 1, 555, 90, 257, 9, 5]
    cache = U.make_cache(8 * 18, kv_heads, head_dim, 32, blocksize, dtype=dtype, seed=5)
    table = U.widen(U.random_table(8, 18, 8 * 18), 32)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    sq = N.Kv4Seqs(1 << 21, table.shape[1], 1 << 22, 1 << 23, sum(new), table.shape[1], 8, 400)
    assert N.lib().mpsbnb_attention_4bit_kernels(cache._ref, sq, heads, 0) == kinds
    q = torch.randn(starts[-1], heads, head_dim, device="cuda").to(dtype)
    want, want_lse, bound = U.attention(q, cache, 0, table, lens, starts, window=window)
    got, lse = bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), 400, window=window, return_lse=True)
    U.check(got, want, bound, dtype)
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -11 * 16 + 2.0 ** -20 * want_lse.abs()).all()
    assert torch.equal(got, bnb.attention_4bit(q, cache, 0, table, _i32(lens), _i32(starts), 400, window=window))
    assert_device_ok()


@pytest.mark.parametrize("new,length", [(10, 40), (10, 2 ** 31 - 1), (3, 33), (32, 64), (40, 40)])
def test_append_leaves_the_tokens_alone_that_are_there_when_the_table_has_no_room(new, length):
    cache = bnb.KVCache4bit(1, 4, 2, 64, page_size=16)
    table = _i32([[3, 1], [0, 2]])
    old = torch.randn(2, 32, 2, 64, device="cuda", dtype=F16)
    bnb.append_kv_4bit(cache, 0, old, old * 2, table, _i32([32, 32]))
    kept = bnb.dequantize_kv_4bit(cache, 0, table, _i32([32, 32]))
    assert_device_ok()
    k = torch.randn(2, new, 2, 64, device="cuda", dtype=F16)
    bnb.append_kv_4bit(cache, 0, k, k * 3, table, _i32([length, 32]))
    assert _status() == 430
    got = bnb.dequantize_kv_4bit(cache, 0, table, _i32([32, 32]))
    first = length - new                                             # the first new token's place
    for x, was, now in zip((k, k * 3), kept, got):
        room = max(0, 32 - first)
        assert torch.equal(now[0, :min(first, 32)], was[0, :min(first, 32)])
        if room:
            want = bnb.dequantize_4bit(*bnb.quantize_4bit(x[0, :room].reshape(-1, 64))).view(room, 2, 64)
            assert torch.equal(now[0, first:], want)
    own = min(new, 32)
    want = bnb.dequantize_4bit(*bnb.quantize_4bit(k[1, new - own:].reshape(-1, 64))).view(own, 2, 64)
    assert torch.equal(got[0][1, 32 - own:], want)
    assert_device_ok()


@pytest.mark.parametrize("heads,kv_heads,new,length", [(8, 2, 10, 5), (32, 8, 300, 200), (32, 8, 300, 300)])
def test_the_largest_window_is_none(heads, kv_heads, new, length):
    """By the C entry point, for a sequence that is shorter than its new tokens too: places are negative there."""
    import kv_util as U
    cache = U.make_cache(10, kv_heads, 128, 32, seed=6)
    table = U.widen(U.random_table(1, 10, 10), 32)
    q = torch.randn(new, heads, 128, device="cuda", dtype=F16)
    lens = _i32([length])
    want = bnb.attention_4bit(q[None], cache, 0, table, lens)[0]
    sq = N.Kv4Seqs(table.data_ptr(), table.shape[1], lens.data_ptr(), None, new, table.shape[1], 1, new)
    nbytes = N.lib().mpsbnb_attention_4bit_workspace_bytes(cache._ref, sq, heads)
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    for window in (1 << 30, (1 << 31) - 1):
        got = torch.full_like(q, 7.0)
        assert N.lib().mpsbnb_attention_4bit(cache._ref, 0, sq, q.data_ptr(), heads * 128, 128, heads, 1, window, 128 ** -0.5, got.data_ptr(), None,
                                             ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(got, want) and want.any()


#  tokens of each sequence; what of them is new
LARGE = [([5200], [5200]), ([1700, 0, 900, 3001, 64, 1], [1700, 0, 333, 3001, 1, 1]), ([3, 1, 2], [3, 1, 1])]


@pytest.mark.parametrize("lens,new", LARGE, ids=["one of many tokens", "ragged", "few"])
@pytest.mark.parametrize("head_dim,blocksize,kv_heads,dtype,quant", [
    (256, 64, 8, BF16, "nf4"), (256, 32, 5, F16, "fp4"), (128, 64, 11, F16, "nf4"), (64, 32, 17, BF16, "fp4"), (128, 32, 1, BF16, "nf4"), (64, 64, 3, F16, "nf4")])
def test_append_and_read_back_of_many_tokens_and_many_heads(lens, new, head_dim, blocksize, kv_heads, dtype, quant):
    """More tokens than there are warps, so that each goes on from one to the next, and more heads than a warp takes at a time; few
    tokens, whose heads several warps share."""
    width = max(-(-max(lens) // 64), 1)
    cache = bnb.KVCache4bit(1, len(lens) * width, kv_heads, head_dim, 64, blocksize, quant, dtype)
    table = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(len(lens), width).cuda()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    k, v = (torch.randn(starts[-1], kv_heads, head_dim, device="cuda").to(dtype) for _ in range(2))
    cache.data.random_(0, 128)
    before = bnb.dequantize_kv_4bit(cache, 0, table, _i32(lens))
    bnb.append_kv_4bit(cache, 0, k, v, table, _i32(lens), _i32(starts))
    after = bnb.dequantize_kv_4bit(cache, 0, table, _i32(lens))
    for x, was, now in zip((k, v), before, after):
        want = bnb.dequantize_4bit(*bnb.quantize_4bit(x.reshape(-1, head_dim), blocksize=blocksize, quant_type=quant)).view(x.shape)
        for b, (n, length) in enumerate(zip(new, lens)):
            assert torch.equal(now[b, length - n:length], want[starts[b]:starts[b + 1]])
            same = now[b, :length - n].view(torch.int16) == was[b, :length - n].view(torch.int16)
            assert same.all() and (now[b, length:] == 0).all()
    assert_device_ok()


def test_read_back_of_more_places_than_there_are_warps():
    import kv_util as U
    lens = [9000, 0, 12345, 700]
    cache = U.make_cache(4 * 200, 5, 256, 64, 64, "nf4", BF16, seed=8)
    table = U.random_table(4, 200, 800)
    k, v = bnb.dequantize_kv_4bit(cache, 0, table, _i32(lens), 12400)
    for x, name in ((k, "k"), (v, "v")):
        for b, length in enumerate(lens):
            for a in range(0, length, 4000):
                e = min(length, a + 4000)
                assert torch.equal(x[b, a:e], U.rows_of(cache, 0, table[b], a, e, name).float().to(BF16))
            assert (x[b, length:] == 0).all()


@pytest.mark.parametrize("head_dim,kv_heads", [(128, 3), (64, 2), (256, 2)])
def test_append_takes_rows_on_uneven_addresses_from_the_c_entry_point(head_dim, kv_heads):
    """Python copies such rows first; the kernel takes them as they are: odd addresses, odd strides, heads between which others lie."""
    tokens, token, head = 37, (kv_heads + 1) * (head_dim + 3) + 5, head_dim + 3
    cache, other = (bnb.KVCache4bit(1, 3, kv_heads, head_dim, page_size=16) for _ in range(2))
    flat = torch.randn(2 * tokens * token + 9, device="cuda", dtype=F16)
    rows = [flat[at:].as_strided((tokens, kv_heads, head_dim), (token, head, 1)) for at in (1, 7 + tokens * token)]
    table, lens = _i32([[2, 0, 1]]), _i32([40])
    bnb.append_kv_4bit(other, 0, *(x.contiguous() for x in rows), table, lens)
    sq = N.Kv4Seqs(table.data_ptr(), 3, lens.data_ptr(), None, tokens, 3, 1, tokens)
    assert N.lib().mpsbnb_kv4_append(cache._ref, 0, sq, rows[0].data_ptr(), token, head, rows[1].data_ptr(), token, head, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(cache.data, other.data) and cache.data.any()
    assert_device_ok()


def test_an_output_that_is_not_contiguous_is_refused():
    cache = bnb.KVCache4bit(1, 4, 2, 128)
    q = torch.zeros(2, 3, 8, 128, device="cuda", dtype=F16)
    for out in (torch.zeros(2, 8, 3, 128, device="cuda", dtype=F16).transpose(1, 2), torch.zeros(2, 3, 8, 136, device="cuda", dtype=F16)[..., :128],
                torch.zeros(2 * 3 * 8 * 128 + 1, device="cuda", dtype=F16)[1:].view(q.shape)):
        with pytest.raises(ValueError, match="out must be"):
            bnb.attention_4bit(q, cache, 0, _i32([[0, 1], [2, 3]]), _i32([3, 4]), out=out)


def test_calls_without_tokens_or_sequences():
    cache = bnb.KVCache4bit(1, 4, 2, 64)
    before = cache.data.clone()
    table, lens = _i32([[0, 1], [2, 3]]), _i32([5, 0])
    for q, args in ((torch.zeros(0, 8, 64, device="cuda", dtype=F16), (table, lens, _i32([0, 0, 0]))), (torch.zeros(2, 0, 8, 64, device="cuda", dtype=F16), (table, lens)),
                    (torch.zeros(0, 8, 64, device="cuda", dtype=F16), (table[:0], lens[:0], _i32([0]))), (torch.zeros(0, 1, 8, 64, device="cuda", dtype=F16), (table[:0], lens[:0]))):
        out, lse = bnb.attention_4bit(q, cache, 0, *args, return_lse=True)
        assert out.shape == q.shape and lse.shape == q.shape[:-1]
        bnb.append_kv_4bit(cache, 0, q[..., :2, :], q[..., :2, :], *args)
    # rows that belong to no sequence, for the kernels of either kind
    for rows in (5, 3000):
        q = torch.randn(rows, 8, 64, device="cuda", dtype=F16)
        out, lse = bnb.attention_4bit(q, cache, 0, table, lens, _i32([0, 0, 0]), return_lse=True)
        assert (out == 0).all() and torch.isinf(lse).all()
        bnb.append_kv_4bit(cache, 0, q[:, :2], q[:, :2], table, lens, _i32([0, 0, 0]))
    assert torch.equal(cache.data, before)
    assert_device_ok()


def test_prompts_done_again_on_two_streams_at_once():
    """Each call has its own list of what is to be done again."""
    import kv_util as U
    cache = U.make_cache(40, 8, 128, 64, dtype=BF16, seed=9)
    plain, wide = U.widen(_i32([list(range(20))]), 64), U.widen(_i32([list(range(20, 40))]), 64)
    cache.v_absmax[0, 25, :, 1, 3] = 1e14
    qs = [torch.randn(1, 1100, 32, 128, device="cuda").to(BF16) for _ in range(2)]
    lens = _i32([1200])
    want = [bnb.attention_4bit(q, cache, 0, t, lens) for q, t in zip(qs, (plain, wide))]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for i, t in enumerate((plain, wide)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(bnb.attention_4bit(qs[i], cache, 0, t, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])
    assert_device_ok()
