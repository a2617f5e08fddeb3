"""The 4-bit key/value cache without a GPU: the book of pages against a plain model of sequences, the refusals of the
C entry points (which check before they touch a device) and of the Python surface."""
import ctypes as C
import os
import random
import re

import numpy as np
import pytest
import torch

import mps_bitsandbytes_b200 as bnb
from mps_bitsandbytes_b200 import _native as N
from mps_bitsandbytes_b200.kv_cache import _PageBook
from oracle import oracle_np as O


class Book(_PageBook):
    """Pages as Python lists, so that a lost or shared write shows."""

    def __init__(self, num_pages, page_size):
        super().__init__(num_pages, page_size)
        self.store = [[None] * page_size for _ in range(num_pages)]

    def _copy_pages(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in zip(src, dst):
            self.store[b] = list(self.store[a])

    def write(self, seq_id, tokens):
        first = self.length(seq_id) - len(tokens)
        for i, t in enumerate(tokens):
            page = self.pages(seq_id)[(first + i) // self.page_size]
            assert self._users[page] == 1, "a shared page is written"
            self.store[page][(first + i) % self.page_size] = t

    def read(self, seq_id):
        return [self.store[self.pages(seq_id)[i // self.page_size]][i % self.page_size] for i in range(self.length(seq_id))]


@pytest.mark.parametrize("seed,page_size", [(0, 16), (1, 16), (2, 32), (3, 64)])
def test_book_against_plain_sequences(seed, page_size):
    rng = random.Random(seed)
    book, plain, token = Book(40, page_size), {}, 0
    for _ in range(600):
        what = rng.choice(["new", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if what == "new" or not plain:
            plain[book.new_sequence()] = []
        elif what == "extend":
            ids = rng.sample(sorted(plain), rng.randint(1, len(plain)))
            counts = [rng.choice([0, 1, 1, 3, page_size, 2 * page_size + 1]) for _ in ids]
            before = (book.num_free_pages, {i: (book.pages(i), book.length(i)) for i in plain})
            try:
                book.extend(ids, counts)
            except RuntimeError as err:
                assert "out of pages" in str(err)
                assert before == (book.num_free_pages, {i: (book.pages(i), book.length(i)) for i in plain})
                gone = rng.choice(sorted(plain))
                book.free(gone)
                del plain[gone]
                continue
            for i, n in zip(ids, counts):
                new = list(range(token, token + n))
                token += n
                book.write(i, new)
                plain[i] += new
        elif what == "fork":
            i = rng.choice(sorted(plain))
            plain[book.fork(i)] = list(plain[i])
        elif what == "truncate":
            i = rng.choice(sorted(plain))
            n = rng.randint(0, len(plain[i]))
            book.truncate(i, n)
            del plain[i][n:]
        elif what == "free" and len(plain) > 3:
            i = rng.choice(sorted(plain))
            book.free(i)
            del plain[i]
        elif what == "compact":
            book.compact()
            live = {p for i in plain for p in book.pages(i)}
            assert live == set(range(len(live)))
        for i, tokens in plain.items():
            assert book.read(i) == tokens
        live = {p for i in plain for p in book.pages(i)}
        assert book.num_free_pages == book.num_pages - len(live)
        assert sorted(book._free) == sorted(set(range(book.num_pages)) - live)


def test_book_refusals():
    book = Book(4, 16)
    a, b = book.new_sequence(), book.new_sequence()
    with pytest.raises(KeyError, match="no sequence 7"):
        book.extend([7], 1)
    with pytest.raises(ValueError, match="named twice"):
        book.extend([a, a], 1)
    with pytest.raises(ValueError, match="2 sequences but 1 counts"):
        book.extend([a, b], [1])
    with pytest.raises(ValueError, match="negative"):
        book.extend([a], -1)
    with pytest.raises(RuntimeError, match="out of pages: 5 needed, 4 free"):
        book.extend([a, b], [48, 17])
    assert book.num_free_pages == 4 and book.length(a) == 0
    with pytest.raises(ValueError, match="between 0 and 0"):
        book.truncate(a, 1)
    book.free(a)
    with pytest.raises(KeyError):
        book.free(a)


def test_a_fork_of_a_full_page_copies_nothing_and_a_shared_tail_is_copied_once_less_than_it_is_shared():
    book = Book(8, 16)
    a = book.new_sequence()
    book.extend([a], 16)
    book.write(a, list(range(16)))
    b = book.fork(a)
    book.extend([a, b], 1)
    assert book.pages(a)[0] == book.pages(b)[0] and book.pages(a)[1] != book.pages(b)[1]
    c = book.fork(b)
    d = book.fork(b)
    used = book.num_pages - book.num_free_pages
    book.extend([b, c, d], 1)                       # three on one tail: two copies
    assert book.num_pages - book.num_free_pages == used + 2
    assert len({book.pages(i)[1] for i in (b, c, d)}) == 3


def test_the_scaled_codebook_rounds_better_than_nf4_itself():
    """Rounding errors of the fp16 table over the codes of normal data, of which the kernel's comment speaks."""
    src = open(os.path.join(os.path.dirname(N.LIB_PATH), "..", "csrc", "attn4.cuh")).read()
    scale = float.fromhex(re.search(r"#define ATTN4_NF4_SCALE (\S+)f\b", src).group(1))
    x = np.random.default_rng(0).standard_normal((20000, 64))
    code = O.NF4_CODE.astype(np.float64)
    idx = np.searchsorted((code[1:] + code[:-1]) / 2, x / np.abs(x).max(1, keepdims=True))
    share = np.bincount(idx.ravel(), minlength=16) / idx.size

    def errors(c):
        table = (code.astype(np.float32) * np.float32(c)).astype(np.float16).astype(np.float64)
        d = table / c - code
        return np.sqrt((share * d * d).sum()), abs((share * d).sum())
    plain, scaled = errors(1.0), errors(scale)
    assert scaled[0] < 0.5 * plain[0] and scaled[1] < 0.25 * plain[1]
    assert plain[0] == pytest.approx(7.3e-5, rel=0.02) and scaled[0] == pytest.approx(3.4e-5, rel=0.03)
    assert np.array_equal(O.FP4_CODE.astype(np.float16).astype(np.float32), O.FP4_CODE)


# ---------------------------------------------------------------------- C entry points
def _cache(**kw):
    base = dict(data=1 << 20, num_pages=8, num_layers=2, kv_heads=2, head_dim=128, page_size=64, blocksize=64, quant_type=0, dtype=0)
    base.update(kw)
    return N.Kv4Cache(*[base[n] for n, _ in N.Kv4Cache._fields_])


def _seqs(**kw):
    base = dict(page_table=1 << 21, table_ld=4, seq_lens=1 << 22, cu_seqlens=None, tokens=3, table_width=4, batch=3, new_tokens=1)
    base.update(kw)
    return N.Kv4Seqs(*[base[n] for n, _ in N.Kv4Seqs._fields_])


P = 1 << 24                                         # an address that nothing reads: every call below is refused
INVALID, UNSUPPORTED, WORKSPACE, TOO_LARGE = -1, -2, -4, -5


def _attention(cache, seqs, layer=0, q=P, ts=1024, hs=128, heads=8, causal=1, window=0, out=P, ws=P, nbytes=1 << 40):
    return N.lib().mpsbnb_attention_4bit(C.byref(cache), layer, C.byref(seqs), q, ts, hs, heads, causal, window, 1.0, out, None, ws, nbytes, None)


def test_sizes():
    lib = N.lib()
    assert lib.mpsbnb_kv4_group_bytes(128, 64) == 16 * 2 * (64 + 4)
    assert lib.mpsbnb_kv4_group_bytes(64, 32) == 16 * 2 * (32 + 4)
    assert lib.mpsbnb_kv4_cache_bytes(C.byref(_cache())) == 2 * 8 * 2 * 4 * 2176
    assert lib.mpsbnb_attention_4bit_workspace_bytes(C.byref(_cache()), C.byref(_seqs()), 8) > 0
    assert lib.mpsbnb_attention_4bit_workspace_bytes(C.byref(_cache()), C.byref(_seqs()), 7) == 0
    assert lib.mpsbnb_attention_4bit_workspace_bytes(C.byref(_cache()), C.byref(_seqs(batch=0, tokens=0)), 8) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(data=None), INVALID), (dict(data=8), INVALID), (dict(num_pages=0), INVALID), (dict(kv_heads=0), INVALID),
    (dict(dtype=2), INVALID), (dict(quant_type=2), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
    (dict(blocksize=128), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
    (dict(page_size=2048), UNSUPPORTED), (dict(num_pages=1 << 31), TOO_LARGE)])
def test_caches_that_are_refused(kw, code):
    lib, bad, sq = N.lib(), _cache(**kw), _seqs()
    one = (C.c_int32 * 1)(0)
    assert _attention(bad, sq) == code
    assert lib.mpsbnb_kv4_append(C.byref(bad), 0, C.byref(sq), P, 256, 128, P, 256, 128, None) == code
    assert lib.mpsbnb_kv4_dequantize(C.byref(bad), 0, C.byref(sq), 4, P, P, None) == code
    assert lib.mpsbnb_kv4_copy_pages(C.byref(bad), one, one, 1, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(batch=-1), INVALID), (dict(tokens=-3), INVALID), (dict(new_tokens=-1), INVALID), (dict(table_width=-1), INVALID),
    (dict(seq_lens=None), INVALID), (dict(page_table=None), INVALID), (dict(table_ld=3), INVALID), (dict(tokens=4), INVALID),
    (dict(table_width=1 << 25, table_ld=1 << 25), TOO_LARGE), (dict(tokens=1 << 31, cu_seqlens=P), TOO_LARGE)])
def test_sequences_that_are_refused(kw, code):
    lib, cache, bad = N.lib(), _cache(), _seqs(**kw)
    assert _attention(cache, bad) == code
    assert lib.mpsbnb_kv4_append(C.byref(cache), 0, C.byref(bad), P, 256, 128, P, 256, 128, None) == code


def test_other_arguments_that_are_refused():
    lib, cache, sq = N.lib(), _cache(), _seqs()
    assert _attention(cache, sq, layer=2) == INVALID and _attention(cache, sq, layer=-1) == INVALID
    assert _attention(cache, sq, heads=7) == INVALID and _attention(cache, sq, heads=0) == INVALID
    assert _attention(cache, sq, window=-1) == INVALID and _attention(cache, sq, causal=0, window=5) == INVALID
    assert _attention(cache, sq, q=None) == INVALID and _attention(cache, sq, out=None) == INVALID
    assert _attention(cache, sq, ts=-8) == INVALID
    assert _attention(cache, sq, ws=None) == WORKSPACE and _attention(cache, sq, ws=P + 8) == WORKSPACE and _attention(cache, sq, nbytes=64) == WORKSPACE
    assert _attention(cache, sq, q=P + 8) == UNSUPPORTED and _attention(cache, sq, ts=1025) == UNSUPPORTED and _attention(cache, sq, out=P + 2) == UNSUPPORTED
    assert _attention(cache, _seqs(batch=0, tokens=0)) == 0 and _attention(cache, _seqs(new_tokens=0, tokens=0)) == 0   # nothing to do
    append = lambda k=P, v=P, ks=256: lib.mpsbnb_kv4_append(C.byref(cache), 0, C.byref(sq), k, ks, 128, v, 256, 128, None)
    assert append(k=None) == INVALID and append(v=None) == INVALID and append(ks=-1) == INVALID
    deq = lambda n=4, k=P, v=P: lib.mpsbnb_kv4_dequantize(C.byref(cache), 0, C.byref(sq), n, k, v, None)
    assert deq(n=-1) == INVALID and deq(k=None) == INVALID and deq(v=P + 8) == INVALID and deq(n=1 << 31) == TOO_LARGE and deq(n=0) == 0

    def copy(src, dst, n=None):
        n = len(src) if n is None else n
        return lib.mpsbnb_kv4_copy_pages(C.byref(cache), (C.c_int32 * len(src))(*src), (C.c_int32 * len(dst))(*dst), n, None)
    assert copy([0], [8]) == INVALID and copy([-1], [1]) == INVALID and copy([0, 1], [2, 2]) == INVALID
    assert copy([0, 1], [1, 2]) == INVALID and copy([3], [3]) == INVALID and copy([0], [1], -1) == INVALID
    assert copy([0] * 9, list(range(9)), 9) == INVALID and copy([0], [1], 0) == 0


# ---------------------------------------------------------------------- Python surface
@pytest.mark.parametrize("kw,match", [
    (dict(quant_type="int4"), "quant_type must be"), (dict(dtype=torch.float32), "dtype must be"), (dict(head_dim=80), "head_dim must be"),
    (dict(blocksize=16), "blocksize must be"), (dict(page_size=100), "page_size must be"), (dict(num_pages=0), "num_pages must be"),
    (dict(num_layers=-1), "num_layers must be"), (dict(device="cpu"), "'cuda' device")])
def test_caches_that_python_refuses(kw, match):
    args = dict(num_layers=1, num_pages=4, num_kv_heads=2, head_dim=128)
    args.update(kw)
    with pytest.raises(ValueError, match=match):
        bnb.KVCache4bit(**args)


def test_operators_want_a_cache():
    x = torch.zeros(1, 2, 128)
    with pytest.raises(TypeError, match="takes a KVCache4bit"):
        bnb.append_kv_4bit(x, 0, x, x, None, None)
    with pytest.raises(TypeError, match="takes a KVCache4bit"):
        bnb.attention_4bit(x, x, 0, None, None)
    with pytest.raises(TypeError, match="takes a KVCache4bit"):
        bnb.dequantize_kv_4bit(x, 0, None, None)
    with pytest.raises(TypeError, match="takes a KVCache4bit"):
        bnb.copy_kv_pages_4bit(x, [0], [1])


@pytest.mark.parametrize("qt,bf16", [(0, 0), (1, 0), (0, 1), (1, 1)])
def test_codes_by_the_reciprocal_are_those_of_the_division(qt, bf16):
    """Every third absmax of the 16-bit types in the range where the cache's quantiser multiplies by 1 / absmax, with every x up
    to it (a stride of 1 also returns 0)."""
    from oracle import oracle_c
    fn = oracle_c.lib().o_prove_kv4_thresholds
    fn.restype, fn.argtypes = C.c_int64, [C.c_int, C.c_int, C.c_int64, C.c_float, C.c_float]
    assert fn(qt, bf16, 3, 1.0001e-8, 1e30) == 0
