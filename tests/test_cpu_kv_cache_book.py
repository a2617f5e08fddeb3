"""The 4-bit key/value cache's storage and book of pages where a step fails, without a GPU."""
import pytest
import torch

import mps_bitsandbytes_b200 as bnb
from mps_bitsandbytes_b200.kv_cache import _PageBook


class FailingBook(_PageBook):
    fail = False

    def _copy_pages(self, src, dst):
        if self.fail:
            raise RuntimeError("copy_kv_pages_4bit failed")


def _all(book):
    return sorted(book._free), list(book._users), {i: (list(s[0]), s[1]) for i, s in book._seqs.items()}


def test_a_copy_that_fails_leaves_the_book_as_it_was():
    book = FailingBook(12, 16)
    a = book.new_sequence()
    book.extend([a], 20)
    b = book.fork(a)
    c = book.new_sequence()
    before = _all(book)
    book.fail = True
    with pytest.raises(RuntimeError, match="copy_kv_pages_4bit failed"):
        book.extend([c, a, b], [5, 30, 1])                           # a's last page would be copied
    assert _all(book) == before
    book.fail = False
    book.extend([c, a, b], [5, 30, 1])
    assert (book.length(a), book.length(b), book.length(c)) == (50, 21, 5)
    assert book.pages(a)[0] == book.pages(b)[0] and book.pages(a)[1] != book.pages(b)[1]
    assert sorted(book._free) == [p for p in range(12) if book._users[p] == 0]


def _cpu_cache(pages=3):
    """A cache's storage without its device."""
    cache = object.__new__(bnb.KVCache4bit)
    cache.head_dim, cache.blocksize, cache.dtype = 128, 64, torch.float16
    from mps_bitsandbytes_b200 import _native as N
    cache._desc = N.Kv4Cache(None, pages, 1, 2, 128, 16, 64, 0, 0)
    cache._bind(torch.zeros(1, pages, 2, 1, 2176, dtype=torch.uint8))
    return cache


def test_the_kernels_get_the_storage_that_has_been_assigned():
    cache = _cpu_cache()
    assert cache._desc.data == cache.data.data_ptr()
    other = torch.randint(0, 256, cache.data.shape, dtype=torch.uint8)
    cache.data = other
    assert cache._desc.data == other.data_ptr() and cache.data is other
    assert cache.v_codes.shape == (1, 3, 2, 1, 16, 64) and cache.v_codes.data_ptr() == other.data_ptr() + 1088
    assert torch.equal(cache.k_absmax.view(torch.uint8).flatten(-2), other[..., 1024:1088])
    for bad in (other[:, :2], other.short(), other.to("meta"), other.transpose(1, 2).contiguous().transpose(1, 2), None,
                torch.empty(other.numel() + 1, dtype=torch.uint8)[1:].view(other.shape)):
        with pytest.raises(ValueError, match="data must be"):
            cache.data = bad
    assert cache.data is other and cache._desc.data == other.data_ptr()
