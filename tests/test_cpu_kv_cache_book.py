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
