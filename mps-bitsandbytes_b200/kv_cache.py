"""Paged key/value cache held in 4 bits, and the attention that reads it.

The rows of keys and values are quantised as ``quantize_4bit`` quantises the rows of a weight (same codebooks, blocks
inside a row, one absmax per block); the absmax is kept in the cache's 16-bit type, in which a 16-bit row's absmax is
exact.  4.25 bits per element with 64-element blocks instead of 16.

    cache = KVCache4bit(num_layers=32, num_pages=4096, num_kv_heads=8, head_dim=128)
    ids = [cache.new_sequence() for _ in prompts]
    cache.extend(ids, [len(p) for p in prompts])                       # reserves pages
    table, lens = cache.batch(ids)
    for layer in ...:
        append_kv_4bit(cache, layer, k, v, table, lens, cu_seqlens)    # quantises the new rows into their pages
        o = attention_4bit(q, cache, layer, table, lens, cu_seqlens=cu_seqlens, max_seqlen=longest)

Decoding goes on with ``cache.extend(ids, 1)`` and one row per sequence.  Tensors must live on ``cuda``; nothing here
has a backward pass.
"""
from __future__ import annotations

import ctypes as C
import heapq
from typing import List, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor

from . import _native as N

_GROUP = 16                                         # tokens per group of the layout (include/mpsbnb_b200.h)


class _PageBook:
    """Which sequence holds which pages: host numbers only; ``_copy_pages`` moves the contents."""

    def __init__(self, num_pages: int, page_size: int):
        self.num_pages, self.page_size = num_pages, page_size
        self._free = list(range(num_pages))             # a heap
        self._users = [0] * num_pages
        self._seqs: dict = {}
        self._next_id = 0

    def _copy_pages(self, src: List[int], dst: List[int]) -> None:
        raise NotImplementedError

    @property
    def num_free_pages(self) -> int:
        return len(self._free)

    def _seq(self, seq_id: int):
        try:
            return self._seqs[seq_id]
        except KeyError:
            raise KeyError(f"no sequence {seq_id} in this cache") from None

    def length(self, seq_id: int) -> int:
        return self._seq(seq_id)[1]

    def pages(self, seq_id: int) -> List[int]:
        """Page numbers of the sequence, in order."""
        return list(self._seq(seq_id)[0])

    def new_sequence(self) -> int:
        """An empty sequence; returns its number."""
        seq_id = self._next_id
        self._next_id += 1
        self._seqs[seq_id] = [[], 0]
        return seq_id

    def extend(self, ids: Sequence[int], counts: Union[int, Sequence[int]]) -> None:
        """Makes room for ``counts`` more tokens in each sequence and raises its length.  A page that the new tokens
        share with another sequence is copied first (one launch for all sequences and layers, on the current stream).
        Raises RuntimeError if the pages do not suffice; nothing has changed after an error, that of a copy included."""
        ids = list(ids)
        counts = [counts] * len(ids) if isinstance(counts, int) else list(counts)
        if len(counts) != len(ids):
            raise ValueError(f"{len(ids)} sequences but {len(counts)} counts")
        if len(set(ids)) != len(ids):
            raise ValueError("a sequence is named twice")
        size = self.page_size
        need, shared, plan = 0, {}, []
        for seq_id, count in zip(ids, counts):
            pages, length = self._seq(seq_id)
            if count < 0:
                raise ValueError(f"counts must not be negative, got {count}")
            fresh = -(-(length + count) // size) - len(pages)
            copy = False
            if count > 0 and length % size:
                last = pages[-1]
                users = shared.get(last, self._users[last])
                copy = users > 1
                shared[last] = users - 1 if copy else users
            need += fresh + copy
            plan.append((pages, fresh, copy))
        if need > len(self._free):
            raise RuntimeError(f"the cache is out of pages: {need} needed, {len(self._free)} free")
        taken = [heapq.heappop(self._free) for _ in range(need)]
        src, dst, at = [], [], 0
        for pages, fresh, copy in plan:
            if copy:
                src.append(pages[-1])
                dst.append(taken[at])
            at += fresh + copy
        if src:
            try:
                self._copy_pages(src, dst)
            except BaseException:
                for page in taken:
                    heapq.heappush(self._free, page)
                raise
        at = 0
        for (pages, fresh, copy), seq_id, count in zip(plan, ids, counts):
            if copy:
                self._users[pages.pop()] -= 1
            pages += taken[at:at + fresh + copy]
            at += fresh + copy
            self._seqs[seq_id][1] += count
        for page in taken:
            self._users[page] = 1

    def fork(self, seq_id: int) -> int:
        """A sequence with the same tokens, sharing all pages; returns its number."""
        pages, length = self._seq(seq_id)
        new = self.new_sequence()
        self._seqs[new] = [list(pages), length]
        for page in pages:
            self._users[page] += 1
        return new

    def _release(self, pages: Sequence[int]) -> None:
        for page in pages:
            self._users[page] -= 1
            if self._users[page] == 0:
                heapq.heappush(self._free, page)

    def truncate(self, seq_id: int, length: int) -> None:
        """Drops the tokens from place ``length`` on (drafted tokens that were not accepted)."""
        seq = self._seq(seq_id)
        if not 0 <= length <= seq[1]:
            raise ValueError(f"length must be between 0 and {seq[1]}, got {length}")
        keep = -(-length // self.page_size)
        self._release(seq[0][keep:])
        del seq[0][keep:]
        seq[1] = length

    def free(self, seq_id: int) -> None:
        """Forgets the sequence; pages that no other sequence shares are free again."""
        self._release(self._seq(seq_id)[0])
        del self._seqs[seq_id]

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers (on the current stream); returns how many were moved.  Page
        tables made before are out of date afterwards."""
        live = self.num_pages - len(self._free)
        holes = [p for p in range(live) if self._users[p] == 0]
        high = [p for p in range(live, self.num_pages) if self._users[p] > 0]
        move = dict(zip(high, holes))
        if not move:
            return 0
        self._copy_pages(list(move), list(move.values()))
        for src, dst in move.items():
            self._users[dst], self._users[src] = self._users[src], 0
        for seq in self._seqs.values():
            seq[0][:] = [move.get(p, p) for p in seq[0]]
        self._free = list(range(live, self.num_pages))
        return len(move)


class KVCache4bit(_PageBook):
    """Storage for ``num_pages`` pages of ``page_size`` tokens in each of ``num_layers`` layers, and the host's book of
    which sequence holds which pages (one book for all layers).

    ``data`` is uint8 [layers, pages, kv heads, page_size / 16, group bytes]; ``k_codes`` / ``v_codes`` (uint8 [..., 16,
    head_dim / 2], low nibble = even element) and ``k_absmax`` / ``v_absmax`` (``dtype`` [..., 16, head_dim /
    blocksize]) are views of it.  Another tensor of its shape may be assigned to it.

    The book: ``new_sequence``, ``extend``, ``fork``, ``truncate``, ``free``, ``compact`` and ``batch``.  Forked
    sequences share their pages; a shared page is copied when one of them is about to write to it.  Pages are handed out
    lowest number first.  Whoever keeps page tables of their own can leave the book unused.  The book is not locked:
    calls from several threads have to be ordered by the caller.
    """

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 blocksize: int = 64, quant_type: str = "nf4", dtype: torch.dtype = torch.float16, device="cuda"):
        if quant_type not in ("nf4", "fp4"):
            raise ValueError(f"quant_type must be 'nf4' or 'fp4', got {quant_type}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if blocksize not in (32, 64):
            raise ValueError(f"blocksize must be 32 or 64, got {blocksize}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        for name, value in (("num_layers", num_layers), ("num_pages", num_pages), ("num_kv_heads", num_kv_heads)):
            if value <= 0:
                raise ValueError(f"{name} must be positive, got {value}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"mps-bitsandbytes_b200 KVCache4bit requires a 'cuda' device, got '{device.type}'")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        super().__init__(num_pages, page_size)
        self.num_layers, self.num_kv_heads, self.head_dim = num_layers, num_kv_heads, head_dim
        self.blocksize, self.quant_type, self.dtype, self.device = blocksize, quant_type, dtype, device
        self._desc = N.Kv4Cache(None, num_pages, num_layers, num_kv_heads, head_dim, page_size, blocksize, N.qt(quant_type), N.dt(dtype))
        self._ref, self._index = C.byref(self._desc), device.index
        half = _GROUP * (head_dim // 2 + 2 * (head_dim // blocksize))
        self._bind(torch.zeros(num_layers, num_pages, num_kv_heads, page_size // _GROUP, 2 * half, dtype=torch.uint8, device=device))

    def _bind(self, data: Tensor) -> None:
        """The storage, its views and the address that the kernels get."""
        nb = self.head_dim // self.blocksize
        codes, half = _GROUP * self.head_dim // 2, data.shape[-1] // 2
        self._data = data
        self.k_codes = data[..., :codes].unflatten(-1, (_GROUP, self.head_dim // 2))
        self.k_absmax = data[..., codes:half].view(self.dtype).unflatten(-1, (_GROUP, nb))
        self.v_codes = data[..., half:half + codes].unflatten(-1, (_GROUP, self.head_dim // 2))
        self.v_absmax = data[..., half + codes:].view(self.dtype).unflatten(-1, (_GROUP, nb))
        self._desc.data = data.data_ptr()

    @property
    def data(self) -> Tensor:
        return self._data

    @data.setter
    def data(self, value: Tensor) -> None:
        old = self._data
        if (not isinstance(value, Tensor) or value.shape != old.shape or value.dtype != old.dtype or value.device != old.device
                or not value.is_contiguous() or value.data_ptr() & 15):
            raise ValueError(f"data must be a contiguous uint8 tensor of shape {tuple(old.shape)} on {old.device}, 16-byte aligned")
        self._bind(value)

    def _copy_pages(self, src: List[int], dst: List[int]) -> None:
        copy_kv_pages_4bit(self, src, dst)

    def batch(self, ids: Sequence[int]) -> Tuple[Tensor, Tensor]:
        """(page table int32 [len(ids), most pages], lengths int32 [len(ids)]) on the cache's device."""
        seqs = [self._seq(i) for i in ids]
        width = max([len(s[0]) for s in seqs], default=0)
        host = torch.tensor([s[0] + [0] * (width - len(s[0])) + [s[1]] for s in seqs], dtype=torch.int32).view(len(seqs), width + 1)
        dev = host.to(self.device)
        return dev[:, :width], dev[:, width].contiguous()

    def extra_repr(self) -> str:
        return (f"num_layers={self.num_layers}, num_pages={self.num_pages}, num_kv_heads={self.num_kv_heads}, "
                f"head_dim={self.head_dim}, page_size={self.page_size}, blocksize={self.blocksize}, "
                f"quant_type={self.quant_type}, dtype={self.dtype}")

    def __repr__(self) -> str:
        return f"KVCache4bit({self.extra_repr()})"


# ---------------------------------------------------------------------- arguments
def _check_cache(cache: KVCache4bit, layer: int, what: str):
    if not isinstance(cache, KVCache4bit):
        raise TypeError(f"{what} takes a KVCache4bit, got {type(cache).__name__}")
    if not 0 <= layer < cache.num_layers:
        raise IndexError(f"layer {layer} is out of range for a cache of {cache.num_layers} layers")


def _check_index(name: str, t: Tensor, dim: int, cache: KVCache4bit):
    if t.dtype is not torch.int32 or t.dim() != dim or t.get_device() != cache._index:
        raise ValueError(f"{name} must be int32 with {dim} dimension{'s' if dim > 1 else ''} on {cache.device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    if not t.is_contiguous() and ((t.stride(-1) != 1 and t.shape[-1] > 1) or (dim == 2 and t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        raise ValueError(f"{name} must have distinct rows, contiguous along the last dimension")


def _seqs(cache: KVCache4bit, page_table: Tensor, seq_lens: Tensor, cu_seqlens: Optional[Tensor], tokens: int,
          max_seqlen: Optional[int]) -> "N.Kv4Seqs":
    _check_index("page_table", page_table, 2, cache)
    _check_index("seq_lens", seq_lens, 1, cache)
    batch, width = page_table.shape
    if seq_lens.shape[0] != batch:
        raise ValueError(f"page_table has {batch} rows, seq_lens {seq_lens.shape[0]}")
    if cu_seqlens is None:
        new = tokens // batch if batch else 0
        if new * batch != tokens:
            raise ValueError(f"{tokens} tokens cannot be shared evenly by {batch} sequences: cu_seqlens is needed")
        if max_seqlen is not None and max_seqlen != new:
            raise ValueError(f"max_seqlen is {max_seqlen}, but every sequence has {new} new tokens")
    else:
        _check_index("cu_seqlens", cu_seqlens, 1, cache)
        if cu_seqlens.shape[0] != batch + 1:
            raise ValueError(f"cu_seqlens has {cu_seqlens.shape[0]} entries, {batch} sequences need {batch + 1}")
        new = tokens if max_seqlen is None else int(max_seqlen)
        if not 0 <= new:
            raise ValueError(f"max_seqlen must not be negative, got {max_seqlen}")
        new = min(new, tokens)
    return N.Kv4Seqs(page_table.data_ptr(), page_table.stride(0) if batch > 1 else width, seq_lens.data_ptr(),
                     None if cu_seqlens is None else cu_seqlens.data_ptr(), tokens, width, batch, new)


def _rows(name: str, t: Tensor, heads: Optional[int], cache: KVCache4bit):
    """[..., heads, head_dim] as rows that can be fetched in 16-byte pieces: (the tensor, or a copy of it, that holds them,
    tokens, heads, strides of a token and of a head)."""
    if t.get_device() != cache._index:
        raise ValueError(f"{name} must be on {cache.device}, got {t.device}")
    if t.dtype is not cache.dtype:
        raise ValueError(f"{name} must have the cache's dtype {cache.dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) not in (3, 4) or shape[-1] != cache.head_dim or (heads is not None and shape[-2] != heads):
        raise ValueError(f"{name} must be [tokens, heads, {cache.head_dim}] or [batch, tokens, heads, {cache.head_dim}]"
                         f"{f' with {heads} heads' if heads is not None else ''}, got {tuple(shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires a gradient, but the 4-bit cache has no backward pass")
    stride = t.stride()
    if len(shape) == 4:
        tokens = shape[0] * shape[1]
        # the tokens of all sequences at one distance (else a copy)
        if shape[0] > 1 and shape[1] > 1 and stride[0] != shape[1] * stride[1]:
            t = t.contiguous()
            stride = t.stride()
        token = stride[1] if shape[1] > 1 else stride[0]
    else:
        tokens, token = shape[0], stride[0]
    head = stride[-2]
    if stride[-1] != 1 or (token | head) & 7 or t.data_ptr() & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:                       # contiguous already, but on an odd address
            t = t.clone(memory_format=torch.contiguous_format)
        head, token = cache.head_dim, shape[-2] * cache.head_dim
    return t, tokens, shape[-2], token, head


def _call(cache: KVCache4bit, what: str, entry, *args):
    """Runs a C entry point on the cache's device and its current stream."""
    index = cache._index
    # (the stream's handle without the Stream object that torch.cuda.current_stream() makes: 3 us of a 20 us call)
    if torch._C._cuda_getDevice() == index:
        status = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        N.check(status, what)


# ---------------------------------------------------------------------- operators
def append_kv_4bit(cache: KVCache4bit, layer: int, k: Tensor, v: Tensor, page_table: Tensor, seq_lens: Tensor,
                   cu_seqlens: Optional[Tensor] = None) -> None:
    """Quantises new tokens' keys and values into the last places of their sequences.

    ``k``, ``v``: [tokens, kv heads, head_dim] (or [batch, new, kv heads, head_dim]) in the cache's dtype, any strides.
    ``page_table`` int32 [batch, pages] and ``seq_lens`` int32 [batch], the lengths WITH the new tokens; sequence b's
    rows are ``cu_seqlens[b]`` .. ``cu_seqlens[b + 1]`` (int32 [batch + 1]), or an equal share of all without it.  Rows
    past ``cu_seqlens[-1]`` and tokens whose place would be negative, or behind what the page table can hold, are skipped.  The
    codes are those of ``quantize_4bit``.  A page that is written must belong to one sequence only (``KVCache4bit.extend`` sees to it).
    """
    _check_cache(cache, layer, "append_kv_4bit")
    kr, tokens, _, k_token, k_head = _rows("k", k, cache.num_kv_heads, cache)
    vr, _, _, v_token, v_head = _rows("v", v, cache.num_kv_heads, cache)
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    sq = _seqs(cache, page_table, seq_lens, cu_seqlens, tokens, None)
    _call(cache, "append_kv_4bit", N.lib().mpsbnb_kv4_append, cache._ref, layer, sq, kr.data_ptr(), k_token, k_head,
          vr.data_ptr(), v_token, v_head)


def dequantize_kv_4bit(cache: KVCache4bit, layer: int, page_table: Tensor, seq_lens: Tensor,
                       max_len: Optional[int] = None) -> Tuple[Tensor, Tensor]:
    """The cached keys and values as they stand, [batch, max_len, kv heads, head_dim] each in the cache's dtype; places
    past a sequence's end are zeros.  ``max_len`` defaults to what the page table can hold."""
    _check_cache(cache, layer, "dequantize_kv_4bit")
    sq = _seqs(cache, page_table, seq_lens, None, 0, None)
    if max_len is None:
        max_len = page_table.shape[1] * cache.page_size
    if max_len < 0:
        raise ValueError(f"max_len must not be negative, got {max_len}")
    shape = (page_table.shape[0], int(max_len), cache.num_kv_heads, cache.head_dim)
    k = cache.k_absmax.new_empty(shape)
    v = torch.empty_like(k)
    _call(cache, "dequantize_kv_4bit", N.lib().mpsbnb_kv4_dequantize, cache._ref, layer, sq, max_len, k.data_ptr(), v.data_ptr())
    return k, v


def attention_4bit(q: Tensor, cache: KVCache4bit, layer: int, page_table: Tensor, seq_lens: Tensor,
                   cu_seqlens: Optional[Tensor] = None, max_seqlen: Optional[int] = None, causal: bool = True,
                   window: Optional[int] = None, scale: Optional[float] = None, out: Optional[Tensor] = None,
                   return_lse: bool = False):
    """softmax(scale q K^T) V over the cached keys and values of each row's sequence.

    ``q``: [tokens, heads, head_dim] or [batch, new, heads, head_dim] in the cache's dtype, the queries of each sequence's
    LAST tokens (the tokens that ``append_kv_4bit`` has just stored, one per sequence when decoding); ``page_table``,
    ``seq_lens`` and ``cu_seqlens`` as there, ``max_seqlen`` the largest number of rows of a sequence: with ``cu_seqlens`` the
    choice of kernels goes by it, not the result.  Without it a call of prompts may launch the kernel for single tokens too,
    which then finds nothing to do.
    heads / kv heads consecutive heads share a key/value head.  The query at place p sees the keys up to p - with ``window``
    only the last ``window`` of them - or all of its sequence when not ``causal``.  ``scale`` defaults to head_dim ** -0.5.

    Returns [..., heads, head_dim] like ``q`` (in ``out``, if given: contiguous), and with ``return_lse`` also the
    natural logarithm of each row's sum of exponentials, fp32 [..., heads].  A row that sees no key gives zeros and
    -inf; rows past ``cu_seqlens[-1]`` stay as they were in ``out``, and are zeros without it.
    """
    _check_cache(cache, layer, "attention_4bit")
    qr, tokens, heads, token, head = _rows("q", q, None, cache)
    if heads == 0 or heads % cache.num_kv_heads:
        raise ValueError(f"q has {heads} heads, which {cache.num_kv_heads} key/value heads do not divide")
    if window is not None and (window <= 0 or not causal):
        raise ValueError(f"window must be positive and needs causal=True, got {window}")
    sq = _seqs(cache, page_table, seq_lens, cu_seqlens, tokens, max_seqlen)
    if out is None:
        like = torch.empty_like if cu_seqlens is None else torch.zeros_like
        out = like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() or out.data_ptr() & 15:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor of shape {tuple(q.shape)} on {q.device}, 16-byte aligned")
    elif out.untyped_storage().data_ptr() == qr.untyped_storage().data_ptr():
        qr = qr.clone(memory_format=torch.contiguous_format)   # rows of q are read after others' outputs have been written
        token, head = heads * cache.head_dim, cache.head_dim
    lse = None
    if return_lse:
        lse = torch.full(q.shape[:-1], float("-inf"), dtype=torch.float32, device=q.device)
    lib = N.lib()
    nbytes = lib.mpsbnb_attention_4bit_workspace_bytes(cache._ref, sq, heads)
    ws = cache.data.new_empty(nbytes)
    _call(cache, "attention_4bit", lib.mpsbnb_attention_4bit, cache._ref, layer, sq, qr.data_ptr(), token, head, heads,
          1 if causal else 0, 0 if window is None else min(window, 1 << 30), cache.head_dim ** -0.5 if scale is None else scale, out.data_ptr(),
          None if lse is None else lse.data_ptr(), ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out


def copy_kv_pages_4bit(cache: KVCache4bit, src: Sequence[int], dst: Sequence[int]) -> None:
    """Copies the pages ``src[i]`` to ``dst[i]`` in every layer.  ``src`` and ``dst`` are lists of page numbers on the host; a page
    may be copied to several places, but not be written twice or both read and written."""
    _check_cache(cache, 0, "copy_kv_pages_4bit")
    src, dst = list(src), list(dst)
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} source pages but {len(dst)} destinations")
    if not src:
        return
    for name, pages in (("src", src), ("dst", dst)):
        if min(pages) < 0 or max(pages) >= cache.num_pages:
            raise IndexError(f"{name} names a page outside the cache's {cache.num_pages}")
    targets = set(dst)
    if len(targets) != len(dst):
        raise ValueError("a page is written twice")
    if not targets.isdisjoint(src):
        raise ValueError("a page is both source and destination")
    array = C.c_int32 * len(src)
    _call(cache, "copy_kv_pages_4bit", N.lib().mpsbnb_kv4_copy_pages, cache._ref, array(*src), array(*dst), len(src))
