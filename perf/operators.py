"""Cases and plain forms of the operators on a paged key/value cache held in 4 bits.

The cache keeps, per layer, page, key/value head and token, the row's NF4 or FP4 codes (two to a byte, the lower
nibble first) and one absmax per block of the row, in the cache's own type: a 16-bit input's absmax loses nothing.
Three operators work on it:

``store``      new tokens are quantised into the pages of their sequences and read back as the values they stand for;
``attention``  softmax(scale q k^T) v over the cached keys and values, for single tokens, for a few tokens that are
               verified together and for whole prompts; a query at position p sees the keys max(0, p - window + 1) .. p;
``copy``       pages are copied within the cache in all layers: what forking a sequence and closing gaps come down to.

``run`` takes the plain form (elementary torch operations in 32 bits) where ``own`` is false and the package's operators
where it is true.
"""
import math
import random

import torch

own = False

_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
_NF4 = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453, -0.28444138169288635,
        -0.18477343022823334, -0.09105003625154495, 0.0, 0.07958029955625534, 0.16093020141124725,
        0.24611230194568634, 0.33791524171829224, 0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
_FP4 = (0.0, 0.0625, 0.125, 0.25, 0.375, 0.5, 0.75, 1.0,
        -0.0, -0.0625, -0.125, -0.25, -0.375, -0.5, -0.75, -1.0)
_CODES = {"nf4": _NF4, "fp4": _FP4}


def _attention(name, batch, new, longest, ragged, heads, kv_heads, head_dim, blocksize, page, quant, dtype, window=0):
    case = {"op": "attention", "batch": batch, "new": new, "longest": longest, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "blocksize": blocksize, "page": page, "quant": quant,
            "dtype": dtype, "window": window}
    return {"name": name, **case} if name else case


def _store(name, batch, new, ragged, kv_heads, head_dim, blocksize, page, quant, dtype):
    case = {"op": "store", "batch": batch, "new": new, "longest": new, "ragged": ragged, "kv_heads": kv_heads,
            "head_dim": head_dim, "blocksize": blocksize, "page": page, "quant": quant, "dtype": dtype}
    return {"name": name, **case} if name else case


def _copy(name, layers, pages, copies, kv_heads, head_dim, blocksize, page, dtype):
    case = {"op": "copy", "layers": layers, "pages": pages, "copies": copies, "kv_heads": kv_heads,
            "head_dim": head_dim, "blocksize": blocksize, "page": page, "quant": "nf4", "dtype": dtype}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one sequence of a 32-head model shortly after its prompt: the step's latency counts
        _attention("token_short", 1, 1, 200, False, 32, 32, 128, 64, 64, "nf4", "float16"),
        # a served batch of a model with 64 query heads on 8, sequences of all lengths
        _attention("token_batch", 32, 1, 4096, True, 64, 8, 128, 64, 64, "nf4", "float16"),
        # the largest batch: the cache's bytes are all that counts
        _attention("token_large", 64, 1, 16384, True, 64, 8, 128, 64, 64, "nf4", "bfloat16"),
        # one sequence with a very long context: its keys have to be shared out over the whole card
        _attention("token_long", 1, 1, 131072, False, 64, 8, 128, 64, 128, "fp4", "bfloat16"),
        # four drafted tokens verified at once, sliding window, one key/value head, small blocks and pages, odd lengths
        _attention("draft_window", 7, 4, 9001, True, 12, 1, 64, 32, 16, "nf4", "bfloat16", 4095),
        # a whole prompt of one sequence
        _attention("prompt", 1, 4096, 4096, False, 64, 8, 128, 64, 64, "nf4", "float16"),
        # prompts of a batch, all of different odd lengths, wide heads
        _attention("prompt_ragged", 6, 1023, 1023, True, 16, 4, 256, 64, 32, "fp4", "bfloat16"),
        # a chunk of a long prompt over what is cached already
        _attention("prompt_chunk", 2, 509, 24000, False, 32, 8, 128, 64, 64, "nf4", "bfloat16"),
        # one decoding step's new rows
        _store("store_tokens", 32, 1, False, 8, 128, 64, 64, "nf4", "float16"),
        # prompts' rows
        _store("store_prompts", 5, 8191, True, 8, 128, 64, 64, "fp4", "bfloat16"),
        # three sequences fork: each copy's last page, which it will write to, in every layer
        _copy("fork", 32, 64, 3, 8, 128, 64, 64, "float16"),
        # half of a cache's pages are gone and the others close the gaps
        _copy("compact", 32, 600, 299, 8, 128, 64, 64, "bfloat16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention", "store", "copy"])
    head_dim, blocksize = rng.choice([(64, 32), (64, 64), (128, 64), (128, 64), (128, 32), (256, 64)])
    page = rng.choice([16, 32, 64, 128])
    quant = rng.choice(["nf4", "fp4"])
    dtype = rng.choice(["float16", "bfloat16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if op == "store":
        batch = _log_int(rng, 1, 32)
        new = _log_int(rng, 1, max(2, 8191 * 8 // (batch * kv_heads)))
        return _store(None, batch, min(new, 8191), rng.random() < 0.5, kv_heads, head_dim, blocksize, page, quant, dtype)
    if op == "copy":
        pages = _log_int(rng, 8, 500)
        return _copy(None, rng.randint(1, 16), pages, rng.randint(1, pages // 2), kv_heads, head_dim, blocksize, page, dtype)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 12, 16])
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 8192)])
    if rng.random() < 0.6:
        batch = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, 1, 2, 3, 5, 8])
        longest = new + _log_int(rng, 1, max(2, min(131072, 4000000 // (batch * kv_heads * head_dim // 64))))
    else:
        batch = _log_int(rng, 1, 8)
        # keeps the scores of a sequence under those of the listed prompts
        new = _log_int(rng, 9, max(10, min(2048, 4096 * 8 // heads)))
        longest = new + rng.choice([0, 0, _log_int(rng, 1, 8000)])
    return _attention(None, batch, new, longest, rng.random() < 0.6, heads, kv_heads, head_dim, blocksize, page, quant, dtype, window)


def _lengths(case):
    """(new tokens, length with them) of every sequence."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    out = []
    for i in range(case["batch"]):
        new, length = case["new"], case["longest"]
        if case["ragged"] and i > 0:
            if new == length:                                # prompts: all of the sequence is new
                new = length = rng.randint(max(1, new // 8), new)
            else:
                new = rng.randint(1, new)
                length = rng.randint(new, length)
        out.append((new, length))
    return out


def _row_bytes(case):
    return case["head_dim"] // 2 + 2 * (case["head_dim"] // case["blocksize"])


def work(case):
    if case["op"] == "copy":
        page_bytes = 2 * case["kv_heads"] * case["page"] * _row_bytes(case)
        return {"bytes": 2 * case["layers"] * case["copies"] * page_bytes, "flops": 0}
    lengths = _lengths(case)
    row = _row_bytes(case)
    if case["op"] == "store":
        rows = 2 * case["kv_heads"] * sum(n for n, _ in lengths)
        # 16-bit rows in, the cache written, the cache read, 16-bit rows out; a division and a search of four steps
        return {"bytes": rows * (2 * 2 * case["head_dim"] + 2 * row), "flops": rows * case["head_dim"] * 6}
    seen = read = 0
    for new, length in lengths:
        first = length - new
        low = max(0, first - case["window"] + 1) if case["window"] else 0
        read += length - low
        if case["window"]:
            seen += sum(min(first + i + 1, case["window"]) for i in range(new))
        else:
            seen += new * first + new * (new + 1) // 2
    rows = sum(n for n, _ in lengths) * case["heads"]
    return {"bytes": 2 * case["kv_heads"] * read * row + rows * case["head_dim"] * 4,
            "flops": 4 * case["heads"] * seen * case["head_dim"]}


def _quantise(x, case):
    """Codes 0 .. 15 of every element and the absmax of every block, in 32 bits (rows of x end in head_dim).
    Values between two codes go to the nearer one; a block of zeros or below 1e-8 keeps 1e-8 as its absmax."""
    code = torch.tensor(_CODES[case["quant"]], dtype=torch.float32, device=x.device)
    blocks = x.float().unflatten(-1, (-1, case["blocksize"]))
    absmax = blocks.abs().amax(-1).clamp_min(1e-8)
    idx = torch.empty(blocks.shape, dtype=torch.uint8, device=x.device)
    flat, a, out = blocks.flatten(0, -2), absmax.flatten(), idx.flatten(0, -2)
    step = 1 << 17
    for i in range(0, flat.shape[0], step):
        v = flat[i:i + step] / a[i:i + step, None]
        out[i:i + step] = (v[..., None] - code).abs().argmin(-1).to(torch.uint8)
    return idx.flatten(-2), absmax.to(x.dtype)


def _values(idx, absmax, case):
    code = torch.tensor(_CODES[case["quant"]], dtype=torch.float32, device=idx.device)
    return (code[idx.long()].unflatten(-1, (-1, case["blocksize"])) * absmax.float()[..., None]).flatten(-2)


def _some_codes(rows, case, gen, spread, device):
    """Codes and absmax of normal rows whose channels have different sizes (for caches that are there already)."""
    d, bs = case["head_dim"], case["blocksize"]
    size = torch.exp(spread * torch.randn(case["kv_heads"], d, generator=gen, device=device))
    code = torch.tensor(_CODES[case["quant"]], dtype=torch.float32, device=device)
    order = torch.argsort(code[:16], stable=True)
    if case["quant"] == "fp4":
        order = order[order != 8]                            # -0.0 is never written
    middles = (code[order][1:] + code[order][:-1]) / 2
    idx = torch.empty(rows, case["kv_heads"], d, dtype=torch.uint8, device=device)
    absmax = torch.empty(rows, case["kv_heads"], d // bs, dtype=_DTYPES[case["dtype"]], device=device)
    for i in range(0, rows, 1 << 14):
        n = min(rows - i, 1 << 14)
        x = torch.randn(n, case["kv_heads"], d, generator=gen, device=device) * size
        blocks = x.unflatten(-1, (-1, bs))
        a = blocks.abs().amax(-1).to(absmax.dtype)
        idx[i:i + n] = order.to(torch.uint8)[torch.bucketize((blocks / a[..., None].float()).flatten(-2), middles)]
        absmax[i:i + n] = a
    return idx, absmax


def _paging(case, gen, device):
    """Pages of every sequence in a shuffled order, some of the cache's pages unused."""
    lengths = _lengths(case)
    need = [-(-length // case["page"]) for _, length in lengths]
    total = sum(need) + 3
    order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
    table = torch.zeros(case["batch"], max(need), dtype=torch.int32, device=device)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    ends = [0]
    for new, _ in lengths:
        ends.append(ends[-1] + new)
    return {"lengths": lengths, "pages": total, "table": table,
            "seq_lens": torch.tensor([length for _, length in lengths], dtype=torch.int32, device=device),
            "ends": torch.tensor(ends, dtype=torch.int32, device=device), "tokens": ends[-1]}


def _slots(state, i, first, last):
    """Places (page * page size + offset) of the positions first .. last - 1 of sequence i."""
    size = state["case"]["page"]
    pos = torch.arange(first, last, device=state["table"].device)
    return state["table"][i, pos // size].long() * size + pos % size


def _own_cache(case, layers, pages, device):
    import mps_bitsandbytes_b200 as bnb
    return bnb.KVCache4bit(layers, pages, case["kv_heads"], case["head_dim"], page_size=case["page"],
                           blocksize=case["blocksize"], quant_type=case["quant"], dtype=_DTYPES[case["dtype"]],
                           device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    heads, d, page, nb = case["kv_heads"], case["head_dim"], case["page"], case["head_dim"] // case["blocksize"]
    state = {"case": case}
    if case["op"] == "copy":
        order = torch.randperm(case["pages"], generator=gen, device=device).tolist()
        state["src"], state["dst"] = order[:case["copies"]], order[case["copies"]:2 * case["copies"]]
        shape = (case["layers"], case["pages"], 2 * heads * page * _row_bytes(case))
        data = torch.randint(0, 256, shape, generator=gen, device=device, dtype=torch.uint8)
        if own:
            state["cache"] = _own_cache(case, case["layers"], case["pages"], device)
            state["cache"].data.copy_(data.view(state["cache"].data.shape))
        else:
            state["data"] = data
        return state
    state.update(_paging(case, gen, device))
    slots = state["pages"] * page
    if case["op"] == "store":
        size = torch.exp(torch.randn(heads, d, generator=gen, device=device))
        state["k"] = (torch.randn(state["tokens"], heads, d, generator=gen, device=device) * size).to(dtype)
        state["v"] = torch.randn(state["tokens"], heads, d, generator=gen, device=device).to(dtype)
        if own:
            state["cache"] = _own_cache(case, 1, state["pages"], device)
        else:
            for name in "kv":
                state[name + "_codes"] = torch.zeros(slots, heads, d, dtype=torch.uint8, device=device)
                state[name + "_absmax"] = torch.zeros(slots, heads, nb, dtype=dtype, device=device)
        return state
    state["q"] = torch.randn(state["tokens"], case["heads"], d, generator=gen, device=device).to(dtype)
    rows = {"k": _some_codes(slots, case, gen, 0.5, device), "v": _some_codes(slots, case, gen, 0.2, device)}
    if own:
        cache = _own_cache(case, 1, state["pages"], device)
        for name, (idx, absmax) in rows.items():
            packed = idx[..., 0::2] | (idx[..., 1::2] << 4)
            # the cache's views: pages, heads, groups of 16 tokens, tokens, bytes or blocks
            for view, rows_ in ((getattr(cache, name + "_codes")[0], packed), (getattr(cache, name + "_absmax")[0], absmax)):
                view.copy_(rows_.view(-1, page // 16, 16, heads, rows_.shape[-1]).permute(0, 3, 1, 2, 4))
        state["cache"] = cache
    else:
        for name, (idx, absmax) in rows.items():
            state[name + "_codes"], state[name + "_absmax"] = idx, absmax
    return state


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "copy":
        src = torch.tensor(state["src"], device=state["data"].device)
        dst = torch.tensor(state["dst"], device=state["data"].device)
        state["data"][:, dst] = state["data"][:, src]
        return state["data"]
    if case["op"] == "store":
        return _plain_store(state, case)
    return _plain_attention(state, case)


def _run_own(state, case):
    import mps_bitsandbytes_b200 as bnb
    cache = state["cache"]
    if case["op"] == "copy":
        bnb.copy_kv_pages_4bit(cache, state["src"], state["dst"])
        return cache.data.view(case["layers"], case["pages"], -1)
    one_each = not case["ragged"]
    if case["op"] == "store":
        k, v = state["k"], state["v"]
        bnb.append_kv_4bit(cache, 0, k, v, state["table"], state["seq_lens"], None if one_each else state["ends"])
        return bnb.dequantize_kv_4bit(cache, 0, state["table"], state["seq_lens"], case["longest"])
    q = state["q"]
    window = case["window"] or None
    if one_each:
        q = q.view(case["batch"], case["new"], *q.shape[1:])
        out = bnb.attention_4bit(q, cache, 0, state["table"], state["seq_lens"], window=window)
        return out.view(state["tokens"], *q.shape[2:])
    return bnb.attention_4bit(q, cache, 0, state["table"], state["seq_lens"], cu_seqlens=state["ends"],
                              max_seqlen=case["new"], window=window)


def _plain_store(state, case):
    at = 0
    slots = []
    for i, (new, length) in enumerate(state["lengths"]):
        slots.append(_slots(state, i, length - new, length))
        at += new
    slots = torch.cat(slots)
    out = []
    for name in "kv":
        idx, absmax = _quantise(state[name], case)
        state[name + "_codes"][slots] = idx
        state[name + "_absmax"][slots] = absmax
        x = state[name]
        dense = x.new_zeros(case["batch"], case["longest"], *x.shape[1:])
        for i, (_, length) in enumerate(state["lengths"]):
            places = _slots(state, i, 0, length)
            dense[i, :length] = _values(state[name + "_codes"][places], state[name + "_absmax"][places], case).to(x.dtype)
        out.append(dense)
    return tuple(out)


def _plain_attention(state, case):
    q = state["q"]
    out = torch.empty_like(q)
    group = case["heads"] // case["kv_heads"]
    at = 0
    for i, (new, length) in enumerate(state["lengths"]):
        low = max(0, length - new - case["window"] + 1) if case["window"] else 0
        places = _slots(state, i, low, length)
        k = _values(state["k_codes"][places], state["k_absmax"][places], case).transpose(0, 1)      # heads, keys, dim
        v = _values(state["v_codes"][places], state["v_absmax"][places], case).transpose(0, 1)
        x = q[at:at + new].float().view(new, case["kv_heads"], group, -1).permute(1, 2, 0, 3).flatten(1, 2)
        s = (x @ k.transpose(1, 2)) * case["head_dim"] ** -0.5
        key = torch.arange(low, length, device=q.device)
        pos = torch.arange(length - new, length, device=q.device).repeat(group)[:, None]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | (key <= pos - case["window"])
        s.masked_fill_(hidden, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        y = (p @ v) / p.sum(-1, keepdim=True)
        out[at:at + new] = y.unflatten(1, (group, new)).permute(2, 0, 1, 3).reshape(new, case["heads"], -1).to(q.dtype)
        at += new
    return out


def exact(case, seed):
    """The operators' definitions in 64 bits, head by head and without the plain form's functions."""
    global own
    if case["op"] == "copy":
        saved, own = own, False
        try:
            state = prepare(case, seed)
        finally:
            own = saved
        data = state["data"].clone()
        for a, b in zip(state["src"], state["dst"]):
            data[:, b] = state["data"][:, a]
        return data
    saved, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = saved
    code = torch.tensor(_CODES[case["quant"]], dtype=torch.float64, device="cuda").float().double()
    d, bs = case["head_dim"], case["blocksize"]
    if case["op"] == "store":
        out = []
        for name in "kv":
            x = state[name]
            dense = torch.zeros(case["batch"], case["longest"], case["kv_heads"], d, dtype=torch.float64, device="cuda")
            at = 0
            for i, (new, _) in enumerate(state["lengths"]):
                for b in range(d // bs):
                    part = x[at:at + new, :, b * bs:(b + 1) * bs].double()
                    a = part.abs().max(-1, keepdim=True).values
                    a = torch.maximum(a, torch.tensor(1e-8, dtype=torch.float32, device="cuda").double())
                    # the quotient and its distances are 32-bit numbers by definition; the first of equal distances wins
                    v = (part / a).float().double()
                    best = torch.full_like(v, math.inf)
                    value = torch.zeros_like(v)
                    for c in code:
                        dist = (v - c).abs().float().double()
                        nearer = dist < best
                        best = torch.where(nearer, dist, best)
                        value = torch.where(nearer, c, value)
                    dense[i, :new, :, b * bs:(b + 1) * bs] = value * a.to(x.dtype).double()
                at += new
            out.append(dense)
        return tuple(out)
    out = torch.empty(state["tokens"], case["heads"], d, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    at = 0
    for i, (new, length) in enumerate(state["lengths"]):
        where = torch.arange(length, device="cuda")
        places = state["table"][i].long()[where // case["page"]] * case["page"] + where % case["page"]
        for h in range(case["kv_heads"]):
            k, v = (code[state[n + "_codes"][places, h].long()] * state[n + "_absmax"][places, h].double().repeat_interleave(bs, -1)
                    for n in "kv")
            for g in range(group):
                s = state["q"][at:at + new, h * group + g].double() @ k.T / math.sqrt(d)
                back = torch.arange(length - new, length, device="cuda")[:, None] - where[None]
                seen = back >= 0
                if case["window"]:
                    seen &= back < case["window"]
                s = torch.where(seen, s, -math.inf)
                out[at:at + new, h * group + g] = torch.softmax(s, -1) @ v
        at += new
    return out
