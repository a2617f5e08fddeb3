"""Which attention kernels a call over the 4-bit cache runs, as the library itself tells it (no GPU: 148 SMs are taken)."""
import ctypes as C

import pytest

from mps_bitsandbytes_b200 import _native as N

TOKENS, PROMPTS, SHARED = 1, 2, 4


def kernels(heads, kv_heads, new, places, head_dim=128, longest=None, window=0, even=False):
    cache = N.Kv4Cache(1 << 20, 1 << 16, 1, kv_heads, head_dim, 64, 64, 0, 0)
    tokens, width = sum(new), -(-places // 64)
    seqs = N.Kv4Seqs(1 << 21, width, 1 << 22, None if even else 1 << 23, tokens, width, len(new), max(new, default=0) if longest is None else longest)
    return N.lib().mpsbnb_attention_4bit_kernels(C.byref(cache), C.byref(seqs), heads, window)


@pytest.mark.parametrize("want,args", [
    (TOKENS, dict(heads=32, kv_heads=8, new=[1], places=200, even=True)),
    (TOKENS, dict(heads=64, kv_heads=8, new=[1] * 64, places=16384, even=True)),
    (TOKENS, dict(heads=12, kv_heads=1, new=[4] * 7, places=9001, head_dim=64, window=4095)),
    (TOKENS, dict(heads=8, kv_heads=8, new=[300], places=300)),                     # too little for the prompt kernel
    (PROMPTS, dict(heads=64, kv_heads=8, new=[4096], places=4096, even=True)),
    (PROMPTS | SHARED, dict(heads=32, kv_heads=8, new=[509, 509], places=24000)),
    (PROMPTS, dict(heads=16, kv_heads=4, new=[1023, 700, 900, 300, 1000, 500], places=1023, head_dim=256)),
    (TOKENS | PROMPTS | SHARED, dict(heads=16, kv_heads=4, new=[1] * 7 + [400], places=4096)),   # 8 x 4 x 7 blocks of rows: under two rounds
    (TOKENS | PROMPTS, dict(heads=32, kv_heads=8, new=[1] * 255 + [2048], places=4096)),
    (0, dict(heads=8, kv_heads=8, new=[], places=64)),
    (-1, dict(heads=9, kv_heads=8, new=[1], places=64)), (-1, dict(heads=8, kv_heads=8, new=[1], places=64, window=-1))])
def test_kernels_of_a_call(want, args):
    assert kernels(**args) == want


@pytest.mark.parametrize("heads,kv_heads,batch,places", [(64, 8, 64, 16384), (64, 8, 32, 4096), (32, 8, 200, 2048), (8, 1, 512, 65536)])
def test_single_tokens_are_seen_for_what_they_are_without_the_longest(heads, kv_heads, batch, places):
    told = dict(heads=heads, kv_heads=kv_heads, new=[1] * batch, places=places)
    assert kernels(**told) == kernels(**told, longest=batch) == TOKENS

    def workspace(longest):
        cache = N.Kv4Cache(1 << 20, 1 << 16, 1, kv_heads, 128, 64, 64, 0, 0)
        seqs = N.Kv4Seqs(1 << 21, places // 64, 1 << 22, 1 << 23, batch, places // 64, batch, longest)
        return N.lib().mpsbnb_attention_4bit_workspace_bytes(C.byref(cache), C.byref(seqs), heads)
    assert workspace(batch) == workspace(1)                          # (the tiles are as wide, too)


def test_prompts_without_the_longest_go_where_prompts_go():
    for new in ([700, 300], [2048] * 8, [1] * 30 + [900]):
        assert kernels(32, 8, new, 4096, longest=sum(new)) & PROMPTS


def test_device_status_codes_say_which_kernel_they_are_from():
    """Page numbers (401) and places without room (430) are the caller's business: no other kernel's code may look like them."""
    import glob
    import os
    import re
    csrc = os.path.join(os.path.dirname(N.LIB_PATH), "..", "csrc")
    owners = {}
    for path in glob.glob(os.path.join(csrc, "*.cu")):
        text = open(path).read()
        codes = set(map(int, re.findall(r"_status, (\d+)\)", text))) | set(map(int, re.findall(r"AP_WAIT\([^;]*?, (\d+)\)", text)))
        for code in codes:
            owners.setdefault(code, set()).add(os.path.basename(path))
    assert len(owners) > 30
    assert not {c: f for c, f in owners.items() if len(f) > 1}
    assert not {401, 430} & set(owners)
