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
