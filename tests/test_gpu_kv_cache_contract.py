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
