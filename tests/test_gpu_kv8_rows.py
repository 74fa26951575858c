"""8-bit cache attention of up to 32 rows per KV head: a row's bits depend on its query, its position and
the cache, not on the rows beside it, so that verifying a draft gives what decoding it gave."""
import math

import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests import _kv8 as ref
from tests._gpu import dev
from tests._kv8 import HD
from tests.test_gpu_kv8 import i32, make_desc, table_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


def attend(desc, q, cache, b, window=0, sinks=0):
    out = torch.full_like(q, 7.25)
    ck.paged_attention_verify_kv8(desc, q, *cache, table_of(b), i32(b.cu), i32(b.ctxs), None, out, window, sinks)
    return out.view(torch.int16)


@pytest.mark.parametrize("q_lens,ctxs,nh,nkv,window,sinks", [
    ([3], [301], 16, 8, 0, 0), ([3] * 5, [900] * 5, 32, 8, 0, 0), ([4], [9000], 16, 2, 0, 0), ([7] * 30, [700] * 30, 32, 8, 0, 0),
    ([2] * 30, [900] * 30, 8, 2, 300, 4), ([8], [5000], 32, 8, 0, 0), ([16, 20], [200, 900], 1, 1, 0, 0),
    ([13], [700], 8, 4, 100, 3)])
@pytest.mark.parametrize("other", [0.0, 0.01, 20.0, math.nan])
def test_the_other_rows_contents(q_lens, ctxs, nh, nkv, window, sinks, other):
    """Every other row zero, small, large (its scores move the references far more often) or NaN."""
    d = dev()
    b = ref.batch(q_lens, ctxs, 1)
    g = torch.Generator(device=d).manual_seed(2)
    q = (torch.randn((b.total, nh * HD), generator=g, device=d) * 1.5).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 3, d)
    desc = make_desc(b, nh, nkv)
    want = attend(desc, q, cache, b, window, sinks)
    row = b.total // 2
    changed = q * other
    changed[row] = q[row]
    assert torch.equal(attend(desc, changed, cache, b, window, sinks)[row], want[row])
    # and one head of the row alone
    changed = q * other
    h = slice((nh // 2) * HD, (nh // 2 + 1) * HD)
    changed[row, h] = q[row, h]
    assert torch.equal(attend(desc, changed, cache, b, window, sinks)[row, h], want[row, h])


@pytest.mark.parametrize("ctx", [17, 20, 30, 32, 301, 2000, 9002])
@pytest.mark.parametrize("nh,nkv,seqs", [(32, 8, 1), (32, 8, 12), (16, 8, 40), (8, 8, 3), (8, 2, 4)])
def test_one_row_and_several(ctx, nh, nkv, seqs):
    """The first row of a verify pass against the same row decoded alone, where the pass ends in the same
    page.  The plans are the same: one bound on the contexts, one row tile, and row counts for which the
    merge takes as many warps per row."""
    d = dev()
    first = (ctx - 1) // 16 * 16 + 1  # context of the first row: the page's first token
    n = min(4, ctx - first + 1)
    many, one = ref.batch([n] * seqs, [first + n - 1] * seqs, 4), ref.batch([1] * seqs, [first] * seqs, 4)
    one.tables, one.blocks, one.max_pages = many.tables, many.blocks, many.max_pages
    q = (torch.randn((many.total, nh * HD), generator=torch.Generator(device=d).manual_seed(5), device=d) * 1.5).to(torch.bfloat16)
    cache = ref.random_cache(many.blocks, nkv, 6, d)
    a = attend(make_desc(many, nh, nkv, max_ctx=9100), q, cache, many)
    c = attend(make_desc(one, nh, nkv, max_ctx=9100), q[::n].contiguous(), cache, one)
    assert torch.equal(a[::n], c)
