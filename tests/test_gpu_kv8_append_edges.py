"""Ends of the scales' range in the 8-bit cache append."""
import pytest
import torch

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests import _kv8 as ref
from tests._gpu import dev
from tests._kv8 import HD, PAGE
from tests.test_gpu_kv8 import check_store, i32, make_desc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    abi.init()
    yield


def put(b, kc, vc, ks, vs, offset, v, rows=1):
    """`rows` rows of value v (and zero keys) from `offset` of the first page on."""
    d = dev()
    page = b.tables[0][0]
    one, cos = torch.ones(HD, dtype=torch.bfloat16, device=d), torch.ones((64, 64), device=d)
    qkv = torch.zeros((rows, 3 * HD), dtype=torch.bfloat16, device=d)
    qkv[:, 2 * HD:] = v
    desc = make_desc(b, 1, 1, rope_rows=64)
    desc.total_q = rows
    slots = [page * PAGE + offset + i for i in range(rows)]
    before, scale_before = vc.clone(), vs.clone()
    ck.qk_norm_rope_kv_append_kv8(desc, qkv, one, one, cos, torch.zeros_like(cos), i32(list(range(offset, offset + rows))),
                                  i32(slots), kc, vc, ks, vs, torch.empty((rows, HD), dtype=torch.bfloat16, device=d))
    check_store(qkv[:, 2 * HD:].double().view(rows, 1, HD), slots, before, scale_before, vc, vs)


@pytest.mark.parametrize("big", [2.0 ** 127, 2.0 ** 60, 1.0])
@pytest.mark.parametrize("small", [2.0 ** -60, 2.0 ** -100, 2.0 ** -115, 0.0])
def test_kept_zeros_of_a_page_whose_scale_falls_far(big, small):
    """A large row raises the scale so far that the tokens before it become zeros; once it is written
    over by a small one, those zeros are still zeros (scales of up to 2^119 and down to 2^-122: their ratio
    may be past fp32's range)."""
    d = dev()
    b = ref.batch([1], [4], 0)
    kc, vc, ks, vs = ref.random_cache(b.blocks, 1, 1, d)
    v = torch.randn(HD, generator=torch.Generator(device=d).manual_seed(2), device=d)
    put(b, kc, vc, ks, vs, 0, v * 2.0 ** -40, rows=2)
    put(b, kc, vc, ks, vs, 2, v.clamp(-1, 1) * big)
    put(b, kc, vc, ks, vs, 2, v * small)
    page = b.tables[0][0]
    assert not ((vc[page, :3] & 0x7F) == 0x7F).any(), "a NaN code was written"


def test_values_below_the_least_scale():
    """The least scale is 2^-126: what is small beside it is rounded to its steps."""
    d = dev()
    b = ref.batch([1], [4], 1)
    kc, vc, ks, vs = ref.random_cache(b.blocks, 1, 2, d)
    v = torch.randn(HD, generator=torch.Generator(device=d).manual_seed(3), device=d).to(torch.bfloat16)
    put(b, kc, vc, ks, vs, 0, v * 2.0 ** -116, rows=2)  # a page of its own scale
    page = b.tables[0][0]
    assert vs[page].item() >= 2.0 ** -126
    qkv = v * 2.0 ** -126
    desc, one, cos = make_desc(b, 1, 1, rope_rows=64), torch.ones(HD, dtype=torch.bfloat16, device=d), torch.ones((64, 64), device=d)
    x = torch.zeros((1, 3 * HD), dtype=torch.bfloat16, device=d)
    x[0, 2 * HD:] = qkv
    ck.qk_norm_rope_kv_append_kv8(desc, x, one, one, cos, torch.zeros_like(cos), i32([0]), i32([page * PAGE]), kc, vc, ks, vs,
                                  torch.empty((1, HD), dtype=torch.bfloat16, device=d))
    assert vs[page].item() == 2.0 ** -126
    y = x[0, 2 * HD:].double() * 2.0 ** 126
    # half a step of the codes at that scale, 2^-10 below 2^-6; the value itself is exact in fp32
    assert ((ref.values(vc[page, 0, 0]) - y).abs() <= ref.e4m3_step(y) / 2).all()
