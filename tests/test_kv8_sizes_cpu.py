"""Descriptor sizes of the 8-bit cache calls whose products or casts would wrap are refused."""
import pytest

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests.test_kv8_cpu import append, attend, desc


@pytest.mark.parametrize("stride", [1 << 31, 1 << 60, (1 << 63) + 1024, (1 << 64) - 1])
def test_append_refuses_strides_that_wrap(stride):
    assert append(desc(total_q=2, qkv_stride=stride)) == -1 and "qkv_stride" in abi.last_error()


@pytest.mark.parametrize("pages", [1 << 31, (1 << 32) + 4, 1 << 63])
def test_attention_refuses_block_tables_that_wrap(pages):
    d = desc(max_blocks_per_seq=pages)
    assert attend(d) == -1 and "max_blocks_per_seq" in abi.last_error()
    assert ck.paged_attention_kv8_workspace_bytes(d) == 0


@pytest.mark.parametrize("rows", [1, 64])
@pytest.mark.parametrize("context", [1 << 31, 1 << 62, (1 << 64) - 1])
def test_context_bounds_past_any_context_plan_as_the_largest(rows, context):
    a = dict(num_seqs=3, total_q=3 * rows, max_q_len=rows, n_heads=32, n_kv_heads=8, max_blocks_per_seq=1 << 27)
    n = ck.paged_attention_kv8_workspace_bytes(desc(max_context=context, **a))
    assert n == ck.paged_attention_kv8_workspace_bytes(desc(max_context=(1 << 31) - 1, **a)) > 0
