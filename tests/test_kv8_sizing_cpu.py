"""The workspace size of the 8-bit cache attention, for batches that have nothing to attend."""
import pytest

from pilm_b200 import bindings as abi
from pilm_b200 import ckernel as ck
from tests.test_kv8_cpu import ADDR, attend, desc


# one row per KV head group (the token kernel's plan) and past its 32 rows (the chunk kernel's)
@pytest.mark.parametrize("rows", [1, 3, 64, 4096])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
@pytest.mark.parametrize("empty", [dict(num_seqs=0), dict(total_q=0), dict(num_seqs=0, total_q=0)])
def test_empty_batches_have_a_size_and_a_call(rows, window, sinks, empty):
    a = dict(num_seqs=2, total_q=2 * rows, max_q_len=rows, n_heads=32, n_kv_heads=8, max_context=8192,
             max_blocks_per_seq=512)
    d = desc(**dict(a, **empty))
    n = ck.paged_attention_kv8_workspace_bytes(d, window, sinks)
    # not the 0 of a refused descriptor, and no more than the batch itself would need
    assert 0 < n <= ck.paged_attention_kv8_workspace_bytes(desc(**a), window, sinks)
    assert attend(d, window, sinks, ADDR, n) == 0, abi.last_error()


@pytest.mark.parametrize("over", [dict(max_q_len=0), dict(max_context=0), dict(max_q_len=0, max_context=0)])
def test_bounds_of_zero_are_taken_as_one(over):
    assert ck.paged_attention_kv8_workspace_bytes(desc(**over)) > 0
