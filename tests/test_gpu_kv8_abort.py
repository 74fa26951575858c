"""The 8-bit cache attention's bounded waits giving up: with the poll limit at zero
(ekernel_set_wait_limit) the first wait not already met raises the CTA's abort flag, every role leaves its loop, the
producer drains its copies, the issuer its products, tensor memory is freed, and the call returns
ECPU_ERR_KERNEL in synchronous mode.  With limits of a few polls some waits are met and others not, so
products and copies are in flight when a role gives up; such a call reports the error or is exact.  The
next call with the kernel's own limit gives the bits of the first.  No fault, trap or endless wait is
involved: every wait is bounded, and what is waited for completes.  In a child process (synchronous mode
is read at load)."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

_SCRIPT = r"""
import sys
import torch
sys.path.insert(0, sys.argv[1])
from pilm_b200 import bindings as abi, ckernel as ck
from tests import _kv8 as ref
from tests.test_gpu_kv8 import i32, make_desc, table_of
abi.init()
lib = abi.lib()
d = torch.device("cuda")
gave_up = 0
# token kernel: a CTA per sequence (one and two row tiles; a ring longer and shorter than the context),
# shares of all pages (one warp per head, and several), with a window; chunk kernel: one and two tiles, splits
for q_lens, ctxs, nh, nkv, window, sinks in [
        ([1], [301], 16, 8, 0, 0), ([6], [301], 12, 3, 0, 0), ([1] * 3, [2900] * 3, 4, 2, 0, 0),
        ([3] * 40, [3000 + i for i in range(40)], 32, 8, 0, 0), ([1], [30000], 16, 2, 0, 0),
        ([7] * 30, [2000] * 30, 32, 8, 0, 0), ([2] * 30, [2000] * 30, 8, 2, 700, 4),
        ([40], [40], 2, 2, 0, 0), ([300, 200], [300, 900], 8, 2, 0, 0), ([12], [9000], 32, 8, 0, 0),
        ([400], [2000], 8, 2, 300, 20)]:
    b = ref.batch(q_lens, ctxs, 1)
    g = torch.Generator(device=d).manual_seed(1)
    q = torch.randn((b.total, nh * 128), generator=g, device=d).to(torch.bfloat16)
    cache = ref.random_cache(b.blocks, nkv, 2, d)
    desc = make_desc(b, nh, nkv)
    args = (desc, q, *cache, table_of(b), i32(b.cu), i32(ctxs), None)

    def call():
        out = torch.full_like(q, 7.25)
        ck.paged_attention_verify_kv8(*args, out, window=window, sinks=sinks)
        return out
    want = call()
    assert want.isfinite().all()
    for polls in (0, 1, 2, 0, 4):
        lib.ekernel_set_wait_limit(polls)
        try:
            got = call()
            assert polls > 0, f"{q_lens[0]} rows of {ctxs[0]}: no wait gave up"
            assert torch.equal(got, want)
        except RuntimeError as e:
            assert "rc=-4" in str(e) and "did not complete" in str(e), e
            gave_up += polls > 0
        lib.ekernel_set_wait_limit(-1)
        for _ in range(2):
            assert torch.equal(call(), want)
print("ABORT_PATH_OK", gave_up)
"""


@pytest.mark.gpu
def test_waits_that_give_up_report_an_error_and_the_next_call_is_exact():
    env = dict(os.environ, PILM_CUDA_SYNC="1", PYTHONPATH=str(ROOT))
    r = subprocess.run([sys.executable, "-c", _SCRIPT, str(ROOT)], capture_output=True, text=True, timeout=600, env=env)
    assert r.returncode == 0 and "ABORT_PATH_OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
