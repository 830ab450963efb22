"""A bounded wait of the attention's tile kernel that runs out ends the kernel cleanly.

tt_test_arm_kv_wait_timeout arms a one-shot test switch: in the kernel's next launch the
queries are never announced, a wait on a flag that nothing sets, which gives up after 2^28
cycles, about 0.15 s. The kernel latches TT_ERR_DEVICE_TIMEOUT, stops issuing work, waits for the products it had issued, frees its tensor memory and
returns. The test checks the latched status, then that the next calls, which allocate tensor
memory on every multiprocessor again, give the bits of those before. No GPU fault, trap or
unbounded wait is involved."""
import pytest
import torch

import kv_helpers as kh
from ttjam_gottagofast_b200 import _lib

# the waits that this holds up, all within microseconds of one another: the MMA warp's for
# the queries, the converters' for a free place, the softmax warps' for the first scores
HELD_UP = (0x6000, 0x6300, 0x6400, 0x6600)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hd,length", [(64, 70), (64, 900), (128, 900), (256, 900)])
def test_wait_that_runs_out_latches_a_timeout_and_the_next_calls_are_clean(hd, length, dtype):
    lib = _lib.load()
    cache, _ = kh.make(400, "e4m3", 40, 15, 4, hd, 64, [length] * 40)
    q = torch.randn((40, 70, 4, hd), generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    want = cache.attend(q)
    assert not torch.isnan(want).any() and cache.read_device_status() == (0, 0)
    assert lib.tt_test_arm_kv_wait_timeout() == 0
    cache.attend(q)
    code, detail = cache.read_device_status()
    assert code == _lib.TT_ERR_DEVICE_TIMEOUT and detail in HELD_UP, (code, hex(detail))
    for _ in range(3):  # the switch was one-shot
        assert kh.same_bits(cache.attend(q), want)
    assert cache.read_device_status() == (0, 0)
