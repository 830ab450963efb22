"""Attention over the 8-bit cache for float16 and bfloat16 rows: fp32 accuracy
before the one rounding to the rows' type, whether a row is alone or has
neighbours."""
import pytest
import torch

import kv_helpers as kh
from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _bound(size, total, reach, hd, tokens, dtype):
    """attention_bound as for fp32 rows: no rounding of a probability to the rows'
    type. The output's own rounding is half a step of that type."""
    eps = kh.attention_bound(size, total, reach, hd, tokens, torch.float32)[0]
    info = torch.finfo(dtype)
    return eps + info.smallest_normal * info.eps / 2, info.eps / 2


SHAPES = [  # batch, tokens, heads, kv_heads, head_dim, page, lengths
    (2, 1, 8, 1, 64, 64, [700, 61]),
    (1, 1, 16, 2, 128, 16, [900]),
    (2, 5, 2, 1, 48, 32, [400, 9]),
    (1, 3, 4, 2, 256, 128, [300]),
    (2, 70, 2, 2, 64, 64, [500, 70]),
    (1, 33, 4, 2, 128, 16, [700]),
    (1, 60, 1, 1, 256, 64, [400]),
    (1, 90, 3, 3, 80, 32, [333]),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_rows_are_rounded_once(case, dtype, fmt):
    batch, n, heads, kv_heads, hd, page, lengths = SHAPES[case]
    cache, want = kh.make(200 + case, fmt, batch, -(-max(lengths) // page), kv_heads, hd, page, lengths)
    q = torch.randn((batch, n, heads, hd), generator=torch.Generator().manual_seed(case))
    q = q.to(DTYPES[dtype]).cuda()
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [n] * batch, hd ** -0.5)
    bound, half_step = _bound(size, total, reach, hd, max(lengths), q.dtype)
    assert not torch.isnan(got).any() and kh.worst(got, exact, bound, half_step) <= 1
    assert cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_row_is_the_same_alone_and_with_neighbours(dtype):
    """The last of 1, 9 and 80 new tokens is the same row: each within the same
    bound, so that what a row gets does not hang on the call's shape."""
    cache, want = kh.make(230, "e4m3", 1, 12, 2, 128, 64, [700])
    q = torch.randn((1, 80, 2, 128), generator=torch.Generator().manual_seed(4)).to(DTYPES[dtype]).cuda()
    exact, size, total, reach = ref.attend(want, q[:, -1:].cpu(), [1], 128 ** -0.5)
    bound, half_step = _bound(size, total, reach, 128, 700, q.dtype)
    for n in (1, 9, 80):
        got = cache.attend(q[:, -n:])[:, -1:]
        assert not torch.isnan(got).any() and kh.worst(got, exact, bound, half_step) <= 1, n
