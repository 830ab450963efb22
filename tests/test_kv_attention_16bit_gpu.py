"""Attention over the 8-bit cache for float16 and bfloat16 rows: fp32 accuracy
before the one rounding to the rows' type, whether a row is alone or has
neighbours, and over long contexts."""
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


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hd,rows,batch", [(64, 70, 160), (128, 48, 160), (256, 40, 160), (128, 48, 30), (256, 40, 30)])
def test_long_contexts_do_not_drift(hd, rows, batch, dtype):
    """400000 tokens a sequence, in 160 sequences (over the same pages, read only), so
    many that no sequence's tokens are shared out, or 30, whose tokens are. Tensor cores
    add by rounding toward zero, which moves every sum the same way: the mean error along
    the output's sign shows it. Sums are taken out after 4096 tokens (bfloat16: 8192), so a
    run is at most 512 (1024) additions, two pieces for 16 tokens, each of which cuts the 16
    products and the sum so far: below 2^-22 of that sum, 2^-13 (2^-12) of the output, and in
    the mean, as the sum so far is half of the run's on average, half of that. All
    else rounds both ways and is within attention_bound (whose runs are of 1024
    tokens). The output's rounding is half a step, eps / 2, at most; the mean over
    rows * hd * 2 elements, whose roundings fall anyhow, is below five times
    eps / 4 / sqrt(rows * hd * 2)."""
    length, page = 400000, 128
    run = (4096 if dtype == "fp16" else 8192) / 8 * 2.0 ** -22
    g = torch.Generator().manual_seed(5)
    columns = length // page
    ramp = torch.linspace(-1, 1, columns).view(-1, 1, 1, 1)
    base = torch.linspace(20, 120, hd)[torch.randperm(hd, generator=g)]
    k = torch.randint(-60, 61, (columns, 1, page, hd), generator=g).float()
    k[..., :1] = ramp * 100
    v = base * (0.6 + 0.4 * ramp) * (0.8 + 0.2 * torch.rand((columns, 1, page, hd), generator=g))
    k, v = (x.round().to(torch.int8)[None].cuda() for x in (k, v))
    from ttjam_gottagofast_b200 import KVCache

    scales = [torch.full((1, columns, 1), 2.0 ** -6, device="cuda") for _ in range(2)]
    table = torch.arange(columns, dtype=torch.int32, device="cuda").expand(batch, columns).contiguous()
    cache = KVCache.from_tensors(k, v, *scales, table,
                                 torch.full((batch,), length, dtype=torch.int32, device="cuda"))
    q = torch.randn((batch, rows, 1, hd), generator=g) * 0.3
    q[..., 0] = 2.0 * torch.randn((batch, rows, 1), generator=g)  # each row leans to a part of the context
    q = q.to(DTYPES[dtype]).cuda()
    got = cache.attend(q, scale=1.0)
    assert cache.read_device_status() == (0, 0)
    kk, vv = (x.double().view(length, hd) / 64 for x in (k, v))
    hidden = torch.arange(length, device="cuda") > torch.arange(length - rows, length, device="cuda")[:, None]
    bias, eps = 0.0, torch.finfo(q.dtype).eps
    for b in (0, batch - 1):
        qq = q[b, :, 0].double()
        exact = torch.softmax((qq @ kk.T).masked_fill_(hidden, float("-inf")), -1) @ vv
        reach = ((qq.abs() + qq.abs().amax(-1, keepdim=True) / 8) @ kk.abs().T).amax(-1)
        bound, half_step = _bound(exact, vv.sum(0), reach, hd, length, q.dtype)  # every value is positive
        off = got[b, :, 0].double() - exact
        bound = bound + run * exact
        assert bool((off.abs() <= bound + half_step * (exact + bound)).all())
        bias += float((off / exact).mean()) / 2
    assert abs(bias) <= run / 2 + 5 * eps / 4 / (rows * hd * 2) ** 0.5


def test_scratch_for_long_sums_is_asked_for_16_bit_rows_alone():
    """The sums of many 16-bit rows over a long cache stand in scratch as fp32 values; fp32
    rows have theirs in the output, and short caches need none."""
    from ttjam_gottagofast_b200 import KVCache, _lib

    lib = _lib.load()
    need = lambda c, dtype: lib.tt_kv_attention_typed_workspace_bytes(c._structs[0], dtype, 256, 2)  # noqa: E731
    values = 160 * 256 * 2 * 128 * 4
    for room, wanted in ((4096, (0, 0, 0)), (8192, (0, values, 0)), (8256, (0, values, values))):
        c = KVCache(160, room, 2, 128, page_size=64)
        assert tuple(need(c, d) for d in (0, 1, 2)) == wanted
        assert lib.tt_kv_attention_workspace_bytes(c._structs[0], 256, 2) == max(wanted)
        assert need(c, 3) == 0
