"""Attention over the 8-bit cache at the ends of its range."""
import pytest
import torch

import kv_helpers as kh
from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu


def _worst(got, exact, bound, half_step=2.0 ** -24):
    """kh.worst, where a NaN on one side alone is as far off as can be."""
    got = got.double().cpu()
    off = (got - exact).abs()
    share = torch.where(off == 0, 0.0, off / (bound + half_step * (exact.abs() + bound)))
    return float(share.masked_fill(torch.isnan(got) & torch.isnan(exact), 0.0).nan_to_num(float("inf")).max())


def _large_beside_small(seed, fmt, length, hd, heads, large, exponent, small):
    """One page of 16 tokens with the value scale 2^exponent, the others with the least
    one (codes 0 where `small` is "zero")."""
    cache, _ = kh.make(seed, fmt, 1, -(-length // 16), heads, hd, 16, [length])
    page = int(cache.block_table[0, large])
    if small == "zero":
        keep = cache.v[0, page].clone()
        cache.v.view(torch.uint8).zero_()
        cache.v[0, page] = keep
    cache.v_scale.fill_(2.0 ** -64)
    cache.v_scale[0, page] = 2.0 ** exponent
    return cache, kh.mirror(cache)


@pytest.mark.parametrize("small", ["zero", "least"])
@pytest.mark.parametrize("exponent", [45, 63])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,length,fmt", [
    (1, 1, 1, 64, 100, "e4m3"), (1, 2, 2, 64, 9000, "int8"),  # a single row: whole segments, and joined ones
    (1, 8, 1, 128, 100, "int8"), (1, 8, 1, 128, 9000, "e4m3"),
    (4, 2, 1, 32, 5000, "int8"),
    (150, 1, 1, 64, 300, "int8"), (150, 1, 1, 64, 6000, "e4m3"),  # tiles: one run of tokens, and shared out
    (60, 1, 1, 128, 3000, "e4m3"), (60, 1, 1, 256, 2000, "int8")])
def test_value_scales_far_apart(tokens, heads, kv_heads, hd, length, fmt, first, exponent, small):
    """The largest values beside pages of zeros (scale 2^-64) or of the smallest values:
    every token's weight counts in the denominator, whichever page comes first."""
    large = 0 if first else (length - tokens) // 16 - (tokens == 1)
    cache, want = _large_beside_small(300, fmt, length, hd, kv_heads, large, exponent, small)
    q = torch.randn((1, tokens, heads, hd), generator=torch.Generator().manual_seed(7)).cuda()
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [tokens], hd ** -0.5)
    bound, _ = kh.attention_bound(size, total, reach, hd, length, torch.float32)
    assert _worst(got, exact, bound) <= 1
    assert float(exact[0, -1].abs().max()) > 2.0 ** (exponent - 12)
    assert cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,hd,size", [(3, 64, 1e-27), (70, 64, 1e-27), (70, 64, 1e-36), (70, 128, 1e-30),
                                            (60, 256, 1e-33)])
def test_keys_of_zero_under_queries_near_zero(tokens, hd, size, dtype):
    """Scores of exactly 0, also where the factor of the scores underflows: the
    output is the mean of the values seen."""
    cache, _ = kh.make(310, "int8", 2, 8, 1, hd, 16, [tokens, tokens + 21])
    cache.k.zero_()
    cache.k_scale.fill_(2.0 ** -64)
    want = kh.mirror(cache)
    q = (torch.randn((2, tokens, 1, hd), generator=torch.Generator().manual_seed(3)) * size).to(dtype).cuda()
    for scale in (None, 1e-30):
        got = cache.attend(q, scale=scale)
        exact, s, total, reach = ref.attend(want, q.cpu(), [tokens] * 2, scale or hd ** -0.5)
        bound, half_step = kh.attention_bound(s, total, reach, hd, tokens + 21, dtype)
        assert _worst(got, exact, bound, half_step) <= 1


@pytest.mark.parametrize("tokens,hd", [(1, 64), (3, 64), (3, 128), (70, 64), (70, 128), (60, 256)])
def test_pages_never_written_read_as_zeros(tokens, hd):
    """A new cache whose lengths were advanced, nothing written."""
    from ttjam_gottagofast_b200 import KVCache

    cache = KVCache(2, 128, 1, hd, page_size=32)
    cache.advance(tokens + 30)
    q = torch.randn((2, tokens, 1, hd), generator=torch.Generator().manual_seed(3)).cuda()
    for k in (q, q * 1e-30):
        assert torch.equal(cache.attend(k), torch.zeros_like(q))
    assert not cache.read()[0].any()
    assert cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("tokens,hd", [(1, 64), (3, 64), (3, 128), (70, 64), (70, 128), (60, 256)])
def test_one_channel_of_a_query_far_above_the_others(tokens, hd, dtype):
    """q's first channel is 2^13 times the others, and the keys are 0 there: the others
    count with all of their bits. A score is off by (hd / 16 + 2) 2^-22 of the sum of
    magnitudes (attention_bound), and the pieces of q lose 2^-22 of an element or 2^-39 of
    the row's largest."""
    length = tokens + 200
    cache, _ = kh.make(320, "int8", 1, 20, 1, hd, 16, [length])
    cache.k[..., 0] = 0
    want = kh.mirror(cache)
    q = torch.randn((1, tokens, 1, hd), generator=torch.Generator().manual_seed(3))
    q[..., 0] = 2.0 ** 13
    q = q.to(dtype).cuda()
    got = cache.attend(q)
    exact, size, total, _ = ref.attend(want, q.cpu(), [tokens], hd ** -0.5)
    k = ref.read(want, "k", 0)[0][:, 0].abs()
    qq = q[0, :, 0].double().abs().cpu()
    reach = hd ** -0.5 * ((qq + qq.amax(-1, keepdim=True) * 2.0 ** -17) @ k.T).amax(-1)[None, :, None]
    bound, half_step = kh.attention_bound(size, total, reach, hd, length, dtype)
    assert _worst(got, exact, bound, half_step) <= 1


@pytest.mark.parametrize("tokens,hd", [(1, 64), (3, 128), (70, 64), (70, 128), (60, 256)])
@pytest.mark.parametrize("bad", [0.3, -1.0, 2.0 ** 70, 2.0 ** -70, float("inf")])
@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
def test_scales_that_no_write_makes_are_latched(name, bad, tokens, hd):
    """Attention takes a value scale by its exponent, so one that is no power of two, or out
    of the format's range, would be wrong without a word: it counts as NaN and is latched.
    Other heads and sequences do not know of it."""
    cache, _ = kh.make(330, "int8", 2, 12, 2, hd, 16, [tokens + 90, tokens + 40])
    q = torch.randn((2, tokens, 2, hd), generator=torch.Generator().manual_seed(3)).cuda()
    want = cache.attend(q)
    getattr(cache, name)[0, int(cache.block_table[0, 2]), 1] = bad
    got = cache.attend(q)
    assert cache.read_device_status() == (-7, 0x5400)
    assert torch.isnan(got[0, :, 1]).all()
    assert kh.same_bits(got[0, :, 0], want[0, :, 0]) and kh.same_bits(got[1], want[1])


@pytest.mark.parametrize("bad", [0.3, -1.0, 2.0 ** 70, float("inf")])
def test_appending_to_a_page_with_such_a_scale(bad):
    """The page's older codes cannot be moved exactly: its scale becomes NaN, latched."""
    cache, _ = kh.make(331, "int8", 2, 2, 1, 16, 16, [5, 16])
    pages = cache.block_table[:, 0].tolist()
    cache.k_scale[0, pages] = bad
    cache.lengths.add_(torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    x = torch.ones((2, 1, 1, 16), device="cuda")
    cache.write(x, x, new_tokens=torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    assert cache.read_device_status() == (-7, 0x5400)
    assert torch.isnan(cache.k_scale[0, pages[0]]).all()
    assert float(cache.k_scale[0, pages[1]]) == pytest.approx(bad)  # no new token there
    cache.lengths.copy_(torch.tensor([6, 0], dtype=torch.int32, device="cuda"))
    assert torch.isnan(cache.read(max_tokens=6)[0][0]).all()
    # started anew, the page is as any other
    cache.lengths.fill_(1)
    cache.write(x, x)
    assert torch.equal(cache.read(max_tokens=1)[0], x) and cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("tokens,heads,hd", [(1, 2, 64), (3, 2, 128), (70, 2, 64), (130, 1, 128), (60, 1, 256)])
def test_moving_references_give_numbers(tokens, heads, hd):
    """Scores that grow along the sequence, so that sums are rescaled all the way."""
    cache, _ = kh.make(72, "int8", 2, 20, heads, hd, 64, [1100, 700])
    order = torch.arange(20).float()
    for b in range(2):
        cache.k_scale[0, cache.block_table[b].long()] = torch.exp2(torch.floor(order / 3) - 6)[:, None].cuda()
    want = kh.mirror(cache)
    q = torch.randn((2, tokens, heads, hd), generator=torch.Generator().manual_seed(3)).cuda()
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [tokens] * 2, hd ** -0.5)
    bound, _ = kh.attention_bound(size, total, reach, hd, 1100, torch.float32)
    assert not torch.isnan(exact).any() and _worst(got, exact, bound) <= 1


def test_shared_pages_and_a_padded_batch_give_numbers():
    """Two sequences over the same pages, read only, padded to more rows than a
    sequence has room for."""
    cache, _ = kh.make(75, "e4m3", 2, 2, 1, 32, 16, [32, 20])
    cache.block_table[1] = cache.block_table[0]
    want = kh.mirror(cache)
    q = torch.randn((2, 40, 3, 32), generator=torch.Generator().manual_seed(4)).cuda()
    got = cache.attend(q, new_tokens=torch.tensor([2, 1], dtype=torch.int32, device="cuda"))
    exact, size, total, reach = ref.attend(want, q.cpu(), [2, 1], 32 ** -0.5)
    bound, _ = kh.attention_bound(size, total, reach, 32, 32, torch.float32)
    assert _worst(got, exact, bound) <= 1 and not got[0, 2:].any() and not got[1, 1:].any()
