"""The key/value cache without a GPU: what its C entry points refuse before
anything is launched, and the oracle that the GPU tests compare with."""
import ctypes
import math

import pytest
import torch

from oracle import kv_reference as ref
from ttjam_gottagofast_b200 import KVCache, _lib

FAKE = 1 << 20  # an aligned address that no call here reads


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _cache(**other):
    c = _lib.TTKVCache()
    fields = dict(k_codes=FAKE, v_codes=FAKE, k_scale=FAKE, v_scale=FAKE, block_table=FAKE,
                  lengths=FAKE, status=None, num_pages=8, page_size=64, kv_heads=2, head_dim=64,
                  batch=2, table_columns=4, format=0, reserved=0)
    for name, value in {**fields, **other}.items():
        setattr(c, name, value)
    return c


def _strides():
    return (ctypes.c_int64 * 3)(512, 128, 64)


def _write(lib, c, dtype=0, k=FAKE, v=FAKE, ks=True, tokens=1, counts=None):
    return lib.tt_kv_write(ctypes.byref(c) if c else None, dtype, k, v, _strides() if ks else None,
                           _strides(), tokens, counts, None)


def _attend(lib, c, dtype=0, q=FAKE, out=2 * FAKE, tokens=1, heads=2, scale=1.0, ws=None, nbytes=0):
    return lib.tt_kv_attention(ctypes.byref(c), dtype, q, _strides(), tokens, heads, None, scale, out,
                               ws, nbytes, None)


@pytest.mark.parametrize("field,value,code", [
    ("page_size", 8, _lib.TT_ERR_UNSUPPORTED), ("page_size", 48, _lib.TT_ERR_UNSUPPORTED),
    ("page_size", 256, _lib.TT_ERR_UNSUPPORTED), ("head_dim", 8, _lib.TT_ERR_UNSUPPORTED),
    ("head_dim", 72, _lib.TT_ERR_UNSUPPORTED), ("head_dim", 272, _lib.TT_ERR_UNSUPPORTED),
    ("kv_heads", 0, _lib.TT_ERR_INVALID_ARGUMENT), ("num_pages", 0, _lib.TT_ERR_INVALID_ARGUMENT),
    ("batch", -1, _lib.TT_ERR_INVALID_ARGUMENT), ("table_columns", 0, _lib.TT_ERR_INVALID_ARGUMENT),
    ("table_columns", 1 << 25, _lib.TT_ERR_UNSUPPORTED), ("format", 2, _lib.TT_ERR_INVALID_ARGUMENT),
    ("reserved", 1, _lib.TT_ERR_INVALID_ARGUMENT), ("k_codes", None, _lib.TT_ERR_INVALID_ARGUMENT),
    ("v_codes", FAKE + 8, _lib.TT_ERR_INVALID_ARGUMENT), ("lengths", None, _lib.TT_ERR_INVALID_ARGUMENT),
    ("block_table", FAKE + 2, _lib.TT_ERR_INVALID_ARGUMENT)])
def test_every_entry_refuses_a_bad_cache(lib, field, value, code):
    c = _cache(**{field: value})
    assert _write(lib, c) == code
    assert "tt_kv_write" in _lib.last_error(lib)
    assert lib.tt_kv_read(ctypes.byref(c), 0, FAKE, FAKE, 1, None) == code
    assert _attend(lib, c) == code
    assert lib.tt_kv_attention_workspace_bytes(ctypes.byref(c), 1, 2) == 0


def test_refused_arguments(lib):
    bad = _lib.TT_ERR_INVALID_ARGUMENT
    c = _cache()
    assert _write(lib, None) == bad
    assert _write(lib, c, dtype=3) == bad
    assert _write(lib, c, k=None) == bad
    assert _write(lib, c, ks=False) == bad
    assert _write(lib, c, tokens=-1) == bad
    assert _write(lib, c, tokens=1 << 31) == bad
    assert _write(lib, c, tokens=257) == bad  # 4 pages of 64
    assert lib.tt_kv_read(ctypes.byref(c), 0, None, FAKE, 1, None) == bad
    assert lib.tt_kv_read(ctypes.byref(c), 0, FAKE + 8, FAKE, 1, None) == bad
    assert lib.tt_kv_read(ctypes.byref(c), 7, FAKE, FAKE, 1, None) == bad
    assert lib.tt_kv_read(ctypes.byref(c), 0, FAKE, FAKE, -1, None) == bad
    assert _attend(lib, c, heads=3) == bad
    assert _attend(lib, c, heads=0) == bad
    assert _attend(lib, c, q=None) == bad
    assert _attend(lib, c, out=FAKE) == bad  # aliases q
    assert _attend(lib, c, out=2 * FAKE + 4) == bad
    assert _attend(lib, c, dtype=-1) == bad
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert _attend(lib, c, scale=scale) == bad
    assert lib.tt_kv_read_status(ctypes.byref(c), None, None, None) == bad
    # nothing to do
    assert _write(lib, c, tokens=0) == 0
    assert _write(lib, _cache(batch=0)) == 0
    assert _attend(lib, c, tokens=0) == 0
    assert lib.tt_kv_read(ctypes.byref(c), 0, None, None, 0, None) == 0


def test_cache_needs_cuda():
    with pytest.raises(RuntimeError, match="CUDA only"):
        KVCache(1, 16, 1, 16, device="cpu")
    k = torch.zeros(1, 2, 1, 16, 16, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA only"):
        KVCache.from_tensors(k, k, torch.zeros(1, 2, 1), torch.zeros(1, 2, 1),
                             torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


# ---- the oracle ------------------------------------------------------------


def test_oracle_codes_are_the_types():
    bits = torch.arange(256, dtype=torch.uint8)
    assert torch.equal(ref.code_values("int8"), bits.view(torch.int8).double())
    assert torch.equal(ref.code_values("e4m3").nan_to_num(999.0),
                       bits.view(torch.float8_e4m3fn).double().nan_to_num(999.0))


def test_oracle_rounding_is_the_nearest_code():
    x = torch.cat([torch.linspace(-448, 448, 20001, dtype=torch.float64),
                   torch.linspace(-0.02, 0.02, 4001, dtype=torch.float64)])
    assert torch.equal(ref.nearest(x, "e4m3"), x.float().to(torch.float8_e4m3fn).double())
    values = ref.code_values("e4m3")
    values = values[values.isfinite()].unique()
    nearest = (x[:, None] - values[None]).abs().amin(1)
    assert torch.equal((x - ref.nearest(x, "e4m3")).abs(), nearest)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_write_then_read_is_within_half_a_step(fmt):
    """Written in one piece, each value is within half a step of its code: e4m3
    2^-4 of the value (or 2^-10 of the scale), int8 half the scale."""
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(2, 20, 3, 16, generator=g).double(), torch.randn(2, 20, 3, 16, generator=g).double()
    cache = {"fmt": fmt, "page": 16, "table": [[3, 1], [0, 2]], "lengths": [20, 20]}
    for name in ("k", "v"):
        cache[name] = torch.zeros(4, 3, 16, 16, dtype=torch.float64)
        cache[name + "_scale"] = torch.zeros(4, 3, dtype=torch.float64)
    ref.write(cache, k, v, [20, 20])
    for name, x in (("k", k), ("v", v)):
        for b in range(2):
            got, there = ref.read(cache, name, b)
            assert bool(there.all())
            s = torch.stack([cache[name + "_scale"][cache["table"][b][t // 16]] for t in range(20)])[..., None]
            half = torch.maximum(x[b].abs() * 2.0 ** -4, s * 2.0 ** -10) if fmt == "e4m3" else s / 2
            assert bool(((got - x[b]).abs() <= half).all())


def test_oracle_appending_grows_a_scale():
    cache = {"fmt": "int8", "page": 16, "table": [[0]], "lengths": [1]}
    for name in ("k", "v"):
        cache[name] = torch.zeros(1, 1, 16, 16, dtype=torch.float64)
        cache[name + "_scale"] = torch.zeros(1, 1, dtype=torch.float64)
    x = torch.full((1, 1, 1, 16), 1.0)
    x[..., 0] = 127.0
    ref.write(cache, x, x, [1])
    assert float(cache["k_scale"][0, 0]) == 1.0
    cache["lengths"] = [2]
    ref.write(cache, x * 4, x * 4, [1])
    assert float(cache["k_scale"][0, 0]) == 4.0
    assert cache["k"][0, 0, 0, :2].tolist() == [32.0, 0.0]  # 127 / 4, and 1 / 4 to the even 0
    assert cache["k"][0, 0, 1, :2].tolist() == [127.0, 1.0]


def test_oracle_attention_is_softmax_over_the_seen_tokens():
    g = torch.Generator().manual_seed(2)
    cache = {"fmt": "int8", "page": 16, "table": [[1, 0]], "lengths": [20]}
    for name in ("k", "v"):
        cache[name] = torch.randint(-127, 128, (2, 2, 16, 16), generator=g).double()
        cache[name + "_scale"] = torch.tensor([[0.5, 1.0], [2.0, 0.25]], dtype=torch.float64) / 64
    q = torch.randn(1, 3, 4, 16, generator=g)
    out, _, _, _ = ref.attend(cache, q, [2], 0.25)
    k, v = (ref.read(cache, n, 0)[0].transpose(0, 1) for n in ("k", "v"))
    want = torch.nn.functional.scaled_dot_product_attention(
        q[0, :2].double().transpose(0, 1), k.repeat_interleave(2, 0), v.repeat_interleave(2, 0),
        attn_mask=torch.arange(20)[None] <= torch.tensor([[18], [19]]), scale=0.25)
    assert torch.allclose(out[0, :2].transpose(0, 1), want, rtol=0, atol=1e-12)
    assert not out[0, 2].any()


def test_sizes_beyond_32_bit_positions_are_refused(lib):
    """Positions, and rows padded to a tile, stay in 32 bits."""
    unsupported = _lib.TT_ERR_UNSUPPORTED
    for columns, page in ((1 << 24, 128), ((1 << 23) + 1, 128), ((1 << 26) + 1, 16)):
        c = _cache(table_columns=columns, page_size=page)
        assert _write(lib, c) == unsupported and _attend(lib, c) == unsupported
        assert lib.tt_kv_read(ctypes.byref(c), 0, FAKE, FAKE, 1, None) == unsupported
    c = _cache(num_pages=(1 << 30) + 1)
    assert _write(lib, c) == unsupported and _attend(lib, c) == unsupported
    c = _cache()
    assert lib.tt_kv_read(ctypes.byref(c), 0, FAKE, FAKE, (1 << 30) + 1, None) == _lib.TT_ERR_INVALID_ARGUMENT
    assert _attend(lib, c, tokens=(1 << 30) + 1) == unsupported
    assert _attend(lib, c, tokens=(1 << 29) + 1, heads=4) == unsupported
    assert lib.tt_kv_attention_workspace_bytes(ctypes.byref(c), (1 << 30) + 1, 2) == 0
