"""The model token by token over the 8-bit key/value cache: write, attention and
the forward's other kernels in one run. Each step is recomputed in 64 bits from
the step's input and the codes that the cache holds after it, layer by layer, so
the 8-bit rounding itself does not blur the comparison; the codes are held to
the keys and values they stand for.

Tolerance of y (a LayerNorm's output, of size 1): the schedules compute each
product to 2^-22 of its operands' sizes and sum at most 1024 of them (2^-24
each): below 6e-5 of a row for each of the up to four chained products of a
layer, 5e-4 for two layers."""
import pytest
import torch

import kv_helpers as kh
from oracle import kv_reference as ref
from oracle import reference_model as oracle
from ttjam_gottagofast_b200 import UserOptimizedTransformer
from ttjam_gottagofast_b200.config import TransformerConfig

pytestmark = pytest.mark.gpu
Y_TOL = 5e-4


def _model(d, heads, f, layers, dtype=torch.float32, seed=11, causal=True):
    cfg = TransformerConfig(2, 64, d, heads, f, layers, causal)
    params = oracle.init_params(cfg, seed=seed)
    model = UserOptimizedTransformer(cfg).cuda().eval()
    model.load_state_dict(params, strict=True)
    model = model.to(dtype)
    return cfg, {k: v.to(dtype).double() for k, v in params.items()}, model


def _check_codes(cache, layer, name, want, counts):
    """The new tokens' codes against the values they stand for: half a step of
    the code for the rounding, half of one more where the page was moved to a
    larger scale, and the tolerance of what was rounded."""
    m = kh.mirror(cache, layer)
    for b, count in enumerate(counts):
        got, _ = ref.read(m, name, b)
        start = m["lengths"][b] - count
        for i in range(count):
            s = m[name + "_scale"][m["table"][b][(start + i) // m["page"]]][:, None]
            x = want[b, i]
            half = torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10) if cache.fmt == "e4m3" else s / 2
            assert bool(((got[start + i] - x).abs() <= 2.1 * half + Y_TOL).all())


def _step64(p, cfg, cache, x, counts):
    """y of new tokens x (float64) given the cache after their step."""
    b, n, d = x.shape
    h = cfg.num_heads
    live = torch.arange(n)[None] < torch.tensor(counts)[:, None]
    for i in range(cfg.num_layers):
        pre = f"layers.{i}."
        lin = lambda t, name: t @ p[pre + name + ".weight"].T + p[pre + name + ".bias"]  # noqa: E731
        t = oracle.layer_norm(x, p[pre + "norm1.weight"], p[pre + "norm1.bias"])
        q, k, v = (lin(t, f"attention.{c}_proj").view(b, n, h, d // h) for c in "qkv")
        _check_codes(cache, i, "k", k, counts)
        _check_codes(cache, i, "v", v, counts)
        ctx = ref.attend(kh.mirror(cache, i), q, counts, (d // h) ** -0.5)[0].view(b, n, d)
        x = x + lin(ctx, "attention.out_proj") * live[..., None]
        t = oracle.layer_norm(x, p[pre + "norm2.weight"], p[pre + "norm2.bias"])
        x = (x + lin(torch.nn.functional.gelu(lin(t, "ffn_in")), "ffn_out")) * live[..., None]
    return oracle.layer_norm(x, p["final_norm.weight"], p["final_norm.bias"]) * live[..., None]


STEPS = [(40, None), (1, None), (1, [1, 0]), (5, [2, 5]), (1, None)]


@pytest.mark.parametrize("plan", ["auto", "ops_ffma", "ops_tc"])
@pytest.mark.parametrize("shape", [(128, 4, 128, 2, 16, "e4m3"), (64, 4, 96, 2, 64, "int8"),
                                   (256, 2, 512, 1, 32, "int8"), (128, 8, 256, 2, 128, "e4m3")])
def test_prompt_and_steps(shape, plan):
    d, heads, f, layers, page, fmt = shape
    cfg, params, model = _model(d, heads, f, layers)
    model.set_plan(plan)
    cache = model.make_cache(2, 60, fmt=fmt, page_size=page)
    g = torch.Generator().manual_seed(d)
    with torch.inference_mode():
        for n, counts in STEPS:
            x = torch.randn((2, n, d), generator=g)
            y = model.forward_cached(x.cuda(), cache, None if counts is None else
                                     torch.tensor(counts, dtype=torch.int32, device="cuda"))
            counts = counts or [n, n]
            want = _step64(params, cfg, cache, x.double(), counts)
            assert float((y.double().cpu() - want).abs().max()) <= Y_TOL
            for b in range(2):
                assert not y[b, counts[b]:].any()
    assert cache.lengths.tolist() == [45, 47]
    assert cache.read_device_status() == (0, 0) and model.read_device_status() == (0, 0)


def test_long_prompt_in_pieces_and_wide_model():
    """Prompts that take the tile kernel and the row lists of padded batches."""
    cfg, params, model = _model(512, 8, 512, 1)
    cache = model.make_cache(2, 700, fmt="e4m3")
    g = torch.Generator().manual_seed(1)
    with torch.inference_mode():
        for n, counts in ((520, [520, 300]), (100, [7, 100]), (1, [1, 1])):
            x = torch.randn((2, n, 512), generator=g)
            y = model.forward_cached(x.cuda(), cache, torch.tensor(counts, dtype=torch.int32, device="cuda"))
            want = _step64(params, cfg, cache, x.double(), counts)
            assert float((y.double().cpu() - want).abs().max()) <= Y_TOL


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_models(dtype):
    cfg, params, model = _model(128, 4, 128, 2, dtype)
    cache = model.make_cache(2, 64)
    g = torch.Generator().manual_seed(2)
    with torch.inference_mode():
        for n in (33, 1):
            x = torch.randn((2, n, 128), generator=g).to(dtype)
            y = model.forward_cached(x.cuda(), cache)
            assert y.dtype == dtype
            want = _step64(params, cfg, cache, x.double(), [n, n])
            off = (y.double().cpu() - want).abs()
            assert bool((off <= Y_TOL + torch.finfo(dtype).eps / 2 * (want.abs() + Y_TOL)).all())


def test_graph_of_a_step_replayed():
    """One captured step, replayed for token after token, gives the bits of the
    calls made one by one."""
    _, _, model = _model(128, 4, 128, 2)
    caches = [model.make_cache(2, 200, page_size=16) for _ in range(2)]
    g = torch.Generator().manual_seed(4)
    prompt = torch.randn((2, 70, 128), generator=g).cuda()
    xs = [torch.randn((2, 1, 128), generator=g).cuda() for _ in range(40)]
    with torch.inference_mode():
        for c in caches:
            model.forward_cached(prompt, c)
        want = [model.forward_cached(x, caches[0]) for x in xs]
        model.forward_cached(xs[0], caches[1])
        static = xs[1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = model.forward_cached(static, caches[1])
        for x, w in zip(xs[1:], want[1:]):
            static.copy_(x)
            graph.replay()
            assert torch.equal(y, w)
    assert caches[0].lengths.tolist() == caches[1].lengths.tolist() == [110, 110]


def test_refusals():
    _, _, model = _model(128, 4, 128, 2)
    cache = model.make_cache(2, 32)
    x = torch.zeros((2, 3, 128), device="cuda")
    other = UserOptimizedTransformer(TransformerConfig(2, 64, 128, 4, 128, 2, False)).cuda()
    odd = UserOptimizedTransformer(TransformerConfig(2, 64, 96, 4, 96, 1, True)).cuda()
    for bad, error in ((lambda: model.forward_cached(x.cpu(), cache), RuntimeError),
                       (lambda: model.forward_cached(x.double(), cache), ValueError),
                       (lambda: model.forward_cached(x[:1], cache), ValueError),
                       (lambda: model.forward_cached(x[..., :64], cache), ValueError),
                       (lambda: model.forward_cached(x.repeat(1, 11, 1), cache), ValueError),
                       (lambda: model.forward_cached(x, cache, torch.ones(2, device="cuda")), ValueError),
                       (lambda: other.forward_cached(x, cache), ValueError),
                       (lambda: odd.make_cache(2, 32), ValueError),  # head_dim 24
                       (lambda: model.forward_cached(x, _model(128, 4, 128, 1)[2].make_cache(2, 32)), ValueError),
                       (lambda: model.forward_cached(x, _model(128, 8, 128, 2)[2].make_cache(2, 32)), ValueError)):
        with pytest.raises(error):
            bad()
    assert cache.lengths.tolist() == [0, 0]
    assert model.forward_cached(x[:, :0], cache).shape == (2, 0, 128)


def test_a_batch_padded_beyond_the_room_is_refused_before_it_counts():
    _, _, model = _model(64, 2, 64, 1)
    cache = model.make_cache(2, 32, page_size=16)
    x = torch.zeros((2, 33, 64), device="cuda")
    counts = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="room"):
        model.forward_cached(x, cache, new_tokens=counts)
    assert cache.lengths.tolist() == [0, 0]
    model.forward_cached(x[:, :32], cache, new_tokens=counts)
    assert cache.lengths.tolist() == [1, 2]
