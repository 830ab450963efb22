"""The 8-bit key/value cache on the GPU against its restatement in 64 bits
(oracle/kv_reference.py). Codes and scales are exact by construction (powers of
two, one rounding), so they are compared bit for bit; attention within a bound
that counts its roundings (kv_helpers.attention_bound)."""
import pytest
import torch

import kv_helpers as kh
from oracle import kv_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _counts(counts):
    return torch.tensor(counts, dtype=torch.int32, device="cuda")


def _check_write(cache, want, before, touched):
    for name in ("k", "v"):
        assert torch.equal(getattr(cache, name + "_scale")[0].double().cpu().nan_to_num(-1.0),
                           want[name + "_scale"].nan_to_num(-1.0)), name
        got = kh.values(getattr(cache, name)[0], cache.fmt)
        live = touched[:, None, :, None].expand_as(got)
        assert torch.equal(got[live], want[name][live]), name
        # every other slot keeps its bits
        kept = getattr(cache, name)[0].view(torch.uint8).cpu()
        assert torch.equal(kept[~live], before[name][~live]), name


def _live_slots(mirror):
    """[pages, page] of the slots that hold a sequence's tokens."""
    live = torch.zeros(mirror["k"].shape[0], mirror["page"], dtype=torch.bool)
    for b, length in enumerate(mirror["lengths"]):
        for t in range(length):
            pg = mirror["table"][b][t // mirror["page"]]
            if 0 <= pg < live.shape[0]:
                live[pg, t % mirror["page"]] = True
    return live


WRITES = [  # batch, tokens, heads, head_dim, page, lengths, counts
    (1, 1, 1, 16, 16, [1], None),
    (3, 1, 4, 32, 64, [1, 64, 65], None),
    (4, 1, 2, 64, 16, [5, 16, 17, 100], [1, 0, 1, 1]),
    (2, 40, 3, 48, 32, [40, 71], None),
    (3, 37, 5, 80, 16, [50, 37, 90], [37, 0, 20]),
    (2, 130, 2, 64, 64, [130, 191], [130, 127]),
    (2, 200, 1, 256, 128, [200, 255], None),
    (1, 65, 2, 128, 64, [65], None),
    (2, 300, 2, 96, 128, [300, 383], [300, 1]),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write_matches_64_bits(case, dtype, fmt):
    batch, n, heads, hd, page, lengths, counts = WRITES[case]
    cache, want = kh.make(case, fmt, batch, -(-max(lengths) // page) + 1, heads, hd, page, lengths)
    before = {name: getattr(cache, name)[0].view(torch.uint8).cpu() for name in ("k", "v")}
    g = torch.Generator().manual_seed(100 + case)
    x = torch.randn((batch, n, 3, heads, hd), generator=g)
    x *= torch.exp(torch.randn((batch, n, 1, heads, 1), generator=g))  # some pages' scales grow
    x = x.to(DTYPES[dtype]).cuda()
    k, v = x[:, :, 1], x[:, :, 2]  # slices of a fused projection
    cache.write(k, v, new_tokens=None if counts is None else _counts(counts))
    ref.write(want, k.cpu(), v.cpu(), counts or [n] * batch)
    _check_write(cache, want, before, _live_slots(want))
    assert cache.read_device_status() == (0, 0)
    # the same call again finds the scales it needs: nothing moves
    kept = cache.k.view(torch.uint8).clone()
    cache.write(k, v, new_tokens=None if counts is None else _counts(counts))
    assert torch.equal(kept, cache.k.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_one_by_one_and_other_strides(fmt):
    """Token after token, each of another size, over page borders; unaligned
    and transposed inputs."""
    cache, want = kh.make(7, fmt, 2, 3, 3, 32, 16, [0, 3])
    g = torch.Generator().manual_seed(8)
    for step in range(40):
        for b in range(2):
            want["lengths"][b] += 1
        cache.lengths.add_(1)
        raw = torch.randn((2, 3, 33, 2), generator=g) * 2.0 ** float(torch.randn((), generator=g) * 3)
        raw = raw.cuda()
        k = raw[:, :, 1:, 0].unsqueeze(1)          # head_dim not contiguous: copied
        v = raw.permute(0, 3, 1, 2).contiguous()[:, 1:, :, 1:]  # rows of 33 floats: unaligned
        cache.write(k, v)
        ref.write(want, k.cpu(), v.cpu(), [1, 1])
    live = _live_slots(want)
    for name in ("k", "v"):
        got = kh.values(getattr(cache, name)[0], fmt)
        assert torch.equal(got[live[:, None, :, None].expand_as(got)],
                           want[name][live[:, None, :, None].expand_as(got)])
        assert torch.equal(getattr(cache, name + "_scale")[0].double().cpu(), want[name + "_scale"])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_edges_of_the_scale(fmt):
    """Zeros, the largest value of a code and the next one up, tiny and huge
    magnitudes, ties, NaN and infinities; a new page forgets a NaN."""
    top = ref.MOST[fmt]
    rows = [0.0, top, float(torch.nextafter(torch.tensor(top), torch.tensor(1e9))), top * 2.0 ** 63,
            top * 2.0 ** 64, 2.0 ** -80, 2.0 ** -149, float("nan"), float("inf"), -float("inf"), 1.0]
    cache, want = kh.make(9, fmt, len(rows), 2, 1, 16, 16, [16] * len(rows))
    before = {name: getattr(cache, name)[0].view(torch.uint8).cpu() for name in ("k", "v")}
    x = torch.zeros(len(rows), 16, 1, 16)
    x[:, 3, 0, 5] = torch.tensor(rows)
    x[:, 4, 0, :] = torch.arange(16) * 0.0625 + 0.03125  # ties of either format
    k, v = x.cuda(), (-x).cuda()
    cache.write(k, v)
    ref.write(want, x, -x, [16] * len(rows))
    _check_write(cache, want, before, _live_slots(want))
    # appended to: a NaN page stays NaN; started anew, it is forgotten
    for length in (17, 32):
        cache.lengths.fill_(length)
        want["lengths"] = [length] * len(rows)
        n = length - 16
        y = torch.ones(len(rows), n, 1, 16)
        y[1, n - 1] = float("nan")
        cache.write(y.cuda(), y.cuda())
        ref.write(want, y, y, [n] * len(rows))
        for name in ("k_scale", "v_scale"):
            assert torch.equal(getattr(cache, name)[0].double().cpu().nan_to_num(-1.0),
                               want[name].nan_to_num(-1.0))
    k, _ = cache.read()
    assert torch.isnan(k[1, 16:]).all() and torch.isnan(k[7, :16]).all() and not torch.isnan(k[7, 16:]).any()
    cache.lengths.fill_(16)
    cache.write(torch.ones_like(x).cuda(), torch.ones_like(x).cuda())
    assert torch.equal(cache.read(max_tokens=16)[0].cpu(), torch.ones_like(x))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(1, 1, 1, 16, 16, [1]), (3, 3, 5, 48, 32, [0, 33, 96]),
                                   (2, 2, 2, 256, 128, [129, 256]), (5, 4, 3, 80, 16, [7, 16, 48, 0, 64])])
def test_read_matches_64_bits(shape, dtype, fmt):
    batch, columns, heads, hd, page, lengths = shape
    cache, want = kh.make(20, fmt, batch, columns, heads, hd, page, lengths)
    for most in (None, 1, page + 3):
        k, v = cache.read(DTYPES[dtype], max_tokens=most)
        most = columns * page if most is None else most
        assert k.shape == v.shape == (batch, most, heads, hd)
        for b, length in enumerate(lengths):
            n = min(length, most)
            for name, got in (("k", k), ("v", v)):
                exact = ref.read(want, name, b)[0][:n]
                # code * scale is exact in fp32; the one rounding is to `dtype`
                assert torch.equal(got[b, :n].cpu(), exact.float().to(DTYPES[dtype]))
                assert not got[b, n:].any()


ATTENDS = [  # batch, tokens, heads, kv_heads, head_dim, page, lengths, counts
    (1, 1, 1, 1, 16, 16, [1], None),
    (1, 1, 4, 4, 32, 64, [128], None),
    (4, 1, 4, 2, 64, 64, [1, 63, 64, 700], None),
    (3, 1, 8, 1, 128, 16, [33, 1000, 0], [1, 1, 0]),
    (2, 1, 12, 4, 80, 32, [513, 40], None),
    (2, 3, 2, 2, 256, 128, [300, 3], None),
    (3, 5, 6, 3, 48, 16, [5, 47, 200], [5, 0, 2]),
    (2, 37, 2, 2, 64, 64, [150, 37], [30, 37]),
    (1, 9, 16, 1, 96, 32, [222], None),
    (2, 70, 3, 1, 32, 16, [70, 131], None),
    (2, 130, 4, 2, 64, 64, [400, 130], [130, 7]),
    (2, 200, 2, 2, 128, 16, [200, 333], None),
    (1, 129, 3, 1, 16, 128, [640], None),
    (1, 300, 2, 1, 256, 64, [300], None),
    (2, 90, 3, 3, 80, 32, [900, 90], None),
    (1, 140, 1, 1, 64, 64, [2000], None),
    (1, 100, 2, 2, 128, 16, [1500], None),
    (3, 300, 1, 1, 48, 32, [300, 0, 1111], [40, 0, 300]),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attend_matches_64_bits(case, dtype, fmt):
    batch, n, heads, kv_heads, hd, page, lengths, counts = ATTENDS[case]
    cache, want = kh.make(40 + case, fmt, batch, -(-max(lengths) // page) + 1, kv_heads, hd, page, lengths)
    g = torch.Generator().manual_seed(case)
    q = torch.randn((batch, n, heads + 1, hd), generator=g).to(DTYPES[dtype]).cuda()[:, :, 1:]
    out = torch.full((batch, n, heads, hd), 7.0, dtype=q.dtype, device="cuda")
    got = cache.attend(q, new_tokens=None if counts is None else _counts(counts), out=out)
    assert got is out
    counts = counts or [n] * batch
    exact, size, total, reach = ref.attend(want, q.cpu(), counts, hd ** -0.5)
    bound, half_step = kh.attention_bound(size, total, reach, hd, max(lengths), q.dtype)
    assert not torch.isnan(got).any() and kh.worst(got, exact, bound, half_step) <= 1
    for b in range(batch):
        assert not got[b, counts[b]:].any()
    assert cache.read_device_status() == (0, 0)
    # again, with the output new: the same bits
    assert kh.same_bits(cache.attend(q, new_tokens=_counts(counts)), got)


@pytest.mark.parametrize("tokens", [1, 4, 150])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attend_bad_pages_nan_pages_and_own_scale(fmt, tokens):
    """Pages that do not exist are unseen; a NaN scale reaches the rows that
    see its page and no other; rows whose every page is missing are 0."""
    lengths = [tokens + 60, tokens + 200, 10 + tokens, tokens + 64]
    cache, want = kh.make(60, fmt, 4, 24, 2, 64, 16, lengths)
    cache.block_table[1, 3] = -1
    cache.block_table[1, 5] = cache.num_pages
    cache.block_table[2] = 1 << 30
    page = int(cache.block_table[3, 4])  # tokens 64 .. 79 of sequence 3: its new ones
    cache.v_scale[0, page, 1] = float("nan")
    want = kh.mirror(cache)
    g = torch.Generator().manual_seed(3)
    q = torch.randn((4, tokens, 4, 64), generator=g).cuda()
    got = cache.attend(q, scale=0.3).cpu().double()
    exact, size, total, reach = ref.attend(want, q.cpu(), [tokens] * 4, 0.3)
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    assert torch.isnan(got[3, :, 2:]).all() and not torch.isnan(got[3, :, :2]).any()
    assert not got[2].any()
    bound, half_step = kh.attention_bound(size, total, reach, 64, max(lengths), torch.float32)
    assert kh.worst(got, exact, bound, half_step) <= 1
    assert cache.read_device_status()[0] != 0  # the entries were latched
    assert cache.read_device_status() == (0, 0)
    k, _ = cache.read(max_tokens=80)
    assert not k[1, 48:64].any() and not k[1, 80:96].any() and k[1, 64:80].any()


@pytest.mark.parametrize("tokens", [20, 150])
def test_attend_nan_pages_reach_only_the_rows_that_see_them(tokens):
    """A page of the new tokens themselves: the rows before it stay numbers."""
    cache, _ = kh.make(65, "int8", 2, 16, 1, 32, 16, [tokens, tokens + 40])
    for b, name in ((0, "v_scale"), (1, "k_scale")):
        getattr(cache, name)[0, int(cache.block_table[b, (tokens + 40 * b - 1) // 16])] = float("nan")
    want = kh.mirror(cache)
    q = torch.randn((2, tokens, 1, 32), generator=torch.Generator().manual_seed(2)).cuda()
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [tokens] * 2, 32 ** -0.5)
    assert torch.isnan(exact).any() and not torch.isnan(exact).all(-1).all()
    assert torch.equal(torch.isnan(got).cpu(), torch.isnan(exact))
    bound, half_step = kh.attention_bound(size, total, reach, 32, tokens + 40, torch.float32)
    assert kh.worst(got, exact, bound, half_step) <= 1


def test_attend_large_scores_and_far_apart_value_scales():
    """Scores of hundreds, and pages whose values differ by 2^40."""
    lengths = [300]
    cache, _ = kh.make(70, "e4m3", 1, 20, 1, 64, 16, lengths)
    cache.k_scale.mul_(8.0)
    cache.v_scale[0, int(cache.block_table[0, 2])] *= 2.0 ** 40
    cache.v_scale[0, int(cache.block_table[0, 3])] *= 2.0 ** -50
    want = kh.mirror(cache)
    q = torch.randn((1, 2, 3, 64), generator=torch.Generator().manual_seed(1)).cuda() * 0.5
    q[0, 1] = 0
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [2], 64 ** -0.5)
    bound, half_step = kh.attention_bound(size, total, reach, 64, 300, torch.float32)
    assert not torch.isnan(got).any() and kh.worst(got, exact, bound, half_step) <= 1


@pytest.mark.parametrize("tokens,heads,hd", [(1, 2, 64), (2, 2, 128), (64, 2, 64), (70, 1, 128), (66, 1, 256), (3, 1, 256)])
def test_attend_long_contexts_do_not_drift(tokens, heads, hd):
    """20000 tokens: fp32 rows stay within 2^-19 of the output in the 2-norm: the
    runs of 1024 tokens lose 128 * 2^-24 / 2 = 2^-18 of themselves at most, all of one
    sign, and their partial sums are about half of that on average."""
    length = 20000
    cache, want = kh.make(77, "e4m3", 1, 160, heads, hd, 128, [length])
    q = torch.randn((1, tokens, heads, hd), generator=torch.Generator().manual_seed(6)).cuda()
    got = cache.attend(q)
    k, v = (x[0, :length].double().transpose(0, 1) for x in cache.read())
    s = hd ** -0.5 * q[0].double().transpose(0, 1) @ k.transpose(1, 2)
    end = torch.arange(length - tokens, length, device="cuda")[:, None]
    s.masked_fill_(torch.arange(length, device="cuda") > end, float("-inf"))
    exact = (torch.softmax(s, -1) @ v).transpose(0, 1)[None]
    assert float((got.double() - exact).norm() / exact.norm()) <= 2.0 ** -19
    assert cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("tokens", [1, 3, 70])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attend_unaligned_and_expanded_queries(dtype, tokens):
    """Rows that start anywhere, and one query for a whole batch (stride 0)."""
    cache, want = kh.make(71, "int8", 3, 8, 2, 48, 32, [200, 90, 133])
    raw = torch.randn((tokens, 5, 49), generator=torch.Generator().manual_seed(9)).to(DTYPES[dtype]).cuda()
    q = raw[:, 1:, 1:].expand(3, tokens, 4, 48)
    got = cache.attend(q)
    exact, size, total, reach = ref.attend(want, q.cpu(), [tokens] * 3, 48 ** -0.5)
    bound, half_step = kh.attention_bound(size, total, reach, 48, 200, q.dtype)
    assert not torch.isnan(got).any() and kh.worst(got, exact, bound, half_step) <= 1
    assert kh.same_bits(cache.attend(q.contiguous()), got)


@pytest.mark.parametrize("tokens,heads,hd", [(1, 2, 64), (3, 2, 128), (70, 2, 64), (130, 1, 128), (60, 1, 256)])
def test_attend_moving_references_give_the_same_bits_every_time(tokens, heads, hd):
    """Scores that grow along the sequence, so that the running reference moves
    and sums are rescaled all the way: right, and the same bits in 20 calls."""
    length = 1100
    cache, _ = kh.make(72, "int8", 2, 20, heads, hd, 64, [length, 700])
    order = torch.arange(20).float()
    for b in range(2):
        cache.k_scale[0, cache.block_table[b].long()] = torch.exp2(torch.floor(order / 3) - 6)[:, None].cuda()
    want = kh.mirror(cache)
    q = torch.randn((2, tokens, heads, hd), generator=torch.Generator().manual_seed(3)).cuda()
    got = cache.attend(q)
    for _ in range(19):
        assert kh.same_bits(cache.attend(q), got)
    exact, size, total, reach = ref.attend(want, q[:, -1:].cpu(), [1, 1], hd ** -0.5)
    bound, half_step = kh.attention_bound(size, total, reach, hd, length, torch.float32)
    assert kh.worst(got[:, -1:], exact, bound, half_step) <= 1
    assert cache.read_device_status() == (0, 0)


@pytest.mark.parametrize("tokens,hd", [(1, 64), (4, 32), (4, 128), (70, 64), (70, 128), (70, 256)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_attend_infinite_queries_give_nan(dtype, tokens, hd):
    """All scores of a row with an infinity are infinite or NaN, and its softmax
    is NaN, also where every one of them is minus infinity (the keys' first
    element is negative throughout). Other rows, and rows that see no token, do
    not know of it."""
    cache, _ = kh.make(76, "int8", 3, 3, 1, hd, 64, [150, tokens, tokens])
    cache.k[:, :, :, :, 0] = -5
    cache.block_table[2, :] = -1
    q = torch.randn((3, tokens, 1, hd), generator=torch.Generator().manual_seed(6)).to(DTYPES[dtype]).cuda()
    want = cache.attend(q)
    q[:, tokens - 1, 0, 0] = float("inf")
    got = cache.attend(q)
    assert torch.isnan(got[:2, -1]).all() and not got[2].any()
    assert kh.same_bits(got[:, :-1], want[:, :-1]) and not torch.isnan(want).any()
    q[:, tokens - 1, 0, 0] = float("nan")
    got = cache.attend(q)
    assert torch.isnan(got[:2, -1]).all() and not got[2].any()


def test_two_graphs_at_once():
    """Two captured calls, each with a workspace of its own, replayed on two
    streams at the same time. 100 new tokens are more than the sequence of 64
    holds: that is latched as a count beyond the length (0x5200), and the rows
    are the same in every call all the same."""
    work = []
    for seed, tokens in ((1, 1), (2, 100)):
        cache, _ = kh.make(73 + seed, "e4m3", 4, 40, 2, 64, 64, [2500, 1800, 64, 900])
        q = torch.randn((4, tokens, 2, 64), generator=torch.Generator().manual_seed(seed)).cuda()
        want = cache.attend(q)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            out = cache.attend(q)
        work.append((cache, stream, graph, out, want))
    torch.cuda.synchronize()
    for _ in range(10):
        for _, stream, graph, _, _ in work:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (cache, _, _, out, want), status in zip(work, ((0, 0), (-7, 0x5200))):
        assert kh.same_bits(out, want)
        assert cache.read_device_status() == status


def test_shared_pages_and_padded_width_beyond_the_room():
    """Two sequences over the same pages, read only; and a batch padded to more
    rows than a sequence has room for."""
    cache, _ = kh.make(75, "e4m3", 2, 2, 1, 32, 16, [32, 20])
    own = cache.block_table[1].clone()
    cache.block_table[1] = cache.block_table[0]
    want = kh.mirror(cache)
    q = torch.randn((2, 40, 3, 32), generator=torch.Generator().manual_seed(4)).cuda()
    counts = [2, 1]
    got = cache.attend(q, new_tokens=_counts(counts))
    exact, size, total, reach = ref.attend(want, q.cpu(), counts, 32 ** -0.5)
    bound, half_step = kh.attention_bound(size, total, reach, 32, 32, torch.float32)
    assert kh.worst(got, exact, bound, half_step) <= 1 and not got[0, 2:].any() and not got[1, 1:].any()
    x = torch.ones((2, 40, 1, 32), device="cuda")
    cache.block_table[1] = own
    cache.write(x, x, new_tokens=_counts(counts))
    k, _ = cache.read()
    assert torch.equal(k[0, 30:], x[0, :2]) and torch.equal(k[1, 19:20], x[0, :1])
    assert cache.read_device_status() == (0, 0)


def test_device_checks_of_lengths_and_counts():
    """A length beyond the room or below zero and a count beyond the length
    are latched and clamped; nothing outside the cache's pages is touched."""
    for name, bad in (("lengths", [1000, 5]), ("lengths", [-3, 5]), ("counts", [9, 2]), ("counts", [-1, 2])):
        cache, _ = kh.make(80, "int8", 2, 2, 1, 16, 16, [20, 5], spare=4)
        spare = [p for p in range(cache.num_pages) if p not in cache.block_table.flatten().tolist()]
        kept = cache.k[0, spare].clone()
        counts = _counts(bad) if name == "counts" else None
        if name == "lengths":
            cache.lengths.copy_(_counts(bad))
        x = torch.ones((2, 2, 1, 16), device="cuda")
        for call in (lambda: cache.write(x, x, new_tokens=counts), lambda: cache.attend(x, new_tokens=counts),
                     lambda: cache.read() if name == "lengths" else cache.attend(x, new_tokens=counts)):
            call()
            assert cache.read_device_status()[0] == -7
        assert torch.equal(cache.k[0, spare], kept)


def test_streams_and_graph_replay():
    """The three calls captured into one graph and replayed on new inputs, and
    on a stream of their own."""
    cache, _ = kh.make(90, "e4m3", 3, 8, 2, 64, 32, [100, 3, 200], layers=2)
    other, _ = kh.make(90, "e4m3", 3, 8, 2, 64, 32, [100, 3, 200], layers=2)
    g = torch.Generator().manual_seed(5)
    inputs = [torch.randn((3, 2, 8, 64), generator=g).cuda() for _ in range(4)]
    x = inputs[0].clone()

    def step(c, x):
        c.advance(2)
        outs = []
        for layer in range(2):
            c.write(x[:, :, 4:6], x[:, :, 6:8], layer=layer)
            outs.append(c.attend(x[:, :, :4], layer=layer))
        return outs + list(c.read(layer=1))

    want = [[t.clone() for t in step(other, i)] for i in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(cache, x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = step(cache, x)
    side.synchronize()
    assert all(kh.same_bits(a, b) for a, b in zip(first, want[0]))
    for i in (1, 2, 3):
        x.copy_(inputs[i])
        graph.replay()
        assert all(kh.same_bits(a, b) for a, b in zip(outs, want[i])), i


def test_lengths_advance_and_refusals():
    from ttjam_gottagofast_b200 import KVCache

    cache = KVCache(2, 40, 2, 32, page_size=16, fmt="int8")
    assert cache.block_table.shape == (2, 3) and cache.max_tokens == 40
    cache.advance(30)
    cache.advance(8, new_tokens=_counts([1, 8]))
    assert cache.lengths.tolist() == [31, 38]
    cache.advance(2, new_tokens=_counts([2, 0]))
    with pytest.raises(ValueError, match="full"):
        cache.advance(3)
    assert cache.lengths.tolist() == [33, 38]
    cache.reset()
    cache.advance(40)
    x = torch.ones((2, 4, 2, 32), device="cuda")
    for bad, error in (
            (lambda: cache.write(x.cpu(), x.cpu()), RuntimeError),
            (lambda: cache.write(x.double(), x.double()), ValueError),
            (lambda: cache.write(x, x.half()), ValueError),
            (lambda: cache.write(x[:1], x[:1]), ValueError),
            (lambda: cache.write(x[:, :, :1], x[:, :, :1]), ValueError),
            (lambda: cache.write(x, x[:, :2]), ValueError),
            (lambda: cache.write(x, x, layer=1), ValueError),
            (lambda: cache.write(x, x, new_tokens=torch.ones(2, device="cuda")), ValueError),
            (lambda: cache.write(x.repeat(1, 13, 1, 1), x.repeat(1, 13, 1, 1)), ValueError),
            (lambda: cache.read(torch.float64), ValueError),
            (lambda: cache.read(max_tokens=-1), ValueError),
            (lambda: cache.attend(x[:, :, :1]), ValueError),
            (lambda: cache.attend(x[..., :16]), ValueError),
            (lambda: cache.attend(x, scale=0.0), ValueError),
            (lambda: cache.attend(x, scale=float("nan")), ValueError),
            (lambda: cache.attend(x, out=x.half()), ValueError),
            (lambda: cache.attend(x, out=x), ValueError),
            (lambda: cache.attend(x.int()), ValueError),
            (lambda: KVCache(2, 40, 2, 24), ValueError),
            (lambda: KVCache(2, 40, 2, 272), ValueError),
            (lambda: KVCache(2, 40, 2, 32, page_size=48), ValueError),
            (lambda: KVCache(2, 40, 2, 32, fmt="int4"), ValueError),
            (lambda: KVCache(0, 40, 2, 32), ValueError),
            (lambda: KVCache(2, 40, 2, 32, device="cpu"), RuntimeError),
            (lambda: KVCache.from_tensors(cache.k, cache.v, cache.k_scale, cache.v_scale[:, :2],
                                          cache.block_table, cache.lengths), ValueError),
            (lambda: KVCache.from_tensors(cache.k, cache.v, cache.k_scale, cache.v_scale,
                                          cache.block_table.long(), cache.lengths), ValueError)):
        with pytest.raises(error):
            bad()
    # nothing to do is not an error
    assert cache.attend(x[:, :0]).shape == (2, 0, 2, 32)
    cache.write(x[:, :0], x[:, :0])
    assert cache.read(max_tokens=0)[0].shape == (2, 0, 2, 32)


def test_advance_knows_of_lengths_that_others_wrote():
    """The caller's own writes into lengths, a graph's replays, and caches made
    or used in inference mode: what has no room is still refused."""
    from ttjam_gottagofast_b200 import KVCache

    cache = KVCache(2, 64, 1, 16, page_size=16)
    cache.advance(4)
    cache.lengths.copy_(_counts([60, 1]))
    with pytest.raises(ValueError, match="full"):
        cache.advance(5)
    cache.reset()
    cache.advance(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.advance(10)
    for _ in range(6):
        graph.replay()
    with pytest.raises(ValueError, match="full"):
        cache.advance(4)
    cache.advance(3)
    graph.replay()
    assert cache.lengths.tolist() == [74, 74]
    with pytest.raises(ValueError, match="full"):
        cache.advance(0)
    with torch.inference_mode():
        for make in (lambda: KVCache(2, 64, 1, 16, page_size=16),
                     lambda: KVCache.from_tensors(*_empty(2, 4, 1, 16, 16))):
            cache = make()
            cache.advance(60)
            cache.lengths.add_(2)
            with pytest.raises(ValueError, match="full"):
                cache.advance(3)
            cache.advance(2)
            assert cache.lengths.tolist() == [64, 64]


def _empty(batch, columns, heads, hd, page):
    pages = batch * columns
    codes = [torch.zeros((1, pages, heads, page, hd), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((1, pages, heads), device="cuda") for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(batch, columns)
    return [*codes, *scales, table, torch.zeros(batch, dtype=torch.int32, device="cuda")]


def test_a_batch_of_none():
    from ttjam_gottagofast_b200 import KVCache

    k, v, ks, vs, table, lengths = _empty(1, 2, 1, 16, 16)
    cache = KVCache.from_tensors(k, v, ks, vs, table[:0], lengths[:0])
    x = torch.ones((0, 3, 1, 16), device="cuda")
    cache.advance(3)
    cache.write(x, x)
    assert cache.attend(x).shape == x.shape and cache.read()[0].shape == (0, 32, 1, 16)
    assert cache.read_device_status() == (0, 0)
