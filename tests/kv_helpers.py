"""Caches for the tests of the 8-bit key/value cache: random pages on the GPU, and
the same contents as the oracle holds them."""
import torch

from oracle import kv_reference as ref

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def values(codes, fmt):
    return ref.code_values(fmt)[codes.cpu().view(torch.uint8).long()]


def make(seed, fmt, batch, columns, heads, hd, page, lengths, layers=1, spare=2, spread=1.0):
    """(KVCache over random pages in random order, the oracle's cache of layer
    0). Slots behind a sequence's end hold any bit pattern."""
    from ttjam_gottagofast_b200 import KVCache

    g = torch.Generator().manual_seed(seed)
    pages = batch * columns + spare
    table = torch.randperm(pages, generator=g)[:batch * columns].view(batch, columns).to(torch.int32)
    pools, scales = [], []
    for _ in range(2):
        codes = torch.randint(0, 256, (layers, pages, heads, page, hd), generator=g, dtype=torch.uint8)
        filled = codes.clone()
        if fmt == "int8":
            filled[filled == 128] = 0
        else:
            filled[(filled & 127) == 127] = 0
        for b, length in enumerate(lengths):
            for col in range(columns):
                used = min(page, max(0, length - col * page))
                pg = int(table[b, col])
                codes[:, pg, :, :used] = filled[:, pg, :, :used]
        # values of about 1: 448 * 2^-8 (e4m3 codes spread over many binades), 127 * 2^-6
        e = torch.randint(-1, 2, (layers, pages, heads), generator=g).float() * spread
        scales.append(torch.exp2(e + (-8 if fmt == "e4m3" else -6)))
        pools.append(codes.view(CODES[fmt]))
    cache = KVCache.from_tensors(*(p.cuda() for p in pools), *(s.cuda() for s in scales),
                                 table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    return cache, mirror(cache)


def mirror(cache, layer=0):
    return {"fmt": cache.fmt, "page": cache.page_size, "k": values(cache.k[layer], cache.fmt),
            "v": values(cache.v[layer], cache.fmt), "k_scale": cache.k_scale[layer].double().cpu(),
            "v_scale": cache.v_scale[layer].double().cpu(), "table": cache.block_table.tolist(),
            "lengths": cache.lengths.tolist()}


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def attention_bound(size, total, reach, hd, tokens, dtype):
    """How far an element may be from the 64-bit value, by counting roundings.

    A score's products are exact (11-bit pieces of q times a code); q's split
    loses 2^-22 of each, or 2^-25 of the row's largest element where that is more
    (an fp16 piece has no step below 2^-24; reach counts 2^-25 of it), and each of the hd / 16 additions of a tensor-core step
    at most 2^-22 of the sum of magnitudes: (hd / 16 + 2) 2^-22 reach. The
    exponent's fused multiply-add rounds a number of up to 2^5 where p matters
    (2^-19 of p after ln 2), exp2 and p's split add less than 2^-21 together.
    The sum of p v takes two additions for 16 tokens, each losing up to 2^-23 of the
    sum, in runs of at most 1024 tokens, and one of 2^-24 for each run; the sum of p
    one of 2^-24 for 16 tokens. Each relative error of p_j counts once in the sum of
    p v and once in the sum of p. 16-bit rows may round p to fp16 for its product
    with v (not in the sum): float16's steps are 2^-10 of a power of two, so half
    a step is at most eps / 2 = 2^-11 of p, once.

    p's pieces have no step below 2^-24 either, and p is scaled to have its largest
    value at 2^6 at least: each p_j is off by up to 2^-31 of the largest, whatever
    its own size, which is 2^-31 of `total` in the sum of p v.

    The output's own rounding adds half a step of its type: eps / 2 of the value,
    and below the type's smallest normal number, where the steps stay as they are
    there, half of smallest_normal * eps (float16: 2^-14 2^-10 / 2 = 2^-25)."""
    sums = min(tokens, 1024) / 8 * 2.0 ** -23 + (tokens / 1024 + tokens / 16 + 8) * 2.0 ** -24
    eps = (hd / 16 + 2) * 2.0 ** -22 * reach + 2.0 ** -18 + sums / 2
    info = torch.finfo(dtype)
    once = 2.0 ** -11 if info.bits == 16 else 0.0
    return (2 * eps[..., None] + once) * size + 2.0 ** -31 * total + info.smallest_normal * info.eps / 2, info.eps / 2


def worst(got, exact, bound, half_step):
    """The largest share of its bound that an element is off; at most 1 is right."""
    off = (got.double().cpu() - exact).abs()
    return float((off / (bound + half_step * (exact.abs() + bound))).nan_to_num(0.0).max())
