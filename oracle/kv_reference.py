"""The 8-bit key/value cache restated in 64 bits on the CPU, one token at a time
where that is the plainest form. Test infrastructure only.

A cache here is a dict: fmt ("e4m3" or "int8"), page, k and v (values of the
codes, [pages, heads, page, head_dim] float64), k_scale and v_scale ([pages,
heads] float64), table (list of lists) and lengths (list)."""
import math

import torch

MOST = {"e4m3": 448.0, "int8": 127.0}
LEAST_EXPONENT = -64
MOST_EXPONENT = 63


def code_values(fmt):
    """The 256 values of a code, by its bits."""
    out = []
    for code in range(256):
        if fmt == "int8":
            out.append(float(code - 256 if code > 127 else code))
            continue
        e, m = code >> 3 & 15, code & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if code & 127 == 127:
            x = math.nan
        out.append(-x if code > 127 else x)
    return torch.tensor(out, dtype=torch.float64)


def scale_of(x, fmt):
    """The scale of a set of values (float64 tensor); NaN when one is not
    finite or beyond the range."""
    if not bool(torch.isfinite(x).all()):
        return math.nan
    most = float(x.abs().max()) if x.numel() else 0.0
    e = LEAST_EXPONENT
    while most > MOST[fmt] * 2.0 ** e:
        e += 1
        if e > MOST_EXPONENT:
            return math.nan
    return 2.0 ** e


def nearest(x, fmt):
    """x (float64) to the nearest code's value, ties to the even code."""
    if fmt == "int8":
        return torch.round(x)
    a = x.abs()
    e = torch.floor(torch.log2(torch.clamp(a, min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def write(cache, k, v, counts):
    """k, v [batch, tokens, heads, head_dim] into the cache, in place. Tokens of
    pages outside the pool are dropped."""
    page, fmt = cache["page"], cache["fmt"]
    for name, x in (("k", k.double()), ("v", v.double())):
        pool, scales = cache[name], cache[name + "_scale"]
        for b, length in enumerate(cache["lengths"]):
            start = length - counts[b]
            for col in range(start // page, -(-length // page)):
                lo, hi = max(start, col * page), min(length, (col + 1) * page)
                pg, slot = cache["table"][b][col], lo - col * page
                if lo >= hi or not 0 <= pg < pool.shape[0]:
                    continue
                for h in range(pool.shape[1]):
                    new = x[b, lo - start:hi - start, h]
                    scale, old = scale_of(new, fmt), float(scales[pg, h])
                    if slot and (math.isnan(scale) or math.isnan(old)):
                        scale = math.nan
                    elif slot:
                        scale = max(scale, old)
                    if math.isnan(scale):
                        pool[pg, h, slot:slot + hi - lo] = 0.0
                    else:
                        if slot:
                            pool[pg, h, :slot] = nearest(pool[pg, h, :slot] * old / scale, fmt)
                        pool[pg, h, slot:slot + hi - lo] = nearest(new / scale, fmt)
                    scales[pg, h] = scale


def read(cache, name, b):
    """Sequence b's keys or values, [length, heads, head_dim] float64, and
    whether each token's page exists."""
    page, pool, scales = cache["page"], cache[name], cache[name + "_scale"]
    length = cache["lengths"][b]
    out = torch.zeros((length, pool.shape[1], pool.shape[3]), dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for t in range(length):
        pg = cache["table"][b][t // page]
        if 0 <= pg < pool.shape[0]:
            out[t] = pool[pg, :, t % page] * scales[pg][:, None]
            there[t] = True
    return out, there


def attend(cache, q, counts, scale):
    """(out, size, total, reach): out [batch, tokens, heads, head_dim] float64;
    size = sum_j p_j |v_j| and total = sum_j |v_j| per element, and reach =
    max_j scale * sum_d (|q_d| + max|q| / 8) |k_jd| per (batch, token, head), which
    bounds of rounding errors go by."""
    batch, n, heads, hd = q.shape
    q = q.double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    size, total = torch.zeros_like(out), torch.zeros_like(out)
    reach = torch.zeros(q.shape[:3], dtype=torch.float64)
    group = heads // cache["k"].shape[1]
    for b in range(batch):
        k, there = read(cache, "k", b)
        v, _ = read(cache, "v", b)
        for i in range(counts[b]):
            end = cache["lengths"][b] - counts[b] + i + 1
            seen = there[:end]
            if not bool(seen.any()):
                continue
            for h in range(heads):
                kk, vv = k[:end, h // group][seen], v[:end, h // group][seen]
                p = torch.softmax(scale * (kk @ q[b, i, h]), 0)
                out[b, i, h] = p @ vv
                size[b, i, h] = p @ vv.abs()
                total[b, i, h] = vv.abs().sum(0)
                qq = q[b, i, h].abs()
                reach[b, i, h] = scale * float((kk.abs() @ (qq + qq.max() / 8)).max())
    return out, size, total, reach
