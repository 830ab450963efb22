"""The 8-bit key/value cache of the causal Transformer: writing new tokens' keys
and values into it, reading them back, and attention over it.

The cache is a pool of pages of `page` tokens, [1, pages, kv_heads, page,
head_dim] in 8 bits (float8_e4m3fn or int8), with one fp32 scale, a power of
two, for each page and head of the keys and of the values. A sequence's tokens
lie in the pages that its row of the block table lists; `lengths` counts them,
the new ones included, so new token i of a sequence with `count` new tokens
stands at position length - count + i.
"""
import torch

own = False

MOST = {"e4m3": 448.0, "int8": 127.0}  # largest value of a code
LEAST_EXPONENT = -64                   # of a scale; that of a page of zeros
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of each of 64 sequences, 16 heads of 64: a decoding batch's write
        {"name": "write step", "op": "write", "fmt": "e4m3", "type": "bf16", "batch": 64, "tokens": 1,
         "context": 2048, "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": True},
        # the prompts of 16 sequences at once
        {"name": "write prompts", "op": "write", "fmt": "e4m3", "type": "bf16", "batch": 16, "tokens": 2048,
         "context": 2048, "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": False},
        # pieces of prompts of unlike lengths, appended in the middle of pages
        {"name": "write pieces", "op": "write", "fmt": "int8", "type": "fp32", "batch": 7, "tokens": 517,
         "context": 1900, "kv_heads": 5, "head_dim": 96, "page": 32, "ragged": True},
        # one long sequence read back, for a program that goes on with it elsewhere
        {"name": "read long", "op": "read", "fmt": "e4m3", "type": "bf16", "batch": 1, "context": 100000,
         "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": False},
        # a few short ones with small pages
        {"name": "read short", "op": "read", "fmt": "int8", "type": "fp32", "batch": 5, "context": 777,
         "kv_heads": 3, "head_dim": 48, "page": 16, "ragged": True},
        # a single sequence's next token, 4 heads of 32: latency
        {"name": "step small", "op": "attend", "fmt": "e4m3", "type": "fp32", "batch": 1, "tokens": 1,
         "context": 128, "heads": 4, "kv_heads": 4, "head_dim": 32, "page": 64, "ragged": False},
        # a decoding batch of 64 sequences of up to 2048 tokens, 16 heads of 64
        {"name": "step batch", "op": "attend", "fmt": "e4m3", "type": "fp32", "batch": 64, "tokens": 1,
         "context": 2048, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": True},
        # two sequences of 100000 tokens: few rows, the work lies along the keys
        {"name": "step long", "op": "attend", "fmt": "int8", "type": "bf16", "batch": 2, "tokens": 1,
         "context": 100000, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 128, "ragged": False},
        # a decoding batch whose eight query heads share a key head of 128
        {"name": "step grouped", "op": "attend", "fmt": "e4m3", "type": "fp16", "batch": 32, "tokens": 1,
         "context": 8192, "heads": 32, "kv_heads": 4, "head_dim": 128, "page": 16, "ragged": True},
        # a few dozen new tokens a sequence (a proposal to check, a short turn), odd lengths
        {"name": "chunk", "op": "attend", "fmt": "int8", "type": "fp32", "batch": 3, "tokens": 37,
         "context": 1501, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": True},
        # prompts of 2048 tokens behind as many in the cache, in the model's own type
        {"name": "prompt", "op": "attend", "fmt": "e4m3", "type": "fp32", "batch": 4, "tokens": 2048,
         "context": 4096, "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 64, "ragged": False},
        # long prompts of unlike lengths, eight query heads on a key head of 128
        {"name": "prompt grouped", "op": "attend", "fmt": "e4m3", "type": "bf16", "batch": 3, "tokens": 4096,
         "context": 8192, "heads": 32, "kv_heads": 4, "head_dim": 128, "page": 64, "ragged": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    case = {"op": rng.choice(["write", "read", "attend", "attend", "attend"]), "fmt": rng.choice(["e4m3", "int8"]),
            "type": rng.choice(["fp32", "fp16", "bf16"])}
    case["kv_heads"] = _log(rng, 1, 16)
    case["head_dim"] = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, 256])
    case["page"] = rng.choice([16, 32, 64, 128])
    case["ragged"] = rng.random() < 0.6
    width = case["kv_heads"] * case["head_dim"]
    if case["op"] == "attend":
        case["heads"] = case["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 8])
        few = rng.random() < 0.6
        case["tokens"] = _log(rng, 1, 16) if few else _log(rng, 16, 3000)
        before = _log(rng, 1, 100000 if few else 6000)
        work = lambda: case["tokens"] * (case["tokens"] + before) * case["heads"] * case["head_dim"]
        while work() > 10**11:  # at most the largest listed case's
            case["tokens"] = case["tokens"] * 2 // 3
        case["context"] = case["tokens"] + before
        case["batch"] = _log(rng, 1, max(1, min(64, 10**11 // work(), 4 * 10**8 // (case["context"] * width))))
    else:
        case["context"] = _log(rng, 1, 50000)
        case["batch"] = _log(rng, 1, max(1, min(64, 10**8 // (case["context"] * width))))
        if case["op"] == "write":
            case["tokens"] = _log(rng, 1, case["context"])
    return case


def _lengths(case):
    """(lengths, counts of new tokens), the same for every seed: the work hangs on them."""
    n, most = case.get("tokens", 0), case["context"]
    if not case["ragged"]:
        return [most] * case["batch"], [n] * case["batch"]
    counts, lengths = [], []
    for b in range(case["batch"]):
        counts.append(min(n, 1 + int((n - 1) * ((b + 1) * 0.7548776662 % 1.0) + 0.5)))
        lengths.append(max(1, counts[-1] + int((most - n) * ((b + 1) * 0.6180339887 % 1.0))))
    return lengths, counts


def work(case):
    lengths, counts = _lengths(case)
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["type"]]
    width = case["kv_heads"] * case["head_dim"]
    if case["op"] == "write":
        return {"bytes": 2 * sum(counts) * width * (size + 1), "flops": 0}
    if case["op"] == "read":
        return {"bytes": 2 * sum(lengths) * width + 2 * len(lengths) * case["context"] * width * size, "flops": 0}
    pairs = sum(c * l - c * (c - 1) // 2 for l, c in zip(lengths, counts))
    rows = len(lengths) * case["tokens"] + sum(counts)
    return {"bytes": 2 * sum(lengths) * width + rows * case["heads"] * case["head_dim"] * size,
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}


def _scale(most, fmt):
    """The smallest power of two (2^-64 at least) that brings values of up to `most` into the code's range."""
    f, e = torch.frexp(most)
    top_f, top_e = (0.875, 9) if fmt == "e4m3" else (0.9921875, 7)  # 448 and 127 as f * 2^e
    e = e - top_e + (f > top_f)
    return torch.ldexp(torch.ones_like(most), torch.where(most > 0, e, LEAST_EXPONENT).clamp(min=LEAST_EXPONENT))


def _codes(x, fmt):
    """Rounded to the nearest code, ties to even; |x| is within the code's range."""
    return x.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(x).to(torch.int8)


def _keys(shape, gen, channels):
    """Values as keys and values have them: of a size of each head's own, with a few large channels."""
    x = torch.randn(shape, generator=gen, device="cuda")
    size = torch.exp(0.3 * torch.randn(shape[-3], generator=gen, device="cuda"))[:, None, None]
    x *= size
    if channels:
        x[..., :: max(1, shape[-1] // 3)] *= 2.5
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, page, heads, hd = TYPES[case["type"]], case["page"], case["kv_heads"], case["head_dim"]
    lengths, counts = _lengths(case)
    batch, columns = case["batch"], -(-case["context"] // page)
    pages = batch * columns + 3
    table = torch.randperm(pages, generator=gen, device="cuda")[: batch * columns].to(torch.int32).view(batch, columns)
    state = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "counts": torch.tensor(counts, dtype=torch.int32, device="cuda") if case["ragged"] else None}
    for name in ("k", "v"):
        x = _keys((pages, heads, page, hd), gen, name == "k")
        scale = _scale(x.abs().amax((2, 3)), case["fmt"])
        state[name] = _codes(x / scale[:, :, None, None], case["fmt"])[None]
        state[name + "_scale"] = scale[None]
        del x
    n = case.get("tokens", 0)
    if case["op"] == "write":
        # k and v as a fused projection leaves them: slices of one [batch, tokens, 3 * heads * head_dim]
        x = _keys((batch, n, 3, heads, hd), gen, True) if n else None
        x = x * torch.exp(0.4 * torch.randn((batch, n, 1, 1, 1), generator=gen, device="cuda"))
        x = x.to(kind)
        state["new_k"], state["new_v"] = x[:, :, 1], x[:, :, 2]
    elif case["op"] == "attend":
        q = 1.5 * torch.randn((batch, n, case["heads"] + 2 * heads, hd), generator=gen, device="cuda")
        state["q"] = q.to(kind)[:, :, : case["heads"]]
    if own:  # the handle that a program keeps for its cache
        from ttjam_gottagofast_b200 import KVCache

        state["cache"] = KVCache.from_tensors(state["k"], state["v"], state["k_scale"], state["v_scale"], table, state["lengths"])
    return state


def _write(state, name):
    """The new tokens of state["new_" + name] into the pool, in place."""
    case, pool, scales = state["case"], state[name][0], state[name + "_scale"][0]
    page, n, batch = case["page"], case["tokens"], case["batch"]
    table, lengths = state["table"].long(), state["lengths"].long()
    counts = torch.full_like(lengths, n) if state["counts"] is None else state["counts"].long()
    start = lengths - counts
    first = start // page
    slots = ((n + page - 1) // page + 1) * page  # tokens of the pages that a sequence's new ones can touch
    at = first[:, None] * page + torch.arange(slots, device="cuda")
    i = at - start[:, None]
    new, old = (i >= 0) & (i < counts[:, None]), i < 0
    x = state["new_" + name].float()
    x = torch.gather(x, 1, i.clamp(0, n - 1)[:, :, None, None].expand(-1, -1, *x.shape[2:]))
    x = torch.where(new[:, :, None, None], x, 0.0)
    x = x.view(batch, slots // page, page, *x.shape[2:]).transpose(2, 3)  # [batch, page of it, heads, page, head_dim]
    new, old = (m.view(batch, slots // page, page) for m in (new, old))
    touched = new.any(2)
    column = (first[:, None] + torch.arange(slots // page, device="cuda")).clamp(max=table.shape[1] - 1)
    where = torch.gather(table, 1, column)[touched]
    x, new, old = x[touched], new[touched][:, None, :, None], old[touched][:, None, :, None]
    before, its_scale = pool[where], scales[where]
    scale = _scale(x.abs().amax((2, 3)), case["fmt"])
    scale = torch.where(old.flatten(1).any(1)[:, None], torch.maximum(scale, its_scale), scale)
    moved = _codes(before.float() * (its_scale / scale)[:, :, None, None], case["fmt"])
    codes = _codes(x / scale[:, :, None, None], case["fmt"])
    kept = torch.where(old, moved.view(torch.uint8), before.view(torch.uint8))
    pool.view(torch.uint8)[where] = torch.where(new, codes.view(torch.uint8), kept)
    scales[where] = scale


def _read(state, name, most):
    """[batch, heads, tokens, head_dim] in fp32, zero behind each sequence's end."""
    pool, scales, table = state[name][0], state[name + "_scale"][0], state["table"].long()
    x = pool.view(torch.uint8)[table].view(pool.dtype).float() * scales[table][..., None, None]
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :most]
    there = torch.arange(most, device="cuda") < state["lengths"][:, None]
    return torch.where(there[:, None, :, None], x, 0.0)


def _attend(state):
    case, q = state["case"], state["q"].float()
    batch, n, heads, hd = q.shape
    most = state["table"].shape[1] * case["page"]
    k, v = _read(state, "k", most), _read(state, "v", most)
    group = heads // case["kv_heads"]
    counts = torch.full_like(state["lengths"], n) if state["counts"] is None else state["counts"]
    i = torch.arange(n, device="cuda")
    end = torch.where(i < counts[:, None], (state["lengths"] - counts)[:, None] + i + 1, 0)  # keys that row i sees
    hidden = torch.arange(most, device="cuda") >= end[:, :, None]
    q = q.view(batch, n, -1, group, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, kv_heads, group * n, head_dim]
    s = q @ k.transpose(2, 3)
    s *= hd ** -0.5
    s = s.view(batch, -1, group, n, most).masked_fill_(hidden[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, 3) @ v).view(batch, -1, group, n, hd) / torch.where(total > 0, total, 1.0)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(TYPES[case["type"]])


def run(state):
    case = state["case"]
    op, kind, most = case["op"], TYPES[case["type"]], case["context"]
    if op == "write":
        if own:
            state["cache"].write(state["new_k"], state["new_v"], new_tokens=state["counts"])
        else:
            _write(state, "k")
            _write(state, "v")
        return {name: state[name] for name in ("k", "v", "k_scale", "v_scale")}
    if op == "read":
        if own:
            k, v = state["cache"].read(kind, max_tokens=most)
        else:
            k, v = (_read(state, name, most).transpose(1, 2).to(kind).contiguous() for name in ("k", "v"))
        return {"k": k, "v": v}
    if own:
        return state["cache"].attend(state["q"], new_tokens=state["counts"])
    return _attend(state)


# ---- the definition in 64 bits ----------------------------------------------


def _value_table(fmt):
    """The value of each of the 256 codes, from the bits."""
    values = []
    for code in range(256):
        if fmt == "int8":
            values.append(float(code - 256 if code > 127 else code))
            continue
        exponent, mantissa = code >> 3 & 15, code & 7
        x = mantissa * 2.0 ** -9 if exponent == 0 else (8 + mantissa) * 2.0 ** (exponent - 10)
        x = float("nan") if code & 127 == 127 else x
        values.append(-x if code > 127 else x)
    return torch.tensor(values, dtype=torch.float64, device="cuda")


def _nearest(x, fmt):
    """x to the nearest value of a code, ties to the even one."""
    if fmt == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step


def _exact_write(state):
    case, out = state["case"], {}
    page, fmt = case["page"], case["fmt"]
    lengths, counts = _lengths(case)
    values, table = _value_table(fmt), state["table"].tolist()
    powers = torch.exp2(torch.arange(LEAST_EXPONENT, 64, dtype=torch.float64, device="cuda"))
    for name in ("k", "v"):
        pool = values[state[name][0].view(torch.uint8).long()]
        scales = state[name + "_scale"][0].double()
        for b, (length, count) in enumerate(zip(lengths, counts)):
            start = length - count
            for column in range(start // page, -(-length // page)):
                low, high = max(start, column * page), min(length, (column + 1) * page)
                x = state["new_" + name][b, low - start : high - start].double().transpose(0, 1)
                where, slot = table[b][column], low - column * page
                fits = x.abs().amax((1, 2))[:, None] <= MOST[fmt] * powers
                scale = powers[fits.int().argmax(1)]
                if slot:
                    scale = torch.maximum(scale, scales[where])
                    pool[where, :, :slot] = _nearest(pool[where, :, :slot] * (scales[where] / scale)[:, None, None], fmt)
                pool[where, :, slot : slot + high - low] = _nearest(x / scale[:, None, None], fmt)
                scales[where] = scale
        # int8 codes are whole numbers, which have to be equal to the plain form's anyway
        out[name], out[name + "_scale"] = pool[None] if fmt == "e4m3" else None, scales[None]
    return out


def _exact_tokens(state, name, b, length):
    case, where = state["case"], state["table"][b].long()
    x = _value_table(case["fmt"])[state[name][0].view(torch.uint8)[where].long()]
    x = x * state[name + "_scale"][0][where].double()[:, :, None, None]
    return x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["head_dim"])[:, :length]


def exact(case, seed):
    state = prepare(case, seed)
    lengths, counts = _lengths(case)
    heads, hd, most = case["kv_heads"], case["head_dim"], case["context"]
    if case["op"] == "write":
        return _exact_write(state)
    if case["op"] == "read":
        out = {}
        for name in ("k", "v"):
            out[name] = torch.zeros((case["batch"], most, heads, hd), dtype=torch.float64, device="cuda")
            for b, length in enumerate(lengths):
                out[name][b, :length] = _exact_tokens(state, name, b, length).transpose(0, 1)
        return out
    group, n = case["heads"] // heads, case["tokens"]
    out = torch.zeros((case["batch"], n, case["heads"], hd), dtype=torch.float64, device="cuda")
    for b, (length, count) in enumerate(zip(lengths, counts)):
        k, v = _exact_tokens(state, "k", b, length), _exact_tokens(state, "v", b, length)
        sees = torch.arange(length, device="cuda")[None] <= length - count + torch.arange(count, device="cuda")[:, None]
        for h in range(case["heads"]):
            s = state["q"][b, :count, h].double() @ k[h // group].T / hd ** 0.5
            out[b, :count, h] = torch.softmax(s.masked_fill(~sees, float("-inf")), -1) @ v[h // group]
    return out
