"""Measured cases of the operators over an 8-bit paged K/V cache: appending with rotary positions,
reading back, and attention for single tokens and for ragged runs of tokens.

The cache (keys and values alike) is blocks of 16 tokens of one kv head:

    codes   u8 [pages, kv_heads, 16, head_dim]   E4M3 values
    scales  u8 [pages, kv_heads]                 E8M0 powers of two, one for each block
    value = e4m3(code) * 2^(scale - 127)

Appending: the new tokens of a sequence are the last ones of its `sequence_lengths`; a key is
rotated in f32 and rounded once, to 8 bits.  A block's exponent is the smallest e in [-48, 48] with
|x| <= 448 * 2^e for all its finite new rows, and not below the exponent it had when older tokens
stay in it (their codes are rounded again to the grown exponent).  A row that holds an infinity or
a NaN is stored as NaN throughout.

Attention: token j is visible to the query at position i when j <= i and (no window, or
j > i - window, or j < first_tokens); `sinks` adds exp(sink) to the denominator; a query that sees
nothing gives zeros.

`own` False: elementary torch operations in f32; True: the framework's operators.
"""
import math
import random

import torch

own = False

PAGE = 16
LOWEST, HIGHEST = -48, 48
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# The shape of the decode step's model: 64 query and 8 kv heads of 64, window 128, YaRN factor 32
# over 4096 original positions.
MODEL = {"dtype": "bf16", "heads": 64, "kv_heads": 8, "dim": 64}
OTHER = {"dtype": "f16", "heads": 32, "kv_heads": 8, "dim": 128}


def _append(name, shape, batch, padded, new, context, ragged, rotary, layout):
    return {"name": name, "op": "append", **shape, "batch": batch, "padded": padded,
            "new_low": new[0], "new_high": new[1], "context_low": context[0],
            "context_high": context[1], "ragged": ragged, "rotary": rotary, "layout": layout}


def _attend(name, shape, batch, padded, new, context, ragged, window, first, sinks):
    return {"name": name, "op": "attend", **shape, "batch": batch, "padded": padded,
            "new_low": new[0], "new_high": new[1], "context_low": context[0],
            "context_high": context[1], "ragged": ragged, "window": window, "first": first,
            "sinks": sinks}


def listed():
    return [
        # one user at the keyboard: a token written far behind the original context
        _append("append one token", MODEL, 1, 0, (1, 1), (90001, 90001), False, 64, "half"),
        # the decode step's batch, three of its places empty
        _append("append a decode batch", MODEL, 64, 3, (1, 1), (5, 4500), False, 64, "half"),
        # prompts of unlike lengths behind what is cached already; half of each head is rotated
        _append("append ragged prompts", OTHER, 7, 0, (0, 1300), (0, 900), True, 64,
                "interleaved"),
        # one prompt of 16384 tokens, the longest row count of the linear benchmark
        _append("append a long prompt", MODEL, 1, 0, (16384, 16384), (0, 0), True, 64, "half"),
        # a short conversation copied out, and a decode batch's whole cache
        {"name": "read one sequence", "op": "read", **MODEL, "batch": 1, "rows_low": 333,
         "rows_high": 333},
        {"name": "read a batch", "op": "read", **MODEL, "batch": 64, "rows_low": 3900,
         "rows_high": 4200},
        # decode: one short conversation, the decode step's batch on a full and on a window layer
        _attend("attend one sequence", MODEL, 1, 0, (1, 1), (412, 412), False, 0, 0, True),
        _attend("attend a decode batch", MODEL, 64, 0, (1, 1), (4096, 4096), False, 0, 0, True),
        _attend("attend in a window", MODEL, 64, 3, (1, 1), (100, 4500), False, 128, 4, True),
        # a few long documents, with wide heads
        _attend("attend long contexts", OTHER, 3, 0, (1, 1), (60000, 100000), False, 0, 0, False),
        # drafted tokens of a decode batch, checked in one pass
        _attend("attend drafted tokens", MODEL, 16, 0, (1, 6), (500, 3000), True, 0, 0, True),
        # prompts of unlike lengths, some behind a cached part
        _attend("attend ragged prompts", MODEL, 4, 0, (1200, 2000), (0, 2000), True, 0, 0, True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kv_heads = rng.choice([1, 2, 4, 8])
    shape = {"dtype": rng.choice(["bf16", "f16"]), "kv_heads": kv_heads,
             "heads": kv_heads * rng.choice([1, 2, 3, 4, 5, 8, 8, 16]),
             "dim": rng.choice([64, 64, 128])}
    op = rng.choice(["append", "read", "attend", "attend"])
    batch = _spread(rng, 1, 64)
    if op == "read":
        rows = _spread(rng, 1, 4200)
        return {"op": op, **shape, "batch": batch, "rows_low": rng.randint(0, rows),
                "rows_high": rows}
    ragged = rng.random() < 0.5
    padded = 0 if ragged else rng.randint(0, batch // 4)
    if op == "append":
        new = _spread(rng, 1, max(1, 16384 // batch)) if ragged else 1
        context = _spread(rng, 1, 100000)
        case = _append("", shape, batch, padded, (rng.randint(0, new) if ragged else 1, new),
                       (rng.randint(0, context), context), ragged,
                       rng.choice([0, 16, 32, 64, shape["dim"]]),
                       rng.choice(["half", "interleaved"]))
    else:
        # at most the listed prompts' pairs of rows and tokens, and the long documents' tokens
        new = _spread(rng, 1, 2000) if ragged else 1
        context = _spread(rng, 1, 100000)
        context = min(context, 300000 * 1024 // (batch * kv_heads * shape["dim"]))
        pairs = 4 * 64 * 2000 * 4000
        while batch * shape["heads"] * new * (new + context) > pairs:
            new, context = (new + 1) // 2, (context + 1) // 2
            batch = max(1, batch - 1)
        padded = min(padded, batch // 4)
        window = rng.choice([0, 0, 0, 1, 100, 128, 500])
        case = _attend("", shape, batch, padded, (rng.randint(0, new) if ragged else 1, new),
                       (rng.randint(0, context), context), ragged, window,
                       rng.choice([0, 1, 4, 20]) if window else 0, rng.random() < 0.5)
    del case["name"]
    return case


def _sizes(case):
    """Host-side (new tokens, length after them) of every sequence, from the case alone."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "read":
        rows = [rng.randint(case["rows_low"], case["rows_high"]) for _ in range(case["batch"])]
        rows[-1] = max(1, rows[-1])
        return rows, rows
    new = [rng.randint(case["new_low"], case["new_high"]) for _ in range(case["batch"])]
    new[-1] = max(1, new[-1])
    lengths = [n + rng.randint(case["context_low"], case["context_high"]) for n in new]
    for b in rng.sample(range(case["batch"]), case["padded"]):
        lengths[b] = 0
    return new, lengths


def _frequencies(rotary, device):
    """YaRN: factor 32 over 4096 original positions, base 150000, between 32 and 1 turns."""
    half = rotary // 2
    index = torch.arange(half, dtype=torch.float64, device=device)
    plain = 150000.0 ** (-index / half)
    low, high = (half * math.log(4096 / (turns * 2 * math.pi)) / math.log(150000.0)
                 for turns in (32.0, 1.0))
    ramp = ((index - low) / max(high - low, 1e-3)).clamp(0, 1)
    return plain * (1 - ramp) + plain / 32.0 * ramp


def _cache(gen, pages, kv_heads, dim, device):
    """Random written blocks: values of order one, a magnitude for each head."""
    sets = []
    for _ in range(2):
        spread = torch.exp2(torch.rand((1, kv_heads, 1, 1), generator=gen, device=device) * 4 - 2)
        x = torch.randn((pages, kv_heads, PAGE, dim), generator=gen, device=device) * spread
        mantissa, exponent = torch.frexp(x.abs().amax(dim=(2, 3)))
        e = (exponent - 8 - (mantissa <= 0.875).int()).clamp(LOWEST, HIGHEST)
        codes = (x * torch.exp2(-e.float())[:, :, None, None]).to(torch.float8_e4m3fn)
        sets += [codes.view(torch.uint8), (e + 127).to(torch.uint8)]
        del x
    return sets


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    order = torch.Generator().manual_seed(seed)
    new, lengths = _sizes(case)
    batch, kv_heads, heads, dim = case["batch"], case["kv_heads"], case["heads"], case["dim"]
    dtype, tokens = TYPES[case["dtype"]], sum(new)
    starts = [max(0, m - n) // PAGE if case["op"] == "append" else 0
              for n, m in zip(new, lengths)]
    counts = [max(0, -(-m // PAGE) - s) for m, s in zip(lengths, starts)]
    # every written page belongs to one sequence; what lies before the append's first page is one
    # shared page; the last page belongs to nobody
    pages = 2 + sum(counts)
    shuffled = (torch.randperm(pages - 2, generator=order) + 1).tolist()
    table = torch.zeros((batch, max(1, max(s + c for s, c in zip(starts, counts))) + 1),
                        dtype=torch.int32)
    at = 0
    for b in range(batch):
        table[b, starts[b]:starts[b] + counts[b]] = torch.tensor(
            shuffled[at:at + counts[b]], dtype=torch.int32)
        at += counts[b]
    offsets = torch.zeros(batch + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(new).cumsum(0)
    state = {"case": case, "longest": max(new), "tokens": tokens, "table": table.to(device),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=device),
             "offsets": offsets.to(device), "cache": _cache(gen, pages, kv_heads, dim, device)}
    # what no token was written to yet holds anything, NaN codes among it
    owner = torch.full((pages,), -1, dtype=torch.int64)
    for b in range(batch):
        if counts[b]:
            owner[table[b, starts[b] + counts[b] - 1].long()] = (lengths[b] - 1) % PAGE
    owner[-1] = -1
    stale = (torch.arange(PAGE)[None] > owner[:, None]) & (owner[:, None] >= 0)
    stale[-1] = True
    stale = stale.to(device)[:, None, :, None]
    for codes in (state["cache"][0], state["cache"][2]):
        junk = torch.randint(0, 256, (pages, kv_heads, PAGE, 1), generator=gen, device=device,
                             dtype=torch.uint8)
        codes.copy_(torch.where(stale, junk, codes))
    if case["op"] == "append":
        # the fused projection's output: the three parts are views of its rows
        qkv = torch.randn((tokens, heads + 2 * kv_heads, dim), generator=gen, device=device)
        qkv = (qkv * torch.exp2(torch.rand((heads + 2 * kv_heads, 1), generator=gen,
                                           device=device) * 4 - 2)).to(dtype)
        state["query"] = qkv[:, :heads]
        state["key"] = qkv[:, heads:heads + kv_heads]
        state["value"] = qkv[:, heads + kv_heads:]
        state["rotary"] = None
        if case["rotary"]:
            angle = torch.arange(max(lengths) + 1, dtype=torch.float64, device=device)[:, None] * \
                _frequencies(case["rotary"], device)
            factor = 0.1 * math.log(32.0) + 1.0
            state["rotary"] = torch.cat((angle.cos() * factor, angle.sin() * factor), 1).float()
    elif case["op"] == "attend":
        state["query"] = torch.randn((tokens, heads, dim), generator=gen, device=device).to(dtype)
        state["sinks"] = torch.randn(heads, generator=gen, device=device) if case["sinks"] \
            else None
    return state


# ---- plain forms -----------------------------------------------------------------------------

def _rows(state):
    """(sequence, position) of every new token's row."""
    token = torch.arange(state["tokens"], device=state["table"].device)
    sequence = torch.searchsorted(state["offsets"][1:].contiguous(), token, right=True)
    last = state["offsets"][sequence + 1].long()
    return sequence, state["lengths"][sequence].long() - last + token


def _rotate(x, table, position, layout):
    if table is None:
        return x
    row = table[position.clamp(min=0)][:, None]
    half = table.shape[1] // 2
    cos, sin = row[..., :half], row[..., half:]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if layout == "half":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, rest), -1)


def _to_codes(x, e):
    """E4M3 codes of x at exponent e; rows with an infinity or a NaN become NaN."""
    fine = torch.isfinite(x).all(-1, keepdim=True)
    scaled = (x * torch.exp2(-e.float())).clamp(-448.0, 448.0)
    return torch.where(fine, scaled, math.nan).to(torch.float8_e4m3fn).view(torch.uint8)


def _write(x, codes, scales, state, sequence, position, valid):
    """Quantises the rows x [tokens, kv_heads, dim] into their blocks, in place."""
    spare = codes.shape[0] - 1
    page = state["table"][sequence, position.clamp(min=0) // PAGE].long()
    page = torch.where(valid, page, spare)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    row = torch.where(fine & valid[:, None, None], x.abs(), 0.0).amax(-1)
    largest = torch.zeros(scales.shape, device=x.device)
    largest = largest.scatter_reduce(0, page[:, None].expand_as(row), row, "amax")
    mantissa, exponent = torch.frexp(largest)
    e = torch.where(largest > 0, exponent - 8 - (mantissa <= 0.875).int(), LOWEST)
    e = e.clamp(LOWEST, HIGHEST)
    # the block that a sequence's first new token shares with older ones
    new = state["offsets"][1:] - state["offsets"][:-1]
    start = (state["lengths"] - new).clamp(min=0).long()
    shares = (new > 0) & (state["lengths"] > 0) & (start % PAGE > 0)
    first = state["table"].gather(1, (start // PAGE)[:, None])[:, 0].long()
    first = torch.where(shares, first, spare)
    before = scales[first].int() - 127
    grown = torch.where(shares[:, None], torch.maximum(e[first], before), before)
    old = codes[first]
    again = _to_codes(old.view(torch.float8_e4m3fn).float() *
                      torch.exp2(before.float())[:, :, None, None], grown[:, :, None, None])
    stays = torch.arange(PAGE, device=x.device)[None] < (start % PAGE)[:, None]
    moved = (shares[:, None] & stays)[:, None, :, None] & (grown != before)[:, :, None, None]
    codes[first] = torch.where(moved, again, old)
    e[first] = grown
    codes[page, :, position % PAGE] = torch.where(
        valid[:, None, None], _to_codes(x, e[page][..., None]), codes[page, :, position % PAGE])
    scales[page] = torch.where(valid[:, None], (e[page] + 127).to(torch.uint8), scales[page])


def _plain_append(state):
    case, (key, key_scales, value, value_scales) = state["case"], state["cache"]
    sequence, position = _rows(state)
    valid = position >= 0
    layout = case["layout"]
    _write(_rotate(state["key"].float(), state["rotary"], position, layout), key, key_scales,
           state, sequence, position, valid)
    _write(state["value"].float(), value, value_scales, state, sequence, position, valid)
    query = _rotate(state["query"].float(), state["rotary"], position, layout)
    return torch.where(valid[:, None, None], query, 0.0).to(state["query"].dtype)


def _decoded(codes, scales, table):
    """f32 [batch, logical pages, kv_heads, 16, dim] of the pages of a table."""
    table = table.long()
    return codes[table].view(torch.float8_e4m3fn).float() * \
        torch.exp2(scales[table].float() - 127.0)[..., None, None]


def _plain_read(state):
    key, key_scales, value, value_scales = state["cache"]
    sequence, position = _rows(state)
    page = state["table"][sequence, position // PAGE].long()
    dtype = TYPES[state["case"]["dtype"]]

    def part(codes, scales):
        rows = codes[page, :, position % PAGE].view(torch.float8_e4m3fn).float()
        return (rows * torch.exp2(scales[page].float() - 127.0)[..., None]).to(dtype)

    return part(key, key_scales), part(value, value_scales)


def _plain_attend(state):
    case, query = state["case"], state["query"]
    batch, longest = case["batch"], state["longest"]
    kv_heads, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // kv_heads
    key, key_scales, value, value_scales = state["cache"]
    new = state["offsets"][1:] - state["offsets"][:-1]
    step = torch.arange(longest, device=query.device)
    row = (state["offsets"][:-1, None] + step).clamp(max=state["tokens"] - 1).long()
    q = query[row].float().view(batch, longest, kv_heads, group, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * longest, dim)
    k = _decoded(key, key_scales, state["table"]).transpose(1, 2).flatten(2, 3)
    v = _decoded(value, value_scales, state["table"]).transpose(1, 2).flatten(2, 3)
    token = torch.arange(k.shape[2], device=query.device)
    written = token[None] < state["lengths"][:, None]
    v = torch.where(written[:, None, :, None], v, 0.0)
    position = (state["lengths"] - new)[:, None] + step[None]
    seen = token <= position[..., None]
    if case["window"]:
        seen &= (token > position[..., None] - case["window"]) | (token < case["first"])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(dim ** -0.5)
    scores = scores.view(batch, kv_heads, group, longest, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    largest = scores.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, kv_heads, group, 1, 1)
        largest = torch.maximum(largest, sink)
    largest = torch.where(largest == -math.inf, 0.0, largest)
    weights = scores.sub_(largest).exp_()
    total = weights.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + torch.exp(sink - largest)
    out = torch.matmul(weights.view(batch, kv_heads, group * longest, -1), v)
    out = out.view(batch, kv_heads, group, longest, dim) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, longest, case["heads"], dim).to(query.dtype)
    sequence, _ = _rows(state)
    return out[sequence, torch.arange(state["tokens"], device=query.device) -
               state["offsets"][sequence].long()]


def _values(state):
    """The cache as the values it stands for: codes and block scales in their 8-bit types."""
    key, key_scales, value, value_scales = state["cache"]
    return {"key": key.view(torch.float8_e4m3fn), "value": value.view(torch.float8_e4m3fn),
            "key_scales": key_scales.view(torch.float8_e8m0fnu),
            "value_scales": value_scales.view(torch.float8_e8m0fnu)}


def run(state):
    case = state["case"]
    if own:
        from nml_b200 import ops
        offsets = state["offsets"] if case["op"] == "read" or case["ragged"] else None
    if case["op"] == "append":
        if own:
            query = ops.paged_append_q8(
                state["key"], state["value"], *state["cache"], state["table"], state["lengths"],
                token_offsets=offsets, query=state["query"], rotary=state["rotary"],
                rotary_layout=case["layout"])
        else:
            query = _plain_append(state)
        return {"query": query, **_values(state)}
    if case["op"] == "read":
        if own:
            key, value = ops.paged_read_q8(*state["cache"], state["table"], offsets,
                                           state["tokens"], TYPES[case["dtype"]])
        else:
            key, value = _plain_read(state)
        return {"key": key, "value": value}
    if own:
        return ops.paged_attention_q8(
            state["query"], *state["cache"], state["table"], state["lengths"],
            query_offsets=offsets, sinks=state["sinks"], sliding_window=case["window"] or None,
            first_tokens=case["first"])
    return _plain_attend(state)


def work(case):
    new, lengths = _sizes(case)
    kv_heads, heads, dim, tokens = case["kv_heads"], case["heads"], case["dim"], sum(new)
    if case["op"] == "read":
        # a code in and a 16-bit value out, keys and values
        blocks = sum(-(-n // PAGE) for n in new)
        return {"bytes": 2 * kv_heads * (tokens * dim * 3 + blocks), "flops": 0}
    if case["op"] == "append":
        # 16-bit query in and out, 16-bit keys and values in, codes out, two f32 for each pair
        live = sum(n for n, m in zip(new, lengths) if m)
        return {"bytes": live * (heads * dim * 4 + kv_heads * dim * 6 + 4 * case["rotary"]),
                "flops": live * (heads + kv_heads) * 3 * case["rotary"]}
    # every visible token's codes once for each sequence, 16-bit query in and out
    pairs = visible = 0
    for n, m in zip(new, lengths):
        if m == 0 or n == 0:
            continue
        window, first = case["window"], case["first"]
        for position in range(m - n, m):
            low = max(0, position + 1 - window) if window else 0
            pairs += position + 1 - low + min(first, low)
        low = max(0, m - n + 1 - window) if window else 0
        visible += m - low + min(first, low)
    return {"bytes": 2 * kv_heads * dim * visible + 4 * tokens * heads * dim,
            "flops": 4 * heads * dim * pairs}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _e4m3_64(x):
    """Nearest E4M3 value of f64 numbers, ties to even, largest 448."""
    _, exponent = torch.frexp(x.abs())
    step = torch.exp2((exponent.double() - 4).clamp(min=-9))
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(case, state):
    """Sequence by sequence, block by block."""
    new, lengths = _sizes(case)
    layout, out = case["layout"], {}
    dim = case["dim"]
    angles = None if state["rotary"] is None else state["rotary"].double()

    def turned(x, position):
        x = x.double()
        if angles is None:
            return x
        half = angles.shape[1] // 2
        cos, sin = (angles[position, i * half:(i + 1) * half].unsqueeze(1) for i in (0, 1))
        low = torch.arange(half, device=x.device) * (1 if layout == "half" else 2)
        high = low + (half if layout == "half" else 1)
        y = x.clone()
        y[..., low] = x[..., low] * cos - x[..., high] * sin
        y[..., high] = x[..., low] * sin + x[..., high] * cos
        return y

    query = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    for name, at in (("key", 0), ("value", 2)):
        codes = state["cache"][at].view(torch.float8_e4m3fn).double()
        exponents = state["cache"][at + 1].double() - 127
        row = 0
        for b, (n, m) in enumerate(zip(new, lengths)):
            begin, row = row, row + n
            if n == 0 or m == 0:
                continue
            position = torch.arange(m - n, m, device="cuda")
            x = state[name][begin:begin + n]
            if name == "key":
                x = turned(x, position)
                query[begin:begin + n] = turned(state["query"][begin:begin + n], position)
            x = x.double().transpose(0, 1)  # [kv_heads, n, dim]
            first_page, lead = (m - n) // PAGE, (m - n) % PAGE
            count = (m - 1) // PAGE - first_page + 1
            page = state["table"][b, first_page:first_page + count].long()
            block = torch.zeros((x.shape[0], count * PAGE, dim), dtype=torch.float64,
                                device="cuda")
            block[:, lead:lead + n] = x
            block = block.view(x.shape[0], count, PAGE, dim)
            largest = block.abs().amax((2, 3))
            e = torch.ceil(torch.log2(largest / 448).clamp(LOWEST, HIGHEST))
            e += (largest > 448 * torch.exp2(e)).double()  # log2 may fall on the wrong side
            e -= ((largest <= 448 * torch.exp2(e - 1)) & (e > LOWEST)).double()
            if lead:
                old = exponents[page[0]]
                e[:, 0] = torch.maximum(e[:, 0], old)
                held = codes[page[0], :, :lead] * torch.exp2(old - e[:, 0])[:, None, None]
                codes[page[0], :, :lead] = _e4m3_64(held)
            fresh = _e4m3_64(block / torch.exp2(e)[..., None, None])
            slot = torch.arange(count * PAGE, device="cuda").view(count, PAGE)
            written = (slot >= lead) & (slot < lead + n)
            codes[page] = torch.where(written[:, None, :, None], fresh.transpose(0, 1),
                                      codes[page])
            exponents[page] = e.transpose(0, 1)
        out[name], out[name + "_scales"] = codes, torch.exp2(exponents)
    return {"query": query, **out}


def _exact_read(case, state):
    new, _ = _sizes(case)

    def part(at):
        codes, scales = state["cache"][at], state["cache"][at + 1]
        rows = []
        for b, n in enumerate(new):
            page = state["table"][b, : -(-n // PAGE)].long()
            block = codes[page].view(torch.float8_e4m3fn).double() * \
                torch.exp2(scales[page].double() - 127)[:, :, None, None]
            rows.append(block.transpose(1, 2).flatten(0, 1)[:n])
        return torch.cat(rows)

    return {"key": part(0), "value": part(2)}


def _exact_attend(case, state):
    new, lengths = _sizes(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((state["tokens"], heads, dim), dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, m) in enumerate(zip(new, lengths)):
        begin, row = row, row + n
        if n == 0 or m == 0:
            continue
        page = state["table"][b, : -(-m // PAGE)].long()

        def part(at):
            codes, scales = state["cache"][at], state["cache"][at + 1]
            block = codes[page].view(torch.float8_e4m3fn).double() * \
                torch.exp2(scales[page].double() - 127)[:, :, None, None]
            return block.transpose(0, 1).flatten(1, 2)[:, :m]

        key, value = part(0), part(2)
        distance = torch.arange(m - n, m, device="cuda")[:, None] - \
            torch.arange(m, device="cuda")[None]
        seen = distance >= 0
        if case["window"]:
            seen &= (distance < case["window"]) | \
                (torch.arange(m, device="cuda")[None] < case["first"])
        for head in range(heads):
            kv = head // (heads // kv_heads)
            scores = state["query"][begin:begin + n, head].double() @ key[kv].T / math.sqrt(dim)
            scores = torch.where(seen, scores, -math.inf)
            if case["sinks"]:
                sink = state["sinks"][head].double().expand(n, 1)
                weights = torch.softmax(torch.cat((scores, sink), 1), 1)[:, :-1]
            else:
                weights = torch.softmax(scores, 1)
            out[begin:begin + n, head] = weights @ value[kv]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, state)
    if case["op"] == "read":
        return _exact_read(case, state)
    return _exact_attend(case, state)
