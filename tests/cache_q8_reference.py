"""64-bit definitions of the operators over the 8-bit paged cache, sequence by sequence on the CPU,
and builders of caches and page tables for their tests."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE = 16


def decode(codes: torch.Tensor) -> torch.Tensor:
    return codes.view(torch.float8_e4m3fn).double()


def block_exponent(largest: float) -> int:
    """Smallest e in [-48, 48] with largest <= 448 * 2^e."""
    e = -48
    while e < 48 and largest > 448.0 * 2.0 ** e:
        e += 1
    return e


def encode(x: torch.Tensor, exponent: int) -> torch.Tensor:
    """E4M3 codes of f64 rows [.., dim] at one exponent; rows with an infinity or NaN become NaN."""
    scaled = (x * 2.0 ** -exponent).clamp(-448.0, 448.0)
    magnitude = scaled.abs()
    _, power = torch.frexp(magnitude)
    step = torch.exp2((power.double() - 4).clamp(min=-9.0))
    rounded = torch.copysign(torch.round(magnitude / step) * step, scaled)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    rounded = torch.where(fine, rounded, math.nan)
    # every value is an E4M3 number by now, so this conversion does not round
    return rounded.float().to(torch.float8_e4m3fn).view(torch.uint8)


def rotate(x: torch.Tensor, angles: torch.Tensor | None, layout: str) -> torch.Tensor:
    """Rows [n, heads, dim] rotated by angles [n, width], every operation in x's own type."""
    if angles is None:
        return x
    half = angles.shape[1] // 2
    cos, sin = angles[:, None, :half].to(x.dtype), angles[:, None, half:].to(x.dtype)
    y = x.clone()
    low = torch.arange(half) if layout == "half" else 2 * torch.arange(half)
    high = low + (half if layout == "half" else 1)
    y[..., low] = x[..., low] * cos - x[..., high] * sin
    y[..., high] = x[..., high] * cos + x[..., low] * sin
    return y


def append(rows, codes, scales, table, lengths, offsets):
    """Writes f64 rows [tokens, kv_heads, dim] into CPU copies of one half of the cache."""
    codes, scales = codes.clone(), scales.clone()
    for b, length in enumerate(lengths):
        begin, end = offsets[b], offsets[b + 1]
        by_page = {}
        for row in range(begin, end):
            position = length - end + row
            if position >= 0:
                by_page.setdefault(position // PAGE, []).append((position % PAGE, row))
        for logical, slots in by_page.items():
            page = int(table[b, logical])
            lead = slots[0][0]
            for head in range(codes.shape[1]):
                new = rows[[r for _, r in slots], head]
                fine = torch.isfinite(new).all(-1)
                largest = float(new[fine].abs().max()) if bool(fine.any()) else 0.0
                e = block_exponent(largest)
                if lead:
                    before = int(scales[page, head]) - 127
                    if e <= before:
                        e = before
                    else:
                        held = decode(codes[page, head, :lead]) * 2.0 ** before
                        codes[page, head, :lead] = encode(held, e)
                scales[page, head] = e + 127
                for slot, r in slots:
                    codes[page, head, slot] = encode(rows[r, head], e)
    return codes, scales


def gather(codes, scales, table, length):
    """f64 values, codes and exponents [tokens, kv_heads, ..] of one sequence."""
    pages = table[: -(-length // PAGE)].long()
    value = decode(codes[pages]).transpose(1, 2).flatten(0, 1)[:length]
    exponent = (scales[pages].double() - 127)[:, None].expand(-1, PAGE, -1).flatten(0, 1)[:length]
    return value * torch.exp2(exponent)[..., None], value, exponent


def attention(query, cache, table, lengths, offsets, sinks, window, first, scale):
    """(output, bound) in 64 bits [tokens, heads, dim].

    The bound covers what the operator documents, before the output's own rounding: a weight
    w = p 2^b / 2^M (b the value block's exponent, M the row's largest log2 of p 2^b) is narrowed
    to F16, off by at most 2^-11 of itself or by half of F16's smallest step, 2^-25; scores, exp2
    and sums in f32 add less than 2^-12 of the weights (their arguments are below 64 in magnitude
    where a weight counts, 2^-18; the score's own sum of 64 or 128 products is good to 2^-15 for
    the magnitudes tested; accumulation over 5000 tokens in steps of 16 to 2^-14)."""
    key, key_scales, value, value_scales = cache
    heads, dim = query.shape[1:]
    out = torch.zeros(query.shape, dtype=torch.float64)
    bound = torch.zeros(query.shape, dtype=torch.float64)
    group = heads // key.shape[1]
    for b, length in enumerate(lengths):
        begin, end = offsets[b], offsets[b + 1]
        if length == 0 or begin == end:
            continue
        keys, _, _ = gather(key, key_scales, table[b], length)
        values, codes, exponents = gather(value, value_scales, table[b], length)
        position = torch.arange(begin, end) + (length - end)
        token = torch.arange(length)
        seen = token[None] <= position[:, None]
        if window:
            seen &= (token[None] > position[:, None] - window) | (token[None] < first)
        for h in range(heads):
            kv = h // group
            scores = query[begin:end, h].double() @ torch.nan_to_num(keys[:, kv]).T * scale
            scores = torch.where(keys[:, kv].isnan().any(-1)[None], math.nan, scores)
            scores = torch.where(seen, scores, -math.inf)
            top = torch.where(scores.isnan(), -math.inf, scores).amax(1, keepdim=True)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.exp(scores - top)
            total = p.sum(1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks[h].double() - top)
            total = torch.where(total == 0, 1.0, total)
            visible = seen.any(0)
            v = torch.where(visible[:, None], values[:, kv], 0.0)
            # a masked token contributes nothing, whatever it holds
            numerator = torch.where(seen[..., None], p[..., None] * v[None], 0.0).sum(1) \
                if bool(v.isnan().any()) else p @ v
            out[begin:end, h] = numerator / total
            weight = p * torch.exp2(exponents[:, kv])[None]
            most = torch.where(weight.isnan(), 0.0, weight).amax(1, keepdim=True).clamp(min=1e-300)
            off = torch.maximum(weight * 2.0 ** -11, most * 2.0 ** -25) + weight * 2.0 ** -12
            off = torch.where(seen & ~weight.isnan(), off, 0.0)
            c = torch.where(visible[:, None], torch.nan_to_num(codes[:, kv]), 0.0).abs()
            bound[begin:end, h] = (off @ c) / total + out[begin:end, h].abs() * 2.0 ** -12
    return out, bound


def bound_of_each_dimension(query, cache, table, lengths, offsets, sinks, scale):
    """A bound [tokens, heads, dim] by what each dimension's own values weigh, whatever other tokens
    hold there: weights narrowed to F16 carry the exponent of their values only from 2^-4 to 2^2 of
    the largest, so that a probability is off by at most 2^-11 of itself or by half of F16's smallest
    step, 2^-25, times 2^6, of the row's largest; f32 adds less than 2^-12 of it, as above."""
    key, key_scales, value, value_scales = cache
    heads = query.shape[1]
    group = heads // key.shape[1]
    bound = torch.zeros(query.shape, dtype=torch.float64)
    for b, length in enumerate(lengths):
        begin, end = offsets[b], offsets[b + 1]
        keys, _, _ = gather(key, key_scales, table[b], length)
        values, _, _ = gather(value, value_scales, table[b], length)
        position = torch.arange(begin, end) + (length - end)
        seen = torch.arange(length)[None] <= position[:, None]
        for h in range(heads):
            scores = query[begin:end, h].double() @ keys[:, h // group].T * scale
            scores = torch.where(seen, scores, -math.inf)
            p = torch.exp(scores - scores.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            if sinks is not None:
                total = total + torch.exp(sinks[h].double() - scores.amax(1, keepdim=True))
            off = torch.clamp(p * 2.0 ** -11, min=2.0 ** -19) + p * 2.0 ** -12
            v = values[:, h // group]
            bound[begin:end, h] = torch.where(seen, off, 0.0) @ v.abs() / total + \
                (p @ v / total).abs() * 2.0 ** -12
    return bound


def assert_attention_close(actual, expected, bound, dtype):
    """|a - e| within the bound plus the output's rounding: half a step of its type, or of its
    smallest number."""
    a = actual.double().cpu()
    assert torch.equal(a.isnan(), expected.isnan())
    smallest = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]
    limit = bound + (expected.abs() + bound) * (torch.finfo(dtype).eps / 2) + smallest
    fine = ~expected.isnan()
    excess = ((a - expected).abs() - limit)[fine]
    assert excess.numel() == 0 or excess.max() <= 0, (
        excess.max().item(), (a - expected).abs()[fine].max().item())


def random_cache(gen, pages, kv_heads, dim, spread=0.0):
    """CPU cache (key, key scales, value, value scales) of random blocks, every page written."""
    halves = []
    for _ in range(2):
        x = torch.randn((pages, kv_heads, PAGE, dim), generator=gen, dtype=torch.float64)
        x = x * torch.exp2(spread * (2 * torch.rand((pages, kv_heads, 1, 1), generator=gen,
                                                    dtype=torch.float64) - 1))
        largest = x.abs().amax((2, 3))
        e = torch.ceil(torch.log2(largest / 448)).clamp(-48, 48)
        scaled = x * torch.exp2(-e)[..., None, None]
        halves += [scaled.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8),
                   (e + 127).to(torch.uint8)]
    return halves


def random_table(gen, lengths, spare=3):
    """(page table, pages): every sequence owns a random set of pages, one logical page unused."""
    width = max(1, max(-(-n // PAGE) for n in lengths)) + 1
    pages = len(lengths) * width + spare
    order = torch.randperm(pages, generator=gen)[: len(lengths) * width]
    return order.view(len(lengths), width).to(torch.int32), pages


def stale(cache, table, lengths, gen):
    """Fills every slot that holds no token of a sequence with random rows, NaN rows among them."""
    key, _, value, _ = cache
    pages = key.shape[0]
    written = torch.zeros((pages, PAGE), dtype=torch.bool)
    for b, n in enumerate(lengths):
        for t in range(n):
            written[int(table[b, t // PAGE]), t % PAGE] = True
    for codes in (key, value):
        junk = torch.randint(0, 256, (pages, codes.shape[1], PAGE, 1), generator=gen,
                             dtype=torch.uint8)
        junk[0::2] = 0x7f
        codes.copy_(torch.where(written[:, None, :, None], codes, junk))
    return cache


def offsets_of(counts):
    return np.concatenate(([0], np.cumsum(counts))).astype(int).tolist()
