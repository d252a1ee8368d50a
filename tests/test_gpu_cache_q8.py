"""Writing and reading the 8-bit paged cache through the C ABI, against the 64-bit definition.

Codes and exponents are held to equality: the rotation is defined operation by operation in f32
(each product and their sum rounded once), which the reference repeats in f32, and from there on
every step (exponent, scaling by a power of two, rounding to nearest even) is exact in 64 bits.
The rotation itself is checked against 64 bits: three roundings of half a step, 3 * 2^-24 of the
products' magnitudes."""
import pytest
import torch

import cache_q8_reference as ref

pytestmark = pytest.mark.gpu


def status():
    from nml_b200 import _abi
    torch.cuda.synchronize()
    return _abi.device_status(0x1)


def to_device(tensors):
    return [t.cuda().contiguous() for t in tensors]


def make_rows(gen, tokens, heads, dim, dtype, spread=2.0):
    x = torch.randn((tokens, heads, dim), generator=gen)
    return (x * torch.exp2(spread * (2 * torch.rand((tokens, heads, 1), generator=gen) - 1))).to(
        dtype)


CASES = [
    # dtype, dim, kv_heads, group, rotary width, layout, new tokens, tokens before them
    (torch.bfloat16, 64, 8, 8, 64, "half", [1, 1, 1, 1], [0, 15, 16, 333]),
    (torch.float16, 64, 1, 1, 32, "half", [1], [7]),
    (torch.bfloat16, 128, 2, 3, 128, "half", [1, 40, 0, 5], [0, 3, 50, 1000]),
    (torch.float16, 128, 3, 2, 48, "interleaved", [33, 16, 1], [16, 0, 31]),
    (torch.bfloat16, 64, 2, 16, 16, "interleaved", [100, 2], [13, 14]),
    (torch.float16, 64, 5, 4, 0, "half", [17, 15], [0, 1]),
    (torch.bfloat16, 64, 8, 8, 64, "half", [1500, 3, 700], [9, 0, 32]),
]


@pytest.mark.parametrize("ragged", [True, False])
@pytest.mark.parametrize("dtype,dim,kv_heads,group,width,layout,new,before", CASES)
def test_append_matches_the_definition(dtype, dim, kv_heads, group, width, layout, new, before,
                                       ragged):
    from nml_b200 import ops
    if not ragged:
        new = [1] * len(new)
    gen = torch.Generator().manual_seed(dim + kv_heads * 10 + sum(new))
    lengths = [n + m for n, m in zip(new, before)]
    table, pages = ref.random_table(gen, lengths)
    cache = ref.stale(ref.random_cache(gen, pages, kv_heads, dim), table, before, gen)
    offsets, tokens = ref.offsets_of(new), sum(new)
    key = make_rows(gen, tokens, kv_heads, dim, dtype)
    value = make_rows(gen, tokens, kv_heads, dim, dtype)
    query = make_rows(gen, tokens, kv_heads * group, dim, dtype)
    position = torch.cat([torch.arange(n) + m for n, m in zip(new, before)])
    rotary = angles = None
    if width:
        frequencies = 10000.0 ** (-torch.arange(width // 2, dtype=torch.float64) / (width // 2))
        rotary = ops.rotary_table(frequencies, max(lengths) + 5, 1.25)
        angles = rotary[position]
    # one fused row holds the three parts
    fused = torch.cat((query, key, value), 1).cuda()
    heads = kv_heads * group
    dev = to_device(cache)
    out = ops.paged_append_q8(
        fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:], *dev, table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(),
        token_offsets=torch.tensor(offsets, dtype=torch.int32).cuda() if ragged else None,
        query=fused[:, :heads], rotary=None if rotary is None else rotary.cuda(),
        rotary_layout=layout)
    assert status() == 0
    turned = ref.rotate(key.float(), angles, layout)
    exact = ref.rotate(key.double(), angles, layout)
    if angles is not None:
        slack = 3 * 2.0 ** -24 * ref.rotate(key.double().abs(), angles.abs(), layout).abs()
        # |a cos| + |b sin| bounds the two products; the reference's first half subtracts
        both = key.double().abs().amax(-1, keepdim=True) * 2 * angles.abs().max()
        assert ((turned.double() - exact).abs() <= slack + 3 * 2.0 ** -24 * both).all()
    expected = [*ref.append(turned.double(), cache[0], cache[1], table, lengths, offsets),
                *ref.append(value.double(), cache[2], cache[3], table, lengths, offsets)]
    for got, want in zip(dev, expected):
        assert torch.equal(got.cpu(), want)
    assert torch.equal(out.cpu(), ref.rotate(query.float(), angles, layout).to(dtype))
    # the same call again finds the same cache: nothing is rounded twice
    ops.paged_append_q8(
        fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:], *dev, table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(),
        token_offsets=torch.tensor(offsets, dtype=torch.int32).cuda() if ragged else None,
        rotary=None if rotary is None else rotary.cuda(), rotary_layout=layout)
    for got, want in zip(dev, expected):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_extremes(dim):
    """Zeros, tiny and huge magnitudes, infinities, NaN, and a block that grows under its tokens."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(dim)
    kv_heads, new, before = 2, [16, 5, 4, 3, 20], [0, 11, 12, 2, 6]
    lengths = [n + m for n, m in zip(new, before)]
    table, pages = ref.random_table(gen, lengths)
    cache = ref.random_cache(gen, pages, kv_heads, dim)
    offsets, tokens = ref.offsets_of(new), sum(new)
    dtype = torch.bfloat16
    value = make_rows(gen, tokens, kv_heads, dim, dtype)
    value[0:16] = 0                      # a block of zeros
    value[16:21, 0] *= 2.0 ** 60         # saturates
    value[16:21, 1] = 2.0 ** -70         # below every code
    value[21:25, 0] *= 1000.0            # older tokens move to a larger exponent
    value[22, 1, 3] = float("inf")
    value[23, 1, dim - 1] = float("nan")
    value[26, 0, 0] = torch.finfo(dtype).min
    value[27, 1, 5] = -float("inf")
    value[28:44, 0] = 448.0              # exactly the largest code
    value[28:44, 1] = 450.0             # one step above it
    dev = to_device(cache)
    key = value.flip(0).contiguous()
    ops.paged_append_q8(key.cuda(), value.cuda(), *dev, table.cuda(),
                        torch.tensor(lengths, dtype=torch.int32).cuda(),
                        token_offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    assert status() == 0
    expected = [*ref.append(key.double(), cache[0], cache[1], table, lengths, offsets),
                *ref.append(value.double(), cache[2], cache[3], table, lengths, offsets)]
    for got, want in zip(dev, expected):
        assert torch.equal(got.cpu(), want)


def test_append_leaves_what_is_not_its_own():
    """Empty places of a padded batch, rows outside every sequence, pages of other sequences."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(5)
    kv_heads, dim, lengths = 2, 64, [17, 0, 3, -2 ** 31]
    table, pages = ref.random_table(gen, [17, 0, 3, 0])
    cache = ref.random_cache(gen, pages, kv_heads, dim)
    dev = to_device(cache)
    rows = make_rows(gen, 4, kv_heads, dim, torch.bfloat16)
    query = make_rows(gen, 4, 6, dim, torch.bfloat16).cuda()
    table[1] = -7  # an empty place's table is not read
    out = ops.paged_append_q8(rows.cuda(), rows.cuda(), *dev, table.cuda(),
                              torch.tensor(lengths, dtype=torch.int32).cuda(), query=query)
    assert status() == 0
    expected = ref.append(rows.double(), cache[0], cache[1], table, lengths, [0, 1, 2, 3, 4])
    assert torch.equal(dev[0].cpu(), expected[0]) and torch.equal(dev[1].cpu(), expected[1])
    assert torch.equal(out[[0, 2]], query[[0, 2]]) and (out[[1, 3]] == 0).all()
    # rows in front of and behind the sequences write nothing
    dev = to_device(cache)
    more = make_rows(gen, 9, kv_heads, dim, torch.bfloat16).cuda()
    ops.paged_append_q8(more, more, *dev, table.cuda(),
                        torch.tensor(lengths, dtype=torch.int32).cuda(),
                        token_offsets=torch.tensor([2, 4, 4, 6, 6], dtype=torch.int32).cuda())
    assert status() == 0
    expected = ref.append(more.double().cpu(), cache[0], cache[1], table, lengths,
                          [2, 4, 4, 6, 6])
    assert torch.equal(dev[0].cpu(), expected[0]) and torch.equal(dev[1].cpu(), expected[1])


def test_append_reports_what_it_cannot_place():
    from nml_b200 import _abi, ops
    gen = torch.Generator().manual_seed(6)
    kv_heads, dim = 2, 64
    cache = ref.random_cache(gen, 6, kv_heads, dim)
    rows = make_rows(gen, 1, kv_heads, dim, torch.bfloat16).cuda()
    rotary = ops.rotary_table(torch.ones(8), 10).cuda()
    for table, length, angles in (([[1, 6]], 17, None), ([[1, -1]], 17, None),
                                  ([[1, 2]], 33, None), ([[1, 2]], 11, rotary)):
        dev = to_device(cache)
        out = ops.paged_append_q8(rows, rows, *dev, torch.tensor(table, dtype=torch.int32).cuda(),
                                  torch.tensor([length], dtype=torch.int32).cuda(), query=rows,
                                  rotary=angles)
        assert status() == _abi.STATUS_INDEX_RANGE
        for got, want in zip(dev, cache):
            assert torch.equal(got.cpu(), want)
        if angles is not None:
            assert (out == 0).all()
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,kv_heads,rows", [(64, 8, [1]), (64, 1, [33, 0, 16, 1]),
                                               (128, 3, [500, 17, 0, 64]), (64, 8, [0, 0, 900])])
def test_read_back_is_exact(dtype, dim, kv_heads, rows):
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(dim + sum(rows))
    table, pages = ref.random_table(gen, rows)
    cache = ref.stale(ref.random_cache(gen, pages, kv_heads, dim, spread=3.0), table, rows, gen)
    offsets = [o + 2 for o in ref.offsets_of(rows)]  # two rows of nobody in front, three behind
    tokens = offsets[-1] + 3
    out = tuple(torch.full((tokens, kv_heads, dim), 7.0, dtype=dtype, device="cuda")
                for _ in range(2))
    got = ops.paged_read_q8(*to_device(cache), table.cuda(),
                            torch.tensor(offsets, dtype=torch.int32).cuda(), tokens, dtype, out)
    assert status() == 0
    for half, at in ((0, 0), (1, 2)):
        expected = torch.full((tokens, kv_heads, dim), 7.0, dtype=torch.float64)
        for b, n in enumerate(rows):
            expected[offsets[b]:offsets[b + 1]] = ref.gather(cache[at], cache[at + 1], table[b],
                                                             n)[0]
        assert torch.equal(got[half].cpu(), expected.to(dtype))


def test_read_back_reports_bad_pages():
    from nml_b200 import _abi, ops
    gen = torch.Generator().manual_seed(7)
    cache = to_device(ref.random_cache(gen, 4, 1, 64))
    key, value = ops.paged_read_q8(*cache, torch.tensor([[2, 9]], dtype=torch.int32).cuda(),
                                   torch.tensor([0, 40], dtype=torch.int32).cuda(), 40)
    assert status() == _abi.STATUS_INDEX_RANGE
    assert (key[16:] == 0).all() and (value[16:] == 0).all() and (key[:16] != 0).any()


def test_cache_past_32_bit_offsets():
    """Blocks more than 2^32 codes into the cache."""
    from nml_b200 import ops
    kv_heads, dim = 8, 128
    pages = (1 << 32) // (kv_heads * 16 * dim) + 40
    codes = [torch.empty((pages, kv_heads, 16, dim), dtype=torch.uint8, device="cuda")
             for _ in range(2)]
    scales = [torch.full((pages, kv_heads), 127, dtype=torch.uint8, device="cuda")
              for _ in range(2)]
    cache = (codes[0], scales[0], codes[1], scales[1])
    gen = torch.Generator().manual_seed(8)
    length = 400
    table = (torch.arange(25, dtype=torch.int32) + pages - 30)[None].contiguous()
    key = make_rows(gen, length, kv_heads, dim, torch.float16, 0.0)
    value = make_rows(gen, length, kv_heads, dim, torch.float16, 0.0)
    offsets = torch.tensor([0, length], dtype=torch.int32).cuda()
    lengths = torch.tensor([length], dtype=torch.int32).cuda()
    ops.paged_append_q8(key.cuda(), value.cuda(), *cache, table.cuda(), lengths,
                        token_offsets=offsets)
    back = ops.paged_read_q8(*cache, table.cuda(), offsets, length, torch.float16)
    assert status() == 0
    small = [x[pages - 40:].cpu() for x in cache]
    want = ref.append(key.double(), torch.zeros_like(small[0]), torch.zeros_like(small[1]),
                      table - (pages - 40), [length], [0, length])
    at = table[0].long() - (pages - 40)
    assert torch.equal(small[0][at], want[0][at]) and torch.equal(small[1][at], want[1][at])
    query = make_rows(gen, length, kv_heads, dim, torch.float16, 0.0)
    for rows, offset in ((query[-1:], None), (query, offsets)):
        out = ops.paged_attention_q8(rows.cuda(), *cache, table.cuda(), lengths,
                                     query_offsets=offset)
        assert status() == 0
        n = rows.shape[0]
        expected, bound = ref.attention(rows, small, table - (pages - 40), [length], [0, n], None,
                                        0, 0, dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, torch.float16)
    assert back[0].shape == (length, kv_heads, dim)


def test_appends_in_graphs_and_on_two_streams():
    """A captured append replayed with new rows, beside an eager one on another stream."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(9)
    kv_heads, dim, lengths = 2, 64, [40, 7, 200]
    table, pages = ref.random_table(gen, lengths)
    caches = [to_device(ref.random_cache(gen, pages, kv_heads, dim)) for _ in range(2)]
    before = [[x.cpu() for x in cache] for cache in caches]
    rows = [make_rows(gen, 3, kv_heads, dim, torch.bfloat16) for _ in range(2)]
    given = torch.zeros((3, kv_heads, dim), dtype=torch.bfloat16, device="cuda")
    arguments = (table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    kept = [x.clone() for x in caches[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        query = ops.paged_append_q8(given, given, *caches[0], *arguments, query=given)
    for cache, old in zip(caches[0], kept):  # capturing runs nothing
        assert torch.equal(cache, old)
    given.copy_(rows[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_append_q8(rows[1].cuda(), rows[1].cuda(), *caches[1], *arguments)
    graph.replay()
    assert status() == 0
    assert torch.equal(query.cpu(), rows[0])
    for cache, old, new in zip(caches, before, rows):
        for at in (0, 2):
            want = ref.append(new.double(), old[at], old[at + 1], table, lengths, [0, 1, 2, 3])
            assert torch.equal(cache[at].cpu(), want[0])
            assert torch.equal(cache[at + 1].cpu(), want[1])


def test_appending_and_reading_nothing():
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(10)
    table, pages = ref.random_table(gen, [20, 20])
    cache = ref.random_cache(gen, pages, 2, 64)
    dev = to_device(cache)
    rows = torch.ones((2, 2, 64), dtype=torch.float16, device="cuda")
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert ops.paged_append_q8(rows, rows, *dev, table.cuda(), none) is None
    empty = torch.zeros(3, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    out = ops.paged_append_q8(rows[:0], rows[:0], *dev, table.cuda(), lengths, empty,
                              query=rows[:0])
    assert out.shape == (0, 2, 64)
    ops.paged_append_q8(rows, rows, *dev, table.cuda(), lengths, empty)
    key, value = ops.paged_read_q8(*dev, table.cuda(), empty, 0)
    assert key.shape == value.shape == (0, 2, 64)
    assert status() == 0
    for got, want in zip(dev, cache):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 60])
def test_blocks_that_grow_are_moved_whole(dim, new):
    """Every sequence's partly filled block grows its exponent: all lanes of the warp that moves the
    older codes go by the exponent from before the call, each time."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(19 + new)
    kv_heads, batch = 4, 24
    counts, before = [new] * batch, [1 + i % 15 for i in range(batch)]
    lengths = [n + m for n, m in zip(counts, before)]
    table, pages = ref.random_table(gen, lengths)
    cache = ref.random_cache(gen, pages, kv_heads, dim)
    offsets, tokens = ref.offsets_of(counts), sum(counts)
    rows = [make_rows(gen, tokens, kv_heads, dim, torch.bfloat16) for _ in range(2)]
    for x in rows:
        x[offsets[:-1]] *= (2.0 ** (1 + torch.arange(batch) % 7))[:, None, None]
    expected = [*ref.append(rows[0].double(), cache[0], cache[1], table, lengths, offsets),
                *ref.append(rows[1].double(), cache[2], cache[3], table, lengths, offsets)]
    arguments = [table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                 torch.tensor(offsets, dtype=torch.int32).cuda()]
    start, rows = to_device(cache), to_device(rows)
    for _ in range(20):
        dev = [x.clone() for x in start]
        ops.paged_append_q8(*rows, *dev, *arguments)
        for got, want in zip(dev, expected):
            assert torch.equal(got.cpu(), want)
    assert status() == 0


@pytest.mark.parametrize("rows", [40, 1100])
def test_more_rows_than_tokens(rows):
    """Rows in front of a sequence's first token write nothing and give zero queries; the sequence
    starts at the row of its first token, wherever that lies among the rows."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(rows)
    kv_heads, dim, counts = 2, 64, [rows, 5, rows]
    lengths = [rows - 21, 3, 17]
    table, pages = ref.random_table(gen, lengths)
    cache = ref.random_cache(gen, pages, kv_heads, dim)
    offsets, tokens = ref.offsets_of(counts), 2 * rows + 5
    key, value = (make_rows(gen, tokens, kv_heads, dim, torch.float16) for _ in range(2))
    query = make_rows(gen, tokens, 4, dim, torch.float16)
    rotary = ops.rotary_table(torch.ones(16, dtype=torch.float64) / 3, rows + 1)
    dev = to_device(cache)
    out = ops.paged_append_q8(key.cuda(), value.cuda(), *dev, table.cuda(),
                              torch.tensor(lengths, dtype=torch.int32).cuda(),
                              torch.tensor(offsets, dtype=torch.int32).cuda(), query=query.cuda(),
                              rotary=rotary.cuda())
    assert status() == 0
    position = torch.cat([torch.arange(n) + m - n for n, m in zip(counts, lengths)])
    angles = rotary[position.clamp(min=0)]
    turned = ref.rotate(key.float(), angles, "half").double()
    expected = [*ref.append(turned, cache[0], cache[1], table, lengths, offsets),
                *ref.append(value.double(), cache[2], cache[3], table, lengths, offsets)]
    for got, want in zip(dev, expected):
        assert torch.equal(got.cpu(), want)
    rotated = ref.rotate(query.float(), angles, "half").to(torch.float16)
    assert torch.equal(out.cpu(), torch.where((position >= 0)[:, None, None], rotated, 0))
