"""Attention over the 8-bit paged cache against its definition in 64 bits over the same codes.
The tolerance is derived in cache_q8_reference.attention from the roundings that the operator
documents; it scales with the weights' own magnitudes, not with the output's."""
import pytest
import torch

import cache_q8_reference as ref

pytestmark = pytest.mark.gpu


def status():
    from nml_b200 import _abi
    torch.cuda.synchronize()
    return _abi.device_status(0x1)


def make(seed, dtype, dim, kv_heads, group, new, before, spread=0.0, with_sinks=False):
    gen = torch.Generator().manual_seed(seed)
    lengths = [n + m if m is not None else 0 for n, m in zip(new, before)]
    table, pages = ref.random_table(gen, lengths)
    cache = ref.stale(ref.random_cache(gen, pages, kv_heads, dim, spread), table, lengths, gen)
    query = torch.randn((sum(new), kv_heads * group, dim), generator=gen).to(dtype)
    sinks = torch.randn(kv_heads * group, generator=gen) if with_sinks else None
    return lengths, table, cache, query, sinks, ref.offsets_of(new)


def call(query, cache, table, lengths, offsets, sinks, **options):
    from nml_b200 import ops
    return ops.paged_attention_q8(
        query.cuda(), *[x.cuda() for x in cache], table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(),
        query_offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda(),
        sinks=None if sinks is None else sinks.cuda(), **options)


SINGLE = [
    # dim, kv_heads, group, tokens before each query (None: an empty place), window, first, sinks
    (64, 8, 8, [0, 15, 16, 4095], 0, 0, True),
    (64, 2, 8, [99, None, 700, None], 0, 0, True),
    (64, 1, 1, [40], 0, 0, False),
    (64, 3, 5, [333, 5, 63], 128, 0, False),
    (64, 2, 16, [1000, 64], 128, 4, True),
    (64, 1, 20, [500], 1, 0, False),
    (128, 8, 4, [2000, 31, 0], 0, 0, False),
    (128, 2, 12, [77, 300], 100, 33, True),
    (128, 1, 128, [400], 0, 0, True),
    (64, 1, 8, [200, 201], 64, 500, False),   # the first tokens cover everything
    (64, 4, 8, [130, 17], 16, 1, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [None, 1, 3])
@pytest.mark.parametrize("dim,kv_heads,group,before,window,first,with_sinks", SINGLE)
def test_single_tokens(dtype, dim, kv_heads, group, before, window, first, with_sinks, splits):
    new = [1] * len(before)
    lengths, table, cache, query, sinks, offsets = make(
        dim + group, dtype, dim, kv_heads, group, new, before, with_sinks=with_sinks)
    out = call(query, cache, table, lengths, None, sinks, sliding_window=window or None,
               first_tokens=first, splits=splits)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, window, first,
                                    dim ** -0.5)
    ref.assert_attention_close(out, expected, bound, dtype)
    for b, m in enumerate(before):
        if m is None:
            assert (out[b] == 0).all()


RUNS = [
    # dim, kv_heads, group, new tokens, tokens before them, window, first, sinks
    (64, 2, 8, [5, 1, 0, 3], [100, 0, 20, 1500], 0, 0, True),
    (64, 1, 8, [200], [0], 0, 0, False),
    (64, 2, 8, [130, 17, 64], [0, 300, 15], 0, 0, True),
    (64, 1, 8, [300, 40], [50, 900], 128, 4, True),
    (64, 1, 4, [150], [37], 20, 0, False),
    (64, 2, 3, [90, 5], [10, 411], 0, 0, False),
    (64, 1, 1, [257, 2], [1, 0], 0, 0, True),
    (64, 1, 16, [33, 20], [0, 140], 50, 1, False),
    (64, 1, 128, [7], [30], 0, 0, False),
    (128, 2, 4, [140, 60], [3, 200], 0, 0, True),
    (128, 1, 8, [100, 1], [0, 260], 64, 5, False),
    (128, 1, 5, [70], [0], 0, 0, False),
    # short runs: a few rows that share what is read of their sequence
    (64, 2, 8, [4, 1, 0, 3, 9], [100, 0, 20, 1500, 37], 0, 0, True),
    (64, 1, 5, [5, 5, 2], [3, 200, 14], 64, 2, False),
    (64, 3, 1, [3, 8], [700, 13], 0, 0, True),
    (64, 1, 8, [5, 4], [126, 60], 16, 20, False),
    (128, 2, 4, [2, 3, 1], [130, 0, 900], 0, 0, True),
    (128, 1, 8, [5, 0, 4], [15, 3, 400], 33, 1, False),
    (64, 1, 16, [2, 2], [500, 30], 0, 0, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [None, 1, 2])
@pytest.mark.parametrize("dim,kv_heads,group,new,before,window,first,with_sinks", RUNS)
def test_runs_of_tokens(dtype, dim, kv_heads, group, new, before, window, first, with_sinks,
                        splits):
    lengths, table, cache, query, sinks, offsets = make(
        dim + group + 1, dtype, dim, kv_heads, group, new, before, with_sinks=with_sinks)
    out = call(query, cache, table, lengths, offsets, sinks, sliding_window=window or None,
               first_tokens=first, splits=splits)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, window, first,
                                    dim ** -0.5)
    ref.assert_attention_close(out, expected, bound, dtype)


@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_of_unlike_magnitudes(dim, runs):
    """Exponents of neighbouring blocks up to 2^40 apart, in keys and in values; queries of every
    magnitude."""
    new, before = ([60, 9], [200, 140]) if runs else ([1, 1], [259, 148])
    lengths, table, cache, query, sinks, offsets = make(3, torch.bfloat16, dim, 2, 8, new, before,
                                                        spread=20.0, with_sinks=True)
    # keys of a common, small magnitude keep the softmax from collapsing onto one block
    cache[1] = torch.full_like(cache[1], 120)
    query = (query.float() * torch.exp2(torch.arange(query.shape[1]) % 7 - 3.0)[:, None]).to(
        torch.bfloat16)
    query[0, 0] *= 2.0 ** -90
    query[0, 1] = 0
    out = call(query, cache, table, lengths, offsets if runs else None, sinks)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, 0, 0,
                                    dim ** -0.5)
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
def test_nan_tokens_reach_only_rows_that_see_them(dim):
    """A row stored as NaN makes NaN of the queries that see it and leaves the others alone."""
    new, before = [100], [30]
    lengths, table, cache, query, sinks, offsets = make(4, torch.bfloat16, dim, 2, 8, new, before)
    for token, at in ((70, 0), (90, 2)):  # a key row of head 0, a value row of head 1
        page, slot = int(table[0, token // 16]), token % 16
        cache[at][page, 0 if at == 0 else 1, slot] = 0x7f
    out = call(query, cache, table, lengths, offsets, None)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, None, 0, 0, dim ** -0.5)
    assert expected[40:, :8].isnan().all() and expected[60:, 8:].isnan().all()
    assert not expected[:40].isnan().any() and not expected[:60, 8:].isnan().any()
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)
    # single tokens, the NaN inside and outside a window
    for window in (0, 10):
        one = call(query[-1:], cache, table, lengths, None, None, sliding_window=window or None)
        expected, bound = ref.attention(query[-1:], cache, table, lengths, [0, 1], None, window, 0,
                                        dim ** -0.5)
        assert expected.isnan().any() == (window == 0)
        ref.assert_attention_close(one, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2])
def test_nan_tokens_in_short_runs(dim, splits):
    """The same for the rows of a short run: values that are NaN inside the run itself and, past a
    window, in front of some of its rows."""
    # row i is at position 200 + i: a window of 8 ends before row 195 + 8 - 200 = 3
    for window, token, first_nan, last_nan in ((0, 201, 1, 5), (8, 195, 0, 3), (8, 203, 3, 5)):
        lengths, table, cache, query, _, offsets = make(17, torch.bfloat16, dim, 2, 8, [5], [200])
        page, slot = int(table[0, token // 16]), token % 16
        cache[2][page, 1, slot] = 0x7f   # a value row of head 1
        cache[0][page, 0, slot] = 0xff   # a key row of head 0
        out = call(query, cache, table, lengths, offsets, None, sliding_window=window or None,
                   splits=splits)
        assert status() == 0
        expected, bound = ref.attention(query, cache, table, lengths, offsets, None, window, 0,
                                        dim ** -0.5)
        rows = expected.isnan().any(-1).all(-1)
        assert rows.tolist() == [first_nan <= i < last_nan for i in range(5)]
        ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("splits", [1, 3])
def test_queries_that_are_not_finite(dtype, runs, splits):
    new, before = ([20, 9], [300, 140]) if runs else ([1, 1], [319, 148])
    lengths, table, cache, query, sinks, offsets = make(13, dtype, 64, 2, 8, new, before)
    query[0, 3, 5] = float("inf")
    query[-1, 9, 63] = -float("inf")
    query[-1, 14, 0] = float("nan")
    out = call(query, cache, table, lengths, offsets if runs else None, None, splits=splits)
    assert status() == 0
    bad = ~torch.isfinite(query).all(-1)
    expected, bound = ref.attention(torch.where(bad[..., None], 0, query), cache, table, lengths,
                                    offsets, None, 0, 0, 0.125)
    expected[bad] = float("nan")
    ref.assert_attention_close(out, expected, bound, dtype)


@pytest.mark.parametrize("runs", [False, True])
def test_windows_past_every_length(runs):
    """The largest windows and counts of first tokens that the call takes."""
    most = 2 ** 31 - 1
    new, before = ([70, 3], [40, 200]) if runs else ([1, 1], [109, 202])
    lengths, table, cache, query, sinks, offsets = make(14, torch.bfloat16, 64, 1, 8, new, before)
    given = offsets if runs else None
    plain = call(query, cache, table, lengths, given, None)
    assert torch.equal(call(query, cache, table, lengths, given, None, sliding_window=most), plain)
    wide = call(query, cache, table, lengths, given, None, sliding_window=5,
                first_tokens=most - 16)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, None, 5, 10 ** 6, 0.125)
    ref.assert_attention_close(wide, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("runs", [False, True])
def test_lengths_below_zero_are_empty(runs):
    new = [5, 4] if runs else [1, 1]
    lengths, table, cache, query, _, offsets = make(16, torch.bfloat16, 64, 2, 8, new, [20, 30])
    given = offsets if runs else None
    want = call(query, cache, table, [0, lengths[1]], given, None)
    for empty in (-1, -2 ** 31):
        assert torch.equal(call(query, cache, table, [empty, lengths[1]], given, None), want)
    assert status() == 0 and (want[: new[0]] == 0).all()


def test_nothing_to_do():
    """No rows, a batch of empty places, sequences without rows."""
    lengths, table, cache, query, _, _ = make(15, torch.bfloat16, 64, 2, 8, [4, 4], [0, 30])
    assert call(query[:0], cache, table, lengths, [0, 0, 0], None).shape == (0, 16, 64)
    assert (call(query[:2], cache, table, [0, 0], None, None) == 0).all()
    from nml_b200 import ops
    out = torch.full((8, 16, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    for splits in (1, 2):
        ops.paged_attention_q8(query.cuda(), *[x.cuda() for x in cache], table.cuda(),
                               torch.tensor(lengths, dtype=torch.int32).cuda(),
                               query_offsets=torch.tensor([3, 3, 3], dtype=torch.int32).cuda(),
                               splits=splits, out=out)
        assert status() == 0 and (out == 3).all()


@pytest.mark.parametrize("splits", [1, 4])
def test_rows_outside_every_sequence_stay(splits):
    lengths, table, cache, query, sinks, _ = make(5, torch.float16, 64, 2, 8, [3, 0, 40, 9],
                                                  [5, 7, 60, 100])
    from nml_b200 import ops
    offsets = [2, 3, 3, 41, 48]  # sequences of 1, 0, 38 and 7 rows
    out = torch.full(query.shape, 5.0, dtype=torch.float16, device="cuda")
    got = ops.paged_attention_q8(
        query.cuda(), *[x.cuda() for x in cache], table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(),
        query_offsets=torch.tensor(offsets, dtype=torch.int32).cuda(), splits=splits, out=out)
    assert status() == 0 and got is out
    expected, bound = ref.attention(query, cache, table, lengths, offsets, None, 0, 0, 0.125)
    assert (out[:2] == 5).all() and (out[48:] == 5).all()
    ref.assert_attention_close(out[2:48], expected[2:48], bound[2:48], torch.float16)


@pytest.mark.parametrize("runs", [False, True])
def test_more_rows_than_tokens(runs):
    """Rows in front of a sequence's first token (a length below its row count) see nothing."""
    new = [6, 4] if runs else [1, 1]
    lengths, table, cache, query, sinks, offsets = make(6, torch.bfloat16, 64, 1, 8, new, [0, 30])
    lengths[0] = 2 if runs else 0
    out = call(query, cache, table, lengths, offsets if runs else None, None)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, None, 0, 0, 0.125)
    assert (expected[: 4 if runs else 1] == 0).all()
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("runs", [False, True])
def test_bad_pages_are_reported_and_unseen(runs):
    from nml_b200 import _abi
    new, before = ([40], [60]) if runs else ([1], [99])
    lengths, table, cache, query, sinks, offsets = make(7, torch.bfloat16, 64, 2, 8, new, before)
    table[0, 2] = cache[0].shape[0]
    table[0, 4] = -5
    out = call(query, cache, table, lengths, offsets if runs else None, None)
    assert status() == _abi.STATUS_INDEX_RANGE
    assert torch.isfinite(out).all()
    # a length past the table is cut to it
    lengths, table, cache, query, sinks, offsets = make(8, torch.bfloat16, 64, 2, 8, new, before)
    full = table.shape[1] * 16
    out = call(query, cache, table, [full + 100], offsets if runs else None, None)
    assert status() == _abi.STATUS_INDEX_RANGE
    if not runs:
        expected, bound = ref.attention(query, [torch.nan_to_num(x) for x in cache], table, [full],
                                        offsets, None, 0, 0, 0.125)
        assert torch.equal(out.isnan().cpu(), expected.isnan())


def test_strided_queries_and_another_stream():
    lengths, table, cache, query, sinks, offsets = make(9, torch.bfloat16, 64, 2, 8, [30, 50],
                                                        [10, 500], with_sinks=True)
    from nml_b200 import ops
    wide = torch.zeros((80, 24, 64), dtype=torch.bfloat16, device="cuda")
    wide[:, 4:20] = query.cuda()
    dev = [x.cuda() for x in cache]
    arguments = (*dev, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(),
                 torch.tensor(offsets, dtype=torch.int32).cuda(), sinks.cuda())
    plain = ops.paged_attention_q8(query.cuda(), *arguments)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        strided = ops.paged_attention_q8(wide[:, 4:20], *arguments)
    torch.cuda.current_stream().wait_stream(side)
    assert status() == 0
    assert torch.equal(plain, strided)


@pytest.mark.parametrize("runs", [False, True])
def test_captured_graphs_share_no_scratch(runs):
    """Two graphs captured on one stream, replayed at once on two streams, with splits."""
    from nml_b200 import ops
    sets = []
    for seed in (10, 11):
        new, before = ([20, 33], [900, 1500]) if runs else ([1, 1], [1900, 2400])
        lengths, table, cache, query, sinks, offsets = make(seed, torch.bfloat16, 64, 2, 8, new,
                                                            before)
        dev = [x.cuda() for x in cache]
        arguments = (query.cuda(), *dev, table.cuda(),
                     torch.tensor(lengths, dtype=torch.int32).cuda(),
                     torch.tensor(offsets, dtype=torch.int32).cuda() if runs else None)
        eager = ops.paged_attention_q8(*arguments, splits=5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention_q8(*arguments, splits=5)
        sets.append((graph, out, eager, arguments))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, out, _, _), stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                out.zero_()
                graph.replay()
        torch.cuda.synchronize()
        for _, out, eager, _ in sets:
            assert torch.equal(out, eager)
    assert status() == 0


def test_prompts_and_tokens_in_a_row():
    """A conversation: ragged prompts appended in two chunks and attended to, then single tokens,
    each step against the 64-bit definition over the values read back from the cache."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(12)
    dtype, dim, kv_heads, group, batch = torch.bfloat16, 64, 2, 8, 3
    total = [150, 40, 90]
    table, pages = ref.random_table(gen, total)
    cache = [x.cuda() for x in ref.stale(ref.random_cache(gen, pages, kv_heads, dim), table,
                                         [0] * batch, gen)]
    rotary = ops.rotary_table(150000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), 200).cuda()
    sinks = torch.randn(kv_heads * group, generator=gen)
    lengths = [0] * batch
    written = [torch.zeros((0, kv_heads, dim), dtype=torch.float64) for _ in range(batch)]
    for step in ([100, 5, 33], [30, 20, 0], [1, 1, 1], [1, 1, 1]):
        lengths = [m + n for m, n in zip(lengths, step)]
        offsets = ref.offsets_of(step)
        single = step == [1, 1, 1]
        rows = torch.randn((sum(step), (group + 2) * kv_heads, dim), generator=gen).to(dtype)
        fused = rows.cuda()
        device_lengths = torch.tensor(lengths, dtype=torch.int32).cuda()
        device_offsets = None if single else torch.tensor(offsets, dtype=torch.int32).cuda()
        heads = group * kv_heads
        query = ops.paged_append_q8(fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:],
                                    *cache, table.cuda(), device_lengths, device_offsets,
                                    query=fused[:, :heads], rotary=rotary)
        out = ops.paged_attention_q8(query, *cache, table.cuda(), device_lengths, device_offsets,
                                     sinks=sinks.cuda(), sliding_window=64, first_tokens=2)
        assert status() == 0
        held = [x.cpu() for x in cache]
        expected, bound = ref.attention(query.cpu(), held, table, lengths, offsets, sinks, 64, 2,
                                        dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, dtype)
        for b in range(batch):
            new = rows[offsets[b]:offsets[b + 1], heads + kv_heads:].double()
            written[b] = torch.cat((written[b], new))
            if lengths[b]:
                # what the cache holds is what was written, to half a code step (2^-4) of each
                # value or of the block's smallest code (two roundings where a block has grown)
                value, _, exponent = ref.gather(held[2], held[3], table[b], lengths[b])
                limit = written[b].abs() * 2.0 ** -4 * 1.07 + \
                    2 * 2.0 ** -10 * torch.exp2(exponent)[..., None]
                assert ((value - written[b]).abs() <= limit).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_runs_repeat_themselves(dim):
    """Every step goes by its own pages' scales: magnitudes that change from page to page, many tiles
    beside each other, the same bits each time."""
    new, before = [90, 33, 150, 64] * 3, [400, 900, 0, 77] * 3
    lengths, table, cache, query, sinks, offsets = make(21, torch.bfloat16, dim, 2, 8, new, before,
                                                        spread=3.0, with_sinks=True)
    out = call(query, cache, table, lengths, offsets, sinks)
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, 0, 0, dim ** -0.5)
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)
    for _ in range(20):
        assert torch.equal(call(query, cache, table, lengths, offsets, sinks), out)
    assert status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("runs", [False, True])
def test_masked_tokens_of_tiny_scores(dim, runs, splits):
    """A score factor below f32's smallest number (tiny queries, or a tiny scale, over blocks of zero
    keys, whose exponent is the least) leaves what is masked out masked: the seen values' mean."""
    new, before = ([40, 9], [60, 140]) if runs else ([1, 1], [99, 148])
    given = None
    for dtype, magnitude, scale in ((torch.bfloat16, 2.0 ** -90, None), (torch.bfloat16, 1.0, 1e-36),
                                    (torch.float16, 1.0, 1e-36), (torch.bfloat16, 2.0 ** -126, 1e-38)):
        lengths, table, cache, query, sinks, offsets = make(22, dtype, dim, 2, 8, new, before)
        cache[0].zero_()
        cache[1].fill_(127 - 48)
        query = (query.float() * magnitude).to(dtype)
        given = offsets if runs else None
        for window in (0, 37):
            out = call(query, cache, table, lengths, given, None, scale=scale, splits=splits,
                       sliding_window=window or None)
            assert status() == 0
            expected, bound = ref.attention(query, cache, table, lengths, offsets, None, window, 0,
                                            dim ** -0.5 if scale is None else scale)
            assert torch.isfinite(expected).all()
            ref.assert_attention_close(out, expected, bound, dtype)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 8])
def test_many_more_rows_than_tokens(dim, group):
    """Rows up to 100 positions in front of the first token share a tile with rows that see some."""
    lengths, table, cache, query, _, offsets = make(23, torch.bfloat16, dim, 2, group, [120, 50],
                                                    [0, 0])
    lengths = [20, 41]
    out = call(query, cache, table, lengths, offsets, None)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, None, 0, 0, dim ** -0.5)
    assert (expected[:100] == 0).all() and (expected[120:129] == 0).all()
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("runs", [False, True])
def test_queries_that_are_not_finite_and_see_nothing(dtype, runs, splits):
    """Empty places of a padded batch, rows in front of the first token and rows whose only page is
    bad give zeros whatever their queries hold, in either kernel."""
    from nml_b200 import _abi
    new, before = ([5, 30, 4, 7], [0, 0, 40, 0]) if runs else ([1, 1, 1, 1], [0, 0, 43, 0])
    lengths, table, cache, query, _, offsets = make(24, dtype, 64, 2, 8, new, before)
    lengths[:2] = [0, 12 if runs else 0]
    given = offsets if runs else None
    query[:, 1::2] = float("nan")
    query[:, 4] = float("inf")
    bad = ~torch.isfinite(query).all(-1)
    expected, bound = ref.attention(torch.where(bad[..., None], 0, query), cache, table, lengths,
                                    offsets, None, 0, 0, 0.125)
    sees = torch.cat([torch.arange(n) + m - n >= 0 for n, m in zip(new, lengths)])
    expected[bad & sees[:, None]] = float("nan")
    out = call(query, cache, table, lengths, given, None, splits=splits)
    assert status() == 0
    assert (out[~sees.cuda()] == 0).all()
    ref.assert_attention_close(out, expected, bound, dtype)
    table[3] = -1  # nothing of the last sequence can be seen
    out = call(query, cache, table, lengths, given, None, splits=splits)
    assert status() == _abi.STATUS_INDEX_RANGE
    assert (out[offsets[3]:] == 0).all()
    ref.assert_attention_close(out[:offsets[3]], expected[:offsets[3]], bound[:offsets[3]], dtype)


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("runs", [False, True])
def test_lengths_past_the_table_keep_their_positions(runs, splits):
    """Rows keep the positions that the given length says; of the tokens that they see, those past
    the table are not there.  A row whose window lies past the table sees its first tokens only."""
    from nml_b200 import _abi
    n = 60 if runs else 1
    for excess in (7, 30, 500, None):
        lengths, table, cache, query, _, offsets = make(25, torch.bfloat16, 64, 2, 8, [n], [140])
        full = table.shape[1] * 16
        given = 2 ** 31 - 1 if excess is None else full + excess
        for x in cache[0::2]:
            x.copy_(torch.where(x & 0x7f == 0x7f, 0x30, x))  # every slot of the table is a token's
        for window, first in ((0, 0), (40, 0), (40, 20)):
            out = call(query, cache, table, [given], offsets if runs else None, None, splits=splits,
                       sliding_window=window or None, first_tokens=first)
            assert status() == _abi.STATUS_INDEX_RANGE
            for i in range(n):
                position = given - n + i
                seen = min(position + 1, full)
                start = max(0, position + 1 - window) if window else 0
                if start < seen:
                    expected, bound = ref.attention(query[i:i + 1], cache, table, [seen], [0, 1],
                                                    None, seen - start if start else 0, first, 0.125)
                elif first:
                    expected, bound = ref.attention(query[i:i + 1], cache, table, [first], [0, 1],
                                                    None, 0, 0, 0.125)
                else:
                    expected = bound = torch.zeros((1, 16, 64), dtype=torch.float64)
                ref.assert_attention_close(out[i:i + 1], expected, bound, torch.bfloat16)


def outlier_pages(dim, new, before, gap, at, dtype, seed):
    """One page of every sequence whose values are 2^gap times the others', in the first half of the
    dimensions only: the second half is the other pages' alone."""
    lengths, table, cache, query, sinks, offsets = make(seed, dtype, dim, 2, 8, new, before,
                                                        with_sinks=True)
    low = max(127 - 9 - gap // 2, 127 - 48)  # the least exponent that a block has
    cache[3].fill_(low)
    for b, length in enumerate(lengths):
        last = (offsets[b + 1] - offsets[b] + 15) // 16 + 1  # in front of what only some rows see
        page = int(table[b, {"first": 0, "inside": (length // 16 - last) // 2,
                             "last": length // 16 - last}[at]])
        cache[3][page] = low + gap
        cache[2][page, :, :, dim // 2:] = 0
    return lengths, table, cache, query * 0.5, sinks, offsets


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("gap", [3, 6, 20, 60, 90])
@pytest.mark.parametrize("at", ["first", "inside", "last"])
@pytest.mark.parametrize("splits", [1, 3])
def test_a_page_of_large_values_takes_nothing_from_the_others(dim, gap, at, splits):
    new, before = [1, 1, 1], [700, 240, 95]
    lengths, table, cache, query, sinks, offsets = outlier_pages(dim, new, before, gap, at,
                                                                 torch.bfloat16, 26)
    for q in (query, torch.zeros_like(query)):
        out = call(q, cache, table, lengths, None, sinks, splits=splits)
        assert status() == 0
        expected, _ = ref.attention(q, cache, table, lengths, offsets, sinks, 0, 0, dim ** -0.5)
        bound = ref.bound_of_each_dimension(q, cache, table, lengths, offsets, sinks, dim ** -0.5)
        assert (bound < 0.05 * expected.abs().amax(-1, keepdim=True)).all()
        ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [8, 12])
def test_values_of_every_magnitude(dim, group):
    """Neighbouring pages up to 2^90 apart, every dimension by its own values."""
    lengths, table, cache, query, sinks, offsets = make(27, torch.bfloat16, dim, 2, group, [1, 1],
                                                        [900, 333], with_sinks=True)
    gen = torch.Generator().manual_seed(27)
    shape = cache[3].shape
    cache[3] = torch.randint(127 - 45, 127 + 46, shape, generator=gen).to(torch.uint8)
    # a dimension holds values of pages of one residue only
    residue = torch.randint(0, 8, (shape[0], 1, 1, 1), generator=gen)
    cache[2] = torch.where(torch.arange(dim) % 8 == residue, cache[2], 0)
    for splits in (1, 2):
        out = call(query, cache, table, lengths, None, sinks, splits=splits)
        assert status() == 0
        expected, _ = ref.attention(query, cache, table, lengths, offsets, sinks, 0, 0, dim ** -0.5)
        bound = ref.bound_of_each_dimension(query, cache, table, lengths, offsets, sinks,
                                            dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("gap", [3, 6, 20, 60, 90])
@pytest.mark.parametrize("at", ["first", "inside", "last"])
@pytest.mark.parametrize("splits", [1, 3])
def test_a_page_of_large_values_takes_nothing_from_the_others_in_runs(dim, gap, at, splits):
    new, before = [40, 9, 25], [700, 240, 95]
    lengths, table, cache, query, sinks, offsets = outlier_pages(dim, new, before, gap, at,
                                                                 torch.bfloat16, 28)
    for q in (query, torch.zeros_like(query)):
        out = call(q, cache, table, lengths, offsets, sinks, splits=splits)
        assert status() == 0
        expected, _ = ref.attention(q, cache, table, lengths, offsets, sinks, 0, 0, dim ** -0.5)
        bound = ref.bound_of_each_dimension(q, cache, table, lengths, offsets, sinks, dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 8, 12])
def test_values_of_every_magnitude_in_runs(dim, group):
    new, before = [50, 3, 200], [900, 333, 0]
    lengths, table, cache, query, sinks, offsets = make(29, torch.bfloat16, dim, 2, group, new,
                                                        before, with_sinks=True)
    gen = torch.Generator().manual_seed(29)
    shape = cache[3].shape
    cache[3] = torch.randint(127 - 45, 127 + 46, shape, generator=gen).to(torch.uint8)
    residue = torch.randint(0, 8, (shape[0], 1, 1, 1), generator=gen)
    cache[2] = torch.where(torch.arange(dim) % 8 == residue, cache[2], 0)
    # (a slot that no row sees may hold NaN: only the tokens' own dimensions were cleared)
    for splits in (1, 2):
        out = call(query, cache, table, lengths, offsets, sinks, splits=splits)
        assert status() == 0
        expected, _ = ref.attention(query, cache, table, lengths, offsets, sinks, 0, 0, dim ** -0.5)
        bound = ref.bound_of_each_dimension(query, cache, table, lengths, offsets, sinks,
                                            dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("dim,kv_heads,group,new,before,window,first,with_sinks",
                         [case for case in RUNS if sum(case[3]) >= 3 * len(case[3])])
def test_runs_over_values_far_apart(dtype, dim, kv_heads, group, new, before, window, first,
                                    with_sinks, splits):
    """The runs above, for which the tile kernel takes its values whole: neighbouring pages up to 2^16
    apart.  Weights are two BF16 terms then, off by 2^-17 of themselves: within the bound for F16."""
    lengths, table, cache, query, sinks, offsets = make(
        dim + group + 2, dtype, dim, kv_heads, group, new, before, with_sinks=with_sinks)
    gen = torch.Generator().manual_seed(30)
    shift = torch.randint(-12, 5, cache[3].shape, generator=gen)
    cache[3] = (cache[3].int() + shift).to(torch.uint8)
    out = call(query, cache, table, lengths, offsets, sinks, sliding_window=window or None,
               first_tokens=first, splits=splits)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, window, first,
                                    dim ** -0.5)
    ref.assert_attention_close(out, expected, bound, dtype)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("splits", [1, 2])
def test_nan_tokens_and_bad_pages_among_values_far_apart(dim, splits):
    from nml_b200 import _abi
    lengths, table, cache, query, _, offsets = make(31, torch.bfloat16, dim, 2, 8, [100, 30],
                                                    [30, 0])
    cache[3][table[0, 1]] -= 20
    cache[3][table[1, 0]] += 15
    for token, at in ((70, 0), (90, 2)):  # a key row of head 0, a value row of head 1
        page, slot = int(table[0, token // 16]), token % 16
        cache[at][page, 0 if at == 0 else 1, slot] = 0x7f
    query[3, 2, 1] = float("nan")
    expected, bound = ref.attention(torch.nan_to_num(query), cache, table, lengths, offsets, None,
                                    0, 0, dim ** -0.5)
    expected[3, 2] = float("nan")
    out = call(query, cache, table, lengths, offsets, None, splits=splits)
    assert status() == 0
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)
    # rows in front of the first token, and a page of nobody in the middle of the walk
    table[0, 3] = -1
    out = call(query, cache, table, [lengths[0], 12], offsets, None, splits=splits)
    assert status() == _abi.STATUS_INDEX_RANGE
    assert (out[100:118] == 0).all() and torch.isfinite(out[118:]).all()
    # rows 0 to 17 see the tokens in front of that page only
    ref.assert_attention_close(out[:18], expected[:18], bound[:18], torch.bfloat16)


@pytest.mark.parametrize("runs", [False, True])
@pytest.mark.parametrize("window", [0, 30])
def test_tables_wider_than_the_sequences(runs, window):
    """Entries behind a sequence's last page are not read, whatever they hold; the library chooses
    splits for the table's width."""
    new, before = ([30, 1, 7], [200, 20, 0]) if runs else ([1, 1, 1], [229, 20, 6])
    lengths, table, cache, query, sinks, offsets = make(32, torch.bfloat16, 64, 2, 8, new, before,
                                                        with_sinks=True)
    wide = torch.full((3, 4096), -7, dtype=torch.int32)
    wide[:, 1000:] = 2 ** 31 - 1
    for b, length in enumerate(lengths):
        pages = -(-length // 16)
        wide[b, :pages] = table[b, :pages]
    out = call(query, cache, wide, lengths, offsets if runs else None, sinks,
               sliding_window=window or None, first_tokens=3)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, window, 3, 0.125)
    ref.assert_attention_close(out, expected, bound, torch.bfloat16)


@pytest.mark.parametrize("chunk", [60, 150])
def test_single_tokens_and_a_chunk_in_one_call(chunk):
    """A chunk of a prompt among the single tokens of a batch: by rows or by tiles as a whole."""
    new = [1] * 20 + [chunk] + [1] * 11
    before = [(37 * i) % 300 for i in range(32)]
    lengths, table, cache, query, sinks, offsets = make(33, torch.float16, 64, 1, 8, new, before,
                                                        with_sinks=True)
    out = call(query, cache, table, lengths, offsets, sinks, sliding_window=128)
    assert status() == 0
    expected, bound = ref.attention(query, cache, table, lengths, offsets, sinks, 128, 0, 0.125)
    ref.assert_attention_close(out, expected, bound, torch.float16)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_captured_step_follows_its_buffers(dim):
    """Append and attention captured once, replayed while lengths, pages and rows change in place: a
    place is taken, freed and taken again, a block grows, splits have nothing to do at first."""
    from nml_b200 import ops
    gen = torch.Generator().manual_seed(34)
    dtype, kv_heads, group, batch, width = torch.bfloat16, 2, 8, 3, 40
    heads, pages = kv_heads * group, batch * width
    start = ref.random_cache(gen, pages, kv_heads, dim)
    dev = [x.cuda() for x in start]
    table = torch.randperm(pages, generator=gen).view(batch, width).to(torch.int32)
    rotary = ops.rotary_table(10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / dim), 700)
    fused = torch.zeros((batch, heads + 2 * kv_heads, dim), dtype=dtype, device="cuda")
    dev_table, dev_lengths = table.cuda(), torch.zeros(batch, dtype=torch.int32, device="cuda")
    dev_rotary = rotary.cuda()

    def step():
        query = ops.paged_append_q8(fused[:, heads:heads + kv_heads], fused[:, heads + kv_heads:],
                                    *dev, dev_table, dev_lengths, query=fused[:, :heads],
                                    rotary=dev_rotary)
        return query, ops.paged_attention_q8(query, *dev, dev_table, dev_lengths, splits=4)

    step()  # every place is empty: nothing is written
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        query, out = step()
    held = [x.clone() for x in start]
    for lengths in ([1, 0, 320], [2, 16, 321], [0, 17, 322], [3, 18, 0], [640, 1, 335]):
        rows = torch.randn(fused.shape, generator=gen) * 2.0 ** (max(lengths) % 5)
        fused.copy_(rows.to(dtype))
        dev_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        table = table.flip(0).contiguous()
        dev_table.copy_(table)
        graph.replay()
        assert status() == 0
        parts = rows.to(dtype).float()
        angles = rotary[torch.tensor(lengths).clamp(min=1) - 1]
        offsets = [0, 1, 2, 3]
        key = ref.rotate(parts[:, heads:heads + kv_heads], angles, "half").double()
        held = [*ref.append(key, held[0], held[1], table, lengths, offsets),
                *ref.append(parts[:, heads + kv_heads:].double(), held[2], held[3], table, lengths,
                            offsets)]
        for got, want in zip(dev, held):
            assert torch.equal(got.cpu(), want)
        expected, bound = ref.attention(query.cpu(), held, table, lengths, offsets, None, 0, 0,
                                        dim ** -0.5)
        ref.assert_attention_close(out, expected, bound, dtype)
        for b in range(batch):
            assert lengths[b] or (out[b] == 0).all()
