"""The decode model over the 8-bit cache: prompts in chunks, then single tokens, through the model's
own entry points; what its first layer caches is checked against the projection of the embeddings."""
import pytest
import torch
import torch.nn.functional as F

import cache_q8_reference as ref

pytestmark = pytest.mark.gpu


def small_shape():
    from nml_b200.decode_step import GptOssShape
    return GptOssShape(layers=2, hidden=256, intermediate=128, query_heads=16, key_value_heads=2,
                       experts=4, experts_per_token=2, vocabulary=1000)


def test_prompts_then_tokens():
    from nml_b200 import _abi, ops
    from nml_b200.decode_step import DecodeModel
    shape = small_shape()
    model = DecodeModel(shape, 3, 0, torch.device("cuda"), cache="e4m3", room=80)
    gen = torch.Generator(device="cuda").manual_seed(3)
    given = [[], [], []]
    for counts in ([40, 1, 17], [9, 20, 0], None, None):
        new = [1, 1, 1] if counts is None else counts
        tokens = torch.randint(0, shape.vocabulary, (sum(new),), device="cuda", generator=gen,
                               dtype=torch.int32)
        out = model.extend(tokens, counts)
        assert out.shape == (sum(new),) and int(out.min()) >= 0
        assert int(out.max()) < shape.vocabulary
        for b, part in enumerate(tokens.split(new)):
            given[b] += part.tolist()
    torch.cuda.synchronize()
    assert _abi.device_status(0x1) == 0
    assert model.cached == [51, 23, 19]
    # layer 0's keys and values follow from the embeddings alone
    layer = model.layers[0]
    key, key_scales, value, value_scales = (x.cpu() for x in layer["cache"])
    table = model.page_table.cpu()
    for b, ids in enumerate(given):
        hidden = ops.token_embedding(model.table, torch.tensor(ids, dtype=torch.int32).cuda())
        x = F.rms_norm(hidden, (shape.hidden,), layer["input_norm"], shape.rms_norm_eps)
        heads = (len(ids), shape.key_value_heads, shape.head_dim)
        # the projections of a row do not depend on its batch beyond the order of f32 sums: one
        # step of the result's type, 2^-7 of it or of the largest products' sum, is allowed beside
        # half a code step (2^-4; two roundings where a block has grown)
        for name, codes, scales in (("k", key, key_scales), ("v", value, value_scales)):
            rows = ops.linear(x, layer[name], layer[name + "_bias"]).view(heads).cpu().double()
            slack = rows.abs().amax(-1, keepdim=True) * 2.0 ** -7
            if name == "k":
                rows = ref.rotate(rows, model.rotary[: len(ids)].cpu(), "half")
                slack = slack * 2 * model.attention_factor
            held, _, exponent = ref.gather(codes, scales, table[b], len(ids))
            limit = rows.abs() * 2.0 ** -4 * 1.07 + slack + \
                2 * 2.0 ** -10 * torch.exp2(exponent)[..., None]
            assert ((held - rows).abs() <= limit).all()


def test_a_step_over_either_cache():
    """The benchmark's step: both caches hold random prior tokens, the step runs and can be
    captured into a graph that gives the same tokens again."""
    from nml_b200 import _abi
    from nml_b200.decode_step import DecodeModel
    for cache in ("bf16", "e4m3"):
        model = DecodeModel(small_shape(), 4, 70, torch.device("cuda"), cache=cache)
        eager = model.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.step()
        graph.replay()
        torch.cuda.synchronize()
        assert _abi.device_status(0x1) == 0
        assert torch.equal(out, eager)


def test_extend_refusals():
    from nml_b200.decode_step import DecodeModel
    device = torch.device("cuda")
    with pytest.raises(ValueError):
        DecodeModel(small_shape(), 2, 0, device, cache="fp4")
    with pytest.raises(ValueError):
        DecodeModel(small_shape(), 2, 0, device, cache="e4m3", room=0)
    tokens = torch.zeros(40, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        DecodeModel(small_shape(), 2, 0, device).extend(tokens[:2])
    model = DecodeModel(small_shape(), 2, 0, device, cache="e4m3", room=20)
    for count, counts in ((2, [1]), (2, [3, -1]), (3, [1, 1]), (0, [0, 0]), (40, [33, 7])):
        with pytest.raises(ValueError):
            model.extend(tokens[:count], counts)
    assert model.cached == [0, 0]


def test_a_step_behind_extended_tokens_is_refused():
    """The step's position would be one of theirs: nothing of the cache changes."""
    from nml_b200.decode_step import DecodeModel
    device = torch.device("cuda")
    for prior in (0, 9):
        model = DecodeModel(small_shape(), 2, prior, device, cache="e4m3", room=60)
        model.step()  # before any token is kept it is what it was
        tokens = torch.arange(23, dtype=torch.int32, device=device)
        model.extend(tokens, [20, 3])
        held = [[x.clone() for x in layer["cache"]] for layer in model.layers]
        with pytest.raises(ValueError, match="extend"):
            model.step()
        torch.cuda.synchronize()
        for layer, before in zip(model.layers, held):
            assert all(torch.equal(a, b) for a, b in zip(layer["cache"], before))
        model.extend(tokens[:2])
        assert model.cached == [prior + 21, prior + 4]
        with pytest.raises(ValueError):
            model.extend(tokens[:4].view(2, 2), [2, 2])


def test_attention_of_every_layer_against_the_definition():
    """What each layer writes and attends to, by the layer's own sinks and window and by lengths that
    the test counts itself, against the 64-bit definition over the cache that the layer leaves."""
    from nml_b200 import _abi
    from nml_b200.decode_step import DecodeModel
    shape = small_shape()
    assert shape.sliding_window == 128
    model = DecodeModel(shape, 3, 0, torch.device("cuda"), cache="e4m3", room=260)
    seen = []
    inner = model._append_and_attend

    def record(layer, q, k, v, lengths, offsets):
        held = [x.cpu() for x in layer["cache"]]
        out = inner(layer, q, k, v, lengths, offsets)
        seen.append((layer, q.cpu(), k.cpu(), v.cpu(), held, [x.cpu() for x in layer["cache"]],
                     out.cpu()))
        return out

    model._append_and_attend = record
    gen = torch.Generator(device="cuda").manual_seed(5)
    table, cached = model.page_table.cpu(), [0, 0, 0]
    heads, kv_heads, dim = shape.query_heads, shape.key_value_heads, shape.head_dim
    for counts in ([190, 1, 140], [40, 30, 0], None, None):
        new = [1, 1, 1] if counts is None else counts
        tokens = torch.randint(0, shape.vocabulary, (sum(new),), device="cuda", generator=gen,
                               dtype=torch.int32)
        seen.clear()
        model.extend(tokens, counts)
        torch.cuda.synchronize()
        assert _abi.device_status(0x1) == 0
        lengths, offsets = [m + n for m, n in zip(cached, new)], ref.offsets_of(new)
        position = torch.cat([torch.arange(n) + m for n, m in zip(new, cached)])
        angles = model.rotary.cpu()[position]
        assert [id(x[0]) for x in seen] == [id(layer) for layer in model.layers]
        for index, (layer, q, k, v, before, after, out) in enumerate(seen):
            rows = [x.view(sum(new), -1, dim).float() for x in (q, k, v)]
            written = [*ref.append(ref.rotate(rows[1], angles, "half").double(), before[0], before[1],
                                   table, lengths, offsets),
                       *ref.append(rows[2].double(), before[2], before[3], table, lengths, offsets)]
            for got, want in zip(after, written):
                assert torch.equal(got, want)
            query = ref.rotate(rows[0], angles, "half").to(torch.bfloat16)
            expected, bound = ref.attention(query, after, table, lengths, offsets,
                                            layer["sinks"].cpu(), 128 if index % 2 == 0 else 0, 0,
                                            dim ** -0.5)
            ref.assert_attention_close(out.view(sum(new), heads, dim), expected, bound,
                                       torch.bfloat16)
        cached = lengths
    assert model.cached == cached
    # the benchmark's step behind random prior tokens, where the window has left some behind
    model = DecodeModel(shape, 2, 150, torch.device("cuda"), cache="e4m3")
    inner = model._append_and_attend
    model._append_and_attend = record
    seen.clear()
    model.step()
    for index, (layer, q, _, _, _, after, out) in enumerate(seen):
        angles = model.rotary.cpu()[150].expand(2, -1)
        query = ref.rotate(q.view(2, heads, dim).float(), angles, "half").to(torch.bfloat16)
        expected, bound = ref.attention(query, after, model.page_table.cpu(), [151, 151], [0, 1, 2],
                                        layer["sinks"].cpu(), 128 if index % 2 == 0 else 0, 0,
                                        dim ** -0.5)
        ref.assert_attention_close(out.view(2, heads, dim), expected, bound, torch.bfloat16)
    assert len(seen) == 2
