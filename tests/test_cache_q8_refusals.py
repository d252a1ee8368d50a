"""What the 8-bit cache operators refuse, before any device call."""
import ctypes

import pytest
import torch

from nml_b200 import _abi, ops

FAKE = 0x1000  # never dereferenced: validation fails before any launch


def cache(**overrides):
    fields = dict(key=FAKE, key_scales=FAKE, value=FAKE, value_scales=FAKE, page_table=FAKE,
                  sequence_lengths=FAKE, batch=2, kv_heads=2, head_dim=64, page_size=16,
                  physical_pages=9, table_width=4)
    fields.update(overrides)
    return _abi.CacheQ8(**fields)


BAD_CACHES = [dict(key=None), dict(value=None), dict(key_scales=None), dict(value_scales=None),
              dict(page_table=None), dict(key=FAKE + 8), dict(value=FAKE + 4), dict(batch=0),
              dict(kv_heads=0), dict(head_dim=96), dict(page_size=32), dict(physical_pages=0),
              dict(table_width=0), dict(table_width=2 ** 28), dict(batch=2 ** 31)]


def append_request(cache_fields=None, **overrides):
    fields = dict(key=FAKE, value=FAKE, query=FAKE, query_output=FAKE + 4096, stream=FAKE, tokens=2,
                  query_heads=16, key_token_stride=128, key_head_stride=64,
                  value_token_stride=128, value_head_stride=64, query_token_stride=1024,
                  query_head_stride=64, output_token_stride=1024, output_head_stride=64,
                  dtype=_abi.BF16)
    fields.update(overrides)
    return _abi.PagedAppendQ8(cache=cache(**(cache_fields or {})), **fields)


def read_request(cache_fields=None, **overrides):
    fields = dict(token_offsets=FAKE, key_output=FAKE, value_output=FAKE, stream=FAKE, tokens=5,
                  dtype=_abi.F16)
    fields.update(overrides)
    return _abi.PagedReadQ8(cache=cache(**(cache_fields or {})), **fields)


def attention_request(cache_fields=None, **overrides):
    fields = dict(query=FAKE, output=FAKE, stream=FAKE, tokens=2, query_heads=16,
                  query_token_stride=1024, query_head_stride=64, scale=0.125, splits=1,
                  dtype=_abi.BF16)
    fields.update(overrides)
    return _abi.PagedAttentionQ8(cache=cache(**(cache_fields or {})), **fields)


def refused(name, request, text="invalid"):
    with pytest.raises(_abi.NvFp4Error) as error:
        _abi.call(name, request)
    assert error.value.code == _abi.INVALID_ARGUMENT
    assert text in error.value.message


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches(bad):
    for name, request in (("nml_sm100_paged_append_q8", append_request),
                          ("nml_sm100_paged_read_q8", read_request),
                          ("nml_sm100_paged_attention_q8", attention_request)):
        refused(name, request(bad))


@pytest.mark.parametrize("bad", [
    dict(key=None), dict(value=None), dict(stream=None), dict(tokens=0), dict(tokens=3),
    dict(key=FAKE + 2), dict(key_token_stride=100), dict(value_head_stride=-64),
    dict(query_output=None), dict(query_output=FAKE), dict(query_heads=0),
    dict(query_token_stride=1)])
def test_bad_appends(bad):
    refused("nml_sm100_paged_append_q8", append_request(**bad))


def test_append_refusals_that_say_why():
    name = "nml_sm100_paged_append_q8"
    refused(name, append_request(dict(sequence_lengths=None)))
    refused(name, append_request(dtype=7), "F16 and BF16 only")
    for width, table, rows in ((24, FAKE, 9), (80, FAKE, 9), (16, FAKE + 4, 9), (0, FAKE, 9),
                               (16, FAKE, 0)):
        refused(name, append_request(rotary=table, rotary_dim=width, rotary_rows=rows),
                "rotary width")


@pytest.mark.parametrize("bad", [dict(token_offsets=None), dict(key_output=None),
                                 dict(value_output=FAKE + 2), dict(stream=None), dict(tokens=0)])
def test_bad_reads(bad):
    refused("nml_sm100_paged_read_q8", read_request(**bad))
    refused("nml_sm100_paged_read_q8", read_request(dtype=0), "F16 and BF16 only")


@pytest.mark.parametrize("bad", [
    dict(query=None), dict(output=None), dict(stream=None), dict(tokens=0), dict(tokens=3),
    dict(query_heads=15), dict(query_heads=2 * 129), dict(query=FAKE + 8), dict(output=FAKE + 8),
    dict(query_token_stride=12), dict(query_head_stride=-8), dict(splits=65), dict(splits=-1),
    dict(sliding_window=-1), dict(first_tokens=-1), dict(scale=0.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(workspace=FAKE + 4)])
def test_bad_attention(bad):
    refused("nml_sm100_paged_attention_q8", attention_request(**bad))


def test_attention_scratch():
    name = "nml_sm100_paged_attention_q8"
    size = _abi.load().nml_sm100_paged_attention_q8_workspace_bytes

    def ask(**fields):
        request = attention_request(**fields)
        request.struct_size = ctypes.sizeof(request)
        return size(ctypes.byref(request))

    refused(name, attention_request(dtype=9), "F16 and BF16 only")
    assert ask(splits=1) == 0
    assert ask(splits=4) >= 2 * 16 * 4 * 68 * 4
    refused(name, attention_request(splits=4), "workspace is too small")
    refused(name, attention_request(splits=4, workspace=FAKE, workspace_bytes=1000),
            "workspace is too small")
    assert ask(tokens=0) == 0 and size(None) == 0


def tensors(**overrides):
    fields = dict(key_cache=torch.zeros((4, 2, 16, 64), dtype=torch.uint8),
                  key_scales=torch.zeros((4, 2), dtype=torch.uint8),
                  value_cache=torch.zeros((4, 2, 16, 64), dtype=torch.uint8),
                  value_scales=torch.zeros((4, 2), dtype=torch.uint8),
                  page_table=torch.zeros((1, 3), dtype=torch.int32),
                  sequence_lengths=torch.ones(1, dtype=torch.int32))
    fields.update(overrides)
    return fields


def test_operators_refuse_cpu_tensors():
    rows = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.paged_append_q8(rows, rows, **tensors())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.paged_attention_q8(rows, **tensors())
    fields = tensors()
    fields.pop("sequence_lengths")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.paged_read_q8(**fields, token_offsets=torch.zeros(2, dtype=torch.int32), tokens=1)


@pytest.mark.parametrize("bad", [
    dict(key_cache=torch.zeros((4, 2, 16, 64), dtype=torch.int8)),
    dict(value_cache=torch.zeros((4, 2, 16, 32), dtype=torch.uint8)),
    dict(key_scales=torch.zeros((4, 3), dtype=torch.uint8)),
    dict(value_scales=torch.zeros((4, 2), dtype=torch.float32)),
    dict(page_table=torch.zeros((1, 3), dtype=torch.int64)),
    dict(page_table=torch.zeros(3, dtype=torch.int32)),
    dict(sequence_lengths=torch.ones(2, dtype=torch.int32)),
    dict(sequence_lengths=torch.ones(1, dtype=torch.int64)),
    dict(key_cache=torch.zeros((4, 16, 2, 64), dtype=torch.uint8).transpose(1, 2)),
])
def test_cache_tensors_are_checked(bad):
    # the checks themselves need no device
    with pytest.raises(ValueError):
        ops._cache_q8(**tensors(**bad), device=torch.device("cpu"))


def test_row_tensors_are_checked():
    cpu = torch.device("cpu")

    def check(x, heads=2):
        return ops._head_rows(x, "keys", x.shape[0], heads, 64, torch.bfloat16, cpu)

    wide = torch.zeros((5, 8, 64), dtype=torch.bfloat16)
    assert check(wide[:, 2:4]) == (512, 64)
    assert check(wide.transpose(0, 1)[:, :2].transpose(0, 1)[:2].transpose(0, 1), 2)[0] >= 0
    for bad in (wide[:, :2].float(), wide[:, :3], wide[:, :2, ::2],
                torch.zeros(5 * 2 * 64 + 1, dtype=torch.bfloat16)[1:].view(5, 2, 64),
                torch.zeros((5, 2 * 64 + 4), dtype=torch.bfloat16)[:, :128].unflatten(1, (2, 64))):
        with pytest.raises(ValueError):
            check(bad)
    offsets = torch.zeros(3, dtype=torch.int32)
    ops._row_offsets(offsets, 2, 7, cpu)
    for arguments in ((None, 2, 7, cpu), (offsets.long(), 2, 7, cpu), (offsets, 3, 7, cpu),
                      (offsets, 2, 7, torch.device("cuda", 0))):
        with pytest.raises(ValueError):
            ops._row_offsets(*arguments)


def test_rotary_table():
    frequencies = torch.tensor([1.0, 0.01], dtype=torch.float64)
    table = ops.rotary_table(frequencies, 100001, 2.0)
    assert table.shape == (100001, 4) and table.dtype == torch.float32
    angle = 100000 * frequencies
    want = 2 * torch.cat((angle.cos(), angle.sin()))
    assert ((table[-1].double() - want).abs() <= 2.0 ** -23).all()
    for bad in (torch.zeros((2, 2)), torch.zeros(0)):
        with pytest.raises(ValueError):
            ops.rotary_table(bad, 4)
    with pytest.raises(ValueError):
        ops.rotary_table(frequencies, 0)


def test_tables_whose_positions_would_pass_32_bits():
    for name, request in (("nml_sm100_paged_append_q8", append_request),
                          ("nml_sm100_paged_read_q8", read_request),
                          ("nml_sm100_paged_attention_q8", attention_request)):
        refused(name, request(dict(table_width=2 ** 27 - 64)))


def test_scratch_of_more_heads_than_32_bits_is_not_computed():
    request = attention_request(dict(kv_heads=2 ** 40), query_heads=2 ** 40)
    request.struct_size = ctypes.sizeof(request)
    assert _abi.load().nml_sm100_paged_attention_q8_workspace_bytes(ctypes.byref(request)) == 0
