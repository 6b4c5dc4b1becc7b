"""The 8-bit cache on the host: refusals before any launch, in Python and at the C entries, and the plain forms against direct statements."""

import ctypes
import math

import pytest
import torch

import plain_quantized as plain
import vllm_rlt_b200 as rlt
from vllm_rlt_b200 import _capi


def cache(pages=4, block=16, heads=2, dim=64, **kw):
    return rlt.QuantizedKV.allocate(pages, block, heads, dim, device="cpu", **kw)


def step(n=2, width=2, lengths=(5, 9), counts=(1, 2)):
    return (torch.zeros(n, width, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), torch.tensor(plain.starts_of(counts), dtype=torch.int32))


def rows(n=3, heads=2, dim=64, dtype=torch.bfloat16):
    return torch.zeros(n, heads, dim, dtype=dtype)


def test_allocate_makes_one_block_of_keys_and_values():
    c = cache()
    assert c.key.shape == (4, 16, 2, 64) and c.key.dtype == torch.float8_e4m3fn and c.key_scale.shape == (4, 2)
    assert c.value.data_ptr() - c.key.data_ptr() == c.key.numel()
    c.check()


@pytest.mark.parametrize("broken, match", [
    (lambda c: rlt.QuantizedKV(c.key.view(torch.uint8), c.value, c.key_scale, c.value_scale), "float8"),
    (lambda c: rlt.QuantizedKV(c.key, c.value[:2], c.key_scale, c.value_scale), "layout"),
    (lambda c: rlt.QuantizedKV(c.key.transpose(1, 2), c.value.transpose(1, 2), c.key_scale, c.value_scale), "tail"),
    (lambda c: rlt.QuantizedKV(c.key, c.value, c.key_scale.double(), c.value_scale), "scales"),
    (lambda c: rlt.QuantizedKV(c.key, c.value, c.key_scale[:, :1], c.value_scale[:, :1]), "scales"),
    (lambda c: rlt.QuantizedKV.allocate(2, 16, 2, 257, device="cpu"), "dim"),
    (lambda c: rlt.QuantizedKV.allocate(2, 0, 2, 64, device="cpu"), "tokens"),
])
def test_a_cache_of_another_form_is_refused(broken, match):
    bad = broken(cache())
    tables, lengths, cu = step()
    with pytest.raises(ValueError, match=match):
        rlt.quantized_kv_write(bad, rows(), rows(), tables, lengths, cu)
    with pytest.raises(ValueError, match=match):
        rlt.quantized_attention(rows(), bad, tables, lengths, cu, 2)


def test_steps_of_another_form_are_refused():
    tables, lengths, cu = step()
    c = cache()
    for t, l, b in ((tables.long(), lengths, cu), (tables, lengths.long(), cu), (tables, lengths[:1], cu), (tables, lengths, cu[:2]),
                    (tables.t(), lengths, cu), (tables, lengths, cu.long())):
        with pytest.raises(ValueError, match="int32"):
            rlt.quantized_kv_write(c, rows(), rows(), t, l, b)
        with pytest.raises(ValueError, match="int32"):
            rlt.quantized_attention(rows(), c, t, l, b, 2)
    for k, v in ((rows(heads=1), rows(heads=1)), (rows(), rows(2)), (rows(), rows(dtype=torch.float16)), (rows(dtype=torch.float64),) * 2):
        with pytest.raises(ValueError, match="k and v"):
            rlt.quantized_kv_write(c, k, v, tables, lengths, cu)
    with pytest.raises(ValueError, match="tail"):
        rlt.quantized_kv_write(c, rows().transpose(1, 2).contiguous().transpose(1, 2), rows(), tables, lengths, cu)
    for q in (rows(dim=32), rows(heads=3), rows(dtype=torch.float64)):
        with pytest.raises(ValueError, match="q must be"):
            rlt.quantized_attention(q, c, tables, lengths, cu, 2)
    for bad in (dict(window=-1), dict(window=True), dict(window=1.0)):
        with pytest.raises(ValueError, match="window"):
            rlt.quantized_attention(rows(), c, tables, lengths, cu, 2, **bad)
    with pytest.raises(ValueError, match="max_new"):
        rlt.quantized_attention(rows(), c, tables, lengths, cu, -1)
    # what is in order reaches the device, and there is no fallback behind it
    with pytest.raises(ValueError, match="CUDA"):
        rlt.quantized_attention(rows(), c, tables, lengths, cu, 2)
    with pytest.raises(ValueError, match="CUDA"):
        rlt.quantized_kv_write(c, rows(), rows(), tables, lengths, cu)


def test_slots_of_another_form_are_refused():
    tables, lengths, _ = step()
    counts, held, free, count = lengths.clone(), lengths.clone(), lengths.clone(), torch.ones(1, dtype=torch.int32)
    for bad in (dict(held=held), dict(held=held, free_pages=free), dict(free_count=count)):
        with pytest.raises(ValueError, match="together"):
            rlt.step_slots(lengths, counts, tables, 16, 8, **bad)
    whole = dict(held=held, free_pages=free, free_count=count)
    for name, t in (("held", held.long()), ("held", held[:1]), ("free_count", count.long()), ("free_count", torch.ones(2, dtype=torch.int32)),
                    ("free_pages", free.long()), ("free_pages", free[None])):
        with pytest.raises(ValueError, match=name):
            rlt.step_slots(lengths, counts, tables, 16, 8, **{**whole, name: t})
        with pytest.raises(ValueError, match=name):
            rlt.return_pages(lengths, tables, 16, **{**whole, name: t})
    for block, count_rows in ((0, 8), (16, -1)):
        with pytest.raises(ValueError, match="block"):
            rlt.step_slots(lengths, counts, tables, block, count_rows)
    with pytest.raises(ValueError, match="counts"):
        rlt.step_slots(lengths, counts[:1], tables, 16, 8)
    with pytest.raises(ValueError, match="CUDA"):
        rlt.step_slots(lengths, counts, tables, 16, 8, **whole)


def test_the_c_entries_refuse_without_a_launch():
    """Sizes that no kernel takes come back as a status, from addresses that are never followed."""
    lib = _capi.load()
    at = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(at) + (-ctypes.addressof(at)) % 256
    null = None

    def write(pages=4, block=16, heads=2, dim=64, token=128, page=2048, scale=2, dtype=2, sequences=1, width=2, rows=1, k=p, k_stride=128, key=p):
        return lib.rlt_quantized_kv_write(key, p, p, p, page, token, scale, pages, block, heads, dim, k, k_stride, p, k_stride, dtype, p, p, p, sequences,
                                          width, rows, null)

    assert write(rows=0) == write(sequences=0) == write(width=0) == _capi.OK
    for bad in (dict(dtype=3), dict(dim=257), dict(dim=0), dict(block=0), dict(heads=0), dict(token=127), dict(page=2047), dict(scale=1), dict(rows=-1),
                dict(width=-1), dict(k=null), dict(key=null), dict(k_stride=127), dict(width=1 << 27)):
        assert write(**bad) == _capi.ERR_INVALID, bad

    def attend(heads=4, kv=2, dim=64, width=2, rows=1, window=0, max_new=1, stride=256, ws=p, nbytes=0, block=16, sequences=1, dtype=2):
        return lib.rlt_quantized_attention(p, stride, p, stride, p, p, p, p, block * kv * dim, kv * dim, kv, 4, block, heads, kv, dim, dtype, p, p, p,
                                           sequences, width, rows, max_new, 1.0, window, ws, nbytes, null)

    assert attend(rows=0) == attend(sequences=0) == _capi.OK
    for bad in (dict(heads=3), dict(heads=0), dict(dim=257), dict(width=0), dict(width=(1 << 22) + 1), dict(window=-1), dict(max_new=-1), dict(stride=255),
                dict(dtype=7), dict(rows=-1)):
        assert attend(**bad) == _capi.ERR_INVALID, bad
    def bytes_of(rows=1, sequences=1, max_new=1, heads=4, kv=2, dim=64, block=16, width=1000, window=0, dtype=2):
        return lib.rlt_quantized_attention_workspace_bytes(rows, sequences, max_new, heads, kv, dim, block, width, window, dtype)

    need = bytes_of()
    assert need == 4 * 10 * 4 * (64 + 4)                              # four parts of 1024 tokens and six of 2048
    assert bytes_of(width=64) == bytes_of(window=1) == bytes_of(window=1900) == bytes_of(rows=0) == bytes_of(sequences=0) == 0
    assert bytes_of(window=1901) == 4 * 3 * 4 * (64 + 4)
    long = dict(rows=256, max_new=256, heads=32)
    parts = 256 * 32 * 10 * 4 * (64 + 4)
    assert bytes_of(**long) > 2 * 16000 * 2 * 64 * 2 + parts          # and 16000 expanded tokens
    for short in (dict(max_new=16), dict(dtype=1), dict(dtype=0), dict(sequences=5), dict(sequences=65536), dict(dim=65 + 31), dict(block=8, width=2000),
                  dict(heads=30), dict(heads=32, kv=32, rows=127)):
        given = dict(long, **short)
        assert bytes_of(**given) == 4 * given["rows"] * given["heads"] * 10 * (given.get("dim", 64) + 4), short
    assert bytes_of(**long, window=5) == 0 and bytes_of(**long, window=3000) == 4 * 256 * 32 * 4 * (64 + 4)
    wide = dict(long, width=1 << 22, heads=64, kv=1, dim=128)         # 2^26 tokens are not expanded
    a_row = 4 * 64 * (4 + (1 << 15) - 2) * 132
    assert bytes_of(**wide) == (2 << 30) // a_row * a_row             # rows whose parts fit in 2 GB are done at a time
    assert attend(width=1000, nbytes=need - 1) == _capi.ERR_WORKSPACE
    assert attend(width=1000, nbytes=need, ws=p + 4) == _capi.ERR_WORKSPACE
    assert attend(width=1000, nbytes=need, ws=null) == _capi.ERR_WORKSPACE

    def slots(n=1, width=2, block=16, rows=1, held=p, free=p, capacity=4, count=p, cu=p):
        return lib.rlt_step_slots(p, p, n, p, width, block, held, free, capacity, count, rows, cu, p, p, p, p, p, p, p, null)

    for bad in (dict(n=8193), dict(n=-1), dict(block=0), dict(rows=-1), dict(capacity=-1), dict(free=null), dict(count=null), dict(cu=null), dict(width=1 << 27)):
        assert slots(**bad) == _capi.ERR_INVALID, bad
    for bad in (dict(n=8193), dict(block=0), dict(count=null)):
        given = dict(dict(n=1, block=16, count=p), **bad)
        assert lib.rlt_return_pages(p, given["n"], p, 2, given["block"], p, p, 4, given["count"], p, null) == _capi.ERR_INVALID, bad


def test_plain_codes_and_scales():
    x = torch.tensor([0.0, 448.0, 449.0, 1e9, -464.1, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9, 1.0625, 1.1875, math.nan], dtype=torch.float64)
    got = plain.nearest_code(x)
    assert got[:10].tolist() == [0.0, 448.0, 448.0, 448.0, -448.0, 0.0, 2.0 ** -8, 2.0 ** -9, 1.0, 1.25] and got[10].isnan()
    near = (torch.rand(4000, generator=torch.Generator().manual_seed(0)) * 900 - 450).double()
    assert torch.equal(plain.nearest_code(near), near.clamp(-448, 448).float().to(torch.float8_e4m3fn).double())
    assert [plain.exponent(v) for v in (448.0, 448.1, 1.0, 0.0, 1e-40, 1e38)] == [0, 1, -8, -100, -100, 100]
    assert [plain.exponent_above(v) for v in (1.0, 1.5, 2.0, 0.75)] == [0, 1, 1, 0]


def test_plain_pages_go_back_where_they_came_from():
    tables = [[5, 6, 0, 0], [7, 0, 0, 0], [0, 0, 0, 0]]
    held, free, count, lengths = [2, 1, 0], [1, 2, 3, 4, 9], [4], [32, 10, 0]
    got = plain.step_slots(lengths, [1, 3, 20], tables, 16, 30, held, free, count)
    assert got[0] == [0, 1, 4, 24] and tables == [[5, 6, 4, 0], [7, 0, 0, 0], [3, 2, 0, 0]] and held == [3, 1, 2] and count == [1]
    assert got[4][:5] == [4, 7, 7, 7, 3] and got[5][:5] == [0, 10, 11, 12, 0] and got[3][24:] == [-1] * 6
    assert plain.return_pages(lengths, tables, 16, held, free, count) == 0
    assert held == [2, 1, 0] and count == [4] and free == [1, 2, 3, 4, 9]
    assert plain.step_slots(lengths, [1, 3, 80], tables, 16, 200, held, free, count)[-1] == 1        # beyond the table
    assert plain.step_slots(lengths, [32, 30, 30], tables, 16, 200, held, free, count)[-1] == 1      # five pages, four free
    assert plain.step_slots(lengths, [1, 3, 20], tables, 16, 23, held, free, count)[-1] == 1         # a row too many
