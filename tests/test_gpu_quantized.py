"""Pages and slots of a step, the 8-bit cache and the attention over it, against plain float64 forms."""

import math
import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import plain_quantized as plain
import vllm_rlt_b200 as rlt

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---- pages and slots -----------------------------------------------------------------------------------
def check_slots(lengths, counts, block, width, rows, *, held=None, free=None, count=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = len(lengths)
    tables = torch.randint(0, 1000, (n, width), generator=g, dtype=torch.int32)
    want_tables, want_held, want_count = tables.tolist(), list(held) if held is not None else None, [count] if count is not None else None
    want = plain.step_slots(lengths, counts, want_tables, block, rows, want_held, free, want_count)
    dev = dict(lengths=plain.words(lengths).cuda(), counts=plain.words(counts).cuda(), tables=tables.cuda())
    state = {} if held is None else dict(held=plain.words(held).cuda(), free_pages=plain.words(free).cuda(), free_count=plain.words([count]).cuda())
    got = rlt.step_slots(dev["lengths"], dev["counts"], dev["tables"], block, rows, **state)
    for name, expected in zip(("cu", "lengths", "positions", "row_seq", "write_blocks", "write_offsets"), want):
        assert getattr(got, name).tolist() == expected, name
    assert int(got.active_rows) == want[6] and int(got.status) == want[7]
    assert got.write_blocks.dtype == got.write_offsets.dtype == torch.int64 and got.active_rows.dim() == 0
    assert dev["tables"].tolist() == want_tables and dev["lengths"].tolist() == list(lengths)
    if held is not None:
        assert state["held"].tolist() == want_held and state["free_count"].tolist() == want_count and state["free_pages"].tolist() == list(free)
        # and back: after a step that was refused there is nothing to give back that was not there before
        want_free = list(free)
        status = rlt.return_pages(dev["lengths"], dev["tables"], block, **state)
        assert int(status) == plain.return_pages(lengths, want_tables, block, want_held, want_free, want_count)
        assert state["held"].tolist() == want_held and state["free_count"].tolist() == want_count and state["free_pages"].tolist() == want_free
    return want[7]


@pytest.mark.parametrize("n, most, block, spare", [(1, 1, 16, 0), (3, 40, 16, 5), (64, 1, 16, 0), (33, 9, 7, 100), (200, 30, 64, 1), (1024, 5, 16, 3),
                                                   (1025, 4, 16, 0), (5, 3000, 16, 9), (8192, 1, 16, 0)])
def test_slots_and_claims_match_the_plain_form(n, most, block, spare):
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 300, (n,), generator=g).tolist()
    counts = torch.randint(-1 if n > 3 else 1, most + 1, (n,), generator=g).tolist()
    width = (300 + most) // block + 1
    rows = sum(max(c, 0) for c in counts) + spare
    assert check_slots(lengths, counts, block, width, rows) == 0
    held = [-(-a // block) + (i % 5 == 0 and -(-a // block) < width) for i, a in enumerate(lengths)]     # some hold a page more than they need
    need = sum(max(-(-(a + max(c, 0)) // block) - h, 0) for a, c, h in zip(lengths, counts, held))
    free = torch.randperm(need + 20, generator=g).tolist()
    assert check_slots(lengths, counts, block, width, rows, held=held, free=free, count=need + 7) == 0
    assert check_slots(lengths, counts, block, width, rows, held=held, free=free, count=need) == 0
    if need:
        assert check_slots(lengths, counts, block, width, rows, held=held, free=free, count=need - 1) == 1
    if rows:
        assert check_slots(lengths, counts, block, width, rows - spare - 1 if rows > spare else rows, held=held, free=free, count=need) == (rows > spare)


def test_steps_that_cannot_be_are_refused_as_a_whole():
    base = dict(held=[1, 2], free=[5, 6, 7], count=3)
    assert check_slots([3, 20], [1, 1], 16, 2, 4, **base) == 0
    assert check_slots([-1, 20], [1, 1], 16, 2, 4, **base) == 1
    assert check_slots([3, 20], [1, 13], 16, 2, 40, **base) == 1                   # one token beyond the table
    assert check_slots([3, 20], [1, 12], 16, 2, 40, **base) == 0
    assert check_slots([3, 20], [2 ** 31 - 1, 2 ** 31 - 1], 16, 2, 40, **base) == 1
    assert check_slots([3, 20], [1, 1], 16, 2, 4, **{**base, "held": [3, 2]}) == 1
    assert check_slots([3, 20], [1, 1], 16, 2, 4, **{**base, "held": [-1, 2]}) == 1
    assert check_slots([3, 20], [0, 0], 16, 2, 0, **base) == 0
    assert check_slots([3, 16], [1, 1], 16, 2, 4, **{**base, "held": [1, 1], "count": -4}) == 1
    assert check_slots([3, 16], [1, 1], 16, 2, 4, **{**base, "held": [1, 1], "count": 9}) == 1


def test_no_requests_and_pages_given_back_twice():
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    got = rlt.step_slots(empty, empty, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 16, 3)
    assert got.cu.tolist() == [0] and got.row_seq.tolist() == [-1] * 3 and int(got.status) == 0 and int(got.active_rows) == 0
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    held, free, count = plain.words([4, 4]).cuda(), torch.zeros(8, dtype=torch.int32, device="cuda"), plain.words([0]).cuda()
    lengths = plain.words([0, 0]).cuda()
    assert int(rlt.return_pages(lengths, tables, 16, held=held, free_pages=free, free_count=count)) == 0
    assert free.tolist() == [7, 6, 5, 4, 3, 2, 1, 0] and count.tolist() == [8] and held.tolist() == [0, 0]
    held.fill_(4)                                                                    # the same pages again: no room
    assert int(rlt.return_pages(lengths, tables, 16, held=held, free_pages=free, free_count=count)) == 1
    assert count.tolist() == [8] and held.tolist() == [4, 4]
    held.fill_(5)
    assert int(rlt.return_pages(lengths, tables, 16, held=held, free_pages=free, free_count=plain.words([0]).cuda())) == 1


# ---- storing --------------------------------------------------------------------------------------------
def layer_of(raw, scales, layer, device="cuda"):
    """The cache of one layer inside pools [2, pages, layers, ...]."""
    codes, scales = raw.to(device).view(plain.CODE), scales.to(device)
    return rlt.QuantizedKV(codes[0][:, layer], codes[1][:, layer], scales[0][:, layer], scales[1][:, layer]), codes, scales


def same_values(got, want):
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def pages_for(lengths, block, g, spare=2, width=None):
    """Tables with a page of its own for every entry in use, and how many pages there are."""
    need = [-(-max(a, 0) // block) for a in lengths]
    width = width or max(need + [1])
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for s, n in enumerate(need):
        for j in range(n):
            tables[s, j] = order.pop()
    return tables, sum(need) + spare


WRITES = [
    # heads, dim, block, lengths, counts
    (2, 128, 16, [1], [1]),
    (8, 128, 16, [17, 16, 32, 5], [1, 1, 1, 1]),
    (3, 64, 16, [40, 7, 0, 33], [25, 7, 0, 16]),
    (5, 80, 8, [30, 3, 9], [13, 1, 9]),
    (1, 33, 3, [10, 4], [7, 4]),
    (4, 8, 64, [130, 64, 65], [130, 1, 2]),
    (2, 256, 16, [20, 50], [9, 50]),
    (2, 16, 1, [4, 3], [2, 3]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, dim, block, lengths, counts", WRITES)
def test_stored_rows_match_the_plain_form(dtype, heads, dim, block, lengths, counts):
    g = torch.Generator().manual_seed(dim * block)
    tables, pages = pages_for(lengths, block, g)
    raw, scales = plain.make_cache(pages, block, heads, dim, g, layers=2)
    rows = sum(counts) + 3                                                           # three behind the last sequence
    size = torch.exp2(torch.randint(-12, 13, (rows, heads, 1), generator=g).float())
    k, v = ((torch.randn(rows, heads, dim, generator=g) * size).to(dtype) for _ in range(2))
    cu = plain.starts_of(counts)
    cache, codes, dev_scales = layer_of(raw, scales, 1)
    rlt.quantized_kv_write(cache, k.cuda(), v.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda())
    want = raw.view(plain.CODE).double()
    want_scales = scales.double()
    for i, x in enumerate((k, v)):
        plain.kv_write(want[i][:, 1], want_scales[i][:, 1], x.double(), tables, lengths, cu)
    assert torch.equal(dev_scales.cpu().double(), want_scales)
    # bytes of slots in front of a page's first new row and of other layers; the rest of a page that was started anew means nothing but stays
    assert same_values(codes.cpu().double(), want)


def test_rows_that_are_slices_of_wider_ones_and_odd_addresses():
    g = torch.Generator().manual_seed(3)
    heads, dim, block, lengths, counts = 2, 64, 16, [20, 9], [20, 2]
    tables, pages = pages_for(lengths, block, g)
    raw, scales = plain.make_cache(pages, block, heads, dim, g)
    wide = torch.randn(22, 3 * heads * dim + 1, generator=g).bfloat16()
    for shift in (0, 1):                                                             # 1: no vector loads
        k, v = (wide[:, shift + i * heads * dim:][:, :heads * dim].unflatten(1, (heads, dim)) for i in (0, 2))
        cache, codes, dev_scales = layer_of(raw, scales, 0)
        on = wide.cuda()
        dk, dv = (on[:, shift + i * heads * dim:][:, :heads * dim].unflatten(1, (heads, dim)) for i in (0, 2))
        rlt.quantized_kv_write(cache, dk, dv, tables.cuda(), plain.words(lengths).cuda(), plain.words([0, 20, 22]).cuda())
        want, want_scales = raw.view(plain.CODE).double(), scales.double()
        for i, x in enumerate((k, v)):
            plain.kv_write(want[i][:, 0], want_scales[i][:, 0], x.double(), tables, lengths, [0, 20, 22])
        assert torch.equal(dev_scales.cpu().double(), want_scales) and same_values(codes.cpu().double(), want)


def test_a_page_filled_token_by_token_grows_its_scale():
    """Rows of rising size, one call each: every growth rounds the page's codes again, and a page as a whole is what the plain form says."""
    g = torch.Generator().manual_seed(1)
    heads, dim, block = 2, 128, 16
    cache = rlt.QuantizedKV.allocate(3, block, heads, dim)
    tables = plain.words([[2, 0]])
    want, want_scales = torch.zeros(2, 3, block, heads, dim, dtype=torch.float64), torch.zeros(2, 3, heads, dtype=torch.float64)
    for t in range(24):
        x = (torch.randn(2, 1, heads, dim, generator=g) * 2.0 ** (t % 16 * 1.7 - 12)).bfloat16()
        rlt.quantized_kv_write(cache, x[0].cuda(), x[1].cuda(), tables.cuda(), plain.words([t + 1]).cuda(), plain.words([0, 1]).cuda())
        for i in range(2):
            plain.kv_write(want[i], want_scales[i], x[i].double(), tables, [t + 1], [0, 1])
    assert torch.equal(cache.key_scale.cpu().double(), want_scales[0]) and torch.equal(cache.value_scale.cpu().double(), want_scales[1])
    assert same_values(cache.key.cpu().double(), want[0]) and same_values(cache.value.cpu().double(), want[1])


def test_values_that_are_not_finite_zero_tiny_and_huge():
    heads, dim, block = 1, 32, 16
    tables, lengths, cu = plain.words([[0], [1], [2], [3]]), [1, 1, 1, 2], plain.starts_of([1, 1, 1, 2])
    x = torch.zeros(5, heads, dim)
    x[0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    x[1, 0, :3] = torch.tensor([3e38, -1e38, 1e25])                                  # beyond 448 * 2^100: saturated
    x[2] = 0
    x[3, 0, :2] = torch.tensor([1e-38, 2.0 ** -101])                                 # below the smallest scale's steps
    x[4, 0, 0] = math.nan
    for dtype in (torch.float32, torch.bfloat16):
        rows = x.to(dtype)
        cache = rlt.QuantizedKV.allocate(4, block, heads, dim)
        rlt.quantized_kv_write(cache, rows.cuda(), rows.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda())
        want, want_scales = torch.zeros(4, block, heads, dim, dtype=torch.float64), torch.zeros(4, heads, dtype=torch.float64)
        plain.kv_write(want, want_scales, rows.double(), tables, lengths, cu)
        assert torch.equal(cache.key_scale.cpu().double(), want_scales) and same_values(cache.key.cpu().double(), want)
        assert torch.equal(cache.value_scale, cache.key_scale)


def test_rows_without_a_place_are_not_stored():
    """Padding sequences of a captured step (length 0), pages outside the cache, rows beyond a table, rows behind the last sequence."""
    g = torch.Generator().manual_seed(2)
    heads, dim, block = 2, 64, 16
    raw, scales = plain.make_cache(3, block, heads, dim, g)
    tables = plain.words([[0, 1], [0, 0], [-1, 7], [2, 2]])
    lengths, cu = [18, 0, 17, 34], plain.starts_of([2, 1, 3, 3])                    # the third's pages do not exist; the fourth's last two rows lie behind its table
    k = torch.randn(12, heads, dim, generator=g).bfloat16()
    cache, codes, dev_scales = layer_of(raw, scales, 0)
    rlt.quantized_kv_write(cache, k.cuda(), -k.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda())
    want, want_scales = raw.view(plain.CODE).double(), scales.double()
    for i, x in enumerate((k, -k)):
        plain.kv_write(want[i][:, 0], want_scales[i][:, 0], x.double(), tables, lengths, cu)
    assert torch.equal(dev_scales.cpu().double(), want_scales) and same_values(codes.cpu().double(), want)
    before = codes.clone().view(torch.uint8)
    rlt.quantized_kv_write(cache, k[:0].cuda(), k[:0].cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words([0] * 5).cuda())
    rlt.quantized_kv_write(cache, k.cuda(), k.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words([0] * 5).cuda())
    assert torch.equal(before, codes.view(torch.uint8))


# ---- attention ------------------------------------------------------------------------------------------
def attention_case(heads, kv_heads, dim, block, lengths, counts, dtype, *, window=0, scale=None, seed=0, spare=2, width=None, strided=False):
    g = torch.Generator().manual_seed(seed + dim + block)
    tables, pages = pages_for(lengths, block, g, spare=3, width=width)
    raw, scales = plain.make_cache(pages, block, kv_heads, dim, g, layers=2)
    rows = sum(counts) + spare
    cu = plain.starts_of(counts)
    q = (torch.randn(rows, heads, dim, generator=g) * 0.1).to(dtype)
    codes = raw.view(plain.CODE).double()
    want, parts = plain.attention(q, (codes[0][:, 1], codes[1][:, 1]), (scales[0][:, 1].double(), scales[1][:, 1].double()), tables, lengths, cu,
                                  scale=scale, window=window, out=torch.full(q.shape, 7.0))
    # slots that no token was stored in: every byte NaN, and NaN scales for pages that nobody holds
    stored = torch.zeros(pages, block, dtype=torch.bool)
    for s, a in enumerate(lengths):
        for t in range(min(max(a, 0), tables.shape[1] * block)):
            stored[int(tables[s, t // block]), t % block] = True
    raw = torch.where(stored[None, :, None, :, None, None], raw, 0x7f)
    scales = torch.where(stored.any(1)[None, :, None, None], scales, math.nan)
    cache, _, _ = layer_of(raw, scales, 1)
    on = q.cuda()
    if strided:
        on = torch.cat((on, torch.full_like(on, math.nan)), 1)[:, :heads]
    call = (on, cache, tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda(), max(counts + [0]))
    return call, dict(window=window, scale=scale), want, parts


def is_expanded(call, options):
    """Whether a step's portions are long enough for pages expanded into bfloat16."""
    q, cache, tables, _, _, most = call
    block, kv_heads, dim = cache.key.shape[1:]
    rows, n, heads = q.shape[0], tables.shape[0], q.shape[1]
    pays = rows * (heads // kv_heads) // 16 >= 8 * n and rows >= 64 * n and (rows // 256 + n) * heads >= 64
    return q.dtype == torch.bfloat16 and most > 16 and not options.get("window") and dim in (64, 128) and block % 16 == 0 and pays


def check_attention(*args, **kw):
    dtype, dim, block = args[6], args[2], args[3]
    call, options, want, parts = attention_case(*args, **kw)
    out = torch.full(call[0].shape, 7.0, dtype=dtype, device="cuda")
    got = rlt.quantized_attention(*call, out=out, **options)
    assert got is out
    tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32, expanded=is_expanded(call, options))
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))
    return call, options, got


LENGTHS = [
    ([1], [1]),
    ([16, 17, 15, 31, 33], [1, 1, 1, 1, 1]),
    ([0, 5, 0], [1, 1, 0]),                                      # a padding sequence, and one without rows
    ([7, 40, 3], [5, 2, 5]),                                     # the third has rows in front of its first token
    ([1023, 1024, 1025, 2049], [1, 3, 2, 4]),                    # around the parts
    ([130, 64], [16, 9]),
    ([90, 3000], [21, 1]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, block", [(4, 4, 128, 16), (8, 2, 128, 16), (16, 1, 64, 32), (3, 3, 64, 16), (14, 2, 64, 64), (5, 1, 80, 8),
                                                         (2, 1, 33, 3), (2, 2, 256, 16), (40, 2, 128, 16)])
@pytest.mark.parametrize("lengths, counts", LENGTHS)
def test_attention_matches_the_plain_form(dtype, heads, kv_heads, dim, block, lengths, counts):
    check_attention(heads, kv_heads, dim, block, lengths, counts, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, block", [(2, 1, 128, 16), (2, 2, 64, 32), (2, 2, 40, 8)])
def test_parts_of_long_contexts(dtype, heads, kv_heads, dim, block):
    check_attention(heads, kv_heads, dim, block, [4096, 4097, 6144, 6145, 9000], [1, 2, 1, 1, 3], dtype)
    check_attention(heads, kv_heads, dim, block, [4096, 6150, 8200], [2, 1, 3], dtype, window=4100)
    check_attention(heads, kv_heads, dim, block, [4096, 6150, 8200, 2000], [2, 1, 20, 17], dtype, window=1900)      # from any place in a tile, in one part


@pytest.mark.parametrize("dim, kv_heads, counts", [(128, 32, 1), (64, 5, 3)])
def test_many_sequences(dim, kv_heads, counts):
    """More sequences than are laid out at a time, with more items for a CTA than it looks up at a time."""
    g = torch.Generator().manual_seed(dim)
    lengths = torch.randint(0, 60, (300,), generator=g).tolist()
    check_attention(kv_heads, kv_heads, dim, 16, lengths, torch.randint(0, counts + 1, (300,), generator=g).tolist(), torch.bfloat16)
    lengths[290] = 1500
    check_attention(kv_heads, kv_heads, dim, 16, lengths, [min(i % 7, 1) for i in range(300)], torch.float16, window=33)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tables_for_the_longest_contexts(dtype):
    """A row of a table of 2^26 tokens can have 32770 parts: three rows' partials fit in the workspace, and the rows are done in turns."""
    check_attention(32, 8, 128, 16, [3000, 40, 2500], [5, 1, 2], dtype, width=1 << 22)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, block", [(128, 16), (64, 32), (48, 5)])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 40, 1000, 1024, 1025, 1900, 1901, 5000])
def test_windows(dtype, dim, block, window):
    check_attention(4, 2, dim, block, [1, 50, 1040, 2100], [1, 4, 17 if window > 100 else 2, 3], dtype, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_scales_of_scores_wide_tables_and_strided_rows(dtype, dim):
    check_attention(4, 2, dim, 16, [100, 33], [2, 3], dtype, scale=0.7, width=300, strided=True)
    check_attention(4, 2, dim, 16, [100, 33], [2, 3], dtype, scale=-0.01, width=7)
    check_attention(4, 2, dim, 16, [100, 33], [2, 3], dtype, scale=0.0, width=7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim, block", [(128, 16), (64, 16), (24, 4)])
def test_a_length_beyond_its_table_is_cut(dtype, dim, block):
    call, options, want, _ = attention_case(2, 2, dim, block, [37, 64], [1, 2], dtype, width=64 // block)
    q, cache, tables, lengths, cu, most = call
    cut = rlt.quantized_attention(q, cache, tables[:, :32 // block].contiguous(), lengths, cu, most)
    again = rlt.quantized_attention(q, cache, tables[:, :32 // block].contiguous(), plain.words([32, 33]).cuda(), cu, most)
    assert torch.equal(cut[0], again[0]) and torch.equal(cut[1], again[1]) and torch.equal(cut[2], again[1].new_tensor(again[2].tolist()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim, block", [(8, 2, 128, 16), (4, 4, 64, 32), (2, 1, 40, 8)])
def test_a_row_is_the_same_alone_and_in_any_batch(dtype, heads, kv_heads, dim, block):
    lengths, counts = [1500, 40, 2100, 17], [3, 1, 5, 2]
    call, _, want, _ = attention_case(heads, kv_heads, dim, block, lengths, counts, dtype, spare=0)
    q, cache, tables, _, _, _ = call
    whole = rlt.quantized_attention(*call)
    row = 0
    for s, (a, c) in enumerate(zip(lengths, counts)):
        for i in range(c):
            one = rlt.quantized_attention(q[row:row + 1], cache, tables[s:s + 1], plain.words([a - c + i + 1]).cuda(), plain.words([0, 1]).cuda(), 1)
            assert torch.equal(one[0], whole[row]), (s, i)
            row += 1
    back = [3, 1, 0, 2]
    order = [r for s in back for r in range(sum(counts[:s]), sum(counts[:s + 1]))]
    turned = rlt.quantized_attention(q[order].contiguous(), cache, tables[back].contiguous(), plain.words([lengths[s] for s in back]).cuda(),
                                     plain.words(plain.starts_of([counts[s] for s in back])).cuda(), 5)
    assert torch.equal(turned, whole[order])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim, block", [(128, 16), (64, 16), (40, 8)])
@pytest.mark.parametrize("window", [0, 12])
def test_what_a_row_does_not_see_may_be_nan(dtype, dim, block, window):
    """NaN in the key and value of a later row's token (and, behind a window, of an earlier one): the rows that see it are NaN, the others
    what they were."""
    call, options, want, parts = attention_case(2, 1, dim, block, [40, 23], [6, 6], dtype, window=window, spare=0)
    q, cache, tables, lengths, cu, most = call
    clean = rlt.quantized_attention(*call, **options)
    for which in ("key", "value"):
        codes = getattr(cache, which).view(torch.uint8)
        page, saved = int(tables[0, 37 // block]), codes.clone()
        codes[page, 37 % block, 0, 3] = 0x7f
        if window:
            codes[int(tables[1, 8 // block]), 8 % block, 0, dim - 1] = 0xff
        got = rlt.quantized_attention(*call, **options)
        hit = torch.zeros(12, dtype=torch.bool)
        hit[3:6] = True                                          # positions 37, 38 and 39 see token 37
        if window:
            hit[6:9] = True                                      # positions 17, 18 and 19 still see token 8 behind a window of 12
        if which == "key":
            assert got[hit.cuda()].isnan().all()
        else:
            assert got[:, :, 3][hit.cuda()][:3].isnan().all() and (not window or got[6:9, :, dim - 1].isnan().all())
            keep = [d for d in range(dim) if d not in (3, dim - 1)]
            assert torch.equal(got[:, :, keep], clean[:, :, keep])
        assert torch.equal(got[~hit.cuda()], clean[~hit.cuda()])
        codes.copy_(saved)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [128, 64, 40])
def test_pages_of_unlike_scales_and_scales_that_are_no_powers_of_two(dtype, dim):
    """Pages 2^40 apart in the size of their values, with the weight on the small ones or on the large ones; a page of scale 0."""
    block, lengths, counts = 16, [160], [2]
    call, options, _, _ = attention_case(2, 2, dim, block, lengths, counts, dtype, spare=0)
    q, cache, tables, _, cu, _ = call
    g = torch.Generator().manual_seed(8)
    order = tables[0, :10].long()
    for kind in range(4):
        cache.key_scale[order] = (torch.rand(10, 2, generator=g) + 0.01).cuda()
        exponents = torch.tensor([[40.0, 0, -40, 0, 3, 40, -40, 0, 0, 0], [0.0] * 10, [-90.0] * 10, [90.0, -90] * 5][kind])
        cache.value_scale[order] = (torch.exp2(exponents)[:, None] * (torch.rand(10, 2, generator=g) + 0.5)).cuda()
        if kind == 1:
            cache.value_scale[order[4]] = 0.0
            cache.key_scale[order[5]] = 0.0
        codes = [t.cpu().double() for t in (cache.key, cache.value)]
        scales = [torch.nan_to_num(t.cpu().double()) for t in (cache.key_scale, cache.value_scale)]
        codes = [torch.nan_to_num(c) for c in codes]
        want, parts = plain.attention(q.cpu(), codes, scales, tables.cpu(), lengths, [0, 2])
        if dtype == torch.float16:
            fits = want.abs() < 60000
        else:
            fits = torch.ones_like(want, dtype=torch.bool)
        got = rlt.quantized_attention(*call, **options).cpu().double()
        tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32)
        err = (got - want).abs()
        assert bool((err[fits] <= tol[fits]).all()), (kind, float((err[fits] / tol[fits]).max()))


LONG = [
    (32, 32, 128, 16, [300, 700], [300, 129], {}),
    (32, 8, 128, 32, [513, 100, 1, 65], [257, 100, 1, 17], {}),
    (14, 2, 64, 64, [4100, 90, 0, 2050], [60, 33, 40, 200], {}),                  # a sequence of padding rows in between
    (16, 1, 64, 16, [1000], [1000], dict(strided=True)),
    (32, 16, 128, 48, [200, 31], [128, 64], dict(scale=0.3, spare=0)),            # rows at negative positions
    (32, 8, 128, 16, [64, 17], [64, 64], dict(width=100)),
    (24, 3, 64, 16, [100, 70, 65, 200], [64, 70, 65, 64], {}),                    # an odd number of 64-wide heads
]


@pytest.mark.parametrize("heads, kv_heads, dim, block, lengths, counts, more", LONG)
def test_long_portions(heads, kv_heads, dim, block, lengths, counts, more):
    args = (heads, kv_heads, dim, block, lengths, counts, torch.bfloat16)
    call, options, got = check_attention(*args, **more)
    assert is_expanded(call, options)
    few = rlt.quantized_attention(*call[:5], 16, out=torch.full(call[0].shape, 7.0, dtype=torch.bfloat16, device="cuda"), **options)
    assert not torch.equal(few, got)                              # another kernel's roundings
    for dtype in (torch.float16, torch.float32):
        check_attention(*args[:-1], dtype, **more)


@pytest.mark.parametrize("dim", [128, 64])
def test_long_portions_that_an_expansion_cannot_hold(dim):
    """A sequence with a NaN value, one with a page scale that is no power of two, one beyond its table: each as from short portions' kernel, and
    the others beside them as they were.  Pages outside the cache are zeros."""
    lengths, counts = [200, 160, 230, 90, 111], [100, 160, 80, 64, 64]
    call, options, _, _ = attention_case(16, 4, dim, 16, lengths, counts, torch.bfloat16, spare=0, width=20)
    q, cache, tables, on, cu, most = call
    assert is_expanded(call, options)
    clean = rlt.quantized_attention(*call)
    starts = plain.starts_of(counts)

    def check(marked, lengths=on):
        long, short = (rlt.quantized_attention(q, cache, tables, lengths, cu, m) for m in (most, 16))
        for s in range(5):
            rows = slice(starts[s], starts[s + 1])
            same = short if s in marked else clean
            assert torch.equal(long[rows].nan_to_num(99.0), same[rows].nan_to_num(99.0)), (marked, s)
        return long

    check([])
    codes = cache.value.view(torch.uint8)
    at = (int(tables[1, 7]), 3, 2, 5)                               # token 115 of sequence 1
    saved = codes[at].clone()
    codes[at] = 0xff
    got = check([1])
    assert got[starts[1] + 115:starts[2], 8:12, 5].isnan().all() and got[starts[1]:starts[1] + 115].isfinite().all()
    for scale in (cache.key_scale, cache.value_scale):
        page = int(tables[2, 3])
        keep = scale[page, 1].clone()
        for odd in (keep * 1.5, keep * 0, keep * 2.0 ** 120):
            scale[page, 1] = odd
            check([1, 2])
        scale[page, 1] = keep
    codes[at] = saved
    far = on.clone()
    far[4] = 20 * 16 + 7                                            # (its table's other entries name pages of other sequences, or none)
    tables[4, 7:] = tables[4, :1]
    check([4], far)
    keys = cache.key.view(torch.uint8)
    keys[int(tables[3, 1])] = 0x7f                                  # keys that are NaN need no marks: who sees them is NaN
    got = rlt.quantized_attention(*call)
    assert got[starts[3]:starts[4]].isnan().all() and torch.equal(got[:starts[3]], clean[:starts[3]])
    tables[0, 2], tables[0, 5] = -1, 1 << 20
    raw = [torch.nan_to_num(t.cpu().double()) for t in (cache.key, cache.value, cache.key_scale, cache.value_scale)]
    raw = [torch.cat((t, torch.zeros_like(t[:1]))) for t in raw]    # a page of zeros behind the others
    named = tables.cpu()[:1].clone()
    named[0, 2] = named[0, 5] = raw[0].shape[0] - 1
    want, parts = plain.attention(q.cpu()[:100], raw[:2], raw[2:], named, [200], [0, 100])
    got = rlt.quantized_attention(*call)[:100]
    tol = plain.allowed(want, parts, torch.bfloat16, dim, tiles=True, expanded=True)
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


def test_long_portions_from_a_graph():
    """A captured call over expanded pages, replayed with other lengths, rows and codes, one of them a value that is NaN."""
    heads, kv_heads, dim, block = 32, 4, 128, 16
    call, _, _, _ = attention_case(heads, kv_heads, dim, block, [300, 200], [130, 130], torch.bfloat16, spare=0, width=30)
    q, cache, tables, lengths, cu, most = call
    assert is_expanded(call, {})
    rlt.quantized_attention(*call)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rlt.quantized_attention(*call)
    codes = cache.value.view(torch.uint8)
    for step in range(3):
        if step == 1:
            lengths.copy_(plain.words([140, 190]).cuda())
            cu.copy_(plain.words([0, 135, 260]).cuda())
            q.neg_()
        if step == 2:
            codes[int(tables[1, 3]), 5, 1, 7] = 0x7f                # token 53 of the second
        graph.replay()
        assert torch.equal(out.nan_to_num(9.0), rlt.quantized_attention(*call).nan_to_num(9.0)), step
        assert bool(out.isnan().any()) == (step == 2)


def test_rows_of_extreme_size():
    """Queries near the largest and smallest numbers of their type, beside ordinary ones."""
    for dtype, sizes in ((torch.bfloat16, [1e30, 1e-30, 0.0, 1.0]), (torch.float16, [60000.0, 1e-6, 0.0, 1.0]), (torch.float32, [1e30, 1e-38, 0.0, 1.0])):
        for dim in (128, 64):
            call, options, _, _ = attention_case(2, 2, dim, 16, [70], [4], dtype, spare=0)
            q, cache, tables, lengths, cu, most = call
            size = torch.tensor(sizes)[:, None, None].cuda()
            big = (torch.nn.functional.normalize(q.float(), dim=-1) * size).to(dtype)
            got = rlt.quantized_attention(big, cache, tables, lengths, cu, most, scale=1e-3)
            codes, scales = ([torch.nan_to_num(t.cpu().double()) for t in pair] for pair in ((cache.key, cache.value), (cache.key_scale, cache.value_scale)))
            want, parts = plain.attention(big.cpu(), codes, scales, tables.cpu(), [70], [0, 4], scale=1e-3)
            assert got.isfinite().all()
            tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32)
            err = (got.cpu().double() - want).abs()
            for r in (1, 2, 3):                                   # of the first, weights are decided by differences of scores of 1e27: finite is all that is said
                assert bool((err[r] <= tol[r]).all()), (dtype, dim, r, float((err[r] / tol[r]).max()))


def test_empty_calls():
    cache = rlt.QuantizedKV.allocate(2, 16, 2, 128)
    tables, lengths, cu = plain.words([[0]]).cuda(), plain.words([4]).cuda(), plain.words([0, 0]).cuda()
    q = torch.zeros(0, 4, 128, device="cuda", dtype=torch.bfloat16)
    assert rlt.quantized_attention(q, cache, tables, lengths, cu, 0).shape == (0, 4, 128)
    q = torch.ones(3, 4, 128, device="cuda", dtype=torch.bfloat16)
    out = torch.full_like(q, 5.0)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    rlt.quantized_attention(q, cache, none.view(0, 3), none, plain.words([0]).cuda(), 1, out=out)
    rlt.quantized_attention(q, cache, tables, lengths, cu, 1, out=out)              # no sequence has rows
    assert (out == 5.0).all()
    with pytest.raises(ValueError, match="page"):
        rlt.quantized_attention(q, cache, tables[:, :0].contiguous(), lengths, cu, 1)
    for other in (out.float(), q):
        with pytest.raises(ValueError, match="out must"):
            rlt.quantized_attention(q, cache, tables, lengths, cu, 1, out=other)
    with pytest.raises(ValueError, match="CUDA"):
        rlt.quantized_attention(q, cache, tables.cpu(), lengths, cu, 1)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GB of codes, with pages at its end."""
    heads, dim, block, pages = 8, 128, 16, 300_000
    raw = torch.zeros(2, pages, block, heads, dim, dtype=torch.uint8, device="cuda")
    cache = rlt.QuantizedKV(raw[0].view(plain.CODE), raw[1].view(plain.CODE), *torch.zeros(2, pages, heads, device="cuda").unbind())
    g = torch.Generator().manual_seed(4)
    tables, lengths, cu = plain.words([[pages - 1, 3, pages - 2]]), [40], [0, 40]
    k, v = (torch.randn(40, heads, dim, generator=g).bfloat16() for _ in range(2))
    rlt.quantized_kv_write(cache, k.cuda(), v.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda())
    few = torch.tensor([pages - 1, 3, pages - 2], device="cuda")
    codes = [raw[i][few].view(plain.CODE).cpu().double() for i in range(2)]
    scales = [t[few].cpu().double() for t in (cache.key_scale, cache.value_scale)]
    want_codes, want_scales = torch.zeros_like(codes[0]), torch.zeros_like(scales[0])
    plain.kv_write(want_codes, want_scales, k.double(), plain.words([[0, 1, 2]]), lengths, cu)
    assert torch.equal(codes[0], want_codes) and torch.equal(scales[0], want_scales)
    for dtype in (torch.bfloat16, torch.float32):
        q = (torch.randn(40, 16, dim, generator=g) * 0.3).to(dtype)
        for rows, most in ((slice(38, 40), 2), (slice(0, 40), 40)):
            n = q[rows].shape[0]
            want, parts = plain.attention(q[rows], codes, scales, plain.words([[0, 1, 2]]), lengths, [0, n])
            got = rlt.quantized_attention(q[rows].cuda(), cache, tables.cuda(), plain.words(lengths).cuda(), plain.words([0, n]).cuda(), most)
            tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32)
            err = (got.cpu().double() - want).abs()
            assert bool((err <= tol).all())


# ---- together ---------------------------------------------------------------------------------------------
class Serving:
    """A layer's 8-bit cache with its pages and state on the GPU, and the same in plain form."""

    def __init__(self, requests, block, width, kv_heads, dim, pages):
        self.block = block
        self.cache = rlt.QuantizedKV.allocate(pages, block, kv_heads, dim)
        self.tables = torch.zeros(requests, width, dtype=torch.int32, device="cuda")
        self.held, self.lengths = (torch.zeros(requests, dtype=torch.int32, device="cuda") for _ in range(2))
        self.free, self.count = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0).contiguous(), plain.words([pages]).cuda()

    def step(self, counts, q, k, v, most, **kw):
        slots = rlt.step_slots(self.lengths, counts, self.tables, self.block, q.shape[0], held=self.held, free_pages=self.free, free_count=self.count)
        rlt.quantized_kv_write(self.cache, k, v, self.tables, slots.lengths, slots.cu)
        out = rlt.quantized_attention(q, self.cache, self.tables, slots.lengths, slots.cu, most, **kw)
        self.lengths.copy_(slots.lengths)
        return out, slots


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, kv_heads, dim, block", [(8, 2, 128, 16), (4, 4, 64, 32)])
def test_a_run_of_steps_from_prompts_to_decoding(dtype, heads, kv_heads, dim, block):
    """Prompts, decoding and verification rows with rollback, in eager calls and from a captured graph: at every step the output is the plain
    attention over what the cache holds, and the cache holds the rows to within a code's rounding."""
    g = torch.Generator().manual_seed(dim)
    n, width, pages = 4, 12, 40
    plan = [([37, 20, 1, 0], 37), ([1, 1, 1, 50], 50), ([1, 1, 1, 1], 1), ([5, 5, 5, 5], 5), ([1, 1, 1, 1], 1), ([1, 1, 1, 1], 1), ([1, 1, 1, 1], 1)]
    keep = {3: [3, 1, 5, 2]}                                                         # of the fourth step's five rows so many stay
    served = Serving(n, block, width, kv_heads, dim, pages)
    kept = [torch.zeros(0, 2, kv_heads, dim, dtype=torch.float64) for _ in range(n)]
    graph, buffers = None, None
    for index, (counts, most) in enumerate(plan):
        rows = sum(counts)
        q = (torch.randn(rows, heads, dim, generator=g) * 0.3).to(dtype).cuda()
        k, v = (torch.randn(rows, kv_heads, dim, generator=g).to(dtype).cuda() for _ in range(2))
        if index < 5:
            out, slots = served.step(plain.words(counts).cuda(), q, k, v, most)
            cu, status, after = slots.cu.tolist(), int(slots.status), slots.lengths.tolist()
        else:
            if graph is None:
                buffers = [torch.zeros_like(t) for t in (q, k, v)]
                state = [t.clone() for t in (served.lengths, served.held, served.count, served.tables, served.cache.key.view(torch.uint8),
                                             served.cache.value.view(torch.uint8), served.cache.key_scale, served.cache.value_scale)]
                one = plain.words(counts).cuda()
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    served.step(one, *buffers, most)
                torch.cuda.current_stream().wait_stream(side)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    captured = served.step(one, *buffers, most)
                for t, before in zip((served.lengths, served.held, served.count, served.tables, served.cache.key.view(torch.uint8),
                                      served.cache.value.view(torch.uint8), served.cache.key_scale, served.cache.value_scale), state):
                    t.copy_(before)
            for b, t in zip(buffers, (q, k, v)):
                b.copy_(t)
            graph.replay()
            out, slots = captured
            cu, status, after = slots.cu.tolist(), int(slots.status), slots.lengths.tolist()
        assert status == 0 and cu == plain.starts_of(counts)
        for s in range(n):
            kept[s] = torch.cat((kept[s], torch.stack((k, v), 1)[cu[s]:cu[s + 1]].cpu().double()))
            assert after[s] == len(kept[s]) and int(served.held[s]) >= -(-after[s] // block)
        pages_of = [served.tables[s, :-(-after[s] // block)].tolist() for s in range(n)]
        assert len({p for ps in pages_of for p in ps}) == sum(map(len, pages_of))   # nobody shares a page
        codes = [t.cpu().double() for t in (served.cache.key, served.cache.value)]
        scales = [t.cpu().double() for t in (served.cache.key_scale, served.cache.value_scale)]
        for s in range(n):
            t = torch.arange(after[s])
            page = served.tables[s].cpu().long()[t // block]
            for i in range(2):
                held = codes[i][page, t % block] * scales[i][page][:, :, None]
                # half a step of e4m3, 2^-4 of the value; where codes are the smallest, half a step of those, 2^-10, once for the rounding at the page's
                # scale and at most as much again for all growths before it (each at a scale of at most half the next one's: a geometric sum)
                assert bool(((held - kept[s][:, i]).abs() <= 2 * (2.0 ** -4 * kept[s][:, i].abs() / 2 + 2.0 ** -10 * scales[i][page][:, :, None])).all())
        want, parts = plain.attention(q.cpu(), codes, scales, served.tables.cpu(), after, cu)
        err, tol = (out.cpu().double() - want).abs(), plain.allowed(want, parts, dtype, dim, tiles=True)
        assert bool((err <= tol).all()), (index, float((err / tol).max()))
        if index in keep:
            for s, m in enumerate(keep[index]):
                kept[s] = kept[s][:len(kept[s]) - counts[s] + m]
            served.lengths.copy_(plain.words([len(x) for x in kept]).cuda())
    # finished requests give everything back
    served.lengths.zero_()
    assert int(rlt.return_pages(served.lengths, served.tables, block, held=served.held, free_pages=served.free, free_count=served.count)) == 0
    assert served.count.tolist() == [pages] and sorted(served.free.tolist()) == list(range(pages))


def test_two_streams_at_once():
    """Calls on two streams share no scratch: long contexts (several parts) in turn, each as if it were alone."""
    calls = [attention_case(8, 2, 128, 16, [3000, 2500], [2, 1], torch.bfloat16, seed=s, spare=0)[0] for s in (0, 1)]
    alone = [rlt.quantized_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(rlt.quantized_attention(*calls[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv_heads, group, counts", [(2, 1, [1, 1, 1]), (2, 4, [5, 2, 3]), (3, 1, [4, 4, 4]), (3, 2, [9, 1, 2]), (5, 7, [3, 1, 2])])
@pytest.mark.parametrize("window", [0, 90])
def test_nan_in_one_head_stays_in_it(dtype, kv_heads, group, counts, window):
    """64-wide heads share lines of the cache: a NaN key or value of one head changes no bit of another one's rows."""
    lengths = [200, 33, 1160]
    call, options, _, _ = attention_case(group * kv_heads, kv_heads, 64, 16, lengths, counts, dtype, window=window, spare=0)
    q, cache, tables, _, cu, most = call
    clean = rlt.quantized_attention(*call, **options)
    starts = plain.starts_of(counts)
    for which in ("key", "value"):
        codes = getattr(cache, which).view(torch.uint8)
        for head in range(kv_heads):
            saved = codes.clone()
            seen = torch.zeros(sum(counts), dtype=torch.bool)
            for s, (a, n) in enumerate(zip(lengths, counts)):
                for token in (a - n - 20, a - 1):                    # one that all rows of the sequence see, one that only the last does
                    codes[int(tables[s, token // 16]), token % 16, head, 7] = 0x7f if token % 2 else 0xff
                seen[starts[s]:starts[s + 1]] = True
            got = rlt.quantized_attention(*call, **options)
            mine = torch.arange(group * kv_heads) // group == head
            assert torch.equal(got[:, ~mine.cuda()], clean[:, ~mine.cuda()]), (which, head)
            hit = got[:, mine.cuda()].isnan()
            assert bool(hit.all() if which == "key" else hit[..., 7].all()), (which, head)
            for s, (a, n) in enumerate(zip(lengths, counts)):
                one = rlt.quantized_attention(q[starts[s]:starts[s + 1]].contiguous(), cache, tables[s:s + 1].contiguous(), plain.words([a]).cuda(),
                                              plain.words([0, n]).cuda(), n, **options)
                assert torch.equal(one.nan_to_num(9.0), got[starts[s]:starts[s + 1]].nan_to_num(9.0)), (which, head, s)
            codes.copy_(saved)


def test_a_stored_infinity_stays_in_its_head():
    """What is not finite is stored as NaN: the rows of its own head are NaN, the neighbour's are as they would be without it."""
    g = torch.Generator().manual_seed(5)
    n, kv_heads, dim = 21, 2, 64
    k, v = (torch.randn(n, kv_heads, dim, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(2, 8, dim, generator=g).bfloat16().cuda()
    tables, lengths, cu = plain.words([[1, 0]]).cuda(), plain.words([n]).cuda(), plain.words([0, n]).cuda()
    outs = []
    for bad in (False, True):
        if bad:
            k[4, 1, 9] = math.inf
        cache = rlt.QuantizedKV.allocate(2, 16, kv_heads, dim)
        rlt.quantized_kv_write(cache, k, v, tables, lengths, cu)
        outs.append(rlt.quantized_attention(q, cache, tables, lengths, plain.words([0, 2]).cuda(), 2))
    assert outs[0].isfinite().all() and torch.equal(outs[0][:, :4], outs[1][:, :4]) and outs[1][:, 4:].isnan().all()


def scale_in_range(scale):
    """The value scale that is read: the nearer end of 2^-100 .. 2^100, zero for zero, NaN for what is negative or NaN."""
    scale = scale.double()
    inside = scale.clamp(2.0 ** -100, 2.0 ** 100)
    return torch.where(scale == 0, 0.0, torch.where(scale >= 0, inside, math.nan))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [128, 64, 40])
@pytest.mark.parametrize("value_scale", [0.0, -0.0, 2.0 ** -110, 1e-35, 1e-40, 2.0 ** -100, 2.0 ** 100, 2.0 ** 110, math.inf])
def test_value_scales_at_and_beyond_their_range(dtype, dim, value_scale):
    """One cache gives one result, whatever kernel reads it: everywhere such a scale, and in one page beside ordinary ones."""
    lengths, counts = [70, 35], [2, 1]
    call, options, _, _ = attention_case(4, 2, dim, 16, lengths, counts, dtype, spare=0)
    q, cache, tables, _, cu, _ = call
    codes = [torch.nan_to_num(t.cpu().double()) for t in (cache.key, cache.value)]
    ordinary = torch.nan_to_num(cache.value_scale, nan=1.0)
    for everywhere in (True, False):
        cache.value_scale.copy_(ordinary)
        if everywhere:
            cache.value_scale.fill_(value_scale)
        else:
            cache.value_scale[int(tables[0, 2])] = value_scale
        scales = [torch.nan_to_num(cache.key_scale.cpu().double()), scale_in_range(cache.value_scale.cpu())]
        want, parts = plain.attention(q.cpu(), codes, scales, tables.cpu(), lengths, plain.starts_of(counts))
        got = rlt.quantized_attention(*call, **options).cpu().double()
        tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32)
        err = (got - want).abs()
        assert bool((err <= tol).all()), (everywhere, float((err / tol).max()))
        if everywhere and value_scale == 0:
            assert bool((got == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [128, 64, 40])
@pytest.mark.parametrize("bad", [math.nan, -1.0, -math.inf])
def test_value_scales_that_are_no_sizes(dtype, dim, bad):
    """The rows that see a token of such a page are NaN in its head, the others what they were."""
    lengths, counts = [70, 35], [9, 2]                               # positions 61 .. 69: of the last page's tokens five rows see some, page 3 ends at 63
    call, options, _, _ = attention_case(4, 2, dim, 16, lengths, counts, dtype, spare=0)
    q, cache, tables, _, cu, _ = call
    cache.value_scale.copy_(torch.nan_to_num(cache.value_scale, nan=1.0))
    clean = rlt.quantized_attention(*call, **options)
    cache.value_scale[int(tables[0, 4]), 1] = bad                    # tokens 64 .. 69
    got = rlt.quantized_attention(*call, **options)
    hit = torch.zeros(11, 4, dtype=torch.bool)
    hit[3:9, 2:] = True
    assert bool(got[hit.cuda()].isnan().all()) and torch.equal(got[~hit.cuda()], clean[~hit.cuda()])


@pytest.mark.parametrize("value_scale", [0.0, 1e-35, 2.0 ** 110, math.nan])
def test_long_portions_over_scales_beyond_their_range(value_scale):
    lengths, counts = [200, 160], [200, 160]
    call, options, _, _ = attention_case(32, 4, 64, 16, lengths, counts, torch.bfloat16, spare=0)
    assert is_expanded(call, options)
    q, cache, tables, on, cu, most = call
    cache.value_scale[int(tables[1, 3]), 2] = value_scale
    long, short = (rlt.quantized_attention(q, cache, tables, on, cu, m) for m in (most, 16))
    assert torch.equal(long[200:].nan_to_num(9.0), short[200:].nan_to_num(9.0))
    assert bool(long[200 + 48:, 16:24].isnan().all()) == math.isnan(value_scale) and bool(long[:200 + 48].isfinite().all())


@pytest.mark.parametrize("dim", [128, 64])
def test_rows_that_see_no_key_in_front_of_others(dim):
    """Hundreds of padding sequences, whose items have nothing to score, in front of sequences that have."""
    n = 700
    lengths, counts = [0] * n, [1] * n
    for s in (3, 299, 300, 511, 512, 640, 699):
        lengths[s] = 200 + s
    for kv_heads in (64, 6):
        check_attention(kv_heads, kv_heads, dim, 16, lengths, counts, torch.bfloat16)


def test_requests_whose_sums_nearly_fill_the_usual_shared_memory():
    """Each in a process that has made no larger call before."""
    code = """
import plain_quantized as plain, torch, vllm_rlt_b200 as rlt
for n in (4053, 4094):
    lengths, counts = [i % 40 for i in range(n)], [1 + i % 2 for i in range(n)]
    tables = torch.randint(0, 1000, (n, 3), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    want = plain.step_slots(lengths, counts, tables.tolist(), 16, 3 * n)
    got = rlt.step_slots(plain.words(lengths).cuda(), plain.words(counts).cuda(), tables.cuda(), 16, 3 * n)
    for name, expected in zip(("cu", "lengths", "positions", "row_seq", "write_blocks", "write_offsets"), want):
        assert getattr(got, name).tolist() == expected, (n, name)
    assert int(got.status) == 0
for n in (6079, 6142):
    lengths, held, free, count = [16 * (i % 3) for i in range(n)], [3] * n, [-1] * (3 * n), [0]
    tables = torch.arange(3 * n, dtype=torch.int32).view(n, 3)
    state = dict(held=plain.words(held).cuda(), free_pages=plain.words(free).cuda(), free_count=plain.words(count).cuda())
    status = rlt.return_pages(plain.words(lengths).cuda(), tables.cuda(), 16, **state)
    assert plain.return_pages(lengths, tables.tolist(), 16, held, free, count) == int(status) == 0
    assert state["held"].tolist() == held and state["free_pages"].tolist() == free and state["free_count"].tolist() == count, n
"""
    root = Path(__file__).resolve().parent
    done = subprocess.run([sys.executable, "-c", code], cwd=root.parent, env=dict(os.environ, PYTHONPATH=f"{root.parent}:{root}"), capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_threads_with_unlike_numbers_of_requests():
    """Steps of 8192, 5000 and 6 requests at once, each from a thread of its own: one does not take another's shared memory away."""
    lib, failed = rlt.load_library(), []
    sizes = (8192, 5000, 8192, 6)
    streams = [torch.cuda.Stream() for _ in sizes]
    arrays = [[torch.zeros(n + 1, dtype=torch.int64, device="cuda") for _ in range(8)] for n in sizes]
    torch.cuda.synchronize()

    def work(n, stream, at):
        torch.cuda.set_device(0)
        for _ in range(4000):
            code = lib.rlt_step_slots(at[0], at[0], n, at[1], 1, 16, None, None, 0, None, 0, at[2], at[3], None, None, None, None, at[4], at[5], stream)
            code = code or lib.rlt_return_pages(at[0], n, at[1], 1, 16, at[0], None, 0, at[6], at[7], stream)
            if code:
                failed.append((n, code, lib.rlt_last_error()))
                return

    threads = [threading.Thread(target=work, args=(n, s.cuda_stream, [t.data_ptr() for t in a])) for n, s, a in zip(sizes, streams, arrays)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]


@pytest.mark.parametrize("heads, kv_heads, dim", [(32, 8, 128), (16, 2, 64)])
def test_short_portions_beside_a_long_one(heads, kv_heads, dim):
    """A prompt's portion beside single tokens and verification rows: the short ones keep the bits that they have without it."""
    lengths, counts = [1500, 900, 3000, 40, 2100, 17, 33, 700], [1, 900, 16, 1, 5, 0, 17, 70]
    call, options, got = check_attention(heads, kv_heads, dim, 16, lengths, counts, torch.bfloat16)
    assert is_expanded(call, options)
    q, cache, tables, _, _, _ = call
    starts = plain.starts_of(counts)
    for s, (a, n) in enumerate(zip(lengths, counts)):
        if n:
            one = rlt.quantized_attention(q[starts[s]:starts[s + 1]].contiguous(), cache, tables[s:s + 1].contiguous(), plain.words([a]).cuda(),
                                          plain.words([0, n]).cuda(), min(n, 16))
            assert torch.equal(one, got[starts[s]:starts[s + 1]]) == (n < 64), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, dim, block", [(8, 2, 128, 16), (6, 3, 64, 32), (4, 2, 40, 8)])
def test_keys_and_values_side_by_side_in_one_pool(dtype, heads, kv_heads, dim, block):
    """A pool [pages, block, keys or values, kv_heads, dim]: tokens are two rows apart, pages further than their tokens."""
    g = torch.Generator().manual_seed(dim)
    lengths, counts = [70, 33, 130], [3, 33, 40]
    tables, pages = pages_for(lengths, block, g)
    raw, scales = plain.make_cache(pages, block, kv_heads, dim, g)                    # [2, pages, 1, block, heads, dim]
    pool = torch.full((pages, block + 2, 2, kv_heads, dim), 0x7f, dtype=torch.uint8, device="cuda")
    pool[:, :block] = raw[:, :, 0].permute(1, 2, 0, 3, 4).cuda()
    before = pool.clone()
    dev_scales = scales[:, :, 0].contiguous().cuda()
    cache = rlt.QuantizedKV(pool[:, :block, 0].view(plain.CODE), pool[:, :block, 1].view(plain.CODE), dev_scales[0], dev_scales[1])
    cu = plain.starts_of(counts)
    k, v = (torch.randn(sum(counts), kv_heads, dim, generator=g).to(dtype) for _ in range(2))
    rlt.quantized_kv_write(cache, k.cuda(), v.cuda(), tables.cuda(), plain.words(lengths).cuda(), plain.words(cu).cuda())
    codes, want_scales = raw[:, :, 0].view(plain.CODE).double(), scales[:, :, 0].double()
    for i, x in enumerate((k, v)):
        plain.kv_write(codes[i], want_scales[i], x.double(), tables, lengths, cu)
    assert torch.equal(dev_scales.cpu().double(), want_scales)
    assert same_values(cache.key.cpu().double(), codes[0]) and same_values(cache.value.cpu().double(), codes[1])
    assert torch.equal(pool[:, block:], before[:, block:])
    for most, some in ((3, [3, 2, 1]), (40, [3, 33, 40])):
        rows = plain.starts_of(some)
        q = (torch.randn(sum(some), heads, dim, generator=g) * 0.1).to(dtype)
        want, parts = plain.attention(q, codes, want_scales, tables, lengths, rows)
        got = rlt.quantized_attention(q.cuda(), cache, tables.cuda(), plain.words(lengths).cuda(), plain.words(rows).cuda(), most).cpu().double()
        tol = plain.allowed(want, parts, dtype, dim, tiles=dtype != torch.float32)
        assert bool(((got - want).abs() <= tol).all()), most


def test_portions_of_a_captured_step_become_short_and_long():
    """A call captured with long portions, replayed with others of any length in the same rows: each portion goes where its rows say, and rows
    behind the last sequence stay."""
    lengths = [300, 500, 200]
    call, _, _, _ = attention_case(32, 8, 128, 16, lengths, [100, 120, 80], torch.bfloat16, spare=0, width=40)
    q, cache, tables, dev_lengths, cu, most = call
    assert is_expanded(call, {})
    out = torch.full_like(q, 7.0)
    rlt.quantized_attention(*call, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rlt.quantized_attention(*call, out=out)
    for counts in ([100, 120, 80], [1, 5, 16], [63, 64, 65], [0, 150, 1], [0, 0, 0], [200, 99, 1]):
        starts = plain.starts_of(counts)
        cu.copy_(plain.words(starts))
        out.fill_(7.0)
        graph.replay()
        for s, n in enumerate(counts):
            if n:
                rows = q[starts[s]:starts[s + 1]].contiguous()
                part = torch.cat((rows, rows.new_zeros(256 - n, *rows.shape[1:]))) if n >= 64 else rows        # (of a step long enough)
                one = rlt.quantized_attention(part, cache, tables[s:s + 1].contiguous(), dev_lengths[s:s + 1], plain.words([0, n]).cuda(), len(part) if n >= 64 else 16)
                assert torch.equal(one[:n], out[starts[s]:starts[s + 1]]), (counts, s)
        assert bool((out[starts[3]:] == 7.0).all())
