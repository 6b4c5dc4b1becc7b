"""The 8-bit paged cache in plain float64 tensors on the CPU: pages and slots, storing, attention, and how far a kernel may be from them."""

from __future__ import annotations

import math

import torch

CODE = torch.float8_e4m3fn
GRID = torch.arange(256, dtype=torch.uint8).view(CODE).double()


def words(values):
    return torch.tensor(values, dtype=torch.int32)


def starts_of(counts):
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    return cu


# ---- pages and slots ----------------------------------------------------------------------------------
def step_slots(lengths, counts, tables, block, rows, held=None, free=None, free_count=None):
    """(cu, lengths, positions, row_seq, write_blocks, write_offsets, active, status); lists, tables / held / free_count changed in place."""
    n, width = len(lengths), len(tables[0]) if tables else 0
    counts = [max(c, 0) for c in counts]
    after = [a + c for a, c in zip(lengths, counts)]
    bad = any(a < 0 or e > width * block for a, e in zip(lengths, after)) or sum(counts) > rows
    if held is not None:
        bad = bad or any(not 0 <= h <= width for h in held)
        need = [max(-(-e // block) - h, 0) for e, h in zip(after, held)]
        bad = bad or sum(need) > free_count[0] or not 0 <= free_count[0] <= len(free)
    padding = ([0], [-1], [-1], [0])
    if bad:
        return [0] * (n + 1), list(lengths), *(p * rows for p in padding), 0, 1
    if held is not None:
        for s in range(n):
            for _ in range(need[s]):
                free_count[0] -= 1
                tables[s][held[s]] = free[free_count[0]]
                held[s] += 1
    positions, owner, blocks, offsets = [], [], [], []
    for s in range(n):
        for p in range(lengths[s], after[s]):
            positions.append(p)
            owner.append(s)
            blocks.append(tables[s][p // block])
            offsets.append(p % block)
    spare = rows - len(positions)
    return (starts_of(counts), after, positions + padding[0] * spare, owner + padding[1] * spare, blocks + padding[2] * spare,
            offsets + padding[3] * spare, sum(counts), 0)


def return_pages(lengths, tables, block, held, free, free_count):
    width = len(tables[0]) if tables else 0
    keep = [min(-(-max(a, 0) // block), h) for a, h in zip(lengths, held)]
    given = [tables[s][j] for s in range(len(held)) for j in range(keep[s], max(held[s], 0))] if all(0 <= h <= width for h in held) else None
    if given is None or free_count[0] < 0 or free_count[0] + len(given) > len(free):
        return 1
    free[free_count[0]:free_count[0] + len(given)] = given[::-1]
    free_count[0] += len(given)
    held[:] = keep
    return 0


# ---- storing ------------------------------------------------------------------------------------------
def nearest_code(x):
    """The e4m3 value nearest to each float64, ties to the even code, saturating; NaN for NaN.  By distance over the 256 codes."""
    order = sorted((c for c in range(256) if math.isfinite(float(GRID[c])) and c != 128), key=lambda c: float(GRID[c]))
    grid = GRID[order]
    even = torch.tensor([c % 2 == 0 for c in order])
    middle = (grid[1:] + grid[:-1]) / 2                       # exact: neighbours differ by one step
    flat = x.reshape(-1).contiguous()
    i = torch.searchsorted(middle, torch.nan_to_num(flat, nan=0.0))
    tie = (i < middle.numel()) & (flat == middle[i.clamp_max(middle.numel() - 1)])
    got = grid[torch.where(tie & ~even[i], i + 1, i)]
    return torch.where(flat.isnan(), math.nan, got).view(x.shape)


def exponent(largest):
    if largest <= 0:
        return -100
    e = math.floor(math.log2(largest)) - 10
    while largest > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, -100), 100)


def exponent_above(scale):
    e = math.floor(math.log2(scale)) - 1
    while 2.0 ** e < scale:
        e += 1
    return min(max(e, -100), 100)


def kv_write(codes, scales, x, tables, lengths, cu):
    """codes (float64 values) [pages, block, heads, dim] and scales [pages, heads] changed in place by x [rows, heads, dim] (float64)."""
    pages, block, heads, _ = codes.shape
    width = tables.shape[1]
    for s in range(len(lengths)):
        n = cu[s + 1] - cu[s]
        runs = {}
        for i in range(n):
            position = lengths[s] - n + i
            if 0 <= position < width * block:
                page = int(tables[s, position // block])
                if 0 <= page < pages:
                    runs.setdefault((position // block, page), []).append((position % block, cu[s] + i))
        for (_, page), rows in runs.items():
            first = rows[0][0]
            new = x[[r for _, r in rows]]
            finite = torch.where(new.isfinite(), new.abs(), 0.0).amax((0, 2))
            for h in range(heads):
                e = exponent(float(finite[h]))
                old = float(scales[page, h])
                if first:
                    e = max(e, exponent_above(old) if old > 0 else -100)
                scale = 2.0 ** e
                if first and scale != old:
                    codes[page, :first, h] = nearest_code(codes[page, :first, h] * (old / scale))
                scales[page, h] = scale
                values = torch.where(new[:, h].isfinite(), new[:, h] / scale, math.nan)
                for (offset, _), v in zip(rows, nearest_code(values)):
                    codes[page, offset, h] = v


# ---- attention ----------------------------------------------------------------------------------------
def attention(q, codes, scales, tables, lengths, cu, *, scale=None, window=0, out=None):
    """(result, slack): float64 [rows, heads, dim], and how far a kernel's sum may be from it before its last rounding, for weights rounded
    to `weights` relative (see `slack`): both as plain sums over the keys a row sees.  codes / scales: (key, value) pairs in float64."""
    rows, heads, dim = q.shape
    kv_heads = codes[0].shape[2]
    group = heads // kv_heads
    block = codes[0].shape[1]
    scale = dim ** -0.5 if scale is None else scale
    result = torch.zeros(rows, heads, dim, dtype=torch.float64) if out is None else out.double().clone()
    spread = torch.zeros(rows, heads, dim, dtype=torch.float64)      # sum of p |v|
    size = torch.zeros(rows, heads, 1, dtype=torch.float64)          # the largest scale * sum |q| |k|
    tiny = torch.zeros(rows, heads, 1, dtype=torch.float64)          # number of keys times the largest p * value scale
    count = torch.zeros(rows, 1, 1, dtype=torch.float64)
    for s in range(len(lengths)):
        n = cu[s + 1] - cu[s]
        for i in range(n):
            row = cu[s] + i
            keys = min(max(lengths[s] - n + i + 1, 0), tables.shape[1] * block)
            low = max(keys - window, 0) if window else 0
            result[row] = 0
            if keys <= low:
                continue
            t = torch.arange(low, keys)
            page = tables[s, t // block].long()
            k = codes[0][page, t % block] * scales[0][page][:, :, None]
            v = codes[1][page, t % block] * scales[1][page][:, :, None]
            for h in range(heads):
                a = q[row, h].double()
                score = scale * (k[:, h // group] @ a)
                p = torch.softmax(score, 0)
                result[row, h] = p @ v[:, h // group]
                spread[row, h] = p @ v[:, h // group].abs()
                size[row, h] = abs(scale) * (k[:, h // group].abs() @ a.abs()).max()
                tiny[row, h] = len(t) * (p * scales[1][page, h // group]).max()
            count[row] = len(t)
    return result, (spread, size, tiny, count)


def allowed(result, parts, dtype, dim, tiles, expanded=False):
    """How far a kernel's output may be from `result`, element by element.

    Half a step of the output's type, eps / 2 * |result|, and the weights' errors, each of which moves the output by at most its relative
    size times sum p |v| (twice where it enters the denominator too):
      scores: products of a row add up in fp32, dim roundings (the tensor cores cut instead of rounding: eps, not eps / 2) of at most
              the sum of |q| |k|; q as three parts of four bits at its largest element's size holds fp16's eleven bits and bf16's eight, and is
              off by half of the last part's smallest step, 2^-10 / 1024 of a largest of 2^7: 2^-27 of it per element, which adds up to at
              most eps of the sum for the sizes tested; times 2
      2^x:    two steps of fp32, 2^-22; the factor 2^(M_c - M) of a part again; sums of `count` terms in fp32: count * 2^-24; times 2
      tiles:  weights are rounded to half precision, 2^-11, and held as three parts of four significant bits, of which eleven bits need no more
              (a part leaves at most 2^-4 of what it took: 2^-4, 2^-8, then three bits for the last); the parts' smallest steps are those of
              the codes, 2^-9 / 1024, half of it 2^-20, at a largest p * value scale of at least 2^6: 2^-26 of it, per key, times
              the largest code 448
      expanded (long portions in bfloat16, over pages expanded into bfloat16 without a rounding): weights are rounded to bfloat16, half a step
              of 2^-7, before they meet the values, not in their sum; q is taken as it is."""
    spread, size, tiny, count = parts
    eps = torch.finfo(torch.float32).eps
    weight = 2 * (dim * eps * size + eps * size) + 2 * (4 * 2.0 ** -22 + count * eps / 2)
    if tiles:
        weight = weight + (2.0 ** -8 if expanded else 2.0 ** -11)
    total = spread * weight + torch.finfo(dtype).eps / 2 * result.abs() + torch.finfo(torch.float32).tiny
    if dtype == torch.float16:
        total = total + 2.0 ** -25                                   # half a step of its smallest numbers
    return total + (tiny * 448 * 2.0 ** -26 if tiles else 0)


# ---- inputs -------------------------------------------------------------------------------------------
def make_cache(pages, block, heads, dim, g, *, layers=1, layer=0, poison=True):
    """A layer's codes and scales inside a pool of several, as the user has them: strided views on the CPU, all bytes random (NaN among them
    unless not `poison`), scales powers of two between 2^-3 and 2^3 for keys and for values."""
    raw = torch.randint(0, 256, (2, pages, layers, block, heads, dim), generator=g, dtype=torch.uint8)
    # most magnitudes around one, as codes of a filled page have them, some at the edges
    small = (torch.randint(0x28, 0x58, raw.shape, generator=g, dtype=torch.uint8) | (raw & 0x80))
    raw = torch.where(torch.rand(raw.shape, generator=g) < 0.02, raw, small)
    raw = torch.where((raw & 0x7f) == 0x7f, raw ^ 1, raw)            # no NaN among what is stored
    scales = torch.exp2(torch.randint(-3, 4, (2, pages, layers, heads), generator=g).float())
    return raw, scales
