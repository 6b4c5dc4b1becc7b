"""A paged key/value cache in 8 bits, as a serving step uses it: where the step's rows go (pages claimed and slots mapped on the GPU), storing
keys and values with a scale for each page and head, and attention that reads them back.

Codes are e4m3, scales are powers of two.  `run` computes a case with elementary tensor operations, or with the framework's calls where `own`
is true."""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
CODE = torch.float8_e4m3fn
LARGEST = 448.0                    # the largest code
SCALES = (-100, 100)               # exponents that a scale may have
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    place = lambda name, requests, fewest, most, stored, width, spare=0, block=16: dict(
        name=name, kind="place", requests=requests, fewest=fewest, most=most, stored=stored, width=width, spare=spare, block=block)
    store = lambda name, requests, fewest, most, stored, heads, dim, block=16, type="bfloat16": dict(
        name=name, kind="store", requests=requests, fewest=fewest, most=most, stored=stored, heads=heads, dim=dim, block=block, type=type)
    attend = lambda name, requests, new, shortest, longest, heads, kv_heads, dim=128, window=0, block=16, type="bfloat16": dict(
        name=name, kind="attend", requests=requests, new=new, shortest=shortest, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim,
        window=window, block=block, type=type)
    return [
        # A decoding batch grows by one token per request; one request in sixteen opens a page.
        place("place decode 64", 64, 1, 1, 2048, 256),
        # Prompts of a serving batch come in, beside requests that wait.
        place("place prompts 16", 16, 0, 2047, 0, 256),
        # A full house with portions of every length over long tables, in a step of a fixed number of rows.
        place("place mixed 1024", 1024, 1, 37, 16000, 1025, 59),
        # The new keys and values of a decoding batch, eight key/value heads.
        store("store decode 128", 128, 1, 1, 2048, 8, 128),
        # Prompts U[128, 1024] of sixteen heads.
        store("store prompts 16", 16, 128, 1024, 0, 16, 128),
        # Ragged portions into 8-token pages, heads of an unusual size, 32-bit rows.
        store("store ragged 53", 53, 1, 33, 700, 5, 80, 8, "float32"),
        # One user's next token over a short context: nothing but latency.
        attend("attend one 500", 1, 1, 500, 500, 16, 16),
        # Verification of 64 requests at once: sixteen rows each (four tokens at four depths of a shared plane), contexts U[512, 4096].
        attend("attend verify 64", 64, 16, 512, 4096, 16, 16),
        # A large decoding batch with grouped heads.
        attend("attend grouped 128", 128, 1, 100, 2048, 32, 8),
        # A few very long contexts, five verification rows each.
        attend("attend long 4", 4, 5, 65001, 131072, 32, 8),
        # 64-wide heads behind a window, half precision, larger pages.
        attend("attend window 96", 96, 3, 200, 4096, 32, 16, 64, 1000, 32, "float16"),
        # A portion of a prompt over what is stored already.
        attend("attend prompts 4", 4, 1021, 1021, 4096, 16, 8),
    ]


def _between(rng, low, high):
    """A whole number, spread over its logarithm where the range is wide."""
    if high > 10 * max(low, 1):
        return int(round(math.exp(rng.uniform(math.log(max(low, 1)), math.log(high)))))
    return rng.randint(low, high)


def draw(rng):
    kind = rng.choice(("place", "store", "attend", "attend"))
    block = rng.choice((16, 16, 32, 64))
    if kind == "place":
        requests, most = _between(rng, 1, 1024), _between(rng, 1, 2000)
        most = max(1, min(most, 65536 // requests))
        stored = _between(rng, 1, 16000)
        return dict(kind=kind, requests=requests, fewest=rng.choice((0, 1)), most=most, stored=stored, width=-(-(stored + most) // block) + rng.randint(0, 9),
                    spare=rng.choice((0, rng.randint(1, 99))), block=block)
    if kind == "store":
        requests, most = _between(rng, 1, 256), _between(rng, 1, 1000)
        heads, dim = rng.choice(((16, 128), (8, 128), (16, 64), (2, 128), (5, 80)))
        most = max(1, min(most, 8192 // requests))
        return dict(kind=kind, requests=requests, fewest=rng.randint(0, 1), most=most, stored=_between(rng, 1, 3000), heads=heads, dim=dim,
                    block=rng.choice((8, block)), type=rng.choice(("bfloat16", "bfloat16", "float16", "float32")))
    heads, kv_heads = rng.choice(((16, 16), (32, 8), (32, 8), (16, 8), (14, 2), (32, 16)))
    dim = rng.choice((128, 128, 64))
    room = 500_000_000 // (kv_heads * dim * 2)         # tokens of all contexts together
    longest = min(_between(rng, 2, 100_000), room)
    requests = max(1, min(_between(rng, 1, 128), room // longest))
    if rng.random() < 0.2:
        longest = min(longest, 4000)
        requests = max(1, min(requests, 4))
        new = _between(rng, min(17, longest), min(1000, longest))
    else:
        new = min(rng.choice((1, 1, 1, 2, 5, 8, 16)), longest)
    window = rng.choice((0, 0, 0, _between(rng, 1, 4000)))
    return dict(kind=kind, requests=requests, new=new, shortest=rng.randint(new, longest), longest=longest, heads=heads, kv_heads=kv_heads,
                dim=dim, window=window, block=block, type=rng.choice(("bfloat16", "bfloat16", "float16")))


def _sizes(case):
    """The requests' lengths and portions: the case's own, whatever the seed."""
    rng = random.Random("-".join(str(case[k]) for k in sorted(case) if k != "name"))
    n = case["requests"]
    if case["kind"] == "attend":
        ends = [rng.randint(case["shortest"], case["longest"]) for _ in range(n)]
        ends[0] = case["longest"]
        counts = [case["new"] if i == 0 else rng.randint(1, case["new"]) for i in range(n)] if case["new"] > 1 else [1] * n
        return [e - c for e, c in zip(ends, counts)], counts
    counts = [rng.randint(case["fewest"], case["most"]) for _ in range(n)]
    counts[0] = case["most"]
    return [rng.randint(min(case["stored"], 1), case["stored"]) for _ in range(n)], counts


def _words(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _sum_before(counts):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return total


def _tables(pages, width, g):
    """Tables that hold so many pages of each request, the pages in no order, and how many there are."""
    total = sum(pages)
    order = torch.randperm(total, generator=g, device=DEVICE).int()
    held = torch.tensor(pages, device=DEVICE)
    at = torch.tensor(_sum_before(pages)[:-1], device=DEVICE)[:, None] + torch.arange(width, device=DEVICE)
    inside = torch.arange(width, device=DEVICE) < held[:, None]
    return torch.where(inside, order[at.clamp_max(max(total - 1, 0))] if total else 0, 0).int().contiguous(), total


def _codes(values):
    """Codes and power-of-two scales of [pages, block, heads, dim] values: a scale for each page and head."""
    scale = _scale_of(values.abs().amax(dim=(1, 3)))
    return (values / scale[:, None, :, None]).to(CODE), scale


def _scale_of(largest):
    """2^e with the smallest e for which `largest` is at most 448 * 2^e."""
    part, exponent = torch.frexp(largest)              # largest = part * 2^exponent, part in [0.5, 1)
    e = exponent - 9 + (part > 0.875).int()            # 448 = 0.875 * 2^9
    e = torch.where(largest > 0, e, torch.full_like(e, SCALES[0])).clamp(*SCALES)
    return torch.ldexp(torch.ones_like(largest), e)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    stored, counts = _sizes(case)
    n, block, kind = case["requests"], case["block"], case["kind"]
    ends = [a + c for a, c in zip(stored, counts)]
    rows = sum(counts)
    state = dict(case=case, rows=rows)
    if kind == "place":
        held = [-(-a // block) for a in stored]
        need = sum(max(-(-e // block) - h, 0) for e, h in zip(ends, held))
        tables, taken = _tables(held, case["width"], g)
        free = need + 7
        state.update(rows=rows + case["spare"], lengths=_words(stored), counts=_words(counts), tables=tables, held=_words(held),
                     free_pages=(torch.randperm(free, generator=g, device=DEVICE) + taken).int(), free_count=_words([free]))
        return state
    pages = [-(-e // block) for e in ends]
    heads, dim, dtype = case["heads"] if kind == "store" else case["kv_heads"], case["dim"], TYPES[case["type"]]
    tables, total = _tables(pages, max(pages + [1]), g)
    codes = torch.empty(2, total, block, heads, dim, dtype=CODE, device=DEVICE)
    scales = torch.empty(2, total, heads, device=DEVICE)
    size = torch.exp2(torch.randint(-2, 2, (heads, 1), generator=g, device=DEVICE).float()) * torch.exp(0.5 * torch.randn(heads, dim, generator=g, device=DEVICE))
    for i in range(2):                                 # heads and channels of unlike sizes, as keys and values have them
        for at in range(0, total, 16384):
            part = torch.randn(min(16384, total - at), block, heads, dim, generator=g, device=DEVICE).mul_(size)
            codes[i, at:at + part.shape[0]], scales[i, at:at + part.shape[0]] = _codes(part)
    state.update(codes=codes, scales=scales, tables=tables, lengths=_words(ends), cu=_words(_sum_before(counts)), new=max(counts), longest=max(ends))
    if kind == "store":
        state["k"], state["v"] = ((torch.randn(rows, heads, dim, generator=g, device=DEVICE) * size).to(dtype) for _ in range(2))
    else:
        q = torch.randn(rows, case["heads"], dim, generator=g, device=DEVICE)
        state["q"] = (q / size.repeat_interleave(case["heads"] // heads, 0).clamp_min(0.25)).to(dtype)
    return state


# ---- the plain forms ---------------------------------------------------------------------------------
def _place(state):
    """Pages claimed from the end of the stack in the order of the requests, the step's rows mapped to their slots, and the pages given back."""
    block, rows = state["case"]["block"], state["rows"]
    lengths, counts, tables, held, free, free_count = (state[k] for k in ("lengths", "counts", "tables", "held", "free_pages", "free_count"))
    n, width = tables.shape
    ends = lengths + counts.clamp_min(0)
    cu = torch.zeros(n + 1, dtype=torch.int32, device=DEVICE)
    cu[1:] = counts.clamp_min(0).cumsum(0)
    need = ((ends + block - 1) // block - held).clamp_min(0)
    before = need.cumsum(0) - need
    refused = (cu[-1] > rows) | (need.sum() > free_count[0]) | (ends > width * block).any() | (lengths < 0).any()
    page = torch.arange(width, device=DEVICE)
    new = (page >= held[:, None]) & (page < (held + need)[:, None]) & ~refused
    which = free_count.long() - 1 - (before[:, None] + page - held[:, None])
    tables.copy_(torch.where(new, free[which.clamp(0, free.numel() - 1)], tables))
    held.add_(torch.where(refused, 0, need))
    free_count.sub_(torch.where(refused, 0, need.sum()).int())
    cu = torch.where(refused, 0, cu).int()
    after = torch.where(refused, lengths, ends)
    row = torch.arange(rows, device=DEVICE)
    owner = torch.searchsorted(cu[1:].contiguous(), row.int(), right=True)
    active = row < cu[-1]
    owner = owner.clamp_max(n - 1)
    positions = torch.where(active, lengths[owner] + row - cu[owner], 0).int()
    blocks = torch.where(active, tables[owner, (positions // block).clamp_max(width - 1).long()], -1).long()
    offsets = torch.where(active, positions % block, 0).long()
    owner = torch.where(active, owner, -1).int()
    # the pages of what is taken back go onto the stack again
    keep = (lengths.clamp_min(0) + block - 1) // block
    given = (held - keep).clamp_min(0)
    first = given.cumsum(0) - given
    leaving = (page >= keep[:, None]) & (page < held[:, None])
    place = free_count.long() + given.sum() - 1 - (first[:, None] + page - keep[:, None])
    free.scatter_(0, place[leaving], tables[leaving])
    free_count.add_(given.sum().int())
    held.copy_(torch.minimum(held, keep))
    return [cu, after, positions, owner, blocks, offsets, refused.int(), cu[-1], tables, held, free, free_count]


def _slots(tables, lengths, cu, rows, block, new):
    """Page and offset of every row, and its request."""
    owner = torch.searchsorted(cu[1:].contiguous(), torch.arange(rows, device=DEVICE, dtype=torch.int32), right=True)
    positions = (lengths[owner] - cu[owner + 1] + torch.arange(rows, device=DEVICE)).long()
    return tables[owner, positions // block].long(), positions % block


def _store(state):
    """Each page's and head's scale grows to what its new rows need; what the page holds already is rounded at the new scale, the rows go behind it."""
    codes, scales, block = state["codes"], state["scales"], state["case"]["block"]
    if not state["rows"]:
        return [codes, scales]
    pages, offsets = _slots(state["tables"], state["lengths"], state["cu"], state["rows"], block, state["new"])
    for i, rows in enumerate((state["k"], state["v"])):
        rows = rows.float()
        largest = torch.where(rows.isfinite(), rows.abs(), 0.0).amax(-1)
        total, heads = scales[i].shape
        most = torch.full((total, heads), -1.0, device=DEVICE).scatter_reduce_(0, pages[:, None].expand_as(largest), largest, "amax")
        first = torch.full((total,), block, device=DEVICE).scatter_reduce_(0, pages, offsets, "amin")
        old = _scale_of(scales[i] * LARGEST)
        touched = most >= 0
        needed = _scale_of(most.clamp_min(0.0))
        scale = torch.where(first[:, None] == 0, needed, torch.maximum(needed, old))
        scale = torch.where(touched, scale, scales[i])
        earlier = torch.arange(block, device=DEVICE) < first[:, None]
        again = (codes[i].float() * (scales[i] / scale)[:, None, :, None]).to(CODE)
        moved = (earlier[:, :, None] & touched[:, None] & (scale != scales[i])[:, None])[..., None]
        codes[i].view(torch.uint8).copy_(torch.where(moved, again.view(torch.uint8), codes[i].view(torch.uint8)))
        new = (rows / scale[pages][:, :, None]).clamp(-LARGEST, LARGEST)
        new = torch.where(rows.isfinite(), new, math.nan).to(CODE)
        codes[i].view(torch.uint8)[pages, offsets] = new.view(torch.uint8)
        scales[i].copy_(scale)
    return [codes, scales]


def _attend(state):
    """Softmax over the keys that a row sees, all requests side by side, padded to the longest."""
    case, q, lengths, cu, tables = state["case"], state["q"], state["lengths"], state["cu"], state["tables"]
    n, block, new, window = case["requests"], case["block"], state["new"], case["window"]
    rows, heads, dim = q.shape
    kv_heads = case["kv_heads"]
    pages = tables[:, :-(-state["longest"] // block)].long()
    keys, values = ((state["codes"][i].view(torch.uint8)[pages].view(CODE).float() * state["scales"][i][pages][:, :, None, :, None]).flatten(1, 2)
                    for i in range(2))                                     # [n, tokens, kv_heads, dim]
    token = torch.arange(keys.shape[1], device=DEVICE)
    counts = cu[1:] - cu[:-1]
    place = torch.arange(new, device=DEVICE)
    row = (cu[:-1, None] + place).clamp_max(rows - 1).long()
    x = q[row].float().view(n, new, kv_heads, heads // kv_heads, dim)
    scores = torch.einsum("nmhgd,nthd->nhgmt", x, keys) / math.sqrt(dim)
    del keys
    ends = (lengths - counts)[:, None] + place + 1                          # keys that each row sees
    seen = token < ends[..., None]
    if window:
        seen = seen & (token >= ends[..., None] - window)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    values = torch.where((token < lengths[:, None])[:, :, None, None], values, 0.0)
    total = scores.sum(-1)
    out = torch.einsum("nhgmt,nthd->nmhgd", scores, values)
    out = out / torch.where(total > 0, total, 1.0).permute(0, 3, 1, 2)[..., None]
    owner = torch.searchsorted(cu[1:].contiguous(), torch.arange(rows, device=DEVICE, dtype=torch.int32), right=True)
    return out[owner, torch.arange(rows, device=DEVICE) - cu[owner]].reshape(rows, heads, dim).to(q.dtype)


def run(state):
    case = state["case"]
    if not own:
        return {"place": _place, "store": _store, "attend": _attend}[case["kind"]](state)
    import vllm_rlt_b200 as rlt
    if case["kind"] == "place":
        lengths, tables, held, free, count = (state[k] for k in ("lengths", "tables", "held", "free_pages", "free_count"))
        s = rlt.step_slots(lengths, state["counts"], tables, case["block"], state["rows"], held=held, free_pages=free, free_count=count)
        rlt.return_pages(lengths, tables, case["block"], held=held, free_pages=free, free_count=count)
        return [s.cu, s.lengths, s.positions, s.row_seq, s.write_blocks, s.write_offsets, s.status, s.active_rows, tables, held, free, count]
    cache = rlt.QuantizedKV(state["codes"][0], state["codes"][1], state["scales"][0], state["scales"][1])
    if case["kind"] == "store":
        rlt.quantized_kv_write(cache, state["k"], state["v"], state["tables"], state["lengths"], state["cu"])
        return [state["codes"], state["scales"]]
    return rlt.quantized_attention(state["q"], cache, state["tables"], state["lengths"], state["cu"], state["new"], window=case["window"])


def work(case):
    stored, counts = _sizes(case)
    n, block, rows = case["requests"], case["block"], sum(counts)
    ends = [a + c for a, c in zip(stored, counts)]
    if case["kind"] == "place":
        claimed = sum(-(-e // block) - -(-a // block) for e, a in zip(ends, stored))
        return {"bytes": 4 * 7 * n + 16 * claimed + 24 * (rows + case["spare"]), "flops": 0}
    size = TYPES[case["type"]].itemsize
    if case["kind"] == "store":
        touched = sum(-(-e // block) - a // block for e, a in zip(ends, stored) if e > a)
        values = 2 * rows * case["heads"] * case["dim"]
        return {"bytes": values * (size + 1) + 2 * 8 * touched * case["heads"], "flops": values}
    window, tokens, pairs, pages = case["window"], 0, 0, 0
    for a, e in zip(stored, ends):
        first = max(a + 1 - window, 0) if window else 0
        tokens += e - first
        pages += -(-e // block) - first // block
        pairs += sum(min(p, window) for p in range(a + 1, e + 1)) if window else (a + 1 + e) * (e - a) // 2
    return {"bytes": 2 * case["kv_heads"] * (tokens * case["dim"] + 4 * pages) + 2 * rows * case["heads"] * case["dim"] * size,
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    if case["kind"] == "place":
        return None
    state = prepare(case, seed)
    stored, counts = _sizes(case)
    at, block = _sum_before(counts), case["block"]
    tables = state["tables"].long()
    codes, scales = state["codes"], state["scales"].double()
    if case["kind"] == "attend":
        kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
        out = torch.empty(state["rows"], case["heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        for s, (a, c) in enumerate(zip(stored, counts)):
            pages = tables[s, :-(-(a + c) // block)]
            for h in range(kv_heads):
                k, v = (codes[i][:, :, h].view(torch.uint8)[pages].view(CODE).double().mul(scales[i][pages, h][:, None, None]).reshape(-1, case["dim"])[:a + c]
                        for i in range(2))
                x = state["q"][at[s]:at[s] + c, h * group:(h + 1) * group].double()
                score = x.reshape(-1, case["dim"]) @ k.t() * case["dim"] ** -0.5
                p = torch.arange(a, a + c, device=DEVICE).repeat_interleave(group)[:, None]
                t = torch.arange(a + c, device=DEVICE)
                hidden = (t > p) | (t <= p - case["window"]) if case["window"] else t > p
                out[at[s]:at[s] + c, h * group:(h + 1) * group] = (torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v).view(c, group, -1)
        return out
    # Store, page by page on the host: the codes are found among all 256, by distance.
    if state["rows"] * case["heads"] * case["dim"] > 2_000_000:
        return None
    table = torch.arange(256, dtype=torch.uint8).view(CODE).double()
    order = [c for c in range(256) if math.isfinite(float(table[c])) and c != 128]
    order.sort(key=lambda c: float(table[c]))
    grid = table[order]
    middle = (grid[1:] + grid[:-1]) / 2
    even = torch.tensor([c % 2 == 0 for c in order])

    def nearest(x):
        i = torch.searchsorted(middle, x.contiguous())               # ties fall to the lower neighbour here
        tie = (i < middle.numel()) & (x == middle[i.clamp_max(middle.numel() - 1)])
        return grid[torch.where(tie & ~even[i], i + 1, i)]

    got, scale = codes.cpu().double(), scales.cpu()
    tables = tables.cpu()
    for i, x in enumerate((state["k"].cpu().double(), state["v"].cpu().double())):
        for s, (a, c) in enumerate(zip(stored, counts)):
            for page in range(a // block, -(-(a + c) // block) if c else 0):
                low, high = max(a, page * block), min(a + c, (page + 1) * block)
                rows, p, offset = x[at[s] + low - a:at[s] + high - a], int(tables[s, page]), low - page * block
                e = torch.tensor([min(max(math.ceil(math.log2(m / LARGEST)), SCALES[0]), SCALES[1]) if m > 0 else SCALES[0] for m in rows.abs().amax((0, 2)).tolist()])
                want = torch.exp2(e.double())
                if offset:
                    want = torch.maximum(want, scale[i, p])
                    got[i, p, :offset] = nearest(got[i, p, :offset] * (scale[i, p] / want)[:, None])
                got[i, p, offset:offset + high - low] = nearest((rows / want[:, None]).clamp(-LARGEST, LARGEST))
                scale[i, p] = want
    return [got, scale]
