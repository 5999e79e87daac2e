"""Measured cases of the paged cache held in 4 bits: the attention that reads it, keys
and values appended to it and read back, and its pages forked, freed and compacted.

The cache.  Keys and values of a layer lie in `pages` [pages, kv_heads, page / 16, 18 D]
bytes; page `tables[s, i]` holds positions i * page .. of sequence s, -1 is no page, and
`refs` counts the table rows that hold a page.  A cell of 18 D bytes holds 16 positions
of one head.  Each 64 elements of a key or value share a zero z and a step s in f16,
  z = f16(min x),  s = f16(max((max x - z) / 15, 0)) (the quotient in f32),
  n = (x - z) / s rounded to the nearest of 0..15, a tie to the even one (0 where s = 0),
and stand for s n + z; where z or s is not finite both are NaN and n is 0.  Within a
cell, position t (0..15), element d:
  bytes 0 .. 8D      keys: the lane's ((t % 8) * 4 + d % 64 / 16) 16 bytes of group d / 64 hold, for
                     t / 8, two words of eight elements each, element e of a word in bits 4e
  bytes 8D .. 16D    values: the 16 bytes of lane (d % 8) * 4 + t % 8 / 2 of group d / 64 hold four words
                     d / 16 % 4, byte (t % 2) * 2 + t / 8 of a word the elements d % 16 / 8 = 0 (low bits) and 1
  bytes 16D .. 17D   keys' s and z: per group, per t % 8 / 2, per t / 8: s, s, z, z of t % 2 = 0, 1
  bytes 17D .. 18D   values' s and z likewise

Definitions.  Sequence b of a call has `lengths[b]` positions, the last n_b of them with
rows in the call, rows starts[b] .. starts[b + 1].

  attention  out = sum_t p_t v_t, p = softmax(scale q k_t) over the positions up to the
             row's own; query head h reads key head h / (q_heads / kv_heads); a row that
             sees no position is 0.
  append     writes the rows' keys and values at their positions; the case reads them
             back together with up to `before` earlier positions.
  fork       a step of a search over sequences: the children are freed, each takes its
             parent's positions (whole pages shared, a partly filled one copied to the
             lowest free page) and is given `count` further positions.
  compact    the live pages above their number move, in ascending order, into the free
             pages below it, and the tables follow.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # A test-sized model's first steps: the smallest call, where only latency counts.
        {"name": "attention_tiny", "op": "attention", "sequences": 1, "length": 9, "spread": 0.0, "queries": 1, "ragged": False,
         "q_heads": 2, "kv_heads": 1, "dim": 64, "page": 16, "type": "f32"},
        # Batched generation of 16 sequences at 4 thousand positions, with the decoder's f32 activations.
        {"name": "attention_batch16", "op": "attention", "sequences": 16, "length": 4113, "spread": 0.0, "queries": 1,
         "ragged": False, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "type": "f32"},
        # One sequence with a long context: all SMs share its positions.
        {"name": "attention_one_long", "op": "attention", "sequences": 1, "length": 131072, "spread": 0.0, "queries": 1,
         "ragged": False, "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16"},
        # A server's step: sequences of very different lengths, groups of seven query heads.
        {"name": "attention_ragged", "op": "attention", "sequences": 61, "length": 5000, "spread": 1.3, "queries": 1,
         "ragged": False, "q_heads": 28, "kv_heads": 4, "dim": 128, "page": 32, "type": "f16"},
        # Up to six drafted tokens a sequence are verified at once, wide heads.
        {"name": "attention_draft", "op": "attention", "sequences": 12, "length": 6001, "spread": 0.3, "queries": 6,
         "ragged": True, "q_heads": 16, "kv_heads": 8, "dim": 256, "page": 16, "type": "bf16"},
        # Two parts of prompts behind what the cache holds already.
        {"name": "attention_prompt", "op": "attention", "sequences": 2, "length": 7001, "spread": 0.1, "queries": 1024,
         "ragged": True, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16"},
        # The step's new keys and values of 16 sequences.
        {"name": "append_batch16", "op": "append", "sequences": 16, "length": 4113, "spread": 0.0, "queries": 1,
         "ragged": False, "kv_heads": 8, "dim": 128, "page": 64, "type": "f32", "before": 3},
        # Prompts of several lengths enter the cache.
        {"name": "append_prompts", "op": "append", "sequences": 5, "length": 5001, "spread": 0.6, "queries": 4096,
         "ragged": True, "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "before": 21},
        # Four beams of a search replaced by forks, a test-sized model.
        {"name": "fork_beams", "op": "fork", "layers": 2, "pages": 64, "rows": 12, "parents": 2, "children": 4, "length": 70,
         "kv_heads": 1, "dim": 64, "page": 16, "count": 1, "kind": "u8"},
        # 48 samples from six prompts in a decoder of 36 layers.
        {"name": "fork_samples", "op": "fork", "layers": 36, "pages": 600, "rows": 64, "parents": 6, "children": 48,
         "length": 2500, "kv_heads": 8, "dim": 128, "page": 64, "count": 5, "kind": "u8"},
        # A quarter of a small cache's pages are free, in two places.
        {"name": "compact_small", "op": "compact", "layers": 2, "pages": 100, "rows": 9, "free": 25, "holes": 13, "kv_heads": 2,
         "dim": 64, "page": 32, "kind": "f16"},
        # Sequences that ended leave holes all over a large cache.
        {"name": "compact_large", "op": "compact", "layers": 28, "pages": 700, "rows": 50, "free": 280, "holes": 170,
         "kv_heads": 8, "dim": 128, "page": 64, "kind": "u8"},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "fork", "compact"])
    heads, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 192, 256])
    page = rng.choice([16, 32, 48, 64, 128])
    if op in ("attention", "append"):
        case = {"op": op, "sequences": _spread(rng, 1, 150), "spread": rng.choice([0.0, round(rng.random(), 2)])}
        if op == "attention":
            queries = rng.choice([1, 1, 1, rng.randint(2, 8), _spread(rng, 9, 900)])
            case["q_heads"] = heads * rng.choice([1, 2, 4, 8, rng.randint(1, 20)])
        else:
            queries = rng.choice([1, rng.randint(2, 40), _spread(rng, 40, 4000)])
            case["before"] = rng.randint(0, 40)
        budget = 16_000_000 // (heads * dim) if queries <= 8 else 12000
        case["sequences"] = max(1, min(case["sequences"], budget // (2 * queries)))
        case["length"] = max(queries, _spread(rng, 1, max(2, min(100_000, budget // case["sequences"]))))
        if rng.random() < 0.5:
            case["length"] |= 1
        case.update({"queries": queries, "ragged": queries > 1 and rng.random() < 0.7, "kv_heads": heads, "dim": dim,
                     "page": page, "type": rng.choice(["f32", "f16", "bf16"])})
        return case
    kind = rng.choice(["u8", "u8", "f16", "f32"])
    width = {"u8": 1, "f16": 2, "f32": 4}[kind]
    case = {"op": op, "layers": rng.choice([1, 2, rng.randint(3, 40)]), "kv_heads": heads, "dim": dim, "page": page, "kind": kind}
    bytes_of_page = case["layers"] * heads * (page // 16) * 18 * dim * width
    pages = max(24, min(_spread(rng, 24, 3000), 700_000_000 // bytes_of_page))
    if op == "fork":
        parents, children = rng.randint(1, 8), _spread(rng, 1, 48)
        length = _spread(rng, 1, max(2, (pages // 2 // parents) * page))
        count = rng.choice([0, 1, rng.randint(1, 40)])
        # room for every parent, every child's copy and its further positions
        children = max(1, min(children, (pages - parents * (-(-length // page))) // (2 + count // page + 1)))
        case.update({"pages": pages, "rows": parents + children + rng.randint(0, 9), "parents": parents, "children": children,
                     "length": length, "count": count})
        return case
    free = rng.randint(1, pages - 4)
    case.update({"pages": pages, "rows": rng.randint(1, 60), "free": free, "holes": rng.randint(0, min(free, pages - free))})
    return case


# ---- the cells' layout ---------------------------------------------------------
def _offsets(dim, device):
    """[16, 18 D / 16] byte offsets in a cell of each position's bytes: key nibbles, value nibbles, key s, key z,
    value s, value z (two bytes each)."""
    t = np.arange(16)[:, None]
    e = np.arange(0, dim, 2)[None]  # a byte of keys holds elements e and e + 1
    keys = (e // 64 * 32 + t % 8 * 4 + e % 64 // 16) * 16 + t // 8 * 8 + e % 16 // 2
    u = np.arange(dim // 16).repeat(8)[None]  # a byte of values holds elements 16 u + i and 16 u + 8 + i
    i = np.tile(np.arange(8), dim // 16)[None]
    values = 8 * dim + (u // 4 * 32 + i * 4 + t % 8 // 2) * 16 + u % 4 * 4 + t % 2 * 2 + t // 8
    g = np.arange(dim // 64)[None]
    s = 16 * dim + g * 64 + t % 8 // 2 * 16 + t // 8 * 8 + t % 2 * 2
    pair = lambda a: (a[:, :, None] + np.arange(2)).reshape(16, -1)  # noqa: E731
    table = np.concatenate([keys, values, pair(s), pair(s + 4), pair(s + dim), pair(s + dim + 4)], 1)
    return torch.from_numpy(table).to(device)


def _group(x):
    """Levels 0..15, s and z of x [..., D] in f32, level decisions in 64 bits."""
    x = x.float().unflatten(-1, (-1, 64))
    z = x.amin(-1).half() + 0.0
    step = (x.amax(-1) - z.float()) / torch.full((), 15.0, device=x.device)
    s = torch.maximum(step, torch.zeros_like(step)).half()
    bad = ~(torch.isfinite(s.float()) & torch.isfinite(z.float()))
    n = (x.double() - z.double()[..., None]) / s.double()[..., None]
    n = torch.where((bad | (s == 0))[..., None], 0.0, n.round().clamp(0, 15)).nan_to_num(0.0)
    nan = torch.full_like(s, math.nan)
    return n.to(torch.uint8).flatten(-2), torch.where(bad, nan, s), torch.where(bad, nan, z)


def _encode(k, v):
    """The bytes of each position [T, heads, 18 D / 16] in _offsets' order."""
    (kn, ks, kz), (vn, vs, vz) = _group(k), _group(v)
    kb = kn[..., 0::2] | (kn[..., 1::2] << 4)
    vn = vn.unflatten(-1, (-1, 2, 8))
    vb = (vn[..., 0, :] | (vn[..., 1, :] << 4)).flatten(-2)
    return torch.cat([kb, vb] + [a.contiguous().view(torch.uint8) for a in (ks, kz, vs, vz)], -1)


def _decode(raw):
    """Keys and values [..., D] in f32 of bytes [..., 18 D / 16] in _offsets' order."""
    dim = raw.shape[-1] * 16 // 18
    kb, vb = raw[..., :dim // 2], raw[..., dim // 2:dim]
    ks, kz, vs, vz = (a.contiguous().view(torch.float16).float() for a in raw[..., dim:].split(dim // 32, -1))
    kn = torch.stack([kb & 15, kb >> 4], -1).flatten(-2).float().unflatten(-1, (-1, 64))
    vb = vb.unflatten(-1, (-1, 8))
    vn = torch.stack([vb & 15, vb >> 4], -2).flatten(-3).float().unflatten(-1, (-1, 64))
    return ((kn * ks[..., None] + kz[..., None]).flatten(-2), (vn * vs[..., None] + vz[..., None]).flatten(-2))


def _cells(pages, table, positions, at):
    """Byte rows [T, heads, 18 D / 16] of positions (1-d tensor) of a sequence's table row."""
    size = pages.shape[2] * 16
    page = table[positions // size].long()
    cell = pages[page, :, positions % size // 16]
    index = at[positions % 16][:, None].expand(-1, pages.shape[1], -1)
    return torch.gather(cell, 2, index)


# ---- inputs --------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _shape(case):
    """Each sequence's positions and its rows in the call: whole numbers that go by the case alone."""
    rng = random.Random(repr(sorted(case.items())).replace(repr(case.get("name")), ""))
    lengths, queries = [], []
    for b in range(case["sequences"]):
        length = max(1, int(case["length"] * math.exp(rng.gauss(0.0, case["spread"]) - case["spread"] ** 2 / 2)))
        n = min(length, case["queries"])
        if case["ragged"]:
            n = rng.randint(min(length, case["queries"] // 2), n)
        lengths.append(length)
        queries.append(n)
    if case["op"] == "attention" and not case["ragged"] and case["sequences"] > 8 and case["spread"]:
        lengths[3] = 0  # a sequence that holds nothing yet (one that is appended to holds its rows)
    return lengths, queries


def prepare(case, seed):
    g, dev = _generator(seed), "cuda"
    if case["op"] in ("fork", "compact"):
        return _prepare_pages(case, g, seed)
    H, D, size, dtype = case["kv_heads"], case["dim"], case["page"], _TYPES[case["type"]]
    lengths, queries = _shape(case)
    width = max(1, max(-(-n // size) for n in lengths)) + 1
    used = sum(-(-n // size) for n in lengths)
    order = torch.randperm(used + 3, generator=g, device=dev).to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device=dev)
    first = 0
    for b, n in enumerate(lengths):
        tables[b, :-(-n // size)] = order[first:first - (-n // size)]
        first += -(-n // size)
    starts = np.concatenate([[0], np.cumsum(queries)])
    s = {"case": dict(case), "tables": tables, "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
         "host": (lengths, queries), "offsets": _offsets(D, dev),
         "starts": torch.tensor(starts, dtype=torch.int32, device=dev) if case["queries"] > 1 else None}
    # cells of ordinary keys and values: a few pages' worth of encoded rows, taken in a random order
    pages = torch.empty(used + 3, H, size // 16, 18 * D, dtype=torch.uint8, device=dev)
    flat = pages.view(-1, 18 * D)
    stock = min(flat.shape[0], 4096)
    tokens = stock * 16
    k = torch.randn(tokens, 1, D, generator=g, device=dev) * (0.4 + 2.0 * torch.rand(D, generator=g, device=dev))
    k += 1.5 * torch.randn(D, generator=g, device=dev)
    v = torch.randn(tokens, 1, D, generator=g, device=dev) + 0.3 * torch.randn(D, generator=g, device=dev)
    raw = _encode(k, v).view(stock, 16, 18 * D // 16)
    cells = torch.empty(stock, 18 * D, dtype=torch.uint8, device=dev)
    cells.scatter_(1, s["offsets"].flatten()[None].expand(stock, -1), raw.flatten(1))
    for a in range(0, flat.shape[0], 1 << 16):
        b = min(flat.shape[0], a + (1 << 16))
        flat[a:b] = cells[torch.randint(0, stock, (b - a,), generator=g, device=dev)]
    s["pages"] = pages
    R = int(starts[-1])
    if case["op"] == "attention":
        s["scale"] = D ** -0.5
        s["q"] = torch.randn(R, case["q_heads"], D, generator=g, device=dev).to(dtype)
        s["out"] = torch.zeros_like(s["q"])
        return s
    packed = torch.randn(R, 2 * H * D + 24, generator=g, device=dev).to(dtype)  # rows of a wider buffer
    s["k"], s["v"] = packed[:, 8:8 + H * D].view(R, H, D), packed[:, 8 + H * D:8 + 2 * H * D].view(R, H, D)
    back = [min(a, n + case["before"]) for a, n in zip(lengths, queries)]
    s["back"] = back
    s["back_starts"] = torch.tensor(np.concatenate([[0], np.cumsum(back)]), dtype=torch.int32, device=dev)
    s["out"] = tuple(torch.zeros(sum(back), H, D, device=dev) for _ in range(2))
    return s


def _pool(case, g):
    shape = (case["layers"], case["pages"], case["kv_heads"], case["page"] // 16, 18 * case["dim"])
    if case["kind"] == "u8":
        pool = torch.empty(shape, dtype=torch.uint8, device="cuda")
        pool.view(torch.int64).random_(generator=g)  # cells are a multiple of 8 bytes
        return pool
    return torch.randn(shape, generator=g, device="cuda").to(_TYPES[case["kind"]])


def _parent_length(case, i):
    return max(1, case["length"] - i * 5 % (case["page"] // 2))


def _prepare_pages(case, g, seed):
    rng = random.Random(f"pages {seed}")
    N, size = case["pages"], case["page"]
    s = {"case": dict(case), "pool": _pool(case, g)}
    if case["op"] == "fork":
        need = -(-case["length"] // size)
        width = need + case["count"] // size + 3
        tables = np.full((case["rows"], width), -1, np.int32)
        lengths, refs = np.zeros(case["rows"], np.int32), np.zeros(N, np.int32)
        rows = rng.sample(range(case["rows"]), case["parents"] + case["children"])
        parents, children = rows[:case["parents"]], rows[case["parents"]:]
        ids = rng.sample(range(N), need * len(parents))
        for i, p in enumerate(parents):
            n = _parent_length(case, i)
            pages = -(-n // size)
            tables[p, :pages] = ids[i * need:i * need + pages]
            refs[tables[p, :pages]] = 1
            lengths[p] = n
        of = [parents[i % len(parents)] for i in range(len(children))]
        rng.shuffle(of)
        counts = [case["count"]] * len(children)
        for name, a in (("parents", of), ("children", children), ("counts", counts)):
            s[name] = torch.tensor(a, dtype=torch.int32, device="cuda")
        s["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["lengths"] = torch.from_numpy(lengths).cuda()
    else:
        live = N - case["free"]
        holes = rng.sample(range(live), case["holes"])
        high = rng.sample(range(live, N), case["holes"])
        alive = sorted(set(range(live)) - set(holes) | set(high))
        rng.shuffle(alive)
        width = -(-live // case["rows"]) + 5
        tables = np.full((case["rows"], width), -1, np.int32)
        refs = np.zeros(N, np.int32)
        for i, p in enumerate(alive):
            tables[i % case["rows"], i // case["rows"]] = p
            refs[p] += 1
        for r in range(1, case["rows"], 3):  # rows that share their first pages
            tables[r, width - 5:width - 3] = tables[0, 0]
            refs[tables[0, 0]] += 2
        s["out"] = (torch.empty(case["rows"], width, dtype=torch.int32, device="cuda"),
                    torch.empty(N, dtype=torch.int32, device="cuda"))
    s["tables"], s["refs"] = torch.from_numpy(tables).cuda(), torch.from_numpy(refs).cuda()
    return s


# ---- the plain forms -------------------------------------------------------------
def _plain_attention(s):
    c, q = s["case"], s["q"]
    H, group = c["kv_heads"], c["q_heads"] // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    row = 0
    for b, (length, n) in enumerate(zip(*s["host"])):
        if n and length:
            at = torch.arange(length, device=q.device)
            k, v = _decode(_cells(s["pages"], s["tables"][b], at, s["offsets"]).transpose(0, 1))
            rows = q[row:row + n].float().unflatten(1, (H, group)).permute(1, 2, 0, 3).flatten(1, 2)  # [H, group n, D]
            score = torch.matmul(rows, k.transpose(1, 2)).mul_(s["scale"])
            if n > 1:
                own_position = torch.arange(length - n, length, device=q.device).repeat(group)
                score.masked_fill_(at > own_position[:, None], -math.inf)
            score = torch.exp(score.sub_(score.amax(2, keepdim=True)))
            got = torch.matmul(score, v) / score.sum(2, keepdim=True)
            out[row:row + n] = got.unflatten(1, (group, n)).permute(2, 0, 1, 3).flatten(1, 2)
        row += n
    return out.to(q.dtype)


def _positions(lengths, rows, device):
    """(sequence, position) of each row of a call."""
    b = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows)).to(device)
    at = torch.cat([torch.arange(a - n, a) for a, n in zip(lengths, rows)]).to(device)
    return b, at


def _plain_append(s):
    pages, dev = s["pages"], s["pages"].device
    size, H = pages.shape[2] * 16, pages.shape[1]
    lengths, queries = s["host"]
    b, at = _positions(lengths, queries, dev)
    page = s["tables"][b, at // size].long()
    cell = (page[:, None] * H + torch.arange(H, device=dev)) * (size // 16) + (at % size // 16)[:, None]
    index = cell[:, :, None] * pages.shape[3] + s["offsets"][at % 16][:, None]
    pages.view(-1).index_copy_(0, index.flatten(), _encode(s["k"], s["v"]).flatten())
    b, at = _positions(lengths, s["back"], dev)
    page = s["tables"][b, at // size].long()
    cell = pages[page, :, at % size // 16]
    return list(_decode(torch.gather(cell, 2, s["offsets"][at % 16][:, None].expand(-1, H, -1))))


def _free_pages(refs):
    """Page ids, the free ones first, in ascending order."""
    return torch.sort((refs > 0).int(), stable=True).indices.int()


def _plain_fork(s):
    c, size = s["case"], s["case"]["page"]
    pool, tables, lengths, refs = s["pool"], s["tables"], s["lengths"], s["refs"]
    parents, children = s["parents"].long(), s["children"].long()
    N, width = refs.shape[0], tables.shape[1]

    def count(pages, by):
        held = torch.where(pages >= 0, pages, N).long().flatten()
        refs.add_(torch.zeros(N + 1, dtype=torch.int32, device=refs.device).index_add_(
            0, held, torch.full(held.shape, by, dtype=torch.int32, device=refs.device))[:N])

    def place(rows, slots, wanted):
        """Gives the wanted [n, w] table slots the lowest free pages, row by row."""
        rank = wanted.flatten().int().cumsum(0) - 1
        ids = torch.where(wanted.flatten(), _free_pages(refs)[rank.clamp_min(0)], -1).view(wanted.shape)
        tables[rows[:, None], slots] = torch.where(wanted, ids, tables[rows[:, None], slots])
        count(ids, 1)
        return ids

    # the children are freed
    count(tables[children], -1)
    tables[children] = -1
    lengths[children] = 0
    # and forked
    n = lengths[parents]
    whole = n // size
    held = torch.where(torch.arange(width, device=n.device) < whole[:, None], tables[parents], -1)
    tables[children] = held
    count(held, 1)
    part = (n % size > 0)[:, None]
    to = place(children, whole[:, None].long(), part)
    source = tables[parents, whole.clamp_max(width - 1).long()]
    to = torch.where(part, to, source[:, None])[:, 0].long()
    pool[:, to] = torch.where(part[:, 0][None, :, None, None, None], pool[:, source.long()], pool[:, to])
    lengths[children] = n
    # and given further positions
    end = n + s["counts"]
    before, after = -(-n // size), -(-end // size)
    slots = torch.arange(c["count"] // size + 2, device=n.device) + before[:, None]
    place(children, slots.clamp_max(width - 1).long(), slots < after[:, None])
    lengths[children] = end
    return [pool, tables, lengths, refs, s["missing"]]


def _plain_compact(s):
    pool, tables, refs = s["pool"], s["tables"], s["refs"]
    N, most = refs.shape[0], s["case"]["holes"]
    alive = refs > 0
    low = torch.arange(N, device=refs.device) < alive.sum()
    to = torch.sort((alive | ~low).int(), stable=True).indices[:most]     # free pages below the number of live ones
    source = torch.sort((~(alive & ~low)).int(), stable=True).indices[:most]  # live pages above it
    for layer in pool:
        layer[to] = layer[source]
    moved = torch.arange(N, dtype=torch.int32, device=refs.device)
    moved[source] = to.int()
    s["out"][0].copy_(torch.where(tables >= 0, moved[tables.clamp_min(0).long()], tables))
    s["out"][1].copy_(refs)
    s["out"][1][to] = refs[source]
    s["out"][1][source] = 0
    return [pool, *s["out"]]


_gpu = None


def run(s):
    op = s["case"]["op"]
    if not own:
        return {"attention": lambda: [_plain_attention(s)], "append": lambda: _plain_append(s),
                "fork": lambda: _plain_fork(s), "compact": lambda: _plain_compact(s)}[op]()
    global _gpu
    from laplacesscissors_b200 import Gpu, cache
    if _gpu is None:
        _gpu = Gpu(torch.cuda.current_device())
    if op == "attention":
        return [cache.attention(_gpu, s["q"], s["pages"], s["tables"], s["lengths"], s["starts"], scale=s["scale"],
                                out=s["out"])]
    if op == "append":
        cache.append(_gpu, s["k"], s["v"], s["pages"], s["tables"], s["lengths"], s["starts"])
        return list(cache.read(_gpu, s["pages"], s["tables"], s["lengths"], s["back_starts"], out=s["out"]))
    if op == "compact":
        cache.compact(_gpu, s["pool"], s["tables"], s["refs"], out=s["out"])
        return [s["pool"], *s["out"]]
    size = s["case"]["page"]
    cache.free(_gpu, s["tables"], s["lengths"], s["refs"], s["children"], size)
    cache.fork(_gpu, s["pool"], s["tables"], s["lengths"], s["refs"], s["parents"], s["children"], size, missing=s["missing"])
    cache.reserve(_gpu, s["tables"], s["lengths"], s["refs"], s["children"], s["counts"], size, missing=s["missing"])
    return [s["pool"], s["tables"], s["lengths"], s["refs"], s["missing"]]


def work(case):
    D, H = case["dim"], case["kv_heads"]
    if case["op"] in ("attention", "append"):
        lengths, queries = _shape(case)
        rows, wide = sum(queries), _BYTES[case["type"]]
        held = 18 * D // 16 * H  # bytes of a position
        if case["op"] == "attention":
            seen = sum(n for n, m in zip(lengths, queries) if m)
            pairs = sum(m * n - m * (m - 1) // 2 for n, m in zip(lengths, queries) if n)
            return {"bytes": float(seen * held + 2 * rows * case["q_heads"] * D * wide),
                    "flops": float(4 * D * case["q_heads"] * pairs)}
        back = sum(min(a, n + case["before"]) for a, n in zip(lengths, queries))
        return {"bytes": float(rows * H * D * 2 * wide + (rows + back) * held + back * H * D * 8),
                "flops": float(rows * H * D * 2 * 4 + back * H * D * 2 * 2)}
    width = {"u8": 1, "f16": 2, "f32": 4}[case["kind"]]
    page = case["layers"] * H * (case["page"] // 16) * 18 * D * width
    if case["op"] == "fork":
        copied = sum(_parent_length(case, i % case["parents"]) % case["page"] > 0 for i in range(case["children"]))
        small = case["children"] * (-(-case["length"] // case["page"])) * 16 + case["pages"] * 4
        return {"bytes": float(2 * copied * page + small), "flops": float(small // 4)}
    small = 16 * case["pages"] + 8 * (case["pages"] - case["free"])
    return {"bytes": float(2 * case["holes"] * page + small), "flops": float(small // 4)}


# ---- the definitions in 64 bits, one element at a time where that is quick ------------
def _exact_values(pages, table, length, device):
    """Keys and values [length, heads, D] in 64 bits, taken from the cells' words."""
    D, size = pages.shape[3] // 18, pages.shape[2] * 16
    cells = pages[table[:-(-length // size)].long()].transpose(1, 2).flatten(0, 1)[:-(-length // 16)]  # [C, H, 18 D]
    C, H = cells.shape[:2]

    def steps(part):
        a = cells[..., part:part + D].contiguous().view(torch.float16).double().view(C, H, D // 64, 4, 2, 2, 2)
        a = a.permute(0, 4, 3, 6, 1, 2, 5).reshape(C * 16, H, D // 64, 2)  # [t / 8, t % 8 / 2, t % 2], group, (s, z)
        return a[..., 0].repeat_interleave(64, 2), a[..., 1].repeat_interleave(64, 2)

    def nibbles(part):
        a = cells[..., part:part + 8 * D]
        return torch.stack([a & 15, a >> 4], -1)  # the low bits first
    k = nibbles(0).view(C, H, D // 64, 8, 4, 2, 16)            # group, t % 8, 16 elements' lane, t / 8, elements
    k = k.permute(0, 5, 3, 1, 2, 4, 6).reshape(C * 16, H, D).double()
    v = nibbles(8 * D).view(C, H, D // 64, 8, 4, 4, 2, 2, 2)   # group, d % 8, t % 8 / 2, word, t % 2, t / 8, d % 16 / 8
    v = v.permute(0, 7, 4, 6, 1, 2, 5, 8, 3).reshape(C * 16, H, D).double()
    (ks, kz), (vs, vz) = steps(16 * D), steps(17 * D)
    return (ks * k + kz)[:length], (vs * v + vz)[:length]


def _exact_attention(s):
    c, q = s["case"], s["q"]
    group, parts = c["q_heads"] // c["kv_heads"], []
    for b, (length, n) in enumerate(zip(*s["host"])):
        first = sum(s["host"][1][:b])
        if not length:
            parts.append(torch.zeros(n, *q.shape[1:], dtype=torch.float64, device=q.device))
            continue
        k, v = _exact_values(s["pages"], s["tables"][b], length, q.device)
        got = torch.empty(n, *q.shape[1:], dtype=torch.float64, device=q.device)
        for h in range(c["q_heads"]):
            for a in range(0, n, 256):
                z = q[first + a:first + min(n, a + 256), h].double() @ k[:, h // group].t() * s["scale"]
                last = torch.arange(length - n + a, length - n + a + z.shape[0], device=q.device)
                z = torch.where(torch.arange(length, device=q.device)[None] <= last[:, None], z, -math.inf)
                got[a:a + z.shape[0], h] = torch.softmax(z, 1) @ v[:, h // group]
        parts.append(got)
    return torch.cat(parts)


def _exact_append(s):
    lengths, queries = s["host"]
    keys, values, row = [], [], 0
    for b, (length, n, back) in enumerate(zip(lengths, queries, s["back"])):
        k, v = _exact_values(s["pages"], s["tables"][b], length, s["k"].device)
        for old, new in ((k, s["k"]), (v, s["v"])):
            x = new[row:row + n].double().unflatten(2, (-1, 64))
            z = x.min(3, keepdim=True).values.to(torch.float16).double()
            step = ((x.max(3, keepdim=True).values - z).float() / torch.full((1,), 15.0, device=x.device)).clamp_min(0)
            step = step.to(torch.float16).double()
            level = torch.where(step > 0, torch.round((x - z) / torch.where(step > 0, step, 1.0)), 0.0).clamp(0, 15)
            old[length - n:] = (z + step * level).flatten(2)
        keys.append(k[length - back:])
        values.append(v[length - back:])
        row += n
    return [torch.cat(keys), torch.cat(values)]


def _exact_fork(s):
    size = s["case"]["page"]
    tables, lengths, refs = (s[n].cpu().numpy().copy() for n in ("tables", "lengths", "refs"))
    pool = s["pool"].clone()

    def lowest():
        page = int(np.flatnonzero(refs == 0)[0])
        refs[page] = 1
        return page
    for child in s["children"].tolist():
        for i in range(-(-int(lengths[child]) // size)):
            refs[tables[child, i]] -= 1
        tables[child], lengths[child] = -1, 0
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        n = int(lengths[parent])
        for i in range(n // size):
            tables[child, i] = tables[parent, i]
            refs[tables[parent, i]] += 1
        lengths[child] = n
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        n = int(lengths[parent])
        if n % size:
            tables[child, n // size] = lowest()
            pool[:, int(tables[child, n // size])] = pool[:, int(tables[parent, n // size])]
    for child, more in zip(s["children"].tolist(), s["counts"].tolist()):
        for i in range(-(-int(lengths[child]) // size), -(-(int(lengths[child]) + more) // size)):
            tables[child, i] = lowest()
        lengths[child] += more
    return [pool, *(torch.from_numpy(a).cuda() for a in (tables, lengths, refs)), torch.zeros(1, dtype=torch.int32, device="cuda")]


def _exact_compact(s):
    tables, refs = s["tables"].cpu().numpy().copy(), s["refs"].cpu().numpy().copy()
    pool, live = s["pool"].clone(), int((refs > 0).sum())
    holes = [p for p in range(live) if refs[p] == 0]
    high = [p for p in range(live, len(refs)) if refs[p] > 0]
    for to, source in zip(holes, high):
        pool[:, to] = pool[:, source]
        tables[tables == source] = to
        refs[to], refs[source] = refs[source], 0
    return [pool, torch.from_numpy(tables).cuda(), torch.from_numpy(refs).cuda()]


def exact(case, seed):
    if case["op"] == "attention" and work(case)["flops"] > 4e12:
        return None  # minutes in 64 bits
    s = prepare(case, seed)
    return {"attention": lambda: [_exact_attention(s)], "append": lambda: _exact_append(s), "fork": lambda: _exact_fork(s),
            "compact": lambda: _exact_compact(s)}[case["op"]]()
