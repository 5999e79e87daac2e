"""The paged cache of include/lsx.h restated in numpy, in 64 bits and one sequence at a time: what its storage
holds, what attention over it gives, and what its bookkeeping leaves."""
import numpy as np


def quantise(x):
    """(n, s, z) of groups of 64 along the last axis: x [..., D] f32."""
    x = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        z = (x.min(-1) + np.float32(0)).astype(np.float16)
        s = np.maximum((x.max(-1) - z.astype(np.float32)) / np.float32(15), np.float32(0)).astype(np.float16)
        bad = ~(np.isfinite(s) & np.isfinite(z) & np.isfinite(x).all(-1))
        s, z = np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(np.nan), z)
        n = np.rint((x.astype(np.float64) - z.astype(np.float64)[..., None]) / s.astype(np.float64)[..., None])
        n = np.where((bad | (s == 0))[..., None], 0, np.clip(n, 0, 15))
    return n.astype(np.uint8).reshape(*x.shape[:-2], -1), s, z


def dequantise(n, s, z):
    groups = n.reshape(*s.shape, 64).astype(np.float64)
    with np.errstate(all="ignore"):
        return (groups * s.astype(np.float64)[..., None] + z.astype(np.float64)[..., None]).reshape(n.shape)


def cell_index(D):
    """[16, 18 D / 16] bytes of a cell by position: key n, value n, key s, key z, value s, value z."""
    out = []
    for t in range(16):
        row = [(32 * (d // 64) + 4 * (t % 8) + d % 64 // 16) * 16 + t // 8 * 8 + d % 16 // 2 for d in range(0, D, 2)]
        row += [8 * D + (32 * (d // 64) + 4 * (d % 8) + t % 8 // 2) * 16 + d // 16 % 4 * 4 + t % 2 * 2 + t // 8
                for d in range(D) if d % 16 < 8]
        for base in (16 * D, 16 * D + 4, 17 * D, 17 * D + 4):
            for g in range(D // 64):
                at = base + 64 * g + t % 8 // 2 * 16 + t // 8 * 8 + t % 2 * 2
                row += [at, at + 1]
        out.append(row)
    index = np.array(out)
    assert len(set(index.reshape(-1))) == 18 * D == index.size
    return index


def encode(k, v):
    """Bytes [..., 18 D / 16] of keys and values [..., D], in cell_index's order."""
    (kn, ks, kz), (vn, vs, vz) = quantise(k), quantise(v)
    D = kn.shape[-1]
    kb = kn[..., 0::2] | kn[..., 1::2] << 4
    low = [d for d in range(D) if d % 16 < 8]
    vb = vn[..., low] | vn[..., [d + 8 for d in low]] << 4
    return np.concatenate([kb, vb] + [np.ascontiguousarray(a).view(np.uint8) for a in (ks, kz, vs, vz)], -1)


def decode(raw):
    """(keys, values, key scale 15 s + |z|, value scale) [..., D] in 64 bits of encode's bytes."""
    D = raw.shape[-1] * 16 // 18
    n = np.zeros((2, *raw.shape[:-1], D), np.uint8)
    n[0][..., 0::2], n[0][..., 1::2] = raw[..., :D // 2] & 15, raw[..., :D // 2] >> 4
    low = [d for d in range(D) if d % 16 < 8]
    n[1][..., low], n[1][..., [d + 8 for d in low]] = raw[..., D // 2:D] & 15, raw[..., D // 2:D] >> 4
    ks, kz, vs, vz = (np.ascontiguousarray(raw[..., D + i * D // 32:D + (i + 1) * D // 32]).view(np.float16) for i in range(4))
    wide = lambda s, z: np.repeat(15 * s.astype(np.float64) + abs(z.astype(np.float64)), 64, -1)  # noqa: E731
    return dequantise(n[0], ks, kz), dequantise(n[1], vs, vz), wide(ks, kz), wide(vs, vz)


class Reference:
    """Pages as numpy bytes [pages, heads, page / 16, 18 D], with tables and lengths."""

    def __init__(self, pages, tables, lengths):
        self.pages, self.tables, self.lengths = pages, tables, lengths
        self.size, self.D = pages.shape[2] * 16, pages.shape[3] // 18
        self.index = cell_index(self.D)

    def rows(self, rows, starts, sequences):
        """(row, table row or None, position, sequence) of each row that belongs to a sequence."""
        names = list(range(len(self.tables))) if sequences is None else list(sequences)
        count = len(names) if sequences is not None else (rows if starts is None else len(starts) - 1)
        for b in range(count):
            first, end = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
            table = names[b] if 0 <= names[b] < len(self.tables) else None
            length = 0 if table is None else int(self.lengths[table])
            for row in range(first, end):
                yield row, table, length - (end - row), b

    def cell(self, table, position):
        """[heads, 18 D] of a position, or None without a page."""
        slot = position // self.size
        page = int(self.tables[table][slot]) if slot < len(self.tables[table]) else -1
        return None if not 0 <= page < len(self.pages) else self.pages[page][:, position % self.size // 16]

    def append(self, k, v, starts=None, sequences=None):
        raw = encode(k, v)
        for row, table, position, _ in self.rows(len(k), starts, sequences):
            cell = self.cell(table, position) if table is not None and position >= 0 else None
            if cell is not None:
                cell[:, self.index[position % 16]] = raw[row]

    def values(self, table, length):
        """decode's four [length, heads, D]; NaN where there is no page."""
        raw, gone = [], []
        for position in range(length):
            cell = self.cell(table, position)
            gone.append(cell is None)
            raw.append(np.zeros((self.pages.shape[1], 18 * self.D // 16), np.uint8) if cell is None
                       else cell[:, self.index[position % 16]])
        parts = decode(np.array(raw).reshape(length, self.pages.shape[1], -1))
        for part in parts:
            part[gone] = np.nan
        return parts

    def read(self, rows, starts=None, sequences=None):
        out = np.zeros((2, rows, self.pages.shape[1], self.D))
        for row, table, position, _ in self.rows(rows, starts, sequences):
            if table is None:
                out[:, row] = np.nan
            elif position >= 0:
                cell = self.cell(table, position)
                if cell is None:
                    out[:, row] = np.nan
                else:
                    out[0, row], out[1, row] = decode(cell[:, self.index[position % 16]])[:2]
        return out

    def attention(self, q, scale, starts=None, sequences=None):
        """(out, the largest scaled sum of |q| (15 s + |z|) over the keys, the sum of p (15 s + |z|) of the values), each
        [rows, q_heads, D], and which rows belong to a sequence."""
        rows, heads, D = q.shape
        group = heads // self.pages.shape[1]
        out, score_bound, wide = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
        held, used = {}, np.zeros(rows, bool)
        for row, table, position, b in self.rows(rows, starts, sequences):
            used[row] = True
            if table is None:
                out[row] = np.nan
                continue
            if position < 0:
                continue
            if table not in held:
                held[table] = self.values(table, int(self.lengths[table]))
            k, v, k_wide, v_wide = (a[:position + 1] for a in held[table])
            for h in range(heads):
                x, g = q[row, h].astype(np.float64), h // group
                z = k[:, g] @ x * scale
                with np.errstate(all="ignore"):
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[row, h] = p @ v[:, g]
                    wide[row, h] = p @ v_wide[:, g]
                    score_bound[row, h] = abs(scale) * (k_wide[:, g] @ abs(x)).max()
        return out, score_bound, wide, used


# ---- bookkeeping, one entry after the other -----------------------------------------
def reserve(tables, lengths, refs, sequences, counts, size):
    """Changes the state in place and returns how many pages were short."""
    state = [a.copy() for a in (tables, lengths, refs)]
    missing, seen = 0, set()
    for s, n in zip(sequences, counts):
        if not 0 <= s < len(tables) or s in seen:
            continue
        seen.add(s)
        before, after = int(state[1][s]), int(state[1][s]) + max(int(n), 0)
        missing += max(0, -(-after // size) - tables.shape[1])
    if missing:
        return missing
    for s, n in [(s, n) for i, (s, n) in enumerate(zip(sequences, counts)) if s in seen and s not in list(sequences[:i])]:
        before, after = int(state[1][s]), int(state[1][s]) + max(int(n), 0)
        for slot in range(-(-before // size), -(-after // size)):
            free = np.flatnonzero(state[2] <= 0)
            if not len(free):
                missing += 1
                continue
            state[0][s, slot] = free[0]
            state[2][free[0]] = 1
        state[1][s] = after
    if not missing:
        tables[:], lengths[:], refs[:] = state
    return missing


def fork(pool, tables, lengths, refs, parents, children, size):
    entries, seen, empty = [], set(), lengths <= 0
    for p, c in zip(parents, children):
        if 0 <= c < len(tables) and 0 <= p < len(tables) and c not in seen and empty[c] and lengths[p] > 0:
            entries.append((p, c))
        seen.add(c)
    part = [e for e in entries if lengths[e[0]] % size]
    free = np.flatnonzero(refs <= 0)
    if len(part) > len(free):
        return len(part) - len(free)
    for page, (p, c) in zip(free, part):
        slot = lengths[p] // size
        tables[c, slot] = page
        refs[page] = 1
        if 0 <= tables[p, slot] < len(refs):
            pool[:, page] = pool[:, tables[p, slot]]
    for p, c in entries:
        for slot in range(lengths[p] // size):
            tables[c, slot] = tables[p, slot]
            if 0 <= tables[p, slot] < len(refs):
                refs[tables[p, slot]] += 1
        lengths[c] = lengths[p]
    return 0


def free(tables, lengths, refs, sequences, size):
    for s in sequences:
        if 0 <= s < len(tables):
            for slot in range(min(-(-int(lengths[s]) // size), tables.shape[1])):
                if 0 <= tables[s, slot] < len(refs):
                    refs[tables[s, slot]] -= 1
                tables[s, slot] = -1
            lengths[s] = 0


def compact(pool, tables, refs):
    live = int((refs > 0).sum())
    holes, high = [p for p in range(live) if refs[p] <= 0], [p for p in range(live, len(refs)) if refs[p] > 0]
    for to, source in zip(holes, high):
        pool[:, to] = pool[:, source]
        tables[tables == source] = to
        refs[to], refs[source] = refs[source], 0
    refs[live:] = 0
