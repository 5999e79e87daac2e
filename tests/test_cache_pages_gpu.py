"""Reserving, forking, freeing, compacting and copying pages against the same steps one entry at a time
(tests/cache_reference.py); the whole as a search over sequences uses it."""
import numpy as np
import pytest
import torch

import cache_reference as ref
from laplacesscissors_b200 import cache

pytestmark = pytest.mark.gpu


def tensor(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


class State:
    """The same tables, lengths, counts and pool on the device and on the host."""

    def __init__(self, seed, pages=40, rows=7, width=6, size=16, layers=2, lengths=(), dtype=torch.uint8, item=(48,)):
        self.size, rng = size, np.random.default_rng(seed)
        self.tables = np.full((rows, width), -1, np.int32)
        self.lengths, self.refs = np.zeros(rows, np.int32), np.zeros(pages, np.int32)
        order = rng.permutation(pages)
        first = 0
        for s, n in enumerate(lengths):
            need = -(-n // size)
            self.tables[s, :need] = order[first:first + need]
            first += need
            self.lengths[s] = n
        np.add.at(self.refs, self.tables[self.tables >= 0], 1)
        self.pool = rng.integers(0, 256, (layers, pages, *item)).astype(np.uint8)
        self.dev = [tensor(a) for a in (self.tables, self.lengths, self.refs)]
        self.dev_pool = tensor(self.pool, torch.uint8).to(dtype)

    def same(self):
        for a, b, name in zip(self.dev, (self.tables, self.lengths, self.refs), ("tables", "lengths", "refs")):
            assert np.array_equal(a.cpu().numpy(), b), name
        assert np.array_equal(self.dev_pool.float().cpu().numpy(), self.pool.astype(np.float32))

    def reserve(self, gpu, sequences, counts):
        got = cache.reserve(gpu, *self.dev, tensor(sequences), tensor(counts), self.size)
        expected = ref.reserve(self.tables, self.lengths, self.refs, sequences, counts, self.size)
        assert int(got) == expected
        self.same()
        return expected

    def fork(self, gpu, parents, children):
        got = cache.fork(gpu, self.dev_pool, *self.dev, tensor(parents), tensor(children), self.size)
        expected = ref.fork(self.pool, self.tables, self.lengths, self.refs, parents, children, self.size)
        assert int(got) == expected
        self.same()
        return expected

    def free(self, gpu, sequences):
        cache.free(gpu, *self.dev, tensor(sequences), self.size)
        ref.free(self.tables, self.lengths, self.refs, sequences, self.size)
        self.same()

    def compact(self, gpu, in_place=True):
        tables, _, refs = self.dev
        before = tables.clone(), refs.clone()
        out = (tables, refs) if in_place else None
        got = cache.compact(gpu, self.dev_pool, tables, refs, out=out)
        if not in_place:
            assert torch.equal(tables, before[0]) and torch.equal(refs, before[1])
            self.dev[0], self.dev[2] = got
        ref.compact(self.pool, self.tables, self.refs)
        self.same()


def test_reserve(gpu):
    s = State(1, lengths=[0, 5, 16, 40])
    assert s.reserve(gpu, [0, 1, 2, 3], [0, 11, 1, 60]) != 0  # the last row of the tables is too short
    assert s.reserve(gpu, [0, 1, 2, 3], [0, 11, 1, 30]) == 0
    assert s.reserve(gpu, [0, 1, 2], [1, 1, 0]) == 0
    assert s.reserve(gpu, [6, 5], [96, 17]) == 0
    assert s.reserve(gpu, [], []) == 0


def test_reserve_passes_over_and_gives_back(gpu):
    s = State(2, pages=12, lengths=[30, 30, 16])
    assert s.reserve(gpu, [-1, 7, 3, 3, 10 ** 9], [5, 5, 20, 99, 1]) == 0
    assert s.reserve(gpu, [4, 5, 0], [60, 60, 20]) == 5  # 5 pages are free, 10 wanted
    assert s.reserve(gpu, [4, 5], [-3, 60]) == 0
    assert s.reserve(gpu, [0], [2 ** 31 - 1]) != 0
    assert s.reserve(gpu, [0, 1], [2, 2]) == 0


@pytest.mark.parametrize("pages", [1, 1023, 4096, 4097, 30001])
def test_reserve_in_large_pools(gpu, pages):
    rng = np.random.default_rng(pages)
    s = State(3, pages=pages, rows=1024, width=64, layers=1, item=(16,))
    used = rng.random(pages) < 0.9
    s.refs[used] = rng.integers(1, 4, used.sum())
    s.dev[2] = tensor(s.refs)
    left = int((~used).sum())
    counts = np.zeros(1024, int)
    for i in rng.integers(0, 1024, min(left, 1000)):
        counts[i] += 16
    counts = np.minimum(counts, 64 * 16)
    order = rng.permutation(1024)
    assert s.reserve(gpu, order.tolist(), counts.tolist()) == 0
    s.reserve(gpu, order.tolist(), (counts + 40).tolist())


def test_fork(gpu):
    s = State(4, lengths=[33, 32, 5])
    assert s.fork(gpu, [0, 1, 2, 0], [3, 4, 5, 6]) == 0
    assert s.lengths.tolist() == [33, 32, 5, 33, 32, 5, 33]
    s.free(gpu, [0, 3])
    assert s.fork(gpu, [6, 4], [3, 0]) == 0


def test_fork_passes_over(gpu):
    s = State(5, lengths=[33, 32, 0, 7])
    # taken children, the same child twice, rows outside, an empty parent, a child that is a parent
    assert s.fork(gpu, [0, 0, 1, 9, 0, -1, 2, 5, 3], [1, 4, 4, 5, 70, 6, 6, 2, 3]) == 0
    assert s.lengths.tolist() == [33, 32, 0, 7, 33, 0, 0]


def test_fork_without_room_changes_nothing(gpu):
    s = State(6, pages=6, lengths=[33, 16, 17])
    assert s.fork(gpu, [0, 1, 2], [3, 4, 5]) == 2
    assert s.fork(gpu, [1, 1, 1, 1], [3, 4, 5, 6]) == 0  # whole pages need none


def test_fork_many(gpu):
    rng = np.random.default_rng(7)
    s = State(7, pages=3000, rows=1100, width=9, lengths=[100, 129, 144, 1], layers=3, item=(5, 32))
    children = rng.permutation(np.arange(4, 1028)).tolist()
    assert s.fork(gpu, rng.integers(0, 4, 1024).tolist(), children) == 0
    s.free(gpu, children[::2] + children[:3])
    s.compact(gpu)


def test_free(gpu):
    s = State(8, lengths=[33, 32, 5, 96])
    s.fork(gpu, [0], [5])
    s.free(gpu, [0, 0, 9, -1, 3, 6, 0])
    s.free(gpu, [5, 1, 2])
    assert not s.refs.any() and (s.tables == -1).all()


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("pages", [3, 40, 1024, 5000])
@pytest.mark.parametrize("dtype,item", [(torch.uint8, (48,)), (torch.float32, (3, 4)), (torch.bfloat16, (7, 2, 8))])
def test_compact(gpu, in_place, pages, dtype, item):
    rng = np.random.default_rng(pages)
    s = State(9, pages=pages, rows=40, width=-(-pages // 20), layers=3, dtype=dtype, item=item)
    live = rng.permutation(pages)[:max(1, pages * 6 // 10)]
    flat = s.tables.reshape(-1)
    flat[rng.permutation(flat.size)[:len(live)]] = live
    flat[flat == live[0]] = live[0]
    for _ in range(3):  # a page that several rows share
        flat[rng.integers(0, flat.size)] = live[-1]
    s.refs[:] = 0
    np.add.at(s.refs, s.tables[s.tables >= 0], 1)
    s.tables[0, 0] = pages + 5 if s.tables[0, 0] < 0 else s.tables[0, 0]  # no page
    s.dev = [tensor(a) for a in (s.tables, s.lengths, s.refs)]
    s.compact(gpu, in_place)
    s.compact(gpu, in_place)  # nothing is left to move


def test_compact_full_and_empty(gpu):
    s = State(10, pages=12, lengths=[64, 64, 64])
    s.compact(gpu)
    s = State(11, pages=12)
    s.compact(gpu)


@pytest.mark.parametrize("item", [(16,), (48,), (2, 9, 1152), (40000 // 16 * 16,)])
def test_copy_pages(gpu, item):
    s = State(12, pages=30, layers=5, item=item)
    pairs = [[0, 7], [3, 29], [0, 8], [-1, 4], [5, 30], [2 ** 31 - 1, 9], [6, -2]]
    cache.copy_pages(gpu, s.dev_pool, tensor(pairs))
    for a, b in pairs[:3]:
        s.pool[:, b] = s.pool[:, a]
    s.same()


def test_layers_apart(gpu):
    """A pool that is a slice of a larger one."""
    s = State(13, pages=20, layers=4, lengths=[30, 40])
    s.dev_pool, s.pool = s.dev_pool[::2], s.pool[::2].copy()
    assert s.fork(gpu, [0, 1], [2, 3]) == 0


def test_a_search_over_sequences(gpu):
    """Prompts, forks, steps, ends and compaction as a server would run them, on a PagedCache: what every sequence
    reads back is what was appended along its branch, and attention over it agrees with the reference."""
    rng = np.random.default_rng(14)
    held = cache.PagedCache(gpu, layers=2, pages=60, kv_heads=2, head_dim=64, sequences=8, longest=160, page_size=16)
    told = {}  # sequence -> list of (k, v) [layers, 2, 64]

    def add(names, counts):
        starts = tensor(np.concatenate([[0], np.cumsum(counts)]))
        assert int(held.reserve(tensor(names), tensor(counts))) == 0
        kv = rng.standard_normal((2, 2, sum(counts), 2, 64)).astype(np.float32)
        for layer in range(2):
            held.append(layer, *(tensor(a, torch.float32) for a in kv[:, layer]), starts, tensor(names))
        row = 0
        for s, n in zip(names, counts):
            told[s] = told.get(s, []) + [kv[:, :, row + i] for i in range(n)]
            row += n

    def look():
        r = None
        for layer in range(2):
            r = ref.Reference(held.pool[layer].cpu().numpy(), held.tables.cpu().numpy(), held.lengths.cpu().numpy())
            for s, rows in told.items():
                assert int(held.lengths[s]) == len(rows)
                starts = tensor([0, len(rows)])
                got = held.read(layer, starts, tensor([s]), rows=len(rows))
                kv = np.array(rows).reshape(-1, 2, 2, 2, 64)[:, :, layer]
                for a, b in zip(got, (kv[:, 0], kv[:, 1])):
                    expected = ref.dequantise(*ref.quantise(b)) if len(rows) else b
                    assert np.allclose(a.cpu().numpy(), expected, rtol=2.0 ** -23, atol=1e-7)
            names = sorted(told)
            q = rng.standard_normal((len(names), 4, 64)).astype(np.float32)
            out = held.attention(layer, tensor(q, torch.float32), sequences=tensor(names)).cpu().numpy()
            expected = r.attention(q, 0.125, None, names)[0]
            assert np.allclose(out, expected, rtol=1e-4, atol=1e-4)
        used = held.refs.cpu().numpy()
        tables = held.tables.cpu().numpy()
        assert np.array_equal(used, np.bincount(tables[tables >= 0], minlength=60))

    add([0, 3], [37, 16])
    look()
    assert int(held.fork(tensor([0, 0, 3]), tensor([1, 2, 4]))) == 0
    told.update({1: list(told[0]), 2: list(told[0]), 4: list(told[3])})
    look()
    for _ in range(13):
        add([0, 1, 2, 3, 4], [1] * 5)
    look()
    held.free(tensor([0, 3]))
    del told[0], told[3]
    held.compact()
    look()
    assert int(held.fork(tensor([2, 1]), tensor([0, 7]))) == 0
    told.update({0: list(told[2]), 7: list(told[1])})
    add([7, 2, 0], [5, 1, 20])
    held.compact()
    look()


class Counted:
    """Tables, lengths and refs whose counts are those of the tables, whatever was done."""

    def __init__(self, pages, rows, width, size=16):
        self.size = size
        self.tables = tensor(np.full((rows, width), -1))
        self.lengths, self.refs = tensor([0] * rows), tensor([0] * pages)
        self.state = (self.tables, self.lengths, self.refs)

    def look(self):
        t, refs = self.tables.cpu().numpy(), self.refs.cpu().numpy()
        assert np.array_equal(refs, np.bincount(t[t >= 0], minlength=len(refs)))
        for row, n in zip(t, self.lengths.tolist()):
            held = int((row >= 0).sum())
            assert (row[:held] >= 0).all() and held >= -(-n // self.size)  # no gaps, and pages for all positions
        return t

    def reserve(self, gpu, sequences, counts):
        missing = int(cache.reserve(gpu, *self.state, tensor(sequences), tensor(counts), self.size))
        self.look()
        return missing


def test_positions_taken_back_keep_their_pages(gpu):
    """Drafts that were rejected: a length that was lowered across pages loses none of them."""
    s = Counted(pages=30, rows=4, width=40)
    assert s.reserve(gpu, [0, 1, 2], [100, 33, 16]) == 0
    before = s.look()
    for lower, more, used in ((70, 20, 7), (32, 1, 7), (0, 112, 7), (97, 30, 8), (1, 300, 19)):
        s.lengths[0] = lower
        assert s.reserve(gpu, [3, 0, 1], [0, more, 0]) == 0
        now = s.look()
        assert int(s.lengths[0]) == lower + more and (now[0] >= 0).sum() == used and np.array_equal(now[0, :7], before[0, :7])
        assert np.array_equal(now[1:], before[1:])
    assert int((s.refs > 0).sum()) == 23
    s.lengths[0], s.lengths[1] = 5, 0
    assert s.reserve(gpu, [0, 1, 3], [16 * 18, 48, 16 * 8]) == 1  # a row's own pages, then the seven that are free
    assert s.lengths.tolist() == [5, 0, 16, 0]
    assert s.reserve(gpu, [0, 1, 3], [16 * 18, 48, 16 * 6]) == 0
    s.lengths[0], s.lengths[1] = 3, 0
    cache.free(gpu, *s.state, tensor([0, 1]), s.size)
    t = s.look()
    assert (t[:2] == -1).all() and int((s.refs > 0).sum()) == 7


@pytest.mark.parametrize("pages,width", [(700, 600), (700, 256), (700, 257), (2000, 1900)])
def test_long_rows_taken_back(gpu, pages, width):
    s = Counted(pages, rows=3, width=width)
    assert s.reserve(gpu, [0, 1], [16 * width, 40]) == 0
    for lower in (16 * (width - 1), 16 * 255 + 1, 16 * 256, 17, 0):
        s.lengths[0] = lower
        assert s.reserve(gpu, [0], [16 * width - lower]) == 0
        assert int((s.refs > 0).sum()) == width + 3
    s.lengths[0] = 16 * (width // 2)
    cache.free(gpu, *s.state, tensor([0]), s.size)
    assert s.look()[0].max() == -1 and int((s.refs > 0).sum()) == 3


def test_a_child_that_kept_its_pages_is_not_empty(gpu):
    s = Counted(pages=20, rows=4, width=6)
    assert s.reserve(gpu, [0, 1], [40, 20]) == 0
    pool = torch.zeros((2, 20, 16), dtype=torch.uint8, device="cuda")
    s.lengths[1] = 0
    assert int(cache.fork(gpu, pool, *s.state, tensor([0, 0]), tensor([1, 2]), s.size)) == 0
    s.look()
    assert s.lengths.tolist() == [40, 0, 40, 0]
    cache.free(gpu, *s.state, tensor([1]), s.size)
    assert int(cache.fork(gpu, pool, *s.state, tensor([0]), tensor([1]), s.size)) == 0
    s.look()
    assert s.lengths.tolist() == [40, 40, 40, 0]
