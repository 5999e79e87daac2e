"""The paged cache as programs run it: captured and replayed, on other streams, from two threads, twice at
once, with pages far into a large pool, and twice with the same answer."""
import threading

import numpy as np
import pytest
import torch

import cache_reference as ref
from laplacesscissors_b200 import LsxError, cache
from test_cache_gpu import check, make, queries, tensor

pytestmark = pytest.mark.gpu


def filled(gpu, seed, lengths, heads=2, D=64, layers=1, page_size=16, longest=1024):
    """A PagedCache whose sequences hold random keys and values."""
    held = cache.PagedCache(gpu, layers=layers, pages=sum(-(-n // page_size) for n in lengths) + 20, kv_heads=heads, head_dim=D,
                            sequences=len(lengths), longest=longest, page_size=page_size)
    assert int(held.reserve(tensor(range(len(lengths))), tensor(lengths))) == 0
    starts = tensor(np.concatenate([[0], np.cumsum(lengths)]))
    for layer in range(layers):
        held.append(layer, *(queries(seed + i, sum(lengths), heads, D, torch.bfloat16) for i in (2 * layer, 2 * layer + 1)), starts)
    return held


def reference(held, layer=0):
    return ref.Reference(held.pool[layer].cpu().numpy(), held.tables.cpu().numpy(), held.lengths.cpu().numpy())


class Step:
    """A decode step of all sequences, captured: reserve, append, attention."""

    def __init__(self, gpu, seed, lengths, D=64):
        self.held = filled(gpu, seed, lengths, D=D)
        n = len(lengths)
        self.names, self.ones = tensor(range(n)), tensor([1] * n)
        self.k, self.v, self.q = (queries(seed + i, n, h, D, torch.float32) for i, h in ((10, 2), (11, 2), (12, 6)))
        self.missing = tensor([0])
        self.out = torch.zeros_like(self.q)
        self.run()  # once before the capture
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.run()

    def run(self):
        self.held.reserve(self.names, self.ones, missing=self.missing)
        self.held.append(0, self.k, self.v)
        self.held.attention(0, self.q, out=self.out)

    def check(self, length_of_first):
        assert int(self.missing) == 0 and int(self.held.lengths[0]) == length_of_first
        r = reference(self.held)
        expected = r.attention(self.q.double().cpu().numpy(), self.q.shape[2] ** -0.5)[0]
        assert np.allclose(self.out.cpu().numpy(), expected, rtol=1e-4, atol=1e-4)


def test_a_captured_step_follows_the_lengths(gpu):
    s = Step(gpu, 1, [5, 31, 200, 630])
    length = 6
    for count in (1, 3, 12):
        for i in range(count):
            s.k.normal_()
            s.v.normal_()
            s.q.normal_()
            s.graph.replay()
        length += count
        torch.cuda.synchronize()
        s.check(length)


def test_two_captured_steps_at_once(gpu):
    steps = [Step(gpu, 2, [700, 31, 650]), Step(gpu, 3, [5, 800, 90, 13], D=128)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(8):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.graph.replay()
    torch.cuda.synchronize()
    for s, first in zip(steps, (709, 14)):
        s.check(first)


def test_two_streams_and_two_threads(gpu):
    caches = [filled(gpu, 20 + i, [900, 3, 400 + i]) for i in range(2)]
    expected = [reference(c).attention(queries(30 + i, 3, 4, 64, torch.float32).double().cpu().numpy(), 0.125)[0]
                for i, c in enumerate(caches)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        q = queries(30 + i, 3, 4, 64, torch.float32)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = caches[i].attention(0, q)
                stream.synchronize()
                if not np.allclose(got.cpu().numpy(), expected[i], rtol=1e-4, atol=1e-4):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_same_call_repeats_its_bits(gpu, dtype):
    held, _ = make(40, [3000, 17, 900, 2500], heads=2, D=128, size=64)
    q = queries(41, 4, 8, 128, dtype)
    first = cache.attention(gpu, q, *held)
    for _ in range(10):
        assert torch.equal(cache.attention(gpu, q, *held), first)


def test_calls_follow_the_current_stream(gpu):
    held, r = make(42, [200, 64], D=64)
    q = queries(43, 2, 4, 64, torch.float32)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        moved = q * 2
        got = cache.attention(gpu, moved, *held)
        back = got + 0
    stream.synchronize()
    expected = r.attention((q * 2).double().cpu().numpy(), 0.125)[0]
    assert np.allclose(back.cpu().numpy(), expected, rtol=1e-4, atol=1e-4)


def test_tensors_that_a_call_writes_count_as_modified(gpu):
    held = filled(gpu, 44, [20, 30])
    x = queries(45, 2, 2, 64, torch.float32)
    before = held.pool._version
    held.append(0, x, x)
    assert held.pool._version > before
    out = torch.zeros(2, 2, 64, device="cuda")
    before = out._version
    held.attention(0, x, out=out)
    assert out._version > before


def test_pages_far_into_a_large_pool(gpu):
    """Bytes past 2^32 from the pool's start, in its second layer too."""
    heads, D, size, count = 8, 128, 64, 60000  # 4.4 GB a layer
    pool = torch.empty((2, *cache.pages_shape(count, heads, size, D)), dtype=torch.uint8, device="cuda")
    tables = tensor([[count - 1, 3, count - 2, -1], [count - 7, count - 30, -1, -1], [-1] * 4])
    lengths = tensor([150, 100, 0])
    refs = torch.zeros(count, dtype=torch.int32, device="cuda")
    refs[tables[tables >= 0].long()] = 1
    refs[:40000] = 1
    starts = tensor([0, 150, 250])
    k, v = (queries(50 + i, 250, heads, D, torch.bfloat16) for i in range(2))
    for layer in range(2):
        cache.append(gpu, k + layer, v, pool[layer], tables, lengths, starts)
    missing = cache.fork(gpu, pool, tables, lengths, refs, tensor([0]), tensor([2]), size)
    assert int(missing) == 0 and tables[2].tolist() == [count - 1, 3, 40000, -1]
    for layer in range(2):
        for rows, at in ((150, 0), (100, 1), (150, 2)):
            got = cache.read(gpu, pool[layer], tables, lengths, tensor([0, rows]), sequences=tensor([at]), rows=rows)
            first = 150 if at == 1 else 0
            expected = ref.dequantise(*ref.quantise((k + layer)[first:first + rows].float().cpu().numpy()))
            assert np.allclose(got[0].cpu().numpy(), expected, rtol=2.0 ** -23, atol=0)
        small = [1, 3, count - 1, count - 2, count - 7, count - 30, 40000]
        pages = pool[layer][small].cpu().numpy()
        index = {p: i for i, p in enumerate(small)}
        local = np.array([[index.get(p, -1) for p in row] for row in tables.tolist()], np.int32)
        r = ref.Reference(pages, local, lengths.cpu().numpy())
        check(gpu, (pool[layer], tables, lengths), r, queries(60, 3, 16, D, torch.bfloat16))
    kept = [pool[layer, 40000].clone() for layer in range(2)]
    refs[:39000] = 0
    refs[3] = 1
    got = cache.compact(gpu, pool, tables, refs)
    live = int((refs > 0).sum())
    assert int(got.tables.max()) < live and int((got.refs > 0).sum()) == live and not got.refs[live:].any()
    for layer in range(2):
        assert torch.equal(pool[layer, int(got.tables[2, 2])], kept[layer])


@pytest.mark.parametrize("rows,sequences", [(1, 1), (1, 300), (2000, 300), (129, 128)])
def test_many_sequences(gpu, rows, sequences):
    """More sequences than threads look them up, most without rows."""
    rng = np.random.default_rng(rows)
    lengths = rng.integers(0, 40, sequences).tolist()
    held, r = make(70, lengths, heads=1, D=64, size=16)
    cuts = np.sort(rng.integers(0, rows + 1, sequences - 1))
    starts = np.concatenate([[0], cuts, [rows]])
    check(gpu, held, r, queries(71, rows, 2, 64, torch.float32), starts)
    k, v = (queries(72 + i, rows, 1, 64, torch.float16) for i in range(2))
    cache.append(gpu, k, v, *held, tensor(starts))
    r.append(k.float().cpu().numpy(), v.float().cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)


def test_sequences_that_share_pages(gpu):
    held = cache.PagedCache(gpu, layers=1, pages=30, kv_heads=2, head_dim=64, sequences=6, longest=200, page_size=16)
    assert int(held.reserve(tensor([0]), tensor([90]))) == 0
    kv = [queries(81 + i, 90, 2, 64, torch.float32) for i in range(2)]
    held.append(0, *kv, tensor([0, 90]), tensor([0]))
    assert int(held.fork(tensor([0] * 5), tensor([1, 2, 3, 4, 5]))) == 0
    r = reference(held)
    check(gpu, (held.pool[0], held.tables, held.lengths), r, queries(83, 6, 4, 64, torch.float32))
    starts = [0, 20, 25, 45, 46, 46, 60]
    check(gpu, (held.pool[0], held.tables, held.lengths), r, queries(84, 60, 4, 64, torch.bfloat16), starts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_long_runs_do_not_drift(gpu, dtype):
    """More positions than fit a sum on the tensor cores, for every warp: 32 sequences of some 40 thousand, whose
    tables name the same pages again and again."""
    heads, D, size, n = 8, 64, 64, 32
    held, r = make(90, [64 * 200], heads=heads, D=D, size=size, spare=0)
    rng = np.random.default_rng(91)
    lengths = rng.integers(39000, 41000, n)
    tables = rng.integers(0, 200, (n, 641)).astype(np.int32)
    q = queries(92, n, 2 * heads, D, dtype, 0.3)  # weights of one size, so that all positions count
    got = cache.attention(gpu, q, held[0], tensor(tables), tensor(lengths)).double()
    order = held[1][0].cpu().numpy()
    k, v, k_wide, v_wide = (torch.from_numpy(a).cuda() for a in r.values(0, 64 * 200))
    place = np.empty(200, np.int64)
    place[order[:200]] = np.arange(200)
    for b in range(0, n, 3):
        at = np.arange(lengths[b])
        at = torch.from_numpy(place[tables[b][at // size]] * size + at % size).cuda()
        z = torch.einsum("hgd,thd->hgt", q[b].double().view(heads, 2, D), k[at]) / 8
        p = torch.softmax(z, 2)
        expected = torch.einsum("hgt,thd->hgd", p, v[at]).reshape(2 * heads, D)
        wide = torch.einsum("hgt,thd->hgd", p, v_wide[at]).reshape(2 * heads, D)
        bound = torch.einsum("hgd,thd->hgt", q[b].double().abs().view(heads, 2, D), k_wide[at]).amax(2).reshape(-1, 1) / 8
        # scores as in test_cache_gpu.tolerance; the sums are put aside after 64 (f16, bf16: 256) steps, which cut up to
        # 2^-23 of the sum each, and meet in f32
        weight = 2 * torch.expm1((D / 8 + 16) * 2.0 ** -22 * bound) + 2.0 ** -20
        steps = (2 * 64 if dtype is torch.float32 else 256) * 2.0 ** -23
        single = 0 if dtype is torch.float32 else 2.0 ** -11
        allowed = (weight + steps + 64 * 2.0 ** -24 + single) * wide + torch.finfo(dtype).eps / 2 * expected.abs()
        error = (got[b] - expected).abs()
        assert (error <= allowed).all(), float((error - allowed).max())
        if dtype is torch.float32:
            assert float(error.norm() / expected.norm()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths_at_the_end_of_their_type(gpu, dtype):
    """A sequence of 2^31 - 16 positions whose table names one page again and again: the attention over it is
    that over the page, and rows behind it, of a length that no table covers, are NaN."""
    held, r = make(95, [16], heads=1, D=64, size=16, spare=0)
    width = (2 ** 31 - 1) // 16
    tables = torch.zeros((2, width), dtype=torch.int32, device="cuda")
    lengths = tensor([16 * width, 2 ** 31 - 1])
    q = queries(96, 21, 1, 64, dtype)
    got = cache.attention(gpu, q, held[0], tables, lengths, tensor([0, 1, 21]))
    # row i of the second's twenty sees 2^31 - 20 + i positions, of which the table covers 16 * width
    seen = np.array([16 * width] + [2 ** 31 - 20 + i for i in range(20)])
    fine = seen <= 16 * width
    assert fine.sum() == 6 and torch.equal(torch.isnan(got).all(2).all(1).cpu(), torch.from_numpy(~fine))
    k, v, _, _ = r.values(0, 16)
    z = np.einsum("bhd,td->bht", q.double().cpu().numpy(), k[:, 0]) / 8
    p = np.exp(z - z.max(2, keepdims=True))
    expected = np.einsum("bht,td->bhd", p / p.sum(2, keepdims=True), v[:, 0])
    # a thread adds less than 2 * 10^5 weights (3 tiles of 2^26 pairs over 2000 warps, two a pair) and as many products
    # with the zeros, each addition off by 2^-25 of the sum at most, all alike where the terms are: 6e-3 each
    error = abs(got.double().cpu().numpy() - expected)[fine]
    assert (error <= 1.2e-2 * abs(v).max() + torch.finfo(dtype).eps / 2 * abs(expected[fine])).all(), error.max()


def test_as_many_rows_of_heads_as_a_call_takes(gpu):
    """2^31 rows of heads, all of them the same ones, appended; of their pages one is there."""
    rows, heads, D = 1 << 16, 1 << 15, 64
    pages = torch.zeros(cache.pages_shape(1, heads, 16, D), dtype=torch.uint8, device="cuda")
    tables = torch.full((1, rows // 16), -1, dtype=torch.int32, device="cuda")
    tables[0, 2000] = 0
    base = queries(97, 1, heads, D, torch.bfloat16)
    k, v = base.expand(rows, heads, D), base.flip(2).contiguous().expand(rows, heads, D)
    cache.append(gpu, k, v, pages, tables, tensor([rows]), tensor([0, rows]))
    raw = ref.encode(base[0].float().cpu().numpy(), base[0].flip(1).float().cpu().numpy())
    expected = np.zeros((heads, 18 * D), np.uint8)
    for index in ref.cell_index(D):
        expected[:, index] = raw
    assert np.array_equal(pages[0, :, 0].cpu().numpy(), expected)
    with pytest.raises(LsxError, match="rows of heads"):
        cache.append(gpu, base.expand(rows + 1, heads, D), base.expand(rows + 1, heads, D), pages, tables, tensor([rows + 1]),
                     tensor([0, rows + 1]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_long_sums_do_not_drift(gpu, dtype):
    """Warps with thousands of pairs of cells each: 200 thousand positions for 256 sequences of 8 heads, whose tables name
    the same pages again and again, values of one sign so that every cut goes the same way."""
    heads, D, size, n, length = 8, 64, 64, 256, 200_000
    held, r = make(98, [64 * 40], heads=heads, D=D, size=size, spare=0)
    rng = np.random.default_rng(99)
    order = held[1][0, :40].cpu().numpy()
    raw = ref.encode(*(np.abs(rng.standard_normal((2, 64 * 40, heads, D))).astype(np.float32)))
    pages = held[0].cpu().numpy()
    for t, index in enumerate(ref.cell_index(D)):  # position t of every cell
        at = np.ix_(order, range(heads), range(size // 16), index)
        pages[at] = raw[t::16].reshape(40, size // 16, heads, -1).transpose(0, 2, 1, 3)
    width = -(-length // size)
    tables = rng.integers(0, 40, (n, width)).astype(np.int32)
    q = queries(100, n, heads, D, dtype, 0.1)
    got = cache.attention(gpu, q, tensor(pages, torch.uint8), tensor(tables), tensor([length] * n)).double()
    place = np.empty(40, np.int64)
    place[order] = np.arange(40)
    k, v, _, _ = (torch.from_numpy(a.reshape(40, size, heads, D)).cuda() for a in ref.decode(raw))
    drift, worst = [], []
    for b in range(0, n, 16):
        count = torch.from_numpy(np.bincount(place[tables[b]], minlength=40).astype(np.float64)).cuda()  # how often each page
        last = (length - 1) % size + 1
        z = torch.einsum("hd,pthd->hpt", q[b].double(), k) / 8
        w = torch.exp(z - z.amax((1, 2), keepdim=True)) * count[None, :, None]
        end = place[tables[b, -1]]
        w[:, end, last:] *= (count[end] - 1) / count[end]
        expected = torch.einsum("hpt,pthd->hd", w, v) / w.sum((1, 2))[:, None]
        error = (got[b] - expected) / expected
        drift.append(error.mean())
        worst.append(error.abs().max())
    # 12.8 million pairs (32 positions of a head) over 2400 warps are 5300 a warp.  Cut by half a unit, 2^-24 of the sum, at each of
    # 2 (f32 4) steps a pair, a sum that is not put aside ends 5300 * 2 * 2^-24 / 2 = 3e-4 too small on average.  Put
    # aside, 256 (f32 128) steps leave 2^-24 * 256 / 2 = 8e-6, and the f32 sums of some 20000 terms a thread, which round to
    # nearest, 2e-6 or so.  The result's rounding (f16 2^-11, bf16 2^-8 at most) is to both sides and, over 512 elements of 16
    # sequences, 1/50 of half a step on average: 5e-6, 4e-5.
    allowed = {torch.float32: 1e-5, torch.float16: 2e-5, torch.bfloat16: 6e-5}[dtype]
    mean = abs(float(torch.stack(drift).mean()))
    assert mean < allowed, mean
    if dtype is torch.float32:
        assert float(torch.stack(worst).max()) < 2e-5
