"""The paged cache in 4 bits against its restatement in 64 bits (tests/cache_reference.py): append, read and
attention at the sizes and tables where they can go wrong."""
import numpy as np
import pytest
import torch

import cache_reference as ref
from laplacesscissors_b200 import cache

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def tensor(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


def make(seed, lengths, heads=2, D=64, size=32, spare=3, offset=1.0):
    """A cache of random cells: (pages, tables, lengths) on the device and the Reference; every cell holds
    encoded keys and values, those behind a sequence's end too."""
    rng = np.random.default_rng(seed)
    need = [-(-n // size) for n in lengths]
    count = sum(need) + spare
    order = rng.permutation(count)
    tables = np.full((len(lengths), max(need) + 2), -1, np.int32)
    first = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[first:first + n]
        first += n
    pages = np.zeros((count, heads, size // 16, 18 * D), np.uint8)
    index = ref.cell_index(D)
    shape = (count, heads, size // 16, 16, D)
    k = (rng.standard_normal(shape) * rng.uniform(0.3, 2, D) + offset * rng.standard_normal(D)).astype(np.float32)
    v = (rng.standard_normal(shape) + 0.3 * rng.standard_normal(D)).astype(np.float32)
    raw = ref.encode(k, v)
    for t in range(16):
        pages[..., index[t]] = raw[..., t, :]
    lengths = np.array(lengths, np.int32)
    return (tensor(pages, torch.uint8), tensor(tables), tensor(lengths)), ref.Reference(pages, tables, lengths)


def queries(seed, rows, heads, D, dtype, size=1.0):
    rng = np.random.default_rng(seed + 1000)
    return tensor(size * rng.standard_normal((rows, heads, D)), torch.float32).to(dtype)


def tolerance(r, q, scale, expected, bound, wide, dtype, longest):
    """What rounding may do.  A score is a sum over D of q (s n + z) held as s sum(q n) + z sum(q), so its terms are
    bounded by |q| (15 s + |z|), whose scaled sum is `bound`.  Queries keep 22 bits or more and a tensor core adds
    16 products at a time, cutting what lies 2^-22 below the largest: D / 16 steps of two terms, the groups' sums and
    the scaling leave (D / 8 + 16) 2^-22 of the bound, and the reference point as much again as one step.  A weight is
    off by that, twice (it and the sum), and by exp2's 2^-21.  The output adds the weights' rounding (2^-22, or 2^-11 of
    the 15 s part where f16 or bf16 rows share a matrix instruction) and the steps' of the sum over the positions,
    against sum p (15 s + |z|) = `wide`."""
    score = (q.shape[2] / 8 + 16) * 2.0 ** -22 * bound
    weight = 2 * np.expm1(score) + 2.0 ** -20
    single = 0 if dtype is torch.float32 else 2.0 ** -11
    output = (longest / 16 + 32) * 2.0 ** -22 + single
    return (weight + output) * wide + torch.finfo(dtype).eps / 2 * abs(expected)


def check(gpu, held, r, q, starts=None, sequences=None, scale=None, out=None):
    tables = [None if a is None else tensor(a) for a in (starts, sequences)]
    got = cache.attention(gpu, q, *held, tables[0], sequences=tables[1], scale=scale, out=out)
    factor = q.shape[2] ** -0.5 if scale is None else scale
    expected, bound, wide, used = r.attention(q.double().cpu().numpy(), factor, starts, sequences)
    allowed = tolerance(r, q, factor, expected, bound, wide, q.dtype, int(max(r.lengths.max(), 1)))
    got = got.double().cpu().numpy()
    assert used.any()
    nan = np.isnan(expected[used])
    assert (np.isnan(got[used]) == nan).all()
    error = np.where(nan, 0, abs(got[used] - expected[used]) - allowed[used])
    assert (error <= 0).all(), (error.max(), np.unravel_index(error.argmax(), error.shape))
    return got


# ---- append and read ------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [0, 17, 5, 40], [3, 0, 0, 0], [70, 1, 33, 2]])
def test_append_writes_the_documented_bytes(gpu, dtype, D, counts):
    held, r = make(D, [3, 40, 33, 97], D=D)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rng = np.random.default_rng(7)
    packed = tensor(rng.standard_normal((starts[-1] + 2, 2, 2, D)) * 3, torch.float32).to(dtype)  # two rows of no sequence
    k, v = packed[:, 0], packed[:, 1]
    cache.append(gpu, k, v, *held, tensor(starts))
    r.append(k.float().cpu().numpy(), v.float().cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)
    for out_type in TYPES:
        back = [torch.full((starts[-1] + 2, 2, D), 7.0, dtype=out_type, device="cuda") for _ in range(2)]
        cache.read(gpu, *held, tensor(starts), out=back)
        expected = r.read(starts[-1], starts)
        for got, e in zip(back, expected):
            # s n + z rounded to f32, then to the type: half a step of each
            assert (abs(got[:starts[-1]].double().cpu().numpy() - e) <= (torch.finfo(out_type).eps / 2 + 2.0 ** -24) * abs(e) * 1.001).all()
            assert (got[starts[-1]:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("size", [16, 48])
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_read_of_many_heads_of_rows(gpu, dtype, D, size, strided):
    counts, heads = [70, 0, 9, 1, 52, 17], 80  # enough for cells to be taken whole
    held, r = make(D + size, [73, 5, 9, 40, 33, 17], D=D, heads=heads, size=size)  # 52 rows, 33 positions
    r.tables[0, 2], r.tables[5, 0] = -1, 10 ** 9
    held = (held[0], tensor(r.tables), tensor(r.lengths))
    starts = np.concatenate([[0], np.cumsum(counts)])
    n = int(starts[-1])
    assert n * heads >= 8192 and n >= 8 * len(counts)
    rng = np.random.default_rng(5)
    wide = D + 1 if strided else D  # rows that lie to no 16 bytes
    k, v = (tensor(rng.standard_normal((n + 1, heads, wide)) * 3, torch.float32).to(dtype)[..., :D] for _ in range(2))
    cache.append(gpu, k, v, *held, tensor(starts))
    r.append(k.float().cpu().numpy(), v.float().cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)
    back = [torch.full((n + 1, heads, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    cache.read(gpu, *held, tensor(starts), out=back)
    for got, e in zip(back, r.read(n, starts)):
        got = got.double().cpu().numpy()
        nan = np.isnan(e)
        assert (np.isnan(got[:n]) == nan).all() and (got[n:] == 7).all()
        # s n + z rounded to f32, then to the type: half a step of each
        assert (abs(got[:n] - e)[~nan] <= (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * abs(e)[~nan] * 1.001).all()


@pytest.mark.parametrize("values", ["ties", "not finite"])
def test_cells_taken_whole_hold_values_at_the_ends(gpu, values):
    held, r = make(4, [300, 41], D=64, heads=40)
    starts = [0, 200, 241]
    x = np.random.default_rng(6).standard_normal((241, 40, 64)).astype(np.float32)
    if values == "ties":
        x[:] = np.arange(64) % 31 * 0.5 + (np.arange(241)[:, None, None] - 120)
        x[::3] = np.nextafter(x[::3], np.float32(1e9))
    else:
        x[3, :, 5], x[17, 1, 9], x[18, 2, 60], x[40], x[41] = np.nan, np.inf, -np.inf, 3.25, 0
        x[60, :, 0], x[61, :, 0], x[62, :, 1] = 1e30, -60000, 65519.0
        x[70:90] *= 10.0 ** np.linspace(-9, 4, 20)[:, None, None]
    k = tensor(x, torch.float32)
    cache.append(gpu, k, k.flip(2), *held, tensor(starts))
    r.append(x, x[..., ::-1], starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("strided", [False, True])
def test_cells_taken_whole_hold_values_at_the_ends_in_all_types(gpu, dtype, D, strided):
    """NaN and infinities at even, odd, first and last elements of a group, alone in their row; ties; groups of one
    value, of zeros of both signs, and of what no f16 holds."""
    held, r = make(21, [300, 41], D=D, heads=40)
    starts = [0, 200, 241]
    x = np.random.default_rng(22).standard_normal((241, 40, D)).astype(np.float32)
    for i, bad in enumerate((np.nan, np.inf, -np.inf)):
        for j, at in enumerate((0, 1, 30, 33, 62, 63, D - 64, D - 1)):
            x[3 + 8 * i + j, i::2, at] = bad
    x[40], x[41], x[42, :, ::2] = 3.25, 0, -0.0
    x[43, :, 0], x[44, :, 63], x[45, :, 1], x[46, :, 62] = 65504, -65504, 60000, -60000
    x[47] = 60000 * (-1.0) ** np.arange(D)  # a step within f16
    # levels and ties between them: s = 1 about several zeros, each of which all three types hold
    x[50:114] = np.arange(D) % 31 * 0.5 + (np.arange(64)[:, None, None] - 32)
    x[114:130] = (np.arange(D) % 31 * 0.5 + np.arange(16)[:, None, None]) * 2.0 ** -6
    x[130:170] *= 10.0 ** np.linspace(-9, 4, 40)[:, None, None]
    if dtype is not torch.float16:
        x[171, 1::3, 5], x[172, ::2, 6], x[173, :, 0] = 1e30, -3e38, 65520.0  # the last rounds to infinity in f16
    wide = D + 1 if strided else D
    k = torch.zeros((241, 40, wide), device="cuda").to(dtype)[..., :D]
    k.copy_(tensor(x, torch.float32))
    v = torch.zeros((241, 40, wide), device="cuda").to(dtype)[..., :D]
    v.copy_(k.flip(2))
    cache.append(gpu, k, v, *held, tensor(starts))
    r.append(k.float().cpu().numpy(), v.float().cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)


def test_append_one_row_a_sequence_and_a_list(gpu):
    held, r = make(1, [3, 40, 33, 97, 64], D=128)
    k, v = (queries(i, 4, 2, 128, torch.float32) for i in (1, 2))
    names = [4, 9, 1, -3]  # two name no sequence
    cache.append(gpu, k, v, *held, sequences=tensor(names))
    r.append(k.cpu().numpy(), v.cpu().numpy(), None, names)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)
    got = cache.read(gpu, *held, sequences=tensor(names))
    expected = r.read(4, None, names)
    for a, e in zip(got, expected):
        assert np.allclose(a.cpu().numpy(), e, rtol=2.0 ** -23, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_values_that_cannot_be_held_or_lie_on_a_tie(gpu, dtype):
    held, r = make(2, [64, 64, 64], D=64, heads=1)
    x = np.zeros((24, 1, 64), np.float32)
    x[0, 0, 5] = np.nan
    x[1, 0, 9], x[2, 0, 9] = np.inf, -np.inf
    x[3], x[4] = 3.25, 0
    x[5, 0] = np.arange(64) % 31 * 0.5          # s = 1: levels and exact ties between them
    x[6, 0] = 100 + np.arange(64) % 31 * 0.5
    x[7, 0] = -1000 + np.arange(64) % 31 * 0.5
    x[8, 0, 3], x[9, 0, 3] = 60000, -60000
    x[10, 0] = 60000 * (-1) ** np.arange(64)
    x[11, 0, :2] = 1e-7, -1e-7
    x[12, 0, 0] = -0.0
    rng = np.random.default_rng(3)
    x[13:] = rng.standard_normal((11, 1, 64)) * 10.0 ** rng.integers(-6, 5, (11, 1, 1))
    if dtype is torch.float32:
        x[14, 0, 1], x[15, 0, 1] = 1e30, -3e38
        x[16, 0] = np.nextafter(x[5, 0], 100)   # next to the ties
        x[17, 0] = np.nextafter(x[5, 0], -100)
        x[18, 0] = 1e-42
    k = tensor(x, torch.float32).to(dtype)
    starts = [0, 8, 16, 24]
    cache.append(gpu, k, k.flip(2), *held, tensor(starts))
    r.append(k.float().cpu().numpy(), k.flip(2).float().cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)


def test_append_passes_over_what_has_no_page(gpu):
    held, r = make(3, [20, 70, 200, 5], D=64, size=16)
    for (b, slot), page in {(0, 1): -1, (1, 2): 10 ** 9, (1, 3): -7}.items():
        r.tables[b, slot] = page
    r.lengths[2] = 300  # beyond its row of the tables
    held = (held[0], tensor(r.tables), tensor(r.lengths))
    counts = [20, 70, 120, 9]  # the last has more rows than positions
    starts = np.concatenate([[0], np.cumsum(counts)])
    k, v = (queries(i, starts[-1], 2, 64, torch.float32) for i in (4, 5))
    cache.append(gpu, k, v, *held, tensor(starts))
    r.append(k.cpu().numpy(), v.cpu().numpy(), starts)
    assert np.array_equal(held[0].cpu().numpy(), r.pages)
    got = cache.read(gpu, *held, tensor(starts), rows=int(starts[-1]))
    expected = r.read(starts[-1], starts)
    for a, e in zip(got, expected):
        assert np.allclose(a.cpu().numpy(), e, rtol=2.0 ** -23, atol=0, equal_nan=True)


# ---- attention -------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("group", [1, 3, 8, 9, 20])
def test_one_row_a_sequence(gpu, dtype, D, group):
    held, r = make(group, [0, 1, 2, 15, 16, 17, 31, 33, 64, 200, 333], D=D)
    check(gpu, held, r, queries(group, 11, 2 * group, D, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [16, 48, 128])
@pytest.mark.parametrize("group,heads", [(1, 3), (2, 1), (7, 2), (16, 1)])
def test_several_rows_a_sequence(gpu, dtype, size, group, heads):
    lengths, counts = [5, 130, 64, 0, 77, 300], [5, 2, 64, 0, 9, 40]
    held, r = make(size + group, lengths, heads=heads, size=size, D=64)
    starts = np.concatenate([[0], np.cumsum(counts)])
    check(gpu, held, r, queries(3, starts[-1], heads * group, 64, dtype), starts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 192, 256])
@pytest.mark.parametrize("counts,group", [([1] * 11 + [37], 1), ([2, 0, 1, 1, 5, 0, 0, 1], 2), ([1, 1, 1, 9, 0, 0], 4), ([1] * 15 + [50], 4)])
def test_few_rows_but_for_one_sequence(gpu, dtype, D, counts, group):
    lengths = [max(n, 700 * (i % 3 == 0) + 13 * i) for i, n in enumerate(counts)]
    held, r = make(group + D, lengths, D=D)
    starts = np.concatenate([[0], np.cumsum(counts)])
    check(gpu, held, r, queries(group, int(starts[-1]), 2 * group, D, dtype), starts)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_rows_than_positions_and_rows_of_no_sequence(gpu, dtype):
    held, r = make(8, [3, 0, 40], D=128)
    starts = [2, 9, 13, 17]
    q = queries(9, 20, 4, 128, dtype)
    out = torch.full_like(q, 5.0)
    got = check(gpu, held, r, q, starts, out=out)
    assert (got[:2] == 5).all() and (got[17:] == 5).all()  # rows before the first and behind the last
    assert (got[2:6] == 0).all() and (got[9:13] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_list_of_sequences(gpu, dtype):
    held, r = make(9, [50, 3, 200, 17], D=64)
    check(gpu, held, r, queries(10, 6, 4, 64, dtype), None, [2, 2, 0, 77, 3, -1])
    check(gpu, held, r, queries(11, 9, 4, 64, dtype), [0, 3, 4, 9], [2, 77, 0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 30, 20]])
def test_pages_that_are_not_there(gpu, dtype, counts):
    """Rows that see a missing page are NaN, rows before it are not."""
    held, r = make(10, [100, 90, 80], D=64, size=16)
    r.tables[0, 4], r.tables[1, 3] = -1, 10 ** 9
    r.tables[2, 4:] = -5
    starts = np.concatenate([[0], np.cumsum(counts)])
    got = check(gpu, (held[0], tensor(r.tables), held[2]), r, queries(12, starts[-1], 4, 64, dtype), starts)
    if counts[0] == 40:
        assert not np.isnan(got[:4]).any() and np.isnan(got[4:40]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_lies_behind_the_end_is_not_seen(gpu, dtype):
    """NaN in the cells' unused positions, in pages of nobody, and in later positions than a row's own."""
    held, r = make(11, [21, 50, 1], D=64, size=16)
    index = ref.cell_index(64)
    for b, n in enumerate([21, 46, 1]):  # positions 46 .. 49 of the second are NaN
        for position in range(n, -(-n // 16) * 16):
            r.cell(b, position)[:, index[position % 16][-16:]] = 0xff
    for page in set(range(len(r.pages))) - set(r.tables.reshape(-1).tolist()):
        r.pages[page] = 0xff
    starts = [0, 3, 13, 14]
    got = check(gpu, (tensor(r.pages, torch.uint8), *held[1:]), r, queries(13, 14, 6, 64, dtype), starts)
    assert not np.isnan(got[:9]).any() and np.isnan(got[9:13]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_at_the_ends_of_their_range(gpu, dtype):
    held, r = make(12, [40, 40, 40, 40, 40, 40], D=64, heads=1)
    q = queries(14, 6, 2, 64, torch.float32)
    q[0] *= 1e-5
    q[1] = 0
    q[2] *= 300      # weights of one position only
    q[3, 0, 7] = float("nan")
    q[4, 1, 9] = float("inf")
    q[5, :, :32] *= 1e-3
    q = q.to(dtype)
    got = cache.attention(gpu, q, *held).double().cpu().numpy()
    for bad in ((3, 0), (4, 1)):
        assert np.isnan(got[bad]).all()
    q[3, 0], q[4, 1] = 0, 0
    expected, bound, wide, _ = r.attention(q.double().cpu().numpy(), 0.125)
    allowed = tolerance(r, q, 0.125, expected, bound, wide, dtype, 40)
    for b in range(6):
        for h in range(2):
            if (b, h) not in ((3, 0), (4, 1)):
                assert (abs(got[b, h] - expected[b, h]) <= allowed[b, h]).all(), (b, h)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_of_many_magnitudes(gpu, dtype):
    """Steps from 2^-20 to 2^11 in one sequence: small values beside large ones, large ones last."""
    held, r = make(13, [160, 160], D=64, heads=1, size=16)
    k, v = (np.random.default_rng(i).standard_normal((320, 1, 64)).astype(np.float32) for i in (1, 2))
    v *= (10.0 ** np.linspace(-5, 4, 320))[:, None, None].astype(np.float32)
    v[160:] = v[160:][::-1].copy()
    starts = [0, 160, 320]
    r.append(k, v, starts)
    cache.append(gpu, tensor(k, torch.float32), tensor(v, torch.float32), *held, tensor(starts))
    check(gpu, held, r, queries(15, 24, 2, 64, dtype), [0, 4, 24])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,ratios", [(128, (1e3, 1e-3)), (128, (1e-4, 1e4)), (256, (3e3, 1e-4, 1.0, 1e-3)), (192, (1e-5, 2e4, 1e-1))])
@pytest.mark.parametrize("rows", [1, 5, 30])
def test_groups_of_many_magnitudes(gpu, dtype, D, ratios, rows):
    """Groups of a head whose steps lie 2^20 and more apart: each is as near to its own sum p (15 s + |z|)."""
    held, r = make(17, [160, 75], D=D, heads=1, size=16)
    k, v = (np.random.default_rng(i).standard_normal((235, 1, D)).astype(np.float32) for i in (3, 4))
    v *= np.repeat(np.array(ratios, np.float32), 64)
    starts = [0, 160, 235]
    r.append(k, v, starts)
    cache.append(gpu, tensor(k, torch.float32), tensor(v, torch.float32), *held, tensor(starts))
    check(gpu, held, r, queries(16, 2 * rows, 2, D, dtype), [0, rows, 2 * rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 4, 17])
@pytest.mark.parametrize("groups", ["all", "first"])
def test_large_values_of_little_weight(gpu, dtype, D, rows, groups):
    """In each sequence a position whose values are 2^28 times the others' and whose weight is below 2^-60 of theirs: what
    the others leave, one of them above all, is held as it is without it."""
    lengths = list(range(rows + 11, rows + 23))
    held, r = make(18, lengths, D=D, heads=1, size=16)
    rng = np.random.default_rng(9)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    k, v = (0.02 * rng.standard_normal((starts[-1], 1, D)).astype(np.float32) for _ in range(2))
    v *= np.float32(5e-3)
    k[starts[:-1] + 5] -= 1.0
    k[starts[:-1] + 7] += 0.2
    v[starts[:-1] + 5, :, :D if groups == "all" else 64] *= np.float32(3e8)
    r.append(k, v, starts)
    cache.append(gpu, tensor(k, torch.float32), tensor(v, torch.float32), *held, tensor(starts))
    q = (42 / D * (1 + 0.01 * queries(17, 12 * rows, 2, D, torch.float32))).to(dtype)  # scores of 42 less: 2^-60
    check(gpu, held, r, q, list(range(0, 12 * rows + 1, rows)), scale=1.0)


@pytest.mark.parametrize("dtype,size,scale", [
    (torch.float32, 1e12, 1.0), (torch.float32, 1e12, -1.0), (torch.float32, 1e32, 1.0), (torch.float32, 3e37, 0.125),
    (torch.float32, 3e37, -1e20), (torch.float32, 1.0, 1e29), (torch.float16, 1e4, 1e9),
    (torch.float16, 1e-3, -1e28), (torch.bfloat16, 1e12, 1.0), (torch.bfloat16, 1e32, -1.0), (torch.bfloat16, 3e37, 1e15)])
@pytest.mark.parametrize("sign", [0, 1, -1])
@pytest.mark.parametrize("rows,length", [(1, 40), (9, 90), (1, 3000)])
def test_scores_of_any_size(gpu, dtype, size, scale, sign, rows, length):
    """Scores up to 10^60 apart, all of one sign or not: the position with the largest has all the weight."""
    held, r = make(19, [length, length], D=64, heads=1, offset=8.0 if sign else 1.0)
    k, v, k_wide, v_wide = r.values(0, length)
    q = queries(18, 2 * rows, 4, 64, torch.float32)
    if sign:  # along the keys' mean, so that all scores have its sign
        mean = np.concatenate([k, r.values(1, length)[0]]).mean((0, 1))
        q = q * 0.05 + sign * tensor(mean / abs(mean).max(), torch.float32)
    q = (q / 6 * size).to(dtype)
    got = cache.attention(gpu, q, *held, tensor([0, rows, 2 * rows]), scale=scale).double().cpu().numpy()
    x = q.double().cpu().numpy()
    used = 0
    for row in range(2 * rows):
        k, v, k_wide, v_wide = (a[:length - rows + 1 + row % rows, 0] for a in r.values(row // rows, length))
        for h in range(4):
            z = k @ x[row, h] * np.sign(scale)
            order = np.argsort(z)[::-1]
            # the score's rounding as in `tolerance`, of differences: further apart than that, and by 40 in the exponent
            apart = z[order[0]] - z[order[1]]
            if apart < 2 * (64 / 8 + 16) * 2.0 ** -22 * (k_wide @ abs(x[row, h])).max() or apart * abs(scale) < 60:
                continue
            used += 1
            error = abs(got[row, h] - v[order[0]])
            single = 0 if dtype is torch.float32 else 2.0 ** -11
            assert (error <= (2.0 ** -19 + single) * v_wide[order[0]] + torch.finfo(dtype).eps / 2 * abs(v[order[0]])).all(), (row, h)
    assert used > 4 * rows


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_queries_and_small_scales(gpu, dtype):
    held, r = make(20, [70, 19], D=128)
    check(gpu, held, r, (queries(16, 2, 4, 128, torch.float32) * 1e35).to(dtype), scale=1e-36)
    check(gpu, held, r, (queries(16, 2, 4, 128, torch.float32) * 1e-35).to(dtype), scale=1e29)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(gpu, scale):
    held, r = make(14, [70, 19], D=128)
    check(gpu, held, r, queries(16, 2, 4, 128, torch.float32), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(gpu, dtype):
    """Queries within a packed projection, an output with rows apart, heads before rows."""
    held, r = make(15, [70, 19, 33], D=64)
    base = queries(17, 3, 9, 64, dtype)
    out = torch.full((3, 7, 64), 3.0, dtype=dtype, device="cuda")
    check(gpu, held, r, base[:, 1:5], out=out[:, 2:6])
    assert (out[:, :2] == 3).all() and (out[:, 6:] == 3).all()
    turned = queries(18, 4, 3, 64, dtype).transpose(0, 1)
    check(gpu, held, r, turned, out=torch.zeros(4, 3, 64, dtype=dtype, device="cuda").transpose(0, 1))
    odd = torch.zeros(3 * 4 * 64 + 1, dtype=dtype, device="cuda")[1:].view(3, 4, 64)  # not aligned to 16 bytes
    check(gpu, held, r, odd.copy_(base[:, :4]), out=torch.zeros(3 * 4 * 64 + 1, dtype=dtype, device="cuda")[1:].view(3, 4, 64))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,heads,group", [([9000], 1, 4), ([5000, 3, 7000], 2, 12), ([1500] * 40, 3, 1)])
def test_long_sequences_are_shared_by_blocks(gpu, dtype, lengths, heads, group):
    held, r = make(16, lengths, heads=heads, D=64, size=64)
    rows = len(lengths)
    if rows > 3:  # the reference is slow: a list of some of them, in two calls that cover the lengths
        check(gpu, held, r, queries(19, 5, heads * group, 64, dtype), None, [0, 39, 7, 7, 20])
        full = cache.attention(gpu, queries(20, rows, heads * group, 64, dtype), *held)
        part = cache.attention(gpu, queries(20, rows, heads * group, 64, dtype)[3:5].contiguous(), *held, sequences=tensor([3, 4]))
        assert torch.allclose(full[3:5].float(), part.float(), rtol=2e-2, atol=2e-3)
    else:
        check(gpu, held, r, queries(19, rows, heads * group, 64, dtype))
