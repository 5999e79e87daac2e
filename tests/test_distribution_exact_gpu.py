"""Sums over rows whose logits are equal or masked count their tokens exactly, so one token that
is dropped or counted twice, anywhere in a row and however many blocks share it, shows.

Every kept logit is the row's maximum, its exponential 1, and sums of ones are exact in f32 below
2^24: s = ln(count) up to the logarithm's own rounding and the storage, 4 u ln(count) together
(2.8e-6 for 151936 tokens), where one token makes 1 / count (6.6e-6) and more."""
import math
import threading

import pytest
import torch

from laplacesscissors_b200 import distribution
from test_distribution_gpu import KINDS, U, check_distill, dev, make, order64, teacher_of, within  # noqa: F401

pytestmark = pytest.mark.gpu

# Numbers of rows that leave a row to 8, 4, 2 and 1 blocks, and to narrower ones, on 148 SMs.
ROWS = [3, 100, 200, 600, 800, 1000]


def rows_at(dev, rows, vocab, dtype, lead, fill):
    """Rows whose first element lies `lead` elements after a 16-byte boundary."""
    n = 16 // torch.empty(0, dtype=dtype).element_size()
    width = (vocab + lead + n - 1) // n * n
    buffer = torch.full((rows, width), 3.0, dtype=dtype, device=dev)
    z = buffer[:, lead:lead + vocab]
    z.fill_(fill)
    return z


def equal_logits(dev, seed, rows, vocab, dtype, lead):
    """Rows of 1.5 with nothing, some and nearly everything masked; rows kept [rows, vocab]."""
    z = rows_at(dev, rows, vocab, dtype, lead, 1.5)
    g = torch.Generator(device=dev).manual_seed(seed)
    drop = torch.tensor([0.0, 0.02, 0.5, 0.999], device=dev)[torch.arange(rows, device=dev) % 4]
    kept = torch.rand(rows, vocab, generator=g, device=dev) >= drop[:, None]
    kept[:, [0, vocab // 2, vocab - 1]] = True
    z.masked_fill_(~kept, -math.inf)
    return z, kept


def layouts(vocab):
    return [(torch.float32, 0), (torch.float32, 3), (torch.float16, 5), (torch.bfloat16, 0), (torch.bfloat16, 1)]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("vocab", [16411, 40003, 151936])
def test_equal_logits_are_counted(gpu, dev, vocab, rows):
    if vocab == 151936 and rows > 600:
        rows = 300  # (a row of its own from 297 rows on)
    for i, (dtype, lead) in enumerate(layouts(vocab)):
        z, kept = equal_logits(dev, i, rows, vocab, dtype, lead)
        count = kept.sum(1).double()
        got = distribution.token_logprobs(gpu, z, alternatives=3)
        want = count.log()
        within(got.stats[:, 0], torch.full_like(want, 1.5), 0.0)
        within(got.stats[:, 1], want, 4 * U * want)
        within(got.entropy, want, 4 * U * want)
        assert torch.equal(got.top_ids.long(), order64(z, 3))
        # listed: tokens of all stretches of the row, each kept
        k = 24
        ids = torch.linspace(0, vocab - 1, k, device=dev).round().int().expand(rows, k).contiguous()
        ids = torch.where(kept.gather(1, ids.long()), ids, -1)
        listed = (ids >= 0).sum(1).double()
        values = torch.zeros(rows, k, device=dev)
        stats = torch.tensor([[0.0, math.log(k)]] * rows, device=dev)
        for gradient in (False, True):
            d = distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=gradient)
            within(d.stats[:, 1], want, 4 * U * want)
            within(d.stats[:, 2], (count - listed).log(), 4 * U * want)
            d = distribution.distill(gpu, z, ids, values, gradient=gradient)
            loss = want - listed.log()  # a uniform teacher over its list
            within(d.loss, loss, 4 * U * (loss.abs() + 1))


@pytest.mark.parametrize("dtype, lead", [(torch.float32, 0), (torch.float32, 1), (torch.float16, 3), (torch.bfloat16, 7)])
def test_single_tokens_at_the_seams(gpu, dev, dtype, lead):
    """One token of all mass, and two that share it, at the ends of a row's vectors and of the
    slices that 2, 4 and 8 blocks take: s is 0 and ln 2 exactly."""
    vocab = 70001
    n = 16 // torch.empty(0, dtype=dtype).element_size()
    first, full = (1 if lead else 0), (lead + vocab) // n - (1 if lead else 0)
    at = {0, 1, n - lead - 1, n - lead, vocab // 2, vocab - 1, vocab - 2}
    for parts in (2, 4, 8):
        step = (full + parts - 1) // parts
        for p in range(1, parts):
            seam = (first + p * step) * n - lead
            at |= {seam - n, seam - 1, seam, seam + n - 1}
    end = (first + full) * n - lead
    at |= {end - 1, min(end, vocab - 1)}
    at = sorted(a for a in at if 0 <= a < vocab)
    assert len(at) <= 74
    for repeat in (1, 2, 4, 9):  # of the rows, for 8, 4, 2 and 1 blocks to each
        one = torch.tensor(at * repeat, device=dev)
        two = (one + 1) % vocab
        R = len(one)
        z = rows_at(dev, R, vocab, dtype, lead, -math.inf)
        z[torch.arange(R), one] = -2.5
        tokens = torch.stack([one, two], 1).int()
        got = distribution.token_logprobs(gpu, z, tokens, alternatives=1)
        assert not bool(got.stats[:, 1].any()) and not bool(got.entropy.any())
        assert not bool(got.logprob[:, 0].any()) and bool((got.logprob[:, 1] == -math.inf).all())
        assert torch.equal(got.top_ids[:, 0].long(), one)
        none = torch.zeros(R, 2, device=dev)
        for gradient in (False, True):
            d = distribution.distill(gpu, z, tokens, none, teacher_stats=none, gradient=gradient)
            assert not bool(d.stats[:, 1].any()) and bool((d.stats[:, 2] == -math.inf).all())
        z[torch.arange(R), two] = -2.5
        got = distribution.token_logprobs(gpu, z, tokens, alternatives=2)
        ln2 = torch.full((R,), math.log(2.0), dtype=torch.float64, device=dev)
        for x in (got.stats[:, 1], got.entropy, -got.logprob[:, 0], -got.logprob[:, 1]):
            within(x, ln2, 2 * U)
        both = torch.stack([torch.minimum(one, two), torch.maximum(one, two)], 1)
        assert torch.equal(got.top_ids.long(), both)
        only = torch.stack([one, torch.full_like(one, -1)], 1).int().contiguous()
        for gradient in (False, True):
            d = distribution.distill(gpu, z, only, none, teacher_stats=none, gradient=gradient)
            within(d.stats[:, 1], ln2, 2 * U)
            assert not bool(d.stats[:, 2].any())


@pytest.mark.parametrize("rows", [3, 100, 200, 600])
def test_peaked_rows_are_counted(gpu, dev, rows):
    """One token, at any place, above equal others that hold 2^-24 of its mass each: where it lies is
    left out of the sum once.  The others' sum goes through at most vocab / 512 + 24 roundings of
    2^-24 and an exponential off by 2^-22: 6.4e-6 relative, where one token makes 2.5e-5."""
    vocab, T = 40003, math.log2(math.e)  # a difference of 1 is one power of two
    tol = (vocab / 512 + 24) * U + 2.0 ** -22
    for dtype, lead in ((torch.float32, 3), (torch.bfloat16, 0), (torch.float16, 1)):
        z = rows_at(dev, rows, vocab, dtype, lead, -8.0)
        n = 16 // torch.empty(0, dtype=dtype).element_size()
        at = (torch.arange(rows, device=dev) * 9973 + torch.tensor([0, n - lead, vocab - 1], device=dev)[
            torch.arange(rows, device=dev) % 3]) % vocab
        z[torch.arange(rows), at] = 16.0
        got = distribution.token_logprobs(gpu, z, at.int()[:, None].contiguous(), temperature=T)
        r = torch.full((rows,), (vocab - 1) * 2.0 ** -24, dtype=torch.float64, device=dev)
        log_sum = torch.log1p(r)
        within(got.stats[:, 1], log_sum, tol * log_sum)
        within(got.logprob[:, 0], -log_sum, tol * log_sum)
        entropy = log_sum + r / (1 + r) * 24 * math.log(2)
        within(got.entropy, entropy, 2 * tol * entropy)


def test_marks_of_rows_longer_than_the_bitmap(gpu, dev):
    """Rows to a block each of 37984 vectors, whose marks share bitmap words: 128 listed tokens put
    fewer vectors aside than are kept, and more."""
    rows, vocab = 298, 151936
    z, kept = equal_logits(dev, 7, rows, vocab, torch.float32, 0)
    count = kept.sum(1).double()
    for k, step in ((100, 600), (128, 512)):  # 235 and 297 vectors of an unmasked row
        ids = (torch.arange(k, device=dev) * step).int().expand(rows, k).contiguous()
        ids = torch.where(kept.gather(1, ids.long()), ids, -1)
        listed = (ids >= 0).sum(1).double()
        stats = torch.tensor([[0.0, math.log(k)]] * rows, device=dev)
        d = distribution.distill(gpu, z, ids, torch.zeros(rows, k, device=dev), teacher_stats=stats)
        within(d.stats[:, 1], count.log(), 4 * U * count.log())
        within(d.stats[:, 2], (count - listed).log(), 4 * U * count.log())
    z = make(dev, 90, rows, vocab, torch.float32)
    ids, values, stats = teacher_of(dev, 91, z, 128, 1.0)
    check_distill(gpu, z, ids, values, stats, torch.ones(rows, device=dev), 1.0)


def test_two_threads_at_once(gpu, dev):
    """Two threads of one program, each with its stream, on one context."""
    inputs = []
    for i, (rows, vocab, dtype) in enumerate([(5, 151936, torch.float32), (300, 20011, torch.bfloat16)]):
        z = make(dev, 95 + i, rows, vocab, dtype)
        inputs.append((z, *teacher_of(dev, i, z, 32, 1.0)))

    def work(z, ids, values, stats):
        return [*distribution.token_logprobs(gpu, z, ids, alternatives=40),
                *distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)]

    want = [work(*x) for x in inputs]
    torch.cuda.synchronize(dev)
    wrong, streams = [], [torch.cuda.Stream(dev) for _ in inputs]

    def run(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(50):
                    got = work(*inputs[i])
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001 (told to the test's own thread)
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize(dev)
    assert not wrong
