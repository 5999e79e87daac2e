"""Operators on rows of logits (laplacesscissors_b200/distribution.py over
lsx_token_logprobs_device, lsx_distill_device and their backward entries) against their
formulas in 64 bits, on every storage type, at odd sizes, strides and masks, with their
gradients also against differences; ordering with torch's streams and captured graphs.

Tolerances, with u = 2^-24 (half a step of f32): a thread adds at most V/128 terms one
after another and the threads' sums meet in a tree, the exponential is off by 2^-22 and its
argument y by 3u|y|, and sum p|y| <= log2 V < 20 for the vocabularies here, so the sum of
exponentials is off by at most (V/128 + 30 + 4 + 0.7 * 3 * 20) u relative: sum_tol() takes
(V/128 + 80) u.  A 16-bit output adds half a step of its type."""
import math

import numpy as np
import pytest
import torch

import laplacesscissors_b200 as lsx
from laplacesscissors_b200 import LsxError, distribution
from laplacesscissors_b200._lib import lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KINDS = [torch.float32, torch.float16, torch.bfloat16]
UNUSED = -1


@pytest.fixture(scope="module")
def dev(gpu):
    return torch.device("cuda", gpu.device)


def sum_tol(vocab):
    return (vocab / 128 + 80) * U


def make(dev, seed, rows, vocab, dtype, pad=0, scale=2.5, masked=0.0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * scale
    likely = torch.randint(0, vocab, (rows, 4), generator=g)
    z[torch.arange(rows)[:, None], likely] = 6.0 + 3.0 * torch.randn(rows, 4, generator=g)
    if masked:
        drop = torch.rand(rows, vocab, generator=g) < masked
        drop[:, vocab // 2] = False
        z.masked_fill_(drop, -math.inf)
    buffer = torch.full((rows, vocab + pad), 7.0, dtype=dtype, device=dev)
    buffer[:, :vocab] = z.to(dtype).to(dev)
    return buffer[:, :vocab]


def softmax64(logits, T):
    """(m, log sum, ln q) in 64 bits, with the statistics of empty rows as documented."""
    z = logits.double()
    m = z.amax(1)
    empty = m == -math.inf
    y = torch.where(z == -math.inf, z, (z - torch.where(empty, 0.0, m)[:, None]) / T)
    s = torch.where(empty, 0.0, torch.log(torch.exp(y).sum(1)))
    return m, s, y - s[:, None]


def entropy64(log_q):
    q = log_q.exp()
    return -torch.where(q > 0, q * log_q, 0.0).sum(1)


def order64(logits, k):
    """Ids by (logit descending, id ascending); NaN first, -0 equal to 0."""
    z = torch.nan_to_num(logits.double(), nan=math.inf, posinf=1e300, neginf=-math.inf) + 0.0
    return torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]


def within(actual, expected, tol):
    a, e = actual.double(), expected.double()
    # outputs are f32: what lies beyond its largest number, 3.4e38, rounds to infinity
    # (the lowest f32 logit at a temperature of 0.05 has a log probability of -6.8e39)
    e = torch.where(e.abs() > torch.finfo(torch.float32).max, torch.sign(e) * math.inf, e)
    tol = torch.as_tensor(tol, dtype=torch.float64, device=a.device).expand_as(e)
    same = (a == e) | (torch.isnan(a) & torch.isnan(e))
    bad = ~same & ~((a - e).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), a[bad][:4], e[bad][:4], tol[bad][:4])


def check_logprobs(gpu, logits, tokens, k, T):
    got = distribution.token_logprobs(gpu, logits, tokens, alternatives=k, temperature=T)
    rows, V = logits.shape
    m, s, log_q = softmax64(logits, T)
    tol = sum_tol(V)
    within(got.stats[:, 0], m, 0.0)
    within(got.stats[:, 1], s, tol + 2 * U * s.abs())
    H = entropy64(log_q)
    # sum p y^2 <= 20^2 * 2: each term's exponent error times its own size, and the sum's rounding
    within(got.entropy, H, 20 * tol + 1200 * U)
    if tokens is not None and tokens.shape[1]:
        t = tokens.long()
        lp = torch.where(t < 0, 0.0, log_q.gather(1, t.clamp_min(0)))
        within(got.logprob, lp, tol + 4 * U * torch.where(lp.isinf(), 0.0, lp.abs()) + 4 * U * s.abs()[:, None])
    if k:
        ids = order64(logits, k)
        assert torch.equal(got.top_ids.long(), ids)
        assert torch.equal(got.top_logits, logits.gather(1, ids).float())
        lp = log_q.gather(1, ids)
        within(got.top_logprobs, lp, tol + 4 * U * torch.where(lp.isinf(), 0.0, lp.abs()) + 4 * U * s.abs()[:, None])
    else:
        assert got.top_ids is None and got.top_logits is None and got.top_logprobs is None
    return got


VOCABS = [1, 2, 3, 7, 8, 9, 31, 33, 127, 512, 1021, 4096, 4099, 16411, 50257, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", KINDS)
def test_logprobs_match(gpu, dev, dtype, vocab):
    for i, (rows, pad, T, k, n, masked) in enumerate([(1, 0, 1.0, min(vocab, 20), 1, 0.0),
                                                      (5, 3, 0.7, min(vocab, 128), 3, 0.5),
                                                      (7, 8, 2.3, min(vocab, 1), 5, 0.97)]):
        z = make(dev, vocab + i, rows, vocab, dtype, pad, masked=masked)
        tokens = torch.randint(-1, vocab, (rows, n), dtype=torch.int32, device=dev)
        check_logprobs(gpu, z, tokens, k, T)


@pytest.mark.parametrize("rows", [1, 2, 9, 18, 37, 75, 149, 300, 600, 1300])
def test_logprobs_row_counts(gpu, dev, rows):
    """Few rows are split over more of the GPU than many: every split gives the formula."""
    for vocab, dtype in ((5003, torch.float32), (33001, torch.bfloat16)):
        z = make(dev, rows, rows, vocab, dtype)
        tokens = torch.randint(0, vocab, (rows, 1), dtype=torch.int32, device=dev)
        check_logprobs(gpu, z, tokens, 11, 1.0)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("vocab", [40, 4099, 70001])
def test_logprobs_special_rows(gpu, dev, dtype, vocab):
    """Masks that leave nothing or one token, the type's lowest value, far offsets, ties,
    signed zeros and rows in order (whose best tokens lie next to one another)."""
    lowest = torch.finfo(dtype).min
    z = torch.zeros(16, vocab, dtype=dtype, device=dev)
    z[0] = -math.inf                                   # no token left
    z[1] = -math.inf
    z[1, vocab - 1] = 3.0                              # one token left
    z[2] = lowest                                      # masked with the type's lowest value throughout
    z[3] = lowest
    z[3, 5] = 1.0
    z[4] = lowest
    z[4, ::2] = -math.inf                              # both masks
    z[5] = torch.finfo(dtype).max                      # a uniform row at the top of the type
    z[6, 1::2] = -0.0                                  # 0 and -0 are equal
    z[7] = torch.linspace(9, -9, vocab).to(dtype)      # descending
    z[8] = torch.linspace(-9, 9, vocab).to(dtype)      # ascending
    z[9] = 1000.0 + torch.randn(vocab, device=dev).to(dtype)
    z[10] = -1000.0 + torch.randn(vocab, device=dev).to(dtype)
    z[11] = -math.inf
    z[11, :3] = 2.0                                    # fewer tokens left than alternatives
    z[12] = torch.randint(0, 2, (vocab,), device=dev).to(dtype)  # two values only
    z[13] = torch.finfo(dtype).tiny
    z[14, vocab // 2:] = 8.0                           # half the row ties for the best
    z[15] = torch.arange(vocab, device=dev).remainder(17).to(dtype)
    tokens = torch.tensor([[0, vocab - 1, 5, UNUSED]] * 16, dtype=torch.int32, device=dev)
    for k in (1, 20, 40, min(vocab, 128)):
        check_logprobs(gpu, z, tokens, k, 1.0)
    check_logprobs(gpu, z, tokens, 3, 0.05)
    check_logprobs(gpu, z, None, 0, 50.0)


@pytest.mark.parametrize("dtype", KINDS)
def test_logprobs_nan_and_infinity(gpu, dev, dtype):
    """A NaN or +inf logit makes its row NaN, leaves the others, and leads the alternatives."""
    vocab = 9001
    z = make(dev, 5, 6, vocab, dtype)
    z[1, 777] = math.nan
    z[2, 8000] = math.inf
    z[3, 3] = -math.nan
    z[3, 5000] = math.inf
    z[4] = math.nan
    tokens = torch.tensor([[4]] * 6, dtype=torch.int32, device=dev)
    got = distribution.token_logprobs(gpu, z, tokens, alternatives=7)
    for r in (1, 2, 3, 4):
        assert bool(got.logprob[r].isnan().all()) and bool(got.entropy[r].isnan()) and bool(got.stats[r, 1].isnan())
        assert bool(got.top_logprobs[r].isnan().all())
    assert torch.equal(got.top_ids.long(), order_special(z, 7))
    fine = [0, 5]
    check_logprobs(gpu, z[fine], tokens[fine], 7, 1.0)
    one = distribution.token_logprobs(gpu, z[fine], tokens[fine], alternatives=7)
    for a, b in zip(got, one):
        within(a[fine], b, 1e-6)


def order_special(z, k):
    rank = z.double()
    rank = torch.where(rank.isnan(), 3.0, torch.where(rank == math.inf, 2.0, torch.where(rank == -math.inf, -2.0,
                                                                                     torch.atan(rank) / 2)))
    return torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :k]


def test_tokens_outside_the_vocabulary(gpu, dev):
    z = make(dev, 6, 3, 500, torch.float32)
    tokens = torch.tensor([[0, 500], [UNUSED, 499], [-2, 2 ** 31 - 1]], dtype=torch.int32, device=dev)
    got = distribution.token_logprobs(gpu, z, tokens)
    nan = got.logprob.isnan().cpu().tolist()
    assert nan == [[False, True], [False, False], [True, True]]
    assert float(got.logprob[1, 0]) == 0.0
    grad = distribution.token_logprobs_backward(gpu, z, tokens, got.stats, got.entropy,
                                                torch.ones(3, 2, device=dev), torch.ones(3, device=dev))
    assert grad.isnan().all(1).cpu().tolist() == [True, False, True]


# ---- gradient of the log probabilities -----------------------------------------------------
def logprobs_gradient64(z, tokens, g, h, T):
    m, s, log_q = softmax64(z, T)
    q = log_q.exp()
    empty = (m == -math.inf)[:, None]
    t = tokens.long()
    g = torch.where(t < 0, 0.0, g.double())
    H = entropy64(log_q)[:, None]
    ln_q = torch.where(q > 0, log_q, 0.0)
    inner = g.sum(1, keepdim=True) + h.double()[:, None] * (ln_q + H)
    out = -q * inner
    out.scatter_add_(1, t.clamp_min(0), g)
    # relative error of q, of the entropy, and of the marked values
    rho = sum_tol(z.shape[1]) + (3 * ln_q.abs() + 3 * s.abs()[:, None] + 10) * 2 * U
    size = g.abs().sum(1, keepdim=True) + h.double().abs()[:, None] * (ln_q.abs() + H)
    tol = q * (size * rho + h.double().abs()[:, None] * (20 * sum_tol(z.shape[1]) + 1200 * U))
    tol += torch.zeros_like(out).scatter_add_(1, t.clamp_min(0), 4 * U * g.abs())
    return torch.where(empty, 0.0, out / T), torch.where(empty, 0.0, tol / T)


def stored(ref, tol, dtype):
    """The tolerance after rounding to the stored type (and its smallest steps)."""
    return tol + torch.finfo(dtype).eps / 2 * (ref.abs() + tol) * (0 if dtype == torch.float32 else 1) + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2 * U * ref.abs()


@pytest.mark.parametrize("vocab", [1, 2, 8, 9, 33, 513, 4099, 50257])
@pytest.mark.parametrize("dtype", KINDS)
def test_logprobs_gradient_matches(gpu, dev, dtype, vocab):
    for i, (rows, pad, T, n, masked) in enumerate([(1, 0, 1.0, 1, 0.0), (6, 5, 0.6, 7, 0.4), (3, 16, 1.9, 128, 0.9)]):
        z = make(dev, vocab * 3 + i, rows, vocab, dtype, pad, masked=masked)
        if rows == 6:
            z[2] = -math.inf
        tokens = torch.randint(-1, vocab, (rows, n), dtype=torch.int32, device=dev)
        g = torch.randn(rows, n, device=dev)
        h = torch.randn(rows, device=dev)
        f = distribution.token_logprobs(gpu, z, tokens, temperature=T)
        grad = distribution.token_logprobs_backward(gpu, z, tokens, f.stats, f.entropy, g, h, temperature=T)
        ref, tol = logprobs_gradient64(z, tokens, g, h, T)
        within(grad, ref, stored(ref, tol, dtype))
        # one of the two gradients alone
        only_g = distribution.token_logprobs_backward(gpu, z, tokens, f.stats, None, g, temperature=T)
        ref, tol = logprobs_gradient64(z, tokens, g, torch.zeros_like(h), T)
        within(only_g, ref, stored(ref, tol, dtype))
        only_h = distribution.token_logprobs_backward(gpu, z, None, f.stats, f.entropy, None, h, temperature=T)
        ref, tol = logprobs_gradient64(z, tokens, torch.zeros_like(g), h, T)
        within(only_h, ref, stored(ref, tol, dtype))


def test_logprobs_gradient_of_a_repeated_token(gpu, dev):
    z = make(dev, 9, 2, 700, torch.float32)
    tokens = torch.tensor([[5, 5, 5, UNUSED], [699, 0, 699, 0]], dtype=torch.int32, device=dev)
    g = torch.tensor([[1.0, -3.0, 0.5, 9.0], [2.0, 1.0, -2.5, 4.0]], device=dev)
    f = distribution.token_logprobs(gpu, z, tokens)
    grad = distribution.token_logprobs_backward(gpu, z, tokens, f.stats, None, g)
    ref, tol = logprobs_gradient64(z, tokens, g, torch.zeros(2, device=dev), 1.0)
    within(grad, ref, stored(ref, tol, torch.float32))


def test_logprobs_gradient_against_differences(gpu, dev):
    """Central differences of the forward call: step 2^-5, third derivatives of the objective
    below 2 (|g| <= 1, |h| <= 1, T = 1: ln q has third derivatives below 1 and the entropy's stay
    below 6 here), so the difference is off by (2^-10 / 6) * 8 < 1.4e-3; rounding adds
    2 * 2e-6 / 2^-4."""
    V, step = 37, 2.0 ** -5
    z = make(dev, 10, 1, V, torch.float32, scale=1.0)
    tokens = torch.tensor([[3, 20]], dtype=torch.int32, device=dev)
    g = torch.tensor([[1.0, -0.5]], device=dev)
    h = torch.tensor([0.7], device=dev)
    f = distribution.token_logprobs(gpu, z, tokens)
    grad = distribution.token_logprobs_backward(gpu, z, tokens, f.stats, f.entropy, g, h)
    up = z.expand(V, V).clone() + step * torch.eye(V, device=dev)
    down = z.expand(V, V).clone() - step * torch.eye(V, device=dev)

    def objective(x):
        r = distribution.token_logprobs(gpu, x, tokens.expand(V, 2).contiguous())
        return (r.logprob.double() * g.double()).sum(1) + 0.7 * r.entropy.double()

    within(grad[0], (objective(up) - objective(down)) / (2 * step), 2e-3)


# ---- distillation ---------------------------------------------------------------------------------
def teacher_of(dev, seed, z, k, T, noise=1.0, unused=0.0):
    """A teacher's top k tokens, logits and statistics, near the student's logits."""
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    t = z.float() + noise * torch.randn(z.shape, generator=g).to(dev)
    top = torch.topk(t, k, dim=1)
    ids = torch.where(top.values > -math.inf, top.indices, UNUSED).to(torch.int32)
    if unused:
        ids[torch.rand(ids.shape, generator=g).to(dev) < unused] = UNUSED
    m, s, _ = softmax64(t, T)
    return ids.contiguous(), top.values.contiguous(), torch.stack([m, s], 1).float()


def distill64(z, ids, values, stats, weights, T):
    """Loss, statistics, gradient and their tolerances in 64 bits from the definition."""
    R, V = z.shape
    m, s, log_q = softmax64(z, T)
    q = log_q.exp()
    empty = m == -math.inf
    inside = torch.zeros(R, V, dtype=torch.bool)
    a = torch.full((R, V), -math.inf, dtype=torch.float64)
    for r in range(R):
        for i, x in zip(ids[r].tolist(), values[r].double().tolist()):
            if i >= 0 and not inside[r, i]:
                inside[r, i] = True
                a[r, i] = x
    inside, a = inside.to(z.device), a.to(z.device)
    if stats is None:
        norm = torch.logsumexp(a / T, 1)
        log_p = a / T - torch.where(norm == -math.inf, 0.0, norm)[:, None]
        rest = torch.zeros(R, dtype=torch.float64, device=z.device)
        log_rest = torch.full_like(rest, -math.inf)
    else:
        log_p = (a - stats[:, :1].double()) / T - stats[:, 1:].double()
        rest = (1 - log_p.exp().sum(1)).clamp_min(0.0)
        log_rest = torch.logsumexp(torch.where(inside, -math.inf, log_q), 1) + s
    p = log_p.exp()
    q_rest = torch.exp(log_rest - s)
    counts = log_rest - s >= math.log(2.0 ** -126)
    rest = torch.where(counts, rest, 0.0)
    terms = torch.where(p > 0, p * (log_p - log_q), 0.0)
    loss = terms.sum(1) + torch.where(rest > 0, rest * (torch.log(rest) - log_rest + s), 0.0)
    mass = (p.sum(1) + rest)[:, None]
    ratio = torch.where(counts, rest / q_rest, 0.0)[:, None]
    w = torch.where(empty, 0.0, weights.double())[:, None] / T
    grad = w * (q * (mass - torch.where(inside, 0.0, ratio)) - p)
    grad = torch.where(empty[:, None], 0.0, grad)
    tol = sum_tol(V)
    ln_q = torch.where(q > 0, log_q, 0.0)
    rho = 3 * tol + (3 * ln_q.abs() + 3 * s.abs()[:, None] + 10) * 2 * U
    grad_tol = w.abs() * (q * (mass + torch.where(inside, 0.0, ratio)) * rho + 4 * U * p)
    loss_tol = 2 * tol * (1 + mass[:, 0]) + 4 * U * (1 + torch.where(loss.isinf(), 0.0, loss.abs()))
    return loss, torch.stack([m, s, log_rest], 1), grad, loss_tol, grad_tol


def check_distill(gpu, z, ids, values, stats, weights, T):
    loss, saved, grad, loss_tol, grad_tol = distill64(z, ids, values, stats, weights, T)
    tol = sum_tol(z.shape[1])
    forward = distribution.distill(gpu, z, ids, values, teacher_stats=stats, temperature=T)
    assert forward.gradient is None
    step = distribution.distill(gpu, z, ids, values, teacher_stats=stats, weights=weights, temperature=T, gradient=True)
    for got in (forward, step):
        within(got.loss, loss, loss_tol)
        within(got.stats[:, 0], saved[:, 0], 0.0)
        within(got.stats[:, 1], saved[:, 1], tol + 2 * U * saved[:, 1].abs())
        within(got.stats[:, 2], saved[:, 2],
               tol + 4 * U * torch.where(saved[:, 2].isinf(), 0.0, saved[:, 2].abs()))
    within(step.gradient, grad, stored(grad, grad_tol, z.dtype))
    back = distribution.distill_backward(gpu, z, ids, values, forward.stats, weights, teacher_stats=stats,
                                         temperature=T)
    within(back, grad, stored(grad, grad_tol, z.dtype))
    return step


@pytest.mark.parametrize("vocab", [1, 2, 7, 9, 33, 512, 4099, 20011])
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_matches(gpu, dev, tail, dtype, vocab):
    for i, (rows, pad, T, k, masked) in enumerate([(1, 0, 1.0, 1, 0.0), (5, 3, 2.0, 20, 0.3), (3, 8, 0.7, 128, 0.0)]):
        z = make(dev, vocab * 5 + i, rows, vocab, dtype, pad, masked=masked)
        ids, values, stats = teacher_of(dev, i, z, min(k, vocab), T, unused=0.1)
        weights = torch.rand(rows, device=dev) + 0.25
        check_distill(gpu, z, ids, values, stats if tail else None, weights, T)


@pytest.mark.parametrize("rows", [1, 4, 20, 40, 160, 320])
def test_distill_row_counts(gpu, dev, rows):
    for vocab, dtype in ((5003, torch.float32), (40001, torch.float16)):
        z = make(dev, rows, rows, vocab, dtype)
        ids, values, stats = teacher_of(dev, rows, z, 16, 1.0)
        check_distill(gpu, z, ids, values, stats, torch.ones(rows, device=dev), 1.0)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", KINDS)
def test_distill_special_rows(gpu, dev, dtype, tail):
    V, k = 900, 6
    z = make(dev, 21, 9, V, dtype)
    ids, values, stats = teacher_of(dev, 22, z, k, 1.0)
    ids[0] = UNUSED                                  # a padded row
    z[1] = -math.inf                                 # a student without any token
    z[2, ids[2, 0].item()] = -math.inf               # a teacher's token that the student forbids: loss inf
    ids[3, 1] = ids[3, 0]                            # listed twice: counts once, at its first slot
    ids[3, 4] = ids[3, 2]
    values[4, 2] = -math.inf                         # a teacher's token without mass
    z[5] = -math.inf
    z[5, ids[5].long()] = 1.0                        # the student has no mass outside the list
    z[6] = torch.finfo(dtype).min
    z[6, ids[6, 0].item()] = 2.0                     # masked with the type's lowest value
    values[7] = -math.inf                            # a teacher without mass
    check_distill(gpu, z, ids, values, stats if tail else None, torch.linspace(0.5, 2, 9, device=dev), 1.0)


def test_distill_confident_student_keeps_its_rest(gpu, dev):
    """The student's mass outside the list is summed by itself, so it holds where it is 1e-12
    of the whole (a difference of sums would leave nothing of it)."""
    V = 3001
    z = make(dev, 30, 4, V, torch.float32, scale=1.0).clamp_(-4, 4)
    ids = torch.tensor([[5, 77]] * 4, dtype=torch.int32, device=dev)
    z[:, 5] = 38.0
    z[:, 77] = 37.0
    values = torch.tensor([[2.0, 1.0]] * 4, device=dev)
    stats = torch.tensor([[2.0, 1.0]] * 4, device=dev)
    step = check_distill(gpu, z, ids, values, stats, torch.ones(4, device=dev), 1.0)
    assert bool((step.stats[:, 2] < -25).all()) and bool(step.loss.isfinite().all())


def test_distill_padded_positions(gpu, dev):
    """Positions where teacher and student hold no token, as token_logprobs hands them on."""
    teacher, student = make(dev, 27, 3, 600, torch.bfloat16), make(dev, 28, 3, 600, torch.bfloat16)
    teacher[1] = -math.inf
    student[1] = -math.inf
    teacher[2] = -math.inf
    top = distribution.token_logprobs(gpu, teacher, alternatives=8)
    for stats in (None, top.stats):
        got = distribution.distill(gpu, student, top.top_ids, top.top_logits, teacher_stats=stats, gradient=True)
        assert got.loss[1:].cpu().tolist() == [0.0, 0.0] and float(got.loss[0]) > 0
        assert not bool(got.gradient[1:].any()) and bool(got.gradient[0].any())
        back = distribution.distill_backward(gpu, student, top.top_ids, top.top_logits, got.stats,
                                             torch.ones(3, device=dev), teacher_stats=stats)
        assert torch.equal(back, got.gradient)


@pytest.mark.parametrize("dtype, vocab", [(torch.float32, 420011), (torch.bfloat16, 850001)])
def test_distill_of_very_long_rows(gpu, dev, dtype, vocab):
    """Rows beyond what a cluster holds in shared memory are read again for the gradient."""
    z = make(dev, 29, 2, vocab, dtype, pad=3)
    ids, values, stats = teacher_of(dev, 30, z, 128, 1.0, unused=0.05)
    for t in (None, stats):
        check_distill(gpu, z, ids, values, t, torch.ones(2, device=dev), 1.0)
    ids[1, 7] = ids[1, 9]
    check_distill(gpu, z, ids, values, stats, torch.ones(2, device=dev), 1.0)


def test_distill_bad_rows_are_nan(gpu, dev):
    z = make(dev, 23, 5, 300, torch.float32)
    ids, values, stats = teacher_of(dev, 24, z, 5, 1.0)
    z[0, 17] = math.nan
    z[1, 299] = math.inf
    ids[2, 3] = 300
    values[3, 1] = math.nan
    for t in (None, stats):
        got = distribution.distill(gpu, z, ids, values, teacher_stats=t, gradient=True)
        assert got.loss.isnan().cpu().tolist() == [True, True, True, True, False]
        assert got.gradient.isnan().any(1).cpu().tolist() == [True, True, True, True, False]
        back = distribution.distill_backward(gpu, z, ids, values, got.stats, torch.ones(5, device=dev),
                                             teacher_stats=t)
        assert back.isnan().any(1).cpu().tolist() == [True, True, True, True, False]


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(gpu, dev, tail):
    """Central differences with step 2^-5: the loss is P lse(z) minus linear terms, and with the
    tail minus p_r lse of the rest, so third derivatives stay below 2 * 1; off by 2^-10 / 6 * 2
    < 4e-4, and rounding adds 4e-6 / 2^-4."""
    V, step = 41, 2.0 ** -5
    z = make(dev, 25, 1, V, torch.float32, scale=1.0)
    ids, values, stats = teacher_of(dev, 26, z, 6, 1.0)
    stats = stats if tail else None
    got = distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)
    many = [t.expand(V, *t.shape[1:]).contiguous() if t is not None else None for t in (ids, values, stats)]
    eye = step * torch.eye(V, device=dev)
    up, down = (distribution.distill(gpu, z + s * eye, many[0], many[1], teacher_stats=many[2]).loss.double()
                for s in (1, -1))
    within(got.gradient[0], (up - down) / (2 * step), 6e-4)


# ---- memory, streams, graphs -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", KINDS)
def test_gradients_in_place_and_elsewhere(gpu, dev, dtype):
    """Written over the logits, into a strided view, at another alignment: the same bits, and
    nothing outside the rows changes."""
    R, V = 11, 5001
    z = make(dev, 31, R, V, dtype, pad=7)
    ids, values, stats = teacher_of(dev, 32, z, 9, 1.0)
    weights = torch.rand(R, device=dev)
    tokens = ids[:, :3].contiguous()
    f = distribution.token_logprobs(gpu, z, tokens)
    g, h = torch.randn(R, 3, device=dev), torch.randn(R, device=dev)
    calls = {
        "step": lambda x, out: distribution.distill(gpu, x, ids, values, teacher_stats=stats, weights=weights,
                                                    gradient=True, out=(None, None, out)).gradient,
        "back": lambda x, out: distribution.distill_backward(
            gpu, x, ids, values, distribution.distill(gpu, x, ids, values, teacher_stats=stats).stats, weights,
            teacher_stats=stats, out=out),
        "logprobs": lambda x, out: distribution.token_logprobs_backward(gpu, x, tokens, f.stats, f.entropy, g, h, out=out),
    }
    for name, call in calls.items():
        plain = call(z, None)
        assert plain.is_contiguous()
        for shift in (0, 1, 3, 8):
            buffer = torch.full((R, V + 40), 5.0, dtype=dtype, device=dev)
            call(z, buffer[:, shift:shift + V])
            assert torch.equal(buffer[:, shift:shift + V], plain), name
            assert bool((buffer[:, :shift] == 5).all()) and bool((buffer[:, shift + V:] == 5).all())
        buffer = torch.full((R, V + 7), 7.0, dtype=dtype, device=dev)
        mine = buffer[:, :V]
        mine.copy_(z)
        assert call(mine, mine) is mine or True
        assert torch.equal(mine, plain), name
        assert bool((buffer[:, V:] == 7).all())


def test_outputs_stay_inside_their_rows(gpu, dev):
    """Buffers longer than the call's rows keep what lies behind."""
    R, V, k = 5, 2003, 9
    z = make(dev, 33, R, V, torch.bfloat16)
    tokens = torch.zeros(R, 2, dtype=torch.int32, device=dev)
    big = [torch.full((R + 3, *s), 3, dtype=d, device=dev)
           for s, d in (((2,), torch.float32), ((), torch.float32), ((2,), torch.float32), ((k,), torch.int32),
                        ((k,), torch.float32), ((k,), torch.float32))]
    got = distribution.token_logprobs(gpu, z, tokens, alternatives=k, out=[b[:R] for b in big])
    plain = distribution.token_logprobs(gpu, z, tokens, alternatives=k)
    for a, b, c in zip(got, plain, big):
        assert torch.equal(a, b) and bool((c[R:] == 3).all())


def test_single_outputs(gpu, dev):
    z = make(dev, 34, 3, 777, torch.float16)
    tokens = torch.zeros(3, 1, dtype=torch.int32, device=dev)
    full = distribution.token_logprobs(gpu, z, tokens, alternatives=4)
    for i in range(6):
        out = [torch.empty_like(t) if j == i else None for j, t in enumerate(full)]
        got = distribution.token_logprobs(gpu, z, tokens, alternatives=4, out=out)
        assert torch.equal(got[i], full[i])


def test_no_rows(gpu, dev):
    z = torch.empty(0, 33, device=dev)
    got = distribution.token_logprobs(gpu, z, torch.empty(0, 2, dtype=torch.int32, device=dev), alternatives=3)
    assert got.logprob.shape == (0, 2) and got.top_ids.shape == (0, 3)
    d = distribution.distill(gpu, z, torch.empty(0, 2, dtype=torch.int32, device=dev), torch.empty(0, 2, device=dev),
                             gradient=True)
    assert d.loss.shape == (0,) and d.gradient.shape == (0, 33)


def test_results_repeat_bit_for_bit(gpu, dev):
    for rows, vocab, dtype in ((3, 151936, torch.float32), (200, 30011, torch.bfloat16)):
        z = make(dev, 35, rows, vocab, dtype)
        tokens = torch.randint(0, vocab, (rows, 4), dtype=torch.int32, device=dev)
        ids, values, stats = teacher_of(dev, 36, z, 50, 1.0)
        first = [*distribution.token_logprobs(gpu, z, tokens, alternatives=50),
                 *distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)]
        for _ in range(3):
            again = [*distribution.token_logprobs(gpu, z, tokens, alternatives=50),
                     *distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)]
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_ordered_with_the_callers_stream(gpu, dev):
    """Inputs written and outputs read on another stream, without a synchronisation between."""
    R, V = 64, 40009
    side = torch.cuda.Stream(dev)
    base = make(dev, 37, R, V, torch.float32)
    ids, values, _ = teacher_of(dev, 38, base, 8, 1.0)
    want = distribution.distill(gpu, base * 0.5, ids, values, gradient=True)
    torch.cuda.synchronize(dev)
    with torch.cuda.stream(side):
        for _ in range(5):
            work = torch.randn(4096, 4096, device=dev)
            for _ in range(4):
                work = work @ work * 1e-3
            z = torch.zeros_like(base)
            z.copy_(base)
            z.mul_(0.5)
            got = distribution.distill(gpu, z, ids, values, gradient=True)
            total = got.gradient.double().abs().sum()
            z.zero_()
        assert torch.equal(total, want.gradient.double().abs().sum())
        assert torch.equal(got.loss, want.loss)
    side.synchronize()


def test_captured_and_replayed(gpu, dev):
    """Two graphs of the same calls, replayed in turn on new inputs, and eager calls between."""
    R, V = 6, 9001
    sources = [make(dev, 40 + i, R, V, torch.bfloat16) for i in range(3)]
    tokens = torch.randint(0, V, (R, 2), dtype=torch.int32, device=dev)
    ids, values, stats = teacher_of(dev, 44, sources[0], 12, 1.0)
    g = torch.ones(R, 2, device=dev)

    def calls(z):
        a = distribution.token_logprobs(gpu, z, tokens, alternatives=12)
        b = distribution.token_logprobs_backward(gpu, z, tokens, a.stats, a.entropy, g, g[:, 0].contiguous())
        c = distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)
        d = distribution.distill_backward(gpu, z, ids, values, c.stats, g[:, 1].contiguous(), teacher_stats=stats)
        return [*a, b, *c, d]

    want = [calls(z) for z in sources]
    graphs = []
    for _ in range(2):
        z = sources[0].clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph):
            out = calls(z)
        graphs.append((graph, z, out))
    for i, source in enumerate(sources):
        for graph, z, _ in graphs:
            z.copy_(source)
            graph.replay()
        eager = calls(sources[(i + 1) % 3])
        torch.cuda.synchronize(dev)
        for _, _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3]))


def test_two_contexts_at_once(gpu, dev):
    """Calls of two contexts share nothing: interleaved, they give what each gives alone."""
    other = lsx.Gpu(gpu.device)
    a, b = make(dev, 50, 32, 60013, torch.float32), make(dev, 51, 32, 60013, torch.float16)
    want = [distribution.token_logprobs(gpu, x, alternatives=30) for x in (a, b)]
    torch.cuda.synchronize(dev)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for _ in range(4):
        for g, s, x in ((gpu, streams[0], a), (other, streams[1], b)):
            with torch.cuda.stream(s):
                got.append(distribution.token_logprobs(g, x, alternatives=30))
    torch.cuda.synchronize(dev)
    for i, r in enumerate(got):
        for x, y in zip(r, want[i % 2]):
            assert (x is None and y is None) or torch.equal(x, y)


def test_long_offsets(gpu, dev):
    """Rows whose offsets pass 2^32 bytes and 2^31 elements."""
    V, stride = 1009, 1 << 26
    buffer = torch.empty(34 * stride, dtype=torch.bfloat16, device=dev)  # 4.25 GiB of addresses
    z = buffer.as_strided((34, V), (stride, 1))
    z.copy_(make(dev, 52, 34, V, torch.bfloat16))
    tokens = torch.zeros(34, 1, dtype=torch.int32, device=dev)
    check_logprobs(gpu, z, tokens, 5, 1.0)
    ids, values, stats = teacher_of(dev, 53, z, 5, 1.0)
    check_distill(gpu, z, ids, values, stats, torch.ones(34, device=dev), 1.0)
    distribution.distill(gpu, z, ids, values, gradient=True, out=(None, None, z))
    assert bool(z[33].float().abs().max() < 1)


def test_python_refusals(gpu, dev):
    z = make(dev, 54, 4, 50, torch.float32)
    ids, values, stats = teacher_of(dev, 55, z, 5, 1.0)
    bad = [
        lambda: distribution.token_logprobs(gpu, z.t()),
        lambda: distribution.token_logprobs(gpu, z[:1].expand(4, 50)),
        lambda: distribution.token_logprobs(gpu, z, ids.long()),
        lambda: distribution.token_logprobs(gpu, z, ids[:3]),
        lambda: distribution.token_logprobs(gpu, z, ids.t().contiguous().t()),
        lambda: distribution.token_logprobs(gpu, z, alternatives=51),
        lambda: distribution.token_logprobs(gpu, z, alternatives=-1),
        lambda: distribution.token_logprobs(gpu, z, ids.cpu()),
        lambda: distribution.token_logprobs(gpu, z, out=[None] * 5),
        lambda: distribution.token_logprobs_backward(gpu, z, ids, stats[:, :1], None, values),
        lambda: distribution.token_logprobs_backward(gpu, z, ids, stats, None, values[:, :2]),
        lambda: distribution.token_logprobs_backward(gpu, z, ids, stats, None, values, stats[:, 0].contiguous()),
        lambda: distribution.token_logprobs_backward(gpu, z, ids, stats, None, values, out=z.half()),
        lambda: distribution.distill(gpu, z, ids, values.half()),
        lambda: distribution.distill(gpu, z, ids, values, weights=stats[:, 0].contiguous()),
        lambda: distribution.distill(gpu, z, ids, values, out=(None, None, z)),
        lambda: distribution.distill(gpu, z, ids[:, :0], values[:, :0]),
        lambda: distribution.distill_backward(gpu, z, ids, values, stats, stats[:, 0].contiguous()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(LsxError, match="temperature"):
        distribution.token_logprobs(gpu, z, temperature=0.0)
    with pytest.raises(LsxError, match="overlaps"):
        both = torch.zeros(4, 60, device=dev)
        distribution.distill(gpu, both[:, :50], ids, values, gradient=True, out=(None, None, both[:, 10:]))


# ---- together -----------------------------------------------------------------------------------------
def test_teacher_to_student_gradient(gpu, dev):
    """The operators as they are used together: a teacher's alternatives and statistics feed the
    distillation of a student, whose gradient step brings the loss down to first order."""
    R, V, k, T = 20, 12007, 32, 1.5
    teacher, student = make(dev, 60, R, V, torch.bfloat16), make(dev, 61, R, V, torch.float32)
    top = distribution.token_logprobs(gpu, teacher, alternatives=k, temperature=T)
    step = distribution.distill(gpu, student, top.top_ids, top.top_logits, teacher_stats=top.stats, temperature=T,
                                gradient=True)
    loss, _, grad, loss_tol, grad_tol = distill64(student, top.top_ids, top.top_logits, top.stats,
                                                  torch.ones(R, device=dev), T)
    within(step.loss, loss, loss_tol)
    within(step.gradient, grad, stored(grad, grad_tol, torch.float32))
    # the listed log probabilities are the teacher's own: their sum and the rest make 1
    p = top.top_logprobs.double().exp().sum(1)
    assert bool((p <= 1 + 1e-5).all())
    # a student equal to the teacher has nothing to learn: the loss is 0 up to the sums' rounding
    same = distribution.distill(gpu, teacher, top.top_ids, top.top_logits, teacher_stats=top.stats, temperature=T,
                                gradient=True)
    assert float(same.loss.abs().max()) <= 6 * sum_tol(V)
    assert lib.lsx_last_error() is not None and np.isfinite(step.loss.cpu().numpy()).all()


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("vocab", [9, 700, 50257])
def test_peaked_rows_keep_the_small_rest(gpu, dev, dtype, vocab):
    """Where one token holds all but a small rest r, log q of that token and the statistics are
    ln(1 + r) and the entropy is about r ln(1/r): they hold to a relative tolerance, which a sum
    of 1 + r in f32 would not give."""
    z = make(dev, 70, 12, vocab, dtype, scale=1.0).clamp_(-4, 4)
    at = torch.tensor([0, vocab - 1, vocab // 2, 7, 8, vocab // 3] * 2, device=dev)
    z[torch.arange(12), at] = torch.tensor([14.0, 18, 20, 22, 26, 30] * 2, device=dev).to(dtype)
    tokens = at.to(torch.int32)[:, None].contiguous()
    got = distribution.token_logprobs(gpu, z, tokens, alternatives=min(vocab, 5))
    rest = torch.where(torch.arange(vocab, device=dev)[None, :] == at[:, None], -math.inf, z.double())
    top = z.double().amax(1)
    r = torch.exp(rest - top[:, None]).sum(1)
    tol = sum_tol(vocab) + 40 * 3 * U  # |y| reaches 40 here
    log_sum = torch.log1p(r)
    within(got.stats[:, 1], log_sum, tol * log_sum)
    within(got.logprob[:, 0], -log_sum, tol * log_sum)
    y = torch.where(rest == -math.inf, 0.0, rest - top[:, None])
    entropy = log_sum - (torch.exp(rest - top[:, None]) * y).sum(1) / (1 + r)
    within(got.entropy, entropy, 2 * tol * entropy)


def test_alternatives_at_neighbouring_values(gpu, dev):
    """Rows of two neighbouring f32 values: the value that separates them is itself a logit, and
    its ties have to stay candidates; with fewer, as many and more of the larger one than
    alternatives."""
    low = torch.nextafter(torch.tensor(2.0), torch.tensor(0.0)).item()
    for vocab in (4099, 1031, 40000):
        for larger in (5, 47, 50, 100, 127, 200, 600):
            z = torch.full((3, vocab), low, device=dev)
            g = torch.Generator().manual_seed(larger)
            for r in range(3):
                z[r, torch.randperm(vocab, generator=g)[:larger].to(dev)] = 2.0
            z[2, ::3] = -math.inf
            for k in (26, 48, 100, 128):
                got = distribution.token_logprobs(gpu, z, alternatives=k)
                assert torch.equal(got.top_ids.long(), order64(z, k)), (vocab, larger, k)


@pytest.mark.parametrize("dtype", KINDS)
def test_alternatives_of_coarse_logits(gpu, dev, dtype):
    """Logits on a coarse grid tie everywhere; masks leave few, some or most of them."""
    g = torch.Generator().manual_seed(71)
    for vocab in (97, 257, 1025, 5000, 33000):
        z = torch.randint(-6, 7, (24, vocab), generator=g).to(dtype)
        for r in range(24):
            z[r, torch.rand(vocab, generator=g) < [0.0, 0.5, 0.99][r % 3]] = -math.inf
        z = z.to(dev)
        for k in (1, 7, 20, 25, 30, 60, min(vocab, 128)):
            got = distribution.token_logprobs(gpu, z, alternatives=k)
            assert torch.equal(got.top_ids.long(), order64(z, k)), (vocab, k)


def test_distill_bad_slot_in_an_empty_row(gpu, dev):
    z = torch.full((2, 40), -math.inf, device=dev)
    ids = torch.tensor([[1, 40], [1, 2]], dtype=torch.int32, device=dev)
    values = torch.zeros(2, 2, device=dev)
    got = distribution.distill(gpu, z, ids, values, gradient=True)
    back = distribution.distill_backward(gpu, z, ids, values, got.stats, torch.ones(2, device=dev))
    for grad in (got.gradient, back):
        assert bool(grad[0].isnan().all()) and not bool(grad[1].any())
    assert bool(got.loss[0].isnan()) and float(got.loss[1]) == math.inf


@pytest.mark.parametrize("rows", [741, 888, 889, 1036, 1037])
@pytest.mark.parametrize("dtype", KINDS)
def test_logprobs_of_a_full_wave(gpu, dev, dtype, rows):
    """Numbers of rows around what a GPU of 148 SMs holds at once, masked in different measure,
    with rows of one token, of none and of ties."""
    for vocab, k in ((4102, 3), (9001, 128)):
        z = make(dev, rows + k, rows, vocab, dtype, 1, masked=0.9)
        z[::7] = -math.inf
        z[::14, 11] = 1.5
        z[1::7, ::2] = 3.0
        z[2::7] = torch.linspace(-9, 9, vocab).to(dtype).to(dev)
        z[3::7] = torch.finfo(dtype).min
        tokens = torch.randint(-1, vocab, (rows, 2), dtype=torch.int32, device=dev)
        check_logprobs(gpu, z, tokens, k, 0.9)
        z[5, 100] = math.nan
        got = distribution.token_logprobs(gpu, z, tokens, alternatives=k)
        assert bool(got.entropy[5].isnan()) and not bool(got.entropy[6:].isnan().any())
        assert torch.equal(got.top_ids.long(), order64(z, k))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", KINDS)
def test_distill_step_of_long_rows(gpu, dev, dtype, tail):
    """Slices of one to many chunks a thread, in numbers of rows that take one to eight blocks
    each; results repeat bit for bit, in place too."""
    n = 16 // torch.empty(0, dtype=dtype).element_size()
    for vectors, rows in ((1024, 600), (1025, 33), (2303, 600), (2305, 593), (3500, 593), (9999, 160), (20001, 3),
                          (20003, 170)):
        vocab = vectors * n + vectors % 3
        z = make(dev, vectors, rows, vocab, dtype, n if vectors % 2 else 1, masked=0.2)
        ids, values, stats = teacher_of(dev, rows, z, 128 if vectors % 2 else 20, 1.4, unused=0.1)
        if not tail:
            stats = None
        weights = torch.rand(rows, device=dev) + 0.25
        got = check_distill(gpu, z, ids, values, stats, weights, 1.4)
        again = distribution.distill(gpu, z, ids, values, teacher_stats=stats, weights=weights, temperature=1.4,
                                     gradient=True, out=(torch.empty_like(got.loss), torch.empty_like(got.stats), z))
        assert again.gradient.data_ptr() == z.data_ptr()
        assert torch.equal(got.loss, again.loss) and torch.equal(got.stats, again.stats)
        assert torch.equal(got.gradient, again.gradient)


def test_two_captured_steps_of_long_rows_at_once(gpu, dev):
    """Two graphs of steps over long rows, replayed on two streams at the same time, give what each
    gives alone."""
    graphs, wanted, held = [], [], []
    for i, (rows, vocab, dtype) in enumerate([(250, 40003, torch.bfloat16), (90, 70001, torch.float32)]):
        z = make(dev, i, rows, vocab, dtype)
        ids, values, stats = teacher_of(dev, i, z, 24, 1.0)
        alone = distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)
        out = (torch.empty_like(alone.loss), torch.empty_like(alone.stats), torch.empty_like(alone.gradient))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True, out=out)
        graphs.append((graph, torch.cuda.Stream(dev)))
        wanted.append(alone)
        held.append((z, ids, values, stats, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for alone, (*_, out) in zip(wanted, held):
        for a, b in zip((alone.loss, alone.stats, alone.gradient), out):
            assert torch.equal(a, b)
