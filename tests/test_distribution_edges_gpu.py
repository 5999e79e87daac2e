"""Edges of the operators on rows of logits (laplacesscissors_b200/distribution.py): a student
whose share of the tokens outside the teacher's list is next to nothing, and logits whose
difference f32 does not hold.  The references compute from the definitions in 64 bits, in
logarithms where 64 bits would leave nothing of a share."""
import math

import pytest
import torch

from laplacesscissors_b200 import distribution
from test_distribution_gpu import KINDS, U, check_distill, dev, make, stored, sum_tol, within  # noqa: F401

pytestmark = pytest.mark.gpu

SHARES = [1e-30, 1e-37, 1e-39, 1e-80, 1e-300]


def lost_bucket(dev, seed, vocab, dtype, T, shares):
    """A student with one likely token and the others about `shares` of the mass together, and a
    teacher with p = 0.5 for that token, 0.1 for another listed one and 0.4 for the rest."""
    g = torch.Generator().manual_seed(seed)
    R = len(shares)
    z = torch.randn(R, vocab, generator=g).clamp_(-2, 2) * T
    z[:, 5] = T * torch.tensor([math.log(vocab / s) for s in shares])
    ids = torch.tensor([[3, 5, -1]] * R, dtype=torch.int32, device=dev)
    values = torch.tensor([[2.0 - T * math.log(5), 2.0, 7.0]] * R, device=dev)
    stats = torch.tensor([[2.0, math.log(2)]] * R, device=dev)
    return z.to(dtype).to(dev), ids, values, stats


def distill_in_logs(z, ids, values, stats, weights, T):
    """Loss, gradient, ln q, ln q_r and the teacher's p, by the definition."""
    log_q = torch.log_softmax(z.double() / T, 1)
    inside = torch.zeros_like(log_q, dtype=torch.bool)
    log_p = torch.full_like(log_q, -math.inf)
    for r in range(z.shape[0]):
        for i, x in zip(ids[r].tolist(), values[r].double().tolist()):
            if i >= 0:
                inside[r, i] = True
                log_p[r, i] = (x - float(stats[r, 0])) / T - float(stats[r, 1])
    p = log_p.exp()
    p_rest = 1 - p.sum(1, keepdim=True)
    log_rest = torch.logsumexp(torch.where(inside, -math.inf, log_q), 1, keepdim=True)
    loss = torch.where(inside, p * (log_p - log_q), 0.0).sum(1) + (p_rest * (p_rest.log() - log_rest))[:, 0]
    P = p.sum(1, keepdim=True) + p_rest
    w = weights.double()[:, None] / T
    grad = w * (log_q.exp() * P - torch.where(inside, p, p_rest * (log_q - log_rest).exp()))
    return loss, grad, log_q, log_rest, p, p_rest, inside, w


@pytest.mark.parametrize("T", [1.0, 0.1])
@pytest.mark.parametrize("vocab", [8, 900, 2500, 20011, 70001])
@pytest.mark.parametrize("dtype", KINDS)
def test_small_share_of_the_other_tokens(gpu, dev, dtype, vocab, T):
    """The other tokens stay one outcome of the loss however little the student gives them, down to
    what 64 bits hold.

    Tolerances, with sum_tol for a sum of exponentials.  Loss: its logarithms are taken in 64 bits of
    sums in f32, and it is stored in f32.  Log of the others' mass: a difference, 1/T, their product
    and a sum, half a step each, and logf's own 2.  A gradient's exponent (z - m) L - log_rest log2e:
    half a step of the difference, of L, and of log_rest's four, of the constant and of two products,
    so 2 u of ln q_i and 8 u of ln q_r at most; the exponential is off by 4 u, the factors by a few."""
    z, ids, values, stats = lost_bucket(dev, vocab, vocab, dtype, T, SHARES)
    weights = torch.linspace(0.5, 2, len(SHARES), device=dev)
    loss, grad, log_q, log_rest, p, p_rest, inside, w = distill_in_logs(z, ids, values, stats, weights, T)
    assert bool((loss > 0).all()) and float(log_rest[-1]) < -680
    tol = sum_tol(vocab)
    rho = 2 * tol + (4 * log_q.abs() + 8 * log_rest.abs() + 20) * U
    parts = log_q.exp() * (p + p_rest).sum(1, keepdim=True) + torch.where(inside, 0.0, p_rest * (log_q - log_rest).exp())
    grad_tol = w * (parts * rho + 4 * U * p)
    forward = distribution.distill(gpu, z, ids, values, teacher_stats=stats, temperature=T)
    step = distribution.distill(gpu, z, ids, values, teacher_stats=stats, weights=weights, temperature=T, gradient=True)
    back = distribution.distill_backward(gpu, z, ids, values, forward.stats, weights, teacher_stats=stats,
                                         temperature=T)
    s = -log_q.amax(1, keepdim=True)  # the likely token's: its logit is the maximum
    for got in (forward, step):
        within(got.loss, loss, 4 * tol + 4 * U * (1 + loss))
        within(got.stats[:, 2:], log_rest + s, tol + 6 * U * log_rest.abs())
    within(step.gradient, grad, stored(grad, grad_tol, dtype))
    within(back, grad, stored(grad, grad_tol, dtype))


@pytest.mark.parametrize("dtype", KINDS)
def test_share_that_64_bits_do_not_hold(gpu, dev, dtype):
    """Below 2^-1074, where q_r is 0 in 64 bits, the others are no outcome: what masks of -inf and of
    a type's lowest value leave."""
    z, ids, values, stats = lost_bucket(dev, 1, 3000, dtype, 1.0, [1e-300] * 3)
    z[:, 5] = torch.tensor([800.0, 2000.0, 30000.0]).to(dtype)
    step = check_distill(gpu, z, ids, values, stats, torch.ones(3, device=dev), 1.0)
    others = torch.ones(3000, dtype=torch.bool, device=dev)
    others[[3, 5]] = False
    assert not bool(step.gradient[:, others].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [40, 4099, 70001])
def test_differences_that_f32_does_not_hold(gpu, dev, dtype, vocab):
    """The type's lowest value next to its largest: the difference passes f32's range, what it
    gives at a temperature above 2 does not.  Half a step for each of two halved logits'
    difference, 1/T and the product, and the statistics' 4."""
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).min
    z = torch.full((3, vocab), low, dtype=dtype, device=dev)
    z[:, 7] = top
    z[1, 9] = top / 2
    z[2] = top
    z[2, 11] = low
    tokens = torch.tensor([[7, 9, 11, 0]] * 3, dtype=torch.int32, device=dev)
    ids = torch.tensor([[7, 30]] * 3, dtype=torch.int32, device=dev)
    values = torch.zeros(3, 2, device=dev)
    for T in (2.5, 4.0, 1000.0, 1e6):
        d = z.double() / T
        m, log_sum = d.amax(1, keepdim=True), torch.logsumexp(d - d.amax(1, keepdim=True), 1, keepdim=True)
        log_q = d - m - log_sum
        assert bool(log_q.isfinite().all())
        got = distribution.token_logprobs(gpu, z, tokens, alternatives=20, temperature=T)
        want = log_q.gather(1, tokens.long())
        within(got.logprob, want, 4 * U * want.abs() + sum_tol(vocab))
        want = log_q.gather(1, got.top_ids.long())
        within(got.top_logprobs, want, 4 * U * want.abs() + sum_tol(vocab))
        outside = d - m
        outside[:, [7, 30]] = -math.inf
        want = torch.logsumexp(outside, 1)
        stats = distribution.distill(gpu, z, ids, values, teacher_stats=torch.zeros(3, 2, device=dev),
                                     temperature=T).stats
        within(stats[:, 2], want, 6 * U * want.abs() + sum_tol(vocab))


@pytest.mark.parametrize("vocab", [1, 8, 900, 2500, 20011, 70001])
@pytest.mark.parametrize("dtype", KINDS)
def test_unused_lists_ask_for_nothing(gpu, dev, dtype, vocab):
    """A row that lists no token has p_r = q_r = 1: loss and gradient are 0, not next to it; so
    has one whose listed tokens neither teacher nor student holds."""
    z = make(dev, vocab, 6, vocab, dtype, 3, masked=0.2 if vocab > 1 else 0.0)
    ids = torch.full((6, 7), -1, dtype=torch.int32, device=dev)
    values = torch.randn(6, 7, generator=torch.Generator().manual_seed(vocab)).to(dev)
    if vocab > 1:
        ids[3:, 2] = 1
        z[3:, 1] = values[3:, 2] = -math.inf
    stats = torch.tensor([[1.0, 2.0]] * 6, device=dev)
    weights = torch.linspace(0.5, 2, 6, device=dev)
    for T in (1.0, 0.3, 2.0):
        for teacher in (None, stats):
            step = distribution.distill(gpu, z, ids, values, teacher_stats=teacher, weights=weights, temperature=T,
                                        gradient=True)
            back = distribution.distill_backward(gpu, z, ids, values, step.stats, weights, teacher_stats=teacher,
                                                 temperature=T)
            assert not bool(step.loss.any()) and not bool(step.gradient.any()) and not bool(back.any())


def test_unused_lists_of_rows_of_every_spread(gpu, dev):
    """Rows from nearly uniform to nearly one token: the logarithms of q_r's two sums are one."""
    R = 4000
    ids = torch.full((R, 3), -1, dtype=torch.int32, device=dev)
    none, stats, ones = torch.zeros(R, 3, device=dev), torch.zeros(R, 2, device=dev), torch.ones(R, device=dev)
    for vocab in (61, 700, 2999):
        g = torch.Generator().manual_seed(vocab)
        z = (torch.randn(R, vocab, generator=g) * torch.rand(R, 1, generator=g) * 12).to(dev)
        step = distribution.distill(gpu, z, ids, none, teacher_stats=stats, gradient=True)
        back = distribution.distill_backward(gpu, z, ids, none, step.stats, ones, teacher_stats=stats)
        assert torch.equal(step.stats[:, 1], step.stats[:, 2])
        assert not bool(step.loss.any()) and not bool(step.gradient.any()) and not bool(back.any())
