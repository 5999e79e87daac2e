"""Distributions at teacher-forced positions (lsx_model_distribution_batch,
lsx_model_divergence_batch, diagnosis.readout_divergence) on the committed tiny
checkpoint: against the formulas in 64 bits on the logits that lsx_model_score_batch
returns for the same cases (the same kernels make them, so they are equal), with and
without a readout edit.

Tolerances: the vocabulary of 512 is summed in f32 with 2^-24 per step, at most 512/128
steps in a row and a tree, exponentials off by 2^-22 and their arguments (below 20 powers
of two in weight) by 3 * 2^-24 each: below 2^-24 * (4 + 80) = 5e-6 relative of the sum."""
import numpy as np
import pytest

import laplacesscissors_b200 as lsx
from conftest import GOLDEN
from laplacesscissors_b200 import DeviceRotation, LsxError, ReadoutRotation, diagnosis

pytestmark = pytest.mark.gpu

SUM = 84 * 2.0 ** -24
CASES = ([[1, 2, 3], [7, 300, 5], [9, 9, 9], [400, 2, 17]], [[5, 9, 200, 7], [11, 400, 2, 1], [3, 3, 3, 3], [8, 1, 0, 511]])


@pytest.fixture(scope="module")
def model(gpu):
    return lsx.Model.load(GOLDEN / "tiny_qwen3", gpu, 32)


@pytest.fixture(scope="module")
def edit(gpu, model, golden_tiny):
    spec = ReadoutRotation(golden_tiny["plane_u"], golden_tiny["plane_v"], float(golden_tiny["plane_tangent"]))
    return DeviceRotation.upload(gpu, spec, model.hidden_size)


def log_softmax(z, T):
    z = z.astype(np.float64) / T
    m = z.max(-1, keepdims=True)
    return z - m - np.log(np.exp(z - m).sum(-1, keepdims=True))


@pytest.mark.parametrize("edited", [False, True])
@pytest.mark.parametrize("temperature, k", [(1.0, 5), (0.5, 128), (2.0, 0)])
def test_distribution_matches_the_logits(model, edit, edited, temperature, k):
    rotation = edit if edited else None
    nll, amax, _, logits = model.score_batch(*CASES, rotation, logits=True)
    got = model.score_distribution(*CASES, rotation, alternatives=k, temperature=temperature)
    lq = log_softmax(logits, temperature)
    target = np.take_along_axis(lq, np.asarray(CASES[1])[..., None], -1)[..., 0]
    assert np.all(np.abs(got.logprob - target) <= SUM + 8 * 2.0 ** -24 * (10 + np.abs(target)))
    entropy = -(np.exp(lq) * lq).sum(-1)
    assert np.all(np.abs(got.entropy - entropy) <= 40 * SUM)
    assert np.array_equal(got.stats[..., 0], logits.max(-1))
    order = np.argsort(-logits.astype(np.float64), axis=-1, kind="stable")[..., :k]
    assert np.array_equal(got.top_ids, order)
    assert np.array_equal(got.top_logits, np.take_along_axis(logits, order, -1))
    want = np.take_along_axis(lq, order, -1)
    assert np.all(np.abs(got.top_logprobs - want) <= SUM + 8 * 2.0 ** -24 * (10 + np.abs(want)))
    if temperature == 1.0:  # the scores of the same cases say the same
        assert np.all(np.abs(got.logprob + nll) <= SUM + 8 * 2.0 ** -24 * (10 + np.abs(nll)))
        assert np.array_equal(got.top_ids[..., 0], amax)


@pytest.mark.parametrize("with_rest", [False, True])
def test_divergence_matches_the_logits(model, edit, with_rest):
    teacher = model.score_distribution(*CASES, alternatives=12)
    before = model.score_batch(*CASES, logits=True)[3]
    after = model.score_batch(*CASES, edit, logits=True)[3]
    got = model.score_divergence(*CASES, teacher.top_ids, teacher.top_logits,
                                 teacher.stats if with_rest else None, edit)
    p_all, lq = np.exp(log_softmax(before, 1.0)), log_softmax(after, 1.0)
    p = np.take_along_axis(p_all, teacher.top_ids.astype(np.int64), -1)
    q = np.take_along_axis(lq, teacher.top_ids.astype(np.int64), -1)
    if with_rest:
        rest, q_rest = 1 - p.sum(-1), 1 - np.exp(q).sum(-1)
        want = (p * (np.log(p) - q)).sum(-1) + rest * np.log(rest / q_rest)
    else:
        p = p / p.sum(-1, keepdims=True)
        want = (p * (np.log(p) - q)).sum(-1)
    # the teacher's statistics are f32 (4 * 2^-24 of about 10), so p and its rest are off by 3e-6
    assert np.all(np.abs(got - want) <= 4 * SUM + 3e-6 * 10)


def test_readout_divergence(gpu, model, edit, golden_tiny):
    """No edit changes nothing; a larger angle changes more."""
    still = ReadoutRotation(golden_tiny["plane_u"], golden_tiny["plane_v"], 0.0)
    none, before = diagnosis.readout_divergence(model, *CASES, DeviceRotation.upload(gpu, still, model.hidden_size))
    some, again = diagnosis.readout_divergence(model, *CASES, edit)
    assert before.top_ids.shape == (4, 4, 20) and np.array_equal(before.top_ids, again.top_ids)
    assert np.all(np.abs(none) <= 4 * SUM + 3e-5)
    assert some.shape == (4, 4) and np.all(some >= -3e-5) and some.max() > none.max()


def test_scores_are_as_before_and_the_cursor_stays(model):
    a = model.score_batch(*CASES, logits=True)
    model.reset()
    model.advance(model.gpu, 3)
    model.score_distribution(*CASES, alternatives=3)
    assert model.position() == 1
    b = model.score_batch(*CASES, logits=True)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_refusals(model, edit):
    ids, values = np.zeros((4, 4, 3), np.uint32), np.zeros((4, 4, 3), np.float32)
    for call in (lambda: model.score_distribution(*CASES, temperature=0.0),
                 lambda: model.score_distribution(*CASES, alternatives=129),
                 lambda: model.score_distribution([[1] * 40], [[2]]),
                 lambda: model.score_distribution([[1]], [[512]]),
                 lambda: model.score_divergence(*CASES, ids, values, temperature=-1.0),
                 lambda: model.score_divergence(*CASES, ids + 512, values),
                 lambda: model.score_divergence(*CASES, ids[..., :0], values[..., :0])):
        with pytest.raises(LsxError):
            call()
    for call in (lambda: model.score_distribution([1, 2], [[3]]),
                 lambda: model.score_distribution(*CASES, alternatives=-1),
                 lambda: model.score_divergence(*CASES, ids[:2], values[:2]),
                 lambda: model.score_divergence(*CASES, ids, values, teacher_stats=np.zeros((4, 4)))):
        with pytest.raises(ValueError):
            call()
