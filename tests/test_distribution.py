"""Argument checks of the distribution operators (lsx_token_logprobs_device and the
entries beside it, laplacesscissors_b200/distribution.py).  No GPU: the C entries check
their arguments before they use the context, and refuse a NULL context last."""
import ctypes as C

import pytest
import torch

from laplacesscissors_b200 import distribution
from laplacesscissors_b200._lib import BF16, F16, F32, lib

A, B, D = 0x10000, 0x4000000, 0x8000000  # addresses that the checks never follow


def message():
    return lib.lsx_last_error().decode()


def logprobs(**change):
    a = dict(ctx=None, logits=A, kind=F32, rows=4, vocab=10, stride=10, temperature=1.0, tokens=B, count=2, k=3,
             logprob=D, entropy=D, stats=D, ids=D, top=D, lp=D, stream=None)
    a.update(change)
    return lib.lsx_token_logprobs_device(*a.values())


def logprobs_backward(**change):
    a = dict(ctx=None, logits=A, kind=F32, rows=4, vocab=10, stride=10, temperature=1.0, tokens=B, count=2, stats=D,
             entropy=D, g=D, h=D, out=B, out_stride=10, stream=None)
    a.update(change)
    return lib.lsx_token_logprobs_backward_device(*a.values())


def distill(**change):
    a = dict(ctx=None, logits=A, kind=F32, rows=4, vocab=10, stride=10, temperature=1.0, ids=D, values=D, count=2,
             tstats=D, weights=D, loss=D, stats=D, out=B, out_stride=10, stream=None)
    a.update(change)
    return lib.lsx_distill_device(*a.values())


def distill_backward(**change):
    a = dict(ctx=None, logits=A, kind=F32, rows=4, vocab=10, stride=10, temperature=1.0, ids=D, values=D, count=2,
             tstats=D, stats=D, g=D, out=B, out_stride=10, stream=None)
    a.update(change)
    return lib.lsx_distill_backward_device(*a.values())


ENTRIES = [logprobs, logprobs_backward, distill, distill_backward]


@pytest.mark.parametrize("entry", ENTRIES)
def test_sound_arguments_reach_the_context(entry):
    assert entry() == 1 and "context" in message()


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("change, says", [
    (dict(logits=None), "invalid"), (dict(kind=3), "kind"), (dict(kind=-1), "kind"), (dict(rows=0), "row count"),
    (dict(rows=(1 << 27) + 1), "row count"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=(1 << 30) + 1, stride=1 << 31), "vocabulary"), (dict(stride=9), "overlap"),
    (dict(stride=(1 << 32) + 1), "overlap"), (dict(logits=A + 2), "aligned"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=float("nan")), "temperature"),
    (dict(temperature=float("inf")), "temperature"), (dict(temperature=1e7), "temperature"),
])
def test_rows_are_checked(entry, change, says):
    assert entry(**change) == 1 and says in message(), message()


@pytest.mark.parametrize("change, says", [
    (dict(count=129), "128"), (dict(tokens=None), "together"), (dict(count=0), "together"),
    (dict(tokens=None, count=0), "together"), (dict(k=129, vocab=200, stride=200), "128"), (dict(k=11), "vocabulary"),
    (dict(k=0), "count"),
])
def test_logprobs_arguments(change, says):
    assert logprobs(**change) == 1 and says in message(), message()


def test_outputs_are_optional():
    assert logprobs(tokens=None, count=0, logprob=None, entropy=None, stats=None, k=0, ids=None, top=None, lp=None) == 1
    assert "context" in message()
    assert distill(loss=None, stats=None, out=None, out_stride=0, weights=None, tstats=None) == 1
    assert "context" in message()
    assert logprobs_backward(entropy=None, h=None) == 1 and "context" in message()
    assert logprobs_backward(tokens=None, count=0, g=None) == 1 and "context" in message()


@pytest.mark.parametrize("change, says", [
    (dict(count=129), "128"), (dict(g=None), "together"), (dict(tokens=None), "together"), (dict(count=0), "together"),
    (dict(h=None), "entropy"), (dict(entropy=None), "entropy"), (dict(stats=None), "invalid"),
])
def test_logprobs_backward_arguments(change, says):
    assert logprobs_backward(**change) == 1 and says in message(), message()


@pytest.mark.parametrize("entry", [distill, distill_backward])
@pytest.mark.parametrize("change, says", [
    (dict(ids=None), "invalid"), (dict(values=None), "invalid"), (dict(count=0), "128"), (dict(count=129), "128"),
])
def test_teacher_arguments(entry, change, says):
    assert entry(**change) == 1 and says in message(), message()


def test_distill_arguments():
    assert distill(out=None) == 1 and "weights" in message()
    assert distill_backward(stats=None) == 1 and "invalid" in message()
    assert distill_backward(g=None) == 1 and "invalid" in message()
    assert distill_backward(out=None) == 1 and "invalid" in message()


@pytest.mark.parametrize("entry", [logprobs_backward, distill, distill_backward])
def test_gradient_memory(entry):
    """In place, or apart from the logits; never partly over them."""
    assert entry(out=A) == 1 and "context" in message()  # in place
    assert entry(out=A, out_stride=12) == 1 and "overlaps" in message()
    assert entry(out=A + 4) == 1 and "overlaps" in message()
    assert entry(out=A + 40 * 4 - 4) == 1 and "overlaps" in message()
    assert entry(out=A + 40 * 4) == 1 and "context" in message()  # right behind
    assert entry(out=A - 40 * 4) == 1 and "context" in message()  # right before
    assert entry(out=A - 40 * 4 + 4) == 1 and "overlaps" in message()
    assert entry(out=B, out_stride=9) == 1 and "overlap" in message()
    assert entry(out=B + 2) == 1 and "aligned" in message()
    # two column blocks of one buffer of 20 columns
    assert entry(stride=20, out=A + 40, out_stride=20) == 1 and "context" in message()
    assert entry(stride=20, out=A + 36, out_stride=20) == 1 and "overlaps" in message()
    assert entry(stride=20, out=A + 44, out_stride=20) == 1 and "overlaps" in message()
    assert entry(stride=20, logits=A + 40, out=A, out_stride=20) == 1 and "context" in message()
    for kind in (F16, BF16):
        assert entry(kind=kind, out=A + 40 * 2) == 1 and "context" in message()
        assert entry(kind=kind, out=A + 40 * 2 - 2) == 1 and "overlaps" in message()


class FakeGpu:
    device = 0
    handle = C.c_void_p(None)


def test_python_refuses_what_is_not_on_the_device():
    z = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="device"):
        distribution.token_logprobs(FakeGpu(), z)
    with pytest.raises(ValueError, match="float32"):
        distribution.token_logprobs(FakeGpu(), z.double())
    with pytest.raises(ValueError, match="rows, vocab"):
        distribution.token_logprobs(FakeGpu(), z[0])
    with pytest.raises(ValueError, match="float32"):
        distribution.distill(FakeGpu(), z.int(), z.int(), z)
