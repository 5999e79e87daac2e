"""Host side of laplacesscissors_b200/distribution.py and its callers: what torch's autograd would
lose is refused, the module can be imported beside a torch without CUDA, and the default call of
diagnosis.readout_divergence suits any vocabulary.  No GPU: refusals come before anything is
launched, and a model of plain Python stands in for the other calls."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT
from laplacesscissors_b200 import LsxError, diagnosis, distribution


class HostGpu:
    """Where CPU tensors say they are (get_device), with no context: a call that passes the Python
    checks is refused by the library, which needs one."""
    device = -1
    handle = C.c_void_p(None)


@pytest.fixture
def host(monkeypatch):
    monkeypatch.setattr(distribution, "_stream", lambda device: 0)
    return HostGpu()


def rows(**kw):
    return torch.zeros(2, 5, **kw)


IDS, ONE = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2)


def test_logits_that_require_grad_are_refused(host):
    z, values = rows(requires_grad=True), torch.zeros(2, 3)
    for call in (lambda: distribution.token_logprobs(host, z, IDS),
                 lambda: distribution.token_logprobs(host, z * 2),
                 lambda: distribution.distill(host, z, IDS, values),
                 lambda: distribution.distill(host, rows(), IDS, values.clone().requires_grad_())):
        with pytest.raises(ValueError, match="detach"):
            call()
        with torch.no_grad(), pytest.raises(LsxError, match="context"):
            call()


def test_calls_that_give_the_gradient_take_logits_that_require_grad(host):
    z, values = rows(requires_grad=True), torch.zeros(2, 3)
    for call in (lambda: distribution.token_logprobs(host, z.detach(), IDS),
                 lambda: distribution.distill(host, z, IDS, values, gradient=True),
                 lambda: distribution.token_logprobs_backward(host, z, IDS, torch.zeros(2, 2), None, values),
                 lambda: distribution.distill_backward(host, z, IDS, values, torch.zeros(2, 3), ONE)):
        with pytest.raises(LsxError, match="context"):
            call()


def test_import_without_the_raw_stream_of_a_cuda_build():
    code = ("import torch\n"
            "del torch._C._cuda_getCurrentRawStream\n"
            "from laplacesscissors_b200 import distribution\n"
            "class Stream: cuda_stream = 77\n"
            "torch.cuda.current_stream = lambda device: Stream if device == 3 else None\n"
            "assert distribution._stream(3) == 77\n")
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


class PlainModel:
    def __init__(self, vocab):
        self.vocab, self.asked = vocab, []

    def vocab_size(self):
        return self.vocab

    def score_distribution(self, prompts, targets, rotation=None, alternatives=0, temperature=1.0):
        self.asked.append(alternatives)
        return _Scored()

    def score_divergence(self, prompts, targets, ids, logits, stats, rotation, temperature):
        return np.zeros((1, 1), np.float32)


class _Scored:
    top_ids = top_logits = stats = None


@pytest.mark.parametrize("vocab, default", [(1, 1), (7, 7), (19, 19), (20, 20), (151936, 20)])
def test_default_alternatives_suit_the_vocabulary(vocab, default):
    model = PlainModel(vocab)
    diagnosis.readout_divergence(model, [[1]], [[0]], None)
    diagnosis.readout_divergence(model, [[1]], [[0]], None, 9)  # as asked, for the library to refuse
    assert model.asked == [default, 9]
