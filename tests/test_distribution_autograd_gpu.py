"""What torch's autograd learns of the calls of laplacesscissors_b200/distribution.py: every tensor
that a call writes counts as modified, and an `out` that a caller gives is what it gets back; a
gradient handed to backward() reaches the weights behind the logits."""
import pytest
import torch

from laplacesscissors_b200 import distribution
from test_distribution_gpu import dev, distill64, logprobs_gradient64, make, stored, teacher_of, within  # noqa: F401

pytestmark = pytest.mark.gpu


def calls(gpu, dev):
    z = make(dev, 80, 3, 900, torch.float32)
    ids, values, stats = teacher_of(dev, 81, z, 6, 1.0)
    one = torch.ones(3, device=dev)
    tokens = ids[:, :2].contiguous()
    first = distribution.token_logprobs(gpu, z, tokens, alternatives=4)
    step = distribution.distill(gpu, z, ids, values, teacher_stats=stats, gradient=True)
    return {
        "logprobs": ([t.clone() for t in first],
                     lambda out: distribution.token_logprobs(gpu, z, tokens, alternatives=4, out=out)),
        "logprobs backward": ([z.clone()], lambda out: (distribution.token_logprobs_backward(
            gpu, z, tokens, first.stats, first.entropy, torch.ones(3, 2, device=dev), one, out=out[0]),)),
        "distill": ([step.loss.clone(), step.stats.clone()],
                    lambda out: distribution.distill(gpu, z, ids, values, out=(*out, None))[:2]),
        "step": ([t.clone() for t in step], lambda out: distribution.distill(
            gpu, z, ids, values, teacher_stats=stats, gradient=True, out=out)),
        "distill backward": ([z.clone()], lambda out: (distribution.distill_backward(
            gpu, z, ids, values, step.stats, one, teacher_stats=stats, out=out[0]),)),
    }


@pytest.mark.parametrize("name", ["logprobs", "logprobs backward", "distill", "step", "distill backward"])
def test_written_tensors_count_as_modified(gpu, dev, name):
    out, call = calls(gpu, dev)[name]
    before = [t._version for t in out]
    got = call(out)
    assert len(got) == len(out)
    for b, t, g in zip(before, out, got):
        assert g is t and t._version > b


@pytest.mark.parametrize("name", ["step", "logprobs backward", "distill backward"])
def test_autograd_notices_a_saved_tensor_that_was_overwritten(gpu, dev, name):
    """exp saves its result: a gradient written over it must not go into exp's own gradient unseen."""
    out, call = calls(gpu, dev)[name]
    leaf = torch.zeros(3, 900, device=dev, requires_grad=True)
    saved = leaf.exp()
    out[-1] = saved.detach()
    call(out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()


def test_modification_is_counted_under_no_grad_and_capture(gpu, dev):
    out, call = calls(gpu, dev)["step"]
    graph = torch.cuda.CUDAGraph()
    before = out[2]._version
    with torch.no_grad():
        call(out)
        after = out[2]._version
        torch.cuda.synchronize(dev)
        with torch.cuda.graph(graph):
            call(out)
    assert before < after < out[2]._version
    with torch.inference_mode():
        mine = [t.clone() for t in out]  # inference tensors have no counter
        call(mine)
    assert all(torch.equal(a, b) for a, b in zip(mine, out))


@pytest.mark.parametrize("step", ["distill", "logprobs"])
def test_a_training_step(gpu, dev, step):
    """Logits of a readout in 64 bits, rounded to f32 on their way: the weights' gradient is the
    states' product with the formula's, within what the states make of its tolerance."""
    g = torch.Generator().manual_seed(82)
    states = torch.randn(6, 24, generator=g, dtype=torch.float64).to(dev)
    weight = (torch.randn(24, 2003, generator=g, dtype=torch.float64) * 0.5).to(dev).requires_grad_()
    logits = (states @ weight).float()
    z = logits.detach()
    ids, values, stats = teacher_of(dev, 83, z, 9, 1.0)
    each = torch.linspace(0.5, 2, 6, device=dev)
    if step == "distill":
        logits.backward(distribution.distill(gpu, z, ids, values, teacher_stats=stats, weights=each,
                                             gradient=True).gradient)
        _, _, want, _, tol = distill64(z, ids, values, stats, each, 1.0)
    else:
        tokens = ids[:, :2].contiguous()
        own = torch.stack([each, -each], 1)
        f = distribution.token_logprobs(gpu, z, tokens)
        logits.backward(distribution.token_logprobs_backward(gpu, z, tokens, f.stats, f.entropy, own, each))
        want, tol = logprobs_gradient64(z, tokens, own, each, 1.0)
    within(weight.grad, states.t() @ want, states.abs().t() @ stored(want, tol, torch.float32))
