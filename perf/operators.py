"""Measured cases of the operators on rows of logits: log probabilities of given
tokens with entropy and top alternatives, and distillation from a teacher's top
logits, each with its backward pass.

A case names one operator ("op"), the rows and the vocabulary, the storage type of
the logits, the distance between rows in elements beyond the vocabulary ("pad"),
and the operator's own sizes.  Token ids are int32; -1 marks an unused slot.

Definitions, per row with z the logits, T the temperature, m = max z,
s = log sum_i exp((z_i - m) / T) and q_i = exp((z_i - m) / T - s):

  logprobs   for given tokens t: log q_t (0 for an unused slot); the entropy
             -sum_i q_i log q_i; (m, s); the k largest z in descending order (the
             lower id first among equals) as ids, logits and log q.
  logprobs_backward
             gradient with respect to z of sum_n g_n log q_{t_n} + h entropy.
  distill    teacher tokens K with logits a: p_j = exp(a_j / T) normalised over K,
             or, where the teacher's (m, s) are given, its own probabilities, with
             p_r = max(0, 1 - sum_K p) and q_r for all tokens outside K;
             loss = sum_K p_j log(p_j / q_j) + p_r log(p_r / q_r).  The loss comes
             with (m, s, log of the student's unnormalised mass outside K, or -inf
             where the teacher's statistics are not given).
  distill_step
             the same, and the gradient with respect to z of weight * loss.
  distill_backward
             that gradient from the logits, the teacher and saved statistics.

A row whose logits are all -inf holds no distribution: its log probabilities are
-inf, its entropy and its gradient 0, and (m, s) = (-inf, 0).
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decode step's answer over a full vocabulary: the emitted token with 20 alternatives.
        {"name": "logprobs_one_row", "op": "logprobs", "rows": 1, "vocab": 151936, "type": "f32", "pad": 0,
         "tokens": 1, "k": 20, "temperature": 1.0, "masked": 0.0},
        # A test-sized vocabulary: the smallest call, where only latency counts.
        {"name": "logprobs_tiny", "op": "logprobs", "rows": 3, "vocab": 512, "type": "f32", "pad": 0,
         "tokens": 1, "k": 5, "temperature": 1.0, "masked": 0.0},
        # A batch of 16 sequences, one step, most of the vocabulary masked by a grammar.
        {"name": "logprobs_batch16_masked", "op": "logprobs", "rows": 16, "vocab": 151936, "type": "bf16", "pad": 0,
         "tokens": 1, "k": 20, "temperature": 0.7, "masked": 0.9},
        # Teacher-forced scoring of many cases: 2048 scored positions of f32 logits.
        {"name": "logprobs_scoring", "op": "logprobs", "rows": 2048, "vocab": 151936, "type": "f32", "pad": 0,
         "tokens": 1, "k": 8, "temperature": 1.0, "masked": 0.0},
        # Rows of odd length, so that no two start at the same alignment; four candidate tokens a row.
        {"name": "logprobs_odd", "op": "logprobs", "rows": 777, "vocab": 50257, "type": "f16", "pad": 0,
         "tokens": 4, "k": 50, "temperature": 1.3, "masked": 0.0},
        # Policy training over scored positions: gradient of the tokens' log probability and the entropy.
        {"name": "logprobs_backward_training", "op": "logprobs_backward", "rows": 2048, "vocab": 151936,
         "type": "bf16", "pad": 0, "tokens": 1, "temperature": 1.0, "masked": 0.0},
        # A few odd rows of a padded buffer, three tokens each.
        {"name": "logprobs_backward_odd", "op": "logprobs_backward", "rows": 45, "vocab": 32003, "type": "f32",
         "pad": 5, "tokens": 3, "temperature": 0.8, "masked": 0.3},
        # How far an edited readout is from the model's own top 20, over scored positions.
        {"name": "distill_divergence", "op": "distill", "rows": 512, "vocab": 151936, "type": "f32", "pad": 0,
         "k": 20, "tail": True, "temperature": 1.0, "masked": 0.0},
        # The same on a test-sized vocabulary.
        {"name": "distill_tiny", "op": "distill", "rows": 4, "vocab": 512, "type": "f32", "pad": 0,
         "k": 8, "tail": True, "temperature": 1.0, "masked": 0.0},
        # One training step's loss and gradient over a full vocabulary.
        {"name": "distill_step_training", "op": "distill_step", "rows": 2048, "vocab": 151936, "type": "bf16", "pad": 0,
         "k": 64, "tail": False, "temperature": 2.0, "masked": 0.0},
        # A short step with the tail bucket, f32 logits in a padded buffer.
        {"name": "distill_step_tail", "op": "distill_step", "rows": 190, "vocab": 128003, "type": "f32", "pad": 61,
         "k": 100, "tail": True, "temperature": 1.0, "masked": 0.2},
        # The gradient alone, from saved statistics.
        {"name": "distill_backward_saved", "op": "distill_backward", "rows": 1000, "vocab": 50257, "type": "f16",
         "pad": 0, "k": 33, "tail": True, "temperature": 1.5, "masked": 0.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_backward", "distill", "distill_step", "distill_backward"])
    vocab = _spread(rng, 130, 200000)
    if rng.random() < 0.5:
        vocab |= 1
    rows = max(1, min(_spread(rng, 1, 3000), 100_000_000 // vocab))
    case = {"op": op, "rows": rows, "vocab": vocab, "type": rng.choice(["f32", "f16", "bf16"]),
            "pad": rng.choice([0, 0, rng.randint(1, 64)]), "temperature": rng.choice([1.0, round(rng.uniform(0.3, 3.0), 2)]),
            "masked": rng.choice([0.0, 0.0, round(rng.random() * 0.999, 3)])}
    if op.startswith("logprobs"):
        case["tokens"] = rng.choice([1, 1, rng.randint(1, 16)])
    else:
        case["tail"] = rng.random() < 0.5
    if op != "logprobs_backward":
        case["k"] = rng.choice([rng.randint(1, 20), rng.randint(1, 128)])
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _blocks(rows, vocab):
    """Row ranges of about 64 Mi elements each."""
    step = max(1, (1 << 26) // vocab)
    return [(a, min(rows, a + step)) for a in range(0, rows, step)]


def prepare(case, seed):
    g = _generator(seed)
    R, V, dtype = case["rows"], case["vocab"], _TYPES[case["type"]]
    dev = "cuda"
    s = {"case": dict(case), "temperature": case["temperature"]}
    buffer = torch.zeros(R, V + case["pad"], dtype=dtype, device=dev)
    logits = buffer[:, :V]
    op = case["op"]
    teach = op.startswith("distill")
    if teach:
        k = case["k"]
        ids = torch.empty(R, k, dtype=torch.int32, device=dev)
        values = torch.empty(R, k, dtype=torch.float32, device=dev)
        stats = torch.empty(R, 2, dtype=torch.float32, device=dev)
    for a, b in _blocks(R, V):
        n = b - a
        z = torch.randn(n, V, generator=g, device=dev) * 2.5
        # a few likely tokens a row, as a language model's logits have
        likely = (torch.randint(0, V, (n, 1), generator=g, device=dev) + torch.arange(0, V, V // 12, device=dev)[:12]) % V
        z.scatter_(1, likely, 6.0 + 3.0 * torch.randn(n, 12, generator=g, device=dev))
        if case["masked"]:
            keep = torch.rand(n, V, generator=g, device=dev) >= case["masked"]
            keep[:, 0] = True
            if a == 0 and R > 2 and not teach:
                keep[1] = False  # a padded position: nothing allowed
            z.masked_fill_(~keep, float("-inf"))
        logits[a:b] = z.to(dtype)
        if teach:
            t = z + torch.randn(n, V, generator=g, device=dev)
            top = torch.topk(t, k, dim=1)
            ids[a:b] = torch.where(top.values > -math.inf, top.indices, -1).to(torch.int32)
            values[a:b] = top.values
            d = t.double() / case["temperature"]
            stats[a:b, 0] = top.values[:, 0]
            stats[a:b, 1] = (torch.logsumexp(d, 1) - d.amax(1)).float()
            del t, d
        del z
    s["logits"] = logits
    grad = torch.zeros_like(buffer)[:, :V] if op not in ("logprobs", "distill") else None
    if not teach:
        n = case["tokens"]
        tokens = torch.randint(0, V, (R, n), generator=g, device=dev)
        likely = logits.float().argmax(1)
        pick = torch.rand(R, n, generator=g, device=dev)
        tokens = torch.where(pick < 0.5, likely[:, None].expand(R, n), tokens)
        if n > 1:
            tokens = torch.where(pick > 0.95, torch.full_like(tokens, -1), tokens)
        s["tokens"] = tokens.to(torch.int32).contiguous()
        if op == "logprobs":
            k = case["k"]
            s["out"] = (torch.empty(R, n, device=dev), torch.empty(R, device=dev), torch.empty(R, 2, device=dev),
                        torch.empty(R, k, dtype=torch.int32, device=dev), torch.empty(R, k, device=dev),
                        torch.empty(R, k, device=dev))
        else:
            s["logprob_grad"] = torch.randn(R, n, generator=g, device=dev)
            s["entropy_grad"] = 0.1 * torch.randn(R, generator=g, device=dev)
            s["stats"], s["entropy"] = _saved(logits, case["temperature"])
            s["out"] = grad
        return s
    # slots that a shorter teacher list leaves unused
    if case["k"] > 4:
        unused = torch.rand(R, case["k"], generator=g, device=dev) < 0.03
        ids = torch.where(unused, torch.full_like(ids, -1), ids)
    s["ids"], s["values"] = ids, values
    s["teacher_stats"] = stats if case["tail"] else None
    if op == "distill":
        s["weights"] = None
        s["out"] = (torch.empty(R, device=dev), torch.empty(R, 3, device=dev), None)
    elif op == "distill_step":
        s["weights"] = 0.5 + torch.rand(R, generator=g, device=dev)
        s["out"] = (torch.empty(R, device=dev), torch.empty(R, 3, device=dev), grad)
    else:
        s["weights"] = 0.5 + torch.rand(R, generator=g, device=dev)
        s["stats"] = _saved(logits, case["temperature"], ids if case["tail"] else False)
        s["out"] = grad
    return s


def _saved(logits, T, ids=None):
    """What a forward pass leaves for the backward one, made in 64 bits."""
    R, V = logits.shape
    stats = torch.empty(R, 2 if ids is None else 3, dtype=torch.float32, device=logits.device)
    entropy = torch.empty(R, dtype=torch.float32, device=logits.device)
    for a, b in _blocks(R, V):
        z = logits[a:b].double()
        m = z.amax(1, keepdim=True)
        y = torch.where(z == -math.inf, z, (z - m) / T)
        e = torch.exp(y)
        total = e.sum(1)
        empty = m[:, 0] == -math.inf
        log_total = torch.where(empty, torch.zeros_like(total), torch.log(total))
        stats[a:b, 0] = m[:, 0]
        stats[a:b, 1] = log_total
        q = e / total.clamp_min(1e-300)[:, None]
        entropy[a:b] = -(q * torch.where(q > 0, y - log_total[:, None], torch.zeros_like(y))).sum(1)
        if ids is False:
            stats[a:b, 2] = -math.inf
        elif ids is not None:
            i = ids[a:b].long()
            e = torch.cat([e, torch.zeros_like(e[:, :1])], 1).scatter(1, torch.where(i < 0, V, i), 0.0)
            stats[a:b, 2] = torch.log(e.sum(1))
    return stats if ids is not None else (stats, entropy)


# ---- the plain forms ---------------------------------------------------------
def _shifted(logits, T):
    """(m, (z - m) / T, exp of it, its sum) in 32 bits; an empty row gets sum 1 of nothing."""
    z = logits.float()
    m = z.amax(1, keepdim=True)
    y = (z - torch.where(m == -math.inf, torch.zeros_like(m), m)) / T
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    return m, y, e, torch.where(m == -math.inf, torch.ones_like(total), total)


def _slots(ids, vocab):
    """Which slots hold a token, each token counted at its first slot; and ids with 0 elsewhere."""
    used = ids >= 0
    same = ids[:, :, None] == ids[:, None, :]
    before = torch.ones(ids.shape[1], ids.shape[1], dtype=torch.bool, device=ids.device).tril(-1)
    used = used & ~(same & before).any(2)
    return used, torch.where(used, ids, torch.zeros_like(ids)).long()


def _plain_logprobs(s):
    c, T, logits = s["case"], s["temperature"], s["logits"]
    m, y, e, total = _shifted(logits, T)
    log_total = torch.log(total)
    used = s["tokens"] >= 0
    at = torch.where(used, s["tokens"], torch.zeros_like(s["tokens"])).long()
    logprob = torch.where(used, y.gather(1, at) - log_total, torch.zeros_like(at, dtype=torch.float32))
    entropy = log_total[:, 0] - (e * torch.where(e > 0, y, torch.zeros_like(y))).sum(1) / total[:, 0]
    stats = torch.cat([m, log_total], 1)
    del y, e
    # the order of (value, lower id first) as one 64-bit key
    bits = (logits.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    ids = torch.arange(c["vocab"], device=logits.device)
    key = (order << 32) | (0xFFFFFFFF - ids)
    del bits, order
    top = 0xFFFFFFFF - (torch.topk(key, c["k"], dim=1).values & 0xFFFFFFFF)
    top_logits = logits.gather(1, top).float()
    shift = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return [logprob, entropy, stats, top.to(torch.int32), top_logits, (top_logits - shift) / T - log_total]


def _plain_logprobs_backward(s):
    T, logits = s["temperature"], s["logits"]
    m, y, e, total = _shifted(logits, T)
    y = y - torch.log(total)
    q = e / total
    used = s["tokens"] >= 0
    at = torch.where(used, s["tokens"], torch.zeros_like(s["tokens"])).long()
    g = torch.where(used, s["logprob_grad"], torch.zeros_like(s["logprob_grad"]))
    h = s["entropy_grad"][:, None]
    inner = g.sum(1, keepdim=True) + h * (torch.where(q > 0, y, torch.zeros_like(y)) + s["entropy"][:, None])
    out = -q * inner
    out.scatter_add_(1, at, torch.where(m == -math.inf, torch.zeros_like(g), g))
    return (out / T).to(logits.dtype)


def _plain_distill(s, gradient, loss=True):
    T, logits, V = s["temperature"], s["logits"], s["case"]["vocab"]
    m, y, e, total = _shifted(logits, T)
    log_total = torch.log(total)
    used, at = _slots(s["ids"], V)
    # the teacher's few numbers in 64 bits: 1 - sum p is next to 0 for a confident teacher
    values = torch.where(used, s["values"].double(), -math.inf)
    none = torch.zeros_like(s["values"])
    tail = s["teacher_stats"] is not None
    if tail:
        stats = s["teacher_stats"].double()
        log_p = (values - stats[:, :1]) / T - stats[:, 1:]
    else:
        top = values.amax(1, keepdim=True)
        shifted = (values - torch.where(top == -math.inf, torch.zeros_like(top), top)) / T
        part = torch.exp(shifted).sum(1, keepdim=True)
        log_p = shifted - torch.log(torch.where(part > 0, part, torch.ones_like(part)))
    p = torch.exp(log_p)
    listed_mass = p.sum(1, keepdim=True)
    rest = torch.clamp(1.0 - listed_mass, min=0.0).float() if tail else none[:, :1]
    p, log_p, listed_mass = p.float(), log_p.float(), listed_mass.float()
    outside = torch.cat([e, torch.zeros_like(e[:, :1])], 1).scatter(1, torch.where(used, at, V), 0.0).sum(1, keepdim=True)
    rest = torch.where(outside > 0, rest, torch.zeros_like(rest))
    log_q = y.gather(1, at) - log_total
    answers = []
    if loss:
        value = torch.where(p > 0, p * (log_p - log_q), none).sum(1, keepdim=True)
        value = value + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(outside) + log_total), torch.zeros_like(rest))
        log_outside = torch.log(outside) if tail else torch.full_like(outside, -math.inf)
        answers += [value[:, 0], torch.cat([m, log_total, log_outside], 1)]
    if gradient:
        q = e / total
        mass = listed_mass + rest
        share = torch.where(rest > 0, rest * total / outside, torch.zeros_like(rest))
        out = q * (mass - share)
        here = q.gather(1, at) * mass - p
        out = torch.cat([out, torch.zeros_like(out[:, :1])], 1)
        out.scatter_(1, torch.where(used, at, V), here)
        w = torch.where(m == -math.inf, torch.zeros_like(m), s["weights"][:, None] / T)
        answers.append((out[:, :V] * w).to(logits.dtype))
    return answers


_gpu = None


def run(s):
    op = s["case"]["op"]
    if own:
        global _gpu
        from laplacesscissors_b200 import Gpu, distribution
        if _gpu is None:
            _gpu = Gpu(torch.cuda.current_device())
        if op == "logprobs":
            return list(distribution.token_logprobs(_gpu, s["logits"], s["tokens"], alternatives=s["case"]["k"],
                                                    temperature=s["temperature"], out=s["out"]))
        if op == "logprobs_backward":
            return [distribution.token_logprobs_backward(_gpu, s["logits"], s["tokens"], s["stats"], s["entropy"],
                                                         s["logprob_grad"], s["entropy_grad"],
                                                         temperature=s["temperature"], out=s["out"])]
        if op == "distill_backward":
            return [distribution.distill_backward(_gpu, s["logits"], s["ids"], s["values"], s["stats"], s["weights"],
                                                  teacher_stats=s["teacher_stats"], temperature=s["temperature"],
                                                  out=s["out"])]
        got = distribution.distill(_gpu, s["logits"], s["ids"], s["values"], teacher_stats=s["teacher_stats"],
                                   weights=s["weights"], temperature=s["temperature"],
                                   gradient=op == "distill_step", out=s["out"])
        return [x for x in got if x is not None]
    if op == "logprobs":
        return _plain_logprobs(s)
    if op == "logprobs_backward":
        return [_plain_logprobs_backward(s)]
    return _plain_distill(s, gradient=op != "distill", loss=op != "distill_backward")


def work(case):
    cells = case["rows"] * case["vocab"]
    wide = _BYTES[case["type"]]
    writes = case["op"] not in ("logprobs", "distill")
    small = case["rows"] * (8 * case.get("tokens", 0) + 8 * case.get("k", 0) + 24)
    # a subtraction, an exponential and a sum for the statistics (and a product and a sum for the entropy);
    # an exponential of a scaled difference and a product for the gradient
    flops = {"logprobs": 6, "logprobs_backward": 7, "distill": 4, "distill_step": 8, "distill_backward": 4}[case["op"]]
    return {"bytes": float(cells * wide * (2 if writes else 1) + small), "flops": float(cells * flops)}


# ---- the definition in 64 bits ------------------------------------------------
def _exact_rows(s, a, b):
    c, T, V = s["case"], float(s["temperature"]), s["case"]["vocab"]
    z = s["logits"][a:b].double()
    m = z.max(dim=1).values
    dead = torch.isinf(m)
    lse = torch.logsumexp(z / T, dim=1)
    logq = z / T - torch.where(dead, 0.0, lse)[:, None]
    logsum = torch.where(dead, 0.0, lse - m / T)
    if c["op"].startswith("logprobs"):
        t = s["tokens"][a:b].long()
        q = logq.exp()
        plogp = torch.nan_to_num(q * logq, nan=0.0)
        if c["op"] == "logprobs":
            lp = torch.where(t < 0, 0.0, logq.gather(1, t.clamp_min(0)))
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :c["k"]]
            return [lp, -plogp.sum(1), torch.stack([m, logsum], 1), order.to(torch.int32), z.gather(1, order),
                    logq.gather(1, order)]
        g = torch.where(t < 0, 0.0, s["logprob_grad"][a:b].double())
        h = s["entropy_grad"][a:b].double()[:, None]
        out = torch.zeros_like(z).scatter_add_(1, t.clamp_min(0), g) - q * g.sum(1, keepdim=True)
        out -= h * (plogp - q * plogp.sum(1, keepdim=True))
        return [torch.where(dead[:, None], 0.0, out / T)]
    ids = s["ids"][a:b].long()
    n, k = ids.shape
    teacher = torch.full((n, V + 1), -math.inf, dtype=torch.float64, device=z.device)
    teacher.scatter_(1, torch.where(ids < 0, V, ids), s["values"][a:b].double() / T)
    teacher = teacher[:, :V]
    inside = torch.zeros(n, V + 1, dtype=torch.bool, device=z.device)
    inside.scatter_(1, torch.where(ids < 0, V, ids), True)
    inside = inside[:, :V]
    q = logq.exp()
    if s["teacher_stats"] is None:
        norm = torch.logsumexp(teacher, 1)
        logp = teacher - torch.where(torch.isinf(norm), 0.0, norm)[:, None]
        rest = torch.zeros(n, dtype=torch.float64, device=z.device)
        logsum_rest = torch.full_like(rest, -math.inf)
    else:
        ts = s["teacher_stats"][a:b].double()
        logp = teacher - (ts[:, 0] / T + ts[:, 1])[:, None]
        rest = (1.0 - logp.exp().sum(1)).clamp_min(0.0)
        logsum_rest = torch.logsumexp(torch.where(inside, -math.inf, z / T), 1) - m / T
    q_rest = torch.where(inside, 0.0, q).sum(1)
    rest = torch.where(q_rest > 0, rest, 0.0)
    p = logp.exp()
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(1) + torch.where(rest > 0, rest * torch.log(rest / q_rest), 0.0)
    answers = [loss, torch.stack([m, logsum, logsum_rest], 1)] if c["op"] != "distill_backward" else []
    if c["op"] != "distill":
        w = s["weights"][a:b].double() / T
        ratio = torch.where(rest > 0, rest / q_rest, 0.0)
        out = q * (p.sum(1) + rest)[:, None] - p - torch.where(inside, 0.0, q) * ratio[:, None]
        answers.append(torch.where(dead, 0.0, w)[:, None] * out)
    return answers


def exact(case, seed):
    s = prepare(case, seed)
    parts = [_exact_rows(s, a, b) for a, b in _blocks(case["rows"], case["vocab"])]
    return [None if column[0] is None else torch.cat(column) for column in zip(*parts)]
