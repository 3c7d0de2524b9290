"""Oracle for the vocabulary-list operators (the k most likely tokens of a row; distillation from a
teacher's top tokens): the definitions written out with library routines, CPU torch, in the dtype
of the inputs (tests pass float64). No reference counterpart: the reference computes the log-prob
of one label per row (openrlhf/models/utils.py:139-163). Test infrastructure."""
import math

import torch


def top_logprobs(logits, k, temperature=1.0, row_mask=None):
    """(top_log_probs, top_ids): the k largest logits, descending, equal logits by ascending id, NaN
    before everything (a stable sort does exactly that)."""
    order = torch.sort(logits + 0.0, dim=-1, descending=True, stable=True).indices[..., :k]
    lp = torch.log_softmax(logits / temperature, dim=-1).gather(-1, order)
    if row_mask is not None:
        keep = (row_mask != 0).unsqueeze(-1)
        lp = torch.where(keep, lp, torch.zeros_like(lp))
        order = torch.where(keep, order, torch.full_like(order, -1))
    return lp, order


def top_objective(logits, labels, top_ids, g_logprob, g_entropy, g_top, temperature=1.0):
    """sum g_lp logprob + g_H entropy + g_k top_logprob, for autograd; absent ids (-1) contribute
    nothing. One row at a time would be the same: rows do not interact."""
    log_t = torch.log_softmax(logits / temperature, dim=-1)
    total = logits.new_zeros(())
    if g_logprob is not None:
        total = total + (log_t.gather(-1, labels.unsqueeze(-1)).squeeze(-1) * g_logprob).sum()
    if g_entropy is not None:
        p = torch.softmax(logits, dim=-1)
        total = total + ((torch.logsumexp(logits, dim=-1) - (p * logits).sum(-1)) * g_entropy).sum()
    if g_top is not None:
        on = (top_ids >= 0).to(logits.dtype)
        total = total + (log_t.gather(-1, top_ids.clamp(min=0)) * g_top * on).sum()
    return total


def distill_kl_row(logits, ids, teacher, temperature=1.0, teacher_temperature=1.0, kl="forward", tail=True):
    """KL divergence of one row, as a Python-level sum over outcomes (differentiable in `logits`).

    The teacher's list is a dict id -> probability: negative ids and log-probs of -inf are absent, an
    id that appears twice has the sum of its probabilities."""
    listed = {}
    for i, v in zip(ids.tolist(), teacher.tolist()):
        if i >= 0 and v != -math.inf:
            listed.setdefault(i, []).append(v / teacher_temperature)
    log_q = torch.log_softmax(logits / temperature, dim=-1)
    zero = torch.where(torch.isfinite(logits), logits, 0.0).sum() * 0.0  # masked logits may be -inf
    if not listed:
        return zero
    joined = lambda off: {i: torch.logsumexp(torch.tensor(v, dtype=torch.float64) - off, 0).item() for i, v in listed.items()}  # noqa: E731
    if kl == "forward" and not tail:  # a softmax: the values may be logits of any size, their largest comes off first
        log_p = joined(max(max(v) for v in listed.values()))
        log_w = torch.log_softmax(torch.tensor(list(log_p.values()), dtype=torch.float64), 0).tolist()
        return zero + sum(math.exp(v) * (v - log_q[i]) for i, v in zip(log_p, log_w))
    log_p = joined(0.0)
    mass = math.fsum(math.exp(v) for v in log_p.values())
    outside = torch.ones_like(logits, dtype=torch.bool)
    outside[list(log_p)] = False
    s = log_q.exp()[outside].sum().clamp(min=2.0 ** -126)
    if kl == "forward":
        t = max(0.0, 1.0 - mass)
        body = sum(math.exp(v) * (v - log_q[i]) for i, v in log_p.items())
        return zero + body + (t * (math.log(t) - s.log()) if t > 0.0 and bool(outside.any()) else 0.0)
    t = max(2.0 ** -24, 1.0 - mass)
    body = sum(log_q[i].exp() * (log_q[i] - v) for i, v in log_p.items())
    return zero + body + (s * (s.log() - math.log(t)) if bool(outside.any()) else 0.0)
