"""What the vocabulary-list operators are timed on, with their plain forms.

Two operators over rows of vocabulary logits [N, V]:

  alternatives  log-prob of a given token, entropy, and the k most likely tokens with their log-probs
                (``openrlhf_amd.models.utils.top_logprobs_from_logits``), forward alone and with the
                gradients of all three;
  distillation  KL divergence between a teacher known by its k most likely tokens and the student's
                full row (``distill_kl_from_logits``, ``fused_distill_kl_fwd_bwd``), forward alone,
                forward and backward as an autograd graph, and both in one pass.

With z = x / T, q = softmax(z), and the list of a row (id_k, p_k = exp(teacher log-prob)):

  forward KL with the tail    sum_k p_k (log p_k - log q_k) + t (log t - log s)
  forward KL without it       sum_k w_k (log w_k - log q_k),  w = p / sum p
  reverse KL with the tail    sum_k q_k (log q_k - log p_k) + s (log s - log t)

where s is the student's mass outside the list and t = 1 - sum p the teacher's (at least 0 in the
forward form, at least 2^-24 in the reverse form, where its logarithm is taken whatever it is).
An entry with a negative id is absent. A row whose mask is 0 gives zeros (ids -1) and no gradient.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_TINY_TAIL = 2.0 ** -24   # least tail mass of the teacher in the reverse form
_TINY_REST = 2.0 ** -126  # least tail mass of the student whose logarithm is taken


def _case(name, op, rows, vocab, k, dtype="bf16", temperature=1.0, pass_="fwd", masked=0.0, pad=0, kl="forward",
          tail=True, ragged=False):
    return dict(name=name, op=op, rows=rows, vocab=vocab, k=k, dtype=dtype, temperature=temperature, masked=masked,
                kl=kl, tail=tail, ragged=ragged, pad=pad, **{"pass": pass_})


def listed():
    return [
        # one new token of a served sequence: the sampled token's log-prob and the usual 20 alternatives
        _case("top_one_token", "top", 1, 151936, 20),
        # a decode batch at a sampling temperature
        _case("top_decode_batch", "top", 48, 151936, 5, temperature=0.6),
        # a small vocabulary in fp32, ragged row count: many short rows
        _case("top_short_rows_fp32", "top", 1021, 32000, 8, dtype="fp32"),
        # odd vocabulary in a padded buffer (rows start off the 16-byte grid), prompt rows left out
        _case("top_odd_fp16", "top", 2003, 50257, 50, dtype="fp16", pad=6, masked=0.25),
        # the teacher's pass that makes distillation targets for a packed micro-batch
        _case("top_teacher", "top", 4096, 151936, 64),
        # the largest vocabulary at a temperature: two softmax sets per row
        _case("top_large_vocab", "top", 4096, 262144, 20, temperature=0.6),
        # training on the alternatives: gradients of log-prob, entropy and the top log-probs
        _case("top_train", "top", 2048, 151936, 32, pass_="train"),
        # the end of a micro-batch: few rows, autograd graph
        _case("distill_few_rows", "distill", 24, 151936, 20, pass_="train"),
        # validation loss of a student: forward only, lists cut by probability
        _case("distill_eval", "distill", 4096, 151936, 64, ragged=True, masked=0.1),
        # the training step of a packed micro-batch in one pass
        _case("distill_step", "distill", 8192, 151936, 64, pass_="fused"),
        # on-policy distillation (reverse KL) of a small fp32 student at a raised temperature
        _case("distill_reverse_fp32", "distill", 2048, 32000, 32, dtype="fp32", temperature=2.0, pass_="train",
              kl="reverse"),
        # the largest vocabulary, longest list, renormalised teacher, ordinary autograd graph
        _case("distill_large_vocab", "distill", 2048, 262144, 128, dtype="fp16", pass_="train", tail=False),
    ]


def draw(rng):
    op = rng.choice(["top", "distill"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = int(round(math.exp(rng.uniform(math.log(2048), math.log(262144)))))
    if rng.random() < 0.3:
        vocab = rng.choice([32000, 50257, 151936, 262144])
    most = min(8192, (1 << 30) // vocab // (2 if dtype == "fp32" else 1))
    rows = max(1, int(math.exp(rng.uniform(0.0, math.log(most)))))
    case = _case(None, op, rows, vocab, max(1, int(math.exp(rng.uniform(0.0, math.log(128.999))))), dtype=dtype,
                 temperature=rng.choice([1.0, 1.0, 0.6, round(rng.uniform(0.5, 2.5), 3)]),
                 pass_=rng.choice(["fwd", "train"] if op == "top" else ["fwd", "train", "fused"]),
                 masked=rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.6), 2)]),
                 pad=rng.choice([0, 0, rng.randint(1, 40)]))
    if op == "distill":
        case["kl"] = rng.choice(["forward", "forward", "reverse"])
        case["tail"] = case["kl"] == "reverse" or rng.random() < 0.6
        case["ragged"] = rng.random() < 0.4
    del case["name"]
    return case


def _kept_rows(case):
    return case["rows"] - int(case["rows"] * case["masked"])


def work(case):
    n, v, k, kept = case["rows"], case["vocab"], case["k"], _kept_rows(case)
    e = 4 if case["dtype"] == "fp32" else 2
    grads = case["pass"] != "fwd"
    nbytes = kept * v * e + (n * v * e if grads else 0) + (n if case["masked"] else 0)
    per_elem = (2 if case["op"] == "distill" else 4) + (4 if grads else 0)
    if case["op"] == "top":
        nbytes += n * (8 + 4 + 4 + 12 * k) + (n * (8 + 4 * k) if grads else 0)
    else:
        nbytes += n * (12 * k + 4) + (n * 4 if grads else 0)
    return {"bytes": nbytes, "flops": kept * v * per_elem}


# ------------------------------------------------------------------------------------ inputs
def _logit_slab(g, rows, vocab):
    """Logits as a language model gives them: a broad body and, on most rows, a few favoured tokens."""
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.5
    sharp = torch.rand(rows, 1, generator=g, device="cuda") * 14.0
    at = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
    fall = torch.tensor([1.0, 0.8, 0.6, 0.5], device="cuda")
    return x.scatter_add_(1, at, sharp * fall)


def prepare(case, seed):
    n, v, k, t = case["rows"], case["vocab"], case["k"], case["temperature"]
    dtype = _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    store = torch.empty(n, v + case["pad"], dtype=dtype, device="cuda")
    logits = store[:, :v]
    state = dict(case=case, logits=logits)
    # fp16 trains with a scaled loss: without it most gradients of a wide row are below its normal range
    scale = 1024.0 if dtype == torch.float16 else 1.0
    if case["op"] == "distill":
        ids = torch.empty(n, k, dtype=torch.int64, device="cuda")
        lps = torch.empty(n, k, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 28) // v)
    for lo in range(0, n, step):
        hi = min(n, lo + step)
        slab = _logit_slab(g, hi - lo, v)
        logits[lo:hi] = slab.to(dtype)
        if case["op"] == "distill":  # a teacher that agrees with the student on much, not on all
            z = (slab * 0.8 + torch.randn(hi - lo, v, generator=g, device="cuda") * 1.5) / t
            top = torch.topk(z, k, dim=1)
            ids[lo:hi] = top.indices
            lps[lo:hi] = top.values - torch.logsumexp(z, 1, keepdim=True)
    if case["op"] == "distill":
        if case["ragged"]:  # lists cut at a random length, as a cut by probability leaves them
            length = torch.randint(1, k + 1, (n, 1), generator=g, device="cuda")
            gone = torch.arange(k, device="cuda")[None] >= length
            ids[gone], lps[gone] = -1, -math.inf
        state["ids"], state["lps"] = ids, lps
        state["weights"] = torch.rand(n, generator=g, device="cuda") * (scale if scale > 1.0 else 1.0 / n)
    else:
        state["labels"] = torch.randint(0, v, (n,), generator=g, device="cuda")
        state["g_lp"] = torch.randn(n, generator=g, device="cuda") * scale
        state["g_ent"] = torch.randn(n, generator=g, device="cuda") * scale
        state["g_top"] = torch.randn(n, k, generator=g, device="cuda") * scale
    state["mask"] = None
    if case["masked"]:
        mask = torch.ones(n, dtype=torch.bool, device="cuda")
        order = torch.argsort(torch.rand(n, generator=g, device="cuda"))
        mask[order[: n - _kept_rows(case)]] = False
        state["mask"] = mask
    if case["pass"] == "train":
        logits.requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own_top(state) if state["case"]["op"] == "top" else _own_distill(state)
    with torch.no_grad():
        n, v = state["logits"].shape
        step = max(1, (1 << 28) // v)
        parts = [(_plain_top if state["case"]["op"] == "top" else _plain_distill)(state, lo, min(n, lo + step))
                 for lo in range(0, n, step)]
        if len(parts) == 1:
            return parts[0]
        return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _own_top(state):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    case = state["case"]
    lp, ent, top_lp, top_ids = top_logprobs_from_logits(state["logits"], state["labels"], case["k"],
                                                        temperature=case["temperature"], row_mask=state["mask"])
    out = dict(log_probs=lp, entropy=ent, top_log_probs=top_lp, top_ids=top_ids)
    if case["pass"] == "train":
        (out["grad_logits"],) = torch.autograd.grad([lp, ent, top_lp], [state["logits"]],
                                                    [state["g_lp"], state["g_ent"], state["g_top"]])
        for name in ("log_probs", "entropy", "top_log_probs"):
            out[name] = out[name].detach()
    return out


def _own_distill(state):
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    case = state["case"]
    how = dict(temperature=case["temperature"], kl=case["kl"], tail=case["tail"], row_mask=state["mask"])
    if case["pass"] == "fused":
        loss, grad = fused_distill_kl_fwd_bwd(state["logits"], state["ids"], state["lps"], state["weights"],
                                              inplace=False, **how)
        return dict(loss=loss, grad_logits=grad)
    loss = distill_kl_from_logits(state["logits"], state["ids"], state["lps"], **how)
    if case["pass"] == "fwd":
        return dict(loss=loss)
    (grad,) = torch.autograd.grad([loss], [state["logits"]], [state["weights"]])
    return dict(loss=loss.detach(), grad_logits=grad)


def _plain_top(state, lo, hi):
    case = state["case"]
    t, k = case["temperature"], case["k"]
    raw = state["logits"][lo:hi].detach()
    x = raw.float()
    v = x.shape[1]
    labels = state["labels"][lo:hi]
    m = x.amax(1, keepdim=True)
    e1 = (x - m).exp()
    s1 = e1.sum(1, keepdim=True)
    ex = (e1 * x).sum(1, keepdim=True) / s1
    entropy = (m + s1.log() - ex)[:, 0]
    if t == 1.0:
        z, et, st, lse = x, e1, s1, m + s1.log()
    else:
        z = x / t
        et = (z - m / t).exp()
        st = et.sum(1, keepdim=True)
        lse = m / t + st.log()
    lp = (z.gather(1, labels[:, None]) - lse)[:, 0]
    # the k largest, equal logits by ascending id: one whole-number key holds both, so none are equal
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (key << 32) + (v - 1 - torch.arange(v, device=x.device))
    top_ids = v - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    del bits, key
    top_lp = z.gather(1, top_ids) - lse
    keep = None if state["mask"] is None else state["mask"][lo:hi]
    out = {}
    if case["pass"] == "train":
        g_lp, g_ent, g_top = state["g_lp"][lo:hi], state["g_ent"][lo:hi], state["g_top"][lo:hi]
        grad = (et / st) * (-(g_lp + g_top.sum(1)) / t)[:, None]
        grad += (e1 / s1) * (ex - x) * g_ent[:, None]
        grad.scatter_add_(1, labels[:, None], (g_lp / t)[:, None])
        grad.scatter_add_(1, top_ids, g_top / t)
        if keep is not None:
            grad[~keep] = 0.0
        out["grad_logits"] = grad.to(raw.dtype)
    if keep is not None:
        lp, entropy = lp * keep, entropy * keep
        top_lp = torch.where(keep[:, None], top_lp, torch.zeros_like(top_lp))
        top_ids = torch.where(keep[:, None], top_ids, torch.full_like(top_ids, -1))
    out.update(log_probs=lp, entropy=entropy, top_log_probs=top_lp, top_ids=top_ids)
    return out


def _plain_distill(state, lo, hi):
    case = state["case"]
    t_, raw = case["temperature"], state["logits"][lo:hi].detach()
    ids, tlp = state["ids"][lo:hi], state["lps"][lo:hi].double()
    on = ids >= 0
    at = ids.clamp(min=0)
    z = raw.float() / t_
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    zk = z.gather(1, at)
    ek = torch.where(on, (zk - m).exp(), torch.zeros_like(zk))
    # the mass outside the list is summed by itself: 1 - sum q would lose it for a sure student
    rest = e.scatter(1, torch.where(on, at, ids.clamp(min=0)[:, :1]), 0.0).sum(1, keepdim=True)
    total = rest + ek.sum(1, keepdim=True)
    lq = (zk - m - total.log()).double()
    q = e / total
    qk = torch.where(on, lq.exp(), torch.zeros_like(lq))
    s = (rest / total).double().clamp(min=_TINY_REST)
    p = torch.where(on, tlp.exp(), torch.zeros_like(tlp))
    safe_tlp = torch.where(on, tlp, torch.zeros_like(tlp))
    if case["kl"] == "reverse":
        t = (1.0 - p.sum(1, keepdim=True)).clamp(min=_TINY_TAIL)
        ratio = torch.where(on, lq - safe_tlp, torch.zeros_like(lq))
        tail = s.log() - t.log()
        loss = (qk * ratio).sum(1, keepdim=True) + s * tail
        listed, other = qk * (ratio - loss), tail - loss
    elif case["tail"]:
        t = (1.0 - p.sum(1, keepdim=True)).clamp(min=0.0)
        loss = (p * (safe_tlp - torch.where(on, lq, torch.zeros_like(lq)))).sum(1, keepdim=True)
        loss = loss + torch.where(t > 0, t * (t.clamp(min=1e-300).log() - s.log()), torch.zeros_like(t))
        mass = p.sum(1, keepdim=True) + t
        listed, other = mass * qk - p, mass - t / s
    else:
        total_p = p.sum(1, keepdim=True)
        w = p / total_p
        loss = (w * (safe_tlp - total_p.log() - torch.where(on, lq, torch.zeros_like(lq)))).sum(1, keepdim=True)
        listed, other = qk - w, torch.ones_like(loss)
    keep = None if state["mask"] is None else state["mask"][lo:hi]
    out = dict(loss=loss[:, 0].float())
    if keep is not None:
        out["loss"] = torch.where(keep, out["loss"], torch.zeros_like(out["loss"]))
    if case["pass"] != "fwd":
        w_row = state["weights"][lo:hi, None]
        grad = q * (other.float() * w_row / t_)
        value = listed.float() * w_row / t_
        # absent entries write what already stands at the row's first listed id
        first = at[:, :1]
        grad.scatter_(1, torch.where(on, at, first), torch.where(on, value, value[:, :1]))
        if keep is not None:
            grad[~keep] = 0.0
        out["grad_logits"] = grad.to(raw.dtype)
    return out


# ------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    logits = state["logits"].detach()
    n, v = logits.shape
    step = max(1, (1 << 27) // v)
    parts = []
    for lo in range(0, n, step):
        rows = slice(lo, min(n, lo + step))
        parts.append((_exact_top if case["op"] == "top" else _exact_distill)(case, state, logits[rows].double(), rows))
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    if state["mask"] is not None:
        for name, value in out.items():
            value[~state["mask"]] = -1 if name == "top_ids" else 0
    return out


def _exact_top(case, state, x, rows):
    k, temp = case["k"], case["temperature"]
    label = state["labels"][rows].view(-1, 1)
    log_p = torch.log_softmax(x / temp, dim=1)
    log_u = torch.log_softmax(x, dim=1)
    entropy = -(log_u.exp() * log_u).sum(1)
    # membership from the k-th value: all above it, and the first of those equal to it
    kth = torch.kthvalue(x, x.shape[1] - k + 1, dim=1, keepdim=True).values
    above = x > kth
    level = x == kth
    room = k - above.sum(1, keepdim=True)
    member = above | (level & (level.cumsum(1) <= room))
    ids = member.nonzero()[:, 1].view(-1, k)  # ascending ids in every row
    order = torch.sort(x.gather(1, ids), dim=1, descending=True, stable=True).indices
    ids = ids.gather(1, order)
    out = {}
    if case["pass"] == "train":
        g_lp, g_ent = state["g_lp"][rows].double().view(-1, 1), state["g_ent"][rows].double().view(-1, 1)
        g_top = state["g_top"][rows].double()
        pick = torch.zeros_like(x).scatter_add_(1, label, g_lp).scatter_add_(1, ids, g_top)
        d_z = pick - log_p.exp() * pick.sum(1, keepdim=True)
        out["grad_logits"] = d_z / temp - g_ent * log_u.exp() * (log_u + entropy[:, None])
    out.update(log_probs=log_p.gather(1, label)[:, 0], entropy=entropy, top_log_probs=log_p.gather(1, ids), top_ids=ids)
    return out


def _exact_distill(case, state, x, rows):
    temp = case["temperature"]
    ids, lt = state["ids"][rows], state["lps"][rows].double()
    n, v = x.shape
    row, col = (ids >= 0).nonzero(as_tuple=True)
    spot = ids[row, col]
    on = torch.zeros(n, v, dtype=torch.bool, device=x.device)
    on[row, spot] = True
    log_t = torch.full((n, v), -math.inf, dtype=torch.float64, device=x.device)
    log_t[row, spot] = lt[row, col]
    log_q = torch.log_softmax(x / temp, dim=1)
    q, p = log_q.exp(), log_t.exp()
    s = torch.where(on, 0.0, q).sum(1, keepdim=True).clamp(min=_TINY_REST)
    mass = p.sum(1, keepdim=True)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    if case["kl"] == "reverse":
        t = (1 - mass).clamp(min=_TINY_TAIL)
        r = torch.where(on, log_q - torch.where(on, log_t, zero), torch.log(s / t))
        loss = (q * r).sum(1)
        d_z = q * (r - loss[:, None])
    elif case["tail"]:
        t = (1 - mass).clamp(min=0)
        loss = torch.where(on, p * (torch.where(on, log_t, zero) - log_q), zero).sum(1)
        loss = loss + torch.xlogy(t, t)[:, 0] - (t * torch.log(s))[:, 0]
        d_z = (mass + t) * q - torch.where(on, p, q * t / s)
    else:
        w = p / mass
        loss = torch.where(on, w * (torch.where(on, log_t, zero) - mass.log() - log_q), zero).sum(1)
        d_z = q - w
    out = dict(loss=loss)
    if case["pass"] != "fwd":
        out["grad_logits"] = d_z * state["weights"][rows].double().view(-1, 1) / temp
    return out
