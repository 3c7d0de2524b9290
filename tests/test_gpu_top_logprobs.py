"""top_logprobs_from_logits against the definition in float64: ids exactly, values and gradients
inside bounds that follow the arithmetic (derived below, before the first run).

Bounds. u = 2^-24. A term exp2(x c - M) carries the rounding of its argument (|x| c + |M| at most
2 X c with X = max |x|, c = log2(e) / T, times u, times ln 2 as a relative error), one ulp of the
exponential and the rounding of c; a sum adds at most one rounding per term of its accumulator (a
row has 4 accumulators in each of 256 lanes, and about 12 further additions). So the sums are
relatively within rel = (V / 1024 + 3 X c + 24) u, and so are, absolutely, the log-sum-exps; a stored
statistic is rounded once more (|lse| u)."""
import math

import pytest
import torch

from oracle import vocab_lists as ov

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FLOOR = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}  # half of the least subnormal, flushed exponentials


def _rel(x64, temperature):
    finite = x64[torch.isfinite(x64) & (x64.abs() < 1e30)]
    big = float(finite.abs().max()) if finite.numel() else 0.0
    c = math.log2(math.e) * max(1.0, 1.0 / temperature)
    return (x64.shape[-1] / 1024 + 3 * big * c + 24) * U, big


def _logits(rows, vocab, dtype, seed, pad=0, offset=0, scale=2.5, spike=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    if spike:
        x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += 12.0 * torch.rand(rows, generator=g)
    store = torch.empty(rows * (vocab + pad) + offset, dtype=TYPES[dtype], device="cuda")
    view = store[offset:].view(rows, vocab + pad)[:, :vocab]
    view.copy_(x.to(TYPES[dtype]))
    labels = torch.randint(0, vocab, (rows,), generator=g)
    return view, labels, g


def _check_forward(view, labels, k, temperature, out, row_mask=None):
    lp, ent, top, ids = (None if t is None else t.cpu() for t in out)
    x64 = view.detach().double().cpu()
    ref_top, ref_ids = ov.top_logprobs(x64, k, temperature, row_mask)
    assert ids.dtype == torch.int64 and torch.equal(ids, ref_ids)
    rel, big = _rel(x64, temperature)
    assert ((top.double() - ref_top).abs() <= rel + 2 * U * (ref_top.abs() + big / temperature)).all()
    keep = torch.ones(x64.shape[0], dtype=torch.bool) if row_mask is None else row_mask.cpu() != 0
    if lp is not None:
        ref = torch.log_softmax(x64 / temperature, -1).gather(-1, labels[:, None])[:, 0] * keep
        assert ((lp.double() - ref).abs() <= rel + 2 * U * (ref.abs() + big / temperature)).all()
    if ent is not None:
        lu = torch.log_softmax(x64, -1)
        ref = -(lu.exp() * lu).sum(-1) * keep
        # lse - E[x]: E[x] is a quotient of two sums, each within rel, of terms of size X
        assert ((ent.double() - ref).abs() <= rel + 2 * rel * big + 2 * U * (ref.abs() + 2 * big + 12)).all()


@pytest.mark.parametrize("rows,vocab,k,dtype,temperature,pad,offset", [
    (1, 1, 1, "fp32", 1.0, 0, 0),
    (3, 2, 2, "bf16", 0.5, 0, 1),
    (5, 7, 3, "fp16", 1.0, 1, 3),
    (4, 128, 128, "bf16", 1.0, 0, 0),
    (4, 129, 128, "fp32", 2.0, 3, 1),
    (17, 1000, 20, "bf16", 0.7, 0, 0),
    (9, 2048, 64, "fp32", 1.0, 0, 0),
    (300, 5003, 50, "fp16", 1.3, 5, 7),
    (260, 32000, 8, "fp32", 1.0, 0, 0),
    (7, 50257, 128, "bf16", 0.6, 2, 1),
    (3, 151936, 1, "bf16", 1.0, 0, 0),
    (1, 151937, 128, "bf16", 1.0, 0, 5),
    (511, 20011, 30, "fp32", 0.9, 0, 0),
    (512, 20011, 30, "bf16", 1.0, 0, 0),
    (2, 524309, 128, "fp32", 1.0, 0, 1),
    (65, 151936, 20, "bf16", 1.0, 0, 0),
    (2, 262144, 100, "fp16", 0.6, 0, 0),
    (270, 70001, 5, "bf16", 1.0, 0, 0),
    (1, 600011, 33, "fp32", 1.0, 0, 2),
])
def test_forward_and_gradients(cuda, rows, vocab, k, dtype, temperature, pad, offset):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    view, labels, g = _logits(rows, vocab, dtype, 11 * rows + vocab, pad, offset)
    view = view.detach().requires_grad_(True)
    out = top_logprobs_from_logits(view, labels.cuda(), k, temperature)
    _check_forward(view, labels, k, temperature, [t.detach() for t in out])
    few = list(range(rows)) if rows * vocab <= 2_000_000 else [0, rows - 1]
    g_lp, g_ent, g_top = (torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g))
    (grad,) = torch.autograd.grad(out[:3], [view], [t.cuda() for t in (g_lp, g_ent, g_top)])
    _check_grad(view, grad, labels, out[3].cpu(), g_lp, g_ent, g_top, temperature, few)


def _check_grad(view, grad, labels, ids, g_lp, g_ent, g_top, temperature, few):
    x64 = view.detach()[few].double().cpu().requires_grad_(True)
    pick = lambda t: None if t is None else t[few].double()  # noqa: E731
    total = ov.top_objective(x64, labels[few], ids[few], pick(g_lp), pick(g_ent), pick(g_top), temperature)
    (ref,) = torch.autograd.grad(total, [x64])
    x64 = x64.detach()
    rel, big = _rel(x64, temperature)
    lse = torch.logsumexp(x64 / temperature, -1, keepdim=True).abs() + torch.logsumexp(x64, -1, keepdim=True).abs()
    slack = 2 * rel + 4 * U * lse  # relative error of a softmax weight: its log-sum-exp (stored in fp32) and its exponent
    none = torch.zeros(len(few), dtype=torch.float64)
    g_all = (none if g_lp is None else pick(g_lp)) + (none if g_top is None else pick(g_top).sum(-1))
    a_all = (none if g_lp is None else pick(g_lp).abs()) + (none if g_top is None else pick(g_top).abs().sum(-1))
    # 140 u: the fp32 sum of up to 128 upstream gradients
    bound = torch.softmax(x64 / temperature, -1) * (g_all.abs().view(-1, 1) * slack + a_all.view(-1, 1) * 140 * U) / temperature
    if g_ent is not None:
        lu = torch.log_softmax(x64, -1)
        ex = (lu.exp() * x64).sum(-1, keepdim=True)
        bound = bound + lu.exp() * pick(g_ent).abs().view(-1, 1) * ((ex - x64).abs() * slack + (2 * rel + 4 * U) * (big + 1))
    # listed entries add their own terms: three fp32 roundings of values up to |g| / T
    bound = bound + 4 * U * (ref.abs() + a_all.view(-1, 1) / temperature * (ref.abs() > 0))
    half = torch.finfo(grad.dtype).eps / 2
    err = (grad[few].double().cpu() - ref).abs()
    assert (err <= half * (ref.abs() + bound) + bound + FLOOR[grad.dtype]).all(), (err - half * ref.abs() - bound).max()


@pytest.mark.parametrize("which", ["logprob", "entropy", "top", "logprob+top", "entropy+top"])
@pytest.mark.parametrize("inplace", [False, True])
def test_gradients_of_each_output_alone_and_in_place(cuda, which, inplace):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    rows, vocab, k, t = 6, 3001, 10, 0.8
    view, labels, g = _logits(rows, vocab, "bf16", 5)
    keep = view.clone()
    view = view.detach().requires_grad_(True)
    lp, ent, top, ids = top_logprobs_from_logits(view, labels.cuda(), k, t, inplace_backward=inplace,
                                                 return_entropy="entropy" in which)
    g_lp = torch.randn(rows, generator=g) if "logprob" in which else None
    g_ent = torch.randn(rows, generator=g) if "entropy" in which else None
    g_top = torch.randn(rows, k, generator=g) if "top" in which else None
    pairs = [(o, q.cuda()) for o, q in ((lp, g_lp), (ent, g_ent), (top, g_top)) if q is not None]
    (grad,) = torch.autograd.grad([p[0] for p in pairs], [view], [p[1] for p in pairs])
    assert (grad.data_ptr() == view.data_ptr()) == inplace
    _check_grad(keep, grad, labels, ids.cpu(), g_lp, g_ent, g_top, t, list(range(rows)))


def test_gradient_against_differences(cuda):
    """Central differences of the float64 objective around the fp32 logits."""
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    rows, vocab, k, t = 3, 40, 4, 1.5
    view, labels, g = _logits(rows, vocab, "fp32", 8, spike=False, scale=1.0)
    view = view.detach().requires_grad_(True)
    out = top_logprobs_from_logits(view, labels.cuda(), k, t)
    gs = [torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g)]
    (grad,) = torch.autograd.grad(out[:3], [view], [q.cuda() for q in gs])
    x, ids = view.detach().double().cpu(), out[3].cpu()
    f = lambda y: ov.top_objective(y, labels, ids, *[q.double() for q in gs], t).item()  # noqa: E731
    h = 1e-5
    for i, j in [(0, int(ids[0, 0])), (0, int(labels[0])), (1, 3), (2, int(ids[2, 3])), (2, 39)]:
        d = torch.zeros_like(x)
        d[i, j] = h
        # truncation h^2 times third derivatives of order 10, rounding 1e-14 / h
        assert abs((f(x + d) - f(x - d)) / (2 * h) - grad[i, j].item()) <= 1e-8 + 1e-5 * (1 + abs(grad[i, j].item()))


def _rows_that_go_wrong(vocab, dtype):
    """Named rows where a selection by threshold, a running maximum or a tie rule can fail."""
    g = torch.Generator().manual_seed(3)
    body = torch.randn(vocab, generator=g) * 2
    low = torch.finfo(TYPES[dtype]).min
    rows = {
        "equal": torch.full((vocab,), 1.5),
        "ascending": torch.sort(body).values,
        "descending": torch.sort(body, descending=True).values,
        "two levels": (body > 1.0).float(),
        "negative zeros": torch.where(torch.arange(vocab) % 3 == 0, -0.0, 0.0),
        "few allowed": torch.where(torch.arange(vocab) % (vocab // 5) == 3, body, torch.tensor(low)),
        "one above all": torch.cat([body[:-1], torch.tensor([60.0])]),
        "far spike": torch.cat([torch.full((vocab - 1,), -300.0), torch.tensor([300.0])]),
        "all lowest": torch.full((vocab,), low),
        "sawtooth": (torch.arange(vocab) % 97).float() / 8,
        "large negative": body - 20000.0,
    }
    return list(rows), torch.stack(list(rows.values())).to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab,k", [(700, 128), (5000, 20), (40009, 7), (33000, 128)])
def test_rows_with_equal_sorted_and_extreme_logits(cuda, dtype, vocab, k):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    names, x = _rows_that_go_wrong(vocab, dtype)
    labels = torch.arange(len(names)) * 31 % vocab
    lp, ent, top, ids = top_logprobs_from_logits(x.cuda(), labels.cuda(), k)
    ref_top, ref_ids = ov.top_logprobs(x.double(), k)
    for i, name in enumerate(names):
        assert torch.equal(ids[i].cpu(), ref_ids[i]), name
    rel, big = _rel(x.double(), 1.0)
    big = torch.where(x.abs().double() < 1e30, x.abs().double(), torch.zeros(())).amax(1, keepdim=True)
    rel = (vocab / 1024 + 5 * big + 24) * U
    ok = (top.cpu().double() - ref_top).abs() <= rel + 2 * U * (ref_top.abs() + big)
    same = top.cpu().double() == ref_top.float().double()
    assert (ok | same).all(), [names[i] for i in (~(ok | same)).any(1).nonzero()[:, 0]]
    ref_lp = torch.log_softmax(x.double(), -1).gather(-1, labels[:, None])
    assert (((lp.cpu().double()[:, None] - ref_lp).abs() <= rel + 2 * U * (ref_lp.abs() + big)) | (lp.cpu()[:, None] == ref_lp.float())).all()
    lu = torch.log_softmax(x.double(), -1)
    ref_ent = -(lu.exp() * lu).sum(-1)
    # E[x] is a quotient of two sums within rel of terms of size big; a logit of weight 0 adds nothing
    close = (ent.cpu().double() - ref_ent).abs() <= rel[:, 0] * (1 + 2 * big[:, 0]) + 4 * U * (ref_ent.abs() + 12)
    assert close.all(), [names[i] for i in (~close).nonzero()[:, 0]]


@pytest.mark.parametrize("vocab", [300, 20011])
def test_infinite_and_nan_logits(cuda, vocab):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    g = torch.Generator().manual_seed(2)
    x = torch.randn(6, vocab, generator=g)
    x[0, : vocab - 4] = -math.inf                 # fewer allowed tokens than k
    x[1, ::2] = -math.inf
    x[2, 17] = math.nan
    x[3, 5], x[3, vocab - 1] = math.nan, -math.nan
    x[4, 250] = math.inf
    x[5] = -math.inf
    lp, _, top, ids = top_logprobs_from_logits(x.cuda(), torch.zeros(6, dtype=torch.long).cuda(), 10, return_entropy=False)
    ref_top, ref_ids = ov.top_logprobs(x.double(), 10)
    assert torch.equal(ids.cpu(), ref_ids)
    top = top.cpu().double()
    assert top[2:4].isnan().all() and top[5].isnan().all()
    assert top[4, 0].isnan() and (top[4, 1:] == -math.inf).all()  # x - lse with lse = +inf
    for r in (0, 1):
        fin = torch.isfinite(ref_top[r])
        assert torch.equal(torch.isfinite(top[r]), fin) and (top[r][~fin] == -math.inf).all()
        assert ((top[r] - ref_top[r])[fin].abs() <= 64 * U * (1 + ref_top[r][fin].abs())).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_gradients_of_masked_vocabularies(cuda, dtype):
    """Logits at the lowest value of their type, some or all of a row: gradients stay those of the
    definition (zero where the softmax is zero), whatever the size of the entropy's upstream gradient."""
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    vocab, k = 2000, 8
    g = torch.Generator().manual_seed(6)
    x = torch.randn(3, vocab, generator=g)
    x[0, 20:] = torch.finfo(TYPES[dtype]).min
    x[2] = torch.finfo(TYPES[dtype]).min
    x = x.to(TYPES[dtype])
    labels = torch.tensor([3, 5, 7])
    view = x.cuda().requires_grad_(True)
    out = top_logprobs_from_logits(view, labels.cuda(), k)
    gs = [torch.tensor([1.0, -2.0, 0.5]), torch.tensor([7.0, -3.0, 0.0]), torch.randn(3, k, generator=g)]
    (grad,) = torch.autograd.grad(out[:3], [view], [t.cuda() for t in gs])
    assert grad.isfinite().all() and (grad[0, 20:] == 0).all()
    small = x.double().clone()
    small[2] = 0.0  # a uniform row
    _check_grad(small[[1, 2]].cuda().to(TYPES[dtype]), grad[[1, 2]], labels[[1, 2]], out[3].cpu()[[1, 2]],
                gs[0][[1, 2]], gs[1][[1, 2]], gs[2][[1, 2]], 1.0, [0, 1])
    _check_grad(x[:1, :20].cuda(), grad[:1, :20], labels[:1], out[3].cpu()[:1], gs[0][:1], gs[1][:1], gs[2][:1], 1.0, [0])


@pytest.mark.parametrize("vocab", [4099, 40009])
def test_masked_rows_and_labels_outside(cuda, vocab):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    view, labels, g = _logits(40, vocab, "bf16", 21)
    view = view.detach().requires_grad_(True)
    mask = torch.rand(40, generator=g) < 0.5
    mask[0], mask[1], mask[2] = True, True, False
    labels[0], labels[1] = -100, vocab
    lp, ent, top, ids = top_logprobs_from_logits(view, labels.cuda().int(), 6, row_mask=mask.cuda())
    assert lp[0].item() == 0.0 and math.isnan(lp[1].item())
    inside = labels.clone()
    inside[:2] = 0
    ok = mask.clone()
    ok[:2] = False
    out = [t.detach().clone() for t in (lp, ent, top, ids)]
    for t, fill in zip(out, (0, 0, 0, -1)):
        t[~ok.cuda()] = fill
    _check_forward(view, inside, 6, 1.0, out, row_mask=ok)
    g_top = torch.randn(40, 6, generator=g)
    (grad,) = torch.autograd.grad([top], [view], [g_top.cuda()])
    assert (grad[~mask.cuda()] == 0).all()
    _check_grad(view, grad, inside, ids.cpu(), None, None, g_top, 1.0, mask.nonzero()[:, 0].tolist())


def test_shapes_strides_and_absent_outputs(cuda):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    x = torch.randn(2, 3, 515, device="cuda")
    labels = torch.randint(0, 515, (2, 3), device="cuda")
    lp, ent, top, ids = top_logprobs_from_logits(x, labels, 4, 0.9)
    assert lp.shape == ent.shape == (2, 3) and top.shape == ids.shape == (2, 3, 4)
    turned = x.permute(0, 2, 1).contiguous().permute(0, 2, 1)  # vocabulary not the fastest axis
    for a, b in zip(top_logprobs_from_logits(turned, labels, 4, 0.9), (lp, ent, top, ids)):
        assert torch.equal(a, b)
    none_lp, none_ent, top2, ids2 = top_logprobs_from_logits(x, None, 4, 0.9, return_entropy=False)
    assert none_lp is None and none_ent is None and torch.equal(ids2, ids)
    assert ((top2 - top).abs() <= 64 * U * (1 + top.abs())).all()
    empty = top_logprobs_from_logits(x[:0], labels[:0], 4)
    assert [tuple(t.shape) for t in empty] == [(0, 3), (0, 3), (0, 3, 4), (0, 3, 4)]


@pytest.mark.parametrize("rows,vocab,k", [(1, 151936, 20), (7, 151936, 128), (300, 50257, 20), (64, 262144, 64)])
def test_cut_rows_merged_in_one_launch_or_two_give_the_same_bits(cuda, rows, vocab, k):
    """The records of a cut row are merged by the workgroup that finishes it (tickets) or by a second
    launch; repeated calls over one ticket array, with masked rows, a row of equal logits (more
    candidates than fit) and one with a NaN among them."""
    from openrlhf_amd import _lib

    view, labels, g = _logits(rows, vocab, "bf16", rows + k)
    if rows > 3:
        view[0] = 0.25
        view[1, 77] = math.nan
        view[2, : vocab - 9] = -math.inf
    lab = labels.cuda()
    mask = torch.ones(rows, dtype=torch.uint8, device="cuda")
    mask[rows // 2 : rows // 2 + rows // 5] = 0
    lib = _lib.load()
    nbytes = lib.orlhf_top_logprobs_workspace_bytes(_lib.BF16, rows, vocab, k)
    assert nbytes > 0
    tickets = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def once(tick):
        ws = torch.randint(0, 255, (nbytes,), dtype=torch.uint8, device="cuda")
        lp, ent = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
        top, stats = torch.full((rows, k), 7.0, device="cuda"), torch.full((rows, 4), 7.0, device="cuda")
        ids = torch.full((rows, k), 7, device="cuda")
        _lib.call("orlhf_top_logprobs_fwd", view.data_ptr(), _lib.BF16, rows, vocab, vocab, lab.data_ptr(), 0.8, k,
                  lp.data_ptr(), ent.data_ptr(), top.data_ptr(), ids.data_ptr(), stats.data_ptr(), mask.data_ptr(),
                  ws.data_ptr(), nbytes, None if tick is None else tick.data_ptr(), _lib.stream_of(view.device))
        return [t.view(torch.int32) if t.dtype == torch.float32 else t for t in (lp, ent, top, ids, stats)]

    want = once(None)
    for _ in range(20):
        got = once(tickets)
        assert int(tickets.abs().sum()) == 0
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [2, 300])
def test_repeats_other_stream_and_replayed_graph_give_the_same_bits(cuda, rows):
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    view, labels, _ = _logits(rows, 50257, "bf16", 4)
    lab = labels.cuda()
    want = top_logprobs_from_logits(view, lab, 12, 0.7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = top_logprobs_from_logits(view, lab, 12, 0.7)
    torch.cuda.current_stream().wait_stream(side)
    static = view.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = top_logprobs_from_logits(static, lab, 12, 0.7)
    other = static.flip(1).contiguous()
    want_other = top_logprobs_from_logits(other, lab, 12, 0.7)
    for a, b in zip(again, want):
        assert torch.equal(a, b)
    for source, expect in ((other, want_other), (view, want), (other, want_other)):
        static.copy_(source)
        graph.replay()
        top_logprobs_from_logits(view, lab, 3)  # eager work between the replays
        torch.cuda.synchronize()
        for a, b in zip(captured, expect):
            assert torch.equal(a, b)


@pytest.mark.parametrize("vocab", [4099, 40009])
@pytest.mark.parametrize("temperature", [1.0, 0.8])
def test_an_ignored_label_has_no_gradient(cuda, vocab, temperature):
    """Label -100: the log-prob is the constant 0, so its upstream gradient reaches no logit; the entropy's
    and the alternatives' do. The same row with a label inside and upstream gradient 0 gives the same bits."""
    from openrlhf_amd.models.utils import top_logprobs_from_logits

    view, labels, g = _logits(6, vocab, "fp32", 12)
    labels[1] = labels[4] = -100
    at = labels == -100
    g_lp, g_ent, g_top = torch.randn(6, generator=g) + 3.0, torch.randn(6, generator=g), torch.randn(6, 5, generator=g)
    zeroed, inside = g_lp.masked_fill(at, 0.0), labels.masked_fill(at, 7)
    for use in ((1, 0, 0), (1, 1, 0), (1, 0, 1), (1, 1, 1)):
        grads = []
        for lab, glp in ((labels, g_lp), (inside, zeroed)):
            leaf = view.detach().requires_grad_(True)
            lp, ent, top, ids = top_logprobs_from_logits(leaf, lab.cuda(), 5, temperature, return_entropy=bool(use[1]))
            pairs = [(o, q.cuda()) for o, q, on in zip((lp, ent, top), (glp, g_ent, g_top), use) if on]
            grads.append(torch.autograd.grad([p[0] for p in pairs], [leaf], [p[1] for p in pairs])[0])
            assert ((lp == 0) == (lab == -100).cuda()).all()
        assert torch.equal(grads[0], grads[1])
        if not use[1] and not use[2]:
            assert (grads[0][at.cuda()] == 0).all() and (grads[0][~at.cuda()] != 0).any(1).all()
    _check_grad(view, grads[0], inside, ids.cpu(), zeroed, g_ent, g_top, temperature, range(6))
