"""distill_kl_from_logits and fused_distill_kl_fwd_bwd against the definition in float64 (a Python sum
over outcomes per row, differentiated by autograd), and the pair of operators as they are used.

Bounds, u = 2^-24. The student's sum outside the list is relatively within rel = (V / 1024 + 3 X c + 24) u
of the exact one (its terms carry the rounding of their exponents, of which X = max |x| and
c = log2(e) / T set the size, and its accumulators one rounding per term); everything after it runs in
fp64. The loss depends on it through log s and the log-sum-exp, with derivatives of at most 2 (forward)
or 2 + |log-ratios| (reverse), and is rounded once."""
import math

import pytest
import torch

from oracle import vocab_lists as ov

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FLOOR = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}
FORMS = [("forward", True), ("forward", False), ("reverse", True)]


def _case(rows, vocab, k, dtype, seed, pad=0, offset=0, sharp=14.0, ragged=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 2
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += sharp * torch.rand(rows, generator=g)
    store = torch.empty(rows * (vocab + pad) + offset, dtype=TYPES[dtype], device="cuda")
    view = store[offset:].view(rows, vocab + pad)[:, :vocab]
    view.copy_(x.to(TYPES[dtype]))
    teacher = x * 0.8 + torch.randn(rows, vocab, generator=g)
    top = torch.topk(torch.log_softmax(teacher.double(), -1), k, dim=1)
    ids, lps = top.indices, top.values.float()
    if ragged:
        gone = torch.arange(k)[None] >= torch.randint(0, k + 1, (rows, 1), generator=g)
        ids[gone] = -1
        lps[gone & (torch.rand(rows, k, generator=g) < 0.5)] = -math.inf
    return view, ids, lps, g


def _reference(view, ids, lps, temperature, form, rows, teacher_temperature=1.0):
    out = []
    for r in rows:
        x = view[r].detach().double().cpu().requires_grad_(True)
        loss = ov.distill_kl_row(x, ids[r], lps[r].double(), temperature, teacher_temperature, *form)
        (grad,) = torch.autograd.grad(loss, [x])
        out.append((loss.item(), grad, x.detach()))
    return out


def _check(view, ids, lps, temperature, form, loss, grad=None, weight=None, rows=None, teacher_temperature=1.0):
    rows = range(view.shape[0]) if rows is None else rows
    c = math.log2(math.e) / temperature
    for r, (want, d, x) in zip(rows, _reference(view, ids, lps, temperature, form, rows, teacher_temperature)):
        fin = x[x.abs() < 1e30]
        big = fin.abs().max().item()
        rel = (x.numel() / 1024 + 3 * big * c + 24) * U
        lt = lps[r][(ids[r] >= 0) & (lps[r] > -math.inf)].double().abs()
        ratios = 2 + (lt.max().item() if lt.numel() else 0.0) + 2 * big / temperature if form[0] == "reverse" else 2.0
        got = loss[r].item()
        assert abs(got - want) <= ratios * rel + 2 * U * abs(want), (r, got, want)
        if grad is not None:
            w = weight[r].item()
            lq = torch.log_softmax(x / temperature, -1)
            q = lq.exp()
            # d / d(log s), d / d(lse) of the coefficient of q: |d| itself, and t / s in the forward form with
            # the tail; a listed entry is a difference of terms up to q and p, rounded in fp32
            slack = 2 * rel + 4 * U * (lq.abs().clamp(max=100) + 4)
            listed = torch.zeros_like(q)
            on = (ids[r] >= 0) & (lps[r] > -math.inf)
            listed[ids[r][on]] = lps[r][on].double().exp()
            bound = (d.abs() * temperature + q * ratios) * slack / temperature + 4 * U * listed / temperature
            if form == ("forward", True) and on.any():
                outside = (listed == 0)
                s = q[outside].sum().clamp(min=2.0 ** -126)
                t = max(0.0, 1.0 - listed.sum().item())
                bound = bound + (t / s) * q * outside * 4 * rel / temperature
            bound = bound * abs(w)
            half = torch.finfo(grad.dtype).eps / 2
            err = (grad[r].double().cpu() - w * d).abs()
            assert (err <= half * (abs(w) * d.abs() + bound) + bound + FLOOR[grad.dtype]).all(), (r, (err - bound).max())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,vocab,k,dtype,temperature,pad,offset,ragged", [
    (1, 1, 1, "fp32", 1.0, 0, 0, False),
    (3, 2, 1, "bf16", 0.5, 0, 1, False),
    (4, 9, 9, "fp32", 1.0, 0, 0, False),
    (5, 131, 128, "fp16", 1.0, 1, 3, True),
    (8, 1000, 20, "bf16", 0.7, 0, 0, True),
    (6, 5003, 65, "fp32", 2.0, 5, 3, True),
    (3, 32000, 1, "fp16", 1.0, 0, 0, False),
    (3, 50257, 128, "bf16", 1.5, 6, 1, True),
    (2, 151936, 64, "bf16", 1.0, 0, 0, False),
    (1, 262144, 50, "fp32", 1.0, 0, 0, True),
    (1, 520192, 20, "fp16", 0.8, 0, 0, False),
    (514, 4099, 7, "bf16", 1.0, 0, 0, True),
    (700, 151936, 64, "bf16", 1.0, 0, 0, False),
    (300, 262144, 100, "fp16", 0.7, 0, 0, True),
    (530, 50257, 128, "fp32", 1.0, 6, 3, True),
    (1031, 33, 33, "fp32", 1.3, 3, 1, True),
    (260, 80001, 11, "fp32", 2.0, 0, 0, False),
    (257, 520192, 20, "bf16", 1.0, 0, 0, True),
])
def test_loss_and_gradients(cuda, form, rows, vocab, k, dtype, temperature, pad, offset, ragged):
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    view, ids, lps, g = _case(rows, vocab, k, dtype, 7 * rows + vocab + k, pad, offset, ragged=ragged)
    scale = 64.0 if dtype == "fp16" else 1.0  # fp16 gradients of a wide row need a scaled loss
    weight = (0.2 + torch.rand(rows, generator=g)) * scale
    few = range(rows) if rows < 20 else [0, 1, rows // 2, rows - 2, rows - 1]
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda(), temperature, *form)
    (grad,) = torch.autograd.grad([loss], [leaf], [weight.cuda()])
    _check(view, ids, lps, temperature, form, loss.detach().cpu(), grad, weight, few)
    for inplace in (False, True):
        x = view.clone() if not inplace else view
        before = view.clone()
        loss2, grad2 = fused_distill_kl_fwd_bwd(x, ids.cuda(), lps.cuda(), weight.cuda(), temperature, *form, inplace=inplace)
        assert (grad2.data_ptr() == x.data_ptr()) == inplace
        _check(before, ids, lps, temperature, form, loss2.cpu(), grad2, weight, few)
        if not inplace:
            assert torch.equal(x, before)


@pytest.mark.parametrize("form", FORMS)
def test_gradient_against_differences(cuda, form):
    from openrlhf_amd.models.utils import distill_kl_from_logits

    view, ids, lps, _ = _case(3, 30, 5, "fp32", 4, sharp=2.0)
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda(), 1.3, *form)
    (grad,) = torch.autograd.grad(loss.sum(), [leaf])
    h = 1e-5
    for r, j in [(0, int(ids[0, 0])), (0, 7), (1, int(ids[1, 4])), (2, 29)]:
        x = view[r].double().cpu()
        d = torch.zeros_like(x)
        d[j] = h
        f = lambda y: ov.distill_kl_row(y, ids[r], lps[r].double(), 1.3, 1.0, *form).item()  # noqa: E731
        # truncation h^2, rounding 1e-14 / h, the kernel's fp32
        assert abs((f(x + d) - f(x - d)) / (2 * h) - grad[r, j].item()) <= 1e-8 + 1e-5 * (1 + abs(grad[r, j].item()))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab", [400, 40011])
def test_lists_with_absent_repeated_and_foreign_ids(cuda, form, vocab):
    from openrlhf_amd.models.utils import distill_kl_from_logits

    view, ids, lps, _ = _case(7, vocab, 6, "fp32", 13)
    lps = lps - 1.0           # leaves mass for the tail
    ids[1] = -1               # nothing listed
    lps[2] = -math.inf        # nothing listed either
    ids[3, 4] = ids[3, 1]     # one id twice
    ids[4, :] = ids[4, 0]     # one id six times
    lps[4] = torch.tensor([-3.0, -2.5, -4.0, -3.0, -6.0, -2.7])
    ids[5, 2] = vocab         # past the vocabulary
    ids[6, 3], lps[6, 5] = -7, -math.inf
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda().int(), lps.cuda(), 1.0, *form)
    weight = torch.ones(7)
    (grad,) = torch.autograd.grad(loss.sum(), [leaf])
    _check(view, ids, lps, 1.0, form, loss.detach().cpu(), grad, weight, [0, 1, 2, 3, 4, 6])
    assert loss[1].item() == 0 and loss[2].item() == 0 and (grad[1:3] == 0).all()
    assert math.isnan(loss[5].item()) and grad[5].isfinite().all()  # the foreign id has no gradient, the others do


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("vocab", [600, 33000])
def test_sure_students_and_masked_vocabularies(cuda, form, dtype, vocab):
    """Rows where 1 - sum q would be rounding noise, and rows whose other logits are masked."""
    from openrlhf_amd.models.utils import distill_kl_from_logits

    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, vocab, generator=g)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:4] for _ in range(6)])
    lps = torch.log(torch.tensor([[0.6, 0.25, 0.1, 0.04]])).repeat(6, 1)
    at = torch.arange(6)
    x[at, ids[:, 0]] += torch.tensor([5.0, 25.0, 40.0, 70.0, 0.0, 120.0])  # student's mass elsewhere: 1e-2 ... 1e-49
    keep = torch.zeros(vocab, dtype=torch.bool)
    keep[ids[4]] = True
    x[4, ~keep] = torch.finfo(TYPES[dtype]).min  # everything outside the list is masked
    x = x.to(TYPES[dtype])
    leaf = x.cuda().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda(), 1.0, *form)
    (grad,) = torch.autograd.grad(loss.sum(), [leaf])
    assert loss.isfinite().all() and grad.isfinite().all()
    _check(x.cuda(), ids, lps, 1.0, form, loss.detach().cpu(), grad, torch.ones(6), [0, 1, 2, 3])
    _check(x.cuda(), ids, lps, 1.0, form, loss.detach().cpu(), None, None, [4, 5])
    low = x.clone()
    low[0, keep.logical_not()] = -math.inf
    low[0, ids[0]] = x[0, ids[0]]
    out = distill_kl_from_logits(low[:1].cuda(), ids[:1].cuda(), lps[:1].cuda(), 1.0, *form)
    assert out.isfinite().all()


@pytest.mark.parametrize("n", [30, 1200])
def test_masked_rows_weights_of_zero_and_teacher_temperature(cuda, n):
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    view, ids, lps, g = _case(n, 6001, 9, "bf16", 3)
    mask = torch.rand(n, generator=g) < 0.5
    mask[0], mask[1] = True, False
    poison = view.clone()
    poison[~mask.cuda()] = math.nan  # masked rows are not read
    leaf = poison.requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda(), row_mask=mask.cuda())
    weight = torch.rand(n, generator=g)
    weight[0] = 0.0
    (grad,) = torch.autograd.grad([loss], [leaf], [weight.cuda()])
    assert (loss[~mask.cuda()] == 0).all() and (grad[~mask.cuda()] == 0).all() and (grad[0] == 0).all()
    rows = mask.nonzero()[:, 0].tolist()
    rows = rows[:12] + rows[-12:]
    _check(view, ids, lps, 1.0, ("forward", True), loss.detach().cpu(), grad, weight, rows)
    loss2, grad2 = fused_distill_kl_fwd_bwd(poison.detach().clone(), ids.cuda(), lps.cuda(), weight.cuda(), row_mask=mask.cuda().float())
    assert (loss2[~mask.cuda()] == 0).all() and (grad2[~mask.cuda()] == 0).all() and (grad2[0] == 0).all()
    _check(view, ids, lps, 1.0, ("forward", True), loss2.cpu(), grad2, weight, rows)
    raw = lps * 3 + 5  # logits of the teacher, at a temperature
    loss3 = distill_kl_from_logits(view, ids.cuda(), raw.cuda(), 1.4, tail=False, teacher_temperature=2.5)
    _check(view, ids, raw, 1.4, ("forward", False), loss3.cpu(), rows=range(5), teacher_temperature=2.5)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab,dtype", [(900, "fp32"), (151937, "bf16"), (200003, "fp16")])
def test_one_pass_on_rows_that_go_wrong(cuda, form, vocab, dtype):
    """The one-pass kernel against the two kernels on a batch that mixes ordinary rows with sure students,
    masked vocabularies, lists that are empty, repeated or out of range, -inf, NaN and far-off logits, so
    that a row's state must not leak into the rows its workgroup takes next."""
    from openrlhf_amd.models.utils import _DistillCall, _distill_backward, fused_distill_kl_fwd_bwd

    rows = 1100
    view, ids, lps, g = _case(rows, vocab, 10, dtype, 77, pad=8 - vocab % 8 if vocab % 8 else 0, ragged=True)
    kind = torch.arange(rows) % 11
    low = torch.finfo(TYPES[dtype]).min
    lps = lps - 0.5
    dev = lambda m: m.cuda()  # noqa: E731
    view[dev(kind == 1)] += 300.0 if dtype != "fp16" else 200.0
    spot = ids[:, 0].clamp(min=0).cuda()
    view[dev(kind == 2), spot[dev(kind == 2)]] = 90.0
    ids[kind == 3] = -1
    ids[kind == 4, 3] = ids[kind == 4, 0]
    ids[kind == 5, 2] = vocab + 5
    view[dev(kind == 6), : vocab - 3] = low
    view[dev(kind == 7)] = -math.inf
    view[dev(kind == 8), 11] = math.nan
    view[dev(kind == 9), 7 : vocab // 2] = -math.inf
    mask = (torch.rand(rows, generator=g) < 0.8).cuda()
    weight = torch.rand(rows, generator=g).cuda()
    weight[::13] = 0.0
    idc, lpc = ids.cuda(), lps.cuda()
    c = _DistillCall(view, idc, lpc, 0.9, *form, 1.0, mask)
    want, saved = c.forward(True)
    want_grad = _distill_backward(c.rows, c.row_stride, c.k, c.temperature, weight, saved, c.rmask, False)
    got, grad = fused_distill_kl_fwd_bwd(view.clone(memory_format=torch.preserve_format) if vocab % 8 == 0 else view, idc, lpc,
                                         weight, 0.9, *form, inplace=True, row_mask=mask)
    finite = want.isfinite()
    assert torch.equal(got.isfinite(), finite) and torch.equal(got.isnan(), want.isnan())
    live = ((kind != 7) & (kind != 8)).cuda() & mask  # rows without a softmax: NaN in both
    # sums of the same terms in another order: twice the bound of each; far-off logits take the exact path
    rel = 4 * (vocab / 1024 + 3 * 64 * 2 + 24) * U
    close = (got - want).abs() <= 4 * rel * (1 + want.abs())
    assert close[finite].all(), (kind.cuda()[finite & ~close], (got - want)[finite & ~close])
    a, b = grad[live].float(), want_grad[live].float()
    half = torch.finfo(TYPES[dtype]).eps / 2
    assert a.isfinite().all() and b.isfinite().all()
    # an element that is not listed: a product, each factor within 4 rel. A listed one is a difference of
    # terms up to w / T, of which the student's, q, moves by q times the change of the log-sum-exp (rel)
    # (reverse: times the log-ratio, up to 2 X / T, as well)
    listed = torch.zeros_like(b, dtype=torch.bool).scatter_(1, idc[live].clamp(0, vocab - 1), True)
    size = 1.0 if form[0] == "forward" else 1.0 + 2 * 100 / 0.9
    tol = (2 * half + 8 * rel) * b.abs() + listed * (rel * size * weight[live][:, None] / 0.9) + 2 * FLOOR[TYPES[dtype]]
    assert ((a - b).abs() <= tol).all(), (((a - b).abs() - tol).max(), kind[live.cpu()][((a - b).abs() > tol).any(1).cpu()])
    assert (grad[~mask] == 0).all() and (grad[::13][live[::13]] == 0).all()


def test_shapes_dtypes_and_empty_batches(cuda):
    from openrlhf_amd.models.utils import distill_kl_from_logits

    view, ids, lps, _ = _case(6, 515, 5, "bf16", 2)
    want = distill_kl_from_logits(view, ids.cuda(), lps.cuda())
    x = view.reshape(2, 3, 515)
    got = distill_kl_from_logits(x, ids.view(2, 3, 5).cuda().int(), lps.view(2, 3, 5).cuda().double())
    assert got.shape == (2, 3) and torch.equal(got.view(-1), want)
    turned = x.permute(0, 2, 1).contiguous().permute(0, 2, 1)
    assert torch.equal(distill_kl_from_logits(turned, ids.view(2, 3, 5).cuda(), lps.view(2, 3, 5).cuda()).view(-1), want)
    assert distill_kl_from_logits(view[:0], ids[:0].cuda(), lps[:0].cuda()).shape == (0,)


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 151936, "bf16"), (9, 50257, "fp16"), (300, 70001, "bf16")])
def test_cut_rows_merged_in_one_launch_or_two_give_the_same_bits(cuda, rows, vocab, dtype):
    from openrlhf_amd import _lib

    view, ids, lps, _ = _case(rows, vocab, 33, dtype, rows, ragged=True)
    if rows > 3:
        view[0, 5] = math.nan
        view[1] = -math.inf
        view[2] = torch.finfo(TYPES[dtype]).min
    code = _lib.dtype_code(view)
    mask = torch.ones(rows, dtype=torch.uint8, device="cuda")
    mask[rows // 2 : rows // 2 + rows // 5] = 0
    nbytes = _lib.load().orlhf_distill_kl_workspace_bytes(code, rows, vocab)
    assert nbytes > 0
    tickets = torch.zeros(rows, dtype=torch.int32, device="cuda")
    idc, lpc = ids.cuda(), lps.cuda()

    def once(tick, kind):
        ws = torch.randint(0, 255, (nbytes,), dtype=torch.uint8, device="cuda")
        loss, stats = torch.full((rows,), 7.0, device="cuda"), torch.full((rows, 4), 7.0, device="cuda")
        lg, at = torch.full((rows, 33), 7.0, device="cuda"), torch.full((rows, 33), 7, device="cuda", dtype=torch.int32)
        _lib.call("orlhf_distill_kl_fwd", view.data_ptr(), code, rows, vocab, vocab, idc.data_ptr(), lpc.data_ptr(), 33, 0.9, 1.0,
                  kind, loss.data_ptr(), stats.data_ptr(), lg.data_ptr(), at.data_ptr(), mask.data_ptr(), ws.data_ptr(), nbytes,
                  None if tick is None else tick.data_ptr(), _lib.stream_of(view.device))
        return [t.view(torch.int32) for t in (loss, stats, lg, at)]

    for kind in (_lib.DISTILL_FORWARD_TAIL, _lib.DISTILL_FORWARD, _lib.DISTILL_REVERSE_TAIL):
        want = once(None, kind)
        for _ in range(8):
            got = once(tickets, kind)
            assert int(tickets.abs().sum()) == 0
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [3, 600])
def test_other_stream_and_replayed_graph_give_the_same_bits(cuda, rows):
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    view, ids, lps, g = _case(rows, 30011, 12, "bf16", 9)
    other, ids2, lps2, _ = _case(rows, 30011, 12, "bf16", 10)
    w = torch.rand(rows, generator=g).cuda()
    args = lambda i, p: (i.cuda(), p.cuda(), w)  # noqa: E731
    want = fused_distill_kl_fwd_bwd(view, *args(ids, lps), inplace=False)
    want2 = fused_distill_kl_fwd_bwd(other, *args(ids2, lps2), inplace=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = fused_distill_kl_fwd_bwd(view, *args(ids, lps), inplace=False)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    sx, si, sl = view.clone(), ids.cuda(), lps.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_distill_kl_fwd_bwd(sx, si, sl, w, inplace=False)
    for x, i, p, expect in ((other, ids2, lps2, want2), (view, ids, lps, want), (other, ids2, lps2, want2)):
        sx.copy_(x), si.copy_(i), sl.copy_(p)
        graph.replay()
        distill_kl_from_logits(view, ids.cuda(), lps.cuda(), 0.5)  # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(out[0], expect[0]) and torch.equal(out[1], expect[1])


def test_teacher_targets_to_aggregated_student_loss(cuda):
    """The operators as they are used: a teacher's alternatives, the student's KL on them aggregated over a
    loss mask, and the same gradient from the one-pass form with the weights known up front."""
    from openrlhf_amd.models.loss import aggregate_loss
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd, top_logprobs_from_logits

    g = torch.Generator().manual_seed(12)
    teacher = (torch.randn(4, 80, 3001, generator=g) * 2).cuda()
    student = (teacher + torch.randn(4, 80, 3001, generator=g).cuda()).requires_grad_(True)
    mask = (torch.rand(4, 80, generator=g) < 0.7).cuda()
    _, _, top, ids = top_logprobs_from_logits(teacher, None, 24, return_entropy=False, row_mask=mask)
    kl = distill_kl_from_logits(student, ids, top, row_mask=mask)
    loss = aggregate_loss(kl, mask.float())
    (grad,) = torch.autograd.grad(loss, [student])
    weights = mask.float() / mask.sum()
    kl2, grad2 = fused_distill_kl_fwd_bwd(student.detach(), ids, top, weights, inplace=False, row_mask=mask)
    assert (kl > -1e-6).all() and (kl[~mask] == 0).all() and (ids[~mask] == -1).all()
    # sums of the same 3001 terms in another order, logits up to 12: 2 (3 + 3 x 12 x 1.45 + 24) u, as above
    rel = 2 * (3 + 3 * 12 * 1.45 + 24) * U
    assert ((kl - kl2).abs() <= 4 * rel * (1 + kl.abs())).all()
    assert ((grad - grad2).abs() <= 8 * rel * grad.abs() + 4 * rel * weights.unsqueeze(-1)).all()


def _sum_error(x, temperature):
    """Relative error of the sum outside the list: one rounding per term of an accumulator (two in each of
    256 lanes: V / 512), the rounding of the exponents (X = max |x|), and the additions that join them."""
    big = x[x.abs() < 1e30].abs().max().item()
    return (x.numel() / 512 + 3 * big * math.log2(math.e) / temperature + 24) * U


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab,dtype", [(2100, "fp32"), (33000, "bf16"), (80011, "fp16")])
@pytest.mark.parametrize("rows", [5, 300, 530])
def test_small_divergences_keep_their_digits(cuda, form, vocab, dtype, rows):
    """Teachers that nearly agree and students that are sure of the listed tokens, where the loss is a
    difference of much larger terms. Only R, the sum outside the list, is an fp32 sum (relative error d):
    the loss moves by dL/dlog R times d, that is ((P + t) s - t) d, s d and s (log(s / t) - L) d, by terms of
    d^2, and is rounded once (1e-12: the fp64 terms that cancel)."""
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    g = torch.Generator().manual_seed(vocab + rows)
    k, temperature = 6, 0.9
    x = torch.randn(rows, vocab, generator=g)
    listed = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)])
    x.scatter_add_(1, listed, torch.rand(rows, k, generator=g) * 3 + math.log(vocab) + torch.arange(rows).view(-1, 1) % 4 * 3.0)
    x = x.to(TYPES[dtype])
    near = x.double() + torch.randn(rows, vocab, generator=g).double() * (0.02 * (torch.arange(rows) % 3)).view(-1, 1)
    lps = torch.log_softmax(near / temperature, -1).gather(1, listed).float()
    view, idc, lpc = x.cuda(), listed.cuda(), lps.cuda()
    outs = [distill_kl_from_logits(view, idc, lpc, temperature, *form),
            fused_distill_kl_fwd_bwd(view, idc, lpc, torch.ones(rows, device="cuda"), temperature, *form, inplace=False)[0]]
    few = range(rows) if rows < 20 else list(range(0, 12)) + [rows - 2, rows - 1]
    small = 0
    for r, (want, _, x64) in zip(few, _reference(view, listed, lps, temperature, form, few)):
        d = _sum_error(x64, temperature)
        q = torch.log_softmax(x64 / temperature, -1).exp()
        inside = torch.zeros(vocab, dtype=torch.bool)
        inside[listed[r]] = True
        s, p = q[~inside].sum().item(), lps[r].double().exp()
        if form == ("forward", False):
            first = s
        elif form == ("forward", True):
            t = max(0.0, 1.0 - p.sum().item())
            first = abs((p.sum().item() + t) * s - t)
        else:
            t = max(2.0 ** -24, 1.0 - p.sum().item())
            first = abs(s * (math.log(s / t) - want))
        small += abs(want) < 1e-3
        for out in outs:
            assert abs(out[r].item() - want) <= first * d + 4 * d * d + 2 * U * abs(want) + 1e-12, (r, out[r].item(), want, s)
    assert small > 0


@pytest.mark.parametrize("teacher_temperature,shift,scale", [
    (1.0, 1000.0, 3.0),    # logits with a constant offset
    (1.0, -1000.0, 3.0),
    (0.05, 40.0, 3.0),     # ordinary logits at a low temperature
    (0.01, -30.0, 1.0),
    (1.0, 0.0, 300.0),     # one token far above the others
    (1.0, -720.0, 2.0),    # probabilities that would be subnormal
    (2.0, 3.0e38, 0.0),    # at the end of fp32
])
@pytest.mark.parametrize("n", [4, 300])
def test_teacher_logits_of_any_size(cuda, teacher_temperature, shift, scale, n):
    """tail=False takes the teacher's logits as they come: w = softmax(values / teacher_temperature), with
    repeated, absent and lowest-value entries among them."""
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    view, ids, _, g = _case(n, 5003, 12, "fp32", 31)
    raw = torch.randn(n, 12, generator=g) * scale + shift
    ids[1, 7] = ids[1, 2]
    ids[2, 3] = ids[2, 9] = ids[2, 0]
    raw[2, 0] = raw[2].max()
    ids[3, 5], raw[3, 6] = -1, -math.inf
    raw[3, 8] = torch.finfo(torch.float32).min
    weight = torch.rand(n, generator=g) + 0.2
    leaf = view.detach().requires_grad_(True)
    idc, rawc = ids.cuda(), raw.cuda()
    loss = distill_kl_from_logits(leaf, idc, rawc, 1.2, tail=False, teacher_temperature=teacher_temperature)
    (grad,) = torch.autograd.grad([loss], [leaf], [weight.cuda()])
    rows = range(4)
    want = _reference(view, ids, raw, 1.2, ("forward", False), rows, teacher_temperature)
    for r, (value, d, x) in zip(rows, want):
        rel = 2 * _sum_error(x, 1.2)
        # w: fp64 quotients of fp32 inputs; log w / q of terms up to max |log w| + max |log q|
        lq = torch.log_softmax(x / 1.2, -1)
        size = 2 * U * (abs(value) + 1)
        bound = (lq.exp() * (rel + 4 * U * (lq.abs() + 4)) + 4 * U * (d.abs() + lq.exp())) / 1.2
        for l, gr in ((loss, grad), fused_distill_kl_fwd_bwd(view, idc, rawc, weight.cuda(), 1.2, tail=False, inplace=False,
                                                             teacher_temperature=teacher_temperature)):
            assert abs(l[r].item() - value) <= rel + size, (r, l[r].item(), value)
            w = weight[r].item()
            assert ((gr[r].double().cpu() - w * d).abs() <= w * bound + 1e-37).all(), r


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows", [4, 300])
@pytest.mark.parametrize("vocab", [3001, 70001])
def test_gradients_of_students_sure_beyond_the_range_of_fp32(cuda, form, dtype, rows, vocab):
    """The student's mass outside the list is 1e-33 to 1e-37 and each weight there far below the least fp32
    number, but the teacher's tail still pulls: d / dz = ((P + t) s - t) r with r the softmax outside the list.
    r is as exact as its sum (d), its stored logarithm (up to 20 in log2 units) and its exponents are."""
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    g = torch.Generator().manual_seed(vocab)
    temperature = 0.25
    x = torch.randn(rows, vocab, generator=g)
    listed = torch.stack([torch.randperm(vocab, generator=g)[:3] for _ in range(rows)])
    gap = (torch.tensor([80.0, 82.5, 84.0, 85.0])[torch.arange(rows) % 4] + math.log(vocab)) * temperature + 0.5 / temperature * 0.9
    x.scatter_(1, listed, torch.tensor([0.0, -0.5, -1.0]).repeat(rows, 1) + gap.view(-1, 1))
    x = x.to(TYPES[dtype])
    lps = torch.log(torch.tensor([[0.6, 0.2, 0.1]])).repeat(rows, 1)
    weight = (0.5 + torch.rand(rows, generator=g)) * (256.0 if dtype == "fp16" else 1.0)
    view, idc, lpc = x.cuda(), listed.cuda(), lps.cuda()
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, idc, lpc, temperature, *form)
    (grad,) = torch.autograd.grad([loss], [leaf], [weight.cuda()])
    _, grad2 = fused_distill_kl_fwd_bwd(view, idc, lpc, weight.cuda(), temperature, *form, inplace=False)
    half = torch.finfo(TYPES[dtype]).eps / 2
    for r, (_, d, x64) in zip(range(4), _reference(view, listed, lps, temperature, form, range(4))):
        outside = torch.ones(vocab, dtype=torch.bool)
        outside[listed[r]] = False
        s = torch.log_softmax(x64 / temperature, -1)[outside].exp().sum().item()
        assert 2.0 ** -126 < s < 1e-32, s  # what the test is about
        d = weight[r].item() * d[outside]
        centred = (x64[outside] - x64[outside].max()).abs() / temperature
        rel = _sum_error(x64, temperature) + (24 + 4 * centred) * U
        for gr in (grad, grad2):
            got = gr[r].double().cpu()[outside]
            assert ((got - d).abs() <= (half + 2 * rel) * d.abs() + 2 * FLOOR[TYPES[dtype]]).all(), (r, s)
    if form == ("forward", True):
        assert (grad[:4].abs().sum(1) > 0.1).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab,dtype", [(9, "bf16"), (33, "fp32"), (515, "fp16"), (4096, "bf16"), (4103, "fp16"), (2051, "fp32"),
                                         (151937, "bf16"), (77827, "fp32"), (155651, "fp16")])
def test_lists_at_the_ends_of_a_row(cuda, form, vocab, dtype):
    """The first and last tokens listed: the bits next to the map's end, lanes whose chunk the row ends in, and
    the elements off the 16-byte grid, in one pass and in two launches."""
    from openrlhf_amd.models.utils import distill_kl_from_logits, fused_distill_kl_fwd_bwd

    view, _, _, g = _case(270, vocab, 4, dtype, vocab, pad=3, offset=1)
    k = min(vocab, 8)
    ids = torch.cat([torch.arange((k + 1) // 2), vocab - 1 - torch.arange(k // 2)]).repeat(270, 1)
    lps = torch.log_softmax(torch.randn(270, k, generator=g), -1) - 0.2
    scale = 64.0 if dtype == "fp16" else 1.0
    weight = (0.2 + torch.rand(270, generator=g)) * scale
    few = [0, 1, 268, 269]
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda(), 0.8, *form)
    (grad,) = torch.autograd.grad([loss], [leaf], [weight.cuda()])
    _check(view, ids, lps, 0.8, form, loss.detach().cpu(), grad, weight, few)
    before = view.clone()
    loss, grad = fused_distill_kl_fwd_bwd(view, ids.cuda(), lps.cuda(), weight.cuda(), 0.8, *form)
    _check(before, ids, lps, 0.8, form, loss.cpu(), grad, weight, few)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab,dtype", [(700, "bf16"), (1500, "fp32"), (3584, "fp16"), (3600, "bf16"), (2100, "fp32")])
def test_short_rows_and_blocked_stretches_in_one_pass(cuda, form, vocab, dtype):
    """Rows that leave waves of the workgroup idle, next to rows whose first or later stretches are -inf (a
    wave then has nothing finite to refer to although it has elements that count)."""
    from openrlhf_amd.models.utils import fused_distill_kl_fwd_bwd

    view, ids, lps, g = _case(256, vocab, 5, dtype, vocab + 2)
    for r, (lo, hi) in enumerate([(0, vocab // 2), (vocab // 2, vocab), (0, min(512, vocab // 3)), (0, vocab - 3), (0, 0)]):
        view[r, lo:hi] = -math.inf
        view[r] -= 20.0 * r  # references that differ from 0
    ids[:5] = torch.arange(vocab // 4, vocab // 4 + 5)
    ids[:5, 0] = vocab - 1
    for r in range(5):
        view[r, ids[r].cuda()] = torch.randn(5, generator=g).to(view.dtype).cuda() - 20.0 * r
    lps[:5] = torch.log_softmax(torch.randn(5, 5, generator=g), -1) - 0.3
    before = view.clone()
    weight = torch.ones(256) * (64.0 if dtype == "fp16" else 1.0)
    loss, grad = fused_distill_kl_fwd_bwd(view, ids.cuda(), lps.cuda(), weight.cuda(), 1.0, *form)
    assert loss.isfinite().all() and grad.isfinite().all()
    few = range(7)
    for r, (want, d, x) in zip(few, _reference(before, ids, lps, 1.0, form, few)):
        lq = torch.log_softmax(x, -1)
        rel = _sum_error(x, 1.0)
        ratios = 2.0 if form[0] == "forward" else 4.0 + 2 * lq[lq > -math.inf].abs().max().item()
        assert abs(loss[r].item() - want) <= ratios * rel + 2 * U * abs(want), (r, loss[r].item(), want)
        w, d = weight[r].item(), torch.nan_to_num(d)
        half = torch.finfo(TYPES[dtype]).eps / 2
        bound = w * (ratios * (d.abs() + lq.exp()) * (2 * rel + 8 * U) + 4 * U)
        assert ((grad[r].double().cpu() - w * d).abs() <= half * w * d.abs() + bound + FLOOR[TYPES[dtype]]).all(), r


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,vocab,k,dtype,temperature,pad,offset,ragged", [
    (1, 1, 1, "fp32", 1.0, 0, 0, False),
    (5, 131, 128, "fp16", 1.0, 1, 3, True),
    (514, 4099, 7, "bf16", 1.0, 0, 0, True),
    (300, 262144, 100, "fp16", 0.7, 0, 0, True),
    (530, 50257, 128, "fp32", 1.0, 6, 3, True),
    (1031, 33, 33, "fp32", 1.3, 3, 1, True),
    (260, 80001, 11, "fp32", 2.0, 0, 0, False),
    (257, 376832, 20, "bf16", 1.0, 0, 0, True),
])
def test_one_pass_kernel_whatever_the_rule(cuda, monkeypatch, form, rows, vocab, k, dtype, temperature, pad, offset, ragged):
    """The one-pass kernel (a public C entry) on shapes for which the Python form takes the two launches."""
    from openrlhf_amd import _lib
    from openrlhf_amd.models import utils

    used, call = [], utils.call
    monkeypatch.setattr(utils, "_one_pass_pays", lambda n_rows, row_bytes: True)
    monkeypatch.setattr(utils, "call", lambda name, *a: (used.append(name), call(name, *a)))
    assert vocab <= _lib.load().orlhf_distill_kl_fwd_bwd_max_vocab(_lib.dtype_code(torch.empty(0, dtype=TYPES[dtype])))
    test_loss_and_gradients(cuda, form, rows, vocab, k, dtype, temperature, pad, offset, ragged)
    assert "orlhf_distill_kl_fwd_bwd" in used  # in place; out of place only rows on the 16-byte grid go through it


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vocab,dtype", [(33, "fp32"), (515, "fp16"), (4103, "bf16"), (2051, "fp32"), (77827, "fp32")])
def test_one_pass_kernel_at_the_ends_of_a_row(cuda, monkeypatch, form, vocab, dtype):
    from openrlhf_amd.models import utils

    monkeypatch.setattr(utils, "_one_pass_pays", lambda n_rows, row_bytes: True)
    test_lists_at_the_ends_of_a_row(cuda, form, vocab, dtype)


@pytest.mark.parametrize("form", FORMS)
def test_one_pass_kernel_on_rows_that_go_wrong_of_every_type(cuda, monkeypatch, form):
    from openrlhf_amd.models import utils

    monkeypatch.setattr(utils, "_one_pass_pays", lambda n_rows, row_bytes: True)
    for vocab, dtype in ((900, "fp32"), (200003, "fp16")):
        test_one_pass_on_rows_that_go_wrong(cuda, form, vocab, dtype)


def test_second_derivatives_are_refused(cuda):
    from openrlhf_amd.models.utils import distill_kl_from_logits, top_logprobs_from_logits

    view, ids, lps, _ = _case(3, 50, 4, "fp32", 1)
    leaf = view.detach().requires_grad_(True)
    loss = distill_kl_from_logits(leaf, ids.cuda(), lps.cuda())
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(loss.sum(), [leaf], create_graph=True)
    assert torch.autograd.grad(loss.sum(), [leaf])[0].isfinite().all()
    _, entropy, top, _ = top_logprobs_from_logits(leaf, None, 4)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(top.sum() + entropy.sum(), [leaf], create_graph=True)
    assert torch.autograd.grad(top.sum(), [leaf])[0].isfinite().all()


# The forms above once more through the one-pass kernel, where the rule gives their sizes to the two launches.
@pytest.fixture
def one_pass(monkeypatch):
    from openrlhf_amd.models import utils

    used, call = [], utils.call
    monkeypatch.setattr(utils, "_one_pass_pays", lambda n_rows, row_bytes: True)
    monkeypatch.setattr(utils, "call", lambda name, *a: (used.append(name), call(name, *a)))
    yield
    assert "orlhf_distill_kl_fwd_bwd" in used


@pytest.mark.parametrize("rows", [3, 600])
def test_one_pass_kernel_on_another_stream_and_in_a_replayed_graph(cuda, one_pass, rows):
    test_other_stream_and_replayed_graph_give_the_same_bits(cuda, rows)


@pytest.mark.parametrize("n", [30, 1200])
def test_one_pass_kernel_with_masked_rows_and_weights_of_zero(cuda, one_pass, n):
    test_masked_rows_weights_of_zero_and_teacher_temperature(cuda, n)


def test_one_pass_kernel_as_the_operators_are_used(cuda, one_pass):
    test_teacher_targets_to_aggregated_student_loss(cuda)


@pytest.mark.parametrize("form", FORMS)
def test_one_pass_kernel_keeps_digits_and_range(cuda, one_pass, form):
    test_small_divergences_keep_their_digits(cuda, form, 33000, "bf16", 530)
    test_small_divergences_keep_their_digits(cuda, form, 2100, "fp32", 300)
    for dtype in ("fp32", "bf16", "fp16"):
        test_gradients_of_students_sure_beyond_the_range_of_fp32(cuda, form, dtype, 300, 70001)
        test_gradients_of_students_sure_beyond_the_range_of_fp32(cuda, form, dtype, 4, 3001)


@pytest.mark.parametrize("teacher_temperature,shift,scale", [(1.0, 1000.0, 3.0), (0.05, 40.0, 3.0), (1.0, -720.0, 2.0), (2.0, 3.0e38, 0.0)])
def test_one_pass_kernel_with_teacher_logits_of_any_size(cuda, one_pass, teacher_temperature, shift, scale):
    test_teacher_logits_of_any_size(cuda, teacher_temperature, shift, scale, 300)


def test_one_pass_kernel_with_every_row_masked_out(cuda, one_pass):
    from openrlhf_amd.models.utils import fused_distill_kl_fwd_bwd

    view, ids, lps, _ = _case(700, 2051, 5, "bf16", 6, pad=5)
    poison = torch.full_like(view, math.nan)
    loss, grad = fused_distill_kl_fwd_bwd(poison, ids.cuda(), lps.cuda(), torch.ones(700, device="cuda"),
                                          row_mask=torch.zeros(700, device="cuda"))
    assert (loss == 0).all() and (grad == 0).all()
