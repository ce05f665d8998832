"""Distillation from a teacher's top logits against the definition in 64 bits."""
import math

import pytest
import torch

from dreamer_amd import _native as N
from dreamer_amd import losses

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def reference(s, values, idx, t, lse, g):
    """Loss, its gradient and q, p dense, row by row from the definition."""
    s, values = s.detach().double(), values.double()
    rows, V = s.shape
    loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, V, dtype=torch.float64)
    qs, ps = torch.zeros_like(grad), torch.zeros_like(grad)
    s, values, idx = s.cpu(), values.cpu(), idx.cpu()
    for r in range(rows):
        ok = (idx[r] >= 0) & (idx[r] < V)
        tv, ti = values[r][ok] / t, idx[r][ok]
        if len(ti) == 0 or (lse is None and bool((tv == -math.inf).all())):
            continue
        logq = torch.log_softmax(s[r] / t, 0)
        q = logq.exp()
        logp = torch.log_softmax(tv, 0) if lse is None else tv - lse[r].double().cpu()
        p = logp.exp()
        for j in range(len(ti)):
            ps[r, ti[j]] += p[j]
            if p[j] != 0:
                loss[r] += p[j] * (logp[j] - logq[ti[j]])
        d = q * p.sum() - ps[r]
        if lse is not None:
            off = torch.ones(V, dtype=torch.bool)
            off[ti] = False
            P = max(0.0, 1.0 - float(p.sum()))
            if bool((logq[off] > -math.inf).any()) and P > 0:
                logQ = torch.logsumexp(logq[off], 0)
                loss[r] += P * (math.log(P) - logQ)
                d = d + q * P - torch.where(off, P * torch.exp(logq - logQ), torch.zeros_like(q))
        grad[r] = d * float(g[r]) / t
        qs[r] = q
    return loss.to(DEV), grad.to(DEV), qs.to(DEV), ps.to(DEV)


def tolerances(s, t, g, ref):
    """fp32 steps: an exponent d / T is off by 2 half steps of its size (factor and product), the hardware's exp2 by 2 more; a row sum
    passes at most 128 + 16 additions in 32 bits.  Entries more than 40 below the maximum do not count, so the exponents that do are at
    most 40: 2 * 40 + 2 + 144 half steps on q and, in logarithms, on the loss."""
    loss, grad, q, p = ref
    rel = (2 * 40 + 2 + 144 + 8) * U
    loss_tol = rel * (1 + loss.abs())
    half = torch.finfo(s.dtype).eps / 2
    tiny = torch.finfo(s.dtype).smallest_normal * torch.finfo(s.dtype).eps
    gs = g.double().abs().unsqueeze(1) / t
    return loss_tol, half * grad.abs() + rel * gs * (2 * q + p) + tiny


def inputs(rows, V, k, dtype, t, rest, seed=0, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed + 31 * rows + V + k)
    teacher = scale * torch.randn(rows, V, generator=g, device=DEV)
    s = (0.5 * teacher + scale * 0.6 * torch.randn(rows, V, generator=g, device=DEV)).to(dtype)
    values, idx = teacher.topk(k, 1)
    order = torch.randperm(k, generator=g, device=DEV)                   # lists need not be sorted
    lse = torch.logsumexp(teacher.double() / t, 1).float() if rest else None
    return s.requires_grad_(), values[:, order].contiguous(), idx[:, order].contiguous(), lse, torch.rand(rows, generator=g, device=DEV) + 0.1


def check(s, values, idx, t, lse, g, rows=None):
    loss = losses.distill_topk_rows(s, values, idx, t, lse)
    (grad,) = torch.autograd.grad(loss, s, g)
    assert grad.dtype == s.dtype and grad.shape == s.shape and loss.dtype == F32
    ref = reference(s, values, idx, t, lse, g)
    lt, gt = tolerances(s, t, g, ref)
    keep = slice(None) if rows is None else rows
    for name, a, b, tol in (("loss", loss.detach(), ref[0], lt), ("grad", grad, ref[1], gt)):
        bad = ((a.double() - b).abs() - tol)[keep]
        assert not torch.isnan(bad).any() and float(bad.max()) <= 0, (name, float(bad.max()))
    return loss.detach(), grad


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,V,k,t", [(1, 1, 1, 1.0), (3, 2, 1, 1.0), (5, 31, 7, 0.5), (240, 255, 16, 1.0), (9, 2048, 64, 2.0),
                                        (4, 2049, 65, 1.0), (6, 32768, 128, 4.0), (3, 32769, 3, 1.0), (2, 70001, 1000, 2.0)])
def test_values_and_gradients(rows, V, k, t, dtype, rest):
    check(*_args(inputs(rows, V, k, dtype, t, rest), t))


def _args(x, t):
    s, values, idx, lse, g = x
    return s, values, idx, t, lse, g


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("V", [50, 5000, 40000])
def test_absent_entries_and_empty_rows(V, rest):
    s, values, idx, lse, g = inputs(6, V, 10, F32, 1.0, rest)
    idx[0, 3:] = -1
    idx[1, :] = V                     # nothing left
    idx[2, ::2] = 2 ** 40
    idx[4, :] = -(2 ** 62)
    with torch.no_grad():
        s[4] = float("nan")           # an empty row is not looked at
    loss, grad = check(s, values, idx, 1.0, lse, g)
    assert float(loss[1]) == 0 and float(loss[4]) == 0 and float(grad[1].abs().max()) == 0 and float(grad[4].abs().max()) == 0


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [4097, 8195, 32771, 36867])
def test_entries_at_the_ends_of_a_rows_pieces(V, dtype, rest):
    s, values, idx, lse, g = inputs(3, V, 8, dtype, 1.0, rest)
    idx[:] = torch.tensor([0, 4095, 4096, V - 1, V - 2, V - 3, V // 2, 31], device=DEV)
    if rest:
        lse = lse + 2.5
    check(s, values, idx, 1.0, lse, g)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("V", [64, 3000, 40000])
def test_an_index_listed_twice_adds_up(V, rest):
    s, values, idx, lse, g = inputs(4, V, 12, F32, 1.0, rest)
    idx[:, 5] = idx[:, 2]
    idx[1, 7] = idx[1, 2]
    idx[2, :] = idx[2, :1]
    if rest:
        lse = lse + 2.5               # the doubled entries must leave something over
    a = check(s, values, idx, 1.0, lse, g)
    b = check(s, values, idx, 1.0, lse, g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rest", [False, True])
def test_masked_logits_and_lowest_values(dtype, rest):
    V = 3001
    s, values, idx, lse, g = inputs(7, V, 9, dtype, 1.0, rest)
    low = torch.finfo(dtype).min
    off = torch.rand(7, V, device=DEV) < 0.4
    off.scatter_(1, idx, False)
    with torch.no_grad():
        s.masked_fill_(off, float("-inf"))
        s[3] = s[3].masked_fill(off[3], low)
    values[5, 2:] = float("-inf")
    values[6, 1:] = torch.finfo(F32).min
    check(s, values, idx, 1.0, lse, g)
    # nothing open outside the list: the rest has nowhere to go and is left out
    with torch.no_grad():
        s[0] = float("-inf")
        s[0, idx[0]] = torch.arange(9, device=DEV).to(dtype)
    check(s, values, idx, 1.0, lse, g)
    # a list of -inf only is an empty one without the teacher's sum
    values[1] = float("-inf")
    loss, grad = check(s, values, idx, 1.0, lse, g)
    if not rest:
        assert float(loss[1]) == 0 and float(grad[1].abs().max()) == 0


def test_everything_listed_with_the_teachers_sum():
    s, values, idx, lse, g = inputs(5, 40, 40, F32, 1.0, True)
    check(s, values, idx, 1.0, lse, g)


def test_a_student_far_from_the_teacher():
    # listed entries 300 above the unlisted ones and the other way round: the small side keeps its logarithm
    V = 500
    s = torch.zeros(2, V, device=DEV)
    idx = torch.arange(4, device=DEV).repeat(2, 1)
    s[0, :4] = 300.0
    s[1, :4] = -300.0
    values = torch.tensor([[1.0, 0.5, 0.0, -0.5]], device=DEV).repeat(2, 1)
    lse = torch.full((2,), 2.5, device=DEV)
    g = torch.ones(2, device=DEV)
    # logits 300 apart: exponents of 300 / ln 2 = 433 carry 2 half steps each into the loss
    loss = losses.distill_topk_rows(s.requires_grad_(), values, idx, 1.0, lse)
    (grad,) = torch.autograd.grad(loss, s, g)
    ref = reference(s, values, idx, 1.0, lse, g)
    assert float((loss.double() - ref[0]).abs().max()) < 300 * 16 * U and torch.isfinite(grad).all()
    assert float((grad.double() - ref[1]).abs().max()) < 300 * 16 * U


def test_nan_and_infinite_logits_stay_in_their_row():
    s, values, idx, lse, g = inputs(5, 4100, 8, F32, 1.0, True)
    clean, cg = check(s, values, idx, 1.0, lse, g)
    with torch.no_grad():
        s[1, 77] = float("nan")
        s[3, 4099] = float("inf")
    loss = losses.distill_topk_rows(s, values, idx, 1.0, lse)
    (grad,) = torch.autograd.grad(loss, s, g)
    keep = [0, 2, 4]
    assert torch.equal(loss[keep], clean[keep]) and torch.equal(grad[keep], cg[keep])
    assert torch.isnan(loss[[1, 3]]).all() and torch.isnan(grad[[1, 3]]).any(1).all()


def test_no_rows_no_list_and_types_of_the_list():
    s, values, idx, lse, g = inputs(4, 100, 5, BF16, 1.0, False)
    a = losses.distill_topk_rows(s, values, idx)
    assert torch.equal(a, losses.distill_topk_rows(s, values, idx.int()))
    half = values.to(BF16)
    assert torch.equal(losses.distill_topk_rows(s, half, idx), losses.distill_topk_rows(s, half.float(), idx))
    empty = losses.distill_topk_rows(s, values[:, :0], idx[:, :0])
    assert float(empty.abs().max()) == 0
    (ge,) = torch.autograd.grad(empty.sum(), s)
    assert float(ge.abs().max()) == 0
    z = torch.zeros(0, 100, device=DEV, requires_grad=True)
    lz = losses.distill_topk_rows(z, values[:0], idx[:0])
    assert lz.shape == (0,) and torch.autograd.grad(lz.sum(), z)[0].shape == (0, 100)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_strided_logits_and_leading_dimensions(dtype):
    full = (torch.randn(12, 333, device=DEV) * 2).to(dtype)
    s = full[:, 1:302].detach().requires_grad_()
    values, idx = torch.randn(12, 301, device=DEV).topk(6, 1)
    g = torch.rand(12, device=DEV)
    loss, grad = check(s, values, idx, 1.0, None, g)
    s3 = s.detach().contiguous().view(3, 4, 301).requires_grad_()
    loss3 = losses.distill_topk_rows(s3, values.view(3, 4, 6), idx.view(3, 4, 6))
    assert torch.equal(loss3.detach(), loss) and torch.equal(torch.autograd.grad(loss3, s3, g)[0].view(12, 301), grad)


def test_gradient_against_differences():
    s, values, idx, lse, g = inputs(2, 37, 5, F32, 1.5, True)
    loss = losses.distill_topk_rows(s, values, idx, 1.5, lse)
    (grad,) = torch.autograd.grad(loss, s, g)
    h = 2.0 ** -6
    for v in (int(idx[0, 0]), int(idx[1, 3]), 0, 36):
        for r in range(2):
            up, dn = s.detach().clone(), s.detach().clone()
            up[r, v] += h
            dn[r, v] -= h
            f = [float((losses.distill_topk_rows(a, values, idx, 1.5, lse).double() * g.double()).sum()) for a in (up, dn)]
            assert abs((f[0] - f[1]) / (2 * h) - float(grad[r, v])) < h * h + 2 * 234 * U * 4 / (2 * h)


def test_logits_beyond_32_bit_offsets():
    stride = 2 ** 30 + 8
    buf = torch.empty(2 * stride + 4000, dtype=BF16, device=DEV)
    s = buf.as_strided((3, 4000), (stride, 1))
    vals, v, i, lse, g = inputs(3, 4000, 20, BF16, 1.0, True)
    s.copy_(vals.detach())
    a = s.detach().requires_grad_()
    la, lb = losses.distill_topk_rows(a, v, i, 1.0, lse), losses.distill_topk_rows(vals, v, i, 1.0, lse)
    assert torch.equal(la, lb) and torch.equal(torch.autograd.grad(la, a, g)[0], torch.autograd.grad(lb, vals, g)[0])


@pytest.mark.parametrize("V", [300, 40000])
def test_on_another_stream_and_in_a_recorded_graph(V):
    s, values, idx, lse, g = inputs(6, V, 11, BF16, 1.0, True)
    eager = losses.distill_topk_rows(s, values, idx, 1.0, lse)
    eager_grad = torch.autograd.grad(eager, s, g, retain_graph=True)[0]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        loss = losses.distill_topk_rows(s, values, idx, 1.0, lse)
        grad = torch.autograd.grad(loss, s, g)[0]
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(loss, eager) and torch.equal(grad, eager_grad)
    del loss, grad
    ss = s.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lg = losses.distill_topk_rows(ss, values, idx, 1.0, lse)
        gg = torch.autograd.grad(lg, ss, g)[0]
    for n in range(3):
        with torch.no_grad():
            ss.copy_(s.detach() * (1 + n))
        graph.replay()
        torch.cuda.synchronize()
        fresh = ss.detach().clone().requires_grad_()
        lr = losses.distill_topk_rows(fresh, values, idx, 1.0, lse)
        assert torch.equal(lg, lr) and torch.equal(gg, torch.autograd.grad(lr, fresh, g)[0])


def test_host_tensors_take_the_formula():
    for rest in (False, True):
        s, values, idx, lse, g = inputs(6, 90, 7, F32, 2.0, rest)
        idx[1, 3:] = -1
        idx[2] = 90
        want, wg = check(s, values, idx, 2.0, lse, g)
        h = s.detach().cpu().requires_grad_()
        loss = losses.distill_topk_rows(h, values.cpu(), idx.cpu(), 2.0, None if lse is None else lse.cpu())
        (grad,) = torch.autograd.grad(loss, h, g.cpu())
        # two fp32 evaluations, each within the bound
        assert float((loss.to(DEV) - want).abs().max()) < 2 * 234 * U * (1 + float(want.abs().max()))
        assert float((grad.to(DEV) - wg).abs().max()) < 4 * 234 * U


def test_refusals_on_the_device():
    s, values, idx, lse, g = inputs(4, 100, 5, F32, 1.0, True)
    with pytest.raises(N.NativeError, match="does not match"):
        losses.distill_topk_rows(s, values[:3], idx)
    with pytest.raises(N.NativeError, match="is on cpu"):
        losses.distill_topk_rows(s, values.cpu(), idx)
    with pytest.raises(N.NativeError, match="top_lse"):
        losses.distill_topk_rows(s, values, idx, 1.0, lse[:2])
    with pytest.raises(ValueError, match="temperature"):
        losses.distill_topk_rows(s, values, idx, 0.0)
    big = torch.zeros(1, 1025, device=DEV)
    with pytest.raises(N.NativeError, match="at most 1024"):
        losses.distill_topk_rows(torch.zeros(1, 2000, device=DEV), big, big.long())
    with pytest.raises(N.NativeError, match="fp32, bf16 or fp16"):
        losses.distill_topk_rows(s.double(), values, idx)
