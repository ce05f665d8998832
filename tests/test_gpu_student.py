"""The new operators together, as a student of a stored teacher uses them: layer norm, frozen 4-bit layers, distillation from the
teacher's top logits, the gradient back through all of it, the same step recorded into a graph, and the acting form on single rows."""
import pytest
import torch

from dreamer_amd import losses, mx4, norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
ROWS, WIDTH, HIDDEN, VOCAB, TOP = 48, 96, 160, 300, 12


def _student(seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    p = dict(w1=(1 + 0.2 * r(WIDTH)), b1=0.2 * r(WIDTH), c1=0.1 * r(HIDDEN), w2=(1 + 0.2 * r(HIDDEN)), b2=0.2 * r(HIDDEN), c2=0.1 * r(VOCAB))
    p = {k: v.requires_grad_() for k, v in p.items()}
    q1, q2 = mx4.quantize(r(HIDDEN, WIDTH) / WIDTH ** 0.5), mx4.quantize(r(VOCAB, HIDDEN) / HIDDEN ** 0.5)
    teacher = 2 * r(ROWS, VOCAB)
    values, idx = teacher.topk(TOP, 1)
    idx[3] = -1
    idx[7, 4:] = -1
    return p, q1, q2, r(ROWS, WIDTH).requires_grad_(), (values, idx, torch.logsumexp(teacher / 2.0, 1))


def _forward(p, q1, q2, x):
    h = mx4.linear(norm.layer_norm(x, p["w1"], p["b1"]), q1, p["c1"])
    return mx4.linear(norm.layer_norm(h, p["w2"], p["b2"]), q2, p["c2"])


def _step(p, q1, q2, x, teacher):
    values, idx, lse = teacher
    loss = losses.distill_topk_rows(_forward(p, q1, q2, x), values, idx, 2.0, lse).sum()
    leaves = [x] + [p[k] for k in sorted(p)]
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves))


def _reference(p, q1, q2, x, teacher):
    values, idx, lse = (t.double() if t.is_floating_point() else t for t in teacher)
    p = {k: v.detach().double().requires_grad_() for k, v in p.items()}
    x = x.detach().double().requires_grad_()
    ln = lambda v, w, b: torch.nn.functional.layer_norm(v, v.shape[-1:], w, b)
    h = ln(x, p["w1"], p["b1"]) @ q1.dequantize().double().t() + p["c1"]
    s = ln(h, p["w2"], p["b2"]) @ q2.dequantize().double().t() + p["c2"]
    logq = torch.log_softmax(s / 2.0, 1)
    loss = 0.0
    for r in range(ROWS):
        ok = idx[r] >= 0
        if not bool(ok.any()):
            continue
        lp = values[r][ok] / 2.0 - lse[r]
        t = lp.exp()
        rest = torch.ones(VOCAB, dtype=torch.bool, device=DEV)
        rest[idx[r][ok]] = False
        P = 1.0 - t.sum()
        loss = loss + (t * (lp - logq[r, idx[r][ok]])).sum() + P * (P.log() - torch.logsumexp(logq[r][rest], 0))
    leaves = [x] + [p[k] for k in sorted(p)]
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves))


def test_a_training_step_of_a_student_with_frozen_4_bit_layers():
    p, q1, q2, x, teacher = _student()
    got = _step(p, q1, q2, x, teacher)
    want = _reference(p, q1, q2, x, teacher)
    # nine operators on the way there and back; each is off by at most 3 * 300 + 256 half steps of its largest magnitudes (the longest
    # sum), and the norms and products that follow enlarge a relative error at most tenfold
    for a, b in zip(got, want):
        assert a.shape == b.shape and float((a.double() - b).abs().max()) <= 9 * 1156 * 10 * U * float(b.abs().max())
    assert float(got[1][3].abs().max()) == 0          # the row without a teacher


def test_the_step_recorded_and_replayed():
    p, q1, q2, x, teacher = _student(1)
    for _ in range(2):
        _step(p, q1, q2, x, teacher)                    # (nothing of these graphs is alive when the step is recorded)
    xs = x.detach().clone().requires_grad_()
    ps = {k: v.detach().clone().requires_grad_() for k, v in p.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(ps, q1, q2, xs, teacher)
    for n in range(3):
        with torch.no_grad():
            xs.copy_(x.detach() * (1.0 + 0.5 * n))
            for k in ps:
                ps[k].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        fresh = {k: v.detach().clone().requires_grad_() for k, v in ps.items()}
        ref = _step(fresh, q1, q2, xs.detach().clone().requires_grad_(), teacher)
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_acting_on_single_rows(dtype):
    """One row at a time, weights and (second form) rows in 4 bits: the layer modules give what the functions give."""
    p, q1, q2, x, _ = _student(2)
    lin = torch.nn.Linear(WIDTH, HIDDEN).to(DEV)
    ln = norm.LayerNorm(WIDTH).to(DEV)
    fl, q4 = mx4.MX4Linear.from_linear(lin), mx4.MX4Linear.from_linear(lin, activations="mx4")
    with torch.no_grad():
        rows = x.detach().to(dtype)
        w = mx4.quantize(lin.weight)
        for r in range(3):
            one = rows[r:r + 1]
            y = ln(one)
            ref = torch.nn.functional.layer_norm(one.double(), (WIDTH,), ln.weight.double(), ln.bias.double())
            assert y.dtype == dtype and float((y.double() - ref).abs().max()) <= (torch.finfo(dtype).eps / 2 + 128 * U) * 6
            a, b = fl(y), q4(y)
            assert torch.equal(a, mx4.linear(y, w, lin.bias)) and torch.equal(b, mx4.linear(mx4.quantize(y), w, lin.bias, dtype))
            full = y.double() @ w.dequantize().double().t() + lin.bias.double()
            mag = y.double().abs() @ w.dequantize().double().abs().t() + lin.bias.double().abs()
            assert float(((a.double() - full).abs() - torch.finfo(dtype).eps / 2 * full.abs() - (3 * WIDTH + 2) * U * mag).max()) <= 0
            four = mx4.quantize(y).dequantize().double() @ w.dequantize().double().t() + lin.bias.double()
            assert float(((b.double() - four).abs() - torch.finfo(dtype).eps / 2 * four.abs() - (WIDTH + 2) * U * mag * 1.5).max()) <= 0
