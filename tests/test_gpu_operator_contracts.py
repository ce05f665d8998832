"""What the layer norm, distillation and 4-bit operators promise beyond their values, on the device."""
import threading

import pytest
import torch
from torch.autograd import forward_ad

from dreamer_amd import _native as N
from dreamer_amd import losses, mx4, norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def test_forward_mode_derivatives_are_refused():
    """The kernels form no tangent: a dual tensor is refused with and without reverse mode, and nothing else is."""
    x, w, b = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    q = mx4.quantize(torch.randn(24, 64, device=DEV))
    b4 = torch.zeros(24, device=DEV)
    layer = mx4.MX4Linear(q, b4, activations="mx4")
    values, idx = torch.randn(4, 64, device=DEV).topk(5, 1)
    plain = norm.layer_norm(x, w, b)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: norm.layer_norm(dual(x), w, b), lambda: norm.layer_norm(x, dual(w), b), lambda: norm.layer_norm(x, None, dual(b)),
                 lambda: norm.layer_norm(dual(x).view(2, 2, 64)), lambda: mx4.linear(dual(x), q), lambda: mx4.linear(x, q, dual(b4)),
                 lambda: losses.distill_topk_rows(dual(x), values, idx)]
        for call in calls:
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        with torch.no_grad(), pytest.raises(N.NativeError, match="no gradient"):
            layer(dual(x))
        # the teacher's side has no derivative by definition, and tensors without a tangent are served as ever
        loss = losses.distill_topk_rows(x, dual(values), idx)
        assert forward_ad.unpack_dual(loss).tangent is None and torch.equal(loss, losses.distill_topk_rows(x, values, idx))
        assert torch.equal(norm.layer_norm(x, w, b), plain)


@pytest.mark.parametrize("rows", [3, 40])
def test_a_4_bit_weight_that_is_exchanged_keeps_the_gradient_of_the_product(rows):
    """Other tensors put into the MX4Tensor between the product and its gradient (a weight that is quantised anew)."""
    for columns in (64, 96):
        w, other = mx4.quantize(torch.randn(24, 64, device=DEV)), mx4.quantize(torch.randn(24, columns, device=DEV))
        x = torch.randn(rows, 64, device=DEV, requires_grad=True)
        dy = torch.randn(rows, 24, device=DEV)
        (want,) = torch.autograd.grad(mx4.linear(x, w), x, dy)
        y = mx4.linear(x, w)
        w.codes, w.scales, w.columns = other.codes, other.scales, columns
        (dx,) = torch.autograd.grad(y, x, dy)
        assert torch.equal(dx, want)


@pytest.mark.parametrize("dtype,bias_dtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_a_product_of_4_bit_rows_has_its_bias_gradient(rows, dtype, bias_dtype):
    g = torch.Generator(device=DEV).manual_seed(rows)
    a, w = mx4.quantize(torch.randn(rows, 96, generator=g, device=DEV)), mx4.quantize(torch.randn(40, 96, generator=g, device=DEV))
    b = torch.randn(2, 40, generator=g, device=DEV).to(bias_dtype).t()[:, 0].requires_grad_()       # (not contiguous)
    y = mx4.linear(a, w, b, out_dtype=dtype)
    dy = torch.randn(rows, 40, generator=g, device=DEV).to(dtype)
    (db,) = torch.autograd.grad(y, b, dy, retain_graph=True)
    ref = dy.double().sum(0)
    tol = torch.finfo(bias_dtype).eps / 2 * ref.abs() + rows * U * dy.double().abs().sum(0)          # rows additions in fp32, one rounding
    assert db.dtype == bias_dtype and float(((db.double() - ref).abs() - tol).max()) <= 0
    (gb,) = torch.autograd.grad(y, b, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        gb.sum().backward()
    with torch.no_grad():
        plain = mx4.linear(a, w, b, out_dtype=dtype)
    assert torch.equal(plain, y.detach()) and not plain.requires_grad and not mx4.linear(a, w).requires_grad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        mx4.linear(a, w, forward_ad.make_dual(b.detach(), torch.ones(40, device=DEV, dtype=bias_dtype)))


def test_on_another_stream_and_in_a_recorded_graph():
    """The product of two 4-bit matrices with the gradient of its bias."""
    g = torch.Generator(device=DEV).manual_seed(5)
    x, w = torch.randn(70, 4096, generator=g, device=DEV), mx4.quantize(torch.randn(200, 4096, generator=g, device=DEV))
    b = torch.randn(200, generator=g, device=DEV)

    def step(rows, bias):
        bias = bias.detach().requires_grad_()                 # a leaf of its own
        y = mx4.linear(mx4.quantize(rows), w, bias)
        return [y.detach(), *torch.autograd.grad((y * rows[:, :200]).sum(), bias)]

    eager = step(x, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step(x, b)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(eager, other))
    xs, bs = x.clone(), b.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, bs)
    for n in range(3):
        xs.copy_(x * (n + 1))
        bs.copy_(b - n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step(xs.clone(), bs.clone())))


def test_two_threads_on_streams_of_their_own():
    """Nothing is shared between calls: two threads, each on its stream with tensors of its own, get what one gets."""
    w = mx4.quantize(torch.randn(300, 2048, device=DEV))

    def step(x, values, idx):
        leaf = x.clone().requires_grad_()
        y = mx4.linear(norm.layer_norm(leaf), w)
        z = mx4.linear(mx4.quantize(leaf), w)
        loss = losses.distill_topk_rows(y, values, idx, 2.0)
        return [y.detach(), z, loss.detach(), torch.autograd.grad(loss.sum(), leaf)[0]]

    work = []
    for n in range(2):
        x = torch.randn(50 + 30 * n, 2048, device=DEV)
        work.append((x, *torch.randn(x.shape[0], 300, device=DEV).topk(7, 1)))
    want = [step(*job) for job in work]
    torch.cuda.synchronize()
    wrong = [None, None]

    def run(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                wrong[n] = [i for i in range(40) if not all(torch.equal(p, q) for p, q in zip(step(*work[n]), want[n]))]
        except Exception as e:                                # (a thread's exception does not reach the test by itself)
            wrong[n] = e

    threads = [threading.Thread(target=run, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [[], []]


# A launch takes fewer than 2^32 threads along an axis: one workgroup per row, or per tile of a weight's rows, reaches that.
def test_distillation_of_more_rows_than_one_grid_axis_takes():
    part, times, V = 1021, 65731, 2                  # 2^26 rows and some of 64 threads each; every row repeats one of 1021
    g = torch.Generator(device=DEV).manual_seed(1)
    s, values = torch.randn(part, V, generator=g, device=DEV).to(F16), torch.randn(part, 1, generator=g, device=DEV)
    idx = torch.randint(-1, V, (part, 1), generator=g, device=DEV)
    lse = values.flatten() + 0.5
    dy = torch.rand(part, generator=g, device=DEV)
    few = s.clone().requires_grad_()
    want = losses.distill_topk_rows(few, values, idx, 1.0, lse)
    (want_grad,) = torch.autograd.grad(want, few, dy)
    many = s.repeat(times, 1).requires_grad_()
    assert many.shape[0] > 2 ** 26
    got = losses.distill_topk_rows(many, values.repeat(times, 1), idx.repeat(times, 1), 1.0, lse.repeat(times))
    (grad,) = torch.autograd.grad(got, many, dy.repeat(times))
    assert bool((got.detach().view(times, part) == want.detach()).all()) and bool((grad.view(times, part, V) == want_grad).all())


@pytest.mark.parametrize("K,rows", [(30, 2 ** 27 + 40), (32, 2 ** 29 + 100)])
def test_few_rows_and_a_weight_of_more_rows_than_one_grid_axis_takes(K, rows):
    part = 3 * 2 ** 12 - 4                           # (no multiple of a workgroup's weight rows)
    g = torch.Generator(device=DEV).manual_seed(2)
    w = mx4.quantize(torch.randn(part, K, generator=g, device=DEV))
    x = torch.randn(1, K, generator=g, device=DEV).to(BF16)
    times = -(-rows // part)
    codes, scales = (t.repeat(times, 1)[:rows] for t in (w.codes, w.scales))
    y = mx4.linear(x, mx4.MX4Tensor(codes, scales, K))
    del codes, scales
    # a sum of K <= 32 exact products in another order (another kernel may serve the short weight), rounded once
    ref = x.double() @ w.dequantize().double().t()
    tol = 2.0 ** -8 * ref.abs() + (K + 2) * U * (x.double().abs() @ w.dequantize().double().abs().t())
    whole = rows // part
    body = y[:, :whole * part].view(whole, part)
    assert bool((body == body[0]).all()) and bool((y[0, whole * part:] == body[0, :rows - whole * part]).all())
    assert float(((body[:1].double() - ref).abs() - tol).max()) <= 0


def test_column_sums_of_rows_longer_than_one_grid_axis_takes():
    E = 2 ** 26 + 3                                  # 2 E sums, joined 32 a workgroup of 1024 threads
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(1, E, generator=g, device=DEV)
    w, b = torch.ones(E, device=DEV, requires_grad=True), torch.zeros(E, device=DEV, requires_grad=True)
    dy = torch.randn(1, E, generator=g, device=DEV)
    y = norm.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(db, dy[0])                    # one row: its own gradient
    # dw = dy xh, and y = xh: one product, of two factors that are each the kernel's own to a few half steps (xh is formed as
    # (x - m) r in both passes: a difference, a product, and a fused step with w = 1, b = 0)
    want = dy[0].double() * y.detach()[0].double()
    assert float(((dw.double() - want).abs() - 8 * U * want.abs()).max()) <= 0
