"""LayerNorm without activation (forward, backward, weight-gradient reduction) against the formula in 64 bits."""
import pytest
import torch

from dreamer_amd import _native as N
from dreamer_amd import norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _reference(x, w, b, dy, eps):
    x, dy = x.detach().double(), dy.double()
    E = x.shape[-1]
    w = torch.ones(E, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    m = x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((x - m).square().mean(1, keepdim=True) + eps)
    xh = (x - m) * r
    g = dy * w
    y = xh * w + (0.0 if b is None else b.detach().double())
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, dx, (dy * xh).sum(0), dy.sum(0), xh, r, w


def _tolerances(x, w, b, dy, ref, n_rows):
    """Half a step of the result's type, and the fp32 arithmetic: a row sum passes at most 16 additions in a thread and 10 between
    threads, each off by half a step of a partial sum that is at most the sum of magnitudes; m, the variance and the two gradient means
    are four such sums, products and differences add fewer than 24 steps: 128 half steps of the largest magnitudes in all."""
    y, dx, dw, db, xh, r, w64 = ref
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    d = dy.double()
    A = x.detach().double().abs().amax(1, keepdim=True) * r          # size of a normalised value, with the row's offset
    y_tol = half * y.abs() + 128 * U * (A * w64.abs() + (0.0 if b is None else b.detach().double().abs())) + tiny
    G = (d * w64).abs().amax(1, keepdim=True)
    dx_tol = half * dx.abs() + 128 * U * r * G * (1 + (A + 1) ** 2) + tiny
    wd = F32 if w is None else w.dtype
    halfw = torch.finfo(wd).eps / 2
    depth = -(-n_rows // 512) + 512 // 4 + 16                        # rows of a workgroup, its partial sums, the columns' tree
    dw_tol = halfw * dw.abs() + U * (depth * (d * xh).abs().sum(0) + 128 * (d.abs() * (A + 1)).sum(0))
    db_tol = halfw * db.abs() + U * depth * d.abs().sum(0)
    return y_tol, dx_tol, dw_tol, db_tol


def _inputs(rows, E, dtype, wdtype, stride=None, seed=0, offset=0.5):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * rows + E)
    x = (torch.randn(rows, stride or E, generator=g, device=DEV) + offset * torch.randn(rows, 1, generator=g, device=DEV)).to(dtype)[:, :E]
    w = (1 + 0.3 * torch.randn(E, generator=g, device=DEV)).to(wdtype)
    b = (0.3 * torch.randn(E, generator=g, device=DEV)).to(wdtype)
    dy = torch.randn(rows, E, generator=g, device=DEV).to(dtype)
    return x.requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy


def _check(x, w, b, dy, eps=1e-5):
    y = norm.layer_norm(x, w, b, eps)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == x.shape
    ref = _reference(x, w, b, dy, eps)
    tols = _tolerances(x, w, b, dy, ref, x.shape[0])
    got = [y.detach(), grads[0]] + list(grads[1:])
    names = ["y", "dx"] + (["dw"] if w is not None else []) + (["db"] if b is not None else [])
    want = {"y": (ref[0], tols[0]), "dx": (ref[1], tols[1]), "dw": (ref[2], tols[2]), "db": (ref[3], tols[3])}
    for name, t in zip(names, got):
        r, tol = want[name]
        bad = (t.double() - r).abs() - tol
        assert not torch.isnan(t).any() and float(bad.max()) <= 0, (name, float(bad.max()), float((t.double() - r).abs().max()))
    return got


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)])
@pytest.mark.parametrize("rows,E", [(1, 1), (3, 2), (5, 7), (130, 31), (9, 64), (16, 512), (33, 255), (17, 1000), (4, 1024), (3, 1025),
                                    (600, 2048), (7, 4095), (5, 4096), (2, 8191), (3, 8200), (2, 16384), (3, 16385), (70, 20001)])
def test_values_and_gradients(rows, E, dtype, wdtype):
    _check(*_inputs(rows, E, dtype, wdtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,E,stride", [(37, 33, 34), (5, 1001, 1009), (3, 4096, 4097), (2, 17001, 17003)])
def test_strided_rows_that_start_anywhere(rows, E, stride, dtype):
    _check(*_inputs(rows, E, dtype, dtype, stride=stride))


@pytest.mark.parametrize("rows,E", [(2500, 24), (1030, 513), (5000, 1100)])
def test_many_rows_reduce_into_the_weight_gradient(rows, E):
    a = _check(*_inputs(rows, E, F32, F32))
    b = _check(*_inputs(rows, E, F32, F32))
    assert all(torch.equal(s, t) for s, t in zip(a, b))              # no order of workgroups in the results


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,E,stride", [(70000, 3, 3), (3000, 7, 9), (257, 1, 5), (64, 4, 4), (40, 17000, 17008), (300, 9001, 9001)])
def test_narrow_rows_and_long_ones(rows, E, stride, dtype):
    _check(*_inputs(rows, E, dtype, F32, stride=stride))


def test_rows_far_from_zero_keep_their_digits():
    x, w, b, dy = _inputs(9, 777, F32, F32, offset=1000.0)
    _check(x, w, b, dy)


@pytest.mark.parametrize("E", [40, 20000])
def test_without_weight_or_bias(E):
    x, w, b, dy = _inputs(6, E, BF16, F32)
    _check(x, None, None, dy)
    _check(x, None, b, dy)
    _check(x, w, None, dy)


def test_constant_rows_and_empty_batches():
    x = torch.full((3, 100), 7.25, device=DEV, requires_grad=True)
    w, b = torch.ones(100, device=DEV, requires_grad=True), torch.full((100,), 0.5, device=DEV, requires_grad=True)
    y = norm.layer_norm(x, w, b)
    assert torch.equal(y, torch.full_like(y, 0.5))
    e = torch.zeros(0, 100, device=DEV, requires_grad=True)
    y = norm.layer_norm(e, w, b)
    dx, dw, db = torch.autograd.grad(y, (e, w, b), torch.zeros_like(y))
    assert y.shape == (0, 100) and dx.shape == (0, 100) and float(dw.abs().max()) == 0 and float(db.abs().max()) == 0


def test_infinities_and_nan_stay_in_their_row():
    x, w, b, dy = _inputs(8, 300, F32, F32)
    clean = norm.layer_norm(x, w, b).detach()
    with torch.no_grad():
        x[2, 5] = float("nan")
        x[6, 299] = float("inf")
    y = norm.layer_norm(x, w, b).detach()
    keep = [0, 1, 3, 4, 5, 7]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[2]).all() and torch.isnan(y[6]).all()


def test_leading_dimensions_views_and_expanded_gradients():
    g = torch.Generator(device=DEV).manual_seed(3)
    base = torch.randn(6, 5, 48, generator=g, device=DEV)
    x = base.transpose(0, 1).detach().requires_grad_()
    ln = norm.LayerNorm(48).to(DEV)
    ln(x).sum().backward()                                            # the incoming gradient is an expanded scalar
    flat = base.transpose(0, 1).reshape(-1, 48).detach().requires_grad_()
    y = norm.layer_norm(flat, ln.weight, ln.bias)
    ref = torch.autograd.grad(y, (flat, ln.weight, ln.bias), torch.ones_like(y))
    assert torch.equal(x.grad.reshape(-1, 48), ref[0]) and torch.equal(ln.weight.grad, ref[1]) and torch.equal(ln.bias.grad, ref[2])
    one = torch.randn(9, generator=g, device=DEV)
    assert torch.equal(norm.layer_norm(one), norm.layer_norm(one.view(1, 9)).view(9))
    col = torch.randn(9, 4, generator=g, device=DEV).t()              # columns not contiguous
    assert torch.equal(norm.layer_norm(col), norm.layer_norm(col.contiguous()))
    rep = torch.randn(1, 16, generator=g, device=DEV).expand(4, 16)   # rows that overlap
    assert torch.equal(norm.layer_norm(rep), norm.layer_norm(rep.contiguous()))


def test_gradients_against_differences():
    x, w, b, dy = _inputs(3, 12, F32, F32)
    y = norm.layer_norm(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    h = 2.0 ** -6

    def value(xx, ww, bb):
        return float((norm.layer_norm(xx, ww, bb).double() * dy.double()).sum())

    for t, gr, pos in ((x, grads[0], (1, 5)), (w, grads[1], (7,)), (b, grads[2], (2,))):
        args = [x.detach(), w.detach(), b.detach()]
        k = [i for i, s in enumerate((x, w, b)) if s is t][0]
        up, dn = [a.clone() for a in args], [a.clone() for a in args]
        up[k][pos] += h
        dn[k][pos] -= h
        # central differences: third-order remainder h^2, rounding of 36 values of about 3 over 2 h
        assert abs((value(*up) - value(*dn)) / (2 * h) - float(gr[pos])) < 20 * h * h + 36 * 3 * 8 * U / (2 * h)


def test_rows_beyond_32_bit_offsets():
    stride = 2 ** 30 + 8
    buf = torch.empty(2 * stride + 64, dtype=BF16, device=DEV)
    x = buf.as_strided((3, 64), (stride, 1))
    vals = torch.randn(3, 64, device=DEV).to(BF16)
    x.copy_(vals)
    assert torch.equal(norm.layer_norm(x), norm.layer_norm(vals))


def test_on_another_stream_and_in_a_recorded_graph():
    x, w, b, dy = _inputs(64, 300, BF16, F32)
    eager = norm.layer_norm(x, w, b)
    eager_grads = torch.autograd.grad(eager, (x, w, b), dy, retain_graph=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = norm.layer_norm(x, w, b)
        grads = torch.autograd.grad(y, (x, w, b), dy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, eager) and all(torch.equal(p, q) for p, q in zip(grads, eager_grads))
    graph = torch.cuda.CUDAGraph()
    # leaves of the recording's own: a recorded backward pass may not meet an eager graph of the same leaves that is alive
    xs, ws, bs = (t.detach().clone().requires_grad_() for t in (x, w, b))
    with torch.cuda.graph(graph):
        yg = norm.layer_norm(xs, ws, bs)
        gg = torch.autograd.grad(yg, (xs, ws, bs), dy)
    for k in range(3):
        with torch.no_grad():
            xs.copy_(x.detach() * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        ref = norm.layer_norm(xs.detach().requires_grad_(), w, b)
        assert torch.equal(yg, ref)
        xr = xs.detach().clone().requires_grad_()
        gr = torch.autograd.grad(norm.layer_norm(xr, w, b), (xr, w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(gg, gr))


def test_refusals_on_the_device():
    x = torch.randn(4, 8, device=DEV)
    with pytest.raises(N.NativeError, match="weight"):
        norm.layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(N.NativeError, match="weight is"):
        norm.layer_norm(x.to(BF16), torch.ones(8, device=DEV), torch.ones(8, device=DEV, dtype=BF16))
    with pytest.raises(N.NativeError, match="element types"):
        norm.layer_norm(x, torch.ones(8, device=DEV, dtype=BF16))
    with pytest.raises(N.NativeError, match="weight is on cpu"):
        norm.layer_norm(x, torch.ones(8))
    with pytest.raises(N.NativeError, match="fp32, bf16 or fp16"):
        norm.layer_norm(x.double())
    y = norm.layer_norm(x.requires_grad_())
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
