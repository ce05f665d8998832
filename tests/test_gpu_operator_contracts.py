"""What the layer norm, distillation and 4-bit operators promise beyond their values, on the device."""
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
        for n, call in enumerate(calls):
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
