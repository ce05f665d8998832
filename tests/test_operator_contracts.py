"""What the layer norm, distillation and 4-bit operators promise beyond their values: derivatives are formed or refused, never lost."""
import pytest
import torch
from torch.autograd import forward_ad

from dreamer_amd import _native as N
from dreamer_amd import losses, norm


def test_a_tensor_with_a_tangent_wants_its_derivative():
    """A dual tensor has requires_grad == False; it must not pass for one without derivatives."""
    x, w = torch.randn(4, 8), torch.ones(8)
    assert not N.wants_grad(x) and not N.wants_grad(x, w, w)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        dual_w = forward_ad.make_dual(w, torch.ones_like(w))
        assert not dual.requires_grad
        for args in ((dual,), (x, dual_w), (x, w, dual_w), (x, None, dual_w)):
            assert N.wants_grad(*args), args
            with torch.no_grad():                       # switches off reverse mode only
                assert N.wants_grad(*args), args
        assert not N.wants_grad(x, w, None)


def test_the_teacher_has_no_derivative_in_either_mode():
    s, t = torch.randn(4, 8), torch.randn(4, 8)
    values, idx = t.topk(3, 1)
    lse = torch.logsumexp(t, 1)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(values, torch.ones_like(values))
        assert forward_ad.unpack_dual(losses.distill_topk_rows(s, dual, idx)).tangent is None
        assert forward_ad.unpack_dual(losses.distill_topk_rows(s, dual, idx, 1.0, forward_ad.make_dual(lse, lse))).tangent is None
        moved = forward_ad.unpack_dual(losses.distill_topk_rows(forward_ad.make_dual(s, torch.ones_like(s)), values, idx)).tangent
    assert moved is not None and float(moved.abs().max()) < 1e-5     # all logits moved alike: the softmax does not change


def test_layer_norm_takes_weight_and_bias_of_one_type():
    """As on the device (a tensor that moves there must not be refused by a call that worked before)."""
    x, one = torch.randn(4, 8).bfloat16(), torch.ones(8)
    for w, b in ((one, one.bfloat16()), (one.bfloat16(), one)):
        with pytest.raises(N.NativeError, match="weight is"):
            norm.layer_norm(x, w, b)
    for w, b in ((one, one), (one.bfloat16(), one.bfloat16()), (one, None), (None, one.bfloat16())):
        assert norm.layer_norm(x, w, b).dtype == torch.bfloat16


def test_products_of_too_many_tiles_are_refused():
    """A launch takes fewer than 2^32 threads along an axis, 512 of them a tile of 128 x 128 outputs."""
    L, P, big = N.lib(), 1 << 20, 1 << 60
    for M, rows in ((33, 2 ** 30), (33, 2 ** 31 - 300), (128 * 65535, 128 * 129)):
        rc = L.drm_mx4_linear(P, 32, 1, P, P, None, 0, P, rows, M, rows, 32, P, big, None)
        assert rc == -95 and "too many tiles" in L.drm_last_error().decode()
    rc = L.drm_mx4_product(P, P, P, P, None, 0, P, 2 ** 30, 1, 128 * 65535, 2 ** 30, 32, P, big, None)
    assert rc == -95 and "too many tiles" in L.drm_last_error().decode()
