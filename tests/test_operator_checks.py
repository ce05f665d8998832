"""Argument checks of the layer norm, distillation and 4-bit entry points (they run before anything touches a device), and the
host forms of the first two."""
import math

import pytest
import torch

from dreamer_amd import _native as N
from dreamer_amd import losses, mx4, norm

EINVAL, ENOTSUP = -22, -95
P = 1 << 20     # stands for an aligned device pointer; the calls below are refused before it is used


def _err(rc, code, text):
    assert rc == code and text in N.lib().drm_last_error().decode(), (rc, N.lib().drm_last_error())


def test_layer_norm_entry_points_refuse():
    L = N.lib()
    fwd = lambda x=P, ldx=8, xt=0, w=P, b=P, wt=0, y=P, ldy=8, m=P, r=P, n=4, e=8: L.drm_layer_norm_forward(x, ldx, xt, w, b, wt, y, ldy, m, r, n, e, 1e-5, None)
    _err(fwd(x=None), EINVAL, "null")
    _err(fwd(y=None), EINVAL, "null")
    _err(fwd(ldx=7), EINVAL, "stride")
    _err(fwd(ldy=7), EINVAL, "stride")
    _err(fwd(xt=3), ENOTSUP, "types")
    _err(fwd(xt=1, wt=2), ENOTSUP, "types")
    _err(fwd(e=0), EINVAL, "E=0")
    _err(fwd(n=-1), EINVAL, "N=-1")
    _err(fwd(m=None), EINVAL, "together")
    assert fwd(n=0) == 0
    need = L.drm_layer_norm_workspace_bytes(4, 8)
    assert need > 0 and L.drm_layer_norm_workspace_bytes(-1, 8) == 0 and L.drm_layer_norm_workspace_bytes(4, 0) == 0
    bwd = lambda ws=P, nbytes=need, dx=P, dw=P, db=P, dy=P, mean=P, n=4, e=8, lddy=8: L.drm_layer_norm_backward(
        P, 8, dy, lddy, 0, P, 0, mean, P, dx, dw, db, n, e, ws, nbytes, None)
    _err(bwd(ws=None), EINVAL, "workspace")
    _err(bwd(nbytes=need - 1), EINVAL, "workspace")
    _err(bwd(dy=None), EINVAL, "null")
    _err(bwd(mean=None), EINVAL, "null")
    _err(bwd(lddy=7), EINVAL, "stride")
    _err(bwd(e=0), EINVAL, "E=0")
    assert bwd(dx=None, dw=None, db=None) == 0
    assert bwd(n=0, dw=None, db=None) == 0


def test_distill_entry_points_refuse():
    L = N.lib()
    fwd = lambda s=P, lds=10, dt=0, val=P, ldv=3, idx=P, ldi=3, rows=4, V=10, k=3, t=1.0, loss=P, p=P, row=P, ws=None, nb=0: L.drm_distill_topk_forward(
        s, lds, dt, val, ldv, idx, ldi, None, rows, V, k, t, loss, p, row, ws, nb, None)
    _err(fwd(s=None), EINVAL, "null")
    _err(fwd(idx=None), EINVAL, "null")
    _err(fwd(val=None), EINVAL, "null")
    _err(fwd(loss=None), EINVAL, "null")
    _err(fwd(p=None), EINVAL, "null")
    _err(fwd(lds=9), EINVAL, "stride")
    _err(fwd(ldv=2), EINVAL, "stride")
    _err(fwd(ldi=2), EINVAL, "stride")
    _err(fwd(dt=7), ENOTSUP, "type")
    _err(fwd(k=-1), EINVAL, "k=-1")
    _err(fwd(k=1025, ldi=1025, ldv=1025), ENOTSUP, "1025")
    _err(fwd(V=0), EINVAL, "V=0")
    _err(fwd(rows=-1), EINVAL, "rows=-1")
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-7):
        _err(fwd(t=t), EINVAL, "temperature")
    _err(fwd(row=P + 8), EINVAL, "aligned")
    assert L.drm_distill_topk_workspace_bytes(4, 1000) == 0
    need = L.drm_distill_topk_workspace_bytes(4, 200000)
    assert need > 0
    _err(fwd(V=200000, lds=200000), EINVAL, "workspace")
    _err(fwd(V=200000, lds=200000, ws=P, nb=need - 1), EINVAL, "workspace")
    _err(fwd(rows=2 ** 31, V=200000, lds=200000, ws=P, nb=2 ** 50), ENOTSUP, "rows")
    assert fwd(rows=0) == 0
    bwd = lambda s=P, p=P, row=P, g=P, d=P, t=1.0: L.drm_distill_topk_backward(s, 10, 0, P, 3, p, row, g, 4, 10, 3, t, d, None)
    for kw in (dict(s=None), dict(p=None), dict(row=None), dict(g=None), dict(d=None)):
        _err(bwd(**kw), EINVAL, "null")
    _err(bwd(row=P + 4), EINVAL, "aligned")
    _err(bwd(t=0.0), EINVAL, "temperature")


def test_mx4_entry_points_refuse():
    L = N.lib()
    _err(L.drm_mx4_quantize(None, 32, 0, 4, 32, P, P, None), EINVAL, "null")
    _err(L.drm_mx4_quantize(P, 31, 0, 4, 32, P, P, None), EINVAL, "stride")
    _err(L.drm_mx4_quantize(P, 32, 5, 4, 32, P, P, None), ENOTSUP, "type")
    _err(L.drm_mx4_quantize(P, 32, 0, 4, 32, P + 8, P, None), EINVAL, "misaligned")
    _err(L.drm_mx4_quantize(P, 32, 0, 4, 0, P, P, None), EINVAL, "K=0")
    _err(L.drm_mx4_quantize(P, 32, 0, -4, 32, P, P, None), EINVAL, "rows=-4")
    assert L.drm_mx4_quantize(None, 32, 0, 0, 32, None, None, None) == 0
    _err(L.drm_mx4_dequantize(P, P, 4, 32, None, 32, 0, None), EINVAL, "null")
    _err(L.drm_mx4_dequantize(P, P, 4, 32, P, 31, 0, None), EINVAL, "stride")
    lin = lambda x=P, ldx=32, dt=0, c=P, s=P, b=None, bt=0, y=P, ldy=8, M=4, n=8, K=32, ws=P, nb=1 << 40: L.drm_mx4_linear(x, ldx, dt, c, s, b, bt, y, ldy, M, n, K, ws, nb, None)
    for kw in (dict(x=None), dict(c=None), dict(s=None), dict(y=None)):
        _err(lin(**kw), EINVAL, "null")
    _err(lin(ldx=31), EINVAL, "stride")
    _err(lin(ldy=7), EINVAL, "stride")
    _err(lin(dt=3), ENOTSUP, "types")
    _err(lin(b=P, bt=3), ENOTSUP, "types")
    _err(lin(M=-1), EINVAL, "M=-1")
    _err(lin(n=0, ldy=0), EINVAL, "N=0")
    _err(lin(M=2 ** 31 - 300), ENOTSUP, "at most")
    assert lin(M=0) == 0
    need = L.drm_mx4_linear_workspace_bytes(0, 100, 128, 4096)
    assert need > 0 and L.drm_mx4_linear_workspace_bytes(0, 4, 128, 4096) == 0 and L.drm_mx4_linear_workspace_bytes(9, 100, 128, 4096) == 0
    for ws, nb in ((None, 0), (P, need - 1), (P + 8, need)):
        _err(lin(M=100, n=128, K=4096, ldx=4096, ldy=128, ws=ws, nb=nb), EINVAL, "workspace")
    grad = lambda **kw: L.drm_mx4_linear_dgrad(*[dict(dict(dy=P, ld=8, dt=0, c=P, s=P, dx=P, ldx=32, M=4, N=8, K=32), **kw)[k] for k in
                                                 ("dy", "ld", "dt", "c", "s", "dx", "ldx", "M", "N", "K")], P, 1 << 40, None)
    for kw in (dict(dy=None), dict(dx=None), dict(c=None)):
        _err(grad(**kw), EINVAL, "null")
    _err(grad(ld=7), EINVAL, "stride")
    _err(grad(ldx=31), EINVAL, "stride")
    prod = lambda **kw: L.drm_mx4_product(*[dict(dict(a=P, sa=P, w=P, sw=P, b=None, bt=0, y=P, ldy=8, yt=0, M=4, N=8, K=32), **kw)[k] for k in
                                            ("a", "sa", "w", "sw", "b", "bt", "y", "ldy", "yt", "M", "N", "K")], P, 1 << 40, None)
    for kw in (dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(y=None)):
        _err(prod(**kw), EINVAL, "null")
    _err(prod(ldy=7), EINVAL, "stride")
    _err(prod(yt=9), ENOTSUP, "types")
    _err(prod(a=P + 4), EINVAL, "misaligned")
    _err(L.drm_mx4_bias_grad(P, 8, 0, P, 0, 4, 8, None, 0, None), EINVAL, "workspace")
    _err(L.drm_mx4_bias_grad(P, 7, 0, P, 0, 4, 8, P, 1 << 20, None), EINVAL, "stride")
    _err(L.drm_mx4_bias_grad(P, 8, 0, None, 0, 4, 8, P, 1 << 20, None), EINVAL, "null")


def test_python_entry_points_refuse_host_tensors_and_shapes():
    x = torch.randn(4, 64)
    with pytest.raises(N.NativeError, match="HIP device"):
        mx4.quantize(x)
    with pytest.raises(N.NativeError, match="HIP device"):
        mx4.MX4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64)
    with pytest.raises(N.NativeError, match="at least one"):
        norm.layer_norm(torch.zeros(4, 0))
    with pytest.raises(N.NativeError, match="weight"):
        norm.layer_norm(x, torch.ones(63))
    with pytest.raises(ValueError, match="last dimension"):
        norm.LayerNorm((4, 64))
    with pytest.raises(ValueError, match="64 elements"):
        norm.LayerNorm(64)(x[:, :32])
    with pytest.raises(N.NativeError, match="does not match"):
        losses.distill_topk_rows(x, x[:, :3], torch.zeros(4, 2, dtype=torch.int64))
    with pytest.raises(ValueError, match="temperature"):
        losses.distill_topk_rows(x, x[:, :2], torch.zeros(4, 2, dtype=torch.int64), temperature=float("nan"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_norm_on_the_host(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 40, generator=g).to(dtype).requires_grad_()
    ln = norm.LayerNorm(40)
    with torch.no_grad():
        ln.weight.uniform_(0.5, 1.5, generator=g)
        ln.bias.uniform_(-1, 1, generator=g)
    y = ln(x)
    ref = torch.nn.functional.layer_norm(x.detach().double(), (40,), ln.weight.double(), ln.bias.double())
    # half a step of the type, and 128 fp32 half steps of values up to 4 * 1.5 + 1
    assert y.dtype == dtype and float(((y.double() - ref).abs() - torch.finfo(dtype).eps / 2 * ref.abs()).max()) < 128 * 2.0 ** -24 * 7
    assert list(ln.state_dict()) == ["weight", "bias"]


def test_distillation_on_the_host_equals_the_divergence_of_full_lists():
    g = torch.Generator().manual_seed(2)
    s, t = torch.randn(6, 20, generator=g), torch.randn(6, 20, generator=g)
    values, idx = t.topk(20, 1)
    for T in (0.5, 1.0, 3.0):
        p = torch.softmax(t.double() / T, 1)
        want = (p * (p.log() - torch.log_softmax(s.double() / T, 1))).sum(1)
        for lse in (None, torch.logsumexp(t / T, 1)):
            got = losses.distill_topk_rows(s, values, idx, T, lse)
            # 20 terms, logarithms up to 10 / T: fp32 half steps
            assert float((got.double() - want).abs().max()) < 20 * 4 * (10 / T) * 2.0 ** -24
    few = losses.distill_topk_rows(s, values[:, :3], idx[:, :3], 1.0, torch.logsumexp(t, 1))
    p = torch.softmax(t.double(), 1)
    q = torch.softmax(s.double(), 1)
    for r in range(6):
        want = sum(float(p[r, i]) * math.log(float(p[r, i] / q[r, i])) for i in idx[r, :3].tolist())
        P, Q = 1 - float(p[r, idx[r, :3]].sum()), 1 - float(q[r, idx[r, :3]].sum())
        assert abs(float(few[r]) - want - P * math.log(P / Q)) < 20 * 40 * 2.0 ** -24
