"""The loops of the layer norm and 4-bit kernels at every number of turns: passes of the few-row products, steps of the tile
products' ring, rows beyond the first that a workgroup of the layer norm takes; and rows of a batch that do not depend on the others."""
import pytest
import torch

from dreamer_amd import losses, mx4, norm
from test_gpu_mx4 import BF16, DEV, F16, F32, PARTS, U, _bound, weight
from test_gpu_norm import _check, _inputs

pytestmark = pytest.mark.gpu


def _against_64_bits(x, w, b, dtype):
    w64, x64 = w.dequantize().double(), x.double()
    y, ref = mx4.linear(x, w, b), x64 @ w64.t() + (0 if b is None else b.double())
    assert float(((y.double() - ref).abs() - _bound(x64, w64, b, ref, x.shape[1], PARTS[dtype], dtype)).max()) <= 0
    return y


# A wave takes 128 of the reduction at a time; eight waves (two-byte rows up to 16) or four share it: up to 4096 gives one to four turns
# of eight and one to eight of four.  The weight's rows choose 16, 32 or 64 of them per workgroup.
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [1, 16, 17, 32])
@pytest.mark.parametrize("Nn", [40, 6150, 12300])
def test_few_rows_at_every_number_of_turns(M, Nn, dtype):
    g = torch.Generator(device=DEV).manual_seed(M + Nn)
    b = torch.randn(Nn, generator=g, device=DEV).to(dtype)
    for K in (8, 512, 520, 1024, 1032, 1544, 2048, 2056, 2568, 3080, 3592, 4096):
        x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
        _against_64_bits(x, weight(Nn, K, scale=0.3), b, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M", [1, 16, 17, 32])
def test_few_rows_that_start_anywhere_at_every_number_of_turns(M, dtype):
    g = torch.Generator(device=DEV).manual_seed(M)
    for K in (1, 7, 1027, 2049, 3100, 4095):
        x = torch.randn(M, K + 3, generator=g, device=DEV).to(dtype)[:, 1:K + 1]
        _against_64_bits(x, weight(70, K, scale=0.3), None, dtype)


# 128 of the reduction a step, three stages: every remainder of the number of steps, with and without a last partial chunk, whole and
# split over workgroups (few tiles, a long reduction)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,Nn,K", [(40, 128 * i, 128 * j) for i, j in ((1, 3), (2, 4), (3, 2), (4, 5), (5, 1), (6, 7), (7, 6))]
                         + [(130, 200, 128 * j + 8) for j in (1, 2, 3, 4)] + [(33, 392, 4224), (64, 4224, 136), (100, 2184, 2176), (129, 1000, 6400)])
def test_tile_products_at_every_number_of_steps(M, Nn, K, dtype):
    g = torch.Generator(device=DEV).manual_seed(M + Nn + K)
    w = weight(Nn, K, scale=0.3)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype).requires_grad_()
    dy = torch.randn(M, Nn, generator=g, device=DEV).to(dtype)
    _against_64_bits(x.detach(), w, None, dtype)
    (dx,) = torch.autograd.grad(mx4.linear(x, w), x, dy)
    w64, d64 = w.dequantize().double(), dy.double()
    ref = d64 @ w64
    assert float(((dx.double() - ref).abs() - _bound(d64, w64.t(), None, ref, Nn, PARTS[dtype], dtype)).max()) <= 0
    a = mx4.quantize(x.detach())
    a64 = a.dequantize().double()
    y, ref = mx4.linear(a, w, out_dtype=dtype), a64 @ w64.t()
    assert float(((y.double() - ref).abs() - _bound(a64, w64, None, ref, K, 1, dtype)).max()) <= 0


# More rows than the workgroups of one launch take at once, with a remainder: 8192 workgroups of several rows (up to 64 threads a row)
# or of one, 4096 and 512 of the larger ones; 64 workgroups of four rows under way backward above 16384 elements.
@pytest.mark.parametrize("rows,E,dtype,wdtype", [
    (262200, 24, F32, F32), (530000, 24, BF16, BF16), (131100, 120, BF16, F32), (33000, 513, F32, F32), (33000, 1000, F16, F16), (8200, 1100, F32, F32),
    (8200, 2048, BF16, F32), (8201, 4000, F16, F32), (4100, 4100, F32, F32), (4099, 8000, BF16, F32), (520, 8200, F32, F32), (515, 16384, BF16, BF16),
    (520, 16392, BF16, F32), (1030, 32768, F16, F16), (261, 16400, F32, F32), (261, 16400, BF16, F32), (4099, 16390, F32, F32), (530000, 3, F32, F32),
    (600001, 7, BF16, F32)])
def test_layer_norm_of_more_rows_than_workgroups(rows, E, dtype, wdtype):
    _check(*_inputs(rows, E, dtype, wdtype))


def _stay_as_they_are(call, x, cut):
    """Rows [0, cut) alone give what they give in the batch, whatever the other rows hold; repeated calls give the same bits."""
    y = call(x)
    assert torch.equal(y, call(x)) and torch.equal(y[:cut], call(x[:cut].contiguous()))
    for other in (1e4, float("nan"), float("inf")):
        z = x.clone()
        z[cut:] = other
        assert torch.equal(y[:cut], call(z)[:cut])
    z = torch.cat([x[cut:], x[:cut]])
    assert torch.equal(call(z), torch.cat([y[cut:], y[:cut]]))


# (the same kernel and the same split of the reduction serve both numbers of rows: 16 or 32 rows a workgroup, or tiles of a
# reduction that is too short to be split)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("M,cut", [(16, 1), (16, 9), (32, 17), (40, 33), (200, 130), (300, 257)])
def test_rows_of_a_product_do_not_depend_on_the_others(M, cut, dtype):
    w = weight(96, 160, 3)
    x = torch.randn(M, 160, device=DEV).to(dtype)
    if cut in (33, 130, 257):                            # the rows behind the cut alone are fewer than a tile kernel's
        y = mx4.linear(x, w)
        assert torch.equal(y[:cut], mx4.linear(x[:cut], w))
        for other in (1e4, float("nan"), float("inf")):
            z = x.clone()
            z[cut:] = other
            assert torch.equal(y[:cut], mx4.linear(z, w)[:cut])
    else:
        _stay_as_they_are(lambda t: mx4.linear(t, w), x, cut)
    _stay_as_they_are(lambda t: mx4.linear(mx4.quantize(t), w, out_dtype=F32), x, cut)
    if M > cut:
        dy = torch.randn(M, 96, device=DEV).to(dtype)

        def grad(t):
            leaf = torch.zeros(t.shape[0], 160, device=DEV, dtype=dtype, requires_grad=True)
            return torch.autograd.grad(mx4.linear(leaf, w), leaf, t)[0]

        _stay_as_they_are(grad, dy, cut)


@pytest.mark.parametrize("E", [5, 100, 700, 5000, 20000])
def test_rows_of_a_layer_norm_do_not_depend_on_the_others(E):
    x = torch.randn(37, E, device=DEV)
    _stay_as_they_are(lambda t: norm.layer_norm(t), x, 20)

    def grad(t):
        leaf = t.clone().requires_grad_()
        return torch.autograd.grad(norm.layer_norm(leaf), leaf, torch.ones_like(leaf) + leaf.detach().sign())[0]

    _stay_as_they_are(grad, x, 20)


@pytest.mark.parametrize("V", [50, 3000, 5000, 40000])
@pytest.mark.parametrize("rest", [False, True])
def test_rows_of_a_distillation_do_not_depend_on_the_others(V, rest):
    teacher = torch.randn(7, V, device=DEV)
    values, idx = teacher[:1].topk(9, 1)                 # one list for every row
    lse = torch.logsumexp(teacher[:1], 1) if rest else None

    def call(t):
        n = t.shape[0]
        return losses.distill_topk_rows(t, values.expand(n, -1), idx.expand(n, -1), 1.0, None if lse is None else lse.expand(n))

    def grad(t):
        leaf = t.clone().requires_grad_()
        return torch.autograd.grad(call(leaf).sum(), leaf)[0]

    _stay_as_they_are(call, teacher + torch.randn(7, V, device=DEV), 4)
    _stay_as_they_are(grad, teacher + torch.randn(7, V, device=DEV), 4)
