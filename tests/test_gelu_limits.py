"""The tanh GELU and its slope far out, where h^2 or h^3 leaves fp32: h or 0, and 1 or 0; NaN stays NaN."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import act8_pack, act8_unpack, linear_act8
from vodascheduler_amd.ops.activation import gelu_tanh
from vodascheduler_amd.ops.ffn import gelu_tanh_grad_ref

U = 2.0 ** -24
SIZES = [0.5, 3.0, 7.5, 8.5, 9.0, 10.0, 50.0, 1e3, 1e6, 1e7, 1e10, 1e20, 1e30, 3e38]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _formulas(h):
    """(gelu, slope) in fp64 by the logistic form, whose terms are products of finite numbers."""
    k, c = (2 / torch.pi) ** 0.5, 0.044715
    u = 2 * k * (h + c * h ** 3)
    s, r = torch.sigmoid(u), torch.sigmoid(-u)
    return h * s, s + h * s * r * 2 * k * (1 + 3 * c * h * h)


def _values(dtype, dev):
    t = torch.tensor(SIZES + [-v for v in SIZES] + [0.0], device=dev)
    return torch.cat([t, t, t, t]).to(dtype)[:113]  # whole vectors and a remainder


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_function_and_its_slope(dtype, dev):
    h = _values(dtype, dev).requires_grad_()
    if dev == "cpu":
        slope = gelu_tanh_grad_ref(h.detach()).to(dtype)
        y = None
    else:
        y = gelu_tanh(h)
        (slope,) = torch.autograd.grad(y, h, torch.ones_like(h))
    want, wslope = _formulas(h.detach().double())
    half = torch.finfo(dtype).eps / 2
    # exp2's argument: three roundings of at most 3.3 (|h| < 3.1), or the exponential is below 2^-24 of the result
    # or the result below 1e-6; what is below 2^-50 is 0
    for got, r in ((y, want), (slope, wslope)):
        if got is not None:
            assert torch.isfinite(got).all()
            off = (got.double() - r).abs()
            assert (off <= (half + 64 * U) * r.abs() + 2.0 ** -24).all(), off.max()
            far = h.detach().double() <= -9
            assert (got.double()[far].abs() <= 2.0 ** -50).all()
            up = h.detach().double() >= 9
            assert torch.equal(got[up], r[up].to(dtype))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_through_the_layer(dtype, dev):
    """One feature in a block at the size: y is that feature's weights or 0, dx its gradient or 0."""
    v = torch.tensor([s * v for v in SIZES[4:-1] for s in (1, -1)], device=dev)
    rows, K, N = len(v), 64, 40
    g = torch.Generator(device="cpu").manual_seed(0)
    x = torch.zeros(rows, K, device=dev)
    x[:, 33] = v
    w = (torch.randn(N, K, generator=g) * 0.1).to(dev).to(dtype)
    x, dy = x.to(dtype).requires_grad_(), torch.randn(rows, N, generator=g).to(dev).to(dtype)
    y = linear_act8(x, w, None, "gelu")
    (dx,) = torch.autograd.grad(y, x, dy)
    half = torch.finfo(dtype).eps / 2
    want = _formulas(x.detach().double())[0] @ w.double().t()
    assert ((y.double() - want).abs() <= (2 * half + 8 * U) * want.abs() + 1e-15).all()
    sl = _formulas(act8_unpack(*act8_pack(x), K).double())[1]
    p = dy.double() @ w.double()
    size = dy.double().abs() @ w.double().abs()
    assert ((dx.double() - p * sl).abs() <= (half * p.abs() + (N + 64) * U * size) * sl.abs() + 1e-15 * size).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_nan(dev):
    h = torch.full((9,), float("nan"), device=dev, requires_grad=True)
    y = gelu_tanh(h)
    assert torch.isnan(y).all() and torch.isnan(torch.autograd.grad(y.sum(), h)[0]).all()
    assert torch.isnan(gelu_tanh_grad_ref(h.detach())).all()
