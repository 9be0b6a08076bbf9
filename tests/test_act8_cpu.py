"""ops/act8.py without a GPU: the checkpoint's format, the layer against the formulas in fp64, refusals."""
import pytest
import torch
import torch.nn.functional as F

from vodascheduler_amd.ops.act8 import Act8Linear, act8_pack, act8_unpack, linear_act8

from act8_bounds import checkpoint, formulas
from xent_bounds import within


def special_values(dtype):
    """Blocks whose scale or rounding is at an edge: zeros, the smallest and largest numbers, powers of
    two, 448 and its neighbours, ties, infinities, NaN."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = [[0.0] * 33, [small, -small / 4, 0.0], [big, -big, 1.0], [448.0, 447.0, 1.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10],
            [449.0, 1.0], [896.0, 464.0, 432.0, 17.0, 19.0, 0.25], [1.0, 1 + 2.0 ** -4, 1 + 3 * 2.0 ** -4, 1.75, 0.875],
            [float("inf"), 2.0, -3.0], [float("nan"), 5.0], [float("-inf"), float("nan")], [-0.0, 1e-30, 3e-38]]
    return torch.tensor([r + [0.0] * (40 - len(r)) for r in rows]).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpoint_of_edges(dtype):
    x = special_values(dtype)
    q, s = act8_pack(x)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float8_e8m0fnu
    assert q.shape == (x.shape[0], 64) and s.shape == (x.shape[0], 2)
    got = act8_unpack(q, s, 40)
    torch.testing.assert_close(got.double(), checkpoint(x), rtol=0, atol=0, equal_nan=True)


def test_checkpoint_error_and_idempotence():
    x = torch.randn(64, 100) * torch.exp(3 * torch.randn(64, 1))
    c = act8_unpack(*act8_pack(x), 100)
    top = F.pad(x, (0, 28)).view(64, 4, 32).abs().amax(2).repeat_interleave(32, 1)[:, :100]
    # half a step: 2^-4 of the value, or half of 2^-9 times a scale of at most top / 224
    assert bool(((c - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, top / 224 * 2.0 ** -10)).all())
    assert torch.equal(act8_unpack(*act8_pack(c), 100), c)
    assert torch.equal(act8_unpack(*act8_pack(x), 100, torch.bfloat16).float(), c)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [(1, 1, 1), (5, 33, 7), (40, 64, 24)])
def test_layer_is_the_formula(rows, K, N, dtype, act):
    g = torch.Generator().manual_seed(rows)
    x, w, b, dy = (torch.randn(*s, generator=g).to(dtype).requires_grad_() for s in ((rows, K), (N, K), (N,), (rows, N)))
    y = linear_act8(x, w, b, act)
    got = (y.detach(), *torch.autograd.grad(y, (x, w, b), dy.detach()))
    want, bound = formulas(x, w, b, dy, act)
    for o, r, d, nm in zip(got, want, bound, ("y", "dx", "dw", "db")):
        within(o, r, d, nm)


def test_gradient_is_the_slope_where_the_checkpoint_is_exact():
    """On values that e4m3 holds the layer's gradient is the plain function's: central differences of the
    loss in fp64 (off by h^2, 1e-8, and by fp32's 1e-6 of the layer)."""
    g = torch.Generator().manual_seed(0)
    x = act8_unpack(*act8_pack(torch.randn(6, 40, generator=g)), 40).requires_grad_()
    w = torch.randn(5, 40, generator=g).requires_grad_()
    dy = torch.randn(6, 5, generator=g)
    gx, gw = torch.autograd.grad(linear_act8(x, w, None, "gelu"), (x, w), dy)
    loss = lambda a, c: float((F.linear(F.gelu(a, approximate="tanh"), c) * dy.double()).sum())  # noqa: E731
    X, W, h = x.detach().double(), w.detach().double(), 1e-4
    for d, grad, at in ((torch.randn(6, 40, generator=g).double(), gx, 0), (torch.randn(5, 40, generator=g).double(), gw, 1)):
        up, down = ((loss(X + s * h * d, W) if at == 0 else loss(X, W + s * h * d)) for s in (1, -1))
        want = (up - down) / (2 * h)
        assert abs(want - float((grad.double() * d).sum())) < 1e-5 * (1 + abs(want))


def test_what_is_kept():
    """A byte a value and one a block of 32: nothing of the input's own size is saved."""
    x = torch.randn(64, 256, requires_grad=True)
    layer = Act8Linear(256, 32, act="gelu")
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel() * t.element_size()) or t, lambda t: t):
        y = layer(x)
    assert sum(sizes) == layer.weight.numel() * 4 + 64 * 256 + 64 * 8
    y.sum().backward()
    assert layer.weight.grad is not None and x.grad is not None
    with torch.no_grad():
        torch.testing.assert_close(layer(x), F.linear(F.gelu(x, approximate="tanh"), layer.weight, layer.bias))


def test_a_frozen_weight_keeps_no_checkpoint():
    """Without the GELU dx needs none; with it the slope does."""
    g = torch.Generator().manual_seed(5)
    for act, extra in ((None, 0), ("gelu", 64 * 256 + 64 * 8)):
        x, layer = torch.randn(64, 256, generator=g).requires_grad_(), Act8Linear(256, 32, act=act)
        layer.weight.requires_grad_(False)
        dy, sizes = torch.randn(64, 32, generator=g), []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel() * t.element_size()) or t, lambda t: t):
            y = layer(x)
        assert sum(sizes) == layer.weight.numel() * 4 + extra
        gx, gb = torch.autograd.grad(y, (x, layer.bias), dy)
        layer.weight.requires_grad_(True)
        wx, wb = torch.autograd.grad(layer(x), (x, layer.bias), dy)
        assert torch.equal(gx, wx) and torch.equal(gb, wb)


def test_shapes_and_empty():
    layer = Act8Linear(6, 3)
    assert layer(torch.zeros(2, 5, 6)).shape == (2, 5, 3)
    x = torch.zeros(0, 6, requires_grad=True)
    layer(x).sum().backward()
    assert x.grad.shape == (0, 6)
    assert act8_unpack(*act8_pack(torch.zeros(0, 6)), 6).shape == (0, 6)


@pytest.mark.parametrize("change,error", [
    (dict(act="relu"), ValueError), (dict(x=torch.zeros(4, 6)), ValueError), (dict(weight=torch.zeros(5)), ValueError),
    (dict(bias=torch.zeros(4)), ValueError), (dict(x=torch.zeros(4, 5).half()), TypeError),
    (dict(weight=torch.zeros(3, 5).bfloat16()), TypeError), (dict(bias=torch.zeros(3).half()), TypeError),
    (dict(bias=torch.zeros(3, device="meta")), ValueError), (dict(weight=torch.zeros(0, 5)), ValueError),
])
def test_refusals(change, error):
    args = dict(x=torch.zeros(4, 5), weight=torch.zeros(3, 5), bias=torch.zeros(3))
    linear_act8(**args)
    with pytest.raises(error):
        linear_act8(**{**args, **change})


def test_checkpoint_refusals():
    q, s = act8_pack(torch.zeros(3, 40))
    with pytest.raises(TypeError):
        act8_pack(torch.zeros(3, 4, dtype=torch.float16))
    with pytest.raises(ValueError):
        act8_pack(torch.zeros(3, 0))
    for a in ((q, s, 65), (q, s, 32), (q, s, 0), (q[:, :32], s, 32), (q.view(torch.uint8), s, 40), (q[:2], s, 40)):
        with pytest.raises(ValueError):
            act8_unpack(*a)
    with pytest.raises(TypeError):
        act8_unpack(q, s, 40, torch.float16)


def test_the_host_refuses():
    from vodascheduler_amd.ops import _native

    h = _native.hip()
    for rows, K, N, dt in ((0, 8, 8, 0), (8, 0, 8, 0), (8, 8, 0, 0), (8, 8, 8, 2), (8, 1 << 21, 8, 0), (1 << 30, 8, 8, 0),
                           (1 << 20, 1 << 15, 8, 1), (1 << 22, 8, 1 << 18, 1)):  # more than a launch's 2^32 threads
        with pytest.raises(ValueError):
            h.linear_act8_sizes(rows, K, N, dt, True)
    with pytest.raises(ValueError):  # bf16 rows off 16 bytes need the copy
        h.linear_act8_fwd(2, 8, 16, 8, 0, 0, 0, 16, 0, 4, 8, 8, 1, False, False, 0, 256, 0)
    with pytest.raises(ValueError):
        h.linear_act8_bwd(2, 8, 16, 8, 16, 0, 0, False, 0, 8, 0, 0, 0, False, 4, 8, 8, 1, False, 0, 256, 0)
