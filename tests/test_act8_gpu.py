"""ops/act8.py on MI355X: the checkpoint bit by bit against the CPU's, the layer against the formulas in
fp64 within bounds that follow from the roundings (tests/act8_bounds.py)."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import Act8Linear, act8_pack, act8_unpack, linear_act8

from act8_bounds import checkpoint, formulas
from test_act8_cpu import special_values
from xent_bounds import within

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _inputs(rows, K, N, dtype, bias, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    x = n(rows, K) * torch.exp(0.5 * n(1, K))
    leaf = lambda t: t.to(dtype).requires_grad_()  # noqa: E731
    return leaf(x), leaf(n(N, K) * 0.1), leaf(n(N)) if bias else None, n(rows, N).to(dtype)


def _run(x, w, b, dy, act):
    leaves = [t for t in (x, w, b) if t is not None]
    y = linear_act8(x, w, b, act)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def _check(x, w, b, dy, act):
    got = _run(x, w, b, dy, act)
    want, bound = formulas(x.reshape(-1, x.shape[-1]), w, b, dy.reshape(-1, w.shape[0]), act)
    for o, r, d, nm in zip(got, want, bound, ("y", "dx", "dw", "db")):
        within(o.reshape(r.shape), r, d, nm)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (2, 7, 33), (130, 264), (1000, 40)])
def test_checkpoint_is_the_cpu_s(shape, dtype):
    x = (torch.randn(*shape) * torch.exp(4 * torch.randn(*shape[:-1], 1))).to(dtype)
    q, s = act8_pack(x)
    for t in (x.to(DEV), torch.cat([x, x], -1).to(DEV)[..., :shape[-1]], x.to(DEV).transpose(0, -1).contiguous().transpose(0, -1)):
        gq, gs = act8_pack(t)
        assert torch.equal(gq.cpu().view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(gs.cpu().view(torch.uint8), s.view(torch.uint8))
        for dt in (torch.float32, torch.bfloat16):
            assert torch.equal(act8_unpack(gq, gs, shape[-1], dt).cpu(), act8_unpack(q, s, shape[-1], dt))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpoint_of_edges(dtype):
    x = special_values(dtype)
    got = act8_unpack(*act8_pack(x.to(DEV)), x.shape[1])
    torch.testing.assert_close(got.cpu().double(), checkpoint(x), rtol=0, atol=0, equal_nan=True)


# rows, features and outputs at, below and past the tiles' edges (32, 128, 256), blocks (32), vectors (8)
# and stages (32, 64)
SIZES = [(1, 1, 1), (1, 264, 130), (3, 32, 8), (31, 100, 5), (32, 64, 128), (33, 31, 129), (128, 33, 40), (130, 520, 24),
         (257, 72, 300), (1000, 264, 96), (700, 1100, 257)]


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_matches_the_formulas(rows, K, N, dtype, act):
    _check(*_inputs(rows, K, N, dtype, bias=rows != 130, seed=rows), act)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [(8192, 1600, 1664), (4100, 384, 6000)])
def test_large_tiles(rows, K, N, dtype, act):
    """Enough tiles for the 256 x 256 and 256 x 128 ones, each of the three products."""
    _check(*_inputs(rows, K, N, dtype, bias=True, seed=rows), act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_shapes(dtype):
    x, w, b, dy = _inputs(24, 40, 27, dtype, bias=True)
    want = _check(x, w, b, dy, "gelu")

    def wide(t, pad):
        buf = torch.full((t.shape[0], t.shape[1] + pad), 7.0, device=DEV, dtype=dtype)
        buf[:, 1:1 + t.shape[1]] = t.detach()
        return buf[:, 1:1 + t.shape[1]]

    strided = torch.zeros(2 * 27, device=DEV, dtype=dtype)[::2]
    strided.copy_(b.detach())
    turned = lambda t: t.detach().t().contiguous().t()  # noqa: E731
    for x2, w2, b2, dy2 in ((x.detach().view(4, 6, 40), w.detach(), b.detach(), dy.view(4, 6, 27)),
                            (wide(x, 7), wide(w, 3), strided, wide(dy, 2)), (turned(x), turned(w), b.detach(), turned(dy))):
        for o, r in zip(_run(x2.requires_grad_(), w2.requires_grad_(), b2.requires_grad_(), dy2, "gelu"), want):
            assert torch.equal(o.reshape(r.shape), r)
    # a gradient that is one number for all
    y = linear_act8(x, w, b)
    g1 = torch.autograd.grad(y.float().sum(), (x, w, b), retain_graph=True)
    g2 = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert all(torch.equal(p, q) for p, q in zip(g1, g2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expanded_operands(dtype):
    """Rows that are all one row: of the gradient (a sum over the rows behind the layer), the input and the
    weight."""
    x, w, b, _ = _inputs(40, 64, 48, dtype, bias=True)
    x1, w1 = (t.detach()[:1].expand(*t.shape) for t in (x, w))
    dy = torch.randn(1, 48, device=DEV).to(dtype).expand(40, 48)
    assert dy.stride(0) == 0
    for xe, we in ((x, w), (x1.requires_grad_(), w1.requires_grad_())):
        y = linear_act8(xe, we, b)
        got = torch.autograd.grad(y, (xe, we, b), dy)
        ref = _run(xe.detach().contiguous().requires_grad_(), we.detach().contiguous().requires_grad_(), b,
                   dy.contiguous(), None)
        assert all(torch.equal(g, r) for g, r in zip((y, *got), ref))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_single_rows_of_any_stride(dtype, act):
    """A matrix of one row is contiguous whatever its row stride says."""
    x, w, b, dy = _inputs(1, 64, 1, dtype, bias=True)
    want = _check(x, w, b, dy, act)
    turned = lambda t: t.detach().reshape(-1, 1).clone().t()  # noqa: E731
    x1, w1 = turned(x), turned(w)
    assert x1.stride() == (1, 1) and w1.is_contiguous()
    for o, r in zip(_run(x1.requires_grad_(), w1.requires_grad_(), b, dy, act), want):
        assert torch.equal(o, r)
    x, w, b, dy = _inputs(1, 40, 48, dtype, bias=True)
    want = _check(x, w, b, dy, act)
    for o, r in zip(_run(x, w, b, turned(dy), act), want):
        assert torch.equal(o, r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [72, 27])
def test_a_frozen_weight(N, dtype):
    """dx and db by themselves; db of the same sums in another order: each within (rows + 1) 2^-24 of the
    sum of magnitudes, and a rounding to the type."""
    x, w, b, dy = _inputs(300, 64, N, dtype, bias=True)
    full = _check(x, w, b, dy, None)
    y = linear_act8(x, w.detach(), b)
    gx, gb = torch.autograd.grad(y, (x, b), dy)
    assert torch.equal(gx, full[1])
    err = (gb.double() - full[3].double()).abs()
    assert (err <= 2 * 301 * 2.0 ** -24 * dy.double().abs().sum(0) + torch.finfo(dtype).eps * full[3].double().abs()).all()


@pytest.mark.parametrize("rows", [20, 900])
def test_bias_of_another_type(rows):
    x, w, b, dy = _inputs(rows, 72, 48, torch.bfloat16, bias=True)
    b = b.detach().float().requires_grad_()
    got = _check(x, w, b, dy, "gelu")
    assert got[3].dtype == torch.float32


def test_offsets_past_32_bits():
    x, w, b, dy = _inputs(700, 64, 700, torch.bfloat16, bias=True)
    want = _check(x, w, b, dy, None)
    ld = (1 << 32) // 600 // 8 * 8

    def far(t):
        v = torch.empty(700 * ld, dtype=torch.bfloat16, device=DEV).view(700, ld)[:, :t.shape[1]]
        v.copy_(t.detach())
        return v

    for o, r in zip(_run(far(x).requires_grad_(), far(w).requires_grad_(), b, far(dy)[:, :700], None), want):
        assert torch.equal(o, r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_non_finite(dtype):
    """NaN and infinities of x reach y; in the checkpoint both are NaN, so they reach dw (and dx through
    the GELU), and only the rows and columns they belong to."""
    x, w, b, dy = _inputs(40, 96, 50, dtype, bias=True)
    with torch.no_grad():
        x[7, 5], x[9, 70] = float("nan"), float("inf")
    y, dx, dw, db = _run(x, w, b, dy, "gelu")
    ok = torch.ones(40, dtype=torch.bool, device=DEV)
    ok[[7, 9]] = False
    assert torch.isfinite(y[ok]).all() and not torch.isfinite(y[~ok]).any()
    bad = torch.zeros(40, 96, dtype=torch.bool, device=DEV)
    bad[7, 5] = bad[9, 70] = True
    assert torch.equal(~torch.isfinite(dx), bad)
    assert not torch.isfinite(dw[:, [5, 70]]).any()
    assert torch.isfinite(dw[:, [k for k in range(96) if k not in (5, 70)]]).all() and torch.isfinite(db).all()


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_asked_for(need):
    x, w, b, dy = _inputs(50, 64, 72, torch.bfloat16, bias=True)
    full = _check(x, w, b, dy, "gelu")
    leaves = [t.detach().requires_grad_(k) for t, k in zip((x, w, b), need)]
    y = linear_act8(*leaves, "gelu")
    got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
    for g, r, nm in zip(got, [r for r, k in zip(full[1:], need) if k], "xwb"):
        assert torch.equal(g, r) or (nm == "b" or need[2]) and torch.allclose(g.float(), r.float(), rtol=2.0 ** -7)
    with torch.no_grad():
        assert torch.equal(linear_act8(x, w, b, "gelu"), full[0])


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [30, 900])
def test_into_the_flat_gradient(rows, grad_dtype):
    from vodascheduler_amd.utils.flat import FlatGroup, grad_of

    x, w, b, dy = _inputs(rows, 72, 48, torch.bfloat16, bias=True)
    want, bound = formulas(x, w, b, dy, "gelu")
    layer = Act8Linear(72, 48, act="gelu", device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        layer.weight.copy_(w), layer.bias.copy_(b)
    group = FlatGroup([layer.weight, layer.bias], grad_dtype=grad_dtype)  # noqa: F841  (owns the gradients)
    seen = []
    for t in (layer.weight, layer.bias):
        t._voda_grad_ready = lambda q: seen.append(q)
        grad_of(t).fill_(0.5)
    layer(x).backward(dy)
    assert [id(q) for q in seen] == [id(layer.weight), id(layer.bias)]
    half = 2.0 ** -8 if grad_dtype == torch.bfloat16 else 2.0 ** -24
    for t, r, d in ((layer.weight, want[2], bound[2]), (layer.bias, want[3], bound[3])):
        within(grad_of(t), r + 0.5, d + half * (r + 0.5).abs() + 2.0 ** -24, "flat gradient")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_residual_sink(dtype):
    """dx is added to the gradient that the residual branch left (one rounding), and returned."""
    from vodascheduler_amd.ops.conv1x1 import GradSink

    x, w, b, dy = _inputs(300, 64, 96, dtype, bias=True)
    want, bound = formulas(x, w, b, dy, None)
    res = torch.randn(300, 64, device=DEV).to(dtype)
    sink = GradSink()
    y = linear_act8(x, w, b, None, sink_in=sink)
    sink.put(res.clone())
    (gx,) = torch.autograd.grad(y, x, dy)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    total = want[1] + res.double()
    within(gx, total, bound[1] + half * (total.abs() + want[1].abs()) + 2.0 ** -24 * res.double().abs(), "dx")


def test_same_bits_every_time_and_on_another_stream():
    for rows, dtype in ((20, torch.bfloat16), (1300, torch.bfloat16), (300, torch.float32)):
        x, w, b, dy = _inputs(rows, 256, 300, dtype, bias=True)
        first = _check(x, w, b, dy, "gelu")
        side = torch.cuda.Stream()
        for k in range(4):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
                got = _run(x, w, b, dy, "gelu")
            torch.cuda.synchronize()
            assert all(torch.equal(g, r) for g, r in zip(got, first))


def test_two_streams_at_once():
    ins = [_inputs(900, 200, 136, torch.float32, bias=True, seed=s) for s in (1, 2)]
    want = [_check(*t, "gelu") for t in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for s, t, o in zip(streams, ins, got):
            with torch.cuda.stream(s):
                o.append(_run(*t, "gelu"))
    torch.cuda.synchronize()
    for o, r in zip(got, want):
        assert all(torch.equal(p, q) for run in o for p, q in zip(run, r))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(dtype):
    x, w, b, dy = _inputs(200, 96, 80, dtype, bias=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(x, w, b, dy, "gelu")
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(x, w, b, dy, "gelu")
        graphs.append((g, out))
    for k in range(4):
        nx, nw, nb, ndy = _inputs(200, 96, 80, dtype, bias=True, seed=10 + k)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), b.copy_(nb), dy.copy_(ndy)
        want = [t.clone() for t in _run(x, w, b, dy, "gelu")]
        g, out = graphs[k % 2]
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip(out, want):
            assert torch.equal(o, r)


def test_refusals_on_the_gpu():
    x, w, b, dy = _inputs(8, 16, 30, torch.bfloat16, bias=True)
    for args in ((x.half(), w.half(), None), (x, w.float(), None), (x, w, b.half())):
        with pytest.raises(TypeError):
            linear_act8(*args)
    with pytest.raises(ValueError):
        linear_act8(x, w.cpu())
    with pytest.raises(RuntimeError):  # first derivatives only
        (g,) = torch.autograd.grad(linear_act8(x, w).float().sum(), x, create_graph=True)
        g.sum().backward()
    assert linear_act8(x[:0], w, b, "gelu").shape == (0, 30)
