"""ops/act8.py in fp32 on elements of any size beside each other: every result within the bounds of fp32
arithmetic on its own terms, whatever else a row, a column or the tensor holds."""
import pytest
import torch

from vodascheduler_amd.ops.act8 import linear_act8

from act8_bounds import U, checkpoint, gelu, slope
from test_act8_gpu import _inputs, _run
from xent_bounds import within

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _terms(x, w, b, dy, act):
    """(y, dx, dw, db) in fp64, and bounds from each one's own terms: a sum of n products in fp32 is off by
    n 2^-24 of the sum of their sizes at most; 4 2^-24 for the planes; the GELU to 8 2^-24
    times 1 + 3 k (|h| + c |h|^3), its argument's error (below 100 2^-24 at |h| <= 3.2)."""
    X, W, G, B = (t.detach().double() for t in (x, w, dy, b))
    c = checkpoint(x)
    a, ac, sl = (X, c, torch.ones_like(c)) if act is None else (gelu(X), gelu(c), slope(c))
    own = 4 * U if act is None else 104 * U
    (M, K), N = X.shape, W.shape[0]
    y, p, dw, db = a @ W.t() + B, G @ W, G.t() @ ac, G.sum(0)
    by = ((K + 64) * U + own) * (a.abs() @ W.abs().t()) + 4 * U * (y.abs() + B.abs())
    bdx = ((N + 64) * U + own) * (G.abs() @ W.abs()) * (sl.abs() + (0.0 if act is None else 1 + c.abs())) + 16 * U * (p * sl).abs()
    bdw = ((M + 64) * U + own) * (G.abs().t() @ ac.abs()) + 16 * U * dw.abs()
    bdb = (M + 64) * U * G.abs().sum(0) + 4 * U * db.abs()
    tiny = 1e-36
    return (y, p * sl, dw, db), (by + tiny, bdx + tiny, bdw + tiny, bdb + tiny)


def _hold(x, w, b, dy, act, rows=slice(None)):
    got = _run(x, w, b, dy, act)
    want, bound = _terms(x, w, b, dy, act)
    for o, r, d, nm in zip(got, want, bound, ("y", "dx", "dw", "db")):
        keep = rows if nm in ("y", "dx") else slice(None)
        within(o[keep], r[keep], d[keep], nm)


SIZES = [(20, 64, 50), (300, 203, 130), (700, 264, 257)]


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("big", [1e10, 1e16, 1e30])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_a_row_of_another_size(rows, K, N, big, act):
    """Padding that holds anything finite: a row of x whose gradient is zero, a row of dy whose input is
    zero; the others, and what all of them add up to, are as ever."""
    x, w, b, dy = _inputs(rows, K, N, torch.float32, bias=True, seed=rows)
    with torch.no_grad():
        x.clamp_(-3, 3)
        x[3] *= big
        x[5] = 0.0
    dy[3] = 0.0
    dy[5] *= big
    others = torch.tensor([r for r in range(rows) if r not in (3, 5)], device=DEV)
    _hold(x, w, b, dy, act, others)


@pytest.mark.parametrize("big", [1e16, 1e30])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_a_feature_and_an_output_of_another_size(rows, K, N, big):
    """A feature that no weight reads, an output that no gradient reaches, one element among ordinary ones."""
    x, w, b, dy = _inputs(rows, K, N, torch.float32, bias=True, seed=rows)
    with torch.no_grad():
        x[:, 7] *= big
        w[:, 7] = 0.0
        w[11] *= big
        w[11, 40] = 0.0
        x[2, 40] = big
    dy[:, 11] = 0.0
    dy[2] = 0.0
    _hold(x, w, b, dy, None)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("rows,K,N", SIZES)
def test_small_features(rows, K, N, act):
    """Blocks of 32 features at 2^-20 to 2^-90 of the others': the checkpoint holds each block by itself, and so
    must dw's columns."""
    x, w, b, dy = _inputs(rows, K, N, torch.float32, bias=True, seed=rows)
    with torch.no_grad():
        x.clamp_(-3, 3)
        for k in range(K // 32):
            x[:, 32 * k:32 * k + 32] *= 2.0 ** -[34, 38, 20, 50, 70, 90, 0][k % 7]
    _hold(x, w, b, dy, act)


@pytest.mark.parametrize("rows,K,N", SIZES)
def test_elements_of_all_sizes(rows, K, N):
    g = torch.Generator(device=DEV).manual_seed(rows)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g) * torch.exp2(60 * torch.rand(*s, device=DEV, generator=g) - 30)  # noqa: E731
    x, w, b = (rnd(*s).requires_grad_() for s in ((rows, K), (N, K), (N,)))
    _hold(x, w, b, rnd(rows, N), None)


def test_the_largest_and_smallest_numbers():
    """What rounds past bf16's largest stays finite; planes below 2^-126 are lost, no more."""
    x, w, b, dy = _inputs(40, 64, 24, torch.float32, bias=True)
    top = torch.finfo(torch.float32).max
    with torch.no_grad():
        x.zero_(), w.zero_(), b.zero_()
        x[:, 0] = top
        x[1::2, 0] = -top
        x[:, 1] = 2.0 ** -100
        w[0, 0], w[1, 0], w[2, 1] = 1.0, 0.5, 2.0 ** 100
    y = _run(x, w, b, dy * 2.0 ** -20, None)[0]
    assert torch.isfinite(y).all()
    assert ((y[:, 0] - x[:, 0]).abs() <= 2 * U * top).all() and ((y[:, 1] - x[:, 0] / 2).abs() <= U * top).all()
    assert ((y[:, 2] - 1).abs() <= 4 * U).all()


@pytest.mark.parametrize("need", [n for n in ((i & 1, i & 2, i & 4) for i in range(1, 8))])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_each_gradient_whatever_else_is_asked_for(dtype, act, need):
    """dx and dw keep their bits.  db is summed with dw, or by itself in another order: each sum of 50 terms
    within 50 2^-24 of their sizes, and a rounding to the type."""
    ins = _inputs(50, 64, 72, dtype, bias=True)
    dy = ins[3]
    full = dict(zip("xwb", _run(*ins, act)[1:]))
    leaves = {nm: t.detach().requires_grad_(bool(k)) for nm, t, k in zip("xwb", ins, need)}
    y = linear_act8(*leaves.values(), act)
    asked = {nm: t for nm, t in leaves.items() if t.requires_grad}
    got = dict(zip(asked, torch.autograd.grad(y, list(asked.values()), dy)))
    assert set(got) == {nm for nm, k in zip("xwb", need) if k}
    for nm, g in got.items():
        r = full[nm]
        if nm != "b" or "w" in got:
            assert torch.equal(g, r), nm
        else:
            off = 2 * 50 * U * dy.double().abs().sum(0) + torch.finfo(dtype).eps * r.double().abs()
            assert ((g.double() - r.double()).abs() <= off).all()
