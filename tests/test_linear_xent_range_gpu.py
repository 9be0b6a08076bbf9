"""ops/linear_xent.py over the whole range of logits: classes masked by any finite value, rows whose logits
are large. Beside the formulas' bounds (tests/xent_bounds.py), cases whose logits are exact products, so
that the softmax is known to the last few bits."""
import math

import pytest
import torch

from vodascheduler_amd.ops.linear_xent import linear_cross_entropy

from test_linear_xent_gpu import _check, _inputs
from xent_bounds import U, formulas, within

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
TYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [-1e4, -1.3e6, -1e9, -1e10, -1e20, -1e30])
def test_classes_masked_by_a_finite_bias(mask, dtype, rows):
    """Whole slots of classes at any low value take no part, and leave the others as they are."""
    x, w, b, y = _inputs(rows, 48, 700, 700, dtype, bias=True)
    y = torch.where(y >= 0, y % 10 + 600, y)
    with torch.no_grad():
        b[:400] = mask
    loss, grads = _check(x, w, b, y, 700)
    assert torch.isfinite(loss) and float(grads[1][:400].float().abs().max()) == 0.0


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [-1e4, 1.3e6, -1.1e9, 1e10, -1e20, 1e30])
def test_every_class_at_one_value(value, dtype, rows):
    """w = 0: every logit is the bias, whatever its size, so the softmax is uniform."""
    C, K = 300, 48
    x, _, _, y = _inputs(rows, K, C, C, dtype, bias=False, ignored=0.0)
    w = torch.zeros(C, K, dtype=dtype, device=DEV, requires_grad=True)
    b = torch.full((C,), value, dtype=dtype, device=DEV, requires_grad=True)
    loss, correct, n = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    assert int(correct) == int((y == 0).sum()) and int(n) == rows
    # log C of a sum of C ones, to the few units of the logarithm and the result
    assert abs(float(loss) - math.log(C)) <= 8 * U * math.log(C)
    G = (torch.full((rows, C), 1 / C, dtype=torch.float64, device=DEV) - torch.nn.functional.one_hot(y, C)) / rows
    # G is 1 / C (the reciprocal's two units) less one, held as an operand; then sums of rows and a rounding
    hold = 2.0 ** -8 if dtype == torch.bfloat16 else 4 * U
    half = torch.finfo(dtype).eps / 2
    assert float(gx.float().abs().max()) == 0.0
    for g, r in ((gw, x.double()), (gb, torch.ones(rows, 1, dtype=torch.float64, device=DEV))):
        want, size = G.t() @ r, G.abs().t() @ r.abs()
        assert ((g.double().reshape(want.shape) - want).abs() <= (hold + (rows + 8) * U) * size + half * want.abs()).all()


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [30.25, 1000.0, 1.3e6, 1.1e9, 1e10, 1e20, 1e29])
def test_rows_of_large_logits(top, dtype, rows):
    """Logits top, 0 and -top, each one product of one term and so exact: a row with its label alone at the
    top has loss 0 and no gradient, one that shares the top with another class log 2 and a half each."""
    C, K = 300, 16
    x = torch.zeros(rows, K, device=DEV)
    at = torch.tensor(top).to(dtype).item()
    x[:, 0], x[:, 1] = at, at
    w = torch.zeros(C, K, device=DEV)
    w[7, 0], w[100:, 0] = 1, -1
    x, w = x.to(dtype).requires_grad_(), w.to(dtype).requires_grad_()
    y = torch.full((rows,), 7, device=DEV)
    tail = 99 * math.exp(-at) + 200 * math.exp(-2 * at)  # of the classes below; 1e-12 at 30
    loss, correct, _ = linear_cross_entropy(x, w, y)
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert 0.0 <= float(loss) <= 2 * tail + 1e-30 and int(correct) == rows
    # dw: the softmax (below tail) times at, over the rows' mean
    assert float(gw.double().abs().max()) <= 4 * tail * at + 1e-30 and float(gx.double().abs().max()) <= 4 * tail + 1e-30
    with torch.no_grad():
        w[200, 0] = 1
    loss, correct, _ = linear_cross_entropy(x, w, y)
    gx, gw = torch.autograd.grad(loss, (x, w))
    assert abs(float(loss) - math.log(2)) <= 4 * U + tail and int(correct) == rows
    want = torch.zeros(C, K, dtype=torch.float64, device=DEV)
    want[7, :2], want[200, :2] = -at / 2, at / 2
    # the halves are exact; the mean's factor, the sums over rows and the result's rounding are not
    off = torch.finfo(dtype).eps / 2 + (rows + 8) * U
    assert ((gw.double() - want).abs() <= off * want.abs() + 4 * tail * at + 1e-30).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_confident_row_s_loss_is_not_negative(dtype):
    """The sum of exponentials holds the largest one's, exactly 1."""
    for seed in range(24):
        x, w, _, _ = _inputs(1, 64, 300, 300, dtype, bias=False, seed=seed, ignored=0.0)
        with torch.no_grad():
            x *= 2.0 ** (seed // 2)
        y = (x.float() @ w.float().t()).argmax(1)
        assert float(linear_cross_entropy(x, w, y)[0]) >= 0.0


def _subset(x, w, b, y, C, keep):
    """The formulas' (dx, dw, db) of some rows alone, in the mean over all of them, and their bounds less the
    one term in them that is no fp32 error (2^-49 of each element of x, for each row)."""
    rows, n = x.shape[0], keep.numel()
    (_, _, _, dx, dw, db), (_, bdx, bdw, bdb) = formulas(x[keep], w, b, y[keep], C, -100, n / rows)
    bdw[:C] -= 2.0 ** -49 / rows * x[keep].detach().double().abs().sum(0)
    bdx -= 2.0 ** -49 / rows * w[:C].detach().double().abs().sum(0)
    return (dx, dw, db), (bdx + 1e-35, bdw + 1e-35, bdb)


@pytest.mark.parametrize("big", [1e10, 1e16, 2.0 ** 60, 1e30])
@pytest.mark.parametrize("rows,K,C", [(20, 64, 300), (200, 203, 500), (600, 264, 1000)])
def test_one_labelled_row_of_another_size(rows, K, C, big):
    """fp32: its logits are far apart, so its softmax is one class; the other rows' gradients, and the weight's of
    all other classes, are as ever."""
    x, w, b, y = _inputs(rows, K, C, C, torch.float32, bias=True, seed=rows, ignored=0.0)
    with torch.no_grad():
        x[3] *= big
    loss, _, n = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    keep = torch.tensor([r for r in range(rows) if r != 3], device=DEV)
    (dx, dw, db), (bdx, bdw, bdb) = _subset(x, w, b, y, C, keep)
    within(gx[keep], dx, bdx, "dx")
    z = x[3].detach().double() @ w.detach().double().t()
    apart = (z.amax() - z) > 200  # certain: its softmax there is 0, in fp32 too
    apart[y[3]] = False
    assert int(apart.sum()) >= C - 3
    within(gw[apart], dw[apart], bdw[apart], "dw")
    within(gb[apart], db[apart], bdb[apart], "db")


@pytest.mark.parametrize("big", [1e16, 1e30])
def test_one_class_and_one_feature_of_another_size(big):
    """fp32: weights of a class that its bias masks, a feature that no class reads."""
    rows, K, C = 300, 72, 400
    x, w, b, y = _inputs(rows, K, C, C, torch.float32, bias=True, ignored=0.1)
    y = torch.where(y == 9, 10, y)
    with torch.no_grad():
        w[9] *= big
        b[9] = float("-inf")
        w[:, 5] = 0.0
        x[:, 5] *= big
        w[9, 5] = 0.0
    loss, _, n = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    with torch.no_grad():
        w[9] = 0.0  # takes no part: any weights give the same
    keep = (y >= 0).nonzero()[:, 0]
    (dx, dw, db), (bdx, bdw, bdb) = _subset(x, w, b, y, C, keep)
    scale = rows / keep.numel()
    assert torch.isfinite(loss)
    within(gx[keep], dx * scale, bdx * scale, "dx")
    within(gw, dw * scale, bdw * scale, "dw")
    within(gb, db * scale, bdb * scale, "db")


@pytest.mark.parametrize("rows", [20, 300])
def test_gradients_of_unlikely_classes(rows):
    """fp32: classes that a bias makes unlikely (2^-40 to 2^-90 of the softmax) get gradients right to
    their own size."""
    K, C = 64, 400
    x, w, b, y = _inputs(rows, K, C, C, torch.float32, bias=True, ignored=0.0)
    y = y % 100
    with torch.no_grad():
        b[100:] -= torch.arange(300, device=DEV) * 0.1 + 28
    loss, _, _ = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    # bounds as the formulas', summed from the relative terms alone: the difference that _subset takes, of
    # numbers near 2^-49 in fp64, is good to 2^-102 only, and these classes' terms lie below 2^-24 2^-90
    X, W, B = (t.detach().double() for t in (x, w, b))
    z = X @ W.t() + B
    gap = z.amax(1, keepdim=True) - z
    p = torch.softmax(z, 1)
    G = p - torch.nn.functional.one_hot(y, C)
    ez = (K + 4) * U * (X.abs() @ W.abs().t()) + 4 * U * (z.abs() + B.abs())
    far = ez + ez.amax(1, keepdim=True)
    dG = p * (far + 4 * U * gap + (C + 16) * U + (p * far).sum(1, keepdim=True)) + 3 * U * G.abs() + U * p
    bound = (dG.t() @ X.abs() + (rows + 68) * U * (G.abs().t() @ X.abs())) / rows
    want = G.t() @ X / rows
    assert float(p[:, 100:].amax()) < 2.0 ** -30 and float(p[:, 399].amax()) < 2.0 ** -75
    within(gw, want, bound + 9 * U * want.abs(), "dw")


@pytest.mark.parametrize("rows", [1, 3, 40, 200, 1100])
@pytest.mark.parametrize("dtype", TYPES)
def test_the_first_of_nothing_but_masks(dtype, rows):
    """Every class at -inf: no loss, and the first maximum is class 0, as argmax has it."""
    x, w, b, y = _inputs(rows, 48, 700, 690, dtype, bias=True, ignored=0.1)
    y = torch.where(y < 0, y, torch.where(torch.arange(rows, device=DEV) % 3 == 0, 0, y))
    with torch.no_grad():
        b[:] = float("-inf")
    loss, correct, n = linear_cross_entropy(x, w, y, b, 690)
    assert torch.isnan(loss) or int(n) == 0
    assert int(correct) == int((y == 0).sum())
    with torch.no_grad():  # one class left, behind several slots of masks
        b[600] = 0.0
    y = torch.where(y == 0, 600, torch.where(y == 600, 5, y))
    assert int(linear_cross_entropy(x, w, y, b, 690)[1]) == int((y == 600).sum())


@pytest.mark.parametrize("dtype,flat", [(d, f) for d in TYPES for f in (None, torch.float32, torch.bfloat16)
                                        if (d, f) != (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows", [20, 300, 700])
def test_pieces_of_the_vocabulary(dtype, rows, flat, monkeypatch):
    """Three pieces, the last of 188 columns, classes < vocabulary: dx gathers over them, dw and db go
    piece by piece to their rows, returned or onto what a flat gradient holds."""
    from vodascheduler_amd.ops import linear_xent
    from vodascheduler_amd.utils.flat import FlatGroup, grad_of

    monkeypatch.setattr(linear_xent, "G_BYTES", 0)
    K, V, C = 72, 730, 700
    x, w, b, y = _inputs(rows, K, V, C, dtype, bias=True, seed=rows)
    if flat is None:
        _check(x, w, b, y, C)
        return
    want, bound = formulas(x, w, b, y, C, -100)
    w, b = torch.nn.Parameter(w.detach()), torch.nn.Parameter(b.detach())
    group = FlatGroup([w, b], grad_dtype=flat)  # noqa: F841  (owns the gradients)
    for t in (w, b):
        grad_of(t).fill_(0.5)
    loss = linear_cross_entropy(x, w, y, b, C)[0]
    monkeypatch.setattr(linear_xent, "G_BYTES", 1 << 20)  # the backward keeps to the forward's limit
    loss.backward()
    within(x.grad, want[3], bound[1], "dx")
    half = torch.finfo(flat).eps / 2
    for t, r, d in ((w, want[4], bound[2]), (b, want[5], bound[3])):
        within(grad_of(t), r + 0.5, d + half * (r + 0.5).abs() + 2.0 ** -24, "flat gradient")
        assert torch.equal(grad_of(t)[C:], torch.full_like(grad_of(t)[C:], 0.5))


def test_the_number_of_pieces(monkeypatch):
    """One piece, two or three: the forward, which has none, keeps its bits, and the gradients their bounds."""
    from vodascheduler_amd.ops import linear_xent

    for dtype, rows in ((torch.bfloat16, 300), (torch.float32, 300), (torch.bfloat16, 40)):
        x, w, b, y = _inputs(rows, 72, 730, 700, dtype, bias=True)
        losses = []
        for limit in (512 << 20, 512 * rows * 2 * 3, 0):
            monkeypatch.setattr(linear_xent, "G_BYTES", limit)
            losses.append(_check(x, w, b, y, 700)[0])
        assert torch.equal(losses[0], losses[1]) and torch.equal(losses[0], losses[2])
