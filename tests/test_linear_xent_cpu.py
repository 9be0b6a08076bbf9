"""ops/linear_xent.py without a GPU: the reference form against the formulas in fp64, its agreement with
ops/xent.py, the refusals, and the host's own checks of the native entry points."""
import pytest
import torch
import torch.nn.functional as F

from vodascheduler_amd.ops.linear_xent import linear_cross_entropy
from vodascheduler_amd.ops.xent import xent_ref

from xent_bounds import formulas


def _inputs(rows, K, V, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g, dtype=dtype).requires_grad_()
    w = torch.randn(V, K, generator=g, dtype=dtype).requires_grad_()
    b = torch.randn(V, generator=g, dtype=dtype).requires_grad_()
    y = torch.randint(0, V, (rows,), generator=g)
    return x, w, b, y


@pytest.mark.parametrize("rows,K,V,C,ignore", [(1, 1, 1, 1, -100), (5, 3, 7, 7, -100), (9, 16, 40, 33, 0), (4, 8, 9, 9, 3)])
def test_reference_is_the_formula(rows, K, V, C, ignore):
    x, w, b, y = _inputs(rows, K, V)
    y[rows // 2] = ignore
    loss, correct, n = linear_cross_entropy(x, w, y, b, C, ignore)
    want, _ = formulas(x, w, b, y, C, ignore, 2.0)
    if n:
        got = torch.autograd.grad(2.0 * loss, (x, w, b))
        torch.testing.assert_close(loss.detach(), want[0])
        for g, r in zip(got, want[3:]):
            torch.testing.assert_close(g, r)
    assert int(correct) == want[1] and int(n) == want[2]


def test_agrees_with_the_loss_of_logits():
    x, w, b, y = _inputs(12, 8, 30, dtype=torch.float32)
    y[3] = -100
    got = linear_cross_entropy(x, w, y, b, 25)
    want = xent_ref(F.linear(x, w, b), torch.where(y < 25, y, -100), 25)
    for g, r in zip(got, want):
        torch.testing.assert_close(g.double(), r.double())


def test_gradient_is_the_loss_s_slope():
    """Central differences of a fp64 loss: off by h^2 / 6 of the third derivative, here below 1e-8."""
    x, w, b, y = _inputs(6, 4, 11, seed=3)
    loss = linear_cross_entropy(x, w, y, b)[0]
    for t, g in zip((x, w, b), torch.autograd.grad(loss, (x, w, b))):
        d = torch.randn(t.shape, generator=torch.Generator().manual_seed(1), dtype=t.dtype)
        h = 1e-4
        with torch.no_grad():
            t += h * d
            up = linear_cross_entropy(x, w, y, b)[0].item()
            t -= 2 * h * d
            down = linear_cross_entropy(x, w, y, b)[0].item()
            t += h * d
        assert abs((up - down) / (2 * h) - float((g * d).sum())) < 1e-6


def test_nothing_labelled_and_no_rows():
    x, w, b, y = _inputs(4, 3, 5)
    loss, correct, n = linear_cross_entropy(x, w, torch.full_like(y, -100), b)
    assert loss.item() == 0.0 and correct.item() == 0 and n.item() == 0
    assert all(float(g.abs().max()) == 0.0 for g in torch.autograd.grad(loss, (x, w, b)))
    loss, correct, n = linear_cross_entropy(x[:0], w, y[:0], b)
    assert loss.item() == 0.0 and n.item() == 0


def test_ignored_rows_may_hold_anything():
    x, w, b, y = _inputs(6, 4, 9)
    y[2], y[4] = -100, 77
    with torch.no_grad():
        x[2], x[4] = float("nan"), float("inf")
    loss, _, n = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    assert n.item() == 4 and torch.isfinite(gw).all() and torch.isfinite(gb).all()
    assert float(gx[[2, 4]].abs().max()) == 0.0


@pytest.mark.parametrize("change,error", [
    (dict(x=torch.zeros(4, 6)), ValueError),                       # widths differ
    (dict(labels=torch.zeros(3, dtype=torch.int64)), ValueError),  # a label too few
    (dict(labels=torch.zeros(4)), TypeError),                      # labels are no integers
    (dict(labels=torch.zeros(4, dtype=torch.bool)), TypeError),
    (dict(bias=torch.zeros(6)), ValueError),
    (dict(num_classes=0), ValueError),
    (dict(num_classes=8), ValueError),
    (dict(weight=torch.zeros(7)), ValueError),
    (dict(weight=torch.zeros(7, 5, device="meta")), ValueError),   # another device
])
def test_refusals(change, error):
    args = dict(x=torch.zeros(4, 5), weight=torch.zeros(7, 5), labels=torch.zeros(4, dtype=torch.int64))
    linear_cross_entropy(**args)
    with pytest.raises(error):
        linear_cross_entropy(**{**args, **change})


def test_the_host_refuses_sizes_out_of_range():
    from vodascheduler_amd.ops import _native

    h = _native.hip()
    assert all(v > 0 for v in h.linear_xent_sizes(20, 256, 15000, 15000, False)[:2])
    for rows, K, C, V in ((0, 8, 8, 8), (1 << 25, 8, 8, 8), (4, 0, 8, 8), (4, 8, 0, 8), (4, 8, 9, 8), (4, 8, 8, 1 << 25),
                          (1 << 24, 8, 1 << 16, 1 << 16), (1 << 22, 1 << 13, 8, 8)):  # more than a launch's 2^32 threads
        with pytest.raises(ValueError):
            h.linear_xent_sizes(rows, K, C, V, False)
    # bf16 weight rows that are no whole 16-byte vectors never reach a kernel
    with pytest.raises(ValueError):
        h.linear_xent_fwd(0, 8, 8, 8, 0, 0, 0, -100, 4, 8, 8, 8, 1, *([0] * 11), 0)


def test_rows_of_whole_vectors():
    """Any bf16 matrix becomes one whose rows the products can read, its values unchanged and zeros behind."""
    from vodascheduler_amd.ops.linear_xent import _rows16

    full = torch.arange(1.0, 5 * 41).bfloat16().reshape(4, 51)
    line = torch.arange(1.0, 65).bfloat16()[:, None]
    for t in (full, full[:, :48], full[:, 1:49], full.t(), full[:1].expand(4, 51), full[:1, :48].expand(4, 48),
              line.t(), line[:61].t(), line, line[:1]):
        r = _rows16(t)
        assert r.stride(1) == 1 and r.shape[1] % 8 == 0 and r.stride(0) % 8 == 0 and r.stride(0) >= r.shape[1]
        assert r.data_ptr() % 16 == 0 and torch.equal(r[:, :t.shape[1]], t) and not r[:, t.shape[1]:].any()


def test_the_workspace_is_bounded():
    """512 MB of G whatever the vocabulary, next to what grows with x and w alone."""
    from vodascheduler_amd.ops import _native

    h = _native.hip()
    mb = [h.linear_xent_sizes(8192, 2048, v, v, False)[1] / 2 ** 20 for v in (1 << 16, 1 << 18, 1 << 20)]
    assert mb[-1] < 1.2 * mb[0] and mb[-1] < 512 + 4 * 64 + 128


def test_the_workspace_s_limit():
    """G goes in pieces of at least 256 columns, of at most ``g_bytes`` otherwise."""
    from vodascheduler_amd.ops import _native

    h = _native.hip()
    for f32, planes in ((False, 1), (True, 3)):
        size = [h.linear_xent_sizes(1000, 64, 20000, 20000, f32, limit)[1] for limit in (0, 4 << 20, 512 << 20)]
        assert size[0] < size[1] < size[2] and size[2] == h.linear_xent_sizes(1000, 64, 20000, 20000, f32)[1]
        assert size[0] >= 1000 * 2 * planes * 256 and size[2] >= 1000 * 2 * planes * 20000
    with pytest.raises(ValueError):
        h.linear_xent_sizes(1000, 64, 20000, 20000, False, -1)
