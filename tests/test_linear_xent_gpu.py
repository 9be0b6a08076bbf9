"""ops/linear_xent.py on MI355X against the formulas in fp64, within bounds that follow from the
roundings (tests/xent_bounds.py)."""
import pytest
import torch

from vodascheduler_amd.ops.linear_xent import linear_cross_entropy

from xent_bounds import formulas, within

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _inputs(rows, K, V, C, dtype, bias, seed=0, ignored=0.2, ignore=-100):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn(V, K, device=DEV, generator=g) * (1.5 / K ** 0.5)
    y = torch.randint(0, C, (rows,), device=DEV, generator=g)
    x = torch.randn(rows, K, device=DEV, generator=g) + 2 * torch.rand(rows, 1, device=DEV, generator=g) * w[y]
    b = torch.randn(V, device=DEV, generator=g) * 0.1 if bias else None
    y = torch.where(torch.rand(rows, device=DEV, generator=g) < ignored, torch.full_like(y, ignore), y)
    leaf = lambda t: None if t is None else t.to(dtype).requires_grad_()  # noqa: E731
    return leaf(x), leaf(w), leaf(b), y


def _check(x, w, b, y, C, ignore=-100, gloss=1.0):
    leaves = [t for t in (x, w, b) if t is not None]
    loss, correct, n = linear_cross_entropy(x, w, y, b, C, ignore)
    grads = torch.autograd.grad(loss * gloss, leaves)
    want, bound = formulas(x.reshape(-1, x.shape[-1]), w, b, y.reshape(-1), C, ignore, gloss)
    assert loss.dtype == torch.float32 and correct.dtype == n.dtype == torch.int64
    assert int(correct) == want[1] and int(n) == want[2]
    within(loss.detach(), want[0], bound[0], "loss")
    for g, r, d, nm, t in zip(grads, want[3:], bound[1:], ("dx", "dw", "db"), leaves):
        assert g.shape == t.shape and g.dtype == t.dtype
        within(g.reshape(r.shape), r, d, nm)
    return loss, grads


# one row to several tiles' worth on each side of every tile's edge (32, 128, 256), the two-plane
# border (128) and the row count from which another tile serves dx (1024); widths below, at and past
# a stage (32, 64) and off 16-byte rows; vocabularies of one class to several slots
SIZES = [(1, 8, 1, 1), (1, 64, 300, 300), (2, 9, 257, 257), (17, 100, 255, 250), (32, 64, 256, 256), (33, 65, 640, 513),
         (64, 264, 1000, 1000), (127, 31, 130, 130), (129, 40, 2, 2), (130, 72, 7, 7), (256, 128, 1030, 1025),
         (300, 203, 4999, 4999), (1024, 96, 384, 384), (1029, 520, 1500, 1490)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,V,C", SIZES)
def test_matches_the_formulas(rows, K, V, C, dtype):
    x, w, b, y = _inputs(rows, K, V, C, dtype, bias=True, seed=rows)
    _check(x, w, b, y, C, gloss=0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,V", [(2050, 1600, 5000), (4096, 64, 33000), (700, 2100, 33000)])
def test_large_tiles(rows, K, V, dtype):
    """Enough tiles and a reduction long enough for the 256 x 256 tile; the last without a bias."""
    x, w, b, y = _inputs(rows, K, V, V, dtype, bias=rows != 700, seed=rows)
    _check(x, w, b, y, V)


def test_several_pieces_of_the_vocabulary(monkeypatch):
    """More rows than one piece of the workspace holds: dx gathers over the pieces."""
    from vodascheduler_amd.ops import _native

    rows, K, V = 70000, 8, 8000
    nb = _native.hip().linear_xent_sizes(rows, K, V, V, False)[1]
    assert nb < rows * V * 2  # G does not fit one piece
    x, w, b, y = _inputs(rows, K, V, V, torch.bfloat16, bias=True, ignored=0.9)
    _check(x, w, b, y, V)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kept", ["none", "first", "last", "outside", "one in 50"])
def test_labels(kept, dtype):
    x, w, b, y = _inputs(600, 40, 300, 290, dtype, bias=True, ignored=0.0, ignore=7)
    y = torch.where(y == 7, 8, y)
    if kept == "none":
        y[:] = 7
    elif kept == "first":
        y[1:] = 7
    elif kept == "last":
        y[:-1] = 7
    elif kept == "outside":  # classes of the padding, negative labels, labels past the weight
        y[::3], y[1::3] = 295, -5
        y[2] = 1 << 40
    else:
        y[torch.arange(600, device=DEV) % 50 != 3] = 7
    _check(x, w, b, y, 290, ignore=7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ignored_rows_may_hold_anything(dtype):
    x, w, b, y = _inputs(300, 64, 500, 500, dtype, bias=True, ignored=0.3)
    clean = _check(x, w, b, y, 500)
    gone = (y == -100).nonzero()[:, 0]
    with torch.no_grad():
        x[gone[::3]] = float("nan")
        x[gone[1::3]] = float("inf")
        x[gone[2::3]] = 3e38
    loss, correct, n = linear_cross_entropy(x, w, y, b)
    grads = torch.autograd.grad(loss, (x, w, b))
    assert torch.equal(loss, clean[0])
    for g, r in zip(grads, clean[1]):
        assert torch.equal(g, r)
    assert float(grads[0][gone].abs().max()) == 0.0


@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_classes(dtype, rows):
    """A bias of -inf, or of the type's lowest value, takes a class out; whole slots of them too."""
    x, w, b, y = _inputs(rows, 48, 700, 700, dtype, bias=True)
    y = torch.where(y >= 0, y % 10 + 600, y)
    with torch.no_grad():
        b[:300] = float("-inf")
        b[300:400] = torch.finfo(dtype).min
    loss, grads = _check(x, w, b, y, 700)
    assert torch.isfinite(loss) and float(grads[1][:400].float().abs().max()) == 0.0


@pytest.mark.parametrize("rows", [2, 200])
def test_a_label_that_is_masked_and_a_row_of_nothing_but_masks(rows):
    x, w, b, y = _inputs(rows, 48, 90, 90, torch.bfloat16, bias=True, ignored=0.0)
    with torch.no_grad():
        b[5] = float("-inf")
    y[0] = 5
    loss, _, _ = linear_cross_entropy(x, w, y, b)
    assert loss.item() == float("inf")  # -log 0
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    assert all(torch.isfinite(g).all() for g in (gx, gw, gb))
    with torch.no_grad():
        b[:] = float("-inf")
    assert torch.isnan(linear_cross_entropy(x, w, y, b)[0])


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_class_at_the_lowest_value(dtype, rows):
    """No logit differs from the mask: a uniform softmax, so G is 1/C less the label's one."""
    C, K = 300, 48
    x, w, b, y = _inputs(rows, K, C, C, dtype, bias=True, ignored=0.0)
    with torch.no_grad():
        b[:] = torch.finfo(dtype).min
    loss, correct, n = linear_cross_entropy(x, w, y, b)
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b))
    assert int(correct) == int((y == 0).sum()) and int(n) == rows
    # log C of a sum of C ones, and the exponents' few units
    assert abs(float(loss) - torch.tensor(float(C)).double().log().item()) < (C + 16) * 2.0 ** -24
    G = (torch.full((rows, C), 1 / C, dtype=torch.float64, device=DEV) - torch.nn.functional.one_hot(y, C)) / rows
    hold = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20  # of G as an operand, and of the result
    for g, l, r in ((gx, G, w), (gw, G.t(), x), (gb, G.t(), torch.ones(rows, 1, dtype=dtype, device=DEV))):
        want, size = l @ r.double(), l.abs() @ r.double().abs()
        assert ((g.double().reshape(want.shape) - want).abs() <= 2 * hold * size + (C + rows) * 2.0 ** -23 * size).all()


def test_rows_past_fp32_s_ordinary_range_beside_others():
    """Logits near 2^110 in some rows: one class takes all of their softmax; the rows between are as ever."""
    x, w, b, y = _inputs(90, 48, 300, 300, torch.bfloat16, bias=True, ignored=0.0)
    big = torch.arange(90, device=DEV) % 4 == 1
    with torch.no_grad():
        x[big] *= 2.0 ** 110
    loss, grads = _check(x, w, b, y, 300)
    assert all(torch.isfinite(t).all() for t in (loss, *grads))
    top = (x[big].double() @ w.double().t()).argmax(1)
    W = w.detach().double()
    want, size = (W[top] - W[y[big]]) / 90, (W[top].abs() + W[y[big]].abs()) / 90
    assert ((grads[0][big].double() - want).abs() <= 2.0 ** -7 * size).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["x", "w"])
def test_non_finite_inputs_reach_the_loss(what, dtype):
    for bad in (float("nan"), float("inf")):
        x, w, b, y = _inputs(40, 64, 300, 300, dtype, bias=False, ignored=0.0)
        with torch.no_grad():
            (x if what == "x" else w)[11, 3] = bad
        assert not torch.isfinite(linear_cross_entropy(x, w, y)[0])


def test_ties_go_to_the_lowest_class():
    for rows, dtype in ((6, torch.bfloat16), (200, torch.float32)):
        x = torch.zeros(rows, 64, device=DEV, dtype=dtype)
        w = torch.ones(400, 64, device=DEV, dtype=dtype)
        y = torch.arange(rows, device=DEV) % 3
        assert int(linear_cross_entropy(x, w, y)[1]) == int((y == 0).sum())
        b = torch.zeros(400, device=DEV, dtype=dtype)
        b[[2, 130, 399]] = 1
        for label, right in ((2, True), (130, False), (399, False), (1, False)):
            y = torch.full((rows,), label, device=DEV)
            assert int(linear_cross_entropy(x, w, y, b)[1]) == (rows if right else 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_shapes(dtype):
    x, w, b, y = _inputs(24, 40, 130, 130, dtype, bias=True)
    want = _check(x, w, b, y, 130)
    base = dict(x=x.detach(), w=w.detach(), b=b.detach())

    def run(x, w, b, y):
        loss, c, n = linear_cross_entropy(x, w, y, b, 130)
        return loss

    def wide(t, pad):  # rows of a wider buffer, starting off 16 bytes
        buf = torch.full((t.shape[0], t.shape[1] + pad), 7.0, device=DEV, dtype=dtype)
        buf[:, 1:1 + t.shape[1]] = t
        return buf[:, 1:1 + t.shape[1]]

    strided = torch.zeros(2 * 130, device=DEV, dtype=dtype)[::2]
    strided.copy_(base["b"])
    for x2, w2, b2, y2 in ((base["x"].view(4, 6, 40), base["w"], base["b"], y.view(4, 6)),
                           (wide(base["x"], 5), wide(base["w"], 9), strided, y.to(torch.int32)),
                           (base["x"].t().contiguous().t(), base["w"].t().contiguous().t(), base["b"], torch.stack([y, y], 1)[:, 0])):
        leaves = [t.requires_grad_() if t.is_leaf else t.detach().requires_grad_() for t in (x2, w2, b2)]
        loss = run(*leaves, y2)
        assert torch.equal(loss, want[0])
        for g, r in zip(torch.autograd.grad(loss, leaves), want[1]):
            assert torch.equal(g.reshape(r.shape), r)


def test_offsets_past_32_bits():
    """Weight and input rows so far apart that their byte offsets, and element offsets, pass 2^32."""
    rows, K, V = 700, 64, 700
    x, w, b, y = _inputs(rows, K, V, V, torch.bfloat16, bias=False)
    want = _check(x, w, b, y, V)
    ld = (1 << 32) // 600 // 8 * 8
    far = torch.empty(rows * ld, dtype=torch.bfloat16, device=DEV).view(rows, ld)[:, :K]
    far.copy_(x.detach())
    far_w = torch.empty(V * ld, dtype=torch.bfloat16, device=DEV).view(V, ld)[:, :K]
    far_w.copy_(w.detach())
    far.requires_grad_(), far_w.requires_grad_()
    loss = linear_cross_entropy(far, far_w, y)[0]
    assert torch.equal(loss, want[0])
    for g, r in zip(torch.autograd.grad(loss, (far, far_w)), want[1]):
        assert torch.equal(g, r)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [12288, 12289, 150000])
def test_many_rows(rows, dtype):
    """Past the row count from which the labelled rows are counted beforehand."""
    x, w, b, y = _inputs(rows, 16, 50, 50, dtype, bias=True, ignored=0.5)
    y[:2500] = -100
    _check(x, w, b, y, 50)


@pytest.mark.parametrize("rows", [20, 900])
def test_bias_of_another_type(rows):
    x, w, b, y = _inputs(rows, 64, 300, 290, torch.bfloat16, bias=True)
    _, grads = _check(x, w, b.detach().float().requires_grad_(), y, 290)
    assert grads[2].dtype == torch.float32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expanded_operands(dtype):
    x, w, b, y = _inputs(40, 64, 300, 300, dtype, bias=False)
    x1, w1 = (t.detach()[:1].expand(*t.shape) for t in (x, w))
    want = _check(x1.contiguous().requires_grad_(), w1.contiguous().requires_grad_(), None, y, 300)
    x1.requires_grad_(), w1.requires_grad_()
    loss = linear_cross_entropy(x1, w1, y)[0]
    assert torch.equal(loss, want[0])
    assert all(torch.equal(g, r) for g, r in zip(torch.autograd.grad(loss, (x1, w1)), want[1]))


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_gradients_asked_for(need):
    x, w, b, y = _inputs(50, 64, 300, 290, torch.bfloat16, bias=True)
    full = _check(x, w, b, y, 290)[1]
    leaves = [t.detach().requires_grad_(k) for t, k in zip((x, w, b), need)]
    loss = linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], 290)[0]
    got = torch.autograd.grad(loss, [t for t in leaves if t.requires_grad])
    for g, r in zip(got, [r for r, k in zip(full, need) if k]):
        assert torch.equal(g, r)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, y, b, 290)[0], loss)


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [30, 700])
def test_into_the_flat_gradient(rows, grad_dtype):
    """Summed onto what the optimizer's flat gradient holds, once a call, the engine signalled; rows of
    the vocabulary's padding are left as they are."""
    from vodascheduler_amd.utils.flat import FlatGroup, grad_of

    V, C = 300, 290
    x, w, b, y = _inputs(rows, 64, V, C, torch.bfloat16, bias=True)
    want, bound = formulas(x, w, b, y, C, -100)
    w, b = torch.nn.Parameter(w.detach()), torch.nn.Parameter(b.detach())
    group = FlatGroup([w, b], grad_dtype=grad_dtype)  # noqa: F841  (owns the gradients)
    seen = []
    for t in (w, b):
        t._voda_grad_ready = lambda q: seen.append(q)
        grad_of(t).fill_(0.5)
    loss = linear_cross_entropy(x, w, y, b, C)[0]
    loss.backward()
    assert [id(q) for q in seen] == [id(w), id(b)]
    half = 2.0 ** -8 if grad_dtype == torch.bfloat16 else 2.0 ** -24
    for t, r, d in ((w, want[4], bound[2]), (b, want[5], bound[3])):
        within(grad_of(t), r + 0.5, d + half * (r + 0.5).abs() + 2.0 ** -24, "flat gradient")
    assert torch.equal(grad_of(w)[C:], torch.full_like(grad_of(w)[C:], 0.5))


def test_same_bits_every_time_and_on_another_stream():
    for rows, dtype in ((20, torch.bfloat16), (1300, torch.bfloat16), (300, torch.float32)):
        x, w, b, y = _inputs(rows, 256, 3000, 3000, dtype, bias=True)
        first = _check(x, w, b, y, 3000)
        side = torch.cuda.Stream()
        for k in range(4):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream()):
                loss = linear_cross_entropy(x, w, y, b)[0]
                grads = torch.autograd.grad(loss, (x, w, b))
            torch.cuda.synchronize()
            assert torch.equal(loss, first[0])
            assert all(torch.equal(g, r) for g, r in zip(grads, first[1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_single_rows_of_any_stride(dtype):
    """A matrix of one row is contiguous whatever its row stride says."""
    turned = lambda t: t.detach().reshape(-1, 1).clone().t().requires_grad_()  # noqa: E731
    for V in (130, 1):
        x, w, b, y = _inputs(1, 64, V, V, dtype, bias=True, ignored=0.0)
        want = _check(x, w, b, y, V)
        leaves = [turned(x), turned(w) if V == 1 else w, b]
        assert leaves[0].stride() == (1, 1)
        loss = linear_cross_entropy(leaves[0], leaves[1], y, b, V)[0]
        assert torch.equal(loss, want[0])
        assert all(torch.equal(g, r) for g, r in zip(torch.autograd.grad(loss, leaves), want[1]))


def test_two_streams_at_once():
    ins = [_inputs(700, 200, 1300, 1290, torch.float32, bias=True, seed=s) for s in (1, 2)]
    want = [_check(*t, 1290) for t in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for s, (x, w, b, y), o in zip(streams, ins, got):
            with torch.cuda.stream(s):
                loss = linear_cross_entropy(x, w, y, b, 1290)[0]
                o.append((loss.detach(), *torch.autograd.grad(loss, (x, w, b))))
    torch.cuda.synchronize()
    for o, r in zip(got, want):
        assert all(torch.equal(p, q) for run in o for p, q in zip(run, (r[0], *r[1])))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(dtype):
    """Two graphs of one program replayed in turn with eager work between, the number of labelled rows
    another each time."""
    rows, K, V = 200, 64, 1000
    x, w, b, y = _inputs(rows, K, V, V, dtype, bias=True)
    leaves = (x, w, b)

    def step():
        loss, correct, n = linear_cross_entropy(x, w, y, b)
        return (loss.detach(), correct, n, *torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(4):
        nx, nw, nb, ny = _inputs(rows, K, V, V, dtype, bias=True, seed=10 + k, ignored=0.3 * k)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), b.copy_(nb), y.copy_(ny)
        want = [t.clone() for t in step()]
        g, out = graphs[k % 2]
        g.replay()
        torch.cuda.synchronize()
        for o, r in zip(out, want):
            assert torch.equal(o, r)


def test_autocast_takes_the_weight_s_type():
    x, w, b, y = _inputs(40, 64, 300, 300, torch.bfloat16, bias=True)
    want = linear_cross_entropy(x, w, y, b)[0]
    xf = x.detach().float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = linear_cross_entropy(xf, w, y, b)[0]
    assert torch.equal(loss, want)
    (g,) = torch.autograd.grad(loss, xf)
    assert g.dtype == torch.float32


def test_refusals_on_the_gpu():
    x, w, b, y = _inputs(8, 16, 30, 30, torch.bfloat16, bias=True)
    for args in ((x.half(), w.half(), y, None), (x, w.float(), y, None), (x, w, y, b.half()), (x.double(), w.double(), y, None)):
        with pytest.raises(TypeError):
            linear_cross_entropy(*args)
    with pytest.raises(ValueError):
        linear_cross_entropy(x, w, y.cpu(), None)
    with pytest.raises(RuntimeError):  # first derivatives only
        loss = linear_cross_entropy(x, w, y)[0]
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        g.sum().backward()
    loss = linear_cross_entropy(x[:0], w, y[:0], b)[0]
    assert loss.item() == 0.0
    assert float(torch.autograd.grad(loss, w)[0].abs().max()) == 0.0
