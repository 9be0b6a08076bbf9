"""Cases of the memory-lean training operators: the loss of a vocabulary head that keeps no logits
(``ops/linear_xent.py``) and the Linear layer that keeps its input in 8 bits (``ops/act8.py``).

``run`` takes one training pass through an operator, forward and backward.  With ``own`` false it is
the plain form, elementary torch operations in 32 bits; with ``own`` true the framework's entry point.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32          # features that share one power-of-two scale of the 8-bit checkpoint
E4M3_MAX = 448.0


def _xent(name, dtype, rows, width, vocab, classes, bias, ignore, kept):
    """``kept``: share of the rows that carry a label; the others have the ``ignore`` label."""
    return {"name": name, "op": "linear_cross_entropy", "dtype": dtype, "rows": rows, "width": width, "vocab": vocab,
            "classes": classes, "bias": bias, "ignore": ignore, "kept": kept}


def _act8(name, dtype, rows, width, out, bias, act):
    return {"name": name, "op": "linear_act8", "dtype": dtype, "rows": rows, "width": width, "out": out,
            "bias": bias, "act": act}


def listed():
    return [
        # one sentence of the translation model through its head: launches are what counts
        _xent("xent sentence", "bfloat16", 20, 256, 15000, 15000, True, 0, 0.85),
        # a batch of 512 sentences of 20 tokens, padding (id 0) ignored
        _xent("xent translation batch", "bfloat16", 10240, 256, 15000, 15000, True, 0, 0.85),
        # BERT-base's masked positions, 64 x 20, over the padded vocabulary
        _xent("xent masked positions", "bfloat16", 1280, 768, 30528, 30522, True, -100, 1.0),
        # the same step at reference precision
        _xent("xent masked positions f32", "float32", 1280, 768, 30528, 30522, True, -100, 1.0),
        # every position handed over, 15 % of them labelled
        _xent("xent all positions", "bfloat16", 8192, 768, 30528, 30522, True, -100, 0.15),
        # odd everything: a ragged batch, a width that is no multiple of a vector, a prime vocabulary
        _xent("xent ragged f32", "float32", 777, 203, 4999, 4999, False, -100, 0.9),
        # a wide model's head over a large vocabulary, every position labelled
        _xent("xent large", "bfloat16", 8192, 2048, 65536, 65536, False, -100, 1.0),
        # a few tokens through an FFN's second projection
        _act8("act8 sentence", "bfloat16", 20, 2048, 256, True, "gelu"),
        # BERT-base's fused q/k/v projection, 64 sequences of 128
        _act8("act8 qkv", "bfloat16", 8192, 768, 2304, True, None),
        # the same at reference precision
        _act8("act8 qkv f32", "float32", 8192, 768, 2304, True, None),
        # odd sizes through the GELU form
        _act8("act8 ragged gelu f32", "float32", 1001, 1348, 331, False, "gelu"),
        # a wide FFN's second projection, its input the GELU's pre-activation
        _act8("act8 wide gelu", "bfloat16", 16384, 8192, 2048, True, "gelu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly whole 16-byte vectors, as layer widths are; one in six is any number."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 1 / 6 else max(8, w // 8 * 8)


def draw(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if rng.random() < 0.5:
        width, vocab = _width(rng, 64, 2048), _log(rng, 500, 65536)
        most = 8192 * 2048 * 65536 // (6 if dtype == "float32" else 1)
        rows = min(_log(rng, 1, 10240), max(1, most // (width * vocab)))
        classes = vocab - rng.choice([0, 0, rng.randint(1, 63)])
        c = _xent("", dtype, rows, width, vocab, classes, rng.random() < 0.5, rng.choice([-100, 0]),
                  rng.choice([1.0, 0.85, 0.5, 0.15]))
    else:
        width, out = _width(rng, 32, 8192), _width(rng, 32, 4096)
        most = 16384 * 8192 * 2048 // (6 if dtype == "float32" else 1)
        rows = min(_log(rng, 1, 16384), max(1, most // (width * out)))
        c = _act8("", dtype, rows, width, out, rng.random() < 0.7, rng.choice([None, "gelu"]))
    del c["name"]
    return c


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    R, K = case["rows"], case["width"]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def leaf(t):
        return t.to(dt).requires_grad_()

    st = {"case": case}
    if case["op"] == "linear_cross_entropy":
        V, C = case["vocab"], case["classes"]
        w = normal(V, K) * (1.5 / math.sqrt(K))
        first = 1 if case["ignore"] == 0 else 0
        labels = torch.randint(first, C, (R,), device=dev, generator=g)
        # a model that has learnt some: a row leans towards its label's weights by a share of its own,
        # up to about half the probability
        lean = torch.rand(R, 1, device=dev, generator=g) * ((math.log(C) + 1) / 2.25)
        x = normal(R, K) + lean * w[labels]
        gone = torch.rand(R, device=dev, generator=g) >= case["kept"]
        gone[0] = False
        st["labels"] = torch.where(gone, torch.full_like(labels, case["ignore"]), labels)
        st["x"], st["w"] = leaf(x), leaf(w)
        st["b"] = leaf(normal(V) * 0.1) if case["bias"] else None
    else:
        # activations: features of different sizes, a few of them large
        size = torch.exp(0.5 * normal(1, K)) * torch.where(torch.rand(1, K, device=dev, generator=g) < 0.01, 20.0, 1.0)
        st["x"] = leaf(normal(R, K) * (size if case["act"] is None else size.clamp(max=4.0)))
        st["w"] = leaf(normal(case["out"], K) * 0.02)
        st["b"] = leaf(normal(case["out"]) * 0.1) if case["bias"] else None
        st["dy"] = (normal(R, case["out"]) * 1e-3).to(dt)
    return st


def run(state):
    case = state["case"]
    x, w, b = state["x"], state["w"], state["b"]
    leaves = [t for t in (x, w, b) if t is not None]
    if case["op"] == "linear_cross_entropy":
        if own:
            from vodascheduler_amd.ops.linear_xent import linear_cross_entropy

            loss, correct, n = linear_cross_entropy(x, w, state["labels"], bias=b, num_classes=case["classes"],
                                                    ignore_index=case["ignore"])
            return (loss.detach(), correct, n, *torch.autograd.grad(loss, leaves))
        return _plain_xent(x.detach(), w.detach(), None if b is None else b.detach(), state["labels"],
                           case["classes"], case["ignore"])
    if own:
        from vodascheduler_amd.ops.act8 import linear_act8

        y = linear_act8(x, w, b, act=case["act"])
        return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))
    return _plain_act8(x.detach(), w.detach(), None if b is None else b.detach(), state["dy"], case["act"])


def _plain_xent(x, w, b, labels, classes, ignore):
    """z = x w^T + b over the first ``classes`` rows of w; loss = mean over the labelled rows of
    logsumexp(z) - z[label]; G = (softmax(z) - onehot) / n; dx = G w, dw = G^T x, db = sum G."""
    xf, wf = x.float(), w[:classes].float()
    z = xf @ wf.t()
    if b is not None:
        z += b[:classes].float()
    kept = labels != ignore
    at = torch.where(kept, labels, 0)[:, None]
    n = kept.sum()
    top = z.amax(1, keepdim=True)
    # the lowest index of the largest value
    best = torch.where(z == top, torch.arange(classes, device=z.device), classes).amin(1)
    correct = ((best == labels) & kept).sum()
    picked = z.gather(1, at)[:, 0]
    p = z.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    loss = torch.where(kept, (top[:, 0] - picked) + total[:, 0].log(), 0.0).sum() / n
    p /= total
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=p.dtype))
    p *= kept[:, None] / n
    pad = w.shape[0] - classes
    grads = [p @ wf, torch.nn.functional.pad(p.t() @ xf, (0, 0, 0, pad))]
    if b is not None:
        grads.append(torch.nn.functional.pad(p.sum(0), (0, pad)))
    return (loss, correct, n, *(t.to(x.dtype) for t in grads))


def _through_8_bits(x):
    """What the checkpoint of x stands for: blocks of BLOCK features, each e4m3 times the smallest
    power of two that keeps the block's largest value within E4M3_MAX."""
    rows, width = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).view(rows, -1, BLOCK)
    mant, exp = torch.frexp(padded.abs().amax(2, keepdim=True))       # amax = mant 2^exp, mant in [0.5, 1)
    exp = (exp - 9 + (mant > E4M3_MAX / 512)).clamp(min=-126)
    held = torch.ldexp(padded, -exp).to(torch.float8_e4m3fn).float()
    return torch.ldexp(held, exp).view(rows, -1)[:, :width]


_C, _D = math.sqrt(2 / math.pi), 0.044715


def _gelu(h):
    return 0.5 * h * (1 + torch.tanh(_C * (h + _D * h * h * h)))


def _gelu_slope(h):
    t = torch.tanh(_C * (h + _D * h * h * h))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * _C * (1 + 3 * _D * h * h)


def _plain_act8(x, w, b, dy, act):
    """y = act(x) w^T + b from x itself; the gradients from its checkpoint c:
    dx = (dy w) act'(c), dw = dy^T act(c), db = sum dy."""
    xf, wf, gf = x.float(), w.float(), dy.float()
    y = (xf if act is None else _gelu(xf)) @ wf.t()
    if b is not None:
        y += b.float()
    c = _through_8_bits(x)
    dx = gf @ wf
    if act is not None:
        dx *= _gelu_slope(c)
    grads = [dx, gf.t() @ (c if act is None else _gelu(c))]
    if b is not None:
        grads.append(gf.sum(0))
    return (y.to(x.dtype), *(t.to(x.dtype) for t in grads))


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    R, K = case["rows"], case["width"]
    if case["op"] == "linear_cross_entropy":
        V, n = case["vocab"], max(1.0, R * case["kept"])
        b = 2 * V * size if case["bias"] else 0
        # x of the labelled rows, w and b in; dx, dw and db out
        return {"bytes": n * K * size + R * K * size + 2 * V * K * size + b + 8 * R, "flops": 6 * n * case["classes"] * K}
    N = case["out"]
    b = 2 * N * size if case["bias"] else 0
    # x, w, dy in; y, dx, dw out; the checkpoint written and read, a byte a value and one a block
    held = 2 * R * (K + -(-K // BLOCK))
    return {"bytes": 2 * (R * K + N * K + R * N) * size + held + b, "flops": 6 * R * K * N}


def exact(case, seed):
    st = prepare(case, seed)
    x, w = st["x"].detach().double().requires_grad_(), st["w"].detach().double().requires_grad_()
    b = None if st["b"] is None else st["b"].detach().double().requires_grad_()
    leaves = [t for t in (x, w, b) if t is not None]
    if case["op"] == "linear_cross_entropy":
        C = case["classes"]
        keep = (st["labels"] != case["ignore"]).nonzero()[:, 0]
        z = torch.nn.functional.linear(x[keep], w[:C], None if b is None else b[:C])
        loss = torch.nn.functional.cross_entropy(z, st["labels"][keep])
        return (loss.detach(), None, None, *torch.autograd.grad(loss, leaves))
    with torch.no_grad():
        v = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))
        top = v.abs().amax(2, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -117) / E4M3_MAX))
        step = torch.exp2(e)
        # a value of e4m3 has three bits behind its first, and none finer than 2^-9
        unit = torch.exp2(torch.floor(torch.log2((v / step).abs().clamp(min=2.0 ** -6))) - 3)
        c = (torch.round(v / step / unit) * unit * step).flatten(1)[:, :x.shape[1]]
    gelu = torch.nn.functional.gelu
    y = torch.nn.functional.linear(x if case["act"] is None else gelu(x, approximate="tanh"), w, b).detach()
    c.requires_grad_()
    through = torch.nn.functional.linear(c if case["act"] is None else gelu(c, approximate="tanh"), w, b)
    grads = torch.autograd.grad(through, [c, w] + ([] if b is None else [b]), st["dy"].double())
    return (y, *grads)
