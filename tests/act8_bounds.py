"""ops/act8.py's results in fp64, and how far the computation's roundings may carry it from them."""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
C, D = (2 / torch.pi) ** 0.5, 0.044715


def gelu(h):
    return 0.5 * h * (1 + torch.tanh(C * (h + D * h ** 3)))


def slope(h):
    t = torch.tanh(C * (h + D * h ** 3))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * C * (1 + 3 * D * h * h)


def checkpoint(x):
    """What x's checkpoint stands for, in fp64: each 32 features' e4m3 values, by rounding to the nearest
    multiple of the step at a value's size, ties to even (torch.round), times the block's power of two."""
    rows, width = x.shape
    v = torch.nn.functional.pad(x.detach().double(), (0, -width % 32)).view(rows, -1, 32)
    fin = torch.isfinite(v)
    top = torch.where(fin, v, 0.0).abs().amax(2, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / 448))
    over, under = top > 448 * torch.exp2(e), top <= 448 * torch.exp2(e - 1)  # log2 rounds
    e = (e + over.double() - under.double()).clamp(min=-126)
    r = torch.where(fin, v, 0.0) / torch.exp2(e)
    step = torch.exp2(torch.frexp(r.abs().clamp(min=2.0 ** -6))[1].double() - 4)
    q = torch.round(r / step) * step
    q = torch.where(e == 120, q.clamp(-240, 240), q)  # 256 2^120 is past fp32
    c = torch.where(fin, q * torch.exp2(e), torch.nan)
    return c.view(rows, -1)[:, :width]


def formulas(x, w, b, dy, act):
    """(y, dx, dw, db) in fp64 with their bounds."""
    dt = x.dtype
    X, W, G = x.detach().double(), w.detach().double(), dy.detach().double()
    M, K = X.shape
    N = W.shape[0]
    c = checkpoint(x)
    f32 = dt == torch.float32
    planes = 4 * U if f32 else 0.0  # two fp16 planes hold a factor to u each, lo.lo (u) is left out
    # gelu and its slope: exp2 and the reciprocal to a unit, the argument's rounding by its size
    arg = lambda h: 1 + 3 * C * (h.abs() + D * h.abs() ** 3)  # noqa: E731
    a = X if act is None else gelu(X)
    ac = c if act is None else gelu(c)
    half = 0.0 if act is None else U * 2 if f32 else 2.0 ** -8  # act's result as an operand
    ea = 0.0 if act is None else half * a.abs() + 8 * U * arg(X) * a.abs()
    eac = 0.0 if act is None else half * ac.abs() + 8 * U * arg(c) * ac.abs()
    y = a @ W.t() + (0.0 if b is None else b.detach().double())
    by = (ea @ W.abs().t() if act else 0.0) + ((K + 64) * U + planes) * (a.abs() @ W.abs().t()) + 4 * U * y.abs()
    by = by + (HALF[dt] * y.abs()) + (0.0 if b is None else 2 * U * b.detach().double().abs())
    sl = torch.ones_like(c) if act is None else slope(c)
    p = G @ W
    dx = p * sl
    bp = ((N + 64) * U + planes) * (G.abs() @ W.abs())
    bdx = bp * sl.abs() + (0.0 if act is None else 8 * U * arg(c) * (1 + c.abs()) * p.abs()) + (HALF[dt] + 8 * U) * dx.abs()
    dw = G.t() @ ac
    bdw = (G.abs().t() @ eac if act else 0.0) + ((M + 64) * U + planes) * (G.abs().t() @ ac.abs()) + (HALF[w.dtype] + 8 * U) * dw.abs()
    # a plane's floor: 2^-50 of a tensor's largest element (an identity c, in one plane: 2^-40)
    if f32:
        floor = 2.0 ** -49
        by = by + floor * (X.abs().max() * W.abs().sum(1) + W.abs().max() * a.abs().sum(1, keepdim=True))
        bdx = bdx + floor * (G.abs().max() * W.abs().sum(0) + W.abs().max() * G.abs().sum(1, keepdim=True)) * (1 + sl.abs())
        bdw = bdw + G.abs().sum(0)[:, None] * X.abs().max() * 2.0 ** -39 + floor * G.abs().max() * ac.abs().sum(0)
    db = G.sum(0)
    bdb = (M + 64) * U * G.abs().sum(0) + (HALF[dt if b is None else b.dtype] + 4 * U) * db.abs()
    if f32:
        bdb = bdb + M * 2.0 ** -49 * G.abs().max() + planes * G.abs().sum(0)
    tiny = 1e-37
    return (y, dx, dw, db), (by + tiny, bdx + tiny, bdw + tiny, bdb + tiny)
