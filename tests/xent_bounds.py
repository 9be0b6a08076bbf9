"""How far ops/linear_xent.py's results may be from the formulas' in 64 bits, element by element.

The bounds follow the roundings of the computation, each taken at its worst: u = 2^-24 is half a step
of fp32, a sum of n terms in fp32 is off by at most n u of the sum of the terms' sizes.
"""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U, torch.float64: 2.0 ** -53}


def formulas(x, w, b, y, C, ignore, gloss=1.0):
    """(loss, correct, n, dx, dw, db) in fp64, and the bounds of loss, dx, dw and db."""
    dt, two = x.dtype, x.dtype == torch.float32 or x.shape[0] <= 128
    X, W = x.detach().double(), w.detach().double()
    B = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    keep = ((y != ignore) & (y >= 0) & (y < C)).nonzero()[:, 0]
    n, K, V = keep.numel(), x.shape[1], w.shape[0]
    yk = y[keep]
    Xk, Wc = X[keep], W[:C]
    z = Xk @ Wc.t() + B[:C]
    top = z.amax(1, keepdim=True) if n else z[:, :1]
    e = (z - top).exp()
    s = e.sum(1, keepdim=True)
    p = e / s
    G = p.clone()
    G[torch.arange(n, device=x.device), yk] -= 1
    scale = gloss / max(1, n)
    lr = (top - z.gather(1, yk[:, None]) + s.log())[:, 0]
    loss = lr.sum() / max(1, n)
    correct = int((z.argmax(1) == yk).sum())
    dx = torch.zeros_like(X)
    dx[keep] = scale * (G @ Wc)
    dw, db = torch.zeros_like(W), torch.zeros(V, dtype=torch.float64, device=x.device)
    dw[:C], db[:C] = scale * (G.t() @ Xk), scale * G.sum(0)
    # logits: products of 16-bit values are exact; fp32 inputs hold each factor to u in two planes and
    # leave lo.lo out (u again)
    planes = 4 * U if dt == torch.float32 else 0.0
    ez = (K * U + planes) * (Xk.abs() @ Wc.abs().t()) + 4 * U * (z.abs() + B[:C].abs())
    there = p > 0  # masked classes take no part
    ez = torch.where(there, ez, 0.0)
    gap = torch.where(there, (z - top).abs(), 0.0)
    far = ez + ez.amax(1, keepdim=True) if n else ez
    # p: both exponents' errors, the argument's scaling by log2(e), exp2 and 1 / sum to a few u
    dp = p * (far + 4 * U * gap + (C + 16) * U + (p * far).sum(1, keepdim=True))
    hold = {True: 2.0 ** -16, False: 2.0 ** -8}[two] if dt == torch.bfloat16 else 2 * U
    dG = dp + hold * G.abs() + U * (G.abs() + p) + 2.0 ** -49
    aG, aX, aW = G.abs(), Xk.abs(), Wc.abs()
    few = 8 * U  # the factors' products
    bdx = torch.zeros_like(X)
    bdx[keep] = scale * (dG @ aW + ((C + 64) * U + planes) * (aG @ aW)) + (HALF[dt] + few) * dx[keep].abs()
    bdw, bdb = torch.zeros_like(W), torch.zeros_like(db)
    bdw[:C] = scale * (dG.t() @ aX + ((n + 64) * U + planes) * (aG.t() @ aX))
    bdb[:C] = scale * (dG.sum(0) + (n + 64) * U * aG.sum(0))
    bdw += (HALF[w.dtype] + few) * dw.abs()
    bdb += (HALF[torch.float32 if b is None else b.dtype] + few) * db.abs()
    tiny = 1e-37
    # the loss: z's errors in max, label and sum; log(s) and the sums to a few u
    bl = ((2 * far.amax(1) + 8 * U * (1 + gap.amax(1)) + (C + 8) * U).sum() / max(1, n) + 4 * U * loss.abs()) if n else 0.0
    return (loss, correct, n, dx, dw, db), (bl, bdx + tiny, bdw + tiny, bdb + tiny)


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    ok = off <= bound
    assert bool(ok.all()), (f"{what}: {int((~ok).sum())} of {ok.numel()} values out of bounds, worst "
                            f"{float((off / bound).max()):.3g} times theirs")
