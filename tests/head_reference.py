"""The vocabulary head's operators from their definitions in 64 bits, with bounds on how far
a result computed as the library does may be off.

The bounds count every rounding the library makes and nothing else.  With u = eps / 2 of the
16-bit type and E = (D + 8) 2^-23 sum |h||w| the worst error of an fp32 dot product of length
D (each of its additions may truncate, which is a whole unit of 2^-23, plus the bias):
  logit           E
  softmax value   a relative 2 E / tau + 2^-18 (its own logit and the denominator's; ex2, its
                  argument's rounding at |z| < 2^6 and the sum)
  P               u |P| (its rounding; u^2 |P| where up to 128 rows let it be held in two
                  parts, whose products are then sums of twice as many terms) + the softmax
                  value's error
  dH = P W, dW = P^T H   |dP| summed against |W|, |H|, fp32 sums of n terms (n 2^-23), and u
                  of the result
fp16 adds the steps of its subnormal numbers: 2^-25 for a result, and for P (scaled so that
the largest row coefficient is 2^14) 2^-25 gmax / 2^14.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUB = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def _products(P, dP, h, w, dt, scale_floor, parts=1):
    """dH, dW, dbias and their bounds from P and its bound."""
    u, sub = U[dt], SUB[dt]
    T, V = P.shape
    aP = P.abs() + dP
    dPr = dP + u ** parts * aP + scale_floor
    ah, aw = h.abs(), w.abs()
    dh, dw, db = P @ w, P.t() @ h, P.sum(0)
    bh = dPr @ aw + (parts * V + 64) * 2.0 ** -23 * (aP @ aw)
    bw = dPr.t() @ ah + (parts * T + 64) * 2.0 ** -23 * (aP.t() @ ah)
    bb = dP.sum(0) + (T + 64) * 2.0 ** -24 * aP.sum(0)
    return (dh, bh * (1 + u) + u * dh.abs() + sub), (dw, bw * (1 + u) + u * dw.abs() + sub), (db, bb)


def softmax_loss(h, w, b, q, live, tau, grads, dt):
    """Losses [T] and gradients for target distributions q [T, V] (64-bit); live [T]; grads [T]
    the gradient of every row's loss.  Everything returned as (value, bound)."""
    h = torch.where(live[:, None], h.double(), 0.0)
    w = w.double()
    s = h @ w.t() + (b.double() if b is not None else 0.0)
    D = h.shape[1]
    E = (D + 8) * 2.0 ** -23 * (h.abs() @ w.abs().t() + (b.double().abs() if b is not None else 0.0))
    z = s / tau
    # words whose bias (below -1e30) takes them out of the vocabulary have a softmax value of
    # exactly 0 in any precision: no error of theirs enters a bound
    out = s < -1e30
    E = torch.where(out, 0.0, E)
    finite = torch.where(out, 0.0, z.abs())
    e = (E.max(dim=1, keepdim=True).values / tau) * 2 + 2.0 ** -18 + finite * 2.0 ** -22
    lse = torch.logsumexp(z, dim=1)
    logq = z - lse[:, None]
    terms = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - logq), 0.0)
    loss = torch.where(live, tau * tau * terms.sum(1), 0.0)
    ent = torch.where(q > 0, q * torch.log(torch.where(q > 0, q, 1.0)), 0.0).sum(1).abs()
    err = e.max(dim=1).values + 2.0 ** -20 * (1 + ent + lse.abs())
    loss_b = torch.where(live, tau * tau * err, 0.0)
    ga = torch.where(live, grads.double() * tau, 0.0)
    sm = torch.exp(logq)
    P = ga[:, None] * (sm - q)
    P = torch.where(live[:, None], P, 0.0)
    dP = ga.abs()[:, None] * (sm * e + 2.0 ** -22 * (sm + q))
    floor = SUB[dt] * float(ga.abs().max()) / 2.0 ** 14 if len(ga) else 0.0
    parts = 2 if len(h) <= 128 and D <= 74 * 256 else 1
    return (loss, loss_b), _products(P, dP, h, w, dt, floor, parts)


def sparse_head(h, w, b, mask, dy, dt, exact=True):
    """y, winner token and gradients; ``exact``: the inputs' products and sums have no rounding."""
    B, Lt, D = h.shape
    m = mask[:, :, None]
    hd = torch.where(m, h.double(), 0.0)
    wd = w.double()
    bd = b.double() if b is not None else torch.zeros(w.shape[0], dtype=torch.float64, device=w.device)
    s = torch.where(m, hd @ wd.t() + bd, float("-inf"))
    best, arg = s.max(dim=1)
    none = ~mask.any(dim=1)
    best = torch.where(none[:, None], 0.0, best)
    y = torch.log1p(best.clamp(min=0.0))
    E = 0.0 if exact else float(((D + 8) * 2.0 ** -23 * (hd.abs() @ wd.abs().t() + bd.abs())).max())
    yb = E + 2.0 ** -22 * y
    if dy is None:
        return (y, yb)
    ds = torch.where(best > 0, dy.double() * torch.exp(-y), 0.0)
    P = torch.zeros(B, Lt, w.shape[0], dtype=torch.float64, device=w.device)
    P.scatter_(1, arg[:, None, :], ds[:, None, :])
    P = P.reshape(B * Lt, -1)
    floor = SUB[dt] * float(dy.abs().max()) / 2.0 ** 14
    grads = _products(P, P.abs() * 2.0 ** -20, hd.reshape(B * Lt, D), wd, dt, 0.0)
    if floor:        # only P's own entries can lose to fp16's subnormal steps
        at = (P != 0).double() * floor
        (dh, bh), (dw, bw), d = grads
        grads = (dh, bh + at @ wd.abs()), (dw, bw + at.t() @ hd.reshape(B * Lt, D).abs()), d
    return (y, yb), grads


def assert_within(got, ref, what):
    value, bound = ref
    got = got.double().cpu()
    value, bound = value.cpu(), bound.cpu() if isinstance(bound, torch.Tensor) else bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - value).abs() - bound
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0.0, (f"{what}: {worst:.3g} beyond its bound, largest error "
                          f"{float((got - value).abs().max()):.3g} of {float(value.abs().max()):.3g}")
