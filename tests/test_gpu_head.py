"""The vocabulary head's operators on the GPU against their definitions in 64 bits."""
import pytest
import torch

import head_reference as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF = torch.bfloat16, torch.float16


def make(T, V, D, dt, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, D, generator=g).to(dt)
    w = (torch.randn(V, D, generator=g) * (2.0 / D ** 0.5)).to(dt)
    b = torch.randn(V, generator=g) * 0.5 if bias else None
    return h.to(DEV), w.to(DEV), b.to(DEV) if bias else None


def leaf(x):
    return x.detach().clone().requires_grad_(True) if x is not None else None


def one_hot(targets, V, live):
    q = torch.zeros(len(targets), V, dtype=torch.float64, device=DEV)
    q[live, targets[live]] = 1.0
    return q


def check_ce(h, w, b, targets, ignore=-100, reduction="mean", grad=None):
    import gpusparse
    T, V = h.shape[0], w.shape[0]
    live = (targets >= 0) & (targets < V) & (targets != ignore)
    n = max(int(live.sum()), 1)
    if reduction == "none":
        rows = grad
    else:
        scale = 1.0 if grad is None else float(grad)
        rows = torch.full((T,), scale / (n if reduction == "mean" else 1), device=DEV)
    ref, (rh, rw, rb) = R.softmax_loss(h, w, b, one_hot(targets, V, live), live, 1.0, rows, h.dtype)
    hl, wl, bl = h.requires_grad_(True), w.requires_grad_(True), leaf(b)
    loss = gpusparse.vocab_cross_entropy(hl, wl, targets, bias=bl, ignore_index=ignore, reduction=reduction)
    assert loss.dtype == torch.float32
    if reduction == "none":
        R.assert_within(loss.detach(), ref, "loss")
    else:
        div = n if reduction == "mean" else 1
        R.assert_within(loss.detach(), (ref[0].sum() / div, ref[1].sum() / div + 2.0 ** -23 * ref[0].sum().abs() / div), "loss")
    leaves = [x for x in (hl, wl, bl) if x is not None]
    go = rows if reduction == "none" else torch.tensor(1.0 if grad is None else float(grad), device=DEV)
    got = torch.autograd.grad(loss, leaves, go.to(torch.float32))
    R.assert_within(got[0], rh, "dh")
    R.assert_within(got[1], rw, "dw")
    if b is not None:
        R.assert_within(got[2], rb, "db")
    assert got[0].dtype == h.dtype and got[1].dtype == w.dtype
    assert (got[0][~live] == 0).all()
    return loss.detach(), got


@pytest.mark.parametrize("T,V,D,dt,frac,bias", [
    (1, 256, 64, BF, 1.0, True),
    (1, 1, 1, BF, 1.0, True),
    (3, 7, 8, HF, 1.0, False),
    (130, 1000, 331, HF, 0.6, True),
    (300, 513, 72, BF, 0.5, False),
    (257, 255, 65, BF, 1.0, True),
    (64, 30522, 768, BF, 1.0, True),
    (5, 30522, 1024, HF, 1.0, False),
    (3000, 300, 128, BF, 0.15, True),
    (20, 90, 19200, BF, 1.0, True),      # more 256-wide tiles of D than pairs of SMs
    (600, 33000, 16, HF, 0.9, True),
])
def test_cross_entropy(T, V, D, dt, frac, bias):
    h, w, b = make(T, V, D, dt, seed=T + V, bias=bias)
    g = torch.Generator().manual_seed(T)
    targets = torch.randint(0, V, (T,), generator=g)
    targets[torch.rand(T, generator=g) >= frac] = -100
    check_ce(h, w, b, targets.to(DEV), grad=1.0 if dt == BF else 1024.0)


@pytest.mark.parametrize("T", [1, 2, 33, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("V,D,dt", [(200, 64, BF), (5000, 96, HF), (90, 331, HF), (3000, 520, BF)])
def test_gradients_of_few_rows(T, V, D, dt):
    """Up to 128 rows the gradients carry the output's rounding alone: losses of few entries a
    row, whose roundings would show."""
    h, w, b = make(T, V, D, dt, seed=T + V)
    targets = torch.arange(T, device=DEV) * 7 % V
    targets[T // 2:][::5] = -100
    if T == 1:
        targets[0] = V - 1
    grad = torch.linspace(-2.0, 3.0, T, device=DEV) + 0.01
    check_ce(h, w, b, targets, reduction="none", grad=grad)
    scores, ids = teacher(T, V, 3, seed=T)
    check_distill(leaf(h), leaf(w), b, scores, ids, 2.0)


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("dt", [BF, HF])
def test_cross_entropy_reductions(reduction, dt):
    h, w, b = make(200, 777, 96, dt, seed=5)
    g = torch.Generator().manual_seed(1)
    targets = torch.randint(0, 777, (200,), generator=g)
    targets[::7] = -100
    grad = torch.randn(200, generator=g).to(DEV) if reduction == "none" else 0.37
    check_ce(h, w, b, targets.to(DEV), reduction=reduction, grad=grad)


def test_cross_entropy_ignored_rows_hold_anything():
    """Ignored tokens and targets outside the vocabulary: NaN and infinities in their hidden
    states reach nothing; the others' results are those without these rows, bit for bit."""
    import gpusparse
    h, w, b = make(140, 500, 80, BF, seed=6)
    targets = torch.arange(140, device=DEV) * 3
    targets[5], targets[9], targets[11], targets[139] = -100, 500, -7, 33
    bad = [5, 9, 11, 139]
    h[5], h[9], h[11], h[139] = float("nan"), float("inf"), float("-inf"), float("nan")
    loss, got = check_ce(h, w, b, targets, ignore=33)
    keep = torch.tensor([r for r in range(140) if r not in bad and int(targets[r]) != 33], device=DEV)
    hl, wl, bl = leaf(h[keep]), leaf(w), leaf(b)
    l2 = gpusparse.vocab_cross_entropy(hl, wl, targets[keep], bias=bl, ignore_index=33)
    g2 = torch.autograd.grad(l2, (hl, wl, bl))
    assert torch.equal(loss, l2) and torch.equal(got[0][keep], g2[0])
    assert torch.equal(got[1], g2[1]) and torch.equal(got[2], g2[2])


def test_cross_entropy_without_any_target():
    import gpusparse
    h, w, b = make(70, 300, 64, BF, seed=7)
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    loss = gpusparse.vocab_cross_entropy(hl, wl, torch.full((70,), -100, device=DEV), bias=bl)
    grads = torch.autograd.grad(loss, (hl, wl, bl))
    assert float(loss.detach()) == 0.0 and all((x == 0).all() for x in grads)
    hl = leaf(h[:0])
    loss = gpusparse.vocab_cross_entropy(hl, wl, torch.zeros(0, dtype=torch.int64, device=DEV))
    grads = torch.autograd.grad(loss, (hl, wl))
    assert float(loss.detach()) == 0.0 and (grads[1] == 0).all() and grads[0].shape == (0, 64)


def test_cross_entropy_masked_vocabulary():
    """A bias of -inf (or the type's lowest value) takes words out of the vocabulary."""
    h, w, b = make(40, 600, 64, BF, seed=8)
    b[100:400] = float("-inf")
    b[400:450] = torch.finfo(torch.float32).min
    targets = torch.arange(40, device=DEV)
    loss, got = check_ce(h, w, b, targets)
    assert (got[1][100:450] == 0).all() and (got[2][100:450] == 0).all()


def test_cross_entropy_layouts():
    """Row strides, unaligned starts, leading dimensions, int32 targets, a 16-bit bias."""
    import gpusparse
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(6, 10, 131, generator=g).to(BF).to(DEV)
    ww = (torch.randn(450, 140, generator=g) * 0.2).to(BF).to(DEV)
    b = torch.randn(450, generator=g).to(BF).to(DEV)
    targets = torch.randint(0, 450, (6, 10), generator=g).to(DEV)
    a = dict(h=wide[..., 3:123], w=ww[:, 5:125])
    dense = gpusparse.vocab_cross_entropy(a["h"].contiguous(), a["w"].contiguous(), targets, bias=b.float())
    assert torch.equal(gpusparse.vocab_cross_entropy(a["h"], a["w"], targets.to(torch.int32), bias=b), dense)
    by_row = gpusparse.vocab_cross_entropy(a["h"], a["w"], targets, bias=b, reduction="none")
    assert by_row.shape == (6, 10)
    t = a["w"].t().contiguous().t()                      # columns contiguous
    assert torch.equal(gpusparse.vocab_cross_entropy(a["h"], t, targets, bias=b), dense)
    # broadcast rows: the gradient of the shared row is the sum over its uses
    one = leaf(wide[0, :1, 3:123])
    loss = gpusparse.vocab_cross_entropy(one.expand(9, 120), a["w"], targets[0, :9])
    (d1,) = torch.autograd.grad(loss, one)
    rep = leaf(one.expand(9, 120))
    (d9,) = torch.autograd.grad(gpusparse.vocab_cross_entropy(rep, a["w"], targets[0, :9]), rep)
    assert d1.shape == one.shape and torch.allclose(d1.float(), d9.float().sum(0, keepdim=True), rtol=2 ** -7, atol=1e-3)


def test_cross_entropy_gradient_matches_differences():
    """The gradient along a direction against a central difference of the 64-bit loss."""
    import gpusparse
    h, w, b = make(60, 400, 64, BF, seed=12)
    targets = torch.arange(60, device=DEV) * 5
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    grads = torch.autograd.grad(gpusparse.vocab_cross_entropy(hl, wl, targets, bias=bl), (hl, wl, bl))
    g = torch.Generator().manual_seed(4)
    for i, (x, d) in enumerate(zip((h, w, b), grads)):
        v = torch.randn(x.shape, generator=g).to(DEV).double()

        def f(step):
            p = [h.double(), w.double(), b.double()]
            p[i] = p[i] + step * v
            return torch.nn.functional.cross_entropy(p[0] @ p[1].t() + p[2], targets)
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        # sum of independent roundings of at most 2^-8 of each term (its own and P's), by the
        # triangle inequality over the terms
        bound = 2.0 ** -7 * (d.double().abs() * v.abs()).sum() + 1e-6
        assert abs(float((d.double() * v).sum() - diff)) <= float(bound)


@pytest.mark.parametrize("dt", [BF, HF])
def test_cross_entropy_in_pieces(dt):
    """More rows x vocabulary than one piece of the backward pass holds: d_hidden is carried
    over the pieces in fp32; the reference is the same formula in fp64 on the GPU, row blocks
    at a time."""
    import gpusparse
    T, V, D = 20000, 15000, 40
    h, w, b = make(T, V, D, dt, seed=9)
    g = torch.Generator().manual_seed(2)
    targets = torch.randint(0, V, (T,), generator=g).to(DEV)
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    loss = gpusparse.vocab_cross_entropy(hl, wl, targets, bias=bl, reduction="sum")
    got = torch.autograd.grad(loss, (hl, wl, bl), torch.tensor(1.0, device=DEV))
    hd, wd, total = h.double(), w.double(), 0.0
    dw = torch.zeros(V, D, dtype=torch.float64, device=DEV)
    db = torch.zeros(V, dtype=torch.float64, device=DEV)
    bw = torch.zeros_like(dw)
    u = R.U[dt]
    for lo in range(0, T, 2500):
        r = slice(lo, lo + 2500)
        s = hd[r] @ wd.t() + b.double()
        P = torch.softmax(s, 1)
        total += float((torch.logsumexp(s, 1) - s.gather(1, targets[r, None]).squeeze(1)).sum())
        P[torch.arange(2500, device=DEV), targets[r]] -= 1.0
        dh = P @ wd
        # P: u + 2^-13 relative (logit errors of 48 * 2^-23 * sum |h||w| < 2^-15, twice), 2^-39
        # absolute in fp16; the sums' own roundings (V + T) 2^-23 are below 2^-8 of u each
        aP = P.abs() * (u + 2.0 ** -13 + V * 2.0 ** -23) + 2.0 ** -39
        bound = (aP @ wd.abs()) * (1 + u) + u * dh.abs() + R.SUB[dt]
        assert ((got[0][r].double() - dh).abs() <= bound).all()
        dw += P.t() @ hd[r]
        bw += aP.t() @ hd[r].abs()
        db += P.sum(0)
    bound = (bw + T * 2.0 ** -23 * bw / u) * (1 + u) + u * dw.abs() + R.SUB[dt]
    assert ((got[1].double() - dw).abs() <= bound).all()
    assert abs(float(loss) - total) <= 2.0 ** -13 * T
    # column sums of 20000 unrounded terms: 2^-13 of the terms' absolute sum (<= 2 per column on
    # average, counted as the target count + the softmax mass)
    mass = torch.bincount(targets, minlength=V).double() * 2 + db.abs()
    assert ((got[2].double() - db).abs() <= (2.0 ** -13 + T * 2.0 ** -24) * (mass + 1)).all()


# ---------------------------------------------------------------------------- distillation
def teacher(T, V, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)])
    scores = torch.sort(torch.randn(T, K, generator=g) * 2 + 6, dim=1, descending=True).values
    return scores.to(DEV), ids.to(DEV)


def check_distill(h, w, b, scores, ids, tau, reduction="mean", grad=1.0):
    import gpusparse
    T, V = h.shape[0], w.shape[0]
    ok = (ids >= 0) & (ids < V) & (scores > float("-inf"))
    live = ok.any(1)
    x = torch.where(ok, scores.double(), float("-inf")) / tau
    p = torch.where(ok, torch.exp(x - torch.where(live, x.max(1).values, 0.0)[:, None]), 0.0)
    p = p / torch.where(live, p.sum(1), 1.0)[:, None]
    q = torch.zeros(T, V, dtype=torch.float64, device=DEV)
    q.scatter_add_(1, torch.where(ok, ids, 0), p)
    n = max(int(live.sum()), 1)
    rows = torch.full((T,), grad / (n if reduction == "mean" else 1), device=DEV)
    ref, (rh, rw, rb) = R.softmax_loss(h, w, b, q, live, tau, rows, h.dtype)
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    loss = gpusparse.topk_distillation(hl, wl, scores, ids, bias=bl, temperature=tau, reduction=reduction)
    div = n if reduction == "mean" else 1
    R.assert_within(loss.detach(), (ref[0].sum() / div, ref[1].sum() / div + 2.0 ** -23 * ref[0].sum().abs() / div), "loss")
    leaves = [t for t in (hl, wl, bl) if t is not None]
    got = torch.autograd.grad(loss, leaves, torch.tensor(grad, device=DEV))
    R.assert_within(got[0], rh, "dh")
    R.assert_within(got[1], rw, "dw")
    if b is not None:
        R.assert_within(got[2], rb, "db")
    return loss.detach(), got


@pytest.mark.parametrize("T,V,D,K,tau,dt,bias", [
    (1, 300, 64, 1, 1.0, BF, True),
    (33, 700, 72, 10, 2.0, BF, True),
    (140, 2000, 100, 100, 0.7, HF, False),
    (70, 5000, 256, 1000, 1.0, BF, True),
    (9, 1024, 64, 1024, 1.5, HF, True),
    (260, 257, 33, 37, 1.0, BF, False),
])
def test_distillation(T, V, D, K, tau, dt, bias):
    h, w, b = make(T, V, D, dt, seed=T, bias=bias)
    scores, ids = teacher(T, V, K, seed=K)
    check_distill(h, w, b, scores, ids, tau, grad=1.0 if dt == BF else 512.0)


@pytest.mark.parametrize("T,V", [(40, 300000), (200, 600000), (40, 1200000)])
def test_distillation_over_wide_vocabularies(T, V):
    """Buckets of 64, 128 and 256 words; the widest in two pieces."""
    h, w, b = make(T, V, 16, BF, seed=T)
    scores, ids = teacher(T, V, 30, seed=T)
    ids[:, :10] = ids[:1, :10] // 5000 * 5000 + torch.arange(10, device=DEV) * 37      # shared blocks
    ids[:, 29] = V - 1 - torch.arange(T, device=DEV) % 3
    check_distill(h, w, b, scores, ids, 1.0)


def test_distillation_padding_duplicates_and_empty_rows():
    h, w, b = make(50, 400, 64, BF, seed=21)
    scores, ids = teacher(50, 400, 16, seed=3)
    scores[3, 10:], ids[3, 10:] = float("-inf"), 0          # compacted_topk's padding
    scores[4, 5:], ids[4, 5:] = float("-inf"), -1           # score_topk's padding
    ids[5] = 77                                             # one word for all
    ids[6, 4], ids[6, 9] = ids[6, 0].clone(), ids[6, 0].clone()
    ids[7, 2], ids[7, 3] = 400, -5                          # outside the vocabulary
    scores[8] = float("-inf")                               # nothing left
    scores[9, 3] = torch.finfo(torch.float32).min           # probability 0
    ids[10] = -1
    h[8], h[10] = float("nan"), float("inf")
    loss, got = check_distill(h, w, b, scores, ids, 1.3)
    assert (got[0][8] == 0).all() and (got[0][10] == 0).all()
    check_distill(h, w, b, scores, ids, 1.3, reduction="sum", grad=0.25)


def test_distillation_from_one_entry_is_cross_entropy():
    import gpusparse
    h, w, b = make(90, 600, 64, BF, seed=22)
    ids = torch.arange(90, device=DEV) * 6
    a, ga = check_ce(h, w, b, ids)
    c, gc = check_distill(h, w, b, torch.zeros(90, 1, device=DEV), ids[:, None], 1.0)
    assert torch.equal(a, c) and all(torch.equal(x, y) for x, y in zip(ga, gc))


# ---------------------------------------------------------------------------- sparse head
def head_inputs(B, Lt, V, D, dt, seed, bias_mean=-1.0):
    """Fixed-point values whose products sum without rounding: maxima and their ties are the
    same in every order of summation."""
    g = torch.Generator().manual_seed(seed)

    def grid(x, step):
        return torch.round(x / step) * step
    h = grid(torch.randn(B, Lt, D, generator=g).clamp(-3.9, 3.9), 2.0 ** -5).to(dt)
    w = grid((torch.randn(V, D, generator=g) / D ** 0.5).clamp(-0.24, 0.24), 2.0 ** -10).to(dt)
    b = grid(torch.randn(V, generator=g) * 0.5 + bias_mean, 2.0 ** -10)
    dy = torch.randn(B, V, generator=g)
    return h.to(DEV), w.to(DEV), b.to(DEV), dy.to(DEV)


def check_head(h, w, b, mask, dy):
    import gpusparse
    ref, (rh, rw, rb) = R.sparse_head(h, w, b, mask != 0 if mask is not None else
                                      torch.ones(h.shape[:2], dtype=torch.bool, device=DEV), dy, h.dtype)
    with torch.no_grad():
        y0 = gpusparse.sparse_head(h, w, bias=b, mask=mask)
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    y = gpusparse.sparse_head(hl, wl, bias=bl, mask=mask)
    assert torch.equal(y, y0)
    R.assert_within(y.detach(), ref, "y")
    leaves = [x for x in (hl, wl, bl) if x is not None]
    got = torch.autograd.grad(y, leaves, dy)
    R.assert_within(got[0].reshape(-1, h.shape[2]), rh, "dh")
    R.assert_within(got[1], rw, "dw")
    if b is not None:
        R.assert_within(got[2], rb, "db")
    return y.detach(), got


@pytest.mark.parametrize("B,Lt,V,D,dt", [
    (1, 1, 5, 8, BF),
    (1, 16, 30522, 256, BF),
    (1, 700, 300, 64, BF),          # one text over many shares
    (3, 700, 300, 72, HF),
    (40, 9, 1000, 331, BF),
    (130, 33, 257, 64, HF),
    (5, 256, 4000, 128, BF),
    (2, 300, 128, 1000, BF),
    (2, 400, 65, 1100, BF),         # more columns than one slice of the gathered sums
    (3, 320, 500, 331, HF),
    (200, 2, 700, 96, BF),          # more texts than one round of the gathered sums
    (150, 300, 40, 96, HF),
])
def test_sparse_head(B, Lt, V, D, dt):
    h, w, b, dy = head_inputs(B, Lt, V, D, dt, seed=B + Lt)
    check_head(h, w, b, None, dy)
    g = torch.Generator().manual_seed(B)
    mask = (torch.rand(B, Lt, generator=g) < 0.6).to(DEV)        # any pattern
    if B > 2:
        mask[1] = False
    check_head(h, w, b, mask, dy)
    check_head(h, w, None, mask, dy)


def test_sparse_head_of_texts_longer_than_the_sort_counts():
    """Texts past 12288 tokens go through the products, however sparse their terms are."""
    h, w, b, dy = head_inputs(2, 13000, 65, 16, BF, seed=36)
    mask = torch.ones(2, 13000, dtype=torch.bool, device=DEV)
    mask[1, 77:] = False
    check_head(h, w, b, mask, dy)


def test_sparse_head_masked_tokens_hold_anything():
    h, w, b, dy = head_inputs(6, 50, 500, 64, BF, seed=31)
    mask = torch.zeros(6, 50, dtype=torch.bool, device=DEV)
    for i, n in enumerate([50, 20, 0, 1, 33, 7]):
        mask[i, :n] = True
    y, got = check_head(h, w, b, mask, dy)
    h2 = h.clone()
    h2[~mask] = float("nan")
    y2, got2 = check_head(h2, w, b, mask.to(torch.int64), dy)
    assert torch.equal(y, y2) and all(torch.equal(a, c) for a, c in zip(got, got2))
    assert (y[2] == 0).all() and (got[0][2] == 0).all()


def test_sparse_head_ties_go_to_the_first_token():
    import gpusparse
    h, w, b, dy = head_inputs(3, 40, 300, 64, BF, seed=32)
    h[:, 20:] = h[:, :20]                     # every token twice
    _, got = check_head(h, w, b, None, dy)
    assert (got[0][:, 20:] == 0).all()


def test_sparse_head_propagates_nan_of_tokens_that_take_part():
    import gpusparse
    h, w, b, dy = head_inputs(3, 40, 300, 64, BF, seed=33)
    h[1, 17] = float("nan")
    y = gpusparse.sparse_head(h, w, bias=b)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()


def test_sparse_head_without_texts_or_tokens():
    import gpusparse
    h, w, b, _ = head_inputs(3, 4, 50, 16, BF, seed=34)
    assert gpusparse.sparse_head(h[:0], w, bias=b).shape == (0, 50)
    assert (gpusparse.sparse_head(h[:, :0], w, bias=b) == 0).all()
    none = torch.zeros(3, 4, dtype=torch.bool, device=DEV)
    wl = leaf(w)
    y = gpusparse.sparse_head(h, wl, bias=b, mask=none)
    (dw,) = torch.autograd.grad(y.sum(), wl)
    assert (y == 0).all() and (dw == 0).all()


# ---------------------------------------------------------------------------- how calls run
def step(h, w, b, targets, scores, ids):
    import gpusparse
    loss = gpusparse.vocab_cross_entropy(h, w, targets, bias=b) + \
        gpusparse.topk_distillation(h, w, scores, ids, bias=b) + \
        gpusparse.sparse_head(h[None], w, bias=b).mean()
    return (loss.detach(),) + torch.autograd.grad(loss, (h, w, b))


def step_inputs(seed):
    h, w, b = make(300, 900, 96, BF, seed=seed)
    targets = torch.arange(300, device=DEV) * 3
    scores, ids = teacher(300, 900, 12, seed=seed)
    return leaf(h), leaf(w), leaf(b), targets, scores, ids


def test_equal_inputs_give_equal_bits_on_any_stream():
    a = step(*step_inputs(41))
    s = torch.cuda.Stream()
    inputs = step_inputs(41)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = step(*inputs)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_captured_training_step_replays_on_new_inputs():
    """Forward and backward in one CUDA graph, then other values in the same tensors; two
    graphs captured over the same leaves keep their own buffers."""
    inputs = step_inputs(42)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*inputs)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*inputs)
        graphs.append((g, out))
    other = step_inputs(43)
    want = step(*other)
    with torch.no_grad():
        for x, y in zip(inputs, other):
            x.copy_(y)
    for g, _ in graphs:
        g.replay()
    for _, out in graphs:
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_wait_that_runs_out_shows_in_the_result():
    """With no polls allowed some wait gives up: the results are NaN, nothing hangs, and the
    next call is right again."""
    import gpusparse
    import gpusparse._lib as L
    h, w, b = make(300, 900, 512, BF, seed=44)
    targets = torch.arange(300, device=DEV) * 3
    want = gpusparse.vocab_cross_entropy(h, w, targets, bias=b)
    lib = L.lib()
    default = lib.gsp_get_wait_limit()
    L.check(lib.gsp_set_wait_limit(0), "wait limit")
    try:
        got = [gpusparse.vocab_cross_entropy(h, w, targets, bias=b) for _ in range(3)]
        y = gpusparse.sparse_head(h[None], w, bias=b)
        torch.cuda.synchronize()
    finally:
        L.check(lib.gsp_set_wait_limit(default), "wait limit")
    assert any(torch.isnan(x).item() for x in got)
    assert torch.isnan(y).any()
    assert torch.equal(gpusparse.vocab_cross_entropy(h, w, targets, bias=b), want)


def test_backward_twice_and_changed_inputs():
    import gpusparse
    h, w, b = make(100, 400, 64, BF, seed=45)
    targets = torch.arange(100, device=DEV)
    hl, wl, bl = leaf(h), leaf(w), leaf(b)
    loss = gpusparse.vocab_cross_entropy(hl, wl, targets, bias=bl)
    first = torch.autograd.grad(loss, (hl, wl, bl), retain_graph=True)
    targets.fill_(7)                              # the forward call kept its own
    second = torch.autograd.grad(loss, (hl, wl, bl), retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(first, second))
    only = torch.autograd.grad(loss, (wl,), retain_graph=True)
    assert torch.equal(only[0], first[1])
    with torch.no_grad():
        wl.add_(1.0)                              # the weight is needed unchanged
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, (hl,))


@pytest.mark.parametrize("which", ["h", "w", "b", "hb", "wb", "hw"])
def test_gradients_asked_for_one_by_one(which):
    """Any subset of the gradients equals the same ones of a full backward pass."""
    import gpusparse
    h, w, b = make(300, 700, 72, BF, seed=46)
    targets = torch.arange(300, device=DEV) * 2
    scores, ids = teacher(300, 700, 9, seed=2)
    dy = torch.randn(3, 700, generator=torch.Generator().manual_seed(1)).to(DEV)
    calls = [lambda a, c, d: gpusparse.vocab_cross_entropy(a, c, targets, bias=d),
             lambda a, c, d: gpusparse.topk_distillation(a, c, scores, ids, bias=d),
             lambda a, c, d: (gpusparse.sparse_head(a.reshape(3, 100, 72), c, bias=d) * dy).sum(),
             lambda a, c, d: (gpusparse.sparse_head(a[:60].reshape(30, 2, 72), c, bias=d)[:3] * dy).sum()]
    for call in calls:
        full = [leaf(h), leaf(w), leaf(b)]
        want = dict(zip("hwb", torch.autograd.grad(call(*full), full)))
        some = [leaf(x) if n in which else x for n, x in zip("hwb", (h, w, b))]
        got = torch.autograd.grad(call(*some), [x for n, x in zip("hwb", some) if n in which])
        for n, x in zip([n for n in "hwb" if n in which], got):
            assert torch.equal(x, want[n]), n


def test_skewed_winners():
    """One token of a long text wins nearly every term: its row of d_hidden sums thousands of
    entries (shared by a CTA's warps), the others few."""
    h, w, b, dy = head_inputs(2, 300, 3000, 96, BF, seed=47, bias_mean=0.0)
    b += 8.0
    h[:, 1:] = 0
    h[:, 0] = (w.float().mean(0) * 0 + 0.03125).to(BF)
    h[1, 7] = 0.0625
    _, got = check_head(h, w, b, None, dy)
    assert int((got[0][0].abs().sum(1) > 0).sum()) <= 300


def test_overlapping_calls_on_two_streams():
    """Calls in flight at the same time keep to their own buffers."""
    import gpusparse
    inputs = [step_inputs(48), step_inputs(49)]
    want = [step(*x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_buffers_are_freed_with_the_backward_pass():
    """A kept loss or kept weights hold none of the buffers of their backward pass once it has
    run, and hooks on saved tensors see all of them."""
    import gpusparse
    h, w, b, targets, scores, ids = step_inputs(52)
    calls = (lambda: gpusparse.vocab_cross_entropy(h, w, targets, bias=b),
             lambda: gpusparse.topk_distillation(h, w, scores, ids, bias=b),
             lambda: gpusparse.sparse_head(h[None], w, bias=b))
    for call in calls:
        want = torch.autograd.grad(call().sum(), (h, w, b))
        del want
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = call()
        torch.autograd.grad(out.sum(), (h, w, b))
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before <= (out.numel() * 4 + 511) // 512 * 512
        with pytest.raises(RuntimeError):
            torch.autograd.grad(out.sum(), (h, w, b))
        want = torch.autograd.grad(call().sum(), (h, w, b))
        with torch.autograd.graph.save_on_cpu():
            out = call()
        got = torch.autograd.grad(out.sum(), (h, w, b))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("D,ld", [(83, 88), (83, 83), (88, 96)])
def test_hooks_may_change_the_layout_of_the_weight(D, ld):
    import gpusparse
    h, _, b = make(20, 300, D, BF, seed=53)
    wide = (torch.randn(300, ld, generator=torch.Generator().manual_seed(54)) * 0.2).to(BF).to(DEV)
    targets = torch.arange(20, device=DEV)
    for call in (lambda h, w: gpusparse.vocab_cross_entropy(h, w, targets, bias=b),
                 lambda h, w: gpusparse.sparse_head(h[None], w, bias=b)):
        got = []
        for hook in (False, True):
            hl, wl = leaf(h), wide[:, :D].requires_grad_(True)
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x.clone(memory_format=torch.contiguous_format)
                                                          if hook else x, lambda x: x):
                out = call(hl, wl)
            got.append(torch.autograd.grad(out.sum(), (hl, wl)))
        assert all(torch.equal(x, y) for x, y in zip(*got))


def test_sparse_head_of_empty_texts_has_zero_gradients():
    import gpusparse
    h, w, b, _ = head_inputs(3, 4, 50, 16, BF, seed=35)
    for some in (h[:, :0], h[:0], h[:0, :0]):
        leaves = [leaf(some), leaf(w), leaf(b)]
        y = gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2])
        assert y.shape == (some.shape[0], 50) and (y == 0).all()
        got = torch.autograd.grad(y.sum(), leaves)
        assert all(g.shape == x.shape and (g == 0).all() for g, x in zip(got, leaves))


# ---------------------------------------------------------------------------- refusals
def test_refusals():
    import gpusparse
    h, w, b = make(10, 50, 16, BF, seed=51)
    t = torch.zeros(10, dtype=torch.int64, device=DEV)
    ce, di, sh = gpusparse.vocab_cross_entropy, gpusparse.topk_distillation, gpusparse.sparse_head
    s, i = torch.zeros(10, 4, device=DEV), torch.zeros(10, 4, dtype=torch.int64, device=DEV)
    for bad in (lambda: ce(h.float(), w.float(), t), lambda: ce(h, w.half(), t), lambda: ce(h, w[:, :8], t),
                lambda: ce(h, w, t[:5]), lambda: ce(h, w, t.float()), lambda: ce(h, w, t, bias=b[:9]),
                lambda: ce(h, w, t, reduction="median"), lambda: ce(h, w[:0], t),
                lambda: ce(h, w, t.cpu()), lambda: ce(h, w.cpu(), t.cpu()) if False else ce(h, w, t, bias=b.cpu()),
                lambda: di(h, w, s, i[:, :3]), lambda: di(h, w, s, i, temperature=0.0),
                lambda: di(h, w, s, i, temperature=float("inf")), lambda: di(h, w, s, s), lambda: di(h, w, i, i),
                lambda: di(h, w, torch.zeros(10, 1025, device=DEV), torch.zeros(10, 1025, dtype=torch.int64, device=DEV)),
                lambda: di(h, w, s[:, :0], i[:, :0]), lambda: sh(h, w), lambda: sh(h[None], w, mask=t[None, :3]),
                lambda: gpusparse.encode_queries(h[None], w, max_terms=0),
                lambda: gpusparse.encode_documents(h[None], w, min_weight=-1.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        ce(h.cpu(), w, t)


# ---------------------------------------------------------------------------- used together
@pytest.mark.parametrize("dt", [BF, HF])
def test_encode_index_search_and_distil(dt):
    """Documents and queries through the head, an index of the documents, the scorer's top-k
    against the dense product of the weights, and a distillation step on what it returned."""
    import gpusparse
    V, D, N, Q = 2000, 64, 300, 20
    h, w, b, _ = head_inputs(N, 24, V, D, dt, seed=61, bias_mean=-3.0)
    hq = head_inputs(Q, 8, V, D, dt, seed=62)[0]
    mask = (torch.arange(24, device=DEV)[None, :] < torch.randint(1, 25, (N, 1), generator=torch.Generator().manual_seed(5)).to(DEV))
    yd = gpusparse.sparse_head(h, w, bias=b, mask=mask)
    ip, ix, dtv = gpusparse.encode_documents(h, w, bias=b, mask=mask)
    dense = torch.zeros_like(yd)
    rows = torch.repeat_interleave(torch.arange(N, device=DEV), ip[1:] - ip[:-1])
    dense[rows, ix.long()] = dtv
    assert torch.equal(dense, yd)
    index = gpusparse.build_index_from_hidden([(h[:128], mask[:128]), (h[128:], mask[128:])], w, bias=b)
    assert index.num_docs == N and index.vocab_size == V
    qi, qs = gpusparse.encode_queries(hq, w, bias=b, max_terms=512)
    yq = gpusparse.sparse_head(hq, w, bias=b)
    assert int((yq > 0).sum(1).max()) <= 512
    back = torch.zeros(Q, V + 1, device=DEV).scatter_(1, qi.long() % (V + 1), qs)[:, :V]
    assert torch.equal(back, yq)
    scores, ids = gpusparse.triton_fused_score(index, qi, qs, top_k=50)
    full = yq.double() @ yd.double().t()
    want = full.topk(50, dim=1).values
    assert torch.allclose(scores.double(), want, rtol=1e-5, atol=1e-6)
    assert torch.allclose(full.gather(1, ids), want, rtol=1e-5, atol=1e-6)
    # a student that scores the documents by dense vectors learns the ranking
    sq, sd = make(Q, N, D, dt, seed=63, bias=False)[:2]
    check_distill(sq, sd, None, scores, ids, 2.0, grad=1.0 if dt == BF else 256.0)


# ---------------------------------------------------------------------------- waits that run out
@pytest.mark.parametrize("limit", [0, 2])
def test_wait_that_runs_out_in_the_backward_pass(limit):
    """The logits' gradient and the products (whole tiles, cut ones, and P in two parts) under a
    wait limit that some wait exceeds: NaN gradients, nothing hangs, and the next pass over the
    same state is right again."""
    import gpusparse
    import gpusparse._lib as L
    h, w, b = make(300, 900, 512, BF, seed=71)
    targets = torch.arange(300, device=DEV) * 3
    scores, ids = teacher(300, 900, 12, seed=71)
    calls = [lambda a, c, d: gpusparse.vocab_cross_entropy(a, c, targets, bias=d),
             lambda a, c, d: gpusparse.vocab_cross_entropy(a[:40], c, targets[:40], bias=d),
             lambda a, c, d: gpusparse.topk_distillation(a, c, scores, ids, bias=d),
             lambda a, c, d: gpusparse.sparse_head(a.reshape(150, 2, 512), c, bias=d).sum()]
    lib = L.lib()
    default = lib.gsp_get_wait_limit()
    for call in calls:
        leaves = [leaf(h), leaf(w), leaf(b)]
        out = call(*leaves)
        want = torch.autograd.grad(out, leaves, retain_graph=True)
        torch.cuda.synchronize()
        L.check(lib.gsp_set_wait_limit(limit), "wait limit")
        try:
            got = [torch.autograd.grad(out, leaves, retain_graph=True) for _ in range(3)]
            torch.cuda.synchronize()
        finally:
            L.check(lib.gsp_set_wait_limit(default), "wait limit")
        if limit == 0:
            assert any(torch.isnan(g).any().item() for grads in got for g in grads)
        after = torch.autograd.grad(out, leaves)
        assert all(torch.equal(x, y) for x, y in zip(after, want))


# ---------------------------------------------------------------------------- NaN
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("Lt,V", [(40, 300), (300, 300), (700, 300), (33, 2000)])
def test_sparse_head_gradients_of_nan_weights(Lt, V, zero, dt):
    """A token that takes part and holds NaN wins every term of its text: its row of d_hidden, and
    all of d_weight and d_bias, are NaN (also where dy is 0, as 0 / (1 + NaN) is), whether rows are
    gathered (long texts) or multiplied, and where shares cut the text.  The other texts' rows of
    d_hidden are those they have without it."""
    import gpusparse
    h, w, b, dy = head_inputs(3, Lt, V, 64, dt, seed=81)
    mask = torch.ones(3, Lt, dtype=torch.bool, device=DEV)
    mask[1] = False
    _, ((rh, bh), _, _) = R.sparse_head(h, w, b, mask, dy, dt)
    h[1, 17] = float("nan")
    h[1, 30] = float("nan")
    if zero:
        dy[1] = 0
    leaves = [leaf(h), leaf(w), leaf(b)]
    y = gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2])
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2]).all()
    dh, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.isnan(dh[1, 17]).all() and torch.isnan(dw).all() and torch.isnan(db).all()
    dh[1, 17] = 0
    assert (dh[1] == 0).all()
    R.assert_within(dh.reshape(3 * Lt, 64), (rh, bh), "dh")


@pytest.mark.parametrize("Lt", [40, 300])
def test_sparse_head_gradients_of_a_nan_bias(Lt):
    import gpusparse
    h, w, b, dy = head_inputs(3, Lt, 300, 64, BF, seed=82)
    b[5] = float("nan")
    leaves = [leaf(h), leaf(w), leaf(b)]
    y = gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2])
    assert torch.equal(torch.isnan(y), (torch.arange(300, device=DEV) == 5).expand(3, 300))
    dh, dw, db = torch.autograd.grad(y, leaves, dy)
    assert torch.isnan(db[5]) and torch.isnan(dw[5]).all()
    assert int(torch.isnan(db).sum()) == 1 and int(torch.isnan(dw).any(1).sum()) == 1
    assert (torch.isnan(dh).all(2).sum(1) == 1).all() and (torch.isnan(dh).any(2).sum(1) == 1).all()


def test_sparse_head_gradients_of_a_wait_that_ran_out():
    """NaN weights of a wait that ran out have NaN gradients, not those of the other terms."""
    import gpusparse
    import gpusparse._lib as L
    h, w, b = make(300, 900, 512, BF, seed=83)
    lib = L.lib()
    default = lib.gsp_get_wait_limit()
    leaves = [leaf(h), leaf(w), leaf(b)]
    L.check(lib.gsp_set_wait_limit(0), "wait limit")
    try:
        y = gpusparse.sparse_head(leaves[0].reshape(3, 100, 512), leaves[1], bias=leaves[2])
        torch.cuda.synchronize()
    finally:
        L.check(lib.gsp_set_wait_limit(default), "wait limit")
    bad = torch.isnan(y)
    assert bad.any()
    dh, dw, db = torch.autograd.grad(y.sum(), leaves)
    terms = bad.any(0)
    assert torch.isnan(db[terms]).all() and torch.isnan(dw[terms]).all() and torch.isnan(dh).any()


def test_encoding_shows_nan_weights():
    """NaN weights of a document or query do not pass for missing terms: encode_documents and
    build_index_from_hidden raise, encode_queries gives the query NaN weights."""
    import gpusparse
    h, w, b, _ = head_inputs(4, 20, 600, 64, BF, seed=84, bias_mean=-2.0)
    qi, qs = gpusparse.encode_queries(h, w, bias=b, max_terms=50)
    ip, ix, dtv = gpusparse.encode_documents(h, w, bias=b)
    h[2, 5] = float("nan")
    with pytest.raises(RuntimeError, match="NaN"):
        gpusparse.encode_documents(h, w, bias=b)
    with pytest.raises(RuntimeError, match="NaN"):
        gpusparse.encode_documents(h, w, bias=b, min_weight=0.5)
    with pytest.raises(RuntimeError, match="NaN"):
        gpusparse.build_index_from_hidden([h[:2], h[2:]], w, bias=b)
    mask = torch.ones(4, 20, dtype=torch.bool, device=DEV)
    mask[2, 5] = False
    gpusparse.encode_documents(h, w, bias=b, mask=mask)
    qi2, qs2 = gpusparse.encode_queries(h, w, bias=b, max_terms=50)
    others = torch.tensor([0, 1, 3], device=DEV)
    assert torch.equal(qi2[others], qi[others]) and torch.equal(qs2[others], qs[others])
    assert torch.isnan(qs2[2]).all() and int(qi2[2, 0]) >= 0
    b[7] = float("nan")                                       # one term of every text
    with pytest.raises(RuntimeError, match="NaN"):
        gpusparse.encode_documents(h[:1], w, bias=b)
    qi3, qs3 = gpusparse.encode_queries(h[:1], w, bias=b, max_terms=700)
    assert torch.isnan(qs3).all() and qs3.shape == (1, 700) and int(qi3[0, 0]) >= 0


def test_encoding_shows_a_wait_that_ran_out():
    import gpusparse
    import gpusparse._lib as L
    h, w, b = make(300, 900, 512, BF, seed=85)
    lib = L.lib()
    default = lib.gsp_get_wait_limit()
    L.check(lib.gsp_set_wait_limit(0), "wait limit")
    try:
        with pytest.raises(RuntimeError, match="NaN"):
            gpusparse.encode_documents(h[None], w, bias=b)
        qs = gpusparse.encode_queries(h[None], w, bias=b)[1]
        torch.cuda.synchronize()
    finally:
        L.check(lib.gsp_set_wait_limit(default), "wait limit")
    assert torch.isnan(qs).all()


@pytest.mark.parametrize("case", ["tiny", "outlier"])
def test_sparse_head_fp16_gradients_scale_with_the_entries_that_have_one(case):
    """The products' 16-bit P is scaled by the largest dy of a term that has a weight: neither a
    dy of 1e-36 (whose reciprocal leaves fp32) nor a huge dy of terms without weight costs the
    others their gradient."""
    import gpusparse
    h, w, b, dy = head_inputs(30, 3, 700, 64, HF, seed=86)
    ref, _ = R.sparse_head(h, w, b, torch.ones(30, 3, dtype=torch.bool, device=DEV), dy, HF)
    live = ref[0] > 0
    assert 0.1 < float(live.double().mean()) < 0.9
    dy = dy * 1e-36 if case == "tiny" else torch.where(live, dy, 1e30)
    _, (rh, rw, rb) = R.sparse_head(h, w, b, torch.ones(30, 3, dtype=torch.bool, device=DEV),
                                    torch.where(live, dy, 0.0), HF)
    leaves = [leaf(h), leaf(w), leaf(b)]
    got = torch.autograd.grad(gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2]), leaves, dy)
    R.assert_within(got[0].reshape(-1, 64), rh, "dh")
    R.assert_within(got[1], rw, "dw")
    # (fp32 results of 1e-36 have no subnormal parts to lose: 2^-126 is 1e-38)
    R.assert_within(got[2], (rb[0], rb[1] + (2.0 ** -126 * 30 if case == "tiny" else 0.0)), "db")


def test_forward_mode_derivatives_are_refused():
    """A dual tensor needs no gradient, but its result without a tangent would be wrong."""
    import torch.autograd.forward_ad as fwd
    import gpusparse
    h, w, b, targets, scores, ids = step_inputs(87)
    h, w, b = h.detach(), w.detach(), b.detach()
    for call in (lambda h, w, b: gpusparse.vocab_cross_entropy(h, w, targets, bias=b),
                 lambda h, w, b: gpusparse.topk_distillation(h, w, scores, ids, bias=b),
                 lambda h, w, b: gpusparse.sparse_head(h[None], w, bias=b),
                 lambda h, w, b: gpusparse.encode_documents(h[None], w, bias=b)):
        want = call(h, w, b)
        for which in range(3):
            with fwd.dual_level():
                args = [h, w, b]
                args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
                with pytest.raises(RuntimeError):
                    call(*args)
                with torch.no_grad(), pytest.raises(RuntimeError):
                    call(*args)
                got = call(h, w, b)                # no tangent: nothing to refuse
        if isinstance(want, torch.Tensor):
            assert torch.equal(got, want)


def test_differentiating_a_gradient_again_is_refused():
    import gpusparse
    h, w, b, targets, scores, ids = step_inputs(88)
    for call in (lambda: gpusparse.vocab_cross_entropy(h, w, targets, bias=b),
                 lambda: gpusparse.topk_distillation(h, w, scores, ids, bias=b),
                 lambda: gpusparse.sparse_head(h[None], w, bias=b).sum()):
        want = torch.autograd.grad(call(), (h, w, b))
        got = torch.autograd.grad(call(), (h, w, b), create_graph=True)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        with pytest.raises(RuntimeError):
            got[0].float().sum().backward()


@pytest.mark.parametrize("D", [83, 88])
def test_hooks_may_change_the_layout_of_all_saved_tensors(D):
    """Matrices saved column by column, and buffers (the state) off their boundaries."""
    import gpusparse
    h, w, b = make(60, 300, D, BF, seed=55)
    targets = torch.arange(60, device=DEV)
    scores, ids = teacher(60, 300, 5, seed=55)
    dy = torch.randn(6, 300, generator=torch.Generator().manual_seed(1)).to(DEV)

    def pack(x):
        if x.dim() == 2:
            return x.detach().t().contiguous()
        return torch.cat((x.detach().new_zeros(8), x.detach()))

    def unpack(x):
        return x.t() if x.dim() == 2 else x[8:]
    for call in (lambda h, w, b: gpusparse.vocab_cross_entropy(h, w, targets, bias=b),
                 lambda h, w, b: gpusparse.topk_distillation(h, w, scores, ids, bias=b),
                 lambda h, w, b: (gpusparse.sparse_head(h.reshape(6, 10, D), w, bias=b) * dy).sum()):
        plain = [leaf(h), leaf(w), leaf(b)]
        want = torch.autograd.grad(call(*plain), plain)
        hooked = [leaf(h), leaf(w), leaf(b)]
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            out = call(*hooked)
        got = torch.autograd.grad(out, hooked)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("tau", [1.1e-19, 1e-6, 1e-2, 1e3, 1e6, 1.8e19])
def test_distillation_at_extreme_temperatures(tau):
    import gpusparse
    h, w, b = make(40, 300, 64, BF, seed=56)
    scores, ids = teacher(40, 300, 7, seed=56)
    leaves = [leaf(h), leaf(w), leaf(b)]
    loss = gpusparse.topk_distillation(*leaves[:2], scores, ids, bias=leaves[2], temperature=tau)
    grads = torch.autograd.grad(loss, leaves)
    assert torch.isfinite(loss.detach()) or tau > 1e18          # (tau^2 ln(300 / 7) leaves fp32)
    assert all(torch.isfinite(g).all() for g in grads)
    if 1e-3 < tau < 1e7:
        p = torch.softmax(scores.double() / tau, 1)
        q = torch.zeros(40, 300, dtype=torch.float64, device=DEV).scatter_(1, ids, p)
        rows = torch.full((40,), 1 / 40, device=DEV)
        ref, refs = R.softmax_loss(h, w, b, q, torch.ones(40, dtype=torch.bool, device=DEV), tau, rows, BF)
        R.assert_within(loss.detach(), (ref[0].mean(), ref[1].mean() + 2.0 ** -23 * ref[0].mean().abs()), "loss")
        # at small temperatures softmax values pass below 2^-126, where they count as 0: P is off
        # by 2^-126 of the row's coefficient tau / 40 there, its sums by that times the other
        # operand (bf16's own subnormal steps are 2^-133 and with that less)
        floor = 2.0 ** -126 * max(tau / 40, 1.0)
        sums = (300 * float(w.abs().max()), 40 * float(h.abs().max()), 40)
        for g, (value, bound), n, what in zip(grads, refs, sums, ("dh", "dw", "db")):
            R.assert_within(g, (value, bound + n * floor), what)
    with pytest.raises(ValueError):
        gpusparse.topk_distillation(h, w, scores, ids, temperature=1e-25)
    with pytest.raises(ValueError):
        gpusparse.topk_distillation(h, w, scores, ids, temperature=1e25)


def test_sparse_head_of_a_text_longer_than_a_grid_is_deep():
    """4.2 million tokens, more than 65535 blocks of 64 rows: the same winners and gradients as any."""
    h, w, b, dy = head_inputs(1, 65535 * 64 + 100, 20, 8, BF, seed=57)
    h[0, -50:] += 4.0           # the last rows, which only a second round reaches, win terms
    _, got = check_head(h, w, b, None, dy)
    assert (got[0][0, -50:] != 0).any()


# ---------------------------------------------------------------------------- sizes and ways
def test_winners_of_thousands_of_terms_are_gathered():
    """The inputs of test_skewed_winners take the way they are meant for: few enough entries to be
    gathered, and tokens with more of them than one warp sums alone (256)."""
    h, w, b, dy = head_inputs(2, 300, 3000, 96, BF, seed=47, bias_mean=0.0)
    b += 8.0
    h[:, 1:] = 0
    h[:, 0] = 0.03125
    h[1, 7] = 0.0625
    s = h.double() @ w.double().t() + b.double()
    best, arg = s.max(dim=1)
    assert (best > 0).all() and (dy != 0).all()
    wins = torch.stack([torch.bincount(a, minlength=300) for a in arg])
    assert (wins.max(dim=1).values > 256).all() and int((wins > 256).sum()) >= 3
    assert dy.numel() * 160 <= 600 * 3000
    check_head(h, w, b, None, dy)


@pytest.mark.parametrize("dt", [BF, HF])
def test_sparse_head_products_in_pieces(dt):
    """Short texts with dense terms, more tokens x vocabulary than one piece of P holds: d_hidden is
    carried over the pieces in fp32.  The reference is the definition, 250 texts at a time."""
    import gpusparse
    B, Lt, V, D = 2000, 10, 15000, 40
    h, w, b, dy = head_inputs(B, Lt, V, D, dt, seed=91)
    dy = dy.clamp_(-3.0, 3.0)
    dy[:, 0] = 3.0                                   # every block of texts has the same largest dy
    leaves = [leaf(h), leaf(w), leaf(b)]
    y = gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2])
    assert int((y > 0).sum()) * 160 > B * Lt * V and B * Lt * V * 2 > 512 << 20
    dh, dw, db = torch.autograd.grad(y, leaves, dy)
    rw = [torch.zeros(V, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    rb = [torch.zeros(V, dtype=torch.float64, device=DEV) for _ in range(2)]
    all_in = torch.ones(250, Lt, dtype=torch.bool, device=DEV)
    for lo in range(0, B, 250):
        r = slice(lo, lo + 250)
        ref, (qh, qw, qb) = R.sparse_head(h[r], w, b, all_in, dy[r], dt)
        R.assert_within(y.detach()[r], ref, "y")
        R.assert_within(dh[r].reshape(-1, D), qh, "dh")
        for total, part in ((rw, qw), (rb, qb)):
            total[0] += part[0]
            total[1] += part[1]
    # the blocks' bounds count sums of 2500 terms; the whole sum has 20000, each of at most the
    # bound / u (the bound has u times every term)
    rw[1] += B * Lt * 2.0 ** -23 * rw[1] / R.U[dt]
    # d_bias: fp32 sums of 2000 terms of at most 3
    rb[1] += B * 2.0 ** -24 * 3.0 * B
    R.assert_within(dw, rw, "dw")
    R.assert_within(db, rb, "db")


def test_cross_entropy_offsets_past_32_bits():
    """2.3e9 hidden values: rows are read, packed and written behind 2^31 elements."""
    import gpusparse
    T, V, D = 3_000_000, 300, 768
    g = torch.Generator(device=DEV).manual_seed(92)
    h = torch.randn(T, D, generator=g, device=DEV, dtype=BF)
    w = (torch.randn(V, D, generator=g, device=DEV) * (2.0 / D ** 0.5)).to(BF)
    targets = torch.randint(0, V, (T,), generator=g, device=DEV)
    targets[torch.rand(T, generator=g, device=DEV) < 0.02] = -100
    rows = torch.randn(T, generator=g, device=DEV)
    hl, wl = h.requires_grad_(True), leaf(w)
    loss = gpusparse.vocab_cross_entropy(hl, wl, targets, reduction="none")
    dh, dw = torch.autograd.grad(loss, (hl, wl), rows)
    loss, h = loss.detach(), h.detach()
    want, off = torch.zeros(V, D, dtype=torch.float64, device=DEV), torch.zeros(V, D, dtype=torch.float64, device=DEV)
    for lo in range(0, T, 100_000):
        r = slice(lo, lo + 100_000)
        live = targets[r] >= 0
        ref, (rh, rw, _) = R.softmax_loss(h[r], w, None, one_hot(targets[r], V, live), live, 1.0, rows[r], BF)
        assert ((loss[r].double() - ref[0]).abs() <= ref[1]).all()      # (compared on the GPU: 2.3e9 values)
        assert ((dh[r].double() - rh[0]).abs() <= rh[1]).all()
        want += rw[0]
        off += rw[1]
    # as above: sums of 3e6 terms instead of 1e5
    R.assert_within(dw, (want, off + T * 2.0 ** -23 * off / R.U[BF]), "dw")


def test_sparse_head_offsets_past_32_bits():
    """60000 texts x 40000 terms, 2.4e9 weights; the gradient comes from the last texts."""
    import gpusparse
    B, V, D = 60_000, 40_000, 16
    g = torch.Generator(device=DEV).manual_seed(93)

    def grid(x, step):
        return torch.round(x / step) * step
    h = grid(torch.randn(B, 1, D, generator=g, device=DEV).clamp(-3.9, 3.9), 2.0 ** -5).to(BF)
    w = grid((torch.randn(V, D, generator=g, device=DEV) / 4).clamp(-0.24, 0.24), 2.0 ** -10).to(BF)
    b = grid(torch.randn(V, generator=g, device=DEV) * 0.5 - 1.0, 2.0 ** -10)
    leaves = [leaf(h), leaf(w), leaf(b)]
    y = gpusparse.sparse_head(leaves[0], leaves[1], bias=leaves[2])
    dy = torch.zeros(B, V, device=DEV)
    dy[-40:] = torch.randn(40, V, generator=g, device=DEV)
    dh, dw, db = torch.autograd.grad(y, leaves, dy)
    one = torch.ones(40, 1, dtype=torch.bool, device=DEV)
    for r in (slice(0, 40), slice(53_680, 53_720), slice(B - 40, B)):       # 53687 x 40000 > 2^31
        ref, (rh, rw, rb) = R.sparse_head(h[r], w, b, one, dy[r], BF)
        R.assert_within(y.detach()[r], ref, "y")
        R.assert_within(dh[r].reshape(40, D), rh, "dh")
    R.assert_within(dw, rw, "dw")
    R.assert_within(db, rb, "db")
    assert (dh[:-40] == 0).all()


@pytest.mark.parametrize("T", [60, 300])
def test_losses_of_rows_with_nan_or_infinities(T):
    """A row that takes part and holds NaN or an infinity has a NaN loss and row of d_hidden, and
    makes d_weight and d_bias NaN; the other rows' losses and gradients keep their bits."""
    import gpusparse
    h, w, b = make(T, 500, 64, BF, seed=94)
    targets = torch.arange(T, device=DEV)
    scores, ids = teacher(T, 500, 6, seed=94)
    rows = torch.linspace(0.5, 2.0, T, device=DEV)
    bad = [3, T - 1]
    for call in (lambda x: gpusparse.vocab_cross_entropy(x[0], x[1], targets, bias=x[2], reduction="none"),
                 lambda x: gpusparse.topk_distillation(x[0], x[1], scores, ids, bias=x[2], reduction="none")):
        clean = [leaf(h), leaf(w), leaf(b)]
        want = call(clean)
        grads = torch.autograd.grad(want, clean, rows)
        h2 = h.clone()
        h2[3, 5], h2[T - 1, 60] = float("nan"), float("inf")
        some = [leaf(h2), leaf(w), leaf(b)]
        got = call(some)
        dh, dw, db = torch.autograd.grad(got, some, rows)
        others = torch.ones(T, dtype=torch.bool, device=DEV)
        others[bad] = False
        assert torch.isnan(got[bad]).all() and torch.equal(got[others], want[others])
        assert torch.isnan(dh[bad]).all() and torch.equal(dh[others], grads[0][others])
        assert torch.isnan(dw).all() and torch.isnan(db).all()


def test_cross_entropy_of_a_target_outside_the_masked_vocabulary():
    """A target whose bias is -inf: an infinite loss with the gradient softmax - one-hot."""
    import gpusparse
    h, w, b = make(50, 300, 64, BF, seed=95)
    targets = torch.arange(50, device=DEV) * 5
    b[20] = float("-inf")                       # row 4's target
    leaves = [leaf(h), leaf(w), leaf(b)]
    loss = gpusparse.vocab_cross_entropy(leaves[0], leaves[1], targets, bias=leaves[2], reduction="none")
    rows = torch.ones(50, device=DEV)
    live = torch.ones(50, dtype=torch.bool, device=DEV)
    ref, (rh, rw, rb) = R.softmax_loss(h, w, b, one_hot(targets, 300, live), live, 1.0, rows, BF)
    assert float(loss[4]) == float("inf") and float(ref[0][4]) == float("inf")
    keep = torch.arange(50, device=DEV) != 4
    R.assert_within(loss.detach()[keep], (ref[0][keep], ref[1][keep]), "loss")
    for g, r, what in zip(torch.autograd.grad(loss, leaves, rows), (rh, rw, rb), ("dh", "dw", "db")):
        R.assert_within(g, r, what)


def test_encoding_of_nothing():
    import gpusparse
    h, w, b, _ = head_inputs(3, 4, 50, 16, BF, seed=96)
    ip, ix, dtv = gpusparse.encode_documents(h[:0], w, bias=b)
    assert ip.tolist() == [0] and ix.numel() == 0 and dtv.numel() == 0
    ip, ix, dtv = gpusparse.encode_documents(h[:, :0], w, bias=b)
    assert ip.tolist() == [0, 0, 0, 0] and ix.numel() == 0
    qi, qs = gpusparse.encode_queries(h[:0], w, bias=b, max_terms=7)
    assert qi.shape == (0, 7) and qs.shape == (0, 7)
    qi, qs = gpusparse.encode_queries(h[:, :0], w, bias=b, max_terms=70)
    assert qi.shape == (3, 70) and (qi == -1).all() and (qs == 0).all()


# ---------------------------------------------------------------------------- threads, devices
def test_calls_from_several_threads():
    """Each thread on a stream of its own, forward and backward passes interleaved."""
    import threading
    inputs = [step_inputs(101 + i) for i in range(4)]
    want = [step(*x) for x in inputs]
    torch.cuda.synchronize()
    got, errors = [[] for _ in inputs], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[i].append(step(*inputs[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:              # noqa: BLE001 (shown by the main thread)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(inputs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for outs, ref in zip(got, want):
        assert len(outs) == 8 and all(torch.equal(x, y) for out in outs for x, y in zip(out, ref))


def test_tensors_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    inputs = step_inputs(105)
    want = step(*inputs)
    there = [x.detach().to("cuda:1").requires_grad_(x.requires_grad) for x in inputs]
    got = step(*there)
    assert torch.cuda.current_device() == 0
    assert all(y.device.index == 1 and torch.equal(x, y.to(x.device)) for x, y in zip(want, got))


def test_weights_on_the_host_are_refused():
    import gpusparse
    h, w, b = make(10, 50, 16, BF, seed=51)
    t = torch.zeros(10, dtype=torch.int64, device=DEV)
    s, i = torch.zeros(10, 4, device=DEV), torch.zeros(10, 4, dtype=torch.int64, device=DEV)
    for bad in (lambda: gpusparse.vocab_cross_entropy(h, w.cpu(), t),
                lambda: gpusparse.topk_distillation(h, w.cpu(), s, i),
                lambda: gpusparse.sparse_head(h[None], w.cpu()),
                lambda: gpusparse.encode_documents(h[None], w.cpu()),
                lambda: gpusparse.encode_queries(h[None], w.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: gpusparse.topk_distillation(h, w, s.cpu(), i), lambda: gpusparse.topk_distillation(h, w, s, i.cpu()),
                lambda: gpusparse.topk_distillation(h, w, s, i, bias=b.cpu()),
                lambda: gpusparse.sparse_head(h[None], w, bias=b.cpu()),
                lambda: gpusparse.sparse_head(h[None], w, mask=torch.ones(1, 10))):
        with pytest.raises(ValueError):
            bad()


def test_batched_transforms_are_refused():
    import gpusparse
    h, w, _ = make(12, 50, 16, BF, seed=51)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: gpusparse.vocab_cross_entropy(x, w, t))(h.reshape(3, 4, 16))
    with pytest.raises(RuntimeError):
        torch.vmap(lambda x: gpusparse.sparse_head(x[None], w))(h.reshape(3, 4, 16))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: gpusparse.vocab_cross_entropy(x, w, t))(h[:4])
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: gpusparse.sparse_head(x[None], w), (h[:4],), (h[4:8],))


def test_compiled_callers():
    """A compiled function around the calls keeps their results and gradients (the calls themselves
    run as they are, between the compiled parts)."""
    import gpusparse
    h, w, b, targets, scores, ids = step_inputs(106)

    def f(h, w, b):
        return gpusparse.vocab_cross_entropy(h * 2, w, targets, bias=b) + \
            gpusparse.topk_distillation(h, w, scores, ids, bias=b) + \
            gpusparse.sparse_head(h[None], w, bias=b).mean()
    want = f(h, w, b)
    grads = torch.autograd.grad(want, (h, w, b))
    compiled = torch.compile(f, backend="eager")
    got = compiled(h, w, b)
    assert torch.equal(got, want)
    assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(got, (h, w, b)), grads))
    with torch.no_grad():
        assert torch.equal(compiled(h, w, b), want)
