"""Cases that measure the vocabulary-head operators: the sparse head that makes term
weights from an encoder's hidden states, the softmax cross entropy over the vocabulary
and the distillation from a teacher's top scores, each forward and in training steps.

A case is a dict of plain values; ``prepare`` makes its inputs on the GPU, ``run`` makes
one pass (the plain torch form, or with ``own`` the framework's operators), ``exact`` is
the same result from the definition in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST_FLOPS = 6 * 16384 * 30522 * 768      # the largest listed case's work
PLAIN_ROWS = 2048                            # rows whose fp32 logits the plain form holds


def _gpusparse():
    root = os.path.join(os.getcwd(), "gpu-sparse_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gpusparse
    return gpusparse


# ---------------------------------------------------------------------------- the cases
def listed():
    return [
        # one labelled token scored by itself, as an evaluation loop over single answers does
        dict(name="ce_one_token", op="ce", T=1, V=30522, D=768, dtype="fp16", frac=1.0, bias=True,
             train=False, scale=1.0),
        # a masked-token training step: 64 texts of 128 tokens, 15 % of them labelled
        dict(name="ce_masked_tokens", op="ce", T=8192, V=30522, D=768, dtype="bf16", frac=0.15,
             bias=True, train=True, scale=1.0),
        # every token labelled, the largest step
        dict(name="ce_every_token", op="ce", T=16384, V=30522, D=768, dtype="bf16", frac=1.0,
             bias=True, train=True, scale=1.0),
        # odd sizes, a projection without bias, fp16 with a scaled loss
        dict(name="ce_odd_fp16", op="ce", T=1237, V=10007, D=331, dtype="fp16", frac=0.6,
             bias=False, train=True, scale=4096.0),
        # a student that learns a few teacher answers for a handful of queries
        dict(name="distill_few", op="distill", T=32, V=30522, D=768, K=10, tau=1.0, dtype="bf16",
             bias=True, train=True, scale=1.0),
        # a teacher's 100 best terms for every token of a batch
        dict(name="distill_terms", op="distill", T=4096, V=30522, D=768, K=100, tau=2.0,
             dtype="bf16", bias=True, train=True, scale=1.0),
        # a teacher's 1000 best documents (what the scorer returns) for 500 queries over 100K
        dict(name="distill_documents", op="distill", T=500, V=100_000, D=256, K=1000, tau=1.0,
             dtype="fp16", bias=False, train=True, scale=1024.0),
        # one query encoded as it arrives
        dict(name="head_one_query", op="head", B=1, L=16, V=30522, D=768, dtype="bf16",
             bias_mean=-4.0, ragged=False, train=False),
        # a batch of queries of a few to some tens of tokens
        dict(name="head_queries", op="head", B=500, L=32, V=30522, D=768, dtype="bf16",
             bias_mean=-4.0, ragged=True, train=False),
        # documents of up to 512 tokens on their way into an index
        dict(name="head_documents", op="head", B=64, L=512, V=30522, D=768, dtype="fp16",
             bias_mean=-4.0, ragged=True, train=False),
        # a training step of the head on texts of up to 256 tokens
        dict(name="head_training", op="head", B=32, L=256, V=30522, D=768, dtype="bf16",
             bias_mean=-3.0, ragged=True, train=True),
        # odd sizes; one of the texts is empty
        dict(name="head_odd_fp16", op="head", B=7, L=77, V=10007, D=331, dtype="fp16",
             bias_mean=-1.0, ragged=True, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["ce", "distill", "head"])
        c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), D=rng.choice([
            _log_int(rng, 64, 1024), 64 * rng.randint(2, 16), 768]))
        c["V"] = rng.choice([30522, _log_int(rng, 1000, 100_000)])
        if op == "head":
            c["B"], c["L"] = _log_int(rng, 1, 500), _log_int(rng, 8, 512)
            c["bias_mean"] = rng.choice([-1.0, -3.0, -4.0])
            c["ragged"] = rng.random() < 0.7
            c["train"] = rng.random() < 0.5
        else:
            c["T"] = _log_int(rng, 1, 16384)
            c["bias"] = rng.random() < 0.5
            c["train"] = rng.random() < 0.7
            c["scale"] = 1024.0 if c["dtype"] == "fp16" and c["train"] else 1.0
            if op == "ce":
                c["frac"] = rng.choice([1.0, 0.6, 0.15])
            else:
                c["K"] = _log_int(rng, 1, 1000)
                c["tau"] = rng.choice([1.0, 2.0, 0.7])
        if op == "head":
            # the dense weights of a batch (and their gradient) are the largest tensors
            if c["B"] * c["V"] > 20_000_000 or (c["train"] and c["B"] * c["L"] > 16384):
                continue
        if work(c)["flops"] <= LARGEST_FLOPS:
            return c


def work(case):
    c = case
    V, D = c["V"], c["D"]
    if c["op"] == "head":
        T = c["B"] * c["L"] * (0.55 if c["ragged"] else 1.0)
        nbytes = 2 * T * D + 2 * V * D + 4 * V + 4 * c["B"] * V
        flops = 2 * T * V * D
        if c["train"]:       # dy in, three gradients out; two products per kept weight
            nbytes += 4 * c["B"] * V + 2 * c["B"] * c["L"] * D + 2 * V * D + 4 * V
            flops += 4 * c["B"] * V * D * 0.1
        return {"bytes": int(nbytes), "flops": int(flops)}
    T = max(1.0, c["T"] * c.get("frac", 1.0))
    nbytes = 2 * T * D + 2 * V * D + (4 * V if c["bias"] else 0) + 8 * c["T"] + 4
    if c["op"] == "distill":
        nbytes += 12 * c["T"] * c["K"]
    flops = 2 * T * V * D
    if c["train"]:
        nbytes += 2 * c["T"] * D + 2 * V * D + (4 * V if c["bias"] else 0)
        flops *= 3
    return {"bytes": int(nbytes), "flops": int(flops)}


# ---------------------------------------------------------------------------- inputs
def _grid(x, step, dtype):
    """Rounded to multiples of ``step``: sums of products of such values are exact in 32
    bits in any order, so that a maximum is won by the same token however it is summed."""
    return (torch.round(x / step) * step).to(dtype)


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    dt, V, D = DTYPES[c["dtype"]], c["V"], c["D"]
    st = {"case": c}
    if c["op"] == "head":
        B, Lq = c["B"], c["L"]
        st["hidden"] = _grid(normal(B, Lq, D).clamp_(-3.9, 3.9), 2.0 ** -5, dt)
        st["weight"] = _grid((normal(V, D) * (1.0 / math.sqrt(D))).clamp_(-0.24, 0.24), 2.0 ** -10, dt)
        st["bias"] = _grid(normal(V) * 0.5 + c["bias_mean"], 2.0 ** -10, torch.float32)
        lens = torch.full((B,), Lq, device=dev)
        if c["ragged"]:
            u = torch.exp(normal(B) * 0.45 - 0.7).clamp_(0.02, 1.0)
            lens = (u * Lq).round().long().clamp_(1, Lq)
            if B >= 7:
                lens[B // 2] = 0
        st["mask"] = torch.arange(Lq, device=dev)[None, :] < lens[:, None]
        if c["train"]:
            st["dy"] = normal(B, V) * 1e-2
    else:
        T = c["T"]
        st["hidden"] = normal(T, D).to(dt)
        st["weight"] = (normal(V, D) * (2.0 / math.sqrt(D))).to(dt)
        st["bias"] = normal(V) * 0.5 if c["bias"] else None
        if c["op"] == "ce":
            tgt = torch.randint(0, V, (T,), generator=g, device=dev)
            lab = torch.rand(T, generator=g, device=dev) < c["frac"]
            lab[0] = True
            st["targets"] = torch.where(lab, tgt, torch.full_like(tgt, IGNORE))
        else:
            K = min(c["K"], V)
            # K distinct ids per row: a random start and an odd stride around the vocabulary
            start = torch.randint(0, V, (T, 1), generator=g, device=dev)
            step = torch.randint(1, max(2, V // K), (T, 1), generator=g, device=dev)
            st["ids"] = (start + step * torch.arange(K, device=dev)[None, :]) % V
            st["scores"] = torch.sort(normal(T, K) * 2.0 + 6.0, dim=1, descending=True).values
        st["scale"] = torch.tensor(c["scale"], device=dev)
    if c["train"]:
        for k in ("hidden", "weight", "bias"):
            if st[k] is not None:
                st[k].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if own:
        return _run_own(c, state)
    with torch.no_grad():
        if c["op"] == "head":
            return _plain_head(c, state)
        return _plain_softmax(c, state)


def _run_own(c, st):
    gs = _gpusparse()
    h, w, b = st["hidden"], st["weight"], st["bias"]
    if c["op"] == "head":
        y = gs.sparse_head(h, w, bias=b, mask=st["mask"])
        if not c["train"]:
            return {"y": y}
        dh, dw, db = torch.autograd.grad(y, (h, w, b), st["dy"])
        return {"y": y.detach(), "dh": dh, "dw": dw, "db": db}
    if c["op"] == "ce":
        loss = gs.vocab_cross_entropy(h, w, st["targets"], bias=b, ignore_index=IGNORE)
    else:
        loss = gs.topk_distillation(h, w, st["scores"], st["ids"], bias=b, temperature=c["tau"])
    if not c["train"]:
        return {"loss": loss}
    leaves = [x for x in (h, w, b) if x is not None]
    grads = torch.autograd.grad(loss, leaves, st["scale"])
    out = {"loss": loss.detach(), "dh": grads[0], "dw": grads[1]}
    if b is not None:
        out["db"] = grads[2]
    return out


def _plain_head(c, st):
    h, w, b, mask = st["hidden"], st["weight"], st["bias"], st["mask"]
    B, V = h.shape[0], w.shape[0]
    wf = w.float()
    y = torch.zeros(B, V, device=h.device)
    if c["train"]:
        dh = torch.zeros(h.shape, device=h.device)
        dw = torch.zeros(w.shape, device=h.device)
        db = torch.zeros(V, device=h.device)
    per = max(1, PLAIN_ROWS // h.shape[1])
    for lo in range(0, B, per):
        hf = h[lo:lo + per].float()
        n, Lq, D = hf.shape
        s = torch.matmul(hf.reshape(n * Lq, D), wf.t()).reshape(n, Lq, V) + b
        s = s.masked_fill(~mask[lo:lo + per, :, None], float("-inf"))
        m, arg = s.max(dim=1)
        del s
        yc = torch.log1p(torch.relu(m))
        y[lo:lo + per] = yc
        if c["train"]:
            ds = torch.where(m > 0, st["dy"][lo:lo + per] * torch.exp(-yc), torch.zeros_like(yc))
            full = torch.zeros(n, Lq, V, device=h.device)
            full.scatter_(1, arg[:, None, :], ds[:, None, :])
            full = full.reshape(n * Lq, V)
            dh[lo:lo + per] = torch.matmul(full, wf).reshape(n, Lq, D)
            dw += torch.matmul(full.t(), hf.reshape(n * Lq, D))
            db += ds.sum(dim=0)
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dh": dh.to(h.dtype), "dw": dw.to(w.dtype), "db": db}


def _plain_softmax(c, st):
    h, w, b = st["hidden"], st["weight"], st["bias"]
    T, V = h.shape[0], w.shape[0]
    dev = h.device
    tau = c.get("tau", 1.0)
    if c["op"] == "ce":
        rows = torch.nonzero(st["targets"] != IGNORE).squeeze(1)
    else:
        rows = torch.arange(T, device=dev)
    n = max(int(rows.numel()), 1)
    wf = w.float()
    total = torch.zeros((), device=dev)
    if c["train"]:
        dh = torch.zeros(h.shape, device=dev)
        dw = torch.zeros(w.shape, device=dev)
        db = torch.zeros(V, device=dev)
        gain = st["scale"] / n
    for lo in range(0, rows.numel(), PLAIN_ROWS):
        r = rows[lo:lo + PLAIN_ROWS]
        hf = h[r].float()
        s = torch.matmul(hf, wf.t())
        if b is not None:
            s += b
        s /= tau
        m = s.max(dim=1, keepdim=True).values
        lse = torch.log(torch.exp(s - m).sum(dim=1, keepdim=True)) + m
        if c["op"] == "ce":
            ids = st["targets"][r][:, None]
            p = torch.ones(r.numel(), 1, device=dev)
            entropy = 0.0
        else:
            ids = st["ids"][r]
            t = st["scores"][r] / tau
            e = torch.exp(t - t.max(dim=1, keepdim=True).values)
            p = e / e.sum(dim=1, keepdim=True)
            entropy = (p * torch.log(p)).sum(dim=1)
        logq = torch.gather(s, 1, ids) - lse
        total += (tau * tau * (entropy - (p * logq).sum(dim=1))).sum()
        if c["train"]:
            d = torch.exp(s - lse)
            del s
            d.scatter_add_(1, ids, -p)
            d *= gain * tau
            dh[r] = torch.matmul(d, wf)
            dw += torch.matmul(d.t(), hf)
            db += d.sum(dim=0)
    out = {"loss": total / n}
    if c["train"]:
        out["dh"], out["dw"] = dh.to(h.dtype), dw.to(w.dtype)
        if b is not None:
            out["db"] = db
    return out


# ---------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    with torch.no_grad():
        st = prepare(case, seed)
        h = st["hidden"].detach().double()
        w = st["weight"].detach().double()
        b = st["bias"].detach().double() if st["bias"] is not None else None
        if case["op"] == "head":
            return _exact_head(case, st, h, w, b)
        return _exact_softmax(case, st, h, w, b)


def _exact_head(c, st, h, w, b):
    """Text by text, only its own tokens; the gradient by the winners' rows."""
    B, V = h.shape[0], w.shape[0]
    y = torch.zeros(B, V, dtype=torch.float64, device=h.device)
    dh, dw, db = torch.zeros_like(h), torch.zeros_like(w), torch.zeros_like(b)
    lens = st["mask"].sum(dim=1).tolist()
    for i in range(B):
        if lens[i] == 0:
            continue
        tok = h[i, :lens[i]]
        best, arg = torch.max(tok @ w.t() + b, dim=0)
        y[i] = torch.log(1.0 + best.clamp(min=0.0))
        if c["train"]:
            ds = torch.where(best > 0, st["dy"][i].double() / (1.0 + best.clamp(min=0.0)), 0.0)
            live = torch.nonzero(ds).squeeze(1)
            dh[i].index_add_(0, arg[live], ds[live, None] * w[live])
            dw[live] += ds[live, None] * tok[arg[live]]
            db += ds
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dh": dh, "dw": dw, "db": db}


def _exact_softmax(c, st, h, w, b):
    """Pieces of the rows, with the targets as a full distribution over the vocabulary."""
    T, V = h.shape[0], w.shape[0]
    tau = c.get("tau", 1.0)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    db = torch.zeros(V, dtype=torch.float64, device=h.device)
    loss = torch.zeros((), dtype=torch.float64, device=h.device)
    if c["op"] == "ce":
        lab = st["targets"] != IGNORE
        rows = torch.arange(T, device=h.device)[lab]
    else:
        rows = torch.arange(T, device=h.device)
    n = rows.numel()
    for r in torch.split(rows, 1024):
        z = h[r] @ w.t()
        if b is not None:
            z = z + b
        logq = torch.log_softmax(z / tau, dim=1)
        target = torch.zeros_like(z)
        if c["op"] == "ce":
            target[torch.arange(r.numel(), device=h.device), st["targets"][r]] = 1.0
        else:
            p = torch.softmax(st["scores"][r].double() / tau, dim=1)
            target.scatter_add_(1, st["ids"][r], p)
        loss += tau * tau * (torch.xlogy(target, target) - target * logq).sum()
        if c["train"]:
            d = (torch.exp(logq) - target) * (tau * float(c["scale"]) / n)
            dh[r] = d @ w
            dw += d.t() @ h[r]
            db += d.sum(dim=0)
    out = {"loss": loss / n}
    if c["train"]:
        out["dh"], out["dw"] = dh, dw
        if b is not None:
            out["db"] = db
    return out
