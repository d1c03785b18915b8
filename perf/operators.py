"""Cases, plain forms and exact values of the vocabulary-sized operators.

Three operators whose size is the vocabulary of a language model, at both ends
of a training step:

* ``nll``      linear head + log-softmax + negative log-likelihood that never
               keeps the logits, forward (scoring) and forward + backward
               (training): hidden rows H [R, d] bf16, head W [V, d] bf16,
               optional bias [V] fp32, target [R] int32 (outside [0, V): the row
               is ignored), optional weight per row, gradients bf16.
* ``distill``  the same head trained towards a teacher's K largest logits per
               row (ids int32, logits fp32; an id outside [0, V) is an absent
               entry) at a temperature T: T^2 KL(softmax(teacher / T) ||
               softmax(student / T)).
* ``embed``    token lookup with a scale (and a position table), and the
               table's gradient summed in token order.

``run`` computes the plain form in elementary torch operations where ``own``
is false and calls the package's operators where it is true.
"""
from __future__ import annotations

import math

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
_DT = {"bf16": BF16, "f32": F32}


# ------------------------------------------------------------------ cases
def _nll(name, R, V, d, train, bias=False, ignored=0.0, weighted=False):
    return {"name": name, "op": "nll", "R": R, "V": V, "d": d, "train": train, "bias": bias, "ignored": ignored,
            "weighted": weighted}


def _distill(name, R, V, d, K, T, train, bias=False, absent=0.0, empty=0.0):
    return {"name": name, "op": "distill", "R": R, "V": V, "d": d, "K": K, "T": T, "train": train, "bias": bias,
            "absent": absent, "empty": empty}


def _embed(name, n, V, d, table, out, train, pos=0, skew=1.0, invalid=0.0):
    return {"name": name, "op": "embed", "n": n, "V": V, "d": d, "table": table, "out": out, "train": train,
            "pos": pos, "skew": skew, "invalid": invalid}


def listed():
    return [
        # the likelihood of one next character under the repository's GPT configuration: latency
        _nll("score one, V=65", 1, 65, 384, False, bias=True),
        # scoring one prompt under a word-piece vocabulary: the head's weights are the traffic
        _nll("score 512, V=32768", 512, 32768, 1024, False),
        # the head of the repository's GPT training step (64 x 256 characters)
        _nll("train 16384, V=65", 16384, 65, 384, True, bias=True),
        # an ordinary language-model batch
        _nll("train 4096, V=32768", 4096, 32768, 1024, True),
        # packed ragged sequences: odd rows and vocabulary, padding rows ignored, rows weighted
        _nll("train 1537, V=50257", 1537, 50257, 768, True, bias=True, ignored=0.2, weighted=True),
        # a large training batch
        _nll("train 8192, V=65536", 8192, 65536, 2048, True),
        # distillation of an ordinary batch from the teacher's 64 stored logits
        _distill("distill 4096, K=64", 4096, 32768, 1024, 64, 2.0, True),
        # a short odd batch; rows with fewer than K stored logits, or none
        _distill("distill 333, K=17", 333, 50257, 512, 17, 1.0, True, bias=True, absent=0.2, empty=0.1),
        # the embedding of one decoded token
        _embed("embed one", 1, 32768, 1024, "bf16", "bf16", False),
        # the repository's GPT training step: every row of a small table is hit hundreds of times
        _embed("embed train 16384, V=65", 16384, 65, 384, "f32", "f32", True, pos=256),
        # word pieces with a long-tailed distribution; padding ids; bf16 activations, fp32 table and gradient
        _embed("embed train 16381, V=50257", 16381, 50257, 1024, "f32", "bf16", True, skew=1.0, invalid=0.1),
        # a large batch on a large bf16 table
        _embed("embed train 65536, V=131072", 65536, 131072, 2048, "bf16", "bf16", True, skew=1.0),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(("nll", "nll", "distill", "embed", "embed"))
    if op == "embed":
        n, V = _log_int(rng, 1, 65536), _log_int(rng, 65, 131072)
        d = 8 * _log_int(rng, 8, 256) if rng.random() < 0.7 else _log_int(rng, 33, 1000)
        c = _embed("", n, V, d, rng.choice(("bf16", "f32")), rng.choice(("bf16", "f32")), rng.random() < 0.7,
                   pos=rng.choice((0, 0, 1)), skew=rng.choice((0.0, 1.0, 1.5)), invalid=rng.choice((0.0, 0.1)))
        if c["pos"]:
            c["pos"] = max(1, n // rng.choice((1, 2, 5)))
            c["pos"] += c["pos"] == 3072
    else:
        while True:
            R, V, d = _log_int(rng, 1, 16384), _log_int(rng, 65, 65536), 8 * _log_int(rng, 8, 256)
            if R * V * d <= 8192 * 65536 * 2048:
                break
        bias = rng.random() < 0.4
        if op == "nll":
            c = _nll("", R, V, d, rng.random() < 0.7, bias, rng.choice((0.0, 0.3)), rng.random() < 0.3)
        else:
            R = max(1, R // 2)
            R += R == 3072
            c = _distill("", R, V, d, rng.choice((1, 3, 8, 20, 32, 64)), rng.choice((1.0, 2.0, 4.0)),
                         rng.random() < 0.8, bias, rng.choice((0.0, 0.2)), rng.choice((0.0, 0.1)))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _zipf(g, n, V, skew):
    """Token ids with P(rank r) ~ 1 / r^skew over a shuffled vocabulary."""
    if skew == 0.0:
        return torch.randint(0, V, (n,), device="cuda", generator=g)
    cdf = torch.cumsum(torch.arange(1, V + 1, device="cuda", dtype=F64) ** -skew, 0)
    ranks = torch.searchsorted(cdf, torch.rand(n, device="cuda", dtype=F64, generator=g) * cdf[-1])
    return torch.randperm(V, device="cuda", generator=g)[ranks.clamp_(max=V - 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    c, V, d = case, case["V"], case["d"]
    if c["op"] == "embed":
        n = c["n"]
        tok = _zipf(g, n, V, c["skew"])
        if c["invalid"]:
            tok = torch.where(rand(n) < c["invalid"], torch.full_like(tok, -1), tok)
        st = {"case": c, "tok": tok.to(torch.int32), "W": (randn(V, d) * 0.02).to(_DT[c["table"]]),
              "pos": randn(c["pos"], d) * 0.02 if c["pos"] else None, "scale": math.sqrt(d)}
        if c["train"]:
            st["dx"] = (randn(n, d) * 1e-3).to(_DT[c["out"]])
        return st
    R = c["R"]
    # logits of standard deviation 3; the target's raised by up to 12, so that
    # its probability runs from near 0 to near 1
    W = (randn(V, d) * (3.0 / math.sqrt(d))).to(BF16)
    lead = torch.randint(0, V, (R,), device="cuda", generator=g)
    H = (randn(R, d) + W[lead].float() * (rand(R, 1) * (12.0 / 9.0))).to(BF16)
    st = {"case": c, "H": H, "W": W, "bias": randn(V) * 0.1 if c["bias"] else None}
    if c["op"] == "nll":
        tgt = torch.where(rand(R) < c["ignored"], torch.full_like(lead, -1), lead)
        st["target"] = tgt.to(torch.int32)
        st["dloss"] = 0.5 + rand(R) if c["weighted"] else None
    else:
        K = min(c["K"], V)
        # the teacher prefers the raised id; the others are drawn without repetition
        key = rand(R, V)
        key[torch.arange(R, device="cuda"), lead] = 2.0
        idx = key.topk(K, dim=1).indices
        del key
        teacher = 8.0 - 8.0 * torch.sort(rand(R, K), dim=1).values
        gone = rand(R, K) < c["absent"]
        gone |= rand(R, 1) < c["empty"]
        st["idx"] = torch.where(gone, torch.full_like(idx, -1), idx).to(torch.int32)
        st["teacher"] = teacher
    st["scale"] = 1.0 / R
    return st


# ------------------------------------------------------------------ the two forms
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    import dreamcompiler_b200 as dgx
    c = st["case"]
    if c["op"] == "embed":
        x = dgx.embed_fwd(st["tok"], st["W"], scale=st["scale"], pos=st["pos"], out_dtype=_DT[c["out"]])
        if not c["train"]:
            return {"x": x}
        return {"x": x, "dW": dgx.embed_bwd(st["tok"], st["dx"], c["V"], scale=st["scale"],
                                            out_dtype=_DT[c["table"]])}
    H, W, b = st["H"], st["W"], st["bias"]
    if c["op"] == "nll":
        loss, lse = dgx.linear_nll_fwd(H, W, st["target"], bias=b)
        if not c["train"]:
            return {"loss": loss, "lse": lse}
        dH, dW, db = dgx.linear_nll_bwd(H, W, st["target"], lse, bias=b, dloss=st["dloss"], scale=st["scale"])
    else:
        loss, lse = dgx.linear_distill_fwd(H, W, st["idx"], st["teacher"], bias=b, temperature=c["T"])
        if not c["train"]:
            return {"loss": loss, "lse": lse}
        dH, dW, db = dgx.linear_distill_bwd(H, W, st["idx"], st["teacher"], lse, bias=b, temperature=c["T"],
                                            scale=st["scale"])
    return {"loss": loss, "lse": lse, "dH": dH, "dW": dW, "db": db}


def _run_plain(st):
    c = st["case"]
    if c["op"] == "embed":
        tok, W, n = st["tok"].long(), st["W"], c["n"]
        valid = (tok >= 0) & (tok < c["V"])
        at = torch.where(valid, tok, 0)
        x = torch.where(valid[:, None], W[at].float() * st["scale"], 0.0)
        if st["pos"] is not None:
            x = x + st["pos"][torch.arange(n, device="cuda") % c["pos"]]
        out = {"x": x.to(_DT[c["out"]])}
        if c["train"]:
            dx = torch.where(valid[:, None], st["dx"].float() * st["scale"], 0.0)
            out["dW"] = torch.zeros(c["V"], c["d"], device="cuda").index_add_(0, at, dx).to(_DT[c["table"]])
        return out
    H, W, R = st["H"].float(), st["W"].float(), c["R"]
    z = H @ W.t()
    if st["bias"] is not None:
        z = z + st["bias"]
    if c["op"] == "nll":
        tgt = st["target"].long()
        valid = (tgt >= 0) & (tgt < c["V"])
        idx, q = torch.where(valid, tgt, 0)[:, None], valid[:, None].float()
        coef = st["scale"] if st["dloss"] is None else st["dloss"][:, None] * st["scale"]
        T = 1.0
    else:
        T = c["T"]
        z = z / T
        idx, q = _soft_target(st["idx"].long(), st["teacher"], c["V"], T)
        coef = st["scale"] * T
    m = z.max(1, keepdim=True).values
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    logp = torch.gather(z, 1, idx) - lse
    entropy = torch.where(q > 0, q * torch.log(torch.where(q > 0, q, 1.0)), 0.0)
    loss = (T * T) * (entropy - torch.where(q > 0, q * logp, 0.0)).sum(1)
    out = {"loss": loss, "lse": lse[:, 0]}
    if c["train"]:
        g = torch.exp(z - lse) * (q.sum(1, keepdim=True) > 0).float()
        g.scatter_add_(1, idx, -q)
        g = g * coef
        out["dH"], out["dW"] = (g @ W).to(BF16), (g.t() @ H).to(BF16)
        out["db"] = g.sum(0) if st["bias"] is not None else None
    return out


def _soft_target(idx, teacher, V, T):
    """Ids (0 for absent entries) and probabilities (0 for them) of the teacher's softmax over its entries."""
    valid = (idx >= 0) & (idx < V)
    t = torch.where(valid, teacher / T, float("-inf"))
    t = t - torch.where(valid.any(1, keepdim=True), t.max(1, keepdim=True).values, 0.0)
    e = torch.exp(t)
    return torch.where(valid, idx, 0), e / torch.clamp(e.sum(1, keepdim=True), min=1e-30)


# ------------------------------------------------------------------ work and exact values
def work(case):
    c, V, d = case, case["V"], case["d"]
    if c["op"] == "embed":
        n, tb, ob = c["n"], 2 if c["table"] == "bf16" else 4, 2 if c["out"] == "bf16" else 4
        rows = min(n, V)  # table rows that a lookup can touch at most
        b = 4 * n + rows * d * tb + n * d * ob + c["pos"] * d * 4
        f = n * d
        if c["train"]:
            b += n * d * ob + V * d * tb
            f += 2 * n * d
        return {"bytes": b, "flops": f}
    R, k = c["R"], 3 if c["train"] else 1
    b = (R + V) * d * 2 * (2 if c["train"] else 1) + 4 * R * 3 + (4 * V * (2 if c["train"] else 1) if c["bias"] else 0)
    if c["op"] == "distill":
        b += 8 * R * c["K"]
    return {"bytes": b, "flops": 2.0 * k * R * V * d}


def exact(case, seed):
    """The outputs in 64 bits, row block by row block."""
    st = prepare(case, seed)
    c, V, d = case, case["V"], case["d"]
    if c["op"] == "embed":
        ok = (st["tok"] >= 0) & (st["tok"] < V)
        rows, ids = ok.nonzero()[:, 0], st["tok"][ok].long()
        x = torch.zeros(c["n"], d, dtype=F64, device="cuda")
        x[rows] = st["W"].to(F64)[ids] * st["scale"]
        if c["pos"]:
            x += st["pos"].to(F64).repeat((c["n"] + c["pos"] - 1) // c["pos"], 1)[:c["n"]]
        out = {"x": x}
        if c["train"]:
            out["dW"] = torch.zeros(V, d, dtype=F64, device="cuda").index_add_(0, ids, st["dx"].to(F64)[rows])
            out["dW"] *= st["scale"]
        return out
    R, W = c["R"], st["W"].to(F64)
    T = c.get("T", 1.0)
    got = {"loss": torch.zeros(R, dtype=F64, device="cuda"), "lse": torch.zeros(R, dtype=F64, device="cuda")}
    if c["train"]:
        got.update(dH=torch.zeros(R, d, dtype=F64, device="cuda"), dW=torch.zeros(V, d, dtype=F64, device="cuda"),
                   db=torch.zeros(V, dtype=F64, device="cuda") if c["bias"] else None)
    for r0 in range(0, R, 2048):
        s = slice(r0, min(R, r0 + 2048))
        h = st["H"][s].to(F64)
        logits = h @ W.T
        if c["bias"]:
            logits += st["bias"].to(F64)
        logits /= T
        lp = torch.log_softmax(logits, 1)
        got["lse"][s] = torch.logsumexp(logits, 1)
        want = torch.zeros_like(lp)
        if c["op"] == "nll":
            live = (st["target"][s] >= 0) & (st["target"][s] < V)
            want[live.nonzero()[:, 0], st["target"][s][live].long()] = 1.0
            weight = torch.full((h.shape[0],), st["scale"], dtype=F64, device="cuda")
            if st["dloss"] is not None:
                weight *= st["dloss"][s].to(F64)
        else:
            ids, there = st["idx"][s].long(), (st["idx"][s] >= 0) & (st["idx"][s] < V)
            t = st["teacher"][s].to(F64) / T
            prob = torch.where(there, t, -torch.inf).softmax(1)
            prob = torch.where(there, prob, 0.0)
            live = there.any(1)
            want.scatter_add_(1, torch.where(there, ids, 0), prob)
            weight = torch.full((h.shape[0],), st["scale"] * T, dtype=F64, device="cuda")
        got["loss"][s] = T * T * (torch.special.xlogy(want, want) - want * lp).sum(1)
        if c["train"]:
            grad = (lp.exp() * live[:, None] - want) * weight[:, None]
            got["dH"][s] = grad @ W
            got["dW"] += grad.T @ h
            if c["bias"]:
                got["db"] += grad.sum(0)
    return got
