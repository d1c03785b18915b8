"""GPU: the vocabulary head (dgx_linear_nll_*, dgx_linear_distill_*) against the
formulas in 64 bits.

Every bound is elementwise and follows from the arithmetic the operator
promises (u = 2^-23, one unit of fp32 rounding or truncation):
  logits   products of bf16 are exact in fp32; a sum of d terms is a chain of
           d/16 tensor-core steps of 16 terms: error at most
           e_z = u (d/16 + 16) max_rj sum_i |h_ri w_ji| (+ the bias add)
  softmax  p = exp(z - lse): relative error e_p = 2 e_z / T + 2u(|z - lse| + 4)
  G        rounded to bf16: 2^-8 |G| + w p e_p
  dH, dW   sum of |dG| |W| (or |H|), fp32 accumulation u (n/16 + 16) sum |G||W|,
           2^-8 |result| when written as bf16
  db       unrounded G, a chain of R fp32 additions
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -23
F64 = torch.float64


class Problem:
    """Inputs, results in 64 bits and their bounds."""

    def __init__(self, R, V, d, *, K=None, T=1.0, bias=None, seed=0, ignored=0.0, weighted=False, pad=0, zstd=3.0,
                 scale=1.0, absent=0.0, dup=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
        randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.R, self.V, self.d, self.K, self.T, self.scale = R, V, d, K, T, scale
        dp = (d + 7) // 8 * 8 + pad
        # pitched buffers whose padding must not be read into the result
        self.Hb = torch.full((R, dp), float("nan"), device="cuda", dtype=torch.bfloat16)
        self.Wb = torch.full((V, dp), float("nan"), device="cuda", dtype=torch.bfloat16)
        self.H, self.W = self.Hb[:, :d], self.Wb[:, :d]
        self.W.copy_(randn(V, d) * (zstd / d ** 0.5))
        lead = torch.randint(0, V, (R,), device="cuda", generator=g)
        self.H.copy_(randn(R, d) + self.W[lead].float() * rand(R, 1) * (10.0 / zstd ** 2))
        self.bias = None
        if bias is not None:
            self.bias = randn(V)
            if bias == "masked" and V > 4:  # some columns masked (never the leading ids)
                off = rand(V) < 0.3
                off[V // 3:V // 3 + 70] = True
                off[lead] = False
                self.bias[off] = float("-inf")
                low = rand(V) < 0.2
                low[V // 2:V // 2 + 70] = True
                low[lead] = False
                self.bias[low] = torch.finfo(torch.float32).min
        self.dloss = rand(R) + 0.5 if weighted else None
        if K is None:
            t = torch.where(rand(R) < ignored, torch.full_like(lead, -1), lead)
            if ignored and R > 2:
                t[1] = V  # the first id past the vocabulary
            self.target = t.to(torch.int32)
        else:
            K = self.K = min(K, V)
            key = rand(R, V)
            key[torch.arange(R, device="cuda"), lead] = 2.0
            idx = key.topk(K, dim=1).indices
            if dup and K > 2:
                idx[:, 1] = idx[:, 0]
            gone = (rand(R, K) < absent) | (rand(R, 1) < absent / 2)
            self.idx = torch.where(gone, torch.full_like(idx, -1), idx).to(torch.int32)
            self.teacher = 6.0 - 7.0 * rand(R, K)
        self._truth()

    def _truth(self):
        H, W, T = self.H.to(F64), self.W.to(F64), self.T
        raw = H @ W.T
        mag = (H.abs() @ W.abs().T).max() if self.R else torch.zeros((), dtype=F64, device="cuda")
        bmag = 0.0
        if self.bias is not None:
            b = self.bias.to(F64)
            raw = raw + b
            ok = b.abs() < 1e30
            bmag = float(b[ok].abs().max()) if ok.any() else 0.0
        e_z = U * ((self.d / 16 + 16) * float(mag) + bmag)
        z = raw / T
        lse = torch.logsumexp(z, 1)
        lp = z - lse[:, None]
        p = lp.exp()
        q = torch.zeros_like(z)
        rows = torch.arange(self.R, device="cuda")
        if self.K is None:
            live = (self.target >= 0) & (self.target < self.V)
            q[rows[live], self.target[live].long()] = 1.0
        else:
            there = (self.idx >= 0) & (self.idx < self.V)
            live = there.any(1)
            t = torch.where(there, self.teacher.to(F64) / T, -torch.inf)
            prob = torch.where(live[:, None], t.softmax(1), 0.0)
            prob = torch.where(there, prob, 0.0)
            q.scatter_add_(1, torch.where(there, self.idx.long(), 0), prob)
        self.live = live
        terms = torch.where(q > 0, q * lp, 0.0)
        ent = torch.special.xlogy(q, q)
        if self.K is not None:  # entropy term per entry, as repeated ids add their probabilities
            ent = torch.special.xlogy(prob, prob).sum(1)
        else:
            ent = ent.sum(1)
        self.lse, self.loss = lse, T * T * (ent - terms.sum(1))
        x = torch.where(torch.isfinite(lp), lp.abs(), 0.0)
        e_p = 2 * e_z / T + 2 * U * (x + 4)
        biggest = torch.where(torch.isfinite(z) & (z.abs() < 1e30), z.abs(), 0.0).amax(1) if self.R else z.sum(1)
        self.tol_lse = e_z / T + 4 * U * (biggest + 16)
        self.tol_loss = T * T * (2 * e_z / T + 8 * U * (biggest + 16 + ent.abs())) + 4 * U * self.loss.abs()
        w = live.to(F64) * self.scale * T
        if self.dloss is not None:
            w = w * self.dloss.to(F64)
        G = (p - q) * w[:, None]
        eG = 2.0 ** -8 * G.abs() + (p * e_p + q * 16 * U) * w.abs()[:, None]
        eG = torch.where(G == 0, (p * e_p + q * 16 * U) * w.abs()[:, None], eG)
        self.dH, self.dW, self.db = G @ W, G.T @ H, G.sum(0)
        aW, aH, aG = W.abs(), H.abs(), G.abs()
        self.tol_dH = eG @ aW + U * (self.V / 16 + 16) * (aG @ aW)
        self.tol_dW = eG.T @ aH + U * (self.R / 16 + 16) * (aG.T @ aH)
        exact_e = (p * e_p + q * 16 * U) * w.abs()[:, None]
        self.tol_db = exact_e.sum(0) + U * (self.R + 8) * aG.sum(0)

    def fwd(self, dgx, **kw):
        if self.K is None:
            return dgx.linear_nll_fwd(self.H, self.W, self.target, bias=self.bias, **kw)
        return dgx.linear_distill_fwd(self.H, self.W, self.idx, self.teacher, bias=self.bias, temperature=self.T, **kw)

    def bwd(self, dgx, lse, **kw):
        kw.setdefault("dloss", self.dloss)
        kw.setdefault("scale", self.scale)
        if self.K is None:
            return dgx.linear_nll_bwd(self.H, self.W, self.target, lse, bias=self.bias, **kw)
        return dgx.linear_distill_bwd(self.H, self.W, self.idx, self.teacher, lse, bias=self.bias, temperature=self.T,
                                      **kw)

    def check_fwd(self, loss, lse):
        within(lse, self.lse, self.tol_lse, "lse")
        within(loss, self.loss, self.tol_loss, "loss")
        assert not loss[~self.live].any()

    def check_bwd(self, dH, dW, db):
        if dH is not None:
            within(dH, self.dH, self.tol_dH + out_round(dH, self.dH), "dH")
            assert not dH[~self.live].any()
        if dW is not None:
            within(dW, self.dW, self.tol_dW + out_round(dW, self.dW), "dW")
        if db is not None:
            within(db, self.db, self.tol_db, "db")


def out_round(t, ref):
    return ref.abs() * (2.0 ** -8 if t.dtype == torch.bfloat16 else U)


def within(got, want, tol, what):
    got = got.to(F64)
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - tol
    if over.numel():
        i = int(over.argmax())
        assert over.max() <= 1e-30, f"{what}[{i}]: {got.flatten()[i]} vs {want.flatten()[i]}, bound {tol.flatten()[i]}"


SIZES = [(1, 1, 8), (1, 2, 8), (2, 65, 384), (3, 31, 20), (64, 257, 64), (129, 300, 72), (257, 1025, 136),
         (1000, 65, 384), (255, 513, 1000), (33, 8209, 256), (700, 2049, 40)]


@pytest.mark.parametrize("R,V,d", SIZES)
@pytest.mark.parametrize("bias,ignored,weighted", [(None, 0.0, False), ("plain", 0.4, True), ("masked", 0.2, False)])
def test_nll_forward_backward(dgx, R, V, d, bias, ignored, weighted):
    p = Problem(R, V, d, bias=bias, ignored=ignored, weighted=weighted, pad=8 * (R % 3), seed=R + V + d, scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))
    dgx.sync_check()


@pytest.mark.parametrize("R,V,d", SIZES)
@pytest.mark.parametrize("K,T,bias,absent,dup", [(1, 1.0, None, 0.0, False), (5, 2.0, "plain", 0.4, True),
                                                 (64, 4.0, "masked", 0.1, False), (256, 1.0, None, 0.2, True)])
def test_distill_forward_backward(dgx, R, V, d, K, T, bias, absent, dup):
    if bias == "masked":  # a masked column may not carry probability: its log is -inf
        bias = "plain"
    p = Problem(R, V, d, K=K, T=T, bias=bias, absent=absent, dup=dup, seed=R + V + d + K, scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))
    dgx.sync_check()


@pytest.mark.parametrize("R,V,d", [(2048, 50257, 64), (16384, 65, 384), (1, 131072, 64), (9000, 33000, 32)])
def test_nll_many_columns_or_rows(dgx, R, V, d):
    """Problems of several pieces of the vocabulary, and of many row tiles."""
    p = Problem(R, V, d, bias="plain", ignored=0.1, seed=1, scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))


@pytest.mark.parametrize("K", [None, 7])
def test_fp32_gradients_accumulate_and_skip(dgx, K):
    p = Problem(300, 777, 96, K=K, T=1.0 if K is None else 2.0, bias="plain", ignored=0.1, absent=0.1, seed=5,
                scale=1 / 300)
    loss, lse = p.fwd(dgx)
    dH = torch.full((300, 104), float("nan"), device="cuda")[:, :96]
    base = torch.randn(777, 96, device="cuda")
    dW, db0 = base.clone(), torch.randn(777, device="cuda")
    db = db0.clone()
    p.bwd(dgx, lse, dH=dH, dW=dW, db=db, accumulate=True)
    within(dH, p.dH, p.tol_dH + out_round(dH, p.dH), "dH")
    within(dW, p.dW + base.to(F64), p.tol_dW + U * (base.abs() + p.dW.abs()), "dW")
    within(db, p.db + db0.to(F64), p.tol_db + U * (db0.abs() + p.db.abs()), "db")
    # each gradient alone has the same bits as with the others
    full = p.bwd(dgx, lse)
    for i, name in enumerate(("dH", "dW", "db")):
        one = p.bwd(dgx, lse, need=(name,))
        assert [t is not None for t in one] == [j == i for j in range(3)]
        assert torch.equal(one[i], full[i])
    assert dH._base[:, 96:].isnan().all()


@pytest.mark.parametrize("R,V,d", [(300, 777, 96), (40, 20000, 64), (9000, 33000, 32)])
def test_losses_sum_into_one_gradient(dgx, R, V, d):
    """Hard and soft target on the same rows, the second call adding to the
    first one's dH, dW and db (direct, sliced and pieced sums)."""
    p = Problem(R, V, d, bias="plain", seed=21, scale=0.25 / R)
    q = Problem(R, V, d, K=5, T=2.0, bias="plain", seed=21, scale=0.75 / R)
    assert torch.equal(p.H, q.H) and torch.equal(p.W, q.W) and torch.equal(p.bias, q.bias)
    out = dict(dH=torch.empty(R, d, device="cuda"), dW=torch.empty(V, d, device="cuda"),
               db=torch.empty(V, device="cuda"))
    p.bwd(dgx, p.fwd(dgx)[1], **out)
    q.bwd(dgx, q.fwd(dgx)[1], accumulate=True, accumulate_dH=True, **out)
    for name, a, b, ta, tb in (("dH", p.dH, q.dH, p.tol_dH, q.tol_dH), ("dW", p.dW, q.dW, p.tol_dW, q.tol_dW),
                               ("db", p.db, q.db, p.tol_db, q.tol_db)):
        within(out[name], a + b, ta + tb + U * 4 * (a.abs() + b.abs()), name)


def test_all_rows_without_target(dgx):
    p = Problem(200, 500, 64, bias="plain", seed=2)
    p.target.fill_(-1)
    p._truth()
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    dH, dW, db = p.bwd(dgx, lse)
    assert not loss.any() and not dH.any() and not dW.any() and not db.any()
    p = Problem(200, 500, 64, K=9, seed=2)
    p.teacher.fill_(float("-inf"))
    loss, lse = p.fwd(dgx)
    dH, dW, _ = p.bwd(dgx, lse)
    assert not loss.any() and not dH.any() and not dW.any()


def test_no_rows(dgx):
    H = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    W = torch.randn(100, 64, device="cuda").bfloat16()
    t = torch.empty(0, device="cuda", dtype=torch.int32)
    mean = torch.ones(1, device="cuda")
    b = torch.zeros(100, device="cuda")
    loss, lse = dgx.linear_nll_fwd(H, W, t, bias=b, mean=mean)
    assert loss.shape == lse.shape == (0,) and mean.item() == 0
    dH, dW, db = dgx.linear_nll_bwd(H, W, t, lse, bias=b)
    assert dH.shape == (0, 64) and not dW.any() and not db.any()


def test_teacher_mask_values(dgx):
    """Teacher logits of -inf or the lowest float carry no probability."""
    p = Problem(100, 400, 64, K=12, T=2.0, seed=3)
    p.teacher[:, 3] = float("-inf")
    p.teacher[:, 5] = torch.finfo(torch.float32).min
    p._truth()
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))


@pytest.mark.parametrize("K", [1, 12, 200])
def test_nan_teacher_rows_are_not_empty_rows(dgx, K):
    """A NaN teacher logit gives its row a NaN loss and gradient, whether it is the row's only entry, one of several
    or beside entries of -inf; the other rows keep their bits. A NaN at an absent entry does not count."""
    p = Problem(70, 300, 64, K=K, seed=30)
    loss0, lse0 = p.fwd(dgx)
    dH0, _, _ = p.bwd(dgx, lse0)
    hit = [5, 33, 66]
    p.teacher[5] = float("nan")
    p.teacher[33, -1] = float("nan")
    p.teacher[66] = float("-inf")
    p.teacher[66, 0] = float("nan")
    p.idx[40, 0] = -1
    loss1 = p.fwd(dgx)[0]
    p.teacher[40, 0] = float("nan")
    loss, lse = p.fwd(dgx)
    dH, dW, _ = p.bwd(dgx, lse)
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[hit] = False
    assert torch.equal(loss[keep], loss1[keep]) and torch.isfinite(loss[keep]).all()
    keep[40] = False
    assert torch.equal(loss[keep], loss0[keep]) and torch.equal(lse, lse0) and torch.equal(dH[keep], dH0[keep])
    assert loss[hit].isnan().all() and dH[hit].isnan().all()
    named = torch.zeros(300, dtype=torch.bool, device="cuda")
    named[p.idx[hit].long()] = True
    assert dW[named].isnan().all() and torch.isfinite(dW[~named]).all()


def test_non_finite_rows_stay_in_their_rows(dgx):
    """A NaN hidden row gives a NaN loss and dH in that row alone; a row without
    a target keeps loss 0 and dH 0 whatever it holds."""
    p = Problem(300, 600, 64, ignored=0.3, seed=4)
    dead = int((~p.live).nonzero()[0])
    alive = int(p.live.nonzero()[5])
    ref_loss, ref_lse = p.fwd(dgx)
    ref_dH, _, _ = p.bwd(dgx, ref_lse)
    p.H[dead] = float("nan")
    p.H[alive, 3] = float("inf")
    loss, lse = p.fwd(dgx)
    dH, _, _ = p.bwd(dgx, lse)
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[dead, alive]] = False
    assert torch.equal(loss[keep], ref_loss[keep]) and torch.equal(dH[keep], ref_dH[keep])
    assert loss[dead] == 0 and not dH[dead].any()
    assert not torch.isfinite(loss[alive])


@pytest.mark.parametrize("R,V,d", [(17, 1, 8), (300, 256, 1000), (700, 129, 64), (60000, 65, 24), (513, 250, 770)])
@pytest.mark.parametrize("bias", [None, "masked"])
def test_nll_vocabulary_of_one_tile(dgx, R, V, d, bias):
    """Up to 256 columns: loss and lse leave the logits kernel itself (60000 rows: several tiles per SM pair)."""
    p = Problem(R, V, d, bias=bias, ignored=0.2, weighted=True, seed=R + V, scale=1.0 / R)
    mean = torch.full((1,), float("nan"), device="cuda")
    loss, lse = p.fwd(dgx, mean=mean)
    p.check_fwd(loss, lse)
    within(mean, p.loss.mean()[None], p.tol_loss.mean()[None] + 2 ** -18 * p.loss.abs().mean(), "mean")
    p.check_bwd(*p.bwd(dgx, lse))
    dgx.sync_check()


@pytest.mark.parametrize("R,V,d,bias", [(1, 65, 64, False), (12, 1000, 64, True), (40, 65, 64, True),
                                        (300, 1000, 1024, False)])
def test_small_losses_keep_their_relative_precision(dgx, R, V, d, bias):
    """A target far above every other column: the loss is log(1 + a small sum), which log of the whole sum would
    round to multiples of 2^-23. All logits are exact (multiples of 1/8), so what is left is the exponentials:
    arguments up to 30 log2(e) < 44 rounded twice (44 * 2^-23), the exponential (2^-21), at most 64 additions in a
    row (64 * 2^-24), log1p and expf (a few 2^-23): below 1.2e-5 of the loss."""
    H = torch.zeros(R, d, device="cuda", dtype=torch.bfloat16)
    H[:, 0] = 1
    W = torch.zeros(V, d, device="cuda", dtype=torch.bfloat16)
    W[:, 0] = -(torch.arange(V, device="cuda") % 9) / 8
    target = (torch.arange(R, device="cuda", dtype=torch.int32) * 7) % V
    rows = torch.arange(R, device="cuda")
    H[rows, 1 + rows] = 1  # column 1 + r lifts row r's target only
    W[target.long(), 1 + rows] = (12 + rows % 8 * 2).to(W.dtype)
    b = None
    if bias:
        b = torch.arange(V, device="cuda", dtype=torch.float32) % 3 / 4
    z = H.to(F64) @ W.to(F64).T + (0 if b is None else b.to(F64))
    zt = z.gather(1, target.long()[:, None])
    others = torch.exp(z - zt).scatter(1, target.long()[:, None], 0.0).sum(1)
    want = torch.log1p(others)
    loss, lse = dgx.linear_nll_fwd(H, W, target, bias=b)[:2]
    assert float(want.max()) < 0.05
    within(loss, want, 1.2e-5 * want, "loss")
    within(lse, zt[:, 0] + want, 2 ** -22 * (zt[:, 0].abs() + want + 1), "lse")


@pytest.mark.parametrize("R", [3, 200])
def test_rows_masked_in_every_column(dgx, R):
    """No distribution: lse is -inf and the loss NaN where a target is asked for, as inf - inf; a masked target
    alone has loss inf; the rows beside them are not touched."""
    H = torch.ones(R, 64, device="cuda", dtype=torch.bfloat16)
    W = torch.ones(10, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.full((R,), 4, device="cuda", dtype=torch.int32)
    t[1] = -1
    b = torch.full((10,), float("-inf"), device="cuda")
    loss, lse = dgx.linear_nll_fwd(H, W, t, bias=b)[:2]
    assert torch.isneginf(lse).all() and loss[1] == 0 and torch.isnan(loss[0]) and torch.isnan(loss[2:]).all()
    b[:3] = 0
    loss, lse = dgx.linear_nll_fwd(H, W, t, bias=b)[:2]
    assert torch.isfinite(lse).all() and loss[1] == 0 and torch.isposinf(loss[0]) and torch.isposinf(loss[2:]).all()


def test_large_logits(dgx):
    """Logits of several thousand: the softmax neither overflows nor loses the
    loss of the leading id."""
    p = Problem(130, 300, 64, zstd=300.0, seed=8)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))


@pytest.mark.parametrize("K", [None, 16])
def test_same_bits_with_any_workspace_and_stream(dgx, K):
    p = Problem(520, 3001, 128, K=K, bias="plain", ignored=0.1, absent=0.1, seed=6, scale=1 / 520)
    loss, lse = p.fwd(dgx)
    ref = p.bwd(dgx, lse)
    if K is None:
        sizes = [dgx.linear_nll_workspace_size(520, 3001, 128, b) for b in (False, True)]
    else:
        sizes = [dgx.linear_distill_workspace_size(520, 3001, 128, K, b) for b in (False, True)]
    ws = [torch.full((n,), 0xFF, device="cuda", dtype=torch.uint8) for n in sizes]  # NaN in every type
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mean = torch.full((1,), float("nan"), device="cuda")
    with torch.cuda.stream(side):
        loss2, lse2 = p.fwd(dgx, workspace=ws[0], mean=mean)
        got = p.bwd(dgx, lse2, workspace=ws[1])
    side.synchronize()
    assert torch.equal(loss, loss2) and torch.equal(lse, lse2)
    for a, b in zip(ref, got):
        assert torch.equal(a, b)
    assert abs(mean.item() - loss.double().mean().item()) <= 520 * U * loss.double().abs().mean().item()


@pytest.mark.parametrize("K", [None, 4])
def test_gradients_against_differences(dgx, K):
    """Central differences of the operator's own loss. H and W lie on a grid of
    2^-4 below 4, so +-2^-6 steps are exact in bf16; the step is taken along
    one random sign direction of H, of W and of the bias."""
    R, V, d = 40, 90, 32
    p = Problem(R, V, d, K=K, T=1.0 if K is None else 2.0, bias="plain", seed=12)
    p.H.copy_((torch.randn(R, d, device="cuda") * 16).round().clamp(-32, 32) / 16)
    p.W.copy_((torch.randn(V, d, device="cuda") * 4).round().clamp(-32, 32) / 16)
    p._truth()
    lse = p.fwd(dgx)[1]
    dH = torch.empty(R, d, device="cuda")
    dW = torch.empty(V, d, device="cuda")
    _, _, db = p.bwd(dgx, lse, dH=dH, dW=dW)
    h = 2.0 ** -6
    # The formula's own central difference in 64 bits at the same points takes
    # the truncation out: what is left is the loss's error over the step and
    # the gradient's bound.
    exact = {"H": p.dH, "W": p.dW, "b": p.db}
    bound = {"H": p.tol_dH + out_round(dH, p.dH), "W": p.tol_dW + out_round(dW, p.dW), "b": p.tol_db}
    for name, t, grad in (("H", p.H, dH), ("W", p.W, dW), ("b", p.bias, db)):
        for k in range(6):
            r = (k * 7) % t.shape[0]
            sign = torch.where(torch.rand(t[r].shape, device="cuda") < 0.5, -1.0, 1.0)
            keep = t[r].clone()
            ends, ends64, tol = [], [], 0.0
            for step in (h, -h):
                t[r] = (keep.float() + step * sign).to(t.dtype)
                ends.append(p.fwd(dgx)[0].to(F64).sum())
                p._truth()
                ends64.append(p.loss.sum())
                tol += float(p.tol_loss.sum())
            t[r] = keep
            slope = float((ends[0] - ends[1]) / (2 * h))
            slope64 = float((ends64[0] - ends64[1]) / (2 * h))
            along = lambda x: float((x[r].to(F64) * sign.to(F64)).sum())  # noqa: E731
            assert abs(slope - slope64) <= tol / (2 * h)
            assert abs(along(grad) - along(exact[name])) <= float(bound[name][r].sum())
            # and the two slopes are the same thing: the step's truncation is small beside them
            assert abs(slope64 - along(exact[name])) <= 0.05 * max(abs(slope64), float(exact[name][r].abs().sum()))
            assert abs(slope - along(grad)) <= tol / (2 * h) + float(bound[name][r].sum()) + abs(
                slope64 - along(exact[name]))


def test_refusals(dgx):
    from dreamcompiler_b200 import DgxError
    H = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    W = torch.zeros(100, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(8, device="cuda", dtype=torch.int32)
    lse = torch.zeros(8, device="cuda")
    with pytest.raises(DgxError, match="pitch"):
        dgx.linear_nll_fwd(torch.zeros(8, 61, device="cuda", dtype=torch.bfloat16), W[:, :61], t)
    with pytest.raises(DgxError, match="aligned"):
        dgx.linear_nll_fwd(torch.zeros(8, 72, device="cuda", dtype=torch.bfloat16)[:, 1:65], W, t)
    with pytest.raises(DgxError, match="pitch"):
        dgx.linear_nll_fwd(H[:1].expand(8, 64), W, t)
    with pytest.raises(DgxError, match="workspace"):
        dgx.linear_nll_fwd(H, W, t, workspace=torch.empty(16, device="cuda", dtype=torch.uint8))
    with pytest.raises(DgxError, match="workspace"):
        dgx.linear_nll_bwd(H, W, t, lse, workspace=torch.empty(16, device="cuda", dtype=torch.uint8))
    with pytest.raises(DgxError, match="fp32 dW"):
        dgx.linear_nll_bwd(H, W, t, lse, dW=torch.zeros_like(W), accumulate=True)
    idx, tea = torch.zeros(8, 300, device="cuda", dtype=torch.int32), torch.zeros(8, 300, device="cuda")
    with pytest.raises(DgxError, match="K=300"):
        dgx.linear_distill_fwd(H, W, idx, tea)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(DgxError, match="temperature"):
            dgx.linear_distill_fwd(H, W, idx[:, :4].contiguous(), tea[:, :4].contiguous(), temperature=bad)
    for wrong in (lambda: dgx.linear_nll_fwd(H.float(), W, t), lambda: dgx.linear_nll_fwd(H, W.float(), t),
                  lambda: dgx.linear_nll_fwd(H, W, t.long()), lambda: dgx.linear_nll_fwd(H, W[:, :32], t),
                  lambda: dgx.linear_nll_fwd(H, W, t[:4]), lambda: dgx.linear_nll_fwd(H, W, t, bias=lse),
                  lambda: dgx.linear_nll_bwd(H, W, t, lse, accumulate=True),
                  lambda: dgx.linear_distill_fwd(H, W, idx[:, :4].contiguous(), tea[:, :5].contiguous())):
        with pytest.raises(AssertionError):
            wrong()
    dgx.sync_check()


def test_mean_must_be_one_float_on_the_device(dgx):
    H = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    W = torch.zeros(100, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(8, device="cuda", dtype=torch.int32)
    for bad in (torch.zeros(1), torch.zeros(1, device="cuda", dtype=torch.bfloat16), torch.zeros(0, device="cuda"),
                torch.zeros(2, device="cuda")):
        with pytest.raises(AssertionError, match="mean"):
            dgx.linear_nll_fwd(H, W, t, mean=bad)
        with pytest.raises(AssertionError, match="mean"):
            dgx.linear_distill_fwd(H, W, t[:, None], torch.zeros(8, 1, device="cuda"), mean=bad)


def test_row_arguments_hold_one_element_per_row(dgx):
    """Tensors whose first extent alone is the number of rows would be read as their leading elements."""
    H = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    W = torch.zeros(100, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.zeros(8, device="cuda", dtype=torch.int32)
    row, rows = torch.zeros(8, device="cuda"), torch.zeros(8, 3, device="cuda")
    i3 = torch.zeros(8, 3, device="cuda", dtype=torch.int32)
    for wrong in (lambda: dgx.linear_nll_fwd(H, W, i3), lambda: dgx.linear_nll_bwd(H, W, i3, row),
                  lambda: dgx.linear_nll_fwd(H, W, t, loss=rows), lambda: dgx.linear_nll_fwd(H, W, t, lse=rows),
                  lambda: dgx.linear_nll_bwd(H, W, t, rows), lambda: dgx.linear_nll_bwd(H, W, t, row, dloss=rows),
                  lambda: dgx.linear_distill_fwd(H, W, i3, rows, lse=rows),
                  lambda: dgx.linear_distill_bwd(H, W, i3, rows, rows),
                  lambda: dgx.linear_distill_bwd(H, W, i3, rows, row, dloss=rows),
                  lambda: dgx.linear_distill_fwd(H, W, i3, rows.double()),
                  lambda: dgx.linear_distill_fwd(H, W, i3, torch.zeros(3, 8, device="cuda").T),
                  lambda: dgx.linear_distill_fwd(H, W, torch.zeros(7, 3, device="cuda", dtype=torch.int32), rows[:7])):
        with pytest.raises(AssertionError):
            wrong()
    dgx.linear_distill_bwd(H, W, i3, rows, dgx.linear_distill_fwd(H, W, i3, rows)[1], dloss=row)
    dgx.sync_check()


def test_workspace_must_be_on_the_device(dgx):
    H = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    t, row = torch.zeros(8, device="cuda", dtype=torch.int32), torch.zeros(8, device="cuda")
    i1, q1 = t[:, None], row[:, None]
    for bad in (torch.empty(1 << 20), torch.empty(1, device="cuda").expand(1 << 20)):
        for call in (lambda: dgx.linear_nll_fwd(H, H, t, workspace=bad),
                     lambda: dgx.linear_nll_bwd(H, H, t, row, workspace=bad),
                     lambda: dgx.linear_distill_fwd(H, H, i1, q1, workspace=bad),
                     lambda: dgx.linear_distill_bwd(H, H, i1, q1, row, workspace=bad)):
            with pytest.raises(AssertionError, match="workspace"):
                call()


def rows_of(p, K, r0, r1):
    """The rows [r0, r1) of a problem that was made without its 64-bit results, with them."""
    b = Problem.__new__(Problem)
    b.__dict__.update(p, R=r1 - r0, K=K, dloss=None, H=p["H"][r0:r1])
    if K is None:
        b.target = p["target"][r0:r1]
    else:
        b.idx, b.teacher = p["idx"][r0:r1], p["teacher"][r0:r1]
    b._truth()
    return b


@pytest.mark.parametrize("R,V,K", [(9000, 262144, None), (9000, 262144, 5), (1100, 2000003, 3), (70000, 31000, None)])
def test_more_logits_than_one_forward_piece(dgx, R, V, K):
    """Above 2^31 logits the forward joins the statistics of several pieces of the vocabulary, and the target lists'
    start table is made anew for each (in the backward for each group of pieces)."""
    g = torch.Generator(device="cuda").manual_seed(R)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    d, T = 16, 1.0 if K is None else 2.0
    W = torch.randn(V, d, device="cuda", generator=g) * 0.75
    lead = torch.randint(0, V, (R,), device="cuda", generator=g)
    H = (torch.randn(R, d, device="cuda", generator=g) + W[lead] * rand(R, 1)).bfloat16()
    bias = torch.randn(V, device="cuda", generator=g)
    p = dict(V=V, d=d, T=T, scale=1.0 / R, H=H, W=W.bfloat16(), bias=bias)
    if K is None:
        p["target"] = torch.where(rand(R) < 0.1, torch.full_like(lead, -1), lead).to(torch.int32)
        call, args = (dgx.linear_nll_fwd, dgx.linear_nll_bwd), (p["target"],)
        kw = dict(bias=bias)
    else:
        p["idx"] = torch.randint(-V // 20, V, (R, K), device="cuda", generator=g).to(torch.int32)
        p["idx"][:, 0] = lead
        p["teacher"] = 6.0 - 7.0 * rand(R, K)
        call, args = (dgx.linear_distill_fwd, dgx.linear_distill_bwd), (p["idx"], p["teacher"])
        kw = dict(bias=bias, temperature=T)
    loss, lse = call[0](H, p["W"], *args, **kw)
    dH, dW = torch.empty(R, d, device="cuda"), torch.empty(V, d, device="cuda")
    _, _, db = call[1](H, p["W"], *args, lse, scale=1.0 / R, dH=dH, dW=dW, **kw)
    dgx.sync_check()
    total = {k: 0.0 for k in ("dW", "tol_dW", "db", "tol_db")}
    step = max(1, (1 << 28) // V)
    blocks = (R + step - 1) // step
    for r0 in range(0, R, step):
        b = rows_of(p, K, r0, min(R, r0 + step))
        b.check_fwd(loss[r0:r0 + step], lse[r0:r0 + step])
        b.check_bwd(dH[r0:r0 + step], None, None)
        for k in total:
            total[k] = total[k] + getattr(b, k)
    # a block's bound counts the additions of its own rows: all R of them are at most `blocks` times as many
    within(dW, total["dW"], blocks * total["tol_dW"], "dW")
    within(db, total["db"], blocks * total["tol_db"], "db")


def masked_distillation(R, V, d, K, T, seed, masked_entries):
    """Columns of -inf and of the lowest float; the teacher's entries there are absent, or present with a logit of -inf."""
    p = Problem(R, V, d, K=K, T=T, bias="masked", absent=0.1, seed=seed, scale=1.0 / R, weighted=True)
    off = (p.idx >= 0) & (p.bias[p.idx.clamp(min=0).long()] < -1e30)
    if masked_entries == "absent":
        p.idx[off] = -1
    else:
        p.teacher[off] = float("-inf")
        p.teacher[(p.idx >= 0).any(1) & ~((p.idx >= 0) & ~off).any(1)] = 0.0  # no row of -inf entries alone ...
        p.idx[off & (p.teacher > -1e30)] = -1  # ... whose masked ids leave instead
    p._truth()
    return p


@pytest.mark.parametrize("R,V,d", [(2, 65, 384), (64, 257, 64), (129, 300, 72), (33, 8209, 256), (700, 2049, 40),
                                   (1000, 65, 384)])
@pytest.mark.parametrize("K,T", [(1, 1.0), (20, 0.25), (64, 4.0), (256, 2.0)])
@pytest.mark.parametrize("masked_entries", ["absent", "-inf"])
def test_distill_with_masked_columns(dgx, R, V, d, K, T, masked_entries):
    """Masked columns have probability 0 whatever 1 / T makes of their logits; rows weighted."""
    p = masked_distillation(R, V, d, K, T, R + V + K, masked_entries)
    off = p.bias < -1e30
    assert off.any() or R > 8 * V  # so many rows that every column leads one, and none may be masked
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    dH, dW, db = p.bwd(dgx, lse)
    p.check_bwd(dH, dW, db)
    assert not dW[off].any() and not db[off].any()


@pytest.mark.parametrize("T", [0.125, 0.5, 30.0])
@pytest.mark.parametrize("R,V,d,K", [(5, 300, 64, 8), (300, 1000, 136, 33)])
def test_distill_temperatures_and_row_weights(dgx, R, V, d, K, T):
    p = Problem(R, V, d, K=K, T=T, bias="plain", absent=0.2, weighted=True, seed=R + K, scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))


@pytest.mark.parametrize("R,V,d,bias", [(9, 65, 384, None), (16, 65, 384, "masked"), (10, 5003, 1000, "plain"),
                                        (13, 300, 20, "masked"), (16, 20011, 1024, None), (17, 5003, 1000, "plain"),
                                        (8, 5003, 1000, "plain"), (15, 2049, 3000, "plain"), (16, 777, 3080, None)])
def test_few_rows_of_ordinary_values(dgx, R, V, d, bias):
    """Both row groups of the thin kernel (up to 16 rows, while their fragments fit shared memory) and what follows it."""
    p = Problem(R, V, d, bias=bias, ignored=0.2, seed=R + V, scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))


@pytest.mark.parametrize("K", [None, 40])
@pytest.mark.parametrize("R,V,d", [(100, 500, 2048), (520, 1300, 2000), (7, 300, 4104)])
def test_long_contractions(dgx, R, V, d, K):
    p = Problem(R, V, d, K=K, T=1.0 if K is None else 2.0, bias="plain", ignored=0.1, absent=0.1, weighted=True, seed=d,
                scale=1.0 / R)
    loss, lse = p.fwd(dgx)
    p.check_fwd(loss, lse)
    p.check_bwd(*p.bwd(dgx, lse))
