"""GPU: dgx_embed_fwd / dgx_embed_bwd against the formulas in 64 bits.

Bounds: forward one product and one sum in fp32, then one rounding to the
output type; backward a sum of L rows (|error| <= u L sum |dx|, u = 2^-24 per
addition), one product, one rounding.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F64 = torch.float64
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def rnd(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else U


def tokens(n, V, kind, g):
    if kind == "one":
        t = torch.full((n,), V // 2, device="cuda")
    elif kind == "hot":  # half the tokens are one id, the rest spread
        t = torch.randint(0, V, (n,), device="cuda", generator=g)
        t = torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, torch.full_like(t, V - 1), t)
    else:
        t = torch.randint(0, V, (n,), device="cuda", generator=g)
    if kind == "invalid":
        r = torch.rand(n, device="cuda", generator=g)
        t = torch.where(r < 0.2, torch.full_like(t, -1), torch.where(r < 0.4, torch.full_like(t, V), t))
    if kind == "none":
        t = torch.full_like(t, -7)
    return t.to(torch.int32)


@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 1000, 1024), (7, 13, 5), (300, 65, 384), (257, 5000, 33),
                                   (1000, 77, 130), (64, 300, 2050)])
@pytest.mark.parametrize("w,x", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("S", [0, 1, 37])
def test_forward(dgx, n, V, d, w, x, S):
    g = torch.Generator(device="cuda").manual_seed(n + V + d)
    W = torch.randn(V, d, device="cuda", generator=g).to(DT[w])
    P = torch.randn(S, d, device="cuda", generator=g) if S else None
    tok = tokens(n, V, "invalid", g)
    scale = 1.7
    got = dgx.embed_fwd(tok, W, scale=scale, pos=P, out_dtype=DT[x])
    ok = (tok >= 0) & (tok < V)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    ref = torch.where(ok[:, None], W.to(F64)[torch.where(ok, tok, 0).long()] * s32, 0.0)
    mag = ref.abs()
    if S:
        p = P.to(F64)[torch.arange(n, device="cuda") % S]
        ref, mag = ref + p, mag + p.abs()
    assert got.dtype == DT[x]
    assert ((got.to(F64) - ref).abs() <= 2 * U * mag + rnd(got.dtype) * ref.abs() * (1 + 2.0 ** -8) + 1e-45).all()


@pytest.mark.parametrize("n,V,d", [(1, 1, 1), (1, 1000, 1024), (7, 13, 5), (300, 65, 384), (257, 5000, 33),
                                   (128, 500, 264), (129, 500, 264), (5000, 77, 130), (64, 300, 2050), (20000, 700, 256), (33, 140000, 64), (100, 70000, 136),
                                   (70000, 3, 40)])
@pytest.mark.parametrize("kind", ["spread", "one", "hot", "invalid", "none"])
@pytest.mark.parametrize("gx,w", [("f32", "f32"), ("f32", "bf16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_backward(dgx, n, V, d, kind, gx, w):
    g = torch.Generator(device="cuda").manual_seed(n + V + d)
    tok = tokens(n, V, kind, g)
    dx = torch.randn(n, d, device="cuda", generator=g).to(DT[gx])
    scale = 0.3
    out = torch.full((V, d), float("nan"), device="cuda", dtype=DT[w])
    got = dgx.embed_bwd(tok, dx, V, scale=scale, out=out)
    ref, mag, cnt = truth(tok, dx, V, scale)
    tol = U * (cnt[:, None] + 2) * mag + rnd(got.dtype) * ref.abs() * (1 + 2.0 ** -8)
    assert ((got.to(F64) - ref).abs() <= tol + 1e-45).all()
    assert not got[cnt == 0].any()
    assert torch.equal(got, dgx.embed_bwd(tok, dx, V, scale=scale, out_dtype=DT[w]))


@pytest.mark.parametrize("before", [0, 1, 127, 128, 33 * 128 + 5])
@pytest.mark.parametrize("span", [1, 128, 129, 31 * 128, 32 * 128 + 1, 33 * 128, 33 * 128 + 1, 65 * 128 - 1])
@pytest.mark.parametrize("after", [0, 40 * 128 + 3])
def test_backward_of_a_token_over_many_blocks(dgx, before, span, after):
    """One id whose sorted run starts and ends at, before and after the edges of the summing blocks."""
    g = torch.Generator(device="cuda").manual_seed(before + span + after)
    n, V, d = before + span + after, 3, 16
    tok = torch.tensor([0] * before + [1] * span + [2] * after, dtype=torch.int32, device="cuda")
    tok = tok[torch.randperm(n, device="cuda", generator=g)].contiguous()
    dx = torch.randn(n, d, device="cuda", generator=g)
    got = dgx.embed_bwd(tok, dx, V)
    ref, mag, cnt = truth(tok, dx, V, 1.0)
    tol = U * (cnt[:, None] + 2) * mag + U * ref.abs()
    assert ((got.to(F64) - ref).abs() <= tol).all()


def truth(tok, dx, V, scale):
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    ok = (tok >= 0) & (tok < V)
    ids = tok[ok].long()
    rows = dx.to(F64)[ok]
    z = torch.zeros(V, dx.shape[1], dtype=F64, device="cuda")
    cnt = torch.zeros(V, dtype=F64, device="cuda").index_add_(0, ids, torch.ones_like(ids, dtype=F64))
    return z.index_add(0, ids, rows) * s32, z.index_add(0, ids, rows.abs()) * s32, cnt


def test_backward_accumulates(dgx):
    g = torch.Generator(device="cuda").manual_seed(1)
    n, V, d = 900, 400, 96
    tok = tokens(n, V // 2, "hot", g)
    dx = torch.randn(n, d, device="cuda", generator=g)
    base = torch.randn(V, d, device="cuda", generator=g)
    base[V - 1] = float("nan")  # a row whose token does not occur is left alone
    got = dgx.embed_bwd(tok, dx, V, scale=2.0, out=base.clone(), accumulate=True)
    ref, mag, cnt = truth(tok, dx, V, 2.0)
    hit = cnt > 0
    assert got[V - 1].isnan().all() and torch.equal(got[~hit][:-1], base[~hit][:-1])
    tol = U * (cnt[:, None] + 4) * (mag + base.abs().to(F64))
    assert ((got.to(F64) - ref - base.to(F64)).abs() <= tol)[hit].all()


def test_pitched_rows_and_unaligned_bases(dgx):
    g = torch.Generator(device="cuda").manual_seed(2)
    n, V, d = 333, 90, 64
    tok = tokens(n, V, "hot", g)
    for dt in (torch.float32, torch.bfloat16):
        Wb = torch.randn(V, d + 9, device="cuda", generator=g).to(dt)
        db = torch.randn(n, d + 3, device="cuda", generator=g).to(dt)
        xb = torch.full((n, d + 5), float("nan"), device="cuda", dtype=dt)
        ob = torch.full((V, d + 7), float("nan"), device="cuda", dtype=torch.float32)
        W, dx, x, o = Wb[:, 3:3 + d], db[:, 1:1 + d], xb[:, 2:2 + d], ob[:, 5:5 + d]
        dgx.embed_fwd(tok, W, scale=1.0, out=x)
        dgx.embed_bwd(tok, dx, V, out=o)
        assert torch.equal(x, dgx.embed_fwd(tok, W.contiguous(), scale=1.0))
        assert torch.equal(o, dgx.embed_bwd(tok, dx.contiguous(), V))
        assert xb[:, :2].isnan().all() and xb[:, 2 + d:].isnan().all()
        assert ob[:, :5].isnan().all() and ob[:, 5 + d:].isnan().all()


def test_backward_workspace_stream_and_no_tokens(dgx):
    g = torch.Generator(device="cuda").manual_seed(3)
    n, V, d = 5000, 300, 128
    tok = tokens(n, V, "hot", g)
    dx = torch.randn(n, d, device="cuda", generator=g)
    ref = dgx.embed_bwd(tok, dx, V)
    ws = torch.full((max(1, dgx.embed_bwd_workspace_size(n, d, V)),), 0xFF, device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dgx.embed_bwd(tok, dx, V, workspace=ws)
    side.synchronize()
    assert torch.equal(ref, got)
    none = dgx.embed_bwd(tok[:0], dx[:0], V)
    assert none.shape == (V, d) and not none.any()
    keep = torch.ones(V, d, device="cuda")
    dgx.embed_bwd(tok[:0], dx[:0], V, out=keep, accumulate=True)
    assert (keep == 1).all()
    assert dgx.embed_fwd(tok[:0], ref).shape == (0, d)


def test_backward_non_finite_rows_stay_in_their_token(dgx):
    tok = torch.tensor([3, 5, 3, -1, 9], device="cuda", dtype=torch.int32)
    dx = torch.ones(5, 40, device="cuda")
    dx[1] = float("inf")
    dx[3] = float("nan")  # a position without a token
    got = dgx.embed_bwd(tok, dx, 12)
    assert (got[3] == 2).all() and got[5].isinf().all() and (got[9] == 1).all()
    got[[3, 5, 9]] = 0
    assert not got.any()


def test_gradient_against_differences(dgx):
    """The lookup is linear: <embed(W + D) - embed(W), G> = <D, embed_bwd(G)>.
    Inputs on a grid of 2^-6 make the products exact; the sums are taken in
    64 bits, the operator's own rounding being one fp32 step per term."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n, V, d = 500, 60, 48
    grid = lambda *s: (torch.randn(*s, device="cuda", generator=g) * 64).round() / 64  # noqa: E731
    W, D, G = grid(V, d), grid(V, d), grid(n, d)
    tok = tokens(n, V, "invalid", g)
    diff = dgx.embed_fwd(tok, W + D, scale=0.5).to(F64) - dgx.embed_fwd(tok, W, scale=0.5).to(F64)
    lhs = (diff * G.to(F64)).sum()
    rhs = (D.to(F64) * dgx.embed_bwd(tok, G, V, scale=0.5).to(F64)).sum()
    assert abs(float(lhs - rhs)) <= 1e-12 * float((diff * G.to(F64)).abs().sum())


def test_refusals(dgx):
    from dreamcompiler_b200 import DgxError
    tok = torch.zeros(4, device="cuda", dtype=torch.int32)
    W = torch.zeros(10, 16, device="cuda")
    dx = torch.zeros(4, 16, device="cuda")
    with pytest.raises(DgxError, match="fp32 dW"):
        dgx.embed_bwd(tok, dx, 10, out=W.bfloat16(), accumulate=True)
    with pytest.raises(DgxError, match="pitch"):
        dgx.embed_bwd(tok, dx[:1].expand(4, 16), 10)
    for wrong in (lambda: dgx.embed_fwd(tok.long(), W), lambda: dgx.embed_fwd(tok, W.half()),
                  lambda: dgx.embed_fwd(tok, W, pos=torch.zeros(3, 8, device="cuda")),
                  lambda: dgx.embed_bwd(tok[:2], dx, 10), lambda: dgx.embed_bwd(tok, dx, 10, accumulate=True),
                  lambda: dgx.embed_bwd(tok, dx, 10, out=torch.zeros(9, 16, device="cuda"))):
        with pytest.raises(AssertionError):
            wrong()


def test_workspace_must_be_on_the_device(dgx):
    tok = torch.zeros(4, device="cuda", dtype=torch.int32)
    dx = torch.zeros(4, 16, device="cuda")
    for bad in (torch.empty(1 << 20), torch.empty(1, device="cuda").expand(1 << 20)):
        with pytest.raises(AssertionError, match="workspace"):
            dgx.embed_bwd(tok, dx, 10, workspace=bad)


@pytest.mark.parametrize("n,V,d", [(100, 262144, 40), (129, 262144, 24), (5000, 262144, 24), (70000, 262144, 17),
                                   (3000, (1 << 27) + 5, 2)])
@pytest.mark.parametrize("kind", ["spread", "hot", "invalid"])
def test_backward_of_a_large_vocabulary(dgx, n, V, d, kind):
    """Three and four passes of the sort (keys of 19 and 28 bits): the order ends in the other buffer, or in one that was
    read before."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    tok = tokens(n, V, kind, g)
    tok[::7] = torch.randint(0, 50, (tok[::7].numel(),), device="cuda", generator=g).to(torch.int32) * (V // 50)
    dx = torch.randn(n, d, device="cuda", generator=g)
    out = torch.full((V, d), float("nan"), device="cuda")
    got = dgx.embed_bwd(tok, dx, V, scale=0.3, out=out)
    ref, mag, cnt = truth(tok, dx, V, 0.3)
    tol = U * (cnt[:, None] + 2) * mag + U * ref.abs()
    assert ((got.to(F64) - ref).abs() <= tol + 1e-45).all()
    assert not got[cnt == 0].any()


@pytest.mark.parametrize("n", [1, 100, 128, 129, 4097])
@pytest.mark.parametrize("V,d", [(70, 40), (500, 264), (300, 33)])
@pytest.mark.parametrize("pad,off", [(0, 0), (3, 1), (8, 8)])
@pytest.mark.parametrize("gx", ["f32", "bf16"])
def test_backward_accumulates_into_pitched_rows(dgx, n, V, d, pad, off, gx):
    """With and without the sort: rows that occur are added to, the others and the padding are left alone; the same
    places without accumulate."""
    g = torch.Generator(device="cuda").manual_seed(n + V + d)
    tok = tokens(n, V, "hot", g)
    dx = torch.randn(n, d + pad + off, device="cuda", generator=g).to(DT[gx])[:, off:off + d]
    ref, mag, cnt = truth(tok, dx, V, 2.0)
    hit = cnt > 0
    tol = U * (cnt[:, None] + 4) * mag
    for accumulate in (True, False):
        base = torch.randn(V, d + pad + off, device="cuda", generator=g)
        base[~hit] = float("nan")
        buf = base.clone()
        got = dgx.embed_bwd(tok, dx, V, scale=2.0, out=buf[:, off:off + d], accumulate=accumulate)
        was = base[:, off:off + d].to(F64) if accumulate else torch.zeros(V, d, dtype=F64, device="cuda")
        assert ((got.to(F64) - ref - was).abs() <= tol + U * 4 * was.abs())[hit].all()
        assert got[~hit].isnan().all() if accumulate else not got[~hit].any()
        keep = torch.ones(V, d + pad + off, dtype=torch.bool, device="cuda")
        keep[:, off:off + d] = False
        assert torch.equal(buf[keep].nan_to_num(7.0), base[keep].nan_to_num(7.0))
