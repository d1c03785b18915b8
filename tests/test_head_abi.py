"""CPU: argument checks of the vocabulary head and the scaled embedding, made
before any device work."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from dreamcompiler_b200 import _lib
    return _lib.load()


FAKE = C.c_void_p(256)


def nll_fwd(lib, H=FAKE, ldh=64, W=FAKE, ldw=64, target=FAKE, R=4, V=10, d=64, loss=FAKE, lse=FAKE, ws=FAKE,
            wsb=1 << 40):
    return lib.dgx_linear_nll_fwd(H, ldh, W, ldw, None, target, R, V, d, loss, lse, None, ws, wsb, None)


def nll_bwd(lib, lse=FAKE, R=4, V=10, d=64, dH=FAKE, dht=1, lddh=64, dW=FAKE, dwt=1, lddw=64, acc=0, ws=FAKE,
            wsb=1 << 40, target=FAKE):
    return lib.dgx_linear_nll_bwd(FAKE, 64, FAKE, 64, None, target, lse, None, 1.0, R, V, d, dH, dht, lddh, dW, dwt,
                                  lddw, None, acc, ws, wsb, None)


def test_head_forward_refusals(lib):
    from dreamcompiler_b200 import _lib as L
    for kw in (dict(R=-1), dict(V=0), dict(d=0), dict(ldh=60), dict(ldw=56), dict(ldh=68), dict(H=None),
               dict(W=None), dict(H=C.c_void_p(264)), dict(target=None), dict(loss=None), dict(lse=None),
               dict(ws=C.c_void_p(272))):
        assert nll_fwd(lib, **kw) == L.DGX_EINVAL, kw
    assert nll_fwd(lib, wsb=8) == L.DGX_ENOMEM
    assert b"workspace" in lib.dgx_last_error()
    assert nll_fwd(lib, R=0, H=None, target=None, loss=None, lse=None) == L.DGX_OK


def test_head_backward_refusals(lib):
    from dreamcompiler_b200 import _lib as L
    for kw in (dict(R=-1), dict(lse=None), dict(target=None), dict(dht=2), dict(dwt=3), dict(lddh=56),
               dict(lddh=66), dict(lddw=62), dict(dH=C.c_void_p(8)), dict(dW=C.c_void_p(8)), dict(ws=C.c_void_p(8))):
        assert nll_bwd(lib, **kw) == L.DGX_EINVAL, kw
    assert nll_bwd(lib, acc=1) == L.DGX_EUNSUPPORTED and nll_bwd(lib, acc=2) == L.DGX_EUNSUPPORTED
    assert nll_bwd(lib, acc=4) == L.DGX_EINVAL
    assert nll_bwd(lib, wsb=8) == L.DGX_ENOMEM
    assert nll_bwd(lib, dH=None, dW=None) == L.DGX_OK  # nothing asked for


def test_head_dimension_limit(lib):
    from dreamcompiler_b200 import _lib as L
    top = 1 << 23
    for kw in (dict(R=top + 1), dict(V=top + 1), dict(d=top + 8, ldh=top + 8, ldw=top + 8)):
        assert nll_fwd(lib, **kw) == L.DGX_EINVAL, kw
        assert b"above" in lib.dgx_last_error()
    assert lib.dgx_linear_nll_workspace_size(4, 10, top + 1, 0) == 0
    assert lib.dgx_linear_distill_workspace_size(4, 10, 64, 4, 1) > 0


def test_distill_refusals(lib):
    from dreamcompiler_b200 import _lib as L

    def fwd(idx=FAKE, teacher=FAKE, K=4, T=1.0):
        return lib.dgx_linear_distill_fwd(FAKE, 64, FAKE, 64, None, idx, teacher, K, T, 4, 10, 64, FAKE, FAKE, None, FAKE,
                                          1 << 40, None)

    def bwd(teacher=FAKE, K=4, T=1.0, lse=FAKE):
        return lib.dgx_linear_distill_bwd(FAKE, 64, FAKE, 64, None, FAKE, teacher, K, T, lse, None, 1.0, 4, 10, 64, FAKE, 1,
                                          64, FAKE, 1, 64, None, 0, FAKE, 1 << 40, None)

    for f in (fwd, bwd):
        for kw in (dict(K=0), dict(K=257), dict(T=0.0), dict(T=-2.0), dict(T=float("nan")), dict(T=float("inf")),
                   dict(T=1e-45), dict(T=4e-39), dict(T=2e19), dict(teacher=None)):
            assert f(**kw) == L.DGX_EINVAL, kw
    assert fwd(idx=None) == L.DGX_EINVAL and bwd(lse=None) == L.DGX_EINVAL


def test_embed_refusals(lib):
    from dreamcompiler_b200 import _lib as L

    def fwd(tok=FAKE, W=FAKE, wt=0, ldw=16, P=None, S=0, x=FAKE, xt=0, ldx=16, n=4, d=16, V=10):
        return lib.dgx_embed_fwd(tok, W, wt, ldw, P, S, 1.0, x, xt, ldx, n, d, V, None)

    def bwd(tok=FAKE, dx=FAKE, gt=0, lddx=16, dW=FAKE, wt=0, lddw=16, n=4, d=16, V=10, acc=0):
        return lib.dgx_embed_bwd(tok, dx, gt, lddx, 1.0, dW, wt, lddw, n, d, V, acc, None, 0, None)

    for kw in (dict(n=-1), dict(d=0), dict(V=0), dict(wt=2), dict(xt=3), dict(ldw=15), dict(ldx=8), dict(tok=None),
               dict(W=None), dict(x=None), dict(P=FAKE, S=0)):
        assert fwd(**kw) == L.DGX_EINVAL, kw
    for kw in (dict(n=-1), dict(d=0), dict(V=0), dict(gt=2), dict(wt=3), dict(lddx=15), dict(lddw=8), dict(tok=None),
               dict(dx=None), dict(dW=None)):
        assert bwd(**kw) == L.DGX_EINVAL, kw
    assert bwd(wt=1, acc=1) == L.DGX_EUNSUPPORTED
    assert fwd(n=0, tok=None, x=None) == L.DGX_OK


def test_embed_token_limit(lib):
    """Positions are counted in 32 bits and stepped past the last one: a count that would wrap is refused before
    anything runs (the last accepted one gets as far as the workspace check)."""
    from dreamcompiler_b200 import _lib as L
    top = (1 << 31) - (1 << 16)

    def bwd(n):
        return lib.dgx_embed_bwd(FAKE, FAKE, 0, 16, 1.0, FAKE, 0, 16, n, 16, 10, 0, FAKE, 16, None)

    assert bwd(top) == L.DGX_ENOMEM
    for n in (top + 1, (1 << 31) - 511, (1 << 31) - 1):
        assert bwd(n) == L.DGX_EINVAL, n
        assert b"above" in lib.dgx_last_error()
        assert lib.dgx_embed_bwd_workspace_size(n, 16, 10) == 0


def test_workspace_sizes(lib):
    assert lib.dgx_linear_nll_workspace_size(0, 10, 8, 0) == 0
    assert lib.dgx_linear_distill_workspace_size(4, 10, 8, 300, 1) == 0
    for b in (0, 1):
        small = lib.dgx_linear_nll_workspace_size(64, 1000, 64, b)
        large = lib.dgx_linear_nll_workspace_size(8192, 131072, 64, b)
        assert 0 < small <= large
        # never the logits: 8192 x 131072 fp32 would be 4 GiB, bf16 2 GiB
        assert large < 2 << 30
        assert lib.dgx_linear_distill_workspace_size(64, 1000, 64, 8, b) >= small


@pytest.mark.parametrize("R,V,d", [(65536, 262144, 4096), (65536, 262144, 256), (16384, 1 << 23, 64), (1 << 23, 65, 64),
                                   (3, 1 << 23, 2048), (300000, 100000, 1024)])
def test_forward_workspace_does_not_grow_with_the_logits(lib, R, V, d):
    """Statistics of 2^31 logits at a time (8 bytes for 64 or, from d = 769 on, 128 of them) and a start table of 2 bytes
    for 64; beside that only K ids, probabilities and logits per row."""
    for K in (1, 20):
        rows = R * (12 * K + 16) + 4096
        stats = (8 << 31) // (128 if d > 768 else 64)
        assert lib.dgx_linear_nll_workspace_size(R, V, d, 0) <= stats + rows
        assert lib.dgx_linear_distill_workspace_size(R, V, d, K, 0) <= stats + (2 << 31) // 64 + rows
        extra = (lib.dgx_linear_distill_workspace_size(R, V, d, K, 1) - lib.dgx_linear_nll_workspace_size(R, V, d, 1))
        assert 0 <= extra <= (2 << 31) // 64 + rows


def test_faults_can_be_injected(lib):
    from dreamcompiler_b200 import _lib as L
    try:
        for call in (lambda: nll_fwd(lib), lambda: nll_bwd(lib),
                     lambda: lib.dgx_embed_fwd(FAKE, FAKE, 0, 16, None, 0, 1.0, FAKE, 0, 16, 4, 16, 10, None),
                     lambda: lib.dgx_embed_bwd(FAKE, FAKE, 0, 16, 1.0, FAKE, 0, 16, 4, 16, 10, 0, None, 0, None)):
            assert lib.dgx_fault_inject(1, L.DGX_ECUDA) == L.DGX_OK
            assert call() == L.DGX_ECUDA
            assert b"injected fault" in lib.dgx_last_error()
    finally:
        lib.dgx_fault_inject(0, 0)


def test_workspace_tensors_are_whole_and_on_the_device():
    """A host tensor, or an expanded one whose bytes are not there, would be written by the kernels."""
    import torch
    from dreamcompiler_b200.ops import _ws
    assert _ws(None, 0) == (None, 0)
    host = torch.empty(64, dtype=torch.uint8)
    assert _ws(host, host.get_device()) == (host.data_ptr(), 64)
    with pytest.raises(AssertionError, match="workspace"):
        _ws(host, 0)
    with pytest.raises(AssertionError, match="workspace"):
        _ws(torch.empty(1).expand(1 << 20), -1)
