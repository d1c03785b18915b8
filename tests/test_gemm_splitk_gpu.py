"""GPU: split-K products whose K blocks do not divide evenly over the slices.

129 K blocks over 16 slices of 9 would leave the sixteenth without a block;
its partial tile would be whatever the accumulator held before.
"""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("M,N,K", [(33, 256, 8209), (65, 40, 8256), (128, 128, 9100), (200, 64, 17 * 64 * 8 + 1)])
def test_uneven_slices(dgx, M, N, K):
    g = torch.Generator(device="cuda").manual_seed(K)
    ld = (K + 7) // 8 * 8
    A = torch.randn(M, ld, device="cuda", generator=g).bfloat16()[:, :K]
    B = torch.randn(K, N, device="cuda", generator=g).bfloat16()
    # the accumulator's earlier contents: a product of large values on the same SMs
    big = torch.full((2048, 1024), 100.0, device="cuda").bfloat16()
    dgx.gemm(big, big, transB=True)
    got = dgx.gemm(A, B).double()
    a, b = A.double(), B.double()
    # exact products; a chain of K/16 tensor-core steps, then up to 16 slices
    tol = 2.0 ** -23 * (K / 16 + 32) * (a.abs() @ b.abs())
    assert ((got - a @ b).abs() <= tol).all()
