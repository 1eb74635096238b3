"""GPU: what the 8-bit linear layer refuses and promises beyond its results (those: test_gpu_linear_fp8.py)."""
import pytest
import torch

from cnmnet_amd import _lib, ops
from oracle import block_fp8 as bf

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_packed_weight_knows_its_columns():
    """A weight of 2100 columns is packed as 2176, as one of 2057 is: the other's input is refused all the same."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(40, 2100, generator=g).to(DEV)
    q, s = ops.pack_linear_fp8(w)
    for M in (1, 30, 200):
        with pytest.raises(_lib.EngineError, match="2100"):
            ops.linear_fp8(torch.randn(M, 2057, device=DEV), q, s)
        assert ops.linear_fp8(torch.randn(M, 2100, device=DEV), q, s).shape == (M, 40)
    a, sa = ops.quantize_fp8(torch.randn(70, 2057, device=DEV))
    with pytest.raises(_lib.EngineError, match="2057"):
        ops.matmul_fp8(a, sa, q, s)
    at, sat = ops.quantize_fp8(torch.randn(2100, 70, device=DEV), transposed=True)[2:]
    assert ops.matmul_fp8(at, sat, q, s).shape == (70, 40)
    # values that do not come from here: the padded length is all there is to compare
    assert ops.linear_fp8(torch.randn(3, 2057, device=DEV), q.clone(), s.clone()).shape == (3, 40)


@pytest.mark.parametrize("M", [3, 40, 200])
def test_scales_at_the_ends_of_their_range(M):
    """16-bit results: the matrix instruction takes every scale there is; fp32 results: exact products for block exponents down to -117, where an e4m3
    value's lowest bit is bf16's smallest normal number."""
    g = torch.Generator().manual_seed(M)
    for dtype, exponent in ((torch.bfloat16, -127), (torch.bfloat16, -120), (torch.float32, -117)):
        a, b = torch.randn(M, 384, generator=g), torch.randn(150, 384, generator=g) * 2.0 ** 100
        a[:, ::128] = 448.0                                              # the largest of every block: e4m3's own, times the power
        a = a.double() * 2.0 ** exponent
        A, B = bf.Operand(a.float(), 1), bf.Operand(b, 1)
        qa = ops.quantize_fp8(a.float().to(DEV))
        assert bool((qa[1].view(torch.uint8) == exponent + 127).all())
        got = ops.matmul_fp8(*qa, *ops.quantize_fp8(b.to(DEV)), dtype=dtype).double().cpu()
        want = bf.product(A, B)
        assert bool(((got - want).abs() <= bf.product_bound(A, B, want, dtype)).all())
