"""GPU: what the 8-bit linear layer refuses and promises beyond its results (those: test_gpu_linear_fp8.py)."""
import pytest
import torch

from cnmnet_amd import _lib, ops

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
