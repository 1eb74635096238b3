"""CPU: the distillation oracle against itself (its gradient is the derivative of the loss that it returns) and the formula; sizes that the 8-bit
linear layer's entries refuse."""
import pytest
import torch

from cnmnet_amd import _lib
from oracle import top_logits as tl


def case(R=7, V=12, K=4, seed=2):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(R, V, dtype=torch.float64, generator=g)
    teacher = torch.randn(R, V, dtype=torch.float64, generator=g)
    val, idx = teacher.topk(K, 1)
    idx[3, 2:] = -1
    return z, idx, val, torch.logsumexp(teacher / 2.0, 1), torch.tensor([0.5, 0.0, -1.5, 2.0, 1.0, 0.25, 3.0], dtype=torch.float64)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_oracle_gradient_is_that_of_its_loss(reduction, tail):
    """Central differences, weights (0 among them) and upstream gradients included; step 1e-5: off by 1e-10 of the third derivative and 1e-16 / 1e-5."""
    z, idx, val, lse, w = case()
    go = torch.linspace(-2, 3, 7, dtype=torch.float64) if reduction == "none" else torch.tensor(1.5, dtype=torch.float64)
    lse = lse if tail else None
    g = tl.distill(z, idx, val, lse, w, 2.0, reduction, go)[1]
    rng = torch.Generator().manual_seed(5)
    for _ in range(6):
        d, h = torch.randn(7, 12, dtype=torch.float64, generator=rng), 1e-5
        num = ((tl.distill(z + h * d, idx, val, lse, w, 2.0, reduction)[0] - tl.distill(z - h * d, idx, val, lse, w, 2.0, reduction)[0]) / (2 * h) * go).sum()
        assert abs(float(num) - float((g * d).sum())) < 1e-8


def test_oracle_weights_each_row():
    z, idx, val, lse, w = case()
    plain, weighted = (tl.distill(z, idx, val, lse, x, 2.0, "none")[0] for x in (None, w))
    assert torch.equal(weighted, w * plain)


def test_oracle_mean_of_weights_of_any_sum():
    z, idx, val, lse, w = case()
    rows = tl.distill(z, idx, val, lse, None, 2.0, "none")[0]
    for w in (-w, torch.linspace(-2, 0.5, 7, dtype=torch.float64)):
        loss, g, _ = tl.distill(z, idx, val, lse, w, 2.0, "mean")
        assert float(w.sum()) < 0 and abs(float(loss) - float((w * rows).sum() / w.sum())) < 1e-14 and float(g.abs().max()) > 0
    w[2] = float("nan")
    loss, g, _ = tl.distill(z, idx, val, lse, w, 2.0, "mean")
    assert bool(torch.isnan(loss)) and bool(torch.isnan(g).any())


@pytest.mark.parametrize("tail", [False, True])
def test_oracle_teacher_entries_that_say_nothing(tail):
    """A NaN among a row's entries is in its loss and gradient; renormalised entries that are all -inf are no entries."""
    z, idx, val, lse, w = case()
    val[0, 1], val[1] = float("nan"), -float("inf")
    loss, g, _ = tl.distill(z, idx, val, lse if tail else None, None, 2.0, "none")
    assert bool(torch.isnan(loss[0])) and bool(torch.isnan(g[0]).any()) and bool(torch.isfinite(loss[1:]).all()) and bool(torch.isfinite(g[1:]).all())
    if not tail:
        assert float(loss[1]) == 0 and float(g[1].abs().max()) == 0


def test_linear_entries_refuse_more_than_one_launch_holds():
    """2^32 threads and more are refused before anything is launched; just below that the workspace (absent here) is what is missed."""
    lib = _lib.load()
    big = 1 << 60
    quantize = lambda rows, cols: lib.cnm_quantize_fp8(64, 0, cols, rows, cols, 1, 4096, 4096, 0, 0, 0)
    assert quantize(1 << 30, 1) == -2 and quantize(1 << 26, 2048) == -2
    matmul = lambda M, N: lib.cnm_matmul_fp8(4096, 64, 8192, 64, 1, 4096, 0, N, M, N, 128, 0, 0, 0)
    assert matmul(1, 1 << 27) == -2 and matmul(64, 1 << 30) == -2 and matmul(1 << 20, 1 << 19) == -2
    linear = lambda M, N, K, n=0: lib.cnm_linear_fp8(64, 1, K, 4096, 64, 4096, N, M, N, K, 4096 if n else 0, n, 0)
    assert linear(1, 1 << 27, 8) == -2 and linear(1 << 30, 100, 8) == -2                  # few rows, few columns
    assert linear(1 << 30, 200, 8, big) == -2 and linear(1 << 20, 1 << 20, 8, big) == -2  # its quantisation, its product
    assert linear(1 << 20, 200, 8) == -5
    forward = lambda M, N, K: lib.cnm_linear_fp8_forward(4096, 0, K, 4096, 0, K, 4096, M, N, K, 0, 0, 0, 0, 4096, big, 0)
    backward = lambda M, N, K: lib.cnm_linear_fp8_backward(4096, 0, N, 4096, big, 4096, 0, 0, 0, M, N, K, 1, 0, 4096, big, 0)
    for f in (forward, backward):
        for shape in ((1 << 22, 8, 1 << 16), (8, 1 << 22, 1 << 16), (1 << 22, 1 << 16, 8)):
            assert f(*shape) == -2
