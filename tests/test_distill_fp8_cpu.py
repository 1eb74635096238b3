"""CPU: refusals of the 8-bit linear layer and the distillation operators (C entry points and Python), and their oracles against torch."""
import pytest
import torch

from cnmnet_amd import _lib, autograd, ops
from cnmnet_amd.depthnet.losses import TopLogitsDistillLoss
from oracle import block_fp8, top_logits as tl


def test_quantize_entry_refuses():
    f = _lib.load().cnm_quantize_fp8
    ok = [64, 0, 256, 4, 200, 1, 4096, 4096, 0, 0, 0]                     # pointers are never followed: every call below is refused before a launch
    def with_(**kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return f(*a)
    assert with_(_0=0) == -1                                            # no input
    assert with_(_2=100) == -1                                          # row stride below the row
    assert with_(_3=0) == -1 and with_(_4=0) == -1
    assert with_(_5=64) == -1                                           # neither kind of block
    assert with_(_6=0) == -1 and with_(_7=0) == -1                      # values without scale and the other way round
    assert with_(_8=4096) == -1
    assert with_(_6=4104) == -1                                         # alignment
    assert with_(_1=3) == -1                                            # element type
    assert with_(_3=1 << 31) == -2


def test_matmul_entry_refuses():
    f = _lib.load().cnm_matmul_fp8
    ok = [4096, 64, 8192, 64, 1, 4096, 0, 64, 8, 64, 256, 0, 0, 0]
    def with_(**kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return f(*a)
    for i in (0, 1, 2, 3, 5):
        assert with_(**{"_%d" % i: 0}) == -1
    assert with_(_4=2) == -1
    assert with_(_6=7) == -1
    assert with_(_7=63) == -1                                           # ldc below N
    assert with_(_8=0) == -1 and with_(_9=0) == -1
    assert with_(_10=200) == -1 and with_(_10=0) == -1                  # K not in blocks
    assert with_(_10=(1 << 23) + 128) == -2
    assert with_(_0=4100) == -1
    n = _lib.load().cnm_matmul_fp8_workspace_bytes(0, 200, 300, 8192)         # few tiles, long reduction: cut into ranges
    assert n > 0 and n % (200 * 300 * 4) == 0 and _lib.load().cnm_matmul_fp8_workspace_bytes(0, 64, 300, 8192) == 0 and _lib.load().cnm_matmul_fp8_workspace_bytes(0, 4096, 4096, 4096) == 0
    assert with_(_7=300, _8=200, _9=300, _10=8192) == -5 and with_(_7=300, _8=200, _9=300, _10=8192, _11=4096, _12=n - 1) == -5


def test_linear_entry_refuses():
    lib = _lib.load()
    n = lib.cnm_linear_fp8_workspace_bytes(100, 300, 200)
    assert n == (100 * 2 * 129 + 15) // 16 * 16 and lib.cnm_linear_fp8_workspace_bytes(16, 300, 200) == 0 and lib.cnm_linear_fp8_workspace_bytes(1000, 64, 200) == 0
    ok = [64, 0, 200, 4096, 64, 4096, 300, 100, 300, 200, 4096, n, 0]
    def with_(**kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.cnm_linear_fp8(*a)
    for i in (0, 3, 4, 5, 7, 8, 9):
        assert with_(**{"_%d" % i: 0}) == -1
    assert with_(_1=3) == -1 and with_(_2=199) == -1 and with_(_3=4100) == -1 and with_(_6=299) == -1
    assert with_(_10=0) == -5 and with_(_11=n - 1) == -5 and with_(_10=4100) == -5
    assert with_(_9=(1 << 23) + 1, _2=1 << 24) == -2


def test_linear_training_entries_refuse():
    lib = _lib.load()
    M, N, K = 100, 300, 200
    nk, nw = lib.cnm_linear_fp8_keep_bytes(M, N, K, 1, 1), lib.cnm_linear_fp8_train_workspace_bytes(M, N, K)
    assert nk >= K * 384 + 6 + K * 128 + K and lib.cnm_linear_fp8_keep_bytes(M, N, K, 0, 0) == 0 and nk % 16 == 0 and nw % 16 == 0
    fwd = [64, 0, 200, 64, 2, 200, 64, M, N, K, 1, 1, 4096, nk, 4096, nw, 0]
    bwd = [64, 0, 300, 4096, nk, 64, 0, 64, 0, M, N, K, 1, 1, 4096, nw, 0]

    def call(f, ok, **kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return f(*a)
    f = lib.cnm_linear_fp8_forward
    for i in (0, 3, 6, 7, 8, 9):
        assert call(f, fwd, **{"_%d" % i: 0}) == -1
    assert call(f, fwd, _2=199) == -1 and call(f, fwd, _5=199) == -1 and call(f, fwd, _1=4) == -1 and call(f, fwd, _4=3) == -1
    assert call(f, fwd, _12=0) == -5 and call(f, fwd, _13=nk - 1) == -5 and call(f, fwd, _14=0) == -5 and call(f, fwd, _15=nw - 1) == -5 and call(f, fwd, _12=4104) == -5
    assert call(f, fwd, _7=1 << 23) == -2
    f = lib.cnm_linear_fp8_backward
    for i in (0, 3, 9, 10, 11):
        assert call(f, bwd, **{"_%d" % i: 0}) == -1
    assert call(f, bwd, _5=0, _7=0) == -1 and call(f, bwd, _2=299) == -1 and call(f, bwd, _12=0) == -1 and call(f, bwd, _13=0) == -1 and call(f, bwd, _1=9) == -1
    assert call(f, bwd, _6=3) == -1 and call(f, bwd, _8=-1) == -1
    assert call(f, bwd, _4=nk - 1) == -5 and call(f, bwd, _14=0) == -5 and call(f, bwd, _15=nw - 1) == -5


def test_top_and_distill_entries_refuse():
    lib = _lib.load()
    top = [64, 0, 100, 1.0, 64, 64, 64, 0, 0, 4, 100, 8, 1, 0]
    def t(**kw):
        a = list(top)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.cnm_top_logits(*a)
    for i in (0, 4, 5, 6):
        assert t(**{"_%d" % i: 0}) == -1
    assert t(_3=0.0) == -1 and t(_3=1e-38) == -1 and t(_3=float("inf")) == -1 and t(_3=float("nan")) == -1
    assert t(_11=101) == -1 and t(_11=0) == -1 and t(_10=1000, _2=1000, _11=257) == -1
    assert t(_2=99) == -1 and t(_12=3) == -1                            # row stride; rows not a multiple of inner
    assert t(_12=4, _11=17) == -1                                        # planes: at most 16
    assert t(_1=5) == -1 and t(_9=1 << 31) == -2 and t(_10=(1 << 20) + 1, _2=1 << 21) == -2
    need = lib.cnm_top_logits_workspace_bytes(0, 2, 100000, 8, 1)          # two long rows: split
    assert need > 0 and lib.cnm_top_logits_workspace_bytes(0, 4, 100, 8, 1) == 0
    assert t(_9=2, _10=100000, _2=100000) == -5 and t(_9=2, _10=100000, _2=100000, _7=64, _8=need - 1) == -5
    n = lib.cnm_distill_workspace_doubles(0, 4, 100, 1)
    assert n >= 4 and lib.cnm_distill_workspace_doubles(0, 5, 100, 2) == 0 and lib.cnm_distill_workspace_doubles(0, 4, 100000, 1) > n
    dis = [64, 0, 100, 64, 0, 64, 0, None, 1.0, None, None, 0, 0, 1, 64, None, 64, n, 0, 4, 100, 8, 1, 0]
    def d(**kw):
        a = list(dis)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.cnm_distill(*a)
    for i in (0, 3, 5):
        assert d(**{"_%d" % i: 0}) == -1
    assert d(_14=0) == -1                                               # nothing to compute
    assert d(_8=-1.0) == -1 and d(_13=3) == -1 and d(_21=257) == -1 and d(_21=0) == -1
    assert d(_2=99) == -1 and d(_6=4) == -1 and d(_1=-1) == -1
    assert d(_11=1) == -1                                               # per-row upstream gradient without one / with a reduction
    assert d(_10=64, _11=1) == -1
    assert d(_16=0) == -5 and d(_17=n - 1) == -5
    assert d(_20=(1 << 20) + 1, _2=1 << 21) == -2
    assert d(_18=1) == -1                                               # a loss needs its own pass
    # more rows than one launch has threads for: refused before anything is launched
    assert t(_9=1 << 27) == -2 and d(_19=1 << 27, _17=1 << 40) == -2 and d(_19=1 << 28, _22=2, _17=1 << 40) == -2
    assert d(_22=2, _20=100000) == -2                                   # planes that do not fit LDS
    assert lib.cnm_distill_planes_ok(64, 8) == 1 and lib.cnm_distill_planes_ok(100000, 8) == 0 and lib.cnm_distill_planes_ok(64, 0) == 0


def test_python_refuses_cpu_tensors_and_bad_arguments():
    x, w = torch.zeros(3, 130), torch.zeros(5, 130)
    with pytest.raises(_lib.EngineError, match="GPU only"):
        ops.quantize_fp8(x)
    with pytest.raises(_lib.EngineError, match="GPU only"):
        ops.pack_linear_fp8(w)
    with pytest.raises(_lib.EngineError, match=r"\[N, K\]"):
        ops.pack_linear_fp8(torch.zeros(5))
    q, s = torch.zeros(5, 256, dtype=torch.float8_e4m3fn), torch.zeros(1, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(_lib.EngineError):
        ops.linear_fp8(x, q, s)
    with pytest.raises(_lib.EngineError, match="values on cpu"):
        ops.matmul_fp8(q, s, q, s)
    with pytest.raises(_lib.EngineError):
        autograd.linear_fp8(x.requires_grad_(), w)
    with pytest.raises(_lib.EngineError, match="against weight"):
        autograd.linear_fp8(x, torch.zeros(5, 131))
    z = torch.zeros(2, 10)
    with pytest.raises(_lib.EngineError, match="GPU only"):
        ops.top_logits(z, 3)
    i = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(_lib.EngineError, match="GPU only"):
        ops.top_logits_distill(z, i, z[:, :3])
    with pytest.raises(_lib.EngineError, match="GPU only"):
        TopLogitsDistillLoss()(z, i, z[:, :3])


def test_class_layouts_on_the_host():
    """How logits reach the engine, on CPU tensors (no launch): in place where rows or planes allow it, copied otherwise."""
    z = torch.randn(4, 12)
    c = ops._Classes(z[:, :10], -1, lambda V: True)
    assert c.z.data_ptr() == z.data_ptr() and c.ld == 12 and (c.rows, c.V, c.inner) == (4, 10, 1)
    c = ops._Classes(z[:1, :10], 1, lambda V: True)
    assert c.ld == 10 and c.rows == 1
    c = ops._Classes(z.t(), -1, lambda V: True)
    assert c.z.is_contiguous() and c.ld == 4 and c.rows == 12
    c = ops._Classes(z[:1].expand(4, 12), -1, lambda V: True)
    assert c.z.is_contiguous() and c.ld == 12
    v = torch.randn(2, 5, 3, 4)
    c = ops._Classes(v, 1, lambda V: True)
    assert c.z.data_ptr() == v.data_ptr() and (c.rows, c.V, c.inner) == (24, 5, 12) and c.sized(2) == (2, 2, 3, 4) and not c.moved
    c = ops._Classes(v, 1, lambda V: False)
    assert c.moved and c.z.shape == (2, 3, 4, 5) and c.inner == 1 and c.back(c.z).equal(v) and c.sized(2) == (2, 3, 4, 2)
    c = ops._Classes(torch.randn(3, 5, 1), 1, lambda V: False)            # one position per plane: rows as they are
    assert not c.moved and c.inner == 1 and c.rows == 3
    c = ops._Classes(torch.randn(7), 0, lambda V: True)
    assert c.rows == 1 and c.row_shape == ()
    for bad in (torch.randn(()), torch.randn(3, 0)):
        with pytest.raises(_lib.EngineError):
            ops._Classes(bad, -1, lambda V: True)
    with pytest.raises(_lib.EngineError):
        ops._Classes(z, 2, lambda V: True)


def test_fp8_oracle_against_torch():
    torch.manual_seed(3)
    x = torch.randn(5, 300) * torch.exp(4 * torch.randn(5, 1))
    q, e = block_fp8.quantize(x, 1)
    got = (x.double() / block_fp8._pow2(e.repeat_interleave(128, 1)[:, :300])).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(got, q[:, :300]) and float(q.abs().max()) <= 448 and bool((q[:, 300:] == 0).all())
    assert bool((block_fp8.exponents(torch.zeros(1, 4), 1) == -127).all())
    edge = torch.tensor([[448.0, 1.0]]), torch.tensor([[448.0000305, 1.0]])
    assert int(block_fp8.exponents(edge[0], 1)) == 0 and int(block_fp8.exponents(edge[1], 1)) == 1


def test_distill_oracle_against_torch_autograd():
    torch.manual_seed(4)
    z = torch.randn(6, 11, dtype=torch.float64, requires_grad=True)
    teacher = torch.randn(6, 11, dtype=torch.float64)
    val, idx = teacher.topk(4, 1)
    T = 2.0
    lse = torch.logsumexp(teacher / T, 1)
    # lumped remainder: the same KL over five classes
    lq = torch.log_softmax(z / T, 1)
    named = lq.gather(1, idx)
    rest = (1 - named.exp().sum(1)).log()
    p = (val / T - lse[:, None]).exp()
    pr = 1 - p.sum(1)
    ref = (T * T * ((p * (p.log() - named)).sum(1) + pr * (pr.log() - rest))).mean()
    loss, g, _ = tl.distill(z.detach(), idx, val, lse, None, T, "mean")
    assert abs(float(loss - ref)) < 1e-12 and float((torch.autograd.grad(ref, z)[0] - g).abs().max()) < 1e-12
    ref = (T * T * torch.nn.functional.kl_div(torch.log_softmax(z / T, 1).gather(1, idx), torch.log_softmax(val / T, 1), log_target=True, reduction="none").sum(1)).sum()
    loss, g, _ = tl.distill(z.detach(), idx, val, None, None, T, "sum")
    assert abs(float(loss - ref)) < 1e-12 and float((torch.autograd.grad(ref, z)[0] - g).abs().max()) < 1e-12
    v, i, l = tl.top(torch.tensor([[1.0, float("nan"), 3.0, 3.0, float("inf")]]), 4, 1.0)
    assert i.tolist() == [[1, 4, 2, 3]]
