"""GPU: a teacher's top logits and the distillation loss against float64 (oracle/top_logits.py).

Bounds, derived from the arithmetic: an exponent (z c - o, one fma, c rounded once) is off by at most 2^-24 (2 X + X) with X the row's range of
z log2(e) / T including its size; the exponential and each of V additions by 2^-23: the log-sum-exp by D = (V + 4 X + 16) 2^-23.  The loss weighs
such errors by at most 1 + sum |terms|; a gradient element by its own q and p."""
import pytest
import torch

from cnmnet_amd import _lib, autograd, ops
from cnmnet_amd.depthnet.losses import TopLogitsDistillLoss
from oracle import top_logits as tl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def delta(z, T):
    fin = torch.where(torch.isfinite(z), z, torch.zeros_like(z)).double()
    return (z.shape[-1] + 8 * float(fin.abs().max()) * 1.4427 / T + 16) * 2.0 ** -23


def rows(t, dim):
    """classes last, 2-D, on the CPU"""
    t = t.detach().cpu()
    return t.movedim(dim, -1).reshape(-1, t.shape[dim])


def check_top(z, k, dim=-1, T=1.0):
    val, idx, lse = ops.top_logits(z, k, dim=dim, temperature=T)
    zr = rows(z, dim)
    v, i, l = tl.top(zr, k, T)
    assert val.dtype == z.dtype and idx.dtype == torch.int32 and lse.dtype == torch.float32
    assert val.shape == idx.shape and lse.numel() == zr.shape[0]
    assert torch.equal(rows(idx, dim).long(), i)
    assert torch.equal(torch.nan_to_num(rows(val, dim).double(), nan=777.0), torch.nan_to_num(v.double(), nan=777.0))
    got = lse.detach().cpu().double().reshape(-1)
    ok = torch.isfinite(l)
    assert torch.equal(torch.isnan(got), torch.isnan(l)) and torch.equal(got[~ok & ~torch.isnan(l)], l[~ok & ~torch.isnan(l)])
    assert bool(((got - l)[ok].abs() <= delta(zr, T) + l[ok].abs() * 2.0 ** -23).all())


@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (5, 17, 17), (4, 64, 8), (7, 100, 1), (2, 256, 256), (3, 1000, 33), (2, 1025, 64), (3, 4097, 5), (2, 9001, 128), (1, 50021, 16), (2, 131072, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_top_rows(R, V, k, dtype):
    g = torch.Generator().manual_seed(V)
    check_top((3 * torch.randn(R, V, generator=g)).to(dtype).to(DEV), k, T=[1.0, 2.0, 0.5][R % 3])


@pytest.mark.parametrize("V", [40, 3000, 20000])
def test_top_ties_and_special_values(V):
    inf, nan = float("inf"), float("nan")
    z = torch.zeros(8, V)
    z[1] = torch.arange(V) % 3                                           # a third of all classes tie for the maximum
    z[2, 5:] = -inf
    z[3] = -inf
    z[4, V - 1], z[4, 3], z[4, 7] = inf, nan, nan
    z[5] = -torch.arange(V, dtype=torch.float32)                         # descending
    z[6] = torch.arange(V, dtype=torch.float32)                          # ascending: the largest are the last
    z[7, ::2] = -0.0                                                     # -0 and +0 are equal
    z[7, V // 2:] = torch.finfo(torch.float32).min
    for k in (1, 7, 30):
        check_top(z.to(DEV), k)
    check_top(z.bfloat16().to(DEV), 20)


def test_top_all_equal_to_the_last_entry():
    z = torch.full((3, 5000), 2.5)
    z[1, 4000] = 3.0
    check_top(z.to(DEV), 256)


@pytest.mark.parametrize("B,V,H,W,k", [(1, 3, 1, 2, 3), (2, 64, 5, 13, 8), (1, 64, 24, 32, 1), (3, 96, 7, 9, 16), (2, 40, 8, 8, 4), (2, 70, 6, 11, 30), (1, 600, 4, 17, 12)])
@pytest.mark.parametrize("dtype", TYPES)
def test_top_planes(B, V, H, W, k, dtype):
    g = torch.Generator().manual_seed(V + W)
    z = (2 * torch.randn(B, V, H, W, generator=g)).to(dtype)
    z[:, ::7] = 1.0                                                      # ties
    check_top(z.to(DEV), k, dim=1)
    check_top(z.to(DEV), k, dim=-3, T=3.0)


def test_top_strides_and_ranks():
    base = torch.randn(6, 300, generator=torch.Generator().manual_seed(0)).to(DEV)
    for z in (base[:, :200], base[:, 1:250], base[::2, 3:], base.t(), base[:1, 7:], base.view(2, 3, 300)):
        check_top(z, 5)
    check_top(base[0], 9)
    assert ops.top_logits(base[:0], 3)[0].shape == (0, 3)


def test_top_refusals():
    z = torch.randn(4, 20, device=DEV)
    for bad in (lambda: ops.top_logits(z, 0), lambda: ops.top_logits(z, 21), lambda: ops.top_logits(z, 3, dim=2), lambda: ops.top_logits(z, 3, temperature=0.0),
                lambda: ops.top_logits(z, 3, temperature=float("nan")), lambda: ops.top_logits(z.double(), 3), lambda: ops.top_logits(torch.randn(2, 400, device=DEV), 257)):
        with pytest.raises(_lib.EngineError):
            bad()


def make(R, V, K, dtype, seed, tail, weighted, short, T, dup=False):
    g = torch.Generator().manual_seed(seed)
    z = (3 * torch.randn(R, V, generator=g)).to(dtype)
    teacher = 0.7 * z.float() + 1.5 * torch.randn(R, V, generator=g)
    val, idx = teacher.topk(K, 1)
    if short:
        n = torch.randint(0, K + 1, (R, 1), generator=g)
        idx = torch.where(torch.arange(K) < n, idx, torch.where(torch.arange(K) % 2 == 0, -1, V + 5))
    if dup and K > 1:
        idx[:, -1] = idx[:, 0]
        val[:, -1] = val[:, 0] - 0.5
    lse = torch.logsumexp(teacher / T, 1) + (0.4 if dup else 0.0) if tail else None
    w = None
    if weighted:
        w = torch.rand(R, generator=g)
        w[::3] = 0.0
    return z, idx, val.to(dtype), lse, w


def dev(t):
    return None if t is None else t.to(DEV)


def check_distill(z, idx, val, lse, w, T, reduction, go=None, view=None, **kw):
    """view: how (z, idx, val, lse, w) are arranged for the call (a function to the call's arrangement and its inverse for gradients)."""
    put, back = view or ((lambda t, c: t), (lambda t: t))
    zd = put(dev(z), True).detach().requires_grad_()
    crit = TopLogitsDistillLoss(temperature=T, reduction=reduction, **kw)
    loss = crit(zd, put(dev(idx), True), put(dev(val), True), None if lse is None else put(dev(lse), False), None if w is None else put(dev(w), False))
    up = torch.ones((), device=DEV) if go is None else dev(go)
    up = up.expand(loss.shape) if up.dim() == 0 else put(up, False)
    (dz,) = torch.autograd.grad(loss, zd, up)
    wl, wg, mag = tl.distill(z, idx, val, lse, w, T, reduction, go)
    d = delta(z, T)
    R = z.shape[0]
    ww = torch.ones(R).double() if w is None else w.double()
    if reduction == "none":
        got = loss.detach().cpu().double().reshape(-1)
        assert bool(((got - wl).abs() <= T * T * d * mag + wl.abs() * 2.0 ** -23).all()), float(((got - wl).abs() / (T * T * d * mag)).max())
        c = ww * (go.double() if go is not None and go.dim() else 1.0)
    else:
        n = (ww.sum() if reduction == "mean" else torch.ones(())).double()
        c = (ww / n if float(n) > 0 else torch.zeros(R)).double()
        assert loss.shape == () and abs(float(loss.detach()) - float(wl)) <= float((T * T * d * mag * c).sum()) + abs(float(wl)) * 2.0 ** -22
        c = c * (float(go) if go is not None else 1.0)
    got = back(dz).detach().cpu().double()
    assert dz.dtype == z.dtype and got.shape == wg.shape
    # q and p of every element, each off by a relative 2 d (q) and (E + 8) 2^-22 (p), plus the output's rounding
    zr = z.double()
    q = torch.softmax(zr / T, 1)
    qmax = torch.where(torch.isfinite(q), q, torch.ones_like(q))
    ok = (idx >= 0) & (idx < z.shape[1])
    lp = val.double() / T - (lse.double()[:, None] if lse is not None else torch.logsumexp(torch.where(ok, val.double() / T, -1e300), 1, keepdim=True))
    p = torch.zeros_like(qmax).scatter_add_(1, torch.where(ok, idx, 0).long(), torch.where(ok, lp.exp(), 0.0))
    if lse is not None:                                                  # an unnamed class also carries p_r q_v / q_r
        named = torch.zeros_like(qmax).scatter_add_(1, torch.where(ok, idx, 0).long(), ok.double()) > 0
        rest = torch.where(named, 0.0, qmax)
        p = p + rest / rest.sum(1, keepdim=True).clamp(min=1e-300)
    bound = T * c.abs()[:, None] * (2 * d * qmax + (d + 64 * 2.0 ** -23) * p) + wg.abs() * torch.finfo(z.dtype).eps / 2 * 1.01 + torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    assert bool(((got - wg).abs() <= bound).all()), float(((got - wg).abs() / bound).max())
    return loss, dz


@pytest.mark.parametrize("R,V,K", [(1, 2, 1), (1, 1, 1), (6, 5, 5), (9, 64, 8), (5, 100, 3), (3, 1000, 64), (4, 1024, 256), (3, 1100, 17), (2, 9001, 32), (2, 50021, 16), (1, 131072, 128)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows(R, V, K, dtype, tail):
    if V == K and tail:
        K = max(1, K - 1) if V > 1 else 1
    T = [1.0, 2.0, 0.5, 4.0][(R + K) % 4]
    for reduction, weighted, short in (("mean", False, False), ("sum", True, R > 2), ("none", R > 1, R > 2), ("mean", R > 3, True)):
        z, idx, val, lse, w = make(R, V, K, dtype, R + V + K, tail and V > K, weighted, short, T)
        check_distill(z, idx, val, lse, w, T, reduction)


@pytest.mark.parametrize("V,dtype", [(131072, torch.bfloat16), (65536, torch.float32), (40000, torch.float32), (60001, torch.float16)])
def test_distill_long_rows_of_many(V, dtype):
    """Rows that one workgroup holds whole (up to 256 KB), and rows of many that are a little longer."""
    for n in (V, V + 40000):
        z, idx, val, lse, w = make(130, n, 20, dtype, V, True, True, True, 2.0)
        check_distill(z, idx, val, lse, w, 2.0, "mean")
    check_top(z.to(DEV), 40)


@pytest.mark.parametrize("B,V,H,W,K", [(1, 2, 1, 2, 1), (2, 64, 3, 21, 8), (1, 64, 16, 16, 4), (2, 96, 5, 7, 16), (1, 33, 2, 65, 33), (2, 128, 4, 4, 64), (1, 700, 3, 5, 6)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_planes(B, V, H, W, K, dtype, tail):
    """Classes in dim 1 of a volume; 700 classes do not fit LDS and go through rows."""
    R, T = B * H * W, 2.0

    def put(t, classes):
        return t.view(B, H, W, -1).permute(0, 3, 1, 2).contiguous() if classes else t.view(B, H, W)

    def back(t):
        return t.permute(0, 2, 3, 1).reshape(R, V)
    for reduction, weighted, short in (("mean", True, True), ("none", False, True), ("sum", False, False)):
        z, idx, val, lse, w = make(R, V, K, dtype, V + K, tail and V > K, weighted, short, T)
        check_distill(z, idx, val, lse, w, T, reduction, view=(put, back), dim=1)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("V,planes", [(50, False), (5000, False), (64, True)])
def test_distill_upstream_gradient(reduction, V, planes):
    R, K, T = 12, 6, 2.0
    z, idx, val, lse, w = make(R, V, K, torch.float16, 5, True, True, True, T)
    view = ((lambda t, c: t.view(3, 4, -1).permute(0, 2, 1).contiguous() if c else t.view(3, 4)), (lambda t: t.permute(0, 2, 1).reshape(R, V))) if planes else None
    kw = {"dim": 1} if planes else {}
    # 1024: a gradient rounded to fp16 before it is scaled would have lost what this one keeps
    go = torch.linspace(-2, 3, R) if reduction == "none" else torch.tensor(1024.0)
    check_distill(z, idx, val, lse, w, T, reduction, go=go, view=view, **kw)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_the_same_class_twice(tail):
    for R, V, K in ((7, 40, 5), (3, 3000, 9)):
        z, idx, val, lse, w = make(R, V, K, torch.float32, 8, tail, True, False, 2.0, dup=True)
        check_distill(z, idx, val, lse, w, 2.0, "none")
        check_distill(z, idx, val, lse, w, 2.0, "mean")


def test_distill_masked_classes():
    """-inf and the type's lowest value in the student's masked classes: no mass, zero gradient; in the teacher's entries: p = 0."""
    inf = float("inf")
    for low in (-inf, torch.finfo(torch.float32).min):
        z, idx, val, lse, w = make(6, 90, 8, torch.float32, 3, True, False, False, 1.0)
        z[:, 50:] = low
        teacher = torch.randn(6, 90, generator=torch.Generator().manual_seed(1))
        teacher[:, 50:] = -inf
        val, idx = teacher.topk(8, 1)
        lse = torch.logsumexp(teacher, 1)
        idx[:, 7], val[:, 7] = 70, -inf                                  # an entry that says "impossible"
        loss, dz = check_distill(z, idx, val, lse, w, 1.0, "none")
        assert bool((dz[:, 50:] == 0).all()) and bool(torch.isfinite(loss).all())
    # every class outside the entries masked in the student: the remainder has nowhere to go and is left out
    z, idx, val, lse, w = make(4, 30, 5, torch.float32, 3, True, False, False, 1.0)
    keep = torch.zeros(4, 30, dtype=torch.bool).scatter_(1, idx, True)
    z = torch.where(keep, z, -inf)
    loss, dz = check_distill(z, idx, val, lse, w, 1.0, "mean")
    assert bool(torch.isfinite(loss)) and bool((dz.cpu()[~keep] == 0).all())
    loss, dz = check_distill(z - 300.0, idx, val, lse, w, 1.0, "mean")   # far from zero as well
    assert bool(torch.isfinite(loss)) and bool((dz.cpu()[~keep] == 0).all())
    view = ((lambda t, c: t.view(1, 4, -1).permute(0, 2, 1).contiguous() if c else t.view(1, 4)), (lambda t: t.permute(0, 2, 1).reshape(4, 30)))
    check_distill(z - 300.0, idx, val, lse, w, 1.0, "mean", view=view, dim=1)


def test_distill_rows_that_count_for_nothing():
    """Zero weight or no entries: zeros out, even where the logits are NaN or infinite; an all-zero weight gives 0, not NaN."""
    for V in (20, 2000):
        z, idx, val, lse, w = make(6, V, 4, torch.float32, 3, True, False, False, 1.0)
        w = torch.tensor([1.0, 0, 1, 0, 1, 1])
        idx[2], idx[4, :] = -1, V
        z[1], z[2, 3], z[4, 5] = float("nan"), float("inf"), float("nan")
        zd = dev(z).requires_grad_()
        loss = TopLogitsDistillLoss()(zd, dev(idx), dev(val), dev(lse), dev(w))
        (dz,) = torch.autograd.grad(loss, zd)
        assert bool(torch.isfinite(loss)) and bool((dz[1:5][[0, 1, 3]] == 0).all()) and bool(torch.isfinite(dz).all())
        none = TopLogitsDistillLoss(reduction="none")(zd, dev(idx), dev(val), dev(lse))
        assert float(none[2]) == 0 and float(none[4]) == 0 and bool(torch.isnan(none[1]))
        loss = TopLogitsDistillLoss()(zd, dev(idx), dev(val), dev(lse), torch.zeros(6, device=DEV))
        (dz,) = torch.autograd.grad(loss, zd)
        assert float(loss) == 0 and bool((dz == 0).all())
    v = torch.full((1, 16, 4, 5), float("nan"), device=DEV, requires_grad=True)
    i = torch.full((1, 2, 4, 5), -1, device=DEV)
    loss = TopLogitsDistillLoss(dim=1)(v, i, torch.zeros(1, 2, 4, 5, device=DEV))
    assert float(loss) == 0 and bool((torch.autograd.grad(loss, v)[0] == 0).all())


def test_distill_gradient_against_differences():
    for tail in (False, True):
        z, idx, val, lse, w = make(5, 40, 6, torch.float32, 6, tail, True, True, 2.0)
        f = lambda zz: float(tl.distill(zz, idx, val, lse, w, 2.0, "mean")[0])
        zd = dev(z).requires_grad_()
        loss = TopLogitsDistillLoss(temperature=2.0)(zd, dev(idx), dev(val), dev(lse), dev(w))
        (dz,) = torch.autograd.grad(loss, zd)
        g = torch.Generator().manual_seed(9)
        for _ in range(4):
            v, h = torch.randn(5, 40, generator=g).double(), 1e-4
            num = (f(z.double() + h * v) - f(z.double() - h * v)) / (2 * h)
            assert abs(num - float((dz.double().cpu() * v).sum())) < 1e-5 * (1 + abs(num))


def test_distill_backward_twice_and_gradient_call():
    z, idx, val, lse, w = make(8, 300, 6, torch.bfloat16, 6, True, True, True, 2.0)
    zd = dev(z).requires_grad_()
    loss = TopLogitsDistillLoss(temperature=2.0)(zd, dev(idx), dev(val), dev(lse), dev(w))
    first = torch.autograd.grad(loss, zd, retain_graph=True)[0]
    keep = first.clone()
    first.zero_()                                                        # its buffer is the caller's now
    assert torch.equal(torch.autograd.grad(loss, zd, retain_graph=True)[0], keep)
    scaled = torch.autograd.grad(loss * 4, zd)[0]                        # a power of two: the same digits
    assert torch.equal(scaled, keep * 4)
    l2, g2 = ops.top_logits_distill(zd.detach(), dev(idx), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
    assert torch.equal(l2, loss.detach()) and torch.equal(g2, keep)
    with torch.no_grad():
        assert torch.equal(TopLogitsDistillLoss(temperature=2.0)(zd, dev(idx), dev(val), dev(lse), dev(w)), loss)
    rowsum = TopLogitsDistillLoss(temperature=2.0, reduction="none")(zd, dev(idx), dev(val), dev(lse), dev(w))
    again = torch.autograd.grad(rowsum, zd, torch.ones(8, device=DEV), retain_graph=True)[0]
    assert torch.equal(again, torch.autograd.grad(rowsum, zd, torch.ones(8, device=DEV))[0])


def test_distill_repeats_bit_by_bit_and_index_types():
    z, idx, val, lse, w = make(300, 700, 9, torch.float32, 6, True, True, True, 2.0)
    a = ops.top_logits_distill(dev(z), dev(idx), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
    for t in (torch.int32, torch.int64):
        b = ops.top_logits_distill(dev(z), dev(idx.to(t)), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_distill_strides():
    z, idx, val, lse, w = make(6, 100, 5, torch.float32, 6, True, True, False, 2.0)
    want = ops.top_logits_distill(dev(z), dev(idx), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
    wide = torch.randn(6, 131, device=DEV)
    for off in (0, 1, 3, 4):
        v = wide[:, off:off + 100]
        v.copy_(dev(z))
        got = ops.top_logits_distill(v, dev(idx), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
        assert float((got[0] - want[0]).abs()) <= 1e-6 * abs(float(want[0])) and float((got[1] - want[1]).abs().max()) <= 1e-6
    tall = dev(z).t().contiguous().t()                                   # classes strided, no planes: copied
    got = ops.top_logits_distill(tall, dev(idx), dev(val), dev(lse), dev(w), temperature=2.0, grad=True)
    assert torch.equal(got[1], want[1])
    wi = dev(idx).t().contiguous().t()
    assert torch.equal(ops.top_logits_distill(dev(z), wi, dev(val), dev(lse), dev(w), temperature=2.0), want[0])


def test_distill_no_rows():
    z = torch.empty(0, 30, device=DEV, requires_grad=True)
    e = torch.empty(0, 4, device=DEV)
    loss = TopLogitsDistillLoss()(z, e.long(), e)
    assert float(loss) == 0
    loss.backward()
    assert z.grad.shape == (0, 30)


def test_distill_refusals():
    z, idx, val, lse, w = (dev(t) for t in make(6, 100, 5, torch.float32, 6, True, True, False, 2.0))
    f = ops.top_logits_distill
    for bad in (lambda: f(z, idx[:, :4], val), lambda: f(z, idx.float(), val), lambda: f(z, idx, val[:5]), lambda: f(z, idx, val, lse[:5]), lambda: f(z, idx, val, lse.double()),
                lambda: f(z, idx, val, lse, w.bool()), lambda: f(z, idx, val, temperature=-1), lambda: f(z, idx, val, reduction="batch"), lambda: f(z, idx, val, dim=3),
                lambda: f(z.double(), idx, val), lambda: f(z, idx.cpu(), val), lambda: f(z, idx, val.cpu()), lambda: f(z, idx[0], val[0]),
                lambda: f(torch.randn(2, 300, device=DEV), torch.zeros(2, 257, device=DEV).long(), torch.zeros(2, 257, device=DEV)),
                lambda: f(torch.randn(1, (1 << 20) + 1, device=DEV), idx[:1], val[:1])):
        with pytest.raises(_lib.EngineError):
            bad()


@pytest.mark.parametrize("planes", [False, True])
def test_distill_captured(planes):
    """A training step's loss and gradient as a graph; two graphs replayed in turn; an eager forward with a captured backward."""
    z, idx, val, lse, w = make(40, 64, 6, torch.float32, 6, True, True, True, 2.0)
    put = (lambda t, c: t.view(2, 20, -1).permute(0, 2, 1).contiguous() if c else t.view(2, 20)) if planes else (lambda t, c: t)
    crit = TopLogitsDistillLoss(temperature=2.0, dim=1)
    rest = [put(dev(idx), True), put(dev(val), True), put(dev(lse), False), put(dev(w), False)]
    made = []
    for scale in (1.0, 0.5):
        zs = put(dev(z), True).requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(crit(zs, *rest) * scale, zs)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss = crit(zs, *rest) * scale
            (dz,) = torch.autograd.grad(loss, zs)
        made.append((g, zs, loss, dz, scale))
    for r in range(3):
        for g, zs, loss, dz, scale in made:
            with torch.no_grad():
                zs.copy_(put(dev(z * (1 + 0.3 * r)), True))
            dz.fill_(7.0)                                                # what a caller did to the last replay's gradient
            g.replay()
            torch.cuda.synchronize()
            ze = zs.detach().clone().requires_grad_()
            le = crit(ze, *rest) * scale
            assert torch.equal(loss, le) and torch.equal(dz, torch.autograd.grad(le, ze)[0])


def test_distill_chain_as_it_is_used():
    """A frozen teacher's 8-bit head over pixels, its top plane logits stored, a student's 8-bit head trained against them with the valid mask:
    every stage fed by the one before it, against the float64 forms of the same stages."""
    import math
    from oracle import block_fp8 as bf
    B, H, W, Cin, P, K, T = 2, 6, 10, 130, 64, 8, 2.0
    R = B * H * W
    g = torch.Generator().manual_seed(2)
    feat = torch.randn(R, Cin, generator=g)
    wt, ws = torch.randn(P, Cin, generator=g) * 3 / math.sqrt(Cin), torch.randn(P, Cin, generator=g) * 3 / math.sqrt(Cin)
    valid = (torch.rand(B, H, W, generator=g) > 0.3).float()
    with torch.no_grad():
        tl_rows = ops.linear_fp8(feat.to(DEV), *ops.pack_linear_fp8(wt.to(DEV)))
        val, idx, lse = ops.top_logits(tl_rows.view(B, H, W, P), K, temperature=T)
    x, w = feat.to(DEV).requires_grad_(), ws.to(DEV).requires_grad_()
    z = autograd.linear_fp8(x, w).view(B, H, W, P)
    loss = TopLogitsDistillLoss(temperature=T)(z, idx, val, lse, valid.to(DEV))
    z.retain_grad()
    loss.backward()
    # the same planes as a volume, classes in dim 1
    vol = z.detach().permute(0, 3, 1, 2).contiguous()
    v2, i2, l2 = ops.top_logits(tl_rows.view(B, H, W, P).permute(0, 3, 1, 2).contiguous(), K, dim=1, temperature=T)
    assert torch.equal(i2.permute(0, 2, 3, 1), idx) and torch.equal(v2.permute(0, 2, 3, 1), val)
    lv, gv = ops.top_logits_distill(vol, i2, v2, l2, valid.to(DEV), temperature=T, dim=1, grad=True)
    zr = z.detach().cpu().reshape(R, P)
    wl, wg, mag = tl.distill(zr, idx.cpu().reshape(R, K), val.cpu().reshape(R, K), lse.cpu().reshape(R), valid.reshape(R), T, "mean")
    d = delta(zr, T)
    assert abs(float(loss) - float(wl)) <= float(mag.max()) * T * T * d + 1e-6 * abs(float(wl))
    assert abs(float(lv) - float(wl)) <= 2 * float(mag.max()) * T * T * d + 1e-6 * abs(float(wl))   # lse of the other layout: off by d as well
    assert float((z.grad.cpu().double().reshape(R, P) - wg).abs().max()) <= 4 * T * d / float(valid.sum()) + 2.0 ** -23 * float(wg.abs().max())
    assert float((gv.permute(0, 2, 3, 1).reshape(R, P).cpu().double() - wg).abs().max()) <= 8 * T * d / float(valid.sum()) + 2.0 ** -23 * float(wg.abs().max())
    dz = z.grad.cpu().reshape(R, P)
    for got, a, b in ((x.grad, bf.Operand(dz, 1), bf.Operand(ws, 128).t()), (w.grad, bf.Operand(dz.t().contiguous(), 1), bf.Operand(feat.t().contiguous(), 1))):
        want = bf.product(a, b)
        assert bool(((got.double().cpu() - want).abs() <= bf.product_bound(a, b, want, torch.float32)).all())


@pytest.mark.parametrize("planes", [False, True])
def test_offsets_beyond_32_bits(planes):
    """More than 2^32 logits: the last rows give what the same rows give alone."""
    g = torch.Generator(device=DEV).manual_seed(3)
    K, T = 5, 2.0
    if planes:
        z = torch.empty(9, 500, 1000000, device=DEV, dtype=torch.float16)
        tail = torch.randn(1, 500, 1000000, device=DEV, generator=g, dtype=torch.float16)
        z[:-1] = 0.25
        z[-1:] = tail
        pick = lambda t: t[-1:]
    else:
        z = torch.empty(140000, 32768, device=DEV, dtype=torch.bfloat16)
        tail = torch.randn(300, 32768, device=DEV, generator=g, dtype=torch.bfloat16)
        z[:-300] = 0.25
        z[-300:] = tail
        pick = lambda t: t[-300:]
    val, idx, lse = ops.top_logits(z, K, dim=1, temperature=T)
    v, i, l = ops.top_logits(tail, K, dim=1, temperature=T)
    assert torch.equal(pick(val), v) and torch.equal(pick(idx), i) and torch.equal(pick(lse), l)
    assert torch.equal(idx[0].reshape(K, -1)[:, 0].cpu(), torch.arange(K, dtype=torch.int32))
    loss, dz = ops.top_logits_distill(z, idx, val - 1, lse, temperature=T, dim=1, reduction="none", grad=True)
    lt, dt = ops.top_logits_distill(tail, i, v - 1, l, temperature=T, dim=1, reduction="none", grad=True)
    assert torch.equal(pick(loss), lt) and torch.equal(pick(dz), dt)
    assert bool((loss[:-300] == loss.reshape(-1)[0]).all()) if not planes else bool((loss[:-1] == loss.reshape(-1)[0]).all())


def test_distill_on_two_streams_at_once():
    z, idx, val, lse, w = (dev(t) for t in make(300, 3000, 9, torch.float32, 6, True, True, True, 2.0))
    want = ops.top_logits_distill(z, idx, val, lse, w, temperature=2.0, grad=True), ops.top_logits_distill(z[:3], idx[:3], val[:3], lse[:3], temperature=2.0, grad=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.top_logits_distill(z, idx, val, lse, w, temperature=2.0, grad=True) if i == 0
                              else ops.top_logits_distill(z[:3], idx[:3], val[:3], lse[:3], temperature=2.0, grad=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for r in got[i] for a, b in zip(r, want[i]))
