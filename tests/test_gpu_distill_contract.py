"""GPU: what the distillation operators promise at the edges of their contract -- weights, special values, reused graphs, memory -- against the
formula in float64, differentiated by torch on the CPU.

Bounds.  A sum of exponentials: a thread adds at most 128 of them one after another, then 6 steps within a wave, 4 across a workgroup and 6 across
segments, three roundings each: 176 times 2^-24; an exponential is off by 2^-23 and its argument by three roundings of its size X = range / T:
D = (178 + 3 X) 2^-24 relative.  A row's loss: D times 1 + the size of its terms, an entry's p by 8 * 2^-24 more; a gradient element: 2 D of its
q, D + 64 * 2^-24 of its p, half a step of its type."""
import math

import pytest
import torch

from cnmnet_amd import _lib, ops
from cnmnet_amd.depthnet.losses import TopLogitsDistillLoss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


def spread(z, T):
    f = z.double()[torch.isfinite(z)]
    return (178 + 3 * float(f.max() - f.min()) / T) * 2.0 ** -24


def formula(z, idx, val, lse, T):
    """[R, V] on the CPU -> rows' losses, their gradients, the size of their terms; float64, the gradient by torch's own differentiation."""
    z = z.double().requires_grad_()
    R, V = z.shape
    lq = torch.log_softmax(z / T, 1)
    ok = (idx >= 0) & (idx < V)
    at = torch.where(ok, idx, 0).long()
    b = torch.where(ok, val.double() / T, -INF)
    lp = b - (lse.double()[:, None] if lse is not None else torch.logsumexp(b, 1, keepdim=True))
    p = torch.where(ok, lp.exp(), 0.0)
    t = torch.where(p > 0, p * (torch.where(p > 0, lp, 0.0) - lq.gather(1, at)), 0.0)
    loss, mag = t.sum(1), t.abs().sum(1).detach()
    if lse is not None:
        named = torch.zeros(R, V).scatter_add_(1, at, ok.float()) > 0
        rest = torch.logsumexp(torch.where(named, torch.full_like(z, -INF), z / T), 1) - torch.logsumexp(z / T, 1)
        pr = (1 - p.sum(1)).clamp(min=0)
        t = torch.where(pr > 0, pr * (torch.where(pr > 0, pr, 1.0).log() - rest), 0.0)
        loss, mag = loss + t, mag + t.abs().detach()
    loss = T * T * loss
    (g,) = torch.autograd.grad(loss.sum(), z)
    return loss.detach(), g, T * T * (1 + mag), lq.exp().detach(), torch.zeros(R, V, dtype=torch.float64).scatter_add_(1, at, p)


def case(R, V, K, seed, T, tail=True):
    g = torch.Generator().manual_seed(seed)
    z = 3 * torch.randn(R, V, generator=g)
    teacher = 0.7 * z + 1.5 * torch.randn(R, V, generator=g)
    val, idx = teacher.topk(K, 1)
    return z, idx, val, torch.logsumexp(teacher / T, 1) if tail else None


class Layout:
    """The same rows as [R, V], or as planes [2, V, R / 4, 2] with the classes in dim 1."""

    def __init__(self, planes, R):
        self.planes, self.R, self.dim = planes, R, 1 if planes else -1

    def put(self, t):
        if t is None:
            return None
        if self.planes:
            t = t.view(2, self.R // 4, 2, -1).permute(0, 3, 1, 2).contiguous() if t.dim() == 2 else t.view(2, self.R // 4, 2)
        return t.to(DEV)

    def back(self, t):
        t = t.detach().cpu()
        if t.dim() == 4:
            return t.permute(0, 2, 3, 1).reshape(self.R, -1)
        return t.reshape(-1) if self.planes or t.dim() == 0 else t


# few short rows, rows of a whole workgroup, rows cut into segments, planes
FORMS = [(8, 50, False), (8, 3000, False), (4, 40000, False), (8, 64, True)]


def bounds(z, T, lossmag, q, p, c, want):
    D = spread(z, T)
    return 2 * (D + 8 * 2.0 ** -24) * lossmag, T * c.abs()[:, None] * (2 * D * q + (D + 64 * 2.0 ** -24) * (p + q)) + want.abs() * 2.0 ** -23


@pytest.mark.parametrize("R,V,planes", FORMS)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_the_gradient_is_that_of_the_returned_loss(R, V, planes, reduction):
    """Weights (0 and others) and upstream gradients: what backward gives is the derivative of what forward returned, for every reduction."""
    T, K = 2.0, 6
    z, idx, val, lse = case(R, V, K, V, T)
    w = torch.linspace(-0.5, 2, R)
    w[1], w[2] = 0.0, 0.5
    up = torch.linspace(1.5, -3, R) if reduction == "none" else torch.tensor(0.75)
    L, g, mag, q, p = formula(z, idx, val, lse, T)
    n = w.double().sum() if reduction == "mean" else 1.0
    c = w.double() / n
    lay = Layout(planes, R)
    zd = lay.put(z).requires_grad_()
    loss = TopLogitsDistillLoss(T, lay.dim, reduction)(zd, lay.put(idx), lay.put(val), lay.put(lse), lay.put(w))
    (dz,) = torch.autograd.grad(loss, zd, lay.put(up) if reduction == "none" else up.to(DEV))
    want = (c * up.double())[:, None] * g
    bl, bg = bounds(z, T, mag, q, p, c * up.double(), want)
    got = lay.back(loss).double()
    if reduction == "none":
        assert bool(((got - c * L).abs() <= c.abs() * (bl + L.abs() * 2.0 ** -23)).all())
    else:
        assert abs(float(got) - float((c * L).sum())) <= float((c.abs() * bl).sum()) + abs(float((c * L).sum())) * 2.0 ** -23
    assert bool(((lay.back(dz).double() - want).abs() <= bg).all())


def test_a_row_of_weight_zero_has_loss_zero():
    z, idx, val, lse = case(6, 30, 4, 1, 1.0)
    z[2] = NAN
    w = torch.tensor([1.0, 0, 0, 2, 1, 0.5])
    loss = ops.top_logits_distill(z.to(DEV), idx.to(DEV), val.to(DEV), lse.to(DEV), w.to(DEV), reduction="none")
    assert float(loss[1]) == 0 and float(loss[2]) == 0 and bool(torch.isfinite(loss).all())


@pytest.mark.parametrize("R,V,planes", FORMS)
def test_mean_over_weights_of_any_sum(R, V, planes):
    """sum w loss / sum w for a negative sum; a NaN or an infinity among the weights is seen; weights that cancel to 0 give 0."""
    T, K = 2.0, 6
    z, idx, val, lse = case(R, V, K, V + 1, T)
    L, g, mag, q, p = formula(z, idx, val, lse, T)
    lay = Layout(planes, R)

    def run(w):
        zd = lay.put(z).requires_grad_()
        loss = TopLogitsDistillLoss(T, lay.dim)(zd, lay.put(idx), lay.put(val), lay.put(lse), lay.put(w))
        return float(loss.detach()), lay.back(torch.autograd.grad(loss, zd)[0]).double()
    w = torch.linspace(-2, 0.25, R)
    loss, dz = run(w)
    c = w.double() / w.double().sum()
    want = c[:, None] * g
    bl, bg = bounds(z, T, mag, q, p, c, want)
    assert abs(loss - float((c * L).sum())) <= float((c.abs() * bl).sum()) + abs(loss) * 2.0 ** -23
    assert bool(((dz - want).abs() <= bg).all())
    w = torch.ones(R)
    w[1] = NAN
    loss, dz = run(w)
    assert math.isnan(loss) and bool(torch.isnan(dz).all())
    w[1] = INF
    loss, dz = run(w)
    assert math.isnan(loss) and bool(torch.isnan(dz[1]).all()) and bool((dz[[0, 2, 3]] == 0).all())   # inf / inf, and 1 / inf
    w = torch.tensor([1.0, -1.0] * (R // 2))
    loss, dz = run(w)
    assert loss == 0 and bool((dz == 0).all())


@pytest.mark.parametrize("R,V,planes", FORMS)
def test_backward_passes_eager_and_captured_over_one_forward(R, V, planes):
    """An eager forward whose backward is captured and run eagerly too, and a captured forward with both: each backward pass gives the gradient,
    whichever comes first."""
    T, K = 2.0, 6
    z, idx, val, lse = case(R, V, K, V + 2, T)
    w = torch.linspace(0.5, 2, R)
    lay = Layout(planes, R)
    args = [lay.put(t) for t in (idx, val, lse, w)]
    crit = TopLogitsDistillLoss(T, lay.dim)
    zd = lay.put(z).requires_grad_()
    up = torch.tensor(2.5, device=DEV)
    (want,) = torch.autograd.grad(crit(zd, *args), zd, up)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def eager(loss, n=2):
        return [torch.autograd.grad(loss, zd, up, retain_graph=True)[0] for _ in range(n)]
    with torch.cuda.stream(side):                                        # (a captured backward pass runs on its forward's stream: the same for all of them)
        loss = crit(zd, *args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        (dg,) = torch.autograd.grad(loss, zd, up, retain_graph=True)
    with torch.cuda.stream(side):
        got = eager(loss)                                                # before the graph has run for the first time
        g.replay()
        got += eager(loss, 1)
    torch.cuda.synchronize()
    for t in got + [dg]:
        assert torch.equal(t, want)
    dg.fill_(7.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(dg, want)

    f = torch.cuda.CUDAGraph()
    with torch.cuda.graph(f, stream=side):
        loss = crit(zd, *args)
    with torch.cuda.stream(side):
        f.replay()
        got = eager(loss, 1)
    torch.cuda.synchronize()
    b = torch.cuda.CUDAGraph()
    with torch.cuda.graph(b, stream=side):
        (d1,) = torch.autograd.grad(loss, zd, up, retain_graph=True)
        (d2,) = torch.autograd.grad(loss, zd, up, retain_graph=True)
    torch.cuda.synchronize()
    junk = [torch.full((1 << k,), NAN, device=DEV) for k in range(4, 22)]    # whatever was freed is somebody else's by now
    for r in range(3):
        if r:                                                            # other inputs in place: the two graphs, replayed in turn, follow
            with torch.no_grad():
                zd.copy_(lay.put(z * (1 + 0.1 * r)))
                args[3].copy_(lay.put(w + r))
            ze = zd.detach().clone().requires_grad_()
            (want,) = torch.autograd.grad(crit(ze, *args), ze, up)
            torch.cuda.synchronize()
        f.replay()
        b.replay()
        torch.cuda.synchronize()
        for t in (got if r == 0 else []) + [d1, d2]:
            assert torch.equal(t, want)
        d1.fill_(7.0), d2.fill_(7.0)
    del junk


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,V,planes", FORMS + [(300, 40000, False), (8, 700, False)])
def test_log_sum_exp_of_infinite_logits(R, V, planes, dtype):
    """+inf among the logits: the log-sum-exp is +inf; NaN beside it: NaN; the values and classes as ever."""
    lay = Layout(planes, R)
    z = torch.randn(R, V, generator=torch.Generator().manual_seed(V)).to(dtype)
    z[0, 3] = INF
    z[1, V - 1], z[1, 0] = INF, -INF
    z[2, 1:] = INF
    z[3, 5], z[3, 7] = INF, NAN
    val, idx, lse = ops.top_logits(lay.put(z), 4, dim=lay.dim, temperature=2.0)
    lse, val, idx = lay.back(lse), lay.back(val), lay.back(idx)
    assert bool((lse[:3] == INF).all()) and bool(torch.isnan(lse[3]))
    assert idx[0, 0] == 3 and idx[1, 0] == V - 1 and idx[2].tolist() == [1, 2, 3, 4] and idx[3, :2].tolist() == [7, 5]
    assert bool((val[[0, 1], 0] == INF).all()) and bool((val[2] == INF).all())
    if R > 4:
        ref = torch.logsumexp(z[4:].double() / 2, 1)
        assert bool(((lse[4:].double() - ref).abs() <= spread(z[4:], 2.0) + ref.abs() * 2.0 ** -24).all())


@pytest.mark.parametrize("R,V,planes", FORMS)
@pytest.mark.parametrize("tail", [False, True])
def test_an_infinite_student_logit_has_no_softmax(R, V, planes, tail):
    """+inf at a named or an unnamed class: loss and gradient of that row are NaN, the other rows' are as ever."""
    T, K = 2.0, 6
    z, idx, val, lse = case(R, V, K, V + 5, T, tail)
    named = torch.zeros(R, V, dtype=torch.bool).scatter_(1, idx, True)
    z[0, idx[0, 2]] = INF
    z[1, int((~named[1]).nonzero()[7])] = INF
    lay = Layout(planes, R)
    zd = lay.put(z).requires_grad_()
    loss = TopLogitsDistillLoss(T, lay.dim, "none")(zd, lay.put(idx), lay.put(val), lay.put(lse))
    dz = lay.back(torch.autograd.grad(loss.sum(), zd)[0])
    loss = lay.back(loss)
    assert bool(torch.isnan(loss[:2]).all()) and bool(torch.isnan(dz[:2]).all())
    assert bool(torch.isfinite(loss[2:]).all()) and bool(torch.isfinite(dz[2:]).all())


def test_nothing_is_held_after_backward():
    """A loss that is kept (for a log) holds none of the step's memory once its backward pass has run."""
    R, V, K = 512, 16384, 8
    leaf = torch.randn(V, R, device=DEV, requires_grad=True)             # classes strided: the operator works on a copy
    idx = torch.zeros(R, K, device=DEV, dtype=torch.int64) + torch.arange(K, device=DEV)
    crit = TopLogitsDistillLoss()
    torch.autograd.grad(crit(leaf.t(), idx, torch.randn(R, K, device=DEV)), leaf)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = crit(leaf.t(), idx, torch.randn(R, K, device=DEV))
    torch.autograd.grad(loss, leaf)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 4096
    assert bool(torch.isfinite(loss))


def test_saved_tensors_follow_the_hooks():
    """torch.autograd.graph.save_on_cpu: the logits leave the card between the passes, and the gradient is the same."""
    R, V, K = 512, 16384, 8
    z0 = torch.randn(R, V, device=DEV, requires_grad=True)
    idx = torch.zeros(R, K, device=DEV, dtype=torch.int64) + torch.arange(K, device=DEV)
    val = torch.randn(R, K, device=DEV)
    for reduction in ("mean", "none"):
        crit = TopLogitsDistillLoss(reduction=reduction)
        (want,) = torch.autograd.grad((crit(z0 * 2, idx, val) * 3).sum(), z0)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with torch.autograd.graph.save_on_cpu():
            z = z0 * 2
            loss = (crit(z, idx, val) * 3).sum()
        del z
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated() - before
        assert held <= (1.1 if reduction == "mean" else 0.1) * R * V * 4     # "mean": the gradient itself is already there
        assert torch.equal(torch.autograd.grad(loss, z0)[0], want)


def test_saved_rows_come_back_dense():
    """Logits that are columns of a wider matrix lose their row stride on the way to the host and back; a hook that changes more is refused."""
    R, V, K = 40, 300, 5
    wide = torch.randn(R, V + 31, device=DEV, requires_grad=True)
    idx = torch.zeros(R, K, device=DEV, dtype=torch.int64) + torch.arange(K, device=DEV)
    val = torch.randn(R, 2 * K, device=DEV)[:, ::2]
    crit = TopLogitsDistillLoss()
    (want,) = torch.autograd.grad(crit(wide[:, 3:V + 3], idx, val) * 3, wide)
    with torch.autograd.graph.save_on_cpu():
        loss = crit(wide[:, 3:V + 3], idx, val) * 3
    assert torch.equal(torch.autograd.grad(loss, wide)[0], want)
    for change in (lambda t: t.half() if t.is_floating_point() else t, lambda t: t[:1], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = crit(wide[:, 3:V + 3], idx, val)
            with pytest.raises(_lib.EngineError, match="came back"):
                torch.autograd.grad(loss * 3, wide)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        loss = crit(wide[:, 3:V + 3], idx, val)
        assert torch.equal(torch.autograd.grad(loss * 3, wide)[0], want)


@pytest.mark.parametrize("R,V,planes", FORMS)
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_tiny_weights_times_large_upstream_gradients(R, V, planes, reduction):
    """Only their product has to be a float32: neither is rounded before it meets the other."""
    T, K = 1.7, 6
    z, idx, val, lse = case(R, V, K, V + 3, T)
    w = torch.full((R,), 1e-43)
    up = torch.tensor(1e35)
    L, g, mag, q, p = formula(z, idx, val, lse, T)
    lay = Layout(planes, R)
    zd = lay.put(z).requires_grad_()
    loss = TopLogitsDistillLoss(T, lay.dim, reduction)(zd, lay.put(idx), lay.put(val), lay.put(lse), lay.put(w))
    (dz,) = torch.autograd.grad(loss, zd, up.to(DEV).expand(loss.shape))
    c = w.double() * up.double()
    want = c[:, None] * g
    _, bg = bounds(z, T, mag, q, p, c, want)
    assert bool(((lay.back(dz).double() - want).abs() <= bg).all())


@pytest.mark.parametrize("R,V,planes", FORMS)
def test_teacher_entries_that_say_nothing(R, V, planes):
    """Renormalised entries that are all -inf hold no mass: a row without entries.  A NaN in the teacher is seen in the loss and in the gradient."""
    T, K = 2.0, 6
    z, idx, val, lse = case(R, V, K, V + 4, T)
    lay = Layout(planes, R)
    none = val.clone()
    none[1] = -INF
    zd = lay.put(z).requires_grad_()
    loss = TopLogitsDistillLoss(T, lay.dim, "none")(zd, lay.put(idx), lay.put(none))
    dz = lay.back(torch.autograd.grad(loss.sum(), zd)[0])
    loss = lay.back(loss)
    assert float(loss[1]) == 0 and bool((dz[1] == 0).all()) and bool(torch.isfinite(loss).all()) and bool(torch.isfinite(dz).all()) and float(loss[0]) > 0
    bad = val.clone()
    bad[0, 2], bad[1, 0], bad[2, 5] = NAN, NAN, INF
    dead = lse.clone()
    dead[3] = NAN
    for l in (None, dead):
        zd = lay.put(z).requires_grad_()
        loss = TopLogitsDistillLoss(T, lay.dim, "none")(zd, lay.put(idx), lay.put(bad), lay.put(l))
        dz = lay.back(torch.autograd.grad(loss.sum(), zd)[0])
        loss = lay.back(loss)
        assert bool(torch.isnan(loss[:2]).all()) and bool(torch.isnan(dz[:2]).any(1).all())
        assert not bool(torch.isfinite(loss[2]))
        assert bool(torch.isnan(loss[3])) == (l is not None) and bool(torch.isnan(dz[3]).any()) == (l is not None)
        assert bool(torch.isfinite(loss[4:]).all()) and bool(torch.isfinite(dz[4:]).all())


@pytest.mark.parametrize("R", [5, 140])
@pytest.mark.parametrize("V,dtype", [(131072, torch.bfloat16), (131069, torch.float16), (65533, torch.float32), (100003, torch.float32), (32768, torch.bfloat16)])
def test_every_class_of_a_long_row_counts(R, V, dtype):
    """Equal logits: the log-sum-exp is log V, and sixteen bytes that a thread leaves out would be missed; a heavy class at either end or at the seams of
    vectors, threads and segments; the bound is that of the sums' depth, not of the row's length."""
    z = torch.zeros(R, V, dtype=dtype)
    seams = [0, V - 1, V - 2, V // 2, 8191, 8192, 4095, 4096, 16384, 32767]
    for r in range(1, R):
        z[r, seams[r % len(seams)]] = 10.0
    val, idx, lse = ops.top_logits(z.to(DEV), 3)
    ref = torch.logsumexp(z.double(), 1)
    D = spread(z, 1.0)
    assert D < 8.0 / V
    assert bool(((lse.cpu().double() - ref).abs() <= D + ref * 2.0 ** -24).all())
    assert idx[1:, 0].cpu().tolist() == [seams[r % len(seams)] for r in range(1, R)]
    # one entry that holds the teacher's whole mass: the loss is log(V) or log(V + e^10 - 1) less the entry's logit
    at = torch.full((R, 1), 7)
    L, g, mag, q, p = formula(z, at, torch.ones(R, 1), None, 1.0)
    zd = z.to(DEV).requires_grad_()
    loss = TopLogitsDistillLoss(reduction="none")(zd, at.to(DEV), torch.ones(R, 1, device=DEV))
    assert bool(((loss.detach().cpu().double() - L).abs() <= D + L * 2.0 ** -24).all())
    (dz,) = torch.autograd.grad(loss.sum(), zd)
    got = dz.cpu().double()
    assert bool(((got - g).abs() <= 2 * D * q + 8 * 2.0 ** -24 * p + g.abs() * torch.finfo(dtype).eps / 2 * 1.01 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())
