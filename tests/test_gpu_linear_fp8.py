"""GPU: 8-bit block quantisation, the block-scaled product and the linear layer against float64 (oracle/block_fp8.py).
Quantised bytes and scales are exact; products are held to block_fp8.product_bound (derived there from the arithmetic of the two paths)."""
import math

import pytest
import torch

from cnmnet_amd import _lib, autograd, ops
from oracle import block_fp8 as bf

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def data(R, C, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, C, generator=g) * torch.exp(spread * torch.randn(R, 1, generator=g)) * torch.exp(spread * torch.randn(1, C, generator=g))).to(dtype)


def same_values(got, want):
    got = got.float().cpu().double()
    assert got.shape == want.shape
    return bool(torch.equal(torch.isnan(got), torch.isnan(want))) and bool(torch.equal(torch.nan_to_num(got), torch.nan_to_num(want)))


def check_quantized(x, block_rows, got):
    R, C = x.shape
    q, e = bf.quantize(x.cpu(), block_rows)
    assert same_values(got[0], q)
    assert torch.equal(got[1].view(torch.uint8).cpu().long(), e + 127)
    if len(got) == 4:
        if block_rows == 1:
            qt, et = bf.quantize(x.cpu().t().contiguous(), 1)
        else:
            qt, et = bf.quantize(x.cpu().t().contiguous(), 128)
        assert same_values(got[2], qt)
        assert torch.equal(got[3].view(torch.uint8).cpu().long(), et + 127)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (3, 130), (127, 257), (128, 128), (130, 64), (300, 1000)])
@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_is_exact(R, C, dtype, block_rows):
    x = data(R, C, dtype, R * 1000 + C).to(DEV)
    check_quantized(x, block_rows, ops.quantize_fp8(x, block_rows, transposed=True))
    q, s = ops.quantize_fp8(x, block_rows)
    check_quantized(x, block_rows, (q, s))


def test_quantize_every_half_and_its_ties():
    """Every finite float16 value (ties of e4m3 among them), each in a block of its own scale."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[torch.isfinite(x)]
    x = torch.nn.functional.pad(x, (0, -x.numel() % 128)).view(-1, 128)
    check_quantized(x.to(DEV), 1, ops.quantize_fp8(x.to(DEV)))
    # the same exponents next to one value that fixes the scale: everything rounds on the same grid, subnormals of e4m3 included
    y = torch.cat([x[:, :127].clamp(-448, 448), torch.full((x.shape[0], 1), 448.0, dtype=torch.float16)], 1)
    check_quantized(y.to(DEV), 1, ops.quantize_fp8(y.to(DEV)))


def test_quantize_extremes():
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 4, [inf, 1.0, -inf, nan], [3.4e38, -3.4e38, 1e30, 0.0], [1e-45, -1e-40, 1e-38, 0.0], [448.0, 1.0, 0.0, -0.0], [448.00003, 1.0, 17.0, 2.0 ** -9],
            [nan] * 4, [-448.0 * 2.0 ** -127, 2.0 ** -126, 0.0, 0.0]]
    x = torch.tensor(rows)
    check_quantized(x.to(DEV), 1, ops.quantize_fp8(x.to(DEV)))
    check_quantized(x.to(DEV), 128, ops.quantize_fp8(x.to(DEV), 128, transposed=True))


def test_quantize_strides_and_alignment():
    base = data(40, 300, torch.bfloat16, 9).to(DEV)
    for view in (base[:, :200], base[:, 1:202], base[1::2, 3:131], base.t(), base[:1, 5:40], base.view(4, 10, 300)):
        flat = view.reshape(-1, view.shape[-1])
        check_quantized(flat, 1, ops.quantize_fp8(view, 1, transposed=True))


def product(M, N, K, dtype, block_rows, seed):
    a, b = data(M, K, torch.float32, seed), data(N, K, torch.float32, seed + 1)
    A, B = bf.Operand(a, 1), bf.Operand(b, block_rows)
    qa, qb = ops.quantize_fp8(a.to(DEV)), ops.quantize_fp8(b.to(DEV), block_rows)
    got = ops.matmul_fp8(*qa, *qb, dtype=dtype).double().cpu()
    want = bf.product(A, B)
    if dtype == torch.float16:
        keep = want.abs() < 6e4
        got, want = torch.where(keep, got, 0.0), torch.where(keep, want, 0.0)
    bound = bf.product_bound(A, B, want, dtype)
    assert got.shape == want.shape and bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 200, 4096), (2, 129, 130), (16, 64, 512), (17, 1000, 640), (33, 31, 1100), (64, 128, 128), (65, 300, 2057), (100, 257, 300), (200, 64, 512),
                                   (257, 129, 385), (300, 500, 1024), (513, 769, 256)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_product(M, N, K, block_rows):
    product(M, N, K, TYPES[(M + N) % 3], block_rows, M + N + K)


@pytest.mark.parametrize("dtype", TYPES)
def test_product_larger(dtype):
    product(1100, 900, 1500, dtype, 128, 5)
    product(600, 1030, 1030, dtype, 1, 6)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_product_long_reduction(block_rows):
    """More blocks than a workgroup holds scales for at once; few rows and many."""
    product(130, 140, 9000, torch.float32, block_rows, 5)
    product(129, 257, 8320, torch.bfloat16, block_rows, 6)
    product(20, 50, 9000, torch.float16, block_rows, 7)
    product(200, 131, 2100, torch.float32, block_rows, 8)               # cut into ranges: uneven last one, odd row length
    product(100, 300, 16400, torch.float16, block_rows, 9)
    product(260, 24, 4224, torch.bfloat16, block_rows, 10)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_product_wide_tiles(dtype):
    """Enough 256 x 256 tiles for the large-tile kernel, ragged at both ends, odd row length; per-row and per-block scales."""
    for block_rows, M, N, K in ((128, 2817, 2999, 130), (1, 3071, 2830, 260)):
        product(M, N, K, dtype, block_rows, M)


def test_product_scales_cover_the_exponent_range():
    """Blocks whose scales are far apart, both ways: every block's own power of two reaches its products and no other's."""
    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(40, 512, generator=g), torch.randn(70, 512, generator=g)
    for kb, e in enumerate((-60, 40, 0, 13)):
        a[:, kb * 128:(kb + 1) * 128] *= 2.0 ** e
        b[:, kb * 128:(kb + 1) * 128] *= 2.0 ** -e
    a *= torch.pow(2.0, torch.arange(40) % 7 - 3.0)[:, None]
    A, B = bf.Operand(a, 1), bf.Operand(b, 1)
    got = ops.matmul_fp8(*ops.quantize_fp8(a.to(DEV)), *ops.quantize_fp8(b.to(DEV)), dtype=torch.float32).double().cpu()
    want = bf.product(A, B)
    assert bool(((got - want).abs() <= bf.product_bound(A, B, want, torch.float32)).all())


def test_product_nan_stays_in_its_row():
    a, b = data(20, 256, torch.float32, 2), data(30, 256, torch.float32, 3)
    a[7, 200] = float("nan")
    b[11, 3] = float("inf")
    got = ops.matmul_fp8(*ops.quantize_fp8(a.to(DEV)), *ops.quantize_fp8(b.to(DEV)), dtype=torch.float32).cpu()
    bad = torch.isnan(got)
    want = torch.zeros(20, 30, dtype=torch.bool)
    want[7], want[:, 11] = True, True
    assert torch.equal(bad, want)


def test_product_leaves_the_gap_between_rows():
    """The C entry writes N columns of ldc and nothing behind the last row."""
    lib = _lib.load()
    for M, N in ((5, 33), (130, 130)):
        a, b = ops.quantize_fp8(data(M, 128, torch.float32, 1).to(DEV)), ops.quantize_fp8(data(N, 128, torch.float32, 2).to(DEV))
        c = torch.full((M + 3, N + 7), 5.0, device=DEV)
        _lib.check(lib.cnm_matmul_fp8(a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), 1, c.data_ptr(), 0, N + 7, M, N, 128, None, 0, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(c[:M, :N], ops.matmul_fp8(*a, *b, dtype=torch.float32))
        assert bool((c[M:] == 5.0).all()) and bool((c[:, N:] == 5.0).all())


@pytest.mark.parametrize("shape,N", [((1, 700), 300), ((3, 5, 64), 17), ((130, 1025), 64), ((64,), 9), ((48, 2048), 515), ((20, 384), 1), ((16, 2057), 100), ((7, 5000), 33), ((1000, 200), 100),
                                     ((5000, 128), 128), ((333, 300), 65), ((300, 301), 200), ((17, 129), 129)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_inference(shape, N, dtype):
    K = shape[-1]
    x, w = data(int(math.prod(shape[:-1])), K, dtype, 11).view(shape), data(N, K, torch.float32, 12) / math.sqrt(K)
    q, s = ops.pack_linear_fp8(w.to(DEV))
    y = ops.linear_fp8(x.to(DEV), q, s)
    assert y.shape == shape[:-1] + (N,) and y.dtype == dtype
    A, B = bf.Operand(x.reshape(-1, K), 1), bf.Operand(w, 128)
    want = bf.product(A, B)
    assert bool(((y.double().cpu().reshape(-1, N) - want).abs() <= bf.product_bound(A, B, want, dtype)).all())


def test_linear_rows_do_not_depend_on_the_batch():
    """A token's result is the same bits alone and in any batch size (each batch size may run another kernel: the order of fp32 sums along the
    reduced axis is compared through its bound, the quantised operands are the same)."""
    x, w = data(300, 640, torch.float32, 21), data(200, 640, torch.float32, 22)
    q, s = ops.pack_linear_fp8(w.to(DEV))
    A, B = bf.Operand(x, 1), bf.Operand(w, 128)
    want = bf.product(A, B)
    bound = bf.product_bound(A, B, want, torch.float32)
    for n in (1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 300):
        y = ops.linear_fp8(x[:n].to(DEV), q, s).double().cpu()
        assert bool(((y - want[:n]).abs() <= bound[:n]).all()), n


def test_linear_nonfinite_and_extreme_inputs():
    """What quantize_fp8 makes of them, also where the layer quantises on the way (few rows, few columns)."""
    for M, N in ((3, 200), (200, 40), (200, 300)):
        x, w = data(M, 300, torch.float32, 5), data(N, 300, torch.float32, 6)
        x[0, 5], x[1, 290] = float("inf"), float("nan")
        x[2] *= 1e-30
        q, s = ops.pack_linear_fp8(w.to(DEV))
        y = ops.linear_fp8(x.to(DEV), q, s).cpu().double()
        assert bool(torch.isnan(y[:2]).all()) and not bool(torch.isnan(y[2:]).any())
        A, B = bf.Operand(x[2:], 1), bf.Operand(w, 128)
        want = bf.product(A, B)
        assert bool(((y[2:] - want).abs() <= bf.product_bound(A, B, want, torch.float32)).all())
        # finite values next to an infinity keep their own scale: the infinity alone makes the row NaN
        z = x.clone()
        z[0, 5] = 0
        assert torch.equal(ops.quantize_fp8(x.to(DEV))[1][0].view(torch.uint8), ops.quantize_fp8(z.to(DEV))[1][0].view(torch.uint8))


def test_linear_row_stride_and_alignment():
    w = data(150, 200, torch.float32, 6)
    q, s = ops.pack_linear_fp8(w.to(DEV))
    for dtype in TYPES:
        base = data(40, 303, dtype, 4).to(DEV)
        for v in (base[:, :200], base[:, 1:201], base[:, 103:], base[::3, 7:207], base[:9, 5:205]):
            assert torch.equal(ops.linear_fp8(v, q, s), ops.linear_fp8(v.contiguous(), q, s))


def test_linear_no_rows():
    q, s = ops.pack_linear_fp8(data(20, 100, torch.float32, 1).to(DEV))
    assert ops.linear_fp8(torch.empty(0, 100, device=DEV), q, s).shape == (0, 20)
    x = torch.empty(0, 100, device=DEV, requires_grad=True)
    w = torch.randn(20, 100, device=DEV, requires_grad=True)
    autograd.linear_fp8(x, w).sum().backward()
    assert x.grad.shape == (0, 100) and bool((w.grad == 0).all())


def test_refusals_on_the_device():
    x = data(4, 256, torch.float32, 1).to(DEV)
    q, s = ops.quantize_fp8(x)
    wq, ws = ops.pack_linear_fp8(x)
    for bad in ((q[:, :100], s, q, s), (q, s[:, :1].contiguous(), q, s), (q, s, q[:, 128:], s), (q.float(), s, q, s), (q, s.view(torch.uint8), q, s),
                (q, s, torch.zeros_like(q[:, :128]).contiguous(), s[:, :1].contiguous()), (wq, ws, q, s)):
        with pytest.raises(_lib.EngineError):
            ops.matmul_fp8(*bad)
    with pytest.raises(_lib.EngineError):
        ops.matmul_fp8(q, s, q, s, dtype=torch.float64)
    with pytest.raises(_lib.EngineError):
        ops.quantize_fp8(x.double())
    with pytest.raises(_lib.EngineError):
        ops.quantize_fp8(x, 64)
    with pytest.raises(_lib.EngineError):
        ops.linear_fp8(x[:, :100], wq, ws)
    with pytest.raises(_lib.EngineError):
        ops.linear_fp8(x, q, s)                                          # per-row scales: not a packed weight


def train_case(M, N, K, xt, wt, seed):
    x, w, dy = data(M, K, xt, seed, 0.3), (data(N, K, torch.float32, seed + 1, 0.3) / math.sqrt(K)).to(wt), data(M, N, xt, seed + 2, 0.3)
    X, W = bf.Operand(x, 1), bf.Operand(w, 128)
    D, Dt, Xt = bf.Operand(dy, 1), bf.Operand(dy.t().contiguous(), 1), bf.Operand(x.t().contiguous(), 1)
    return x, w, dy, ((X, W), (D, W.t()), (Dt, Xt))


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 40, 300), (5, 129, 64), (130, 65, 257), (300, 200, 520), (1000, 96, 128), (3001, 70, 66)])
@pytest.mark.parametrize("xt,wt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
def test_linear_training(M, N, K, xt, wt):
    x, w, dy, pairs = train_case(M, N, K, xt, wt, M + N)
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y = autograd.linear_fp8(xg, wg)
    y.backward(dy.to(DEV))
    for got, (a, b), dtype in zip((y, xg.grad, wg.grad), pairs, (xt, xt, wt)):
        want = bf.product(a, b)
        assert got.dtype == dtype and got.shape == want.shape
        assert bool(((got.detach().double().cpu() - want).abs() <= bf.product_bound(a, b, want, dtype)).all())


def test_linear_training_gradients_are_those_of_the_layer():
    """Against the unquantised layer: each operand value is off by at most 2^-4 of itself or, below e4m3's normal range, 2^-10 of its scale
    (<= 2^-10 * block max / 224), so a product sum is off by at most the sum over |a||b| of the operands' errors; and a directional difference of the
    float64 layer agrees with those float64 gradients."""
    M, N, K = 60, 50, 200
    x, w, dy, _ = train_case(M, N, K, torch.float32, torch.float32, 7)
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    autograd.linear_fp8(xg, wg).backward(dy.to(DEV))
    X, W, D = x.double(), w.double(), dy.double()

    def off(t, rows):                                                    # bound of |Q(t) - t| elementwise
        e = bf.exponents(t, rows)
        per = bf._pow2(e.repeat_interleave(rows, 0)[:t.shape[0]].repeat_interleave(128, 1)[:, :t.shape[1]])
        return torch.maximum(t.double().abs() * 2.0 ** -4, per * 2.0 ** -10)

    def bound(a, ea, b, eb):
        return (ea @ b.abs().t() + a.abs() @ eb.t() + ea @ eb.t()) * (1 + 1e-6) + 1e-6 * (a.abs() @ b.abs().t())
    dx, dw = D @ W, D.t() @ X
    assert bool(((xg.grad.double().cpu() - dx).abs() <= bound(D, off(dy, 1), W.t(), off(w, 128).t())).all())
    assert bool(((wg.grad.double().cpu() - dw).abs() <= bound(D.t(), off(dy.t().contiguous(), 1), X.t(), off(x.t().contiguous(), 1))).all())
    g = torch.Generator().manual_seed(0)
    vx, vw, h = torch.randn(M, K, generator=g).double(), torch.randn(N, K, generator=g).double(), 1e-4
    f = lambda t: float((((X + t * vx) @ (W + t * vw).t()) * D).sum())
    num = (f(h) - f(-h)) / (2 * h)
    assert abs(num - float((dx * vx).sum() + (dw * vw).sum())) < 1e-6 * (1 + abs(num))


def test_linear_partial_gradients_and_broadcast_upstream():
    x, w, dy, pairs = train_case(40, 30, 140, torch.float32, torch.float32, 3)
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV)
    (dx,) = torch.autograd.grad(autograd.linear_fp8(xg, wg), xg, dy.to(DEV))
    xg2, wg2 = x.to(DEV), w.to(DEV).requires_grad_()
    (dw,) = torch.autograd.grad(autograd.linear_fp8(xg2, wg2), wg2, dy.to(DEV))
    xb, wb = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    both = torch.autograd.grad(autograd.linear_fp8(xb, wb), (xb, wb), dy.to(DEV))
    assert torch.equal(dx, both[0]) and torch.equal(dw, both[1])
    y = autograd.linear_fp8(xb, wb)
    one = torch.autograd.grad(y.sum(), xb, retain_graph=True)[0]         # an expanded (stride 0) upstream gradient
    assert torch.equal(one, torch.autograd.grad(y, xb, torch.ones(40, 30, device=DEV))[0])


def test_linear_on_a_side_stream_and_captured():
    x, w, dy, _ = train_case(200, 130, 300, torch.bfloat16, torch.bfloat16, 3)
    q, s = ops.pack_linear_fp8(w.to(DEV))
    xd = x.to(DEV)
    want = ops.linear_fp8(xd, q, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.linear_fp8(xd, q, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    graphs = []
    for n in (1, 200):                                                   # two graphs, replayed in turn, each with its own buffers
        g = torch.cuda.CUDAGraph()
        src = xd[:n].clone()
        with torch.cuda.graph(g):
            out = ops.linear_fp8(src, q, s)
        graphs.append((g, src, out))
    for r in range(3):
        for g, src, out in graphs:
            src.copy_((x[:src.shape[0]] * (r + 1)).to(DEV))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.linear_fp8(src, q, s))


def test_linear_training_step_captured():
    x, w, dy, _ = train_case(150, 70, 260, torch.float32, torch.float32, 3)
    xs, ws, ds = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_(), dy.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(autograd.linear_fp8(xs, ws), (xs, ws), ds)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = autograd.linear_fp8(xs, ws)
        got = torch.autograd.grad(y, (xs, ws), ds)
    for r in range(3):
        with torch.no_grad():
            xs.copy_((x * (1 + r)).to(DEV))
        g.replay()
        torch.cuda.synchronize()
        xe, we = xs.detach().clone().requires_grad_(), ws.detach().clone().requires_grad_()
        ye = autograd.linear_fp8(xe, we)
        want = torch.autograd.grad(ye, (xe, we), ds)
        assert torch.equal(y, ye) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_linear_offsets_beyond_32_bits():
    """More than 2^32 elements of x: the last rows are those of the same rows alone (within the product's bound of float64)."""
    M, K, N = 530000, 8192, 160
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(M, K, device=DEV, dtype=torch.bfloat16)
    x[:1000].zero_()
    x[-300:] = torch.randn(300, K, device=DEV, generator=g)
    x[1000:-300] = 0.5
    w = torch.randn(N, K, device=DEV, generator=g) / 90
    q, s = ops.pack_linear_fp8(w)
    y = ops.linear_fp8(x, q, s)
    A, B = bf.Operand(x[-300:].cpu(), 1), bf.Operand(w.cpu(), 128)
    want = bf.product(A, B)
    assert bool(((y[-300:].double().cpu() - want).abs() <= bf.product_bound(A, B, want, torch.bfloat16)).all())
    assert bool((y[:1000] == 0).all()) and bool((y[1000:-300] == y[1000]).all())
    qx = ops.quantize_fp8(x, 1, transposed=True)
    tail = ops.quantize_fp8(x[-300:])
    assert torch.equal(qx[0][-300:].view(torch.uint8), tail[0].view(torch.uint8)) and torch.equal(qx[1][-300:].view(torch.uint8), tail[1].view(torch.uint8))
    last = (M // 128) * 128                                              # the last block of rows, transposed
    qt = ops.quantize_fp8(x[last:].t().contiguous())
    assert torch.equal(qx[2][:, last:].view(torch.uint8), qt[0].view(torch.uint8)) and torch.equal(qx[3][:, -1:].view(torch.uint8), qt[1].view(torch.uint8))


def test_two_streams_at_once():
    x, w = data(700, 640, torch.bfloat16, 1).to(DEV), data(300, 640, torch.float32, 2).to(DEV)
    q, s = ops.pack_linear_fp8(w)
    want = ops.linear_fp8(x, q, s), ops.linear_fp8(x[:20], q, s)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.linear_fp8(x if i == 0 else x[:20], q, s))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
