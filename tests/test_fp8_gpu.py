"""The 8-bit operand form and product (csrc/fp8.hip).  The form is compared value by value with the format's definition in 64 bits; products
with the 64-bit product of the operands' own values.

Tolerance of a product: every value an operand stands for is exact, so only the fp32 accumulation (at most one rounding, 2^-24, per product
added, K of them and the K slices' joins) and the final rounding are off: (K + 32) 2^-24 sum_k |a w| + half step |y|.  16-bit outputs come from the
8-bit matrix pipe, which cuts each product at 2^-13 of the largest exponent among its neighbours (inside a block of 128, so at most 2^-13 of the
block's largest |a| times its largest |w|): K 2^-13 max|a| max|w| summed per block on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def two(p):
    return ((p.long() + 1023) << 52).view(torch.float64)


def grid(x):
    """(values, exponents) of x's 8-bit rows from the definition: 2^e smallest with max|finite x| <= 448 2^e, e >= -126; three fraction bits,
    exponents -6 .. 8, subnormal step 2^-9, ties to even; non-finite -> NaN"""
    M, K = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -K % 128)).view(M, -1, 128)
    mag = x.abs()
    top = torch.where(x.isfinite(), mag, torch.zeros_like(mag)).amax(2)
    m, e = torch.frexp(top)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    u = torch.where(x.isfinite(), x, torch.full_like(x, float('nan'))) * two(-e)[:, :, None]
    _, p = torch.frexp(u.abs().clamp(min=2.0 ** -6).nan_to_num(1.0))
    p = p.double() - 1
    q = torch.round(u * two(3 - p)) * two(p - 3) * two(e)[:, :, None]
    return q.view(M, -1)[:, :K], e


def same(a, b):
    a = a.double()
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0)), float((a - b).abs().nan_to_num(0.0).max())


def rand(M, K, dtype, seed, spread=3.0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp2(spread * torch.randn(M, K, generator=g, device=DEV)) * scale
    return x.to(dtype)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('M,K', [(1, 1), (1, 128), (2, 130), (31, 127), (128, 128), (129, 257), (300, 1100), (1000, 64), (5, 5000)])
def test_operand_form_is_the_definition(M, K, dtype):
    from sgg_amd import ops
    x = rand(M, K, dtype, M + K)
    r, c = ops.quantize_fp8(x, 'both')
    assert r.shape == (M, K) and c.shape == (K, M) and r.data.shape == ((K + 127) // 128 * 2, M + M % 2, 64)
    for q, src in ((r, x), (c, x.t().contiguous())):
        v, e = grid(src)
        assert torch.equal(q.exponents(), e.int())
        same(q.dequantize(), v)
        assert not q.codes().view(torch.uint8)[:, q.shape[1]:].any() and not q.data.view(torch.uint8)[:, q.shape[0]:].any()     # zeros past the last column and row
    alone, alone_t = ops.quantize_fp8(x), ops.quantize_fp8(x, 'cols')
    assert torch.equal(alone.data.view(torch.uint8), r.data.view(torch.uint8)) and torch.equal(alone.scale, r.scale)
    assert torch.equal(alone_t.data.view(torch.uint8), c.data.view(torch.uint8)) and torch.equal(alone_t.scale, c.scale)


@pytest.mark.parametrize('dtype,bits', [(F32, 0x7f800001), (F32, -0x7fffff), (F16, 0x7c01), (BF16, 0x7f81)])
def test_signalling_nan_changes_nothing_but_itself(dtype, bits):
    from sgg_amd import ops
    x = rand(130, 140, dtype, 2)
    ref = [q.dequantize() for q in ops.quantize_fp8(x, 'both')]
    x.view(torch.int32 if dtype == F32 else torch.int16)[7, 9] = bits
    x0 = x.clone()
    x0[7, 9] = 0
    for q, r, z in zip(ops.quantize_fp8(x, 'both'), ref, ops.quantize_fp8(x0, 'both')):
        v, w = q.dequantize(), z.dequantize()
        at = (7, 9) if v.shape[0] == 130 else (9, 7)
        assert bool(v[at].isnan()) and int(v.isnan().sum()) == 1 and torch.equal(q.exponents(), z.exponents())
        v[at] = w[at]
        assert torch.equal(v, w)


def test_column_sums_ride_along():
    """quantize_fp8(colsum=True): f32 sums of 128 rows at a time, then of the tiles: off by (rows + 8) half steps of the sum of magnitudes"""
    from sgg_amd import ops
    for M, K, dtype in ((1, 5, F32), (700, 300, BF16), (1300, 130, F16), (0, 7, F32)):
        x = rand(M, K, dtype, M, 0.5)
        for form in ('cols', 'both'):
            q, sums = ops.quantize_fp8(x, form, colsum=True)
            assert sums.shape == (K,) and sums.dtype == F32
            assert float(((sums.double() - x.double().sum(0)).abs() - (M + 8) * U * x.double().abs().sum(0)).max()) <= 0
            plain = ops.quantize_fp8(x, form)
            for a, b in zip(q if form == 'both' else (q,), plain if form == 'both' else (plain,)):
                assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scale, b.scale)
    with pytest.raises(ValueError):
        ops.quantize_fp8(rand(3, 4, F32, 1), colsum=True)


def test_every_code_ties_extremes_and_non_finite():
    from sgg_amd import ops
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).float()
    codes = codes[codes.isfinite()]
    x = torch.zeros(6, 256, device=DEV)
    x[0, :254] = codes                                               # every value of the format, 448 among them: exponent 0, exact
    x[1, :253] = (codes[:-1] + codes[1:]) / 2                        # every midpoint of neighbours: ties to even
    x[1, 0], x[1, 128] = 448.0, 448.0
    x[2, :254] = codes * 2.0 ** 100
    x[3, 3], x[3, 4], x[3, 130] = float('inf'), 1.0, float('nan')    # their block keeps the others' scale
    x[4] = torch.linspace(1e-45, 3e-38, 256, device=DEV)             # fp32 subnormals and just above: the smallest scale
    x[5] = torch.finfo(F32).max
    r, c = ops.quantize_fp8(x, 'both')
    v, e = grid(x)
    assert torch.equal(r.exponents(), e.int())
    same(r.dequantize(), v)
    vt, et = grid(x.t().contiguous())
    assert torch.equal(c.exponents(), et.int())
    same(c.dequantize(), vt)
    same(r.dequantize()[0, :254], codes.double())


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('M,K,ld,off', [(40, 200, 201, 1), (70, 128, 136, 3), (130, 129, 160, 8)])
def test_strided_rows(M, K, ld, off, dtype):
    from sgg_amd import ops
    x = rand(M, K, dtype, 7)
    buf = torch.full((M * ld + 32,), float('nan'), dtype=dtype, device=DEV)
    view = buf[off:off + M * ld].view(M, ld)[:, :K]
    view.copy_(x)
    for a, b in zip(ops.quantize_fp8(view, 'both'), ops.quantize_fp8(x, 'both')):
        assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scale, b.scale)


def cut(a, w):
    """the 8-bit pipe's share: 2^-13 max|a| max|w| for each product, block by block"""
    tops = [torch.stack([v[:, k:k + 128].abs().amax(1) * min(128, v.shape[1] - k) ** 0.5 for k in range(0, v.shape[1], 128)], 1) for v in (a, w)]
    return 2.0 ** -13 * torch.mm(tops[0], tops[1].t().contiguous())


def product(A, W, bias=None, relu=False, dtype=F32):
    a, w = A.dequantize().double(), W.dequantize().double()
    y = torch.mm(a, w.t().contiguous())
    tol = (a.shape[1] + 32) * U * torch.mm(a.abs(), w.abs().t().contiguous())
    if dtype != F32:
        tol = tol + cut(a, w)
    if bias is not None:
        y, tol = y + bias.double(), tol + 2 * U * bias.double().abs()
    return (y.clamp(min=0) if relu else y), tol


def check(got, want, tol):
    over = (got.double() - want).abs() - (tol + torch.finfo(got.dtype).eps / 2 * (want.abs() + tol) + torch.finfo(got.dtype).tiny)
    assert got.numel() == 0 or float(over.max()) <= 0, (float(over.max()), float(want.abs().max()))


SIZES = [(1, 1, 1), (1, 128, 128), (2, 100, 5), (1, 4096, 1000), (3, 25088, 300), (16, 1000, 4096), (17, 640, 33), (31, 3000, 100), (32, 2048, 512),
         (33, 1100, 129), (64, 5000, 64), (100, 4096, 700), (128, 128, 128), (127, 257, 129), (256, 12544, 256), (256, 640, 512), (300, 1024, 300),
         (513, 512, 257), (1000, 384, 1000), (1985, 1100, 333), (2048, 896, 2048), (2304, 640, 2300), (4097, 256, 260), (5000, 130, 3), (7, 130, 5000),
         (24, 25088, 300), (40, 25088, 300), (300, 12544, 200), (90, 12800, 1900), (700, 12800, 1900), (2500, 25088, 2500),      # K slices of each kind
         (2304, 100, 2300), (2500, 1000, 2450), (2561, 129, 2000),                     # 256 x 128 tiles: one block, several, ragged edges
         (3000, 100, 3000), (3001, 256, 2901), (3000, 385, 3000), (4352, 700, 4500), (2816, 2048, 3328)]   # 256 x 256 tiles


@pytest.mark.parametrize('out', [F32, F16, BF16])
@pytest.mark.parametrize('M,K,N', SIZES)
def test_product(M, K, N, out):
    from sgg_amd import ops
    A, W = ops.quantize_fp8(rand(M, K, F32, M, 1.0)), ops.quantize_fp8(rand(N, K, F32, N + 1, 1.0, K ** -0.5))
    bias = torch.randn(N, device=DEV)
    for b, relu in ((None, False), (bias, True)):
        y = ops.gemm_fp8(A, W, b, ops.ACT_RELU if relu else ops.ACT_NONE, out_dtype=out)
        assert y.dtype == out and y.shape == (M, N)
        check(y, *product(A, W, b, relu, out))
        assert torch.equal(y, ops.gemm_fp8(A, W, b, ops.ACT_RELU if relu else ops.ACT_NONE, out_dtype=out))      # same bits every time


@pytest.mark.parametrize('M,K,N,ld', [(5, 300, 70, 75), (200, 256, 130, 137), (600, 384, 600, 640)])
def test_product_into_a_strided_buffer_leaves_the_rest(M, K, N, ld):
    from sgg_amd import ops
    A, W = ops.quantize_fp8(rand(M, K, F16, 1, 1.0)), ops.quantize_fp8(rand(N, K, F16, 2, 1.0))
    for dtype in (F32, F16, BF16):
        buf = torch.full((M + 2, ld), 9.0, dtype=dtype, device=DEV)
        ops.gemm_fp8(A, W, out=buf[1:M + 1, 3:3 + N])
        check(buf[1:M + 1, 3:3 + N], *product(A, W, dtype=dtype))
        assert bool((buf[0] == 9).all()) and bool((buf[M + 1] == 9).all()) and bool((buf[:, :3] == 9).all()) and bool((buf[:, 3 + N:] == 9).all())


@pytest.mark.parametrize('M,N', [(4, 64), (20, 64), (100, 64), (4096, 2048), (4096, 4096)])
def test_operands_near_the_smallest(M, N):
    """one product per output: exact down to operands of 2^-133 (bf16's smallest), below that exact or zero"""
    from sgg_amd import ops
    e = -(112 + torch.arange(N, device=DEV) % 24)                        # down to 2^-135 = e4m3's smallest times the smallest scale
    x, w = torch.zeros(M, 128, device=DEV), torch.zeros(N, 128, device=DEV)
    x[:, 0] = 2.0 ** 118
    w[:, 0] = ((e.clamp(min=-126).int() + 127) << 23).view(torch.float32)
    w[:, 0] *= ((e - e.clamp(min=-126) + 127).int() << 23).view(torch.float32)
    A, W = ops.quantize_fp8(x), ops.quantize_fp8(w)
    want = (A.dequantize()[:1, :1] * W.dequantize()[:, :1].t())
    assert torch.equal(want[0], ((e.long() + 118 + 1023) << 52).view(torch.float64))
    for out in (F32, F16, BF16):
        y = ops.gemm_fp8(A, W, out_dtype=out)
        exact, low = want.to(out).expand(M, N), e < -133
        assert torch.equal(y[:, ~low], exact[:, ~low])
        assert bool(((y[:, low] == exact[:, low]) | (y[:, low] == 0)).all())


@pytest.mark.parametrize('M', [3, 20, 100, 250, 600])
def test_operands_past_4_gigabytes(M):
    """W's codes are 4.4 GB (and its f16 source 8.8): a few rows that hold something, the last ones among them"""
    from sgg_amd import ops
    N, K = 40001, 110100
    g = torch.Generator(device=DEV).manual_seed(M)
    at = torch.tensor([0, 1, 127, 20000, N - 129, N - 2, N - 1], device=DEV)
    some = (torch.randn(7, K, generator=g, device=DEV) / 300).half()
    w = torch.zeros(N, K, dtype=F16, device=DEV)
    w[at] = some
    W = ops.quantize_fp8(w)
    del w
    A = ops.quantize_fp8(torch.randn(M, K, generator=g, device=DEV))
    few = ops.quantize_fp8(some)
    for out in (F32, F16):
        y = ops.gemm_fp8(A, W, out_dtype=out)
        check(y[:, at], *product(A, few, dtype=out))
        y[:, at] = 0
        assert not y.any()
    del W
    torch.cuda.empty_cache()


def test_scales_far_apart_and_zero_operands():
    """blocks of one row 2^60 apart, rows of zeros, a whole zero operand"""
    from sgg_amd import ops
    x, w = rand(300, 512, F32, 3, 1.0), rand(280, 512, F32, 4, 1.0)
    x[:, 128:256] *= 2.0 ** 40
    x[:, 256:384] *= 2.0 ** -60
    w[:, 128:256] *= 2.0 ** -45
    x[7] = 0
    w[11] = 0
    A, W = ops.quantize_fp8(x), ops.quantize_fp8(w)
    y = ops.gemm_fp8(A, W)
    check(y, *product(A, W))
    assert not y[7].any() and not y[:, 11].any()
    assert not ops.gemm_fp8(ops.quantize_fp8(torch.zeros_like(x)), W).any()


@pytest.mark.parametrize('M,K,N', [(1, 300, 40), (20, 1000, 70), (200, 300, 300), (600, 512, 600)])
def test_nan_reaches_its_own_outputs_only(M, K, N):
    from sgg_amd import ops
    x, w = rand(M, K, F32, 5, 1.0), rand(N, K, F32, 6, 1.0)
    x[M // 2, K - 1] = float('inf')
    w[N // 3, 0] = float('nan')
    for act in (ops.ACT_NONE, ops.ACT_RELU):
        bad = ops.gemm_fp8(ops.quantize_fp8(x), ops.quantize_fp8(w), act=act).isnan()
        want = torch.zeros_like(bad)
        want[M // 2], want[:, N // 3] = True, True
        assert torch.equal(bad, want)


def quant(x):
    return grid(x.contiguous())[0]


@pytest.mark.parametrize('M,K,N', [(1, 5, 3), (37, 29, 13), (300, 216, 64), (700, 663, 129)])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_affine_forward_and_gradients(M, K, N, dtype):
    """y, dx, dw, db against the formulas on 64-bit quantised operands"""
    from sgg_amd import dense
    torch.manual_seed(M)
    x = rand(M, K, dtype, 1, 1.0).requires_grad_()
    w = rand(N, K, F32, 2, 1.0, K ** -0.5).requires_grad_()
    b = torch.randn(N, device=DEV, requires_grad=True)
    y = dense.affine_fp8(x, w, b)
    assert y.dtype == dtype
    dy = rand(M, N, dtype, 3, 1.0)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xd, wd = x.detach(), w.detach()

    def mm(p, q, dtype=dtype):
        tol = (p.shape[1] + 32) * U * torch.mm(p.abs(), q.abs().t().contiguous())
        return torch.mm(p, q.t().contiguous()), tol if dtype == F32 else tol + cut(p, q)
    want, tol = mm(quant(xd), quant(wd))
    check(y.detach(), want + b.detach().double(), tol + 2 * U * b.detach().abs())
    check(dx, *mm(quant(dy), quant(wd.t())))
    check(dw, *mm(quant(dy.t()), quant(xd.t()), F32))
    check(db, dy.double().sum(0), (M + 4) * U * dy.double().abs().sum(0))
    assert dx.dtype == dtype and dw.dtype == F32 and db.dtype == F32
    # only what is asked for is computed, and it is the same
    y2 = dense.affine_fp8(x.detach(), w, None)
    assert torch.equal(torch.autograd.grad(y2, w, dy)[0], dw)
    y3 = dense.affine_fp8(x, w.detach(), b.detach())
    assert torch.equal(torch.autograd.grad(y3, x, dy)[0], dx)
    assert torch.equal(dense.affine_fp8(x.detach().view(1, M, K), w.detach(), b.detach(), out_dtype=dtype).view(M, N), y.detach())
    with torch.no_grad():
        assert torch.equal(dense.affine_fp8(x, w, b), y)
    # a gradient that autograd hands over as one broadcast number, transposed weights, strided inputs
    ys = dense.affine_fp8(x, w.t().contiguous().t(), b)
    assert torch.equal(ys, y)
    gs = torch.autograd.grad(ys.sum(), (x, w, b))
    gf = torch.autograd.grad(dense.affine_fp8(x, w, b), (x, w, b), torch.ones_like(dy))
    assert all(torch.equal(p, q) for p, q in zip(gs, gf))


def test_relative_error_against_the_unquantised_product():
    """each operand value is off by at most 2^-4 of itself (2^-10 of its block's scale below that): the product by at most the sum of both"""
    from sgg_amd import dense
    x, w = rand(200, 600, F32, 1, 0.5), rand(90, 600, F32, 2, 0.5)
    y = dense.affine_fp8(x, w).double()
    a, c = x.double(), w.double()
    want = torch.mm(a, c.t().contiguous())
    e = 2.0 ** -4
    floor_x, floor_w = 2.0 ** -10 * two(grid(x)[1]).amax(1, keepdim=True), 2.0 ** -10 * two(grid(w)[1]).amax(1, keepdim=True)
    ex, ew = (e * a.abs()).clamp(min=0) + floor_x, e * c.abs() + floor_w
    bound = torch.mm(ex, c.abs().t().contiguous()) + torch.mm(a.abs() + ex, ew.t().contiguous())
    assert float(((y - want).abs() - bound * (1 + 1e-4)).max()) <= 0


def test_dense_layers_in_the_fp8_arithmetic():
    """set_compute('fp8'): Linear and Conv2d forward and backward against the same layers built from 64-bit quantised products"""
    from sgg_amd import dense
    torch.manual_seed(0)
    conv = dense.Conv2d(9, 12, 3, padding=1).to(DEV)
    lin = dense.Linear(12, 7).to(DEV)
    x = torch.randn(2, 6, 5, 9, device=DEV, requires_grad=True)
    prev = dense.set_compute('fp8')
    try:
        h = conv(x)
        y = lin(h)
        dy = torch.randn_like(y)
        grads = torch.autograd.grad(y, (x, conv.weight, conv.bias, lin.weight, lin.bias), dy, retain_graph=True)
        dh = torch.autograd.grad(y, h, dy)[0]
        assert torch.equal(dense.product(x.detach().reshape(-1, 9), lin.weight.detach()[:, :9].contiguous()).isfinite().all(), torch.tensor(True, device=DEV))
    finally:
        dense.set_compute(prev)
    cols = torch.nn.functional.unfold(x.detach().permute(0, 3, 1, 2), 3, padding=1)                      # [B, C*9, L], (c, ky, kx)
    cols = cols.view(2, 9, 9, 30).permute(0, 3, 2, 1).reshape(60, 81)                                     # rows, (ky, kx, c)
    cols = torch.nn.functional.pad(cols, (0, 15))
    wm = torch.nn.functional.pad(conv.weight.detach().permute(0, 2, 3, 1).reshape(12, 81), (0, 15))
    hq = torch.mm(quant(cols), quant(wm).t().contiguous()) + conv.bias.detach().double()
    assert float((h.detach().reshape(60, 12).double() - hq).abs().max()) <= 200 * U * float(hq.abs().max() + 10)
    dhm, dym = dh.reshape(60, 12), dy.reshape(60, 7)
    dw = torch.mm(quant(dhm.t()), quant(cols.t()).t().contiguous())[:, :81].view(12, 3, 3, 9).permute(0, 3, 1, 2)
    assert float((grads[1].double() - dw).abs().max()) <= 200 * U * float(dhm.abs().sum(0).max() * cols.abs().max())
    dl = torch.mm(quant(dym.t()), quant(h.detach().reshape(60, 12).t()).t().contiguous())
    assert float((grads[3].double() - dl).abs().max()) <= 200 * U * float((dym.abs().sum(0).max() * h.abs().max()).detach())
    assert grads[0].shape == x.shape and grads[2].shape == (12,) and grads[4].shape == (7,)


def test_empty_batches():
    from sgg_amd import dense, ops
    w = torch.randn(5, 40, device=DEV, requires_grad=True)
    b = torch.randn(5, device=DEV, requires_grad=True)
    x = torch.zeros(0, 40, device=DEV, requires_grad=True)
    y = dense.affine_fp8(x, w, b)
    assert y.shape == (0, 5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 5, device=DEV))
    assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == (5, 40)
    y = ops.gemm_fp8(ops.quantize_fp8(torch.zeros(3, 0, device=DEV)), ops.quantize_fp8(torch.zeros(5, 0, device=DEV)), b.detach())
    assert torch.equal(y, b.detach().expand(3, 5))                                                        # an empty reduction: the bias
    assert ops.gemm_fp8(ops.quantize_fp8(torch.zeros(3, 8, device=DEV)), ops.quantize_fp8(torch.zeros(0, 8, device=DEV))).shape == (3, 0)


def test_replayed_graphs_and_another_stream():
    from sgg_amd import ops
    w = ops.quantize_fp8(rand(600, 2000, F32, 1, 1.0))
    xs = [rand(m, 2000, F16, m, 1.0) for m in (1, 40, 256)]

    def step():
        return [ops.gemm_fp8(ops.quantize_fp8(x), w, act=ops.ACT_RELU) for x in xs]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(side, step()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        for x in xs:
            x.copy_(rand(x.shape[0], 2000, F16, 50 + k, 1.0))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_a_training_step_of_all_three_together():
    """normalise -> multiply in 8 bits -> ReLU -> multiply -> backward -> unscale and clip -> an optimiser that is not FusedSGD: the gradients
    the optimiser sees are the layers' own, clipped"""
    from sgg_amd import dense
    from sgg_amd.gan_ops import build_mlp
    from sgg_amd.trainer import clip_grad_norm_
    torch.manual_seed(3)
    net = build_mlp([70, 96, 50], batch_norm='layer').to(DEV)
    opt = torch.optim.Adam(net.parameters(), lr=1e-3)
    x, t = torch.randn(230, 70, device=DEV), torch.randn(230, 50, device=DEV)
    prev = dense.set_compute('fp8')
    try:
        for step in range(2):
            opt.zero_grad()
            ((net(x) - t).square().mean() * 64.0).backward()
            raw = [p.grad.double().clone() for p in net.parameters()]
            norm = clip_grad_norm_(net.parameters(), 0.01, grad_scale=1.0 / 64)
            want = sum(g.square().sum() for g in raw).sqrt() / 64
            assert abs(float(norm.double() - want)) <= 2 * U * float(want)
            for p, g in zip(net.parameters(), raw):
                assert float((p.grad.double() - g / 64 * min(1.0, 0.01 / (float(want) + 1e-6))).abs().max()) <= 4 * U * float(g.abs().max())
            before = [p.detach().clone() for p in net.parameters()]
            opt.step()
            assert all(not torch.equal(a, p.detach()) for a, p in zip(before, net.parameters()))
    finally:
        dense.set_compute(prev)


def test_refusals():
    from sgg_amd import dense, ops
    x = torch.randn(4, 256, device=DEV)
    A = ops.quantize_fp8(x)
    with pytest.raises(ValueError):
        ops.quantize_fp8(x, 'diagonal')
    with pytest.raises(ValueError):
        ops.quantize_fp8(x.t())
    with pytest.raises(ValueError):
        ops.quantize_fp8(x[0])
    with pytest.raises(TypeError):
        ops.quantize_fp8(x.double())
    with pytest.raises(RuntimeError):
        ops.quantize_fp8(x.cpu())
    with pytest.raises(TypeError):
        ops.gemm_fp8(x, A)
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, ops.quantize_fp8(x[:, :255]))                     # same padded width, another reduction
    for bad in (ops.Fp8Rows(A.data[:3], A.scale, (4, 256)), ops.Fp8Rows(A.data, A.scale[:100], (4, 256)), ops.Fp8Rows(A.data, A.scale, (4, 300)), ops.Fp8Rows(A.codes(), A.scale, (4, 256)),
                ops.Fp8Rows(A.data.view(torch.uint8), A.scale, (4, 256))):
        with pytest.raises(ValueError):                                   # an operand whose memory is not its shape's
            ops.gemm_fp8(bad, bad)
    by_hand = ops.Fp8Rows(A.data, A.scale, A.shape)
    assert torch.equal(ops.gemm_fp8(by_hand, A), ops.gemm_fp8(A, by_hand))
    A.shape = (1000, 256)
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, A)
    A.shape = (4, 256)
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, A, torch.zeros(5, device=DEV))
    with pytest.raises(TypeError):
        ops.gemm_fp8(A, A, torch.zeros(4, device=DEV).half())
    with pytest.raises(TypeError):
        ops.gemm_fp8(A, A, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, A, out=torch.empty(4, 5, device=DEV))
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, A, out=torch.empty(4, 4, device=DEV).t())
    with pytest.raises(ValueError):
        ops.gemm_fp8(A, A, act=7)
    with pytest.raises(ValueError):
        dense.affine_fp8(x, torch.zeros(3, 255, device=DEV))
    with pytest.raises(RuntimeError):
        dense.affine_fp8(x.cpu(), torch.zeros(3, 256))
