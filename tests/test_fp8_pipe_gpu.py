"""16-bit results of the 8-bit products (more than 32 rows: the 8-bit matrix instructions) and, where the same can be asked of them, fp32 ones: exact
where nothing can be cut, NaN and infinities, scales far apart, and random operands within tests/fp8_bounds.py."""
import pytest
import torch

from .fp8_bounds import inside

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

#  M, K, N: 128 x 128 tiles whole and in 8 .. 18 K slices; 256 x 128 whole and in slices; 256 x 256 whole and in slices; blocks in odd numbers, ragged ends
SHAPES = [(33, 1100, 129), (100, 640, 130), (64, 5000, 64), (128, 4096, 700), (300, 12544, 200), (40, 25088, 300), (90, 12800, 1900), (2304, 640, 2300),
          (2561, 129, 2000), (700, 12800, 1900), (512, 7936, 4608), (3000, 385, 3000), (2816, 2048, 3328), (2500, 25088, 2500)]


def same(got, want):
    a, b = got.double(), want.to(got.dtype).double()
    assert torch.equal(a, b), (int((a != b).sum()), float((a - b).abs().nan_to_num(0.0).max()))


def spread_exponents(rows, blocks, lo, n, s, t):
    return lo + (s * torch.arange(rows, device=DEV)[:, None] + t * torch.arange(blocks, device=DEV)[None, :]) % n


def wide(e, K):
    return torch.exp2(e.double()).repeat_interleave(128, 1)[:, :K]


def operands(a, w):
    from sgg_amd import ops
    A, W = ops.quantize_fp8(a), ops.quantize_fp8(w)
    assert torch.equal(A.dequantize(), a.double()) and torch.equal(W.dequantize(), w.double())       # what is multiplied is what was asked for
    return A, W


@pytest.mark.parametrize('M,K,N', SHAPES)
def test_small_integers_are_exact(M, K, N):
    """values -2 .. 2 times scales 1, 2, 4, 8 of their row and block: products of a block lie within a factor 4, every sum below 2^24: nothing is cut,
    nothing rounds before the output does"""
    from sgg_amd import ops
    g = torch.Generator(device=DEV).manual_seed(M + K)
    blocks = (K + 127) // 128
    a = torch.randint(-2, 3, (M, K), generator=g, device=DEV) * wide(spread_exponents(M, blocks, 0, 4, 1, 3), K)
    w = torch.randint(-2, 3, (N, K), generator=g, device=DEV) * wide(spread_exponents(N, blocks, 0, 4, 3, 1), K)
    A, W = operands(a.float(), w.float())
    want = torch.mm(a, w.t().contiguous())
    for out in (F16, BF16, F32):
        same(ops.gemm_fp8(A, W, out_dtype=out), want)


@pytest.mark.parametrize('M,K,N', SHAPES)
def test_one_product_per_output_in_every_block(M, K, N):
    """one element per row of A, in turn in each block of K (the last one and every K slice's first and last among them); powers of two that differ by
    row, block and side pick every byte of the scale words: the product itself, to the bit"""
    from sgg_amd import ops
    blocks = (K + 127) // 128
    m = torch.arange(M, device=DEV)
    frac = 1 + (torch.arange(N, device=DEV)[:, None] + torch.arange(K, device=DEV)[None, :]) % 8 / 8.0
    for far in (5, 40):                                                  # f16 holds the first kind; the second kind bf16 and fp32
        w = frac * wide(spread_exponents(N, blocks, -far, 2 * far + 1, 5, 3), K)
        ea = -(far // 2) + (7 * m) % (far + 1)
        for p in range(-(-blocks // M)):
            k = ((m + p * M) % blocks * 128 + (37 * m) % 128).clamp(max=K - 1)
            a = torch.zeros(M, K, dtype=torch.float64, device=DEV)
            a[m, k] = torch.exp2(ea.double())
            A, W = operands(a.float(), w.float())
            want = torch.exp2(ea.double())[:, None] * w.t()[k]
            for out in (F16, BF16, F32) if far == 5 else (BF16, F32):
                same(ops.gemm_fp8(A, W, out_dtype=out), want)


@pytest.mark.parametrize('out', [F16, BF16, F32])
@pytest.mark.parametrize('M,K,N', [(40, 300, 140), (64, 5000, 64), (200, 300, 300), (2304, 200, 2300), (700, 12800, 1900), (3000, 200, 3000)])
def test_nan_and_infinity_reach_their_own_outputs_only(M, K, N, out):
    from sgg_amd import ops
    g = torch.Generator(device=DEV).manual_seed(5)
    x, w = torch.randn(M, K, generator=g, device=DEV), torch.randn(N, K, generator=g, device=DEV)
    x[M // 2, K - 1], x[M - 1, 0] = float('inf'), float('nan')
    w[N // 3, K // 2] = float('-inf')
    clean = ops.gemm_fp8(ops.quantize_fp8(x.nan_to_num(0.0, 0.0, 0.0)), ops.quantize_fp8(w.nan_to_num(0.0, 0.0, 0.0)), out_dtype=out)
    y = ops.gemm_fp8(ops.quantize_fp8(x), ops.quantize_fp8(w), out_dtype=out)
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[M // 2], bad[M - 1], bad[:, N // 3] = True, True, True
    assert torch.equal(y.isnan(), bad)
    assert torch.equal(y[~bad], clean[~bad])


def held(x, w, outs=(F16, BF16)):
    from sgg_amd import ops
    A, W = ops.quantize_fp8(x), ops.quantize_fp8(w)
    a, b = A.dequantize(), W.dequantize()
    for out in outs:
        ok, share = inside(ops.gemm_fp8(A, W, out_dtype=out), a, A.exponents(), b, W.exponents())
        assert ok, (out, share)


@pytest.mark.parametrize('spread', [0.0, 1.0, 3.0])
@pytest.mark.parametrize('M,K,N', SHAPES)
def test_random_operands(M, K, N, spread):
    g = torch.Generator(device=DEV).manual_seed(M + K + N)
    x, w = (torch.randn(r, K, generator=g, device=DEV) * torch.exp2(spread * torch.randn(r, K, generator=g, device=DEV)) for r in (M, N))
    held(x, w / K ** 0.5)
    if spread == 0.0:
        held(x.clamp(min=0), w / K ** 0.5)                              # behind a ReLU: half of the codes are zeros


@pytest.mark.parametrize('M,K,N', [(300, 512, 280), (64, 5000, 64), (2304, 640, 2300), (700, 12800, 1900), (3000, 512, 3000)])
def test_scales_far_apart(M, K, N):
    """blocks of one row 2^100 apart (bf16 holds what comes of them), rows of zeros"""
    from sgg_amd import ops
    g = torch.Generator(device=DEV).manual_seed(3)
    x, w = torch.randn(M, K, generator=g, device=DEV), torch.randn(N, K, generator=g, device=DEV)
    x[:, 128:256] *= 2.0 ** 40
    x[:, 256:384] *= 2.0 ** -60
    w[:, 128:256] *= 2.0 ** -45
    x[7], w[11] = 0, 0
    held(x, w, (BF16,))
    held(x * 2.0 ** -20, w * 2.0 ** 20, (BF16, F16))
    y = ops.gemm_fp8(ops.quantize_fp8(x), ops.quantize_fp8(w), out_dtype=BF16)
    assert not y[7].any() and not y[:, 11].any()


@pytest.mark.parametrize('M', [33, 300, 2304])
def test_the_cut_is_what_the_header_says(M):
    """a product 2^-13 of the largest among its 8 columns counts, one of 2^-14 does not, one a group further counts at 2^-14 too; up to 32 rows and fp32
    outputs lose none of them"""
    from sgg_amd import ops
    x, w = torch.zeros(M, 384, device=DEV), torch.ones(M, 384, device=DEV)
    x[:, 0], x[:, 256] = 256.0, -256.0
    rows = torch.arange(M, device=DEV)
    at = 1 + rows % 12
    for small, lost in ((2.0 ** -5, False), (2.0 ** -6, True)):
        x[:, 1:128] = 0
        x[rows, at] = small
        A, W = operands(x, w)
        want = torch.full((M, M), small, dtype=torch.float64, device=DEV)
        same(ops.gemm_fp8(A, W), want)
        few = ops.quantize_fp8(x[:32])
        same(ops.gemm_fp8(few, W, out_dtype=BF16), want[:32])
        want[at < 8] = 0.0 if lost else small
        same(ops.gemm_fp8(A, W, out_dtype=BF16), want)


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('M,K,N', [(300, 216, 64), (700, 663, 129), (1985, 1100, 333)])
def test_gradients_of_16_bit_activations(M, K, N, dtype):
    """y and dx of affine_fp8 come from the 8-bit pipe, dw from fp32 sums"""
    from sgg_amd import dense, ops
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(N, K, generator=g, device=DEV) / K ** 0.5).requires_grad_()
    dy = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    y = dense.affine_fp8(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    form = lambda t: ops.quantize_fp8(t.detach().contiguous())                                   # noqa: E731
    for got, p, q in ((y.detach(), form(x), form(w)), (dx, form(dy), form(w.t()))):
        ok, share = inside(got, p.dequantize(), p.exponents(), q.dequantize(), q.exponents())
        assert ok, share
    p, q = form(dy.t()).dequantize(), form(x.t()).dequantize()
    tol = (M + 32) * 2.0 ** -24 * torch.mm(p.abs(), q.abs().t().contiguous())
    assert bool(((dw.double() - torch.mm(p, q.t().contiguous())).abs() <= tol + 1e-30).all())
