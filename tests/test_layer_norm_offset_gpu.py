"""Layer normalisation of rows whose mean is far larger than their spread, and constant rows, against the formulas in 64 bits.

Tolerances.  u = 2^-24.  The mean is summed in 64 bits: off by C 2^-53 max|x| (16-bit values within a factor 4 in fp32, where their sum is whole; else by
16 u max|x|); x - mean is rounded twice.  The variance's sum takes at most C/64 + 16 = k
steps.  So xh is off by 2 k u |xh| + r C 2^-53 max|x| -- nothing here grows with r max|x| u, an fp32 mean's error.  The backward centres
u = (x - m) r, m the mean as one float, by the fp32 mean a of u, |a| <= r u |m|: off by 2 k u (|xh| + mean|xh| + r u |m|)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24


def reference(x, w, b, dy, eps):
    """(y, dx, dw, db) and their tolerances"""
    narrow = x.dtype != torch.float32
    x, dy, w, b = x.double(), dy.double(), w.double(), b.double()
    M, C = x.shape
    mu = x.sum(1, keepdim=True) / C
    r = (((x - mu) ** 2).sum(1, keepdim=True) / C + eps) ** -0.5
    xh = (x - mu) * r
    g = dy * w
    m1, m2 = g.sum(1, keepdim=True) / C, (g * xh).sum(1, keepdim=True) / C
    k = C / 64 + 16
    big = x.abs().amax(1, keepdim=True)
    far = r * C * 2.0 ** -53 * big
    if narrow:
        far = far + torch.where(x.abs().amin(1, keepdim=True) * 4 <= big, r * 16 * U * big, torch.zeros_like(r))
    e_y = 2 * k * U * xh.abs() + far
    left = r * U * mu.abs()                                                # |a| at most
    e_xh = 2 * k * U * (xh.abs() + xh.abs().mean(1, keepdim=True) + left) + far
    gm = g.abs().mean(1, keepdim=True)
    e_m2 = 2 * k * U * (g.abs() * (xh.abs() + left)).mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    y, dx = xh * w + b, r * (g - m1 - xh * m2)
    t_y = w.abs() * e_y + 4 * U * (y.abs() + b.abs())
    t_dx = r * (2 * k * U * (g.abs() + gm + (xh * m2).abs()) + 2 * k * U * (g.abs() + gm) + xh.abs() * e_m2 + e_xh * m2.abs() + 4 * U * (xh * m2).abs())
    t_dw = (M + 4) * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    return (y, dx, (dy * xh).sum(0), dy.sum(0)), (t_y, t_dx, t_dw, (M + 4) * U * dy.abs().sum(0))


def check(got, want, tol, name):
    t = torch.finfo(got.dtype)
    over = (got.double() - want).abs() - (tol + t.eps / 2 * want.abs() + t.tiny)
    assert bool((over <= 0).all()), (name, float(over.max()), float(want.abs().max()))


def held(x, w, b, dy):
    from sgg_amd import ops
    want, tol = reference(x, w, b, dy, 1e-5)
    y, mean, rstd = ops.layer_norm(x, w, b)
    got = (y,) + ops.layer_norm_bwd(dy, x, mean, rstd, w)
    for p in zip(got, want, tol, ('y', 'dx', 'dw', 'db')):
        check(*p)
    none, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dx=False)
    assert torch.equal(dw, got[2]) and torch.equal(db, got[3])
    dx, none, none = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dw=False, want_db=False)
    assert torch.equal(dx, got[1])


def vectors(M, C, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)                # noqa: E731
    return rand(M, C), 1 + 0.3 * rand(C), 0.3 * rand(C), rand(M, C).to(dtype)


WIDTHS = [1, 2, 41, 64, 100, 200, 300, 512, 1001, 2049, 4096, 5000, 12345, 16384]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('C', WIDTHS)
def test_constant_rows_give_the_bias(C, dtype):
    """the sum of C equal floats is exact in 64 bits, its quotient the float itself: x - mean is 0, y the bias to the bit, dx r (g - mean g)"""
    from sgg_amd import ops
    c = torch.tensor([5.0, 1000.3, 12345.6, 100000.5, 1e6, -7.7e8, 3e-20] if dtype == torch.float32 else [5.0, -1000.3, 31000.0, 3e-4], device=DEV)
    x = c[:, None].expand(-1, C).contiguous().to(dtype)
    _, w, b, dy = vectors(len(c), C, dtype, C)
    y, mean, rstd = ops.layer_norm(x, w, b)
    assert torch.equal(y, b.to(dtype).expand(len(c), C)) and torch.equal(mean, x[:, 0].float())
    held(x, w, b, dy)


@pytest.mark.parametrize('dtype,offset,spread', [(torch.float32, 1e4, 1.0), (torch.float32, -3e4, 0.1), (torch.float32, 1e6, 1.0), (torch.float32, 1e8, 1e3),
                                                 (torch.float16, 3e4, 50.0), (torch.bfloat16, -1e4, 200.0), (torch.bfloat16, 1e30, 1e28)])
@pytest.mark.parametrize('C', WIDTHS)
def test_rows_far_from_zero(C, dtype, offset, spread):
    x, w, b, dy = vectors(33, C, dtype, C)
    held((x * spread + offset * (1 + torch.arange(33, device=DEV)[:, None] / 64)).to(dtype), w, b, dy)


@pytest.mark.parametrize('C', WIDTHS[1:])
def test_two_neighbouring_floats(C):
    """a row of c and the next float after it: a mean that no float holds, a spread of half a step"""
    x, w, b, dy = vectors(5, C, torch.float32, C)
    c = torch.tensor([1e3, -1e4, 1e6, 3.3e7, 1.0], device=DEV)[:, None]
    held(torch.where(x > 0, c, torch.nextafter(c, torch.full_like(c, 1e30))), w, b, dy)


@pytest.mark.parametrize('C', [40, 300, 1000, 1100, 2049, 5000, 9000])
def test_a_rows_result_does_not_hang_on_its_neighbours(C):
    """many rows per workgroup, one after the other: each gets the bits that it gets alone"""
    from sgg_amd import ops
    x, w, b, dy = vectors(2500, C, torch.float16, 1)
    x = (x * 3 + 100).half()
    y, mean, rstd = ops.layer_norm(x, w, b)
    dx = ops.layer_norm_bwd(dy, x, mean, rstd, w)[0]
    at = torch.tensor([0, 1, 255, 256, 257, 1023, 1024, 1800, 2498, 2499], device=DEV)
    ya, ma, ra = ops.layer_norm(x[at], w, b)
    assert torch.equal(ya, y[at]) and torch.equal(ma, mean[at]) and torch.equal(ra, rstd[at])
    assert torch.equal(ops.layer_norm_bwd(dy[at], x[at], ma, ra, w, want_dw=False, want_db=False)[0], dx[at])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('C', [40, 300, 1000, 1500, 2048, 4000, 9000])
def test_differences_whose_squares_pass_fp32(C, dtype):
    """every third row 1e25 times the others: their variance is past 3.4e38, their normalised values are not"""
    from sgg_amd import ops
    x, w, b, dy = vectors(700, C, dtype, 2)
    x[::3] *= 1e25
    x[600:] = x[600:].abs()                                                 # (and a last run of rows without one, and with ordinary signs)
    x = x.to(dtype)
    held(x, w, b, dy)
    y = ops.layer_norm(x, w, b)[0]
    assert torch.equal(ops.layer_norm(x[5:40], w, b)[0], y[5:40])


def test_a_weight_changed_between_forward_and_backward_is_refused():
    """another type, another device or fewer columns behind the saved parameter: an error, no launch; an in-place change is autograd's own"""
    from sgg_amd import dense
    x = torch.randn(30, 64, device=DEV, requires_grad=True)
    for change, error in ((lambda w: w.half(), TypeError), (lambda w: w.cpu(), RuntimeError), (lambda w: w[:32].clone(), ValueError),
                          (lambda w: w.expand(2, 64), ValueError)):
        m = dense.LayerNormRows(64).to(DEV)
        y = m(x)
        m.weight.data = change(m.weight.data)
        with pytest.raises(error):
            y.sum().backward()
    m = dense.LayerNormRows(64).to(DEV)
    y = m(x)
    with torch.no_grad():
        m.weight.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
