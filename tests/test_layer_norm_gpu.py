"""Layer normalisation (csrc/layernorm.hip) against the formulas in 64 bits: forward, gradients, row strides, odd widths, empty batches.

Tolerances.  u = 2^-24 is fp32's half step.  A row's sums are added in at most C/64 + 16 steps, so mean and variance are off by at most
k u relative to the largest magnitude, k = C/64 + 16; xh = (x - mu) r is then off by 2 k u (r max|x| + |xh|), y by |w| times that plus its own
half step.  dx adds the two row means of g and g xh (k u of their magnitudes' means) and the error of xh in each.  A column sum over M
rows is off by at most M u times the sum of its terms' magnitudes plus the terms' own errors."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def make(M, C, dtype, seed, offset=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(M, C, generator=g, device=DEV) + offset * torch.randn(M, 1, generator=g, device=DEV)
    w = 1 + 0.3 * torch.randn(C, generator=g, device=DEV)
    b = 0.3 * torch.randn(C, generator=g, device=DEV)
    dy = torch.randn(M, C, generator=g, device=DEV)
    return x.to(dtype), w, b, dy.to(dtype)


def reference(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    C = x.shape[1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    mu = x.sum(1, keepdim=True) / C
    var = ((x - mu) ** 2).sum(1, keepdim=True) / C
    r = (var + eps) ** -0.5
    xh = (x - mu) * r
    y = xh * w + (0 if b is None else b.double())
    g = dy * w
    m1, m2 = g.sum(1, keepdim=True) / C, (g * xh).sum(1, keepdim=True) / C
    dx = r * (g - m1 - xh * m2)
    k = C / 64 + 16
    big = x.abs().amax(1, keepdim=True)
    e_xh = 2 * k * U * (r * big + xh.abs())
    e_r = 2 * k * U * (1 + (r * big) ** 2 * U * k)
    gm = g.abs().mean(1, keepdim=True)
    ghm = (g * xh).abs().mean(1, keepdim=True)
    e_m2 = k * U * ghm + (g.abs() * e_xh).mean(1, keepdim=True)
    t_y = w.abs() * e_xh + 4 * U * y.abs()
    t_dx = r * (e_r * (g.abs() + gm + (xh * m2).abs()) + 2 * k * U * (g.abs() + gm) + xh.abs() * e_m2 + e_xh * m2.abs() + 4 * U * (xh * m2).abs())
    M = x.shape[0]
    t_dw = (M + 4) * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    t_db = (M + 4) * U * dy.abs().sum(0)
    return (y, dx, (dy * xh).sum(0), dy.sum(0)), (t_y, t_dx, t_dw, t_db)


def check(got, want, tol, name):
    slack = tol + half(got.dtype) * want.abs() + torch.finfo(got.dtype).tiny       # (f16: a subnormal's step is below tiny)
    over = (got.double() - want).abs() - slack
    assert bool((over <= 0).all()), (name, float(over.max()), float(want.abs().max()))


SHAPES = [(1, 1), (1, 512), (3, 2), (5, 63), (7, 64), (33, 65), (64, 200), (130, 511), (257, 1001), (1000, 512), (9, 2048), (4, 2049),
          (40, 4096), (3, 5000), (6, 8192), (2, 12345), (5, 16384), (2049, 40)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,C', SHAPES)
def test_forward_and_gradients(M, C, dtype):
    from sgg_amd import ops
    x, w, b, dy = make(M, C, dtype, M * 7 + C)
    (ry, rdx, rdw, rdb), (ty, tdx, tdw, tdb) = reference(x, w, b, dy, 1e-5)
    y, mean, rstd = ops.layer_norm(x, w, b)
    assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
    check(y, ry, ty, 'y')
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    assert dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
    check(dx, rdx, tdx, 'dx')
    check(dw, rdw, tdw, 'dw')
    check(db, rdb, tdb, 'db')
    y2, none, none2 = ops.layer_norm(x, w, b, stats=False)
    assert none is None and none2 is None and torch.equal(y, y2)
    again = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(torch.equal(a, c) for a, c in zip((dx, dw, db), again))          # fixed order of every sum


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('M,C,ld,off', [(50, 96, 100, 0), (50, 97, 101, 3), (9, 512, 513, 1), (70, 40, 47, 5), (6, 4000, 4097, 9)])
def test_strided_rows_at_any_alignment(M, C, ld, off, dtype):
    """views into wider buffers: row strides and starts that no vector load is aligned to; what lies between the rows is not touched"""
    from sgg_amd import ops
    x, w, b, dy = make(M, C, dtype, C)
    bufs = [torch.full((M * ld + 64,), float('nan'), dtype=dtype, device=DEV) for _ in range(2)]
    views = [t[off:off + M * ld].view(M, ld)[:, :C] for t in bufs]
    views[0].copy_(x), views[1].copy_(dy)
    y, mean, rstd = ops.layer_norm(views[0], w, b)
    y0, mean0, rstd0 = ops.layer_norm(x, w, b)
    (ry, rdx, rdw, rdb), (ty, tdx, tdw, tdb) = reference(x, w, b, dy, 1e-5)
    check(y, ry, ty, 'y')
    dx, dw, db = ops.layer_norm_bwd(views[1], views[0], mean, rstd, w)
    for got, want, tol, name in ((dx, rdx, tdx, 'dx'), (dw, rdw, tdw, 'dw'), (db, rdb, tdb, 'db')):
        check(got, want, tol, name)


def test_without_weight_and_bias_and_partial_gradients():
    from sgg_amd import ops
    x, w, b, dy = make(77, 130, torch.float32, 3)
    (ry, rdx, rdw, rdb), (ty, tdx, tdw, tdb) = reference(x, None, None, dy, 1e-3)
    y, mean, rstd = ops.layer_norm(x, eps=1e-3)
    check(y, ry, ty, 'y')
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, want_dw=False, want_db=False)
    assert dw is None and db is None
    check(dx, rdx, tdx, 'dx')
    none, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, want_dx=False)
    assert none is None
    check(dw, rdw, tdw, 'dw')
    none, none2, db2 = ops.layer_norm_bwd(dy, x, mean, rstd, want_dx=False, want_dw=False)
    assert none2 is None and torch.equal(db, db2)


def test_constant_rows_large_offsets_and_non_finite_rows():
    from sgg_amd import ops
    x = torch.randn(8, 300, device=DEV)
    x[1] = 5.0                                       # variance 0: xh = 0, r = eps^-1/2
    x[2] += 3.0e4                                    # a mean far from the spread: the centred sum keeps the variance
    x[4, 7] = float('inf')
    x[5, 9] = float('nan')
    w, b = torch.ones(300, device=DEV), torch.full((300,), 0.25, device=DEV)
    y, mean, rstd = ops.layer_norm(x, w, b)
    assert torch.equal(y[1], b)
    check(y[2:3], *[t for t in (reference(x[2:3], w, b, x[2:3], 1e-5)[0][0], reference(x[2:3], w, b, x[2:3], 1e-5)[1][0])], 'offset')
    assert bool(y[4:6].isnan().all()) and bool(y[[0, 1, 2, 3, 6, 7]].isfinite().all())       # a bad row stays its own


def test_empty_batch():
    from sgg_amd import dense, ops
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    m = dense.LayerNormRows(32).to(DEV)
    y = m(x)
    assert y.shape == (0, 32)
    y.sum().backward()
    assert x.grad.shape == (0, 32) and float(m.weight.grad.abs().max()) == 0 and float(m.bias.grad.abs().max()) == 0


@pytest.mark.parametrize('shape', [(50, 24), (3, 5, 5, 24), (24,)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_module_autograd_and_state_names(shape, dtype):
    from sgg_amd import dense
    torch.manual_seed(2)
    mine, ref = dense.LayerNormRows(24).to(DEV), torch.nn.LayerNorm(24)
    assert sorted(mine.state_dict()) == sorted(ref.state_dict())
    with torch.no_grad():
        mine.weight.uniform_(0.5, 1.5), mine.bias.normal_()
    x = torch.randn(shape, device=DEV).to(dtype).requires_grad_()
    y = mine(x)
    assert y.shape == x.shape and y.dtype == dtype
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, (x, mine.weight, mine.bias), dy)
    want, tol = reference(x.detach().reshape(-1, 24), mine.weight.detach(), mine.bias.detach(), dy.reshape(-1, 24), mine.eps)
    check(y.detach().reshape(-1, 24), want[0], tol[0], 'y')
    for g, r, t, n in zip((got[0].reshape(-1, 24), got[1], got[2]), want[1:], tol[1:], ('dx', 'dw', 'db')):
        check(g, r, t, n)
    with torch.no_grad():
        assert not mine(x).requires_grad


def test_gradients_against_differences():
    """the derivative of a weighted sum of y along a direction, by central differences of the forward in 64 bits"""
    from sgg_amd import dense
    torch.manual_seed(4)
    x, w, b = torch.randn(6, 37, device=DEV), 1 + 0.2 * torch.randn(37, device=DEV), torch.randn(37, device=DEV)
    c = torch.randn(6, 37, device=DEV)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad((dense.layer_norm(*leaves) * c).sum(), leaves)

    def f(x, w, b):
        mu = x.mean(1, keepdim=True)
        return (((x - mu) / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + 1e-5) * w + b) * c.double()).sum()
    for i, g in enumerate(grads):
        d = torch.randn_like(g).double()
        at = [t.detach().double() for t in leaves]
        h = 1e-6
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        want = (f(*up) - f(*down)) / (2 * h)
        # third-order term h^2 and 64-bit cancellation 1e-16 / h are far below fp32's share: ~100 u of the sum of magnitudes
        assert abs(float((g.double() * d).sum() - want)) <= 100 * U * float((g.double() * d).abs().sum()) + 1e-6


def test_broadcast_gradients_and_another_stream():
    from sgg_amd import dense
    torch.manual_seed(6)
    for shape in ((5, 7), (4, 1), (1, 9)):
        m = dense.LayerNormRows(shape[1]).to(DEV)
        x = torch.randn(shape, device=DEV, requires_grad=True)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            a = torch.autograd.grad(m(x).sum(), (x, m.weight, m.bias))             # dy: one number, strides 0
        s.synchronize()
        b = torch.autograd.grad(m(x), (x, m.weight, m.bias), torch.ones(shape, device=DEV))
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x = torch.randn(3, 4, 10, device=DEV, requires_grad=True)
    assert torch.equal(dense.layer_norm(x.transpose(0, 1)[..., :8]), dense.layer_norm(x.detach().transpose(0, 1)[..., :8].contiguous()))


def test_graph_convolution_net_with_layer_norm_trains():
    """build_mlp(batch_norm='layer'): the scene-graph convolutions run forward and backward through it, every parameter gets a gradient"""
    from sgg_amd import dense
    from sgg_amd.gan_ops import GraphTripleConvNet
    torch.manual_seed(0)
    net = GraphTripleConvNet(12, input_edge_dim=8, output_dim=20, num_layers=2, hidden_dim=16, mlp_normalization='layer').to(DEV)
    assert sum(isinstance(m, dense.LayerNormRows) for m in net.modules()) == 4 + 2
    obj, pred = torch.randn(9, 12, device=DEV), torch.randn(14, 8, device=DEV)
    edges = torch.stack((torch.arange(14) % 9, (torch.arange(14) * 5 + 1) % 9), 1).to(DEV)
    o, p = net(obj, pred, edges)
    (o.square().sum() + p.square().sum()).backward()
    for n, q in net.named_parameters():
        assert q.grad is not None and bool(q.grad.isfinite().all()), n


def test_replayed_graph_equals_eager():
    from sgg_amd import ops
    x, w, b, dy = make(300, 96, torch.float16, 8)

    def step():
        y, mean, rstd = ops.layer_norm(x, w, b)
        return (y,) + ops.layer_norm_bwd(dy, x, mean, rstd, w)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for k in range(3):
        nx, _, _, ndy = make(300, 96, torch.float16, 20 + k)
        x.copy_(nx), dy.copy_(ndy)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(out, step()))


def test_rows_past_4_gigabytes():
    """17 GB of bf16 rows; the last ones and some on the way hold something, the others zeros"""
    from sgg_amd import ops
    M, C = 540001, 16001
    at = torch.tensor([0, 134218, 268436, M - 2, M - 1], device='cuda:0')
    xs, w, b, gs = make(5, C, torch.bfloat16, 5)
    x = torch.zeros(M, C, dtype=torch.bfloat16, device='cuda:0')
    x[at] = xs
    dy = torch.zeros_like(x)
    dy[at] = gs
    y, mean, rstd = ops.layer_norm(x, w, b)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    want, tol = reference(xs, w, b, gs, 1e-5)
    for got, v, t, name in ((y[at], want[0], tol[0], 'y'), (dx[at], want[1], tol[1], 'dx'), (dw, want[2], tol[2], 'dw'), (db, want[3], tol[3], 'db')):
        check(got, v, t, name)
    y[at] = b.to(y.dtype)
    assert bool((y == b.to(y.dtype)).all())
    dx[at] = 0
    assert not dx.any()
    del x, dy, y, dx
    torch.cuda.empty_cache()


def test_refusals():
    from sgg_amd import dense, ops
    x = torch.randn(4, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    with pytest.raises(ValueError):
        ops.layer_norm(x.t())                                       # columns not contiguous
    with pytest.raises(ValueError):
        ops.layer_norm(torch.randn(1, 8, device=DEV).expand(4, 8))  # rows on top of each other
    with pytest.raises(ValueError):
        ops.layer_norm(x, w[:7])
    with pytest.raises(TypeError):
        ops.layer_norm(x, w.half())
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError):
        ops.layer_norm(x, w, eps=0.0)
    with pytest.raises(ValueError):
        ops.layer_norm(x, w, eps=float('nan'))
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(1, 16385, device=DEV))
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(3, 0, device=DEV))
    with pytest.raises(ValueError):
        ops.layer_norm(x.view(2, 2, 8))
    y, mean, rstd = ops.layer_norm(x, w)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x.half(), x, mean, rstd, w)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, x, mean[:3], rstd, w)
    with pytest.raises(ValueError):
        dense.LayerNormRows(9).to(DEV)(x)
    with pytest.raises(RuntimeError):
        dense.layer_norm(x.cpu())
