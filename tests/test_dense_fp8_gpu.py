"""The 'fp8' arithmetic of the dense layers on the GPU: the row product itself, widths that do not fit, a mode switched between forward and backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def mode():
    from sgg_amd import dense
    prev = dense.compute_mode()
    yield
    dense.set_compute(prev)


@pytest.mark.parametrize('M,K,N', [(1, 32, 5), (40, 64, 70), (300, 1056, 129)])
def test_product_is_the_product_of_the_8_bit_forms(M, K, N):
    """fp32 sums of whole products: (K + 32) 2^-24 of the sum of magnitudes, the bias one rounding more"""
    from sgg_amd import dense, ops
    torch.manual_seed(M)
    x, w, b = torch.randn(M, K, device=DEV), torch.randn(N, K, device=DEV), torch.randn(N, device=DEV)
    dense.set_compute('fp8')
    y = dense.product(x, w, b)
    a, c = ops.quantize_fp8(x).dequantize(), ops.quantize_fp8(w).dequantize()
    tol = (K + 33) * U * (torch.mm(a.abs(), c.abs().t().contiguous()) + b.double().abs())
    assert y.dtype == torch.float32 and bool(((y.double() - torch.mm(a, c.t().contiguous()) - b.double()).abs() <= tol).all())
    dense.set_compute('f32')
    assert torch.equal(dense.product(x, w, b, mode='fp8'), y)


def test_a_mode_switched_between_forward_and_backward():
    from sgg_amd import dense
    torch.manual_seed(1)
    x = torch.randn(70, 96, device=DEV, requires_grad=True)
    lin = dense.Linear(96, 40).to(DEV)
    dy = torch.randn(70, 40, device=DEV)
    leaves = (x, lin.weight, lin.bias)

    def grads(forward, backward):
        dense.set_compute(forward)
        y = lin(x)
        dense.set_compute(backward)
        return torch.autograd.grad(y, leaves, dy)
    for other in ('f32', 'x3', 'f16'):
        for a, b in zip(grads(other, 'fp8'), grads(other, other)):
            assert torch.equal(a, b)
        for a, b in zip(grads('fp8', other), grads('fp8', 'fp8')):
            assert torch.equal(a, b)


@pytest.mark.parametrize('grad', [True, False])
def test_widths_that_do_not_fit_are_refused(grad):
    from sgg_amd import dense
    dense.set_compute('fp8')
    lin = dense.Linear(100, 5).to(DEV)
    with torch.set_grad_enabled(grad):
        for width in (64, 99, 101, 130):
            with pytest.raises(ValueError):
                lin(torch.randn(3, width, device=DEV))
        assert lin(torch.randn(2, 3, 100, device=DEV)).shape == (2, 3, 5)


def test_gan_iteration_clips_any_gradients():
    """ordinary ones on the kernels; fp64 and rows with gaps as torch's function does; one gradient of two parameters, which that scales once or twice
    in a race of its threads, is refused and left as it was"""
    from sgg_amd.feature_gan import _clip_gradients

    def params(kind):
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.zeros(40, 40, device=DEV, dtype=torch.float64 if kind == 'double' and i else torch.float32)) for i in range(3)]
        for p in ps:
            p.grad = torch.randn(40, 80, device=DEV)[:, ::2].to(p.dtype) if kind == 'gaps' else torch.randn(40, 40, device=DEV).to(p.dtype)
        return ps
    for kind in ('plain', 'double', 'gaps'):
        mine, ref = params(kind), params(kind)
        assert kind != 'gaps' or not mine[0].grad.is_contiguous()
        n, r = _clip_gradients(mine, 0.5), torch.nn.utils.clip_grad_norm_(ref, 0.5)
        assert abs(float(n) - float(r)) <= 2404 * U * float(r)              # (torch: 4800 fp32 squares, a rounding each at most, their root half of that)
        for a, b in zip(mine, ref):
            assert float((a.grad - b.grad).abs().max()) <= 2408 * U * float(b.grad.abs().max())
    ps = params('plain')
    ps[1].grad = ps[0].grad
    before = [p.grad.clone() for p in ps]
    with pytest.raises(ValueError):
        _clip_gradients(ps, 0.5)
    assert all(torch.equal(p.grad, g) for p, g in zip(ps, before))


@pytest.mark.parametrize('shape,N', [((2, 3, 0), 5), ((0,), 5), ((3, 0), 5), ((2, 0, 7), 5), ((4, 7), 0), ((33, 7), 0), ((0, 0), 0)])
def test_no_rows_columns_or_outputs(shape, N):
    """forward and every gradient of a product with a length of zero; the operand forms' own readings"""
    from sgg_amd import dense, ops
    K = shape[-1]
    x = torch.randn(shape, device=DEV, requires_grad=True)
    w, b = torch.randn(N, K, device=DEV, requires_grad=True), torch.randn(N, device=DEV, requires_grad=True)
    dense.set_compute('fp8')
    for call in (dense.affine_fp8, dense.affine):
        y = call(x, w, b)
        dy = torch.randn_like(y)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert y.shape == shape[:-1] + (N,) and dx.shape == shape and dw.shape == (N, K) and db.shape == (N,)
        want = b.detach().expand_as(y) if not K else y.detach()
        assert torch.equal(y.detach(), want) and not dw.any() and (N or not dx.any())
        assert float((db - dy.reshape(dy.numel() // N if N else 0, N).sum(0)).abs().sum()) <= 1e-5
        assert torch.autograd.grad(call(x.detach(), w.detach(), b), b, dy)[0].shape == (N,)
    for q in ops.quantize_fp8(torch.zeros(shape[-2] if len(shape) > 1 else 1, K, device=DEV), 'both'):
        assert q.codes().shape[0] == q.shape[0] and q.exponents().shape[0] == q.shape[0] and q.dequantize().shape == q.shape


def test_layer_norm_of_no_columns_is_refused():
    from sgg_amd import dense
    for shape in ((3, 0), (2, 3, 0), (0,)):
        with pytest.raises(ValueError):
            dense.layer_norm(torch.zeros(shape, device=DEV))


def test_gan_iteration_in_8_bits_with_clipped_gradients():
    """a whole iteration: the generator's and the discriminators' layers in the fp8 arithmetic, the relation model's gradients clipped before an
    optimiser that is not FusedSGD; every part learns, and the same iteration gives the same weights (but for the two discriminators' first layers: the
    gradient of their lookup of class columns is an indexed sum of torch's, in the order its threads run -- in every arithmetic)"""
    import sgg_amd
    from sgg_amd import dense
    from sgg_amd.feature_gan import GAN, gan_train_step
    from sgg_amd.synthetic import SyntheticData, init_weights, synthetic_batch

    def iteration():
        torch.manual_seed(3)
        data = SyntheticData()
        model = init_weights(sgg_amd.RelModelStanford(data, mode='sgcls')).to(DEV)
        model.set_compute_dtype(torch.float32)
        for n, p in model.named_parameters():
            if n.startswith('detector.'):
                p.requires_grad = False
        gan = GAN(data.ind_to_classes, data.ind_to_predicates, n_ch=model.edge_dim, pool_sz=model.pool_sz, fmap_sz=model.fmap_sz, n_layers_G=2,
                  device=DEV).to(DEV)
        batch = tuple(t.to(DEV) if isinstance(t, torch.Tensor) else t for t in synthetic_batch(B=2, n_boxes=5, n_fg=4, seed=8))
        model.train()
        res = model([batch])
        opt = torch.optim.SGD([p for p in model.parameters() if p.requires_grad], lr=1e-3)
        G_opt = torch.optim.SGD([p for n, p in gan.named_parameters() if n.startswith('G_')], lr=1e-2)
        D_opt = torch.optim.SGD([p for n, p in gan.named_parameters() if n.startswith('D_')], lr=1e-2)
        named = dict([('sgg.' + n, p) for n, p in model.named_parameters() if p.requires_grad] + list(gan.named_parameters()))
        before = {n: p.detach().clone() for n, p in named.items()}
        losses = gan_train_step(model, gan, res, batch[3].clone(), batch[4].clone(), batch[5].clone(), opt, G_opt, D_opt, clip=0.1)
        assert all(torch.isfinite(v) for v in losses.values())
        for n, p in named.items():
            assert bool(torch.isfinite(p).all()) and (p.grad is None or bool(torch.isfinite(p.grad).all())), n
        step = sum((p.detach().double() - before[n].double()).square().sum() for n, p in named.items() if n.startswith('sgg.')) ** 0.5
        assert 0 < float(step) <= 1e-3 * 0.1 * 1.01                       # lr times the clipped norm (and the weights' own rounding)
        for must in ('G_obj_embed.weight', 'G_gcn.gconvs.0.net1.0.weight', 'G_node.0.weight', 'G_proj.weight', 'G_refine.output_conv.0.weight',
                     'D_nodes.0.weight_orig', 'D_edges.6.weight_orig', 'D_global.15.weight_orig', 'sgg.rel_fc.weight', 'sgg.roi_fmap.1.0.weight'):
            assert not torch.equal(before[must], named[must].detach()), must
        return {n: p.detach().clone() for n, p in named.items()}
    dense.set_compute('fp8')
    a, b = iteration(), iteration()
    assert [n for n in a if not torch.equal(a[n], b[n]) and n not in ('D_nodes.0.weight_orig', 'D_edges.0.weight_orig')] == []
