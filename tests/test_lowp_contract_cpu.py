"""What the 8-bit layers, layer norm and clipping refuse or leave to others before any kernel is launched: the launches are stubs here, on the CPU."""
import pytest
import torch


class Form(object):
    """stands for an operand form"""
    def __init__(self, t):
        self._mem, self.shape = t, tuple(t.shape)


@pytest.fixture
def stubbed(monkeypatch):
    """dense with products that multiply in torch: what reaches them was let through"""
    from sgg_amd import dense, ops
    monkeypatch.setattr(dense, '_need_gpu', lambda x: None)
    monkeypatch.setattr(ops, 'quantize_fp8', lambda x, form='rows', colsum=False: Form(x) if form == 'rows' else (Form(x), Form(x.t())))
    monkeypatch.setattr(ops, '_vector', lambda t, n, what: None)
    monkeypatch.setattr(ops, '_gemm_fp8', lambda a, w, b=None, act=0, out_dtype=torch.float32, out=None: a._mem @ w._mem.t())
    prev = dense.set_compute('fp8')
    yield dense
    dense.set_compute(prev)


@pytest.mark.parametrize('grad', [True, False])
def test_fp8_layers_refuse_another_width(stubbed, grad):
    lin = stubbed.Linear(100, 5)
    with torch.set_grad_enabled(grad):
        assert lin(torch.randn(3, 100)).shape == (3, 5)
        for width in (64, 96, 99, 101, 130):
            with pytest.raises(ValueError):
                lin(torch.randn(3, width))
            with pytest.raises(ValueError):
                stubbed.affine(torch.randn(2, 3, width), lin.weight)


@pytest.mark.parametrize('grad', [True, False])
@pytest.mark.parametrize('which', ['input', 'weight', 'bias'])
def test_forward_mode_tangents_are_not_dropped(stubbed, monkeypatch, grad, which):
    """a dual tensor, whatever it is an argument of and whether or not a backward is recorded: no layer answers without its derivative"""
    import torch.autograd.forward_ad as fwd
    from sgg_amd import ops
    monkeypatch.setattr(ops, '_layer_norm', lambda x, w, b, eps, stats: (x * 1.0, torch.zeros(2, x.shape[0])))
    args = {'input': torch.randn(3, 7), 'weight': torch.randn(7, 7), 'bias': torch.randn(7)}
    vec = {'input': args['input'], 'weight': torch.randn(7), 'bias': args['bias']}
    calls = (lambda a, v: stubbed.layer_norm(v['input'], v['weight'], v['bias']), lambda a, v: stubbed.affine_fp8(a['input'], a['weight'], a['bias']),
             lambda a, v: stubbed.affine(a['input'], a['weight'], a['bias']))
    with torch.set_grad_enabled(grad):
        for call in calls:
            call(args, vec)
            with fwd.dual_level():
                call(args, vec)                                              # nothing carries a tangent: as outside
                dual = [{k: fwd.make_dual(v, torch.ones_like(v)) if k == which else v for k, v in d.items()} for d in (args, vec)]
                with pytest.raises(Exception, match='jvp'):
                    call(*dual)


@pytest.mark.parametrize('forward,backward,want', [('f32', 'fp8', 'f32'), ('x3', 'fp8', 'x3'), ('f16', 'fp8', 'f16'), ('f32', 'f16', 'f16'), ('f32', 'f32', 'f32')])
def test_a_backward_is_not_done_in_8_bits_unless_its_forward_was(monkeypatch, forward, backward, want):
    """set_compute between a forward and its backward"""
    from sgg_amd import dense, ops
    seen = []

    def product(x, w, bias=None, mode=None):
        seen.append(mode or dense.compute_mode())
        return x @ w.t()
    monkeypatch.setattr(dense, '_need_gpu', lambda x: None)
    monkeypatch.setattr(dense, 'product', product)
    monkeypatch.setattr(ops, 'transpose', lambda t, pad_to=1: torch.nn.functional.pad(t.t(), (0, -t.shape[0] % 32)).contiguous())
    x, w = torch.randn(5, 32, requires_grad=True), torch.randn(7, 32, requires_grad=True)
    prev = dense.set_compute(forward)
    try:
        y = dense.affine(x, w)
        dense.set_compute(backward)
        dy = torch.randn(5, 7)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
    finally:
        dense.set_compute(prev)
    assert seen == [forward, want, want]
    assert torch.allclose(dx, dy @ w) and torch.allclose(dw, dy.t() @ x, atol=1e-5)


def test_a_weight_that_is_elsewhere_by_the_time_of_the_backward(monkeypatch):
    """module.cpu() between forward and backward gives the saved parameter other memory under the same name and version: its address must not reach
    a kernel (here every tensor is on the CPU, as that one would be)"""
    from sgg_amd import dense, ops
    monkeypatch.setattr(dense, '_need_gpu', lambda x: None)
    monkeypatch.setattr(ops, '_layer_norm', lambda x, w, b, eps, stats: (x * 1.0, torch.zeros(2, x.shape[0])))
    launched = []
    monkeypatch.setattr(ops, '_layer_norm_bwd', lambda *a: (launched.append(a), (None, None, None))[1])
    x, m = torch.randn(3, 7, requires_grad=True), dense.LayerNormRows(7)
    y = m(x)
    with pytest.raises(RuntimeError, match='not on the GPU'):
        y.sum().backward()
    assert not launched


def test_gan_iteration_clips_what_the_kernels_do_not_take():
    """fp64, gaps, memory on the host: as torch's function clips them"""
    from sgg_amd.feature_gan import _clip_gradients

    def params():
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.zeros(4, 4, dtype=t)) for t in (torch.float32, torch.float64, torch.float32, torch.float32, torch.float32)]
        grads = [torch.randn(4, 4), torch.randn(4, 4).double(), torch.randn(4, 8)[:, ::2], torch.randn(4, 4)]
        for p, g in zip(ps, grads):
            p.grad = g
        return ps
    mine, ref = params(), params()
    assert torch.equal(_clip_gradients(iter(mine), 0.5), torch.nn.utils.clip_grad_norm_(ref, 0.5))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(mine[:4], ref[:4])) and mine[4].grad is None


@pytest.mark.parametrize('M,K', [(0, 0), (0, 200), (3, 0), (1, 1), (129, 130)])
def test_operand_forms_of_no_rows_or_columns_can_be_read(M, K):
    from sgg_amd import ops
    slabs, R, scales = ops._fp8_dims(M, K)
    blocks = (K + 127) // 128
    for q in (ops.Fp8Rows._of(torch.full((slabs * R * 64 + scales,), 127, dtype=torch.uint8), (M, K)),
              ops.Fp8Rows(torch.zeros(slabs, R, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.full((scales,), 127, dtype=torch.uint8), (M, K))):
        assert q.codes().shape == (M, blocks * 128) and q.exponents().shape == (M, blocks) and q.dequantize().shape == (M, K)
        assert not q.exponents().any()


def test_8_bit_layers_of_no_columns_give_the_bias(stubbed):
    for shape in ((0,), (3, 0), (2, 3, 0), (2, 0, 4, 0)):
        for call in (stubbed.affine_fp8, stubbed.affine):
            assert call(torch.zeros(shape), torch.zeros(5, 0)).shape == shape[:-1] + (5,)
    assert stubbed.affine_fp8(torch.zeros(2, 0, 7), torch.zeros(5, 7)).shape == (2, 0, 5)
