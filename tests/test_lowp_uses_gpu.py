"""Layer norm, 8-bit layers and clipping as programs use them: a captured training step, two streams at once, operands of mixed types."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def leaves(M, C, N, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)                # noqa: E731
    return [rand(M, C).to(dtype), 1 + 0.2 * rand(C), 0.2 * rand(C), rand(N, C) / C ** 0.5, 0.1 * rand(N), rand(M, N).to(dtype)]


def step(x, w, b, W, B, dy):
    """normalise, multiply, differentiate, clip"""
    from sgg_amd import dense, ops
    ins = [t.detach().requires_grad_() for t in (x, w, b, W, B)]
    y = dense.affine_fp8(dense.layer_norm(*ins[:3]), *ins[3:])
    grads = torch.autograd.grad(y, ins, dy)
    norm = ops.clip_grads_(list(grads), 0.5)
    return [y.detach(), norm] + list(grads)


@pytest.mark.parametrize('M,C,N,dtype', [(5, 100, 40, F32), (300, 1100, 333, F16), (2500, 512, 2400, BF16)])
def test_a_captured_training_step_replays(M, C, N, dtype):
    data = leaves(M, C, N, dtype, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(*data)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*data)
    for k in range(3):
        for t, n in zip(data, leaves(M, C, N, dtype, 20 + k)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(*data)))


def test_two_streams_at_once():
    """nothing is shared between calls: what runs beside each other gives what runs alone gives"""
    jobs = [leaves(300, 1100, 333, F16, 1), leaves(2500, 512, 2400, BF16, 2), leaves(33, 5000, 64, F32, 3)]
    alone = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None] * len(jobs)
    for _ in range(4):
        for i, (s, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i] = step(*j)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize('wt,bt', [(F16, F16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize('xt,out', [(F32, F16), (F16, F32), (BF16, F16)])
def test_mixed_types(xt, out, wt, bt):
    """every gradient in its leaf's type, from the same products as leaves of f32 that hold the same values"""
    from sgg_amd import dense
    x, _, _, W, B, dy = leaves(70, 300, 90, xt, 4)
    x, W, B, dy = x.requires_grad_(), W.to(wt).requires_grad_(), B.to(bt).requires_grad_(), dy.to(out)
    y = dense.affine_fp8(x, W, B, out_dtype=out)
    grads = torch.autograd.grad(y, (x, W, B), dy)
    assert y.dtype == out and [g.dtype for g in grads] == [xt, wt, bt]
    W32, B32 = W.detach().float().requires_grad_(), B.detach().float().requires_grad_()
    y2 = dense.affine_fp8(x, W32, B32, out_dtype=out)
    ref = torch.autograd.grad(y2, (x, W32, B32), dy)
    assert torch.equal(y, y2) and all(torch.equal(a, b.to(a.dtype)) for a, b in zip(grads, ref))


def test_layer_norm_with_one_of_weight_and_bias():
    from sgg_amd import dense
    x, w, b, _, _, _ = leaves(50, 130, 1, F32, 6)
    dy = torch.randn_like(x)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    one, zero = torch.ones(130, device=DEV), torch.zeros(130, device=DEV)
    for args, full, wanted in (((None, b), (one, b), (x, b)), ((w, None), (w, zero), (x, w)), ((None, None), (one, zero), (x,))):
        y, ref = dense.layer_norm(x, *args), dense.layer_norm(x, *full)
        assert torch.equal(y, ref)
        for p, q in zip(torch.autograd.grad(y, wanted, dy), torch.autograd.grad(ref, wanted, dy)):
            assert torch.equal(p, q)
    # rows that are one row in memory: copied, their gradients added up by autograd
    row = torch.randn(1, 130, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(dense.layer_norm(row.expand(50, 130), w, b), row, dy)
    want, = torch.autograd.grad(dense.layer_norm(row.detach().repeat(50, 1).requires_grad_(), w, b).sum() * 0 + (dense.layer_norm(row, w, b) * dy.sum(0)).sum(), row)
    assert float((dx - want).abs().max()) <= 400 * U * 50 * float(dy.abs().max())


def test_an_input_changed_in_place_after_the_forward_is_noticed():
    from sgg_amd import dense
    x, w, b, W, B, dy = leaves(20, 64, 10, F32, 7)
    w.requires_grad_()
    h = x * 1.0
    y = dense.layer_norm(h, w, b)
    h.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    W.requires_grad_()                                  # (the 8-bit layer keeps forms of its own: the gradient is that of the forward's values)
    h = x * 1.0
    y = dense.affine_fp8(h, W, B)
    h.zero_()
    assert torch.equal(torch.autograd.grad(y, W, dy)[0], torch.autograd.grad(dense.affine_fp8(x, W, B), W, dy)[0])
