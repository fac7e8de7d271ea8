"""Global gradient norm and clipping (csrc/clip.hip) against 64-bit arithmetic: one to many tensors, mixed types, any alignment, overflow.

Tolerances: the sum of squares is held in 64 bits (n 2^-53, nothing here), the norm is rounded to fp32 once (half a step, 2^-24), the factor
once, a clipped value once more in fp32 and, for a 16-bit output, once in its type: |got - want| <= (2 * 2^-24 + half step) |want|, and a 16-bit
subnormal's step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def want_of(grads, max_norm, scale=1.0):
    norm = abs(scale) * float(sum(g.double().square().sum() for g in grads)) ** 0.5 if grads else 0.0
    c = scale * min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.double() * c for g in grads]


def check(norm, got, want):
    wn, wg = want
    assert abs(float(norm.double()) - wn) <= 2 * U * wn
    for a, w in zip(got, wg):
        half = torch.finfo(a.dtype).eps / 2
        step = torch.finfo(a.dtype).tiny * torch.finfo(a.dtype).eps
        over = (a.double() - w).abs() - ((2 * U + (half if a.dtype != F32 else U)) * w.abs() + step)
        assert a.numel() == 0 or float(over.max()) <= 0, float(over.max())


def tensors(sizes, types, seed, scale=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(scale * torch.randn(n, generator=g, device=DEV)).to(t) for n, t in zip(sizes, types)]


@pytest.mark.parametrize('sizes', [[1], [0], [3, 0, 5], [64, 1000, 8193], [8191, 8192, 8193, 16385], [7] * 96, [13] * 97, [5, 100001] * 110, [3000001]])
@pytest.mark.parametrize('types', [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize('max_norm', [0.05, 1e6])
def test_in_place(sizes, types, max_norm):
    from sgg_amd import ops
    grads = tensors(sizes, [types[i % len(types)] for i in range(len(sizes))], len(sizes))
    want = want_of(grads, max_norm)
    before = [g.clone() for g in grads]
    assert abs(float(ops.grad_norm(grads)) - want[0]) <= 2 * U * want[0]
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    versions = [g._version for g in grads]
    norm = ops.clip_grads_(grads, max_norm)
    check(norm, grads, want)
    assert all(g._version > v for g, v in zip(grads, versions))
    if want[0] < max_norm:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))             # nothing to clip: not a bit changes


@pytest.mark.parametrize('src,dst', [(F16, F32), (BF16, F32), (F32, BF16), (F32, F16), (F16, F16)])
def test_unscale_into_other_buffers(src, dst):
    from sgg_amd import ops
    grads = tensors([4097, 1, 77, 9000], [src] * 4, 5, scale=30.0)
    out = [torch.full_like(g, 7.0, dtype=dst) for g in grads]
    before = [g.clone() for g in grads]
    for max_norm in (0.5, 1e9):
        norm = ops.clip_grads_(grads, max_norm, grad_scale=1.0 / 1024, out=out)
        check(norm, out, want_of(grads, max_norm, 1.0 / 1024))
        assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize('off', [1, 2, 3, 5, 7])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_any_alignment_and_neighbours_untouched(off, dtype):
    from sgg_amd import ops
    buf = torch.randn(30000, device=DEV).to(dtype)
    ref = buf.clone()
    grads = [buf[off:off + 9001], buf[10000 + off:10000 + off + 5]]
    norm = ops.clip_grads_(grads, 1.0)
    check(norm, grads, want_of([ref[off:off + 9001], ref[10000 + off:10000 + off + 5]], 1.0))
    mask = torch.ones(30000, dtype=torch.bool, device=DEV)
    mask[off:off + 9001] = False
    mask[10000 + off:10000 + off + 5] = False
    assert torch.equal(buf[mask], ref[mask])
    out = torch.zeros(9010, device=DEV)
    check(ops.clip_grads_([ref[off:off + 9001]], 1.0, out=[out[9 - off:9 - off + 9001]]), [out[9 - off:9 - off + 9001]], want_of([ref[off:off + 9001]], 1.0))


def test_large_and_tiny_values_neither_overflow_nor_vanish():
    from sgg_amd import ops
    big = [torch.full((1000,), 1e30, device=DEV), torch.full((7,), -2e38, device=DEV)]
    check(ops.grad_norm([big[0]]), [], (float(1e30 * 1000 ** 0.5), []))
    want = want_of(big, 1.0)
    norm = ops.clip_grads_(big, 1.0)                        # (the norm itself is past fp32's largest: inf, the factor is not)
    assert float(norm) == float('inf') or abs(float(norm) - want[0]) <= 2 * U * want[0]
    for g, w in zip(big, want[1]):
        assert float((g.double() - w).abs().max()) <= 4 * U * float(w.abs().max())
    small = [torch.full((1000,), 1e-30, device=DEV)]
    assert abs(float(ops.grad_norm(small)) - 1e-30 * 1000 ** 0.5) <= 2 * U * 1e-30 * 1000 ** 0.5 + 1e-37


def test_non_finite_norms_are_not_hidden():
    from sgg_amd import ops
    for bad in (float('nan'), float('inf')):
        mine = [torch.ones(10, device=DEV), torch.ones(5000, device=DEV)]
        mine[1][77] = bad
        ref = [torch.nn.Parameter(torch.zeros_like(g)) for g in mine]
        for p, g in zip(ref, mine):
            p.grad = g.clone()
        rn = torch.nn.utils.clip_grad_norm_(ref, 1.0)
        norm = ops.clip_grads_(mine, 1.0)
        assert torch.equal(norm.isnan(), rn.isnan()) and torch.equal(norm.isinf(), rn.isinf())
        for g, p in zip(mine, ref):
            assert torch.equal(g.isnan(), p.grad.isnan()) and torch.equal(g.nan_to_num(0.0), p.grad.nan_to_num(0.0))


def test_parameters_form_follows_torch():
    from sgg_amd.trainer import clip_grad_norm_
    torch.manual_seed(1)
    net = torch.nn.Sequential(torch.nn.Conv2d(3, 5, 3), torch.nn.Linear(40, 30), torch.nn.Linear(9, 9)).to(DEV)
    for i, p in enumerate(net.parameters()):
        if i != 5:
            p.grad = torch.randn_like(p)
    net[0].weight.grad = net[0].weight.grad.contiguous(memory_format=torch.channels_last)      # dense in another order
    net.register_parameter('turned', torch.nn.Parameter(torch.randn(6, 7, 5, device=DEV).permute(2, 0, 1)))
    net.turned.grad = torch.randn(6, 7, 5, device=DEV).permute(2, 0, 1)
    grads = [p.grad for p in net.parameters() if p.grad is not None]
    want = want_of(grads, 2.0)
    check(clip_grad_norm_(net.parameters(), 2.0), grads, want)
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    p = net[1].weight
    want = want_of([p.grad], 0.1)
    check(clip_grad_norm_(p, 0.1), [p.grad], want)
    assert clip_grad_norm_(torch.nn.Parameter(torch.zeros(3, device=DEV)), 1.0).item() == 0.0


def test_same_bits_every_time_and_in_a_replayed_graph():
    from sgg_amd import ops
    sizes = [100001, 33, 8192, 70000]
    grads = tensors(sizes, [F32, F16, BF16, F32], 9)
    out = [torch.empty_like(g, dtype=F32) for g in grads]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.clip_grads_(grads, 0.3, 0.5, out=out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads_(grads, 0.3, 0.5, out=out)
    for k in range(3):
        for g, n in zip(grads, tensors(sizes, [F32, F16, BF16, F32], 30 + k)):
            g.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        out2 = [torch.empty_like(o) for o in out]
        n2 = ops.clip_grads_(grads, 0.3, 0.5, out=out2)
        assert torch.equal(norm, n2) and all(torch.equal(a, b) for a, b in zip(out, out2))


def test_one_tensor_past_4_gigabytes_on_another_stream():
    from sgg_amd import ops
    n = (1 << 32) + 12345
    g = torch.zeros(n, dtype=F16, device=DEV)
    at = torch.tensor([0, 5, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1], device=DEV)
    g[at] = torch.tensor([3.0, -1.0, 2.0, 5.0, -4.0, 7.0], device=DEV).half()
    want = want_of([g[at]], 2.0, 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = torch.ones(n, dtype=BF16, device=DEV)
        norm = ops.clip_grads_(g, 2.0, 0.5, out=out)
    torch.cuda.current_stream().wait_stream(s)
    check(norm, [out[at]], want)
    out[at] = 0
    assert not out.any()
    del g, out
    torch.cuda.empty_cache()


def test_inference_tensors_are_clipped():
    from sgg_amd import ops
    with torch.inference_mode():
        g = torch.full((100,), 3.0, device=DEV)
        ops.clip_grads_([g], 1.0)
        assert abs(float(g.norm()) - 1.0) < 1e-5


def test_refusals():
    from sgg_amd import ops
    g = torch.randn(100, device=DEV)
    with pytest.raises(ValueError):
        ops.clip_grads_([g, g], 1.0)                               # the same tensor twice
    with pytest.raises(ValueError):
        ops.clip_grads_([g[:60], g[50:]], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grads_([g[::2]], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grads_([g[:1].expand(5)], 1.0)
    with pytest.raises(ValueError):
        ops.clip_grads_([g], -1.0)
    with pytest.raises(ValueError):
        ops.clip_grads_([g], float('nan'))
    with pytest.raises(ValueError):
        ops.clip_grads_([g], 1.0, out=[])
    with pytest.raises(ValueError):
        ops.clip_grads_([g], 1.0, out=[torch.empty(99, device=DEV)])
    with pytest.raises(ValueError):
        ops.clip_grads_([g[:50]], 1.0, out=[g[10:60]])             # output over its own input, shifted
    h = torch.randn(100, device=DEV).half()
    with pytest.raises(ValueError):
        ops.clip_grads_([h], 1.0, out=[h.view(torch.bfloat16)])    # the same memory as another type
    with pytest.raises(TypeError):
        ops.clip_grads_([g.double()], 1.0)
    with pytest.raises(TypeError):
        ops.clip_grads_([torch.zeros(4, 4, device=DEV).to_sparse()], 1.0)
    with pytest.raises(RuntimeError):
        ops.clip_grads_([g.cpu()], 1.0)
    assert abs(float(ops.grad_norm([g, g])) - (2.0 * float(g.double().square().sum())) ** 0.5) < 1e-4      # reading twice is fine
    assert abs(float(ops.grad_norm([g[::2]])) - float(g[::2].double().norm())) < 1e-4
