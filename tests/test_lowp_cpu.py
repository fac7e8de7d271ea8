"""What of layer norm, the 8-bit product and gradient clipping can be checked without a GPU: the C entries refuse bad arguments before any
launch, CPU tensors are refused, the operand form's index rule, the modules' parameters."""
import ctypes

import pytest
import torch

ERR_ARG, ERR_DTYPE = -1, -2
P = 4096                                         # an address that is never followed: every call here ends in a check on the host


def test_layer_norm_entries_refuse():
    from sgg_amd import _lib
    lib = _lib.load()

    def fwd(x=P, ldx=8, y=P, mean=P, rstd=P, M=4, C=8, eps=1e-5, dtype=0):
        return lib.sgg_layer_norm_fwd(x, ldx, None, None, y, mean, rstd, M, C, eps, dtype, None)
    for bad in (dict(x=None), dict(y=None), dict(mean=None), dict(rstd=None), dict(ldx=7), dict(C=0), dict(C=16385, ldx=16385), dict(M=-1), dict(eps=0.0),
                dict(eps=float('nan')), dict(M=1 << 31)):
        assert fwd(**bad) == ERR_ARG, bad
    assert fwd(dtype=3) == ERR_DTYPE and fwd(dtype=-1) == ERR_DTYPE
    assert fwd(M=0, x=None, y=None) == 0

    def bwd(dy=P, ld=8, x=P, mean=P, rstd=P, dx=P, dw=P, db=P, ws=P, M=4, C=8, dtype=0):
        return lib.sgg_layer_norm_bwd(dy, ld, x, 8, None, mean, rstd, dx, dw, db, ws, M, C, dtype, None)
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(ws=None), dict(ld=7), dict(C=0), dict(M=-1)):
        assert bwd(**bad) == ERR_ARG, bad
    assert bwd(dtype=9) == ERR_DTYPE
    assert lib.sgg_layer_norm_bwd_parts(-1, 8, 0) == ERR_ARG and lib.sgg_layer_norm_bwd_parts(5, 8, 7) == ERR_DTYPE
    for M in (0, 1, 1000, 70000):
        for C in (1, 512, 16384):
            assert 0 <= lib.sgg_layer_norm_bwd_parts(M, C, 0) <= max(M, 1)


def test_fp8_entries_refuse():
    from sgg_amd import _lib
    lib = _lib.load()

    def q(x=P, ldx=256, M=4, K=256, rows=P, rs=P, cols=P, cs=P, sums=None, ws=None, dtype=0):
        return lib.sgg_fp8_quantize(x, ldx, M, K, rows, rs, cols, cs, sums, ws, dtype, None)
    for bad in (dict(x=None), dict(ldx=255), dict(M=-1), dict(K=-1), dict(rows=None), dict(rs=None), dict(cols=None), dict(cs=None),
                dict(rows=None, rs=None, cols=None, cs=None), dict(rows=P + 8), dict(cols=P + 4), dict(rs=P + 2), dict(M=1 << 40),
                dict(sums=P), dict(sums=P, ws=P, cols=None, cs=None)):
        assert q(**bad) == ERR_ARG, bad
    assert q(dtype=5) == ERR_DTYPE and q(M=0, x=None) == 0

    def g(A=P, As=P, W=P, Ws=P, C=P, ldc=64, M=4, N=64, Kp=256, act=0, dtype=0):
        return lib.sgg_gemm_fp8(A, As, W, Ws, None, C, ldc, M, N, Kp, act, dtype, None, None)
    for bad in (dict(A=None), dict(As=None), dict(W=None), dict(Ws=None), dict(C=None), dict(ldc=63), dict(M=-1), dict(N=-1), dict(Kp=200), dict(Kp=-128),
                dict(act=2), dict(A=P + 8), dict(Ws=P + 1), dict(M=1 << 33)):
        assert g(**bad) == ERR_ARG, bad
    assert g(dtype=3) == ERR_DTYPE and g(M=0, A=None) == 0 and g(N=0, C=None) == 0
    assert lib.sgg_gemm_fp8_splits(-1, 4, 128, 0) == ERR_ARG and lib.sgg_gemm_fp8_splits(4, 4, 100, 0) == ERR_ARG and lib.sgg_gemm_fp8_splits(4, 4, 128, 9) == ERR_DTYPE
    for M, N, Kp in ((1, 4096, 25088), (256, 4096, 25088), (8192, 8192, 128), (1, 1, 128), (0, 0, 0), (333, 1100, 2048)):
        for code in (0, 1, 2):
            s = lib.sgg_gemm_fp8_splits(M, N, Kp, code)
            assert 1 <= s <= max(1, Kp // 128), (M, N, Kp, s)
    assert lib.sgg_fp8_scale_bytes(1, 1) == 128 and lib.sgg_fp8_scale_bytes(129, 257) == 3 * 256 and lib.sgg_fp8_scale_bytes(0, 5) == 0


def test_clip_entry_refuses():
    from sgg_amd import _lib
    lib = _lib.load()
    ptr = (ctypes.c_void_p * 2)(P, 2 * P)
    null = (ctypes.c_void_p * 2)(P, None)
    n, neg = (ctypes.c_int64 * 2)(5, 6), (ctypes.c_int64 * 2)(5, -1)
    f32, odd = (ctypes.c_int * 2)(0, 0), (ctypes.c_int * 2)(0, 3)

    def c(g=ptr, out=ptr, n=n, gd=f32, od=f32, count=2, max_norm=1.0, ws=P, norm=P):
        return lib.sgg_clip_grads(g, out, n, gd, od, count, max_norm, 1.0, ws, norm, None)
    for bad in (dict(g=None), dict(g=null), dict(out=null), dict(n=None), dict(n=neg), dict(gd=None), dict(od=None), dict(count=-1), dict(max_norm=-1.0),
                dict(max_norm=float('nan')), dict(ws=None), dict(norm=None), dict(n=(ctypes.c_int64 * 2)(1 << 62, 1 << 62)),
                dict(g=(ctypes.c_void_p * 2)(P, P), out=(ctypes.c_void_p * 2)(P, P)), dict(g=(ctypes.c_void_p * 2)(P, P + 16), out=(ctypes.c_void_p * 2)(P, P + 16)),
                dict(out=(ctypes.c_void_p * 2)(P + 4, 2 * P)), dict(gd=(ctypes.c_int * 2)(1, 1), od=(ctypes.c_int * 2)(2, 1))):          # shared memory
        assert c(**bad) == ERR_ARG, bad
    assert c(gd=odd) == ERR_DTYPE and c(od=odd) == ERR_DTYPE
    assert lib.sgg_clip_grads_parts(-1) == ERR_ARG and 0 < lib.sgg_clip_grads_parts(0) <= lib.sgg_clip_grads_parts(1000)


def test_cpu_tensors_are_refused():
    from sgg_amd import dense, ops
    from sgg_amd.trainer import clip_grad_norm_
    x = torch.zeros(4, 8)
    p = torch.nn.Parameter(x.clone())
    p.grad = x.clone()
    for call in (lambda: ops.layer_norm(x), lambda: dense.layer_norm(x), lambda: dense.LayerNormRows(8)(x), lambda: ops.quantize_fp8(x),
                 lambda: dense.affine_fp8(x, x), lambda: ops.layer_norm_bwd(x, x, x[:, 0], x[:, 0])):
        with pytest.raises(RuntimeError):
            call()
    for call in (lambda: ops.clip_grads_([x], 1.0), lambda: ops.grad_norm([x]), lambda: clip_grad_norm_([p], 1.0)):
        with pytest.raises(RuntimeError):
            call()


def test_operand_form_index_rule():
    """byte ((b G + m / 128) 32 + m % 32) 4 + (m / 32) % 4 holds the exponent of row m, block b; byte ((k / 64) R + m) 64 + k % 64 the code of row m,
    column k; values are e4m3 times 2^e"""
    from sgg_amd import ops
    M, K = 300, 200
    G, blocks = 3, 2
    gen = torch.Generator().manual_seed(0)
    e = torch.randint(-20, 20, (M, blocks), generator=gen)
    scale = torch.zeros(blocks * G * 128, dtype=torch.uint8)
    for m in range(M):
        for b in range(blocks):
            scale[((b * G + m // 128) * 32 + m % 32) * 4 + m // 32 % 4] = int(e[m, b]) + 127
    data = torch.randint(0, 127, (M, 256), dtype=torch.uint8, generator=gen).view(torch.float8_e4m3fn)
    slabs = torch.zeros(4 * 300 * 64, dtype=torch.uint8)
    for k in range(256):
        slabs[(k // 64 * 300 + torch.arange(M)) * 64 + k % 64] = data.view(torch.uint8)[:, k]
    q = ops.Fp8Rows(slabs.view(torch.float8_e4m3fn).view(4, 300, 64), scale, (M, K))
    assert torch.equal(q.codes().view(torch.uint8), data.view(torch.uint8))
    assert torch.equal(q.exponents(), e.int())
    want = data.double() * (2.0 ** e.double()).repeat_interleave(128, 1)
    assert q.dequantize().shape == (M, K) and torch.equal(q.dequantize().double(), want[:, :K])


def test_layers_and_modes():
    from sgg_amd import dense
    from sgg_amd.gan_ops import build_mlp
    net = build_mlp([6, 9, 4], batch_norm='layer')
    kinds = [type(m).__name__ for m in net]
    assert kinds == ['Linear', 'LayerNormRows', 'ReLU', 'Linear', 'LayerNormRows', 'ReLU']
    assert sorted(net.state_dict()) == sorted('%d.%s' % (i, k) for i in (0, 1, 3, 4) for k in ('weight', 'bias'))
    assert [type(m).__name__ for m in build_mlp([6, 9, 4], batch_norm='batch')][1] == 'BatchNormRows'
    prev = dense.set_compute('fp8')
    assert dense.compute_mode() == 'fp8' and dense.set_compute(prev) == 'fp8'
    assert dense.LayerNormRows(5, elementwise_affine=False).weight is None
