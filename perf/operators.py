"""The cases of the operators for low-precision dense training: layer norm, the block-scaled 8-bit product, and gradient clipping.

`own` False: plain torch forms in 32 bits.  `own` True: the calls a user makes of sgg_amd.  `exact`: the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}
EPS = 1e-5
BLOCK = 128

# the trainable tensors of the relation head, in elements: fc6 / fc7 of the edge and the object branch with their biases, the heads, the
# unary layers, the two GRU cells, the rect convolution with its norms and the gates (247.75 M parameters in all)
HEAD = ('102760448,4096,16777216,4096,102760448,4096,16777216,4096,25088,256,256,256,1179648,512,512,512,26112,51,77312,151,'
        '2097152,512,2097152,512,786432,786432,1536,1536,786432,786432,1536,1536,1024,1,1024,1,1024,1,1024,1')


def listed():
    return [
        # one object's 512-wide state normalised while answering: nothing but latency
        {'name': 'norm_one_row', 'op': 'layernorm', 'rows': 1, 'cols': 512, 'type': 'float32', 'grad': False},
        # the edge states of 8 images of 992 candidate edges, hidden width 512, in a training step
        {'name': 'norm_edges', 'op': 'layernorm', 'rows': 7936, 'cols': 512, 'type': 'float16', 'grad': True},
        # a ragged batch with an odd width (embedding + box columns)
        {'name': 'norm_ragged', 'op': 'layernorm', 'rows': 12345, 'cols': 1001, 'type': 'float32', 'grad': True},
        # the widest rows of the head (4096) over a large batch: the bandwidth case
        {'name': 'norm_wide', 'op': 'layernorm', 'rows': 65536, 'cols': 4096, 'type': 'bfloat16', 'grad': True},
        # one box through fc6 with kept 8-bit weights: streams 103 MB of weights
        {'name': 'fp8_one_box', 'op': 'fp8', 'rows': 1, 'inner': 25088, 'outer': 4096, 'type': 'float16', 'grad': False},
        # the 256 boxes of 8 images through fc6
        {'name': 'fp8_boxes', 'op': 'fp8', 'rows': 256, 'inner': 25088, 'outer': 4096, 'type': 'float16', 'grad': False},
        # the 7936 candidate edges of 8 images through fc6: the largest product of the framework
        {'name': 'fp8_edges', 'op': 'fp8', 'rows': 7936, 'inner': 25088, 'outer': 4096, 'type': 'float16', 'grad': False},
        # fc7 of the edge branch, forward and both gradients
        {'name': 'fp8_train_edges', 'op': 'fp8', 'rows': 7936, 'inner': 4096, 'outer': 4096, 'type': 'bfloat16', 'grad': True},
        # a graph convolution's layer with odd sizes, fp32 activations
        {'name': 'fp8_train_ragged', 'op': 'fp8', 'rows': 1985, 'inner': 1100, 'outer': 333, 'type': 'float32', 'grad': True},
        # a small network's gradients
        {'name': 'clip_small', 'op': 'clip', 'sizes': '64,4096,64,4096,1,129,8193,51', 'type': 'float32', 'scale': 1.0, 'norm': 1.0},
        # a generator's half-precision gradients of a loss scaled by 1024, into fp32
        {'name': 'clip_unscale', 'op': 'clip', 'sizes': ','.join(['589824,256,2359296,512,1179647,512,33,200001'] * 4), 'type': 'float16',
         'scale': 1.0 / 1024, 'norm': 5.0},
        # every gradient of the relation head
        {'name': 'clip_head', 'op': 'clip', 'sizes': HEAD, 'type': 'float32', 'scale': 1.0, 'norm': 5.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['layernorm', 'fp8', 'fp8', 'clip'])
    name = rng.choice(sorted(TYPES))
    if kind == 'layernorm':
        cols = _log(rng, 8, 8192)
        rows = _log(rng, 1, min(65536, 65536 * 4096 // 2 // cols))
        return {'op': 'layernorm', 'rows': rows, 'cols': cols, 'type': name, 'grad': rng.random() < 0.6}
    if kind == 'fp8':
        grad = rng.random() < 0.5
        inner, outer = _log(rng, 64, 8192 if grad else 25088), _log(rng, 16, 4096)
        rows = _log(rng, 1, 7936)
        if rng.random() < 0.5:
            inner, outer = (inner + 127) // 128 * 128, (outer + 15) // 16 * 16
            inner = min(inner, 8192 if grad else 25088)
        return {'op': 'fp8', 'rows': rows, 'inner': inner, 'outer': outer, 'type': name, 'grad': grad}
    count = _log(rng, 1, 150)
    sizes = [_log(rng, 1, 1 << rng.randint(8, 21)) for _ in range(count)]
    return {'op': 'clip', 'sizes': ','.join(str(n) for n in sizes), 'type': name, 'scale': rng.choice([1.0, 1.0 / 1024]),
            'norm': rng.choice([0.1, 1.0, 5.0, 1e6])}


def _sizes(case):
    return [int(s) for s in case['sizes'].split(',')]


def _starts(case):
    at = [0]
    for n in _sizes(case):
        at.append(at[-1] + (n + 15) // 16 * 16)
    return at


def _inputs(case, seed):
    """what both sides and the exact form start from, made from the seed alone"""
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device='cuda')

    kind = TYPES[case['type']]
    if case['op'] == 'layernorm':
        M, C = case['rows'], case['cols']
        x = normal(M, C).mul_(1.5)
        x += normal(M, 1) + 0.5 * normal(1, C)                       # rows and channels with means of their own
        s = {'x': x.to(kind), 'w': 1.0 + 0.2 * normal(C), 'b': 0.2 * normal(C)}
        if case['grad']:
            s['dy'] = normal(M, C).mul_(0.1).to(kind)
        return s
    if case['op'] == 'fp8':
        M, K, N = case['rows'], case['inner'], case['outer']
        x = normal(M, K).clamp_(min=0)                               # activations after a ReLU, rows of unlike size
        x *= torch.exp2(normal(M, 1))
        s = {'x': x.to(kind), 'w': normal(N, K) / K ** 0.5, 'b': 0.1 * normal(N)}
        if case['grad']:
            s['dy'] = (1e-3 * normal(M, N) * torch.exp2(normal(M, 1))).to(kind)
        return s
    grads = [(0.02 * normal(n)) for n in _sizes(case)]
    if case['scale'] != 1.0:
        grads = [g / case['scale'] * 0.05 for g in grads]            # gradients of a scaled loss
    return {'grads': [g.to(kind) for g in grads]}


def prepare(case, seed):
    s = _inputs(case, seed)
    s['case'] = case
    if case['op'] == 'fp8' and not case['grad']:                     # weights laid out once, as a serving program keeps them
        if own:
            from sgg_amd import ops
            s['wq'] = ops.quantize_fp8(s.pop('w'))
        else:
            s['wq'] = _quantized(s.pop('w'))
    if case['op'] == 'clip':
        # the fp32 gradients lie in one flat buffer, as a bucket of an optimiser or a reduction does; each starts on a multiple of 16
        at = _starts(case)
        s['flat'] = torch.zeros(at[-1], device='cuda')
        s['out'] = [s['flat'][o:o + g.numel()] for o, g in zip(at, s['grads'])]
    if own and case.get('grad'):                                     # a training program's leaves
        for k in ('x', 'w', 'b'):
            s[k].requires_grad_()
    return s


def _pow2(e):
    """2^e in 32 bits for whole -126 <= e <= 127, exact (a power function may be off by a last bit, which decides ties)"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantized(x):
    """the values that the 8-bit rows of x stand for, in 32 bits: blocks of 128 along the row, the smallest power of two that brings the
    block's largest magnitude to 448 or less, e4m3 with round to nearest even"""
    M, K = x.shape
    pad = -K % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(M, -1, BLOCK)
    m, e = torch.frexp(v.abs().amax(2, keepdim=True))                # max = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = (e - 9 + (m > 0.875)).clamp(min=-126)
    q = (v * _pow2(-e)).to(torch.float8_e4m3fn).float()
    return (q * _pow2(e)).view(M, -1)[:, :K]


def run(s):
    case = s['case']
    return (_run_own if own else _run_plain)(s, case)


def _run_own(s, case):
    from sgg_amd import dense, ops
    if case['op'] == 'layernorm':
        if not case['grad']:
            return {'y': dense.layer_norm(s['x'], s['w'], s['b'], EPS)}
        y = dense.layer_norm(s['x'], s['w'], s['b'], EPS)
        dx, dw, db = torch.autograd.grad(y, (s['x'], s['w'], s['b']), s['dy'])
        return {'y': y.detach(), 'dx': dx, 'dw': dw, 'db': db}
    if case['op'] == 'fp8':
        if not case['grad']:
            return {'y': ops.gemm_fp8(ops.quantize_fp8(s['x']), s['wq'], s['b'], ops.ACT_RELU, out_dtype=s['x'].dtype)}
        y = dense.affine_fp8(s['x'], s['w'], s['b'])
        dx, dw, db = torch.autograd.grad(y, (s['x'], s['w'], s['b']), s['dy'])
        return {'y': y.detach(), 'dx': dx, 'dw': dw, 'db': db}
    norm = ops.clip_grads_(s['grads'], case['norm'], grad_scale=case['scale'], out=s['out'])
    return {'norm': norm, 'grads': s['flat']}


def _run_plain(s, case):
    if case['op'] == 'layernorm':
        x, w, b = s['x'].float(), s['w'], s['b']
        mean = x.mean(1, keepdim=True)
        d = x - mean
        r = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        xh = d * r
        y = (xh * w + b).to(s['x'].dtype)
        if not case['grad']:
            return {'y': y}
        dy = s['dy'].float()
        g = dy * w
        dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return {'y': y, 'dx': dx.to(s['x'].dtype), 'dw': (dy * xh).sum(0), 'db': dy.sum(0)}
    if case['op'] == 'fp8':
        x = s['x']
        if not case['grad']:
            return {'y': (_quantized(x) @ s['wq'].t() + s['b']).clamp(min=0).to(x.dtype)}
        w, dy = s['w'], s['dy']
        y = _quantized(x) @ _quantized(w).t() + s['b']
        dx = _quantized(dy) @ _quantized(w.t()).t()
        dw = _quantized(dy.t()) @ _quantized(x.t()).t()
        return {'y': y.to(x.dtype), 'dx': dx.to(x.dtype), 'dw': dw, 'db': dy.float().sum(0)}
    total = torch.zeros((), dtype=torch.float64, device='cuda')
    for g in s['grads']:
        total = total + (g.double() * g.double()).sum()
    norm = torch.sqrt(total) * case['scale']
    c = ((case['norm'] / (norm + 1e-6)).clamp(max=1.0) * case['scale']).float()
    for g, o in zip(s['grads'], s['out']):
        o.copy_(g.float() * c)
    return {'norm': norm.float(), 'grads': s['flat']}


def work(case):
    if case['op'] == 'layernorm':
        M, C, z = case['rows'], case['cols'], SIZE[case['type']]
        if not case['grad']:
            return {'bytes': 2 * z * M * C + 8 * C, 'flops': 8 * M * C}
        return {'bytes': 4 * z * M * C + 16 * C, 'flops': 24 * M * C}           # x, dy in; y, dx, dw, db out
    if case['op'] == 'fp8':
        M, K, N, z = case['rows'], case['inner'], case['outer'], SIZE[case['type']]
        if not case['grad']:
            return {'bytes': z * M * K + N * K + N * ((K + 127) // 128) + 4 * N + z * M * N, 'flops': 2 * M * N * K}
        return {'bytes': 2 * z * M * K + 8 * N * K + 2 * z * M * N + 8 * N, 'flops': 6 * M * N * K}
    n = sum(_sizes(case))
    return {'bytes': n * (SIZE[case['type']] + 4) + 4, 'flops': 3 * n}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _two(p):
    """2^p in 64 bits, p whole numbers held as floats: the exponent field itself"""
    return ((p.long() + 1023) << 52).view(torch.float64)


def _grid8(x):
    """x in 64 bits -> what its e4m3 rows with a power of two per 128 columns stand for, from the format's definition: exponents
    -6 .. 8, three fraction bits, largest value 448, subnormal step 2^-9"""
    M, K = x.shape
    out = torch.empty_like(x)
    for k0 in range(0, K, BLOCK):
        v = x[:, k0:k0 + BLOCK]
        top = v.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0))
        e = e.clamp(min=-126.0)
        e = torch.where(top > 448.0 * _two(e), e + 1, e)                        # (a logarithm next to a whole number)
        e = torch.where(top <= 448.0 * _two(e - 1), e - 1, e).clamp(min=-126.0)
        u = v * _two(-e)
        mag = u.abs().clamp(min=2.0 ** -6)
        p = torch.floor(torch.log2(mag))
        p = torch.where(mag < _two(p), p - 1, p)
        p = torch.where(mag >= _two(p + 1), p + 1, p)
        out[:, k0:k0 + BLOCK] = torch.round(u * _two(3 - p)) * _two(p - 3) * _two(e)    # torch.round: ties to even
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    if case['op'] == 'layernorm':
        x, w, b = s.pop('x').double(), s['w'].double(), s['b'].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        xh = (x - mean).div_(torch.sqrt(var + EPS))
        del x
        out = {'y': xh * w + b}
        if case['grad']:
            dy = s.pop('dy').double()
            out['db'] = dy.sum(0)
            out['dw'] = (dy * xh).sum(0)
            g = dy.mul_(w)
            a, c = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
            out['dx'] = g.sub_(a).sub_(xh.mul_(c)).div_(torch.sqrt(var + EPS))
        return out
    if case['op'] == 'fp8':
        x, w, b = s['x'].double(), s['w'].double(), s['b'].double()
        y = torch.mm(_grid8(x), _grid8(w).t()) + b
        if not case['grad']:
            return {'y': torch.relu(y)}
        dy = s['dy'].double()
        return {'y': y, 'dx': torch.mm(_grid8(dy), _grid8(w.t().contiguous()).t()),
                'dw': torch.mm(_grid8(dy.t().contiguous()), _grid8(x.t().contiguous()).t()), 'db': dy.sum(0)}
    sq = 0.0
    for g in s['grads']:
        sq += float(g.double().square().sum())
    norm = math.sqrt(sq) * case['scale']
    c = case['scale'] * min(1.0, case['norm'] / (norm + 1e-6))
    at = _starts(case)
    flat = torch.zeros(at[-1], dtype=torch.float64, device='cuda')
    for o, g in zip(at, s['grads']):
        flat[o:o + g.numel()] = g.double() * c
    return {'norm': torch.tensor(norm, dtype=torch.float64), 'grads': flat}
