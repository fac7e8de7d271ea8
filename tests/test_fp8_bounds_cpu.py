"""The bound that 16-bit results of the 8-bit products are held to (tests/fp8_bounds.py) sees the mistakes that such a kernel makes: planted in the
result here, on the CPU."""
import pytest
import torch

from .fp8_bounds import inside


@pytest.mark.parametrize('out', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('K', [130, 1100, 12544])
@pytest.mark.parametrize('spread', [0.0, 1.0])
def test_planted_mistakes_are_outside(K, spread, out):
    torch.manual_seed(K)
    M, N = 70, 90
    blocks = (K + 127) // 128

    def operand(rows):
        x = torch.randn(rows, K).double() * torch.exp2(spread * torch.randn(rows, K).double())
        e = torch.floor(torch.log2(torch.nn.functional.pad(x.abs(), (0, -K % 128)).view(rows, blocks, 128).amax(2))) - 8
        step = torch.exp2(torch.floor(torch.log2(x.abs())) - 3)
        return torch.round(x / step) * step, e
    (a, ea), (w, ew) = operand(M), operand(N)
    right = torch.mm(a, w.t())
    ok, share = inside(right.to(out), a, ea, w, ew)
    assert ok, share
    short = right - torch.mm(a[:, (K - 1) // 128 * 128:], w[:, (K - 1) // 128 * 128:].t())    # the last block of K is not there
    assert not inside(short.to(out), a, ea, w, ew)[0]
    assert not inside((right * 1.02).to(out), a, ea, w, ew)[0]
    row = right.clone()
    row[M - 1] = right[M - 2]                                                               # one row is another's
    assert not inside(row.to(out), a, ea, w, ew)[0]
    column = right.clone()
    column[:, N - 1] = 0
    assert not inside(column.to(out), a, ea, w, ew)[0]
    scale = right.clone()
    scale[:32] += torch.mm(a[:32, :128], w[:, :128].t())                                    # one block's scale of 32 rows is twice what it should be
    assert not inside(scale.to(out), a, ea, w, ew)[0]
