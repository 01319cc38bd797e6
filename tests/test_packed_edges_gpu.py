"""Edges of the packed-batch operators on the GPU: how exact the gate's gradient is, data at any address, infinities,
offsets beyond the rows, places without an entry.  Tolerances count roundings (see packed_ref.py)."""
import pytest
import torch

import packed_ref as ref
import pytorch_scatter_b200 as ts

pytestmark = pytest.mark.gpu

F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype)


def gate_gradient(src, gate, grad, ends):
    """The 64-bit gradient of the gate [E, heads, 1] of data [E, heads, width], and what 32-bit sums may be off by: h and dh
    within their bounds, their product and the sum over the width; no rounding of h to the data's type."""
    E, H, P = src.shape
    flat = lambda t: t.double().expand(E, H, P).reshape(E, H * P)  # noqa: E731
    h, before, _, mass, way = ref.scan(flat(src), flat(gate), ends, None)
    dh, dg, _, dmass, dway, _, _ = ref.scan_backward(flat(grad), None, flat(gate), before, ends)
    u = ref.unit(F32)
    first = torch.zeros(E, 1)
    first[[lo for lo, hi in zip(ends[:-1], ends[1:]) if hi > lo]] = 1
    err = dh.abs() * torch.roll(u * (4 * way + 32 * mass), 1, 0) * (1 - first) + u * (4 * dway + 32 * dmass) * before.abs() + u * dg.abs()
    total = lambda t: t.reshape(E, H, P).sum(-1, keepdim=True)  # noqa: E731
    return total(dg), total(err) + u * P * total(dg.abs())


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('heads,width', [(64, 1), (9, 1), (333, 1), (2, 64), (7, 8), (5, 6), (3, 33)])
def test_gate_gradient_of_16_bit_data_is_rounded_once(heads, width, dtype):
    """The backward multiplies by h as the recurrence held it: one rounding to 16 bits, that of the gradient itself."""
    gen = torch.Generator().manual_seed(heads + width)
    ends = [0, 150, 151, 151, 400]
    src, grad = rand(gen, 400, heads, width, dtype=dtype), rand(gen, 400, heads, width, dtype=dtype)
    gate = torch.sigmoid(rand(gen, 400, heads, 1) + 2).to(dtype)
    want, err = gate_gradient(src, gate, grad, ends)
    xs, xg = src.cuda().requires_grad_(), gate.cuda().requires_grad_()
    out = ts.scan_csr(xs, xg, torch.tensor(ends, device='cuda'))
    got = torch.autograd.grad(out, xg, grad.cuda())[0]
    assert got.dtype == dtype and out.dtype == dtype
    ref.assert_within(got, want, err + ref.last_rounding(want, dtype), 'grad_gate')
