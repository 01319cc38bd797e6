"""Host-side contract of the packed-batch operators (expert_*, scan_*), checked without a GPU: names, TorchScript,
shapes on fake tensors, and the calls they refuse."""
import ctypes
import os.path as osp

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import pytorch_scatter_b200 as ts

LIB = osp.join(osp.dirname(osp.dirname(osp.abspath(__file__))), 'pytorch_scatter_b200', 'libtsb200.so')
NAMES = ['expert_topk', 'expert_sort', 'expert_dispatch', 'expert_combine', 'scan_csr', 'scan_csr_state', 'scan_step']


@pytest.mark.parametrize('name', NAMES)
def test_names_and_torchscript(name):
    assert name in ts.__all__
    assert torch.jit.script(getattr(ts, name)) is not None


def test_cpu_tensors_fail_loudly():
    x, i = torch.randn(4, 2), torch.zeros(4, 1, dtype=torch.long)
    p = torch.tensor([0, 4])
    for fn in (lambda: ts.expert_topk(x, 1), lambda: ts.expert_sort(i, 2), lambda: ts.expert_dispatch(x, i, p),
               lambda: ts.expert_combine(x, i, p), lambda: ts.scan_csr(x, x, p), lambda: ts.scan_csr_state(x, x, p),
               lambda: ts.scan_step(x, x, x)):
        with pytest.raises(RuntimeError, match='must be CUDA tensor'):
            fn()


def cuda(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device='cuda')


def test_fake_tensor_shapes():
    with FakeTensorMode():
        bf16, f64, i64 = torch.bfloat16, torch.float64, torch.long
        w, i = ts.expert_topk(cuda(5, 7, 16, dtype=bf16), 3)
        assert w.shape == i.shape == (5, 7, 3) and w.dtype == torch.float32 and i.dtype == i64
        slot, order, indptr = ts.expert_sort(i, 16)
        assert slot.shape == (5, 7, 3) and order.shape == (105,) and indptr.shape == (17,)
        rows = ts.expert_dispatch(cuda(5, 7, 4, 8, dtype=bf16), slot, indptr, w)
        assert rows.shape == (105, 4, 8) and rows.dtype == bf16
        out = ts.expert_combine(rows, slot, indptr, w)
        assert out.shape == (5, 7, 4, 8) and out.dtype == bf16
        src, gate, p = cuda(3, 50, 4, 8, dtype=bf16), cuda(3, 50, 4, 1), cuda(1, 6, dtype=i64)
        assert ts.scan_csr(src, gate, p).shape == src.shape
        out, last = ts.scan_csr_state(src, gate, p, cuda(3, 5, 4, 8))
        assert out.dtype == bf16 and last.shape == (3, 5, 4, 8) and last.dtype == torch.float32
        out, last = ts.scan_csr_state(cuda(9, 2, dtype=f64), cuda(9, 2, dtype=f64), cuda(4, dtype=i64))
        assert last.shape == (3, 2) and last.dtype == f64
        assert ts.scan_step(cuda(3, 4, dtype=bf16), cuda(3, 1, dtype=bf16), cuda(3, 4)).shape == (3, 4)


def refusals():
    i64, f64, bf16 = torch.long, torch.float64, torch.bfloat16
    x, slot, p, w = cuda(6, 8), cuda(6, 2, dtype=i64), cuda(4, dtype=i64), cuda(6, 2)
    many = cuda(12, 8)
    seg = cuda(4, dtype=i64)
    return {
        'topk: integers': lambda: ts.expert_topk(cuda(4, 8, dtype=i64), 2),
        'topk: float64': lambda: ts.expert_topk(cuda(4, 8, dtype=f64), 2),
        'topk: k above experts': lambda: ts.expert_topk(cuda(4, 8), 9),
        'topk: k = 0': lambda: ts.expert_topk(cuda(4, 8), 0),
        'topk: no experts': lambda: ts.expert_topk(cuda(4, 0), 1),
        'topk: 1025 experts': lambda: ts.expert_topk(cuda(4, 1025), 1),
        'topk: a number': lambda: ts.expert_topk(cuda(), 1),
        'sort: int32': lambda: ts.expert_sort(cuda(4, 2, dtype=torch.int32), 4),
        'sort: no experts': lambda: ts.expert_sort(slot, 0),
        'sort: 4097 experts': lambda: ts.expert_sort(slot, 4097),
        'dispatch: integers': lambda: ts.expert_dispatch(cuda(6, 8, dtype=i64), slot, p),
        'dispatch: slot without k': lambda: ts.expert_dispatch(x, cuda(6, dtype=i64), p),
        'dispatch: other tokens': lambda: ts.expert_dispatch(cuda(5, 8), slot, p),
        'dispatch: int32 slot': lambda: ts.expert_dispatch(x, cuda(6, 2, dtype=torch.int32), p),
        'dispatch: empty indptr': lambda: ts.expert_dispatch(x, slot, cuda(0, dtype=i64)),
        'dispatch: weight shape': lambda: ts.expert_dispatch(x, slot, p, cuda(6, 1)),
        'dispatch: weight type': lambda: ts.expert_dispatch(cuda(6, 8, dtype=bf16), slot, p, cuda(6, 2, dtype=bf16)),
        'dispatch: weight type with float64': lambda: ts.expert_dispatch(cuda(6, 8, dtype=f64), slot, p, w),
        'combine: too few rows': lambda: ts.expert_combine(cuda(11, 8), slot, p, w),
        'combine: 2-D indptr': lambda: ts.expert_combine(many, slot, cuda(1, 4, dtype=i64), w),
        'scan: integers': lambda: ts.scan_csr(cuda(6, 8, dtype=i64), cuda(6, 8, dtype=i64), seg),
        'scan: int32 indptr': lambda: ts.scan_csr(x, x, cuda(4, dtype=torch.int32)),
        'scan: empty indptr': lambda: ts.scan_csr(x, x, cuda(0, dtype=i64)),
        'scan: gate of fewer dimensions': lambda: ts.scan_csr(x, cuda(6), seg),
        'scan: gate of another shape': lambda: ts.scan_csr(x, cuda(6, 4), seg),
        'scan: 16-bit gate with float32': lambda: ts.scan_csr(x, cuda(6, 8, dtype=bf16), seg),
        'scan: float32 gate with float64': lambda: ts.scan_csr(cuda(6, 8, dtype=f64), x, seg),
        'scan: state of 16 bits': lambda: ts.scan_csr(cuda(6, 8, dtype=bf16), cuda(6, 8), seg, cuda(3, 8, dtype=bf16)),
        'scan: state of another shape': lambda: ts.scan_csr(x, x, seg, cuda(4, 8)),
        'scan: more dimensions in indptr': lambda: ts.scan_csr(cuda(6), cuda(6), cuda(6, 4, dtype=i64)),
        'scan: batch of indptr': lambda: ts.scan_csr(cuda(2, 6, 8), cuda(2, 6, 8), cuda(3, 4, dtype=i64)),
        'step: state shape': lambda: ts.scan_step(x, x, cuda(5, 8)),
        'step: state type': lambda: ts.scan_step(x, x, cuda(6, 8, dtype=bf16)),
        'step: needs a gradient': lambda: ts.scan_step(cuda(6, 8).requires_grad_(), x, cuda(6, 8)),
        'step: overlapping states': lambda: ts.scan_step(x, x, cuda(1, 8).expand(6, 8)),
        'step: state with strides': lambda: ts.scan_step(x, x, cuda(8, 6).t()),
    }


with FakeTensorMode():
    REFUSED = sorted(refusals())


@pytest.mark.parametrize('what', REFUSED)
def test_refusals(what):
    with FakeTensorMode():
        with pytest.raises((RuntimeError, ValueError)):
            refusals()[what]()


def test_c_entries_report_errors_before_any_launch():
    lib = ctypes.CDLL(LIB)
    I, P = ctypes.c_int64, ctypes.c_void_p(256)  # never dereferenced
    size = ctypes.c_size_t
    assert lib.tsb_expert_topk(P, P, P, I(4), I(8), I(9), 0, 0, None) == 3
    assert lib.tsb_expert_topk(P, P, P, I(4), I(2000), I(2), 0, 0, None) == 6
    assert lib.tsb_expert_topk(P, P, P, I(4), I(8), I(2), 0, 1, None) == 1
    assert lib.tsb_expert_topk(None, P, P, I(4), I(8), I(2), 0, 0, None) == 3
    assert lib.tsb_expert_topk(None, None, None, I(0), I(8), I(2), 0, 0, None) == 0
    assert lib.tsb_expert_topk_backward(P, P, P, None, P, I(4), I(8), I(2), 0, 0, None) == 3
    assert lib.tsb_expert_sort(P, P, P, P, I(-1), I(8), P, size(1 << 20), None) == 3
    assert lib.tsb_expert_sort(P, P, P, P, I(10), I(5000), P, size(1 << 20), None) == 6
    assert lib.tsb_expert_sort(P, P, P, P, I(1 << 31), I(8), P, size(1 << 20), None) == 6
    assert lib.tsb_expert_sort(P, None, P, P, I(10), I(8), P, size(1 << 20), None) == 3
    assert lib.tsb_expert_spread(P, P, P, None, P, P, None, I(4), I(2), I(8), 0, None) == 3
    assert lib.tsb_expert_spread(P, P, P, None, None, P, None, I(4), I(0), I(8), 0, None) == 3
    assert lib.tsb_expert_spread(P, P, P, None, None, P, None, I(4), I(2), I(8), 4, None) == 1
    assert lib.tsb_expert_fold(P, None, None, None, P, None, I(4), I(2), I(8), 0, None) == 3
    assert lib.tsb_expert_fold(P, P, None, None, P, P, I(4), I(2), I(8), 0, None) == 3
    assert lib.tsb_expert_fold(None, None, None, None, None, None, I(0), I(2), I(8), 0, None) == 0
    shape = (I(1), I(6), I(8), I(3))
    assert lib.tsb_scan_csr(P, P, P, None, P, None, None, *shape, I(3), I(0), 0, 0, None) == 3
    assert lib.tsb_scan_csr(P, P, P, None, P, None, None, *shape, I(1), I(0), 0, 3, None) == 1
    assert lib.tsb_scan_csr(P, P, None, None, P, None, None, *shape, I(1), I(0), 0, 0, None) == 3
    assert lib.tsb_scan_csr(P, P, P, None, P, None, P, *shape, I(1), I(0), 0, 0, None) == 3
    assert lib.tsb_scan_csr_backward(P, None, P, None, P, None, P, P, None, *shape, I(1), I(0), 0, 0, P, size(1 << 20), None) == 3
    odd = (I(1), I(6), I(9), I(3))  # nine channels share a gate: their products are summed through the workspace
    assert lib.tsb_scan_csr_backward(P, None, P, P, P, None, P, P, None, *odd, I(9), I(0), 0, 0, None, size(0), None) == 4
    assert lib.tsb_scan_step(P, P, P, P, I(4), I(8), I(1), I(7), 0, 0, None) == 3
    assert lib.tsb_scan_step(P, P, P, P, I(4), I(8), I(1), I(8), 4, 4, None) == 1
    assert lib.tsb_scan_step(None, None, None, None, I(0), I(8), I(1), I(8), 0, 0, None) == 0
