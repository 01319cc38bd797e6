"""Edges of the packed-batch operators on the GPU: how exact the gate's gradient is, data at any address, infinities,
offsets beyond the rows, places without an entry.  Tolerances count roundings (see packed_ref.py)."""
import ctypes

import pytest
import torch

import cabi
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


def at_offset(t, nbytes):
    """The tensor's values `nbytes` behind a 256-byte boundary, with as much room behind them."""
    n = t.numel() * t.element_size()
    buf = torch.zeros(n + nbytes + 256, dtype=torch.uint8, device='cuda')
    room = buf[nbytes:nbytes + n].view(t.dtype)
    assert buf.data_ptr() % 256 == 0 and room.data_ptr() % 256 == nbytes
    return room.view(t.shape).copy_(t)


@pytest.mark.parametrize('dtype,gdtype', [(BF16, F32), (BF16, BF16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize('heads,width', [(3, 6), (2, 8), (1, 33), (24, 1)])
@pytest.mark.parametrize('data_off,h_off', [(0, 4), (0, 8), (4, 4), (4, 8), (8, 12), (4, 16)])
def test_raw_pointers_at_any_address_of_their_type(data_off, h_off, heads, width, dtype, gdtype):
    """The C entries, with every array where its type alone allows it and h (fp32) on another boundary than the data: two
    16-bit channels are 4 bytes, two of h are 8."""
    gen = torch.Generator().manual_seed(heads + width)
    E, K, ends = 170, heads * width, [0, 60, 170]
    src, grad = rand(gen, E, heads, width, dtype=dtype), rand(gen, E, heads, width, dtype=dtype)
    gate = torch.sigmoid(rand(gen, E, heads, 1) + 2).to(gdtype)
    x, d, g = at_offset(src, data_off), at_offset(grad, data_off), at_offset(gate, 4)
    out, dx, dg = at_offset(torch.zeros_like(src), data_off), at_offset(torch.zeros_like(src), data_off), at_offset(torch.zeros_like(gate), 4)
    wide = at_offset(torch.zeros(E, K), h_off) if dtype != F32 else None
    p, lib, dt = torch.tensor(ends, device='cuda'), cabi.lib(), (cabi.DTYPE[dtype], cabi.DTYPE[gdtype])
    shape = [cabi._i(v) for v in (1, E, K, 2, width, 0)]
    ptr = cabi._p
    cabi._check(lib.tsb_scan_csr(ptr(x), ptr(g), ptr(p), None, ptr(out), None, ptr(wide), *shape, *dt, cabi._stream()), 'tsb_scan_csr')
    h = wide if wide is not None else at_offset(out.cpu(), h_off)
    need = lib.tsb_scan_csr_backward_workspace_bytes
    need.restype = ctypes.c_size_t
    n = need(*shape[:5], *dt)
    ws = torch.empty(n + 1, dtype=torch.uint8, device='cuda')
    cabi._check(lib.tsb_scan_csr_backward(ptr(d), None, ptr(g), ptr(h), ptr(p), None, ptr(dx), ptr(dg), None, *shape, *dt, ptr(ws),
                                          ctypes.c_size_t(n), cabi._stream()), 'tsb_scan_csr_backward')
    torch.cuda.synchronize()
    flat = lambda t: t.double().expand(E, heads, width).reshape(E, K)  # noqa: E731
    want, before, _, mass, way = ref.scan(flat(src), flat(gate), ends, None)
    dh, _, _, dmass, dway, _, _ = ref.scan_backward(flat(grad), None, flat(gate), before, ends)
    u = ref.unit(F32)
    ref.assert_within(out.reshape(E, K), want, u * (4 * way + 32 * mass) + ref.last_rounding(want, dtype), 'out')
    ref.assert_within(h.reshape(E, K), want, u * (4 * way + 32 * mass), 'h')
    ref.assert_within(dx.reshape(E, K), dh, u * (4 * dway + 32 * dmass) + ref.last_rounding(dh, dtype), 'grad_src')
    total, err = gate_gradient(src, gate, grad, ends)
    ref.assert_within(dg, total, err + ref.last_rounding(total, gdtype), 'grad_gate')


def test_tangents_of_incoming_gradients_raise():
    """Forward over reverse: a backward pass whose incoming gradient carries a tangent."""
    fwd = torch.autograd.forward_ad
    slot, _, p = ts.expert_sort(torch.tensor([[0, 1], [1, 2], [2, 0], [0, 2]], device='cuda'), 3)
    x = torch.randn(4, 6, device='cuda', requires_grad=True)
    for f in (lambda: ts.expert_topk(x, 2)[0], lambda: ts.expert_dispatch(x, slot, p), lambda: ts.expert_combine(torch.cat([x, x]), slot, p),
              lambda: ts.scan_csr(x, torch.sigmoid(x), torch.tensor([0, 1, 4], device='cuda'))):
        with fwd.dual_level():
            y = f()
            for again in (False, True):
                g = fwd.make_dual(torch.ones_like(y), torch.ones_like(y))
                with pytest.raises(RuntimeError, match='forward-mode|jvp'):
                    torch.autograd.grad(y, x, g, retain_graph=True, create_graph=again)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('shape,gate_shape', [((4, 3, 0), (4, 3, 1)), ((4, 0, 5), (4, 1, 1)), ((4, 0, 5), (4, 0, 1)), ((4, 3, 0), (4, 1, 1)),
                                              ((0, 3, 0), (0, 3, 1)), ((4, 3, 0), (4, 3, 0)), ((4, 0), (4, 1))])
def test_scan_of_no_channels(shape, gate_shape, dtype):
    """Shared gates of rows without channels: empty outputs, and gradients of zero where the gates exist."""
    p = torch.tensor([0, shape[0] // 2, shape[0]], device='cuda')
    src = torch.zeros(shape, dtype=dtype, device='cuda', requires_grad=True)
    gate = torch.ones(gate_shape, dtype=dtype, device='cuda', requires_grad=True)
    state = torch.zeros((2,) + shape[1:], device='cuda', requires_grad=True)
    out, last = ts.scan_csr_state(src, gate, p, state)
    assert out.shape == shape and out.dtype == dtype and last.shape == state.shape
    assert ts.scan_csr(src.detach(), gate.detach(), p).shape == shape
    torch.full((64,), float('nan'), device='cuda')  # (what a gradient left unwritten might hold)
    gs, gg, gst = torch.autograd.grad((out, last), (src, gate, state), (torch.ones_like(out), torch.ones_like(last)))
    assert gs.shape == shape and gst.shape == state.shape and torch.equal(gg, torch.zeros_like(gate))
    if shape[0]:
        with torch.no_grad():
            assert ts.scan_step(src[:2], gate[:2], state.detach()).shape == (2,) + shape[1:]


def same_kind(got, want, what):
    """NaN, +inf and -inf at the same places."""
    got = got.detach().cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), f'{what}: NaN'
    assert torch.equal(got == float('inf'), want == float('inf')) and torch.equal(got == -float('inf'), want == -float('inf')), f'{what}: infinities'


@pytest.mark.parametrize('dtype', [F32, BF16, F64])
@pytest.mark.parametrize('heads,width', [(40, 1), (7, 1), (3, 16), (1, 33)])
@pytest.mark.parametrize('decay', [0.5, -0.5, 1e-3, 1e-12, 0.0])
def test_infinite_values_stay_infinite(decay, heads, width, dtype):
    """An infinity stays one under gates that are not 0, however small their product; a gate of 0 makes it NaN.  Over
    sequences that a thread, a tile and a cluster of tiles hold."""
    gen = torch.Generator().manual_seed(heads)
    ends, H, P = [0, 12, 400, 6400], heads, width
    E, inf = ends[-1], float('inf')
    src, grad = rand(gen, E, H, P, dtype=dtype), rand(gen, E, H, P, dtype=dtype)
    gate = torch.full((E, H, 1), 0.75).to(dtype)
    gate[::3] = decay if decay else 0.75
    if not decay:
        gate[[8, 300, 3000]] = 0.0
    for lo, hi in zip(ends[:-1], ends[1:]):
        src[lo + (hi - lo) // 4, 0, 0], src[lo + (hi - lo) // 2, H - 1, P - 1] = inf, -inf
        grad[hi - 1 - (hi - lo) // 4, 0, 0], grad[hi - 1 - (hi - lo) // 2, H - 1, P - 1] = -inf, inf
    flat = lambda t: t.double().expand(E, H, P).reshape(E, H * P)  # noqa: E731
    want, before, last, mass, way = ref.scan(flat(src), flat(gate), ends, None)
    dh, dg, _, dmass, dway, _, _ = ref.scan_backward(flat(grad), None, flat(gate), before, ends)
    assert bool(want.isinf().any()) and bool(dh.isinf().any()) and bool(want.isnan().any()) == (decay == 0)
    xs, xg = src.cuda().requires_grad_(), gate.cuda().requires_grad_()
    out, state = ts.scan_csr_state(xs, xg, torch.tensor(ends, device='cuda'))
    gs, gg = torch.autograd.grad(out, (xs, xg), grad.cuda())
    same_kind(out.reshape(E, H * P), want, 'out')
    same_kind(state.reshape(3, H * P), last, 'last')
    same_kind(gs.reshape(E, H * P), dh, 'grad_src')
    # An infinite dh times an h whose roundings reach 0 may be infinite or NaN, and so may an infinite h times such a dh:
    # with bf16 data 0.75 a + b is exactly 0 for some a and b, and the 1e-12 of the row before them, which 64 bits still hold
    # next to a, is below half a step of 32 bits.  Both are within u (4 way + 32 mass) of their values, so only where that
    # reaches 0 is nothing asked.
    u = ref.unit(dtype)
    may_be_0 = lambda v, by: v.isfinite() & (v != 0) & (v.abs() <= by)  # noqa: E731
    unsure = dh.isinf() & may_be_0(before, torch.roll(u * (4 * way + 32 * mass), 1, 0))
    unsure |= before.isinf() & may_be_0(dh, u * (4 * dway + 32 * dmass))
    assert int(unsure.sum()) < unsure.numel() // 100
    sure = ~unsure.reshape(E, H, P).any(-1, keepdim=True)
    same_kind(gg.cpu()[sure], dg.reshape(E, H, P).sum(-1, keepdim=True)[sure], 'grad_gate')


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('K', [64, 7])
@pytest.mark.parametrize('ends', [[-3, 20, 90, 130], [-9, -4, 100, 300], [0, 40, 128, 129, 140], [-50, 200], [130, 140], [-7, -2, 0, 100]])
def test_scan_offsets_beyond_the_rows(ends, K, dtype):
    """A segment that reaches over the rows' ends is what of it lies inside, as in segment_csr: its state comes in at its
    first row, its last state and the gradient of its state are written."""
    gen = torch.Generator().manual_seed(K)
    E, N = 100, len(ends) - 1
    inside = [min(max(e, 0), E) for e in ends]
    src, grad = rand(gen, E, K, dtype=dtype).cuda(), rand(gen, E, K, dtype=dtype).cuda()
    gate = torch.sigmoid(rand(gen, E, K)).to(dtype).cuda()
    state, grad_last = rand(gen, N, K).cuda(), rand(gen, N, K).cuda()

    def both(offsets):
        leaves = [t.clone().requires_grad_() for t in (src, gate, state)]
        out, last = ts.scan_csr_state(leaves[0], leaves[1], torch.tensor(offsets, device='cuda'), leaves[2])
        return (out.detach(), last.detach()) + torch.autograd.grad((out, last), leaves, (grad, grad_last))

    for got, want, what in zip(both(ends), both(inside), ('out', 'last', 'grad_src', 'grad_gate', 'grad_state')):
        assert torch.equal(got, want), what


def leave_nan(*sizes):
    """Memory of these sizes (bytes) that the next allocations will probably get, full of NaN."""
    blocks = [torch.full((n // 4 + 1,), float('nan'), device='cuda') for n in sizes]
    torch.cuda.synchronize()
    del blocks


@pytest.mark.parametrize('dtype', [F32, BF16, F64])
@pytest.mark.parametrize('T,k,K', [(1, 1, 5), (6, 2, 64), (40, 3, 129), (700, 8, 256), (1000, 8, 33), (1025, 8, 40), (30000, 4, 16), (9000, 2, 7),
                                   (2400, 2, 1032), (2400, 8, 520)])
@pytest.mark.parametrize('drop', ['some', 'one expert', 'all'])
def test_rows_that_no_entry_names_are_zero(T, k, K, drop, dtype):
    """Entries dropped after the sort, as a capacity limit does it: holes among the rows, in few and many entries, in every
    way that the rows move (with and without weights, with their gradient, rows off a 16-byte boundary)."""
    gen = torch.Generator().manual_seed(T + k + K)
    index = torch.randint(-1, 7, (T, k), generator=gen)
    slot, _, indptr = ts.expert_sort(index.cuda(), 7)
    gone = {'some': torch.rand(T, k, generator=gen) < 0.3, 'one expert': index == 3, 'all': torch.ones(T, k, dtype=torch.bool)}[drop]
    slot = slot.masked_fill(gone.cuda(), -1)
    named = torch.zeros(T * k, dtype=torch.bool, device='cuda')
    named[slot[slot >= 0]] = True
    acc = F64 if dtype == F64 else F32
    few, many = rand(gen, T, K, dtype=dtype).cuda(), rand(gen, T * k, K, dtype=dtype).cuda()
    weight = rand(gen, T, k, dtype=acc).cuda()
    size = many.numel() * many.element_size()
    rows_of = torch.zeros(T * k, dtype=torch.long, device='cuda')
    rows_of[slot[slot >= 0]] = torch.arange(T, device='cuda').repeat_interleave(k).view(T, k)[slot >= 0]
    for w in (None, weight):
        leave_nan(size, size)
        rows = ts.expert_dispatch(few, slot, indptr, w)
        assert not bool(rows[~named].any())
        if w is None:
            assert torch.equal(rows[named], few[rows_of[named]])
    for w, dots in ((None, False), (weight, False), (weight, True)):
        leaf = many.clone().requires_grad_()
        wl = None if w is None else w.clone().requires_grad_(dots)
        out = ts.expert_combine(leaf, slot, indptr, wl)
        leave_nan(size, size)
        grads = torch.autograd.grad(out, [leaf] + ([wl] if dots else []), few)
        assert not bool(grads[0][~named].any())
        if w is None:
            assert torch.equal(grads[0][named], few[rows_of[named]])
        if dots:
            assert bool((grads[1][slot < 0] == 0).all())


@pytest.mark.parametrize('T,k,K', [(300, 4, 64), (4000, 4, 72), (4000, 4, 1024)])
def test_dropped_entries_captured_and_on_two_streams(T, k, K):
    """Plans with holes in a captured graph that is replayed with other slots, followed at once by a kernel that reads the
    rows; two streams at a time."""
    gen = torch.Generator().manual_seed(K)
    x, w = rand(gen, T, K, dtype=BF16).cuda(), rand(gen, T, k).cuda()
    many = rand(gen, T * k, K, dtype=BF16).cuda().requires_grad_()
    plans = []
    for i in range(3):
        slot, _, p = ts.expert_sort(torch.randint(-i, 9, (T, k), generator=gen).cuda(), 9)
        plans.append((slot.masked_fill(torch.rand(T, k, generator=gen).cuda() < 0.2 * i, -1), p))
    at, ptr = plans[0][0].clone(), plans[0][1].clone()

    def both(slot, p):
        rows = ts.expert_dispatch(x, slot, p)
        wl = w.detach().requires_grad_()
        grads = torch.autograd.grad(ts.expert_combine(many, slot, p, wl), (many, wl), x)
        return (rows + 1,) + tuple(g + 1 for g in grads)  # (a kernel that reads them at once)

    def plain(slot, p):
        named = slot >= 0
        rows, grad = torch.zeros(T * k, K, dtype=BF16, device='cuda'), torch.zeros(T * k, K, dtype=BF16, device='cuda')
        token = torch.arange(T, device='cuda').repeat_interleave(k).view(T, k)
        rows[slot[named]] = x[token[named]]
        grad[slot[named]] = (x[token[named]].float() * w[named].unsqueeze(1)).to(BF16)
        return rows + 1, grad + 1

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(at, ptr)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(at, ptr)
    for slot, p in plans + plans[::-1]:
        at.copy_(slot)
        ptr.copy_(p)
        leave_nan(2 * T * k * K)
        graph.replay()
        for got, want in zip(out, plain(slot, p)):
            assert torch.equal(got, want)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for stream, plan in zip(streams * 3, plans * 2):
        with torch.cuda.stream(stream):
            outs.append(both(*plan))
    torch.cuda.synchronize()
    for got, plan in zip(outs, plans * 2):
        for a, b in zip(got, plain(*plan)):
            assert torch.equal(a, b)


def test_step_on_overlapping_memory():
    """The state itself as src or gate is fine; other values of its memory would be read before or after they change."""
    buf = torch.rand(24, device='cuda')
    state, x, g = buf[:16].view(2, 8), torch.rand(2, 8, device='cuda'), torch.rand(2, 8, device='cuda')
    for src, gate in ((buf[8:].view(2, 8), g), (x, buf[4:20].view(2, 8)), (x, buf[2:4].view(2, 1)), (buf[1:17].view(2, 8), g)):
        before = buf.clone()
        with pytest.raises(RuntimeError, match='overlap'):
            ts.scan_step(src, gate, state)
        assert torch.equal(buf, before)
    u = ref.unit(F32)
    for src, gate in ((state, g), (x, state)):
        s64, g64, h64 = src.double().cpu(), gate.double().cpu(), state.double().cpu()
        want = g64 * h64 + s64
        out = ts.scan_step(src, gate, state)
        tol = 2 * u * ((g64 * h64).abs() + s64.abs())
        ref.assert_within(state, want, tol, 'state')
        ref.assert_within(out, want, tol, 'out')


def test_more_elements_than_32_bits_count():
    """The last segment, and the last tokens, of arrays of more than 2^31 elements: the bits of the same rows by themselves."""
    gen = torch.Generator(device='cuda').manual_seed(1)
    E, tail = 66000, 500
    for K in (33000, 32997):  # 2.18e9 elements, rows on a 16-byte boundary and off it
        src = torch.rand(E, K, device='cuda', generator=gen, dtype=BF16)
        gate = torch.rand(E, K, device='cuda', generator=gen, dtype=BF16)
        p = torch.tensor([0, 3, E - tail, E], device='cuda')
        out = ts.scan_csr(src.requires_grad_(), gate.requires_grad_(), p)
        gs, gg = torch.autograd.grad(out, (src, gate), out.detach())
        with torch.no_grad():
            x, g = src[-tail:].clone().requires_grad_(), gate[-tail:].clone().requires_grad_()
        # (cut into other tiles, so the roundings differ: both within a bf16 step of the exact values)
        few = ts.scan_csr(x, g, torch.tensor([0, tail], device='cuda'))
        fs, fg = torch.autograd.grad(few, (x, g), few.detach())
        for a, b in ((out[-tail:], few), (gs[-tail:], fs), (gg[-tail:], fg)):
            assert bool(((a.float() - b.float()).abs() <= 2.0 ** -6 * b.float().abs()).all())
        del src, gate, out, gs, gg
    T, k, K = 140000, 8, 2048  # 2.29e9 elements of rows
    slot, order, ptr = ts.expert_sort(torch.randint(-1, 16, (T, k), device='cuda', generator=gen), 16)
    x = torch.rand(T, K, device='cuda', generator=gen, dtype=BF16)
    rows = ts.expert_dispatch(x, slot, ptr)
    used = int(ptr[-1])
    assert not bool(rows[used:].any())
    for places in (slice(0, 1000), slice(used - 1000, used)):
        assert torch.equal(rows[places], x[order[places] // k])
    slot[-3:, :] = -1  # holes far behind
    rows = ts.expert_dispatch(x, slot, ptr)
    named = torch.zeros(T * k, dtype=torch.bool, device='cuda')
    named[slot[slot >= 0]] = True
    assert not bool(rows[~named].any())
    w = torch.rand(T, k, device='cuda', generator=gen)
    out = ts.expert_combine(rows, slot, ptr, w)
    want = (rows[slot[-1003:-3].clamp_min(0)].double() * (w[-1003:-3] * (slot[-1003:-3] >= 0)).double().unsqueeze(-1)).sum(1)
    assert bool(((out[-1003:-3].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * want.abs()).all()) and not bool(out[-3:].any())


def test_16_bit_recurrence_compiles():
    """A traced training step keeps h in fp32 as the eager one does."""
    gen = torch.Generator().manual_seed(3)
    p = torch.tensor([0, 30, 31, 100], device='cuda')
    x, g, s = rand(gen, 100, 24, dtype=BF16).cuda(), torch.sigmoid(rand(gen, 100, 24) + 1).to(BF16).cuda(), rand(gen, 3, 24).cuda()
    d = rand(gen, 100, 24, dtype=BF16).cuda()

    def step(f):
        leaves = [t.clone().requires_grad_() for t in (x, g, s)]
        out, last = f(*leaves)
        return (out.detach(), last.detach()) + torch.autograd.grad((out, last), leaves, (d, torch.ones_like(last)))

    f = lambda a, b, c: ts.scan_csr_state(a, b, p, c)  # noqa: E731
    for got, want in zip(step(torch.compile(f, fullgraph=True)), step(f)):
        assert torch.equal(got, want)
