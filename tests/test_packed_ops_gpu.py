"""The packed-batch operators on the GPU against plain 64-bit implementations (packed_ref.py), at the sizes, masks and
layouts where they can go wrong.  Tolerances count roundings (see packed_ref.py)."""
import math

import pytest
import torch

import packed_ref as ref
import pytorch_scatter_b200 as ts

pytestmark = pytest.mark.gpu

F32, F64, F16, BF16 = torch.float32, torch.float64, torch.float16, torch.bfloat16


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen).to(dtype)


# ---- expert_topk ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('normalize', [True, False])
@pytest.mark.parametrize('T,E,k', [(1, 1, 1), (3, 5, 5), (7, 8, 2), (33, 32, 4), (20, 33, 33), (50, 64, 6), (129, 100, 7),
                                   (64, 256, 8), (17, 257, 40), (9, 512, 16), (5, 1000, 10), (4, 1024, 1)])
def test_topk(T, E, k, normalize, dtype):
    gen = torch.Generator().manual_seed(T * 1000 + E)
    logits = (2 * rand(gen, T, E)).to(dtype)  # 16-bit values hold many ties
    if E > 2:
        logits[torch.rand(T, E, generator=gen) < 0.2] = -math.inf
        logits[::5, 2:] = -math.inf           # at most two experts left
        logits[:, 0] = 0.25                   # and at least one
    grad = rand(gen, T, k)
    want_in = logits.double().requires_grad_()
    want, index = ref.topk(want_in, k, normalize)
    (want_grad,) = torch.autograd.grad(want, want_in, grad.double())

    x = logits.cuda().requires_grad_()
    w, i = ts.expert_topk(x, k, normalize)
    (g,) = torch.autograd.grad(w, x, grad.cuda())
    assert torch.equal(i.cpu(), index) and w.dtype == F32 and g.dtype == dtype
    # a weight: difference and exponential of logits up to 10 apart (12 u + 3 u), a sum of E of them, a quotient
    want = want.detach()
    rel = ref.unit(F32) * (E + k + 40)
    ref.assert_within(w, want, want * rel + 1e-38, 'weight')
    mass = (want * grad.double()).abs().sum(1, keepdim=True)
    p = torch.softmax(want_in.detach(), 1)
    p = torch.maximum(p, torch.zeros_like(p).scatter(1, index.clamp_min(0), want))
    ref.assert_within(g, want_grad, 4 * rel * p * (mass + grad.double().abs().amax(1, keepdim=True)) + ref.last_rounding(want_grad, dtype), 'grad')


def test_topk_extremes():
    inf, low = math.inf, torch.finfo(F32).min
    x = torch.tensor([[-inf, -inf, -inf, -inf], [low, low, low, low], [inf, 0.0, 1.0, 2.0], [0.0, math.nan, 5.0, -inf],
                      [-0.0, 0.0, -inf, -1.0], [low, -inf, 3e38, 3.1e38]], device='cuda', requires_grad=True)
    w, i = ts.expert_topk(x, 2)
    assert i.tolist() == [[-1, -1], [0, 1], [0, 3], [1, 2], [0, 1], [3, 2]]
    (g,) = torch.autograd.grad(w, x, torch.tensor([1.0, 2.0], device='cuda').expand(6, 2))
    assert w[0].tolist() == [0, 0] and g[0].tolist() == [0, 0, 0, 0]
    assert w[1].tolist() == [0.5, 0.5] and w[4].tolist() == [0.5, 0.5] and w[5].tolist() == [1, 0]
    assert bool(w[3].isnan().all())
    one, idx = ts.expert_topk(x[:1].detach(), 4, False)
    assert one.tolist() == [[0, 0, 0, 0]] and idx.tolist() == [[-1] * 4]


def test_topk_empty_and_batched():
    w, i = ts.expert_topk(torch.empty(0, 8, device='cuda'), 2)
    assert w.shape == i.shape == (0, 2)
    x = torch.randn(3, 5, 16, device='cuda').transpose(0, 1)
    w, i = ts.expert_topk(x, 3)
    w2, i2 = ts.expert_topk(x.reshape(15, 16), 3)
    assert torch.equal(w.reshape(15, 3), w2) and torch.equal(i.reshape(15, 3), i2)


# ---- expert_sort ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('n,k,E', [(0, 2, 4), (1, 1, 1), (1, 8, 64), (5, 3, 2), (31, 1, 7), (33, 4, 128), (700, 6, 256),
                                   (1500, 3, 1000), (4097, 1, 4096), (9000, 2, 513), (40000, 3, 60), (140000, 8, 300)])
@pytest.mark.parametrize('load', ['even', 'one', 'dropped'])
def test_sort(n, k, E, load):
    gen = torch.Generator().manual_seed(n + E)
    index = torch.randint(0, E, (n, k), generator=gen)
    if load == 'one':
        index.fill_(E - 1)
    if load == 'dropped':
        index[torch.rand(n, k, generator=gen) < 0.4] = -1
        index[torch.rand(n, k, generator=gen) < 0.1] = E
        index[torch.rand(n, k, generator=gen) < 0.05] = -(1 << 40)
        index[torch.rand(n, k, generator=gen) < 0.05] = (1 << 32) + 1
    want = ref.sort(index, E)
    got = ts.expert_sort(index.cuda(), E)
    for g, w, name in zip(got, want, ('slot', 'order', 'indptr')):
        assert torch.equal(g.cpu(), w), name


def test_sort_strided_index():
    index = torch.randint(0, 9, (4, 50), device='cuda')
    for g, w in zip(ts.expert_sort(index.t(), 9), ref.sort(index.t().cpu().contiguous(), 9)):
        assert torch.equal(g.cpu(), w)


# ---- expert_dispatch / expert_combine ---------------------------------------------------------------------------

ROWS = [(1, 1, 1, 1), (1, 8, 4096, 64), (5, 2, 64, 3), (33, 3, 7, 8), (40, 4, 129, 5), (16, 8, 1030, 16), (9, 11, 72, 4),
        (64, 1, 2048, 8), (130, 6, 36, 20), (3, 40, 20, 50), (257, 2, 514, 2)]


def plan(gen, T, k, E, dropped=0.15):
    index = torch.randint(0, E, (T, k), generator=gen)
    index[torch.rand(T, k, generator=gen) < dropped] = -1
    if T > 2:
        index[1] = -1  # a token that is dropped altogether
    slot, _, indptr = ref.sort(index, E)
    return slot, indptr


@pytest.mark.parametrize('dtype', [F32, F16, BF16, F64])
@pytest.mark.parametrize('weighted', [False, True])
@pytest.mark.parametrize('T,k,K,E', ROWS)
def test_dispatch_and_combine(T, k, K, E, weighted, dtype):
    gen = torch.Generator().manual_seed(T * 100 + k + K)
    slot, indptr = plan(gen, T, k, E)
    few, many = rand(gen, T, K, dtype=dtype), rand(gen, T * k, K, dtype=dtype)
    many[indptr[-1]:] = math.nan  # rows of dropped entries are not read
    acc = F64 if dtype == F64 else F32
    weight = rand(gen, T, k, dtype=acc) if weighted else None
    u, w64 = ref.unit(dtype), None if weight is None else weight.double()
    a64 = None if weight is None else w64.abs()
    clean = many.double().nan_to_num(0)

    spread, fold = ref.spread(few.double(), slot, w64), ref.fold(clean, slot, w64)
    dots = ref.dots(few.double(), clean, slot)
    spread_tol = (spread.abs() * u + ref.last_rounding(spread, dtype)) if weighted else torch.zeros_like(spread)
    fold_tol = ref.fold(clean.abs(), slot, a64) * u * (k + 2) + ref.last_rounding(fold, dtype)
    dots_tol = ref.dots(few.double().abs(), clean.abs(), slot) * u * (K + 2) + 1e-300

    slot_d, indptr_d = slot.cuda(), indptr.cuda()
    for name, x, grad, call, want, want_grad, tol, grad_tol in (
            ('dispatch', few, many, ts.expert_dispatch, spread, fold, spread_tol, fold_tol),
            ('combine', many, few, ts.expert_combine, fold, spread, fold_tol, spread_tol)):
        xd = x.cuda().requires_grad_()
        wd = None if weight is None else weight.cuda().requires_grad_()
        out = call(xd, slot_d, indptr_d, wd)
        assert out.dtype == dtype
        ref.assert_within(out, want, tol, name)
        leaves = (xd,) if wd is None else (xd, wd)
        grads = torch.autograd.grad(out, leaves, grad.cuda())
        assert [g.dtype for g in grads] == [t.dtype for t in leaves]
        ref.assert_within(grads[0], want_grad, grad_tol, name + ' grad')
        if weighted:
            ref.assert_within(grads[1], dots, dots_tol, name + ' grad of the weights')


@pytest.mark.parametrize('dtype', [F32, F16, BF16, F64])
@pytest.mark.parametrize('weighted', [False, True])
@pytest.mark.parametrize('T,k,K', [(2500, 1, 256), (2400, 2, 1032), (2371, 8, 520), (2400, 3, 1027), (3001, 9, 264), (2368, 33, 256)])
def test_many_tokens(T, k, K, weighted, dtype):
    """Tokens enough for the kernels that keep a pipeline per warp: rows of one and more pieces, ragged last pieces."""
    gen = torch.Generator().manual_seed(T + k + K)
    slot, indptr = plan(gen, T, k, 13)
    few, many = rand(gen, T, K, dtype=dtype), rand(gen, T * k, K, dtype=dtype)
    many[indptr[-1]:] = math.nan
    acc = F64 if dtype == F64 else F32
    weight = rand(gen, T, k, dtype=acc) if weighted else None
    u, w64 = ref.unit(dtype), None if weight is None else weight.double()
    # the 64-bit results by indexing, all tokens at once
    at, named = slot.clamp_min(0), (slot >= 0).unsqueeze(-1)
    clean = many.double().nan_to_num(0)
    picked = clean[at] * named
    factor = named.double() * (1 if w64 is None else w64.unsqueeze(-1))
    fold, mass = (picked * factor).sum(1), (picked * factor).abs().sum(1)
    spread = torch.zeros(T * k, K, dtype=torch.float64)
    spread[slot[slot >= 0]] = (few.double().unsqueeze(1) * factor)[slot >= 0]
    dots, dmass = (picked * few.double().unsqueeze(1)).sum(-1), (picked * few.double().unsqueeze(1)).abs().sum(-1)
    spread_tol = (spread.abs() * u + ref.last_rounding(spread, dtype)) if weighted else torch.zeros_like(spread)
    fold_tol = mass * u * (k + 2) + ref.last_rounding(fold, dtype)
    for name, x, grad, call, want, want_grad, tol, grad_tol in (
            ('dispatch', few, many, ts.expert_dispatch, spread, fold, spread_tol, fold_tol),
            ('combine', many, few, ts.expert_combine, fold, spread, fold_tol, spread_tol)):
        xd = x.cuda().requires_grad_()
        wd = None if weight is None else weight.cuda().requires_grad_()
        out = call(xd, slot.cuda(), indptr.cuda(), wd)
        ref.assert_within(out, want, tol, name)
        grads = torch.autograd.grad(out, (xd,) if wd is None else (xd, wd), grad.cuda())
        ref.assert_within(grads[0], want_grad, grad_tol, name + ' grad')
        if weighted:
            ref.assert_within(grads[1], dots, dmass * u * (K + 2) + 1e-300, name + ' grad of the weights')


def test_rows_of_several_dimensions_strides_and_alignment():
    gen = torch.Generator().manual_seed(3)
    slot, indptr = plan(gen, 12, 2, 4)
    x = rand(gen, 12, 24)
    want = ref.spread(x.double(), slot, None)
    s, p = slot.cuda(), indptr.cuda()
    flat = ts.expert_dispatch(x.cuda(), s, p)
    assert torch.equal(flat.cpu().double(), want)
    assert torch.equal(ts.expert_dispatch(x.cuda().reshape(12, 4, 6), s, p).reshape(24, 24), flat)
    assert torch.equal(ts.expert_dispatch(x.cuda().reshape(3, 4, 24), s.reshape(3, 4, 2), p), flat)
    assert torch.equal(ts.expert_dispatch(x.t().contiguous().cuda().t(), s, p), flat)
    for off in (1, 2, 3):  # data that begins off a 16-byte boundary
        buf = torch.zeros(12 * 24 + 8, device='cuda')
        y = buf[off:off + 288].view(12, 24).copy_(x)
        assert torch.equal(ts.expert_dispatch(y, s, p), flat)
        assert torch.equal(ts.expert_combine(buf[off:off + 240].view(24, 10), s, p), ts.expert_combine(buf[off:off + 240].view(24, 10).clone(), s, p))
    # gradient that arrives broadcast
    xd = x.cuda().requires_grad_()
    ts.expert_dispatch(xd, s, p).sum().backward()
    assert torch.equal(xd.grad.cpu(), (slot >= 0).sum(1, keepdim=True).float().expand(12, 24))


def test_empty_rows():
    z = torch.zeros
    p = z(4, dtype=torch.long, device='cuda')
    none, slot = z(0, 2, dtype=torch.long, device='cuda'), z(3, 0, dtype=torch.long, device='cuda')
    assert ts.expert_dispatch(z(0, 8, device='cuda'), none, p).shape == (0, 8)
    assert ts.expert_combine(z(0, 8, device='cuda'), none, p).shape == (0, 8)
    assert torch.equal(ts.expert_combine(z(0, 8, device='cuda'), slot, p), z(3, 8, device='cuda'))
    assert ts.expert_dispatch(z(3, 8, device='cuda'), slot, p).shape == (0, 8)
    two = z(3, 2, dtype=torch.long, device='cuda') - 1
    w = torch.ones(3, 2, device='cuda', requires_grad=True)
    assert ts.expert_dispatch(z(3, 0, device='cuda'), two, p).shape == (6, 0)
    out = ts.expert_combine(z(6, 0, device='cuda', requires_grad=True), two, p, w)
    assert out.shape == (3, 0) and torch.equal(torch.autograd.grad(out.sum(), w)[0], z(3, 2, device='cuda'))


# ---- scan ---------------------------------------------------------------------------------------------------------

def lengths(kind, gen):
    if kind == 'one':
        return [1]
    if kind == 'ones':
        return [1] * 70
    if kind == 'empty':
        return [0, 0, 0]
    if kind == 'ragged':
        return [0, 3, 1, 0, 40, 2, 130, 0, 0, 7, 64, 65, 1, 1, 33, 0]
    if kind == 'long':
        return [2900]
    if kind == 'two':
        return [1300, 1251]
    raise ValueError(kind)


@pytest.mark.parametrize('dtype,gdtype', [(F32, F32), (F64, F64), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize('kind,heads,width', [('one', 1, 1), ('ones', 40, 1), ('empty', 8, 1), ('ragged', 5, 1), ('ragged', 64, 1),
                                              ('ragged', 130, 1), ('ragged', 3, 33), ('ragged', 2, 64), ('ragged', 7, 8),
                                              ('ragged', 1, 300), ('long', 24, 1), ('long', 3, 16), ('two', 2, 24), ('two', 9, 1)])
@pytest.mark.parametrize('states', [False, True])
def test_scan(kind, heads, width, states, dtype, gdtype):
    gen = torch.Generator().manual_seed(heads * 100 + width)
    lens = lengths(kind, gen)
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    front, pad, K = (3 if kind == 'ragged' else 0), 5, heads * width
    ends = [e + front for e in ends]
    E, N = ends[-1] + pad, len(lens)
    acc = F64 if dtype == F64 else F32
    src, grad = rand(gen, E, heads, width, dtype=dtype), rand(gen, E, heads, width, dtype=dtype)
    gate = torch.sigmoid(rand(gen, E, heads, 1) * 2 + 3).to(gdtype)
    gate[torch.rand(E, heads, 1, generator=gen) < 0.02] = 0.0
    gate[torch.rand(E, heads, 1, generator=gen) < 0.02] = -1.0
    outside = torch.ones(E, dtype=torch.bool)
    outside[ends[0]:ends[-1]] = False
    for t in (src, gate, grad):  # what is behind and before the sequences takes no part
        t[outside] = math.nan
    state, grad_last = rand(gen, N, heads, width, dtype=acc), rand(gen, N, heads, width, dtype=acc)

    s64, g64 = src.double().reshape(E, K), gate.double().expand(E, heads, width).reshape(E, K)
    st64, gl64 = (state.double().reshape(N, K), grad_last.double().reshape(N, K)) if states else (None, None)
    h, before, last, mass, way = ref.scan(s64, g64, ends, st64)
    dh, dg, dstate, dmass, dway, smass, sway = ref.scan_backward(grad.double().reshape(E, K), gl64, g64, before, ends)
    u = ref.unit(dtype)
    bound = u * (4 * way + 32 * mass)
    dbound = u * (4 * dway + 32 * dmass)

    xs, xg = src.cuda().requires_grad_(), gate.cuda().requires_grad_()
    xst = state.cuda().requires_grad_() if states else None
    indptr = torch.tensor(ends, device='cuda')
    out, got_last = ts.scan_csr_state(xs, xg, indptr, xst)
    assert out.dtype == dtype and got_last.dtype == acc
    ref.assert_within(out.reshape(E, K), h, bound + ref.last_rounding(h, dtype), 'out')
    lmass, lway = torch.zeros_like(last), torch.zeros_like(last)
    for n in range(N):
        if lens[n]:
            lmass[n], lway[n] = mass[ends[n + 1] - 1], way[ends[n + 1] - 1]
    ref.assert_within(got_last.reshape(N, K), last, u * (4 * lway + 32 * lmass), 'last')
    assert torch.equal(ts.scan_csr(xs, xg, indptr, xst), out)

    if states:
        grads = torch.autograd.grad((out, got_last), (xs, xg, xst), (grad.cuda(), grad_last.cuda()))
        ref.assert_within(grads[2].reshape(N, K), dstate, u * (4 * sway + 32 * smass), 'grad_state')
    else:
        grads = torch.autograd.grad(out, (xs, xg), grad.cuda())
    assert grads[0].dtype == dtype and grads[1].dtype == gdtype
    ref.assert_within(grads[0].reshape(E, K), dh, dbound + ref.last_rounding(dh, dtype), 'grad_src')
    # grad_gate = sum dh * before; `before` is the rounded output (unrounded where the gate is wider than the data), its
    # first row of a segment the state itself
    rounded = ref.last_rounding(before, dtype) if gdtype == dtype else 0
    first = torch.zeros(E, 1)
    first[[e for e, n in zip(ends, lens) if n]] = 1
    err = dh.abs() * (torch.roll(bound, 1, 0) + rounded) * (1 - first) + dbound * before.abs() + u * dg.abs()
    dg3, err3 = dg.reshape(E, heads, width), err.reshape(E, heads, width)
    want = dg3.sum(-1, keepdim=True)
    err3 = err3.sum(-1, keepdim=True) + u * width * dg3.abs().sum(-1, keepdim=True) + ref.last_rounding(want, gdtype)
    ref.assert_within(grads[1], want, err3, 'grad_gate')


def test_scan_forms_of_the_gate_agree():
    """A gate that is shared, expanded, flattened or constant: each form within the roundings of the formula (they are cut
    into tiles of different lengths, so the bits of two forms need not be the same)."""
    gen = torch.Generator().manual_seed(5)
    E, H, P = 700, 6, 16
    ends = [0, 100, 100, 650, 700]
    indptr = torch.tensor(ends, device='cuda')
    src = rand(gen, E, H, P).cuda()
    gate = torch.rand(E, H, 1, generator=gen).cuda()

    def bounds(g):
        h, _, _, mass, way = ref.scan(src.cpu().double().reshape(E, H * P), g.cpu().double().expand(E, H, P).reshape(E, H * P), ends, None)
        return h, ref.unit(F32) * (4 * way + 32 * mass) + ref.last_rounding(h, F32)

    want, tol = bounds(gate)
    ref.assert_within(ts.scan_csr(src, gate, indptr).reshape(E, H * P), want, tol, 'shared')
    ref.assert_within(ts.scan_csr(src, gate.expand(E, H, P), indptr).reshape(E, H * P), want, tol, 'expanded')
    flat = gate.expand(E, H, P).reshape(E, H * P)
    ref.assert_within(ts.scan_csr(src.reshape(E, H * P), flat, indptr), want, tol, 'flat')

    one = torch.rand(E, 1, 1, generator=gen).cuda().requires_grad_()
    full = one.detach().expand(E, H, P).contiguous().requires_grad_()
    want, tol = bounds(one.detach())
    a, b = ts.scan_csr(src, one, indptr), ts.scan_csr(src, full, indptr)
    ref.assert_within(a.reshape(E, H * P), want, tol, 'one gate')
    ref.assert_within(b.reshape(E, H * P), want, tol, 'its copies')
    g = rand(gen, E, H, P)
    before = torch.roll(want, 1, 0)
    before[[0, 100, 650]] = 0
    gates = full.detach().cpu().double().reshape(E, H * P)
    dh, dg, _, dmass, dway, _, _ = ref.scan_backward(g.double().reshape(E, H * P), None, gates, before, ends)
    # each product: dh and h within their bounds; then the sum of H * P of them
    dtol = dh.abs() * torch.roll(tol, 1, 0) + ref.unit(F32) * (4 * dway + 32 * dmass) * before.abs() + 2 * ref.unit(F32) * dg.abs()
    total = dg.sum(1, keepdim=True)
    ttol = dtol.sum(1, keepdim=True) + ref.unit(F32) * (H * P + 4) * dg.abs().sum(1, keepdim=True)
    ga, gb = torch.autograd.grad(a, one, g.cuda())[0], torch.autograd.grad(b, full, g.cuda())[0]
    ref.assert_within(ga.reshape(E, 1), total, ttol, 'gradient of one gate')
    ref.assert_within(gb.reshape(E, H * P), dg, dtol, 'gradient of its copies')

    decay = torch.rand(P, generator=gen).cuda().reshape(1, 1, P).requires_grad_()  # a constant decay: expanded, gradient summed
    out = ts.scan_csr(src, decay, indptr)
    assert torch.equal(out, ts.scan_csr(src, decay.expand(E, H, P).contiguous(), indptr))
    assert torch.autograd.grad(out.sum(), decay)[0].shape == decay.shape


def test_scan_batches_of_sequences():
    gen = torch.Generator().manual_seed(6)
    src, gate = rand(gen, 3, 90, 10).cuda(), torch.rand(3, 90, 10, generator=gen).cuda()
    shared = torch.tensor([[0, 40, 90]], device='cuda')
    own = torch.tensor([[0, 40, 90], [5, 5, 80], [0, 90, 90]], device='cuda')
    state = rand(gen, 3, 2, 10).cuda()
    for p in (shared, own):
        out, last = ts.scan_csr_state(src, gate, p, state)
        for b in range(3):
            row = p[b if p.size(0) > 1 else 0]
            o, l = ts.scan_csr_state(src[b], gate[b], row, state[b])
            assert torch.equal(out[b], o) and torch.equal(last[b], l)


def test_scan_sequences_do_not_leak():
    """Infinities and NaN of one sequence stay in it, and in their channel."""
    src, gate = torch.ones(300, 40, device='cuda'), torch.full((300, 40), 0.5, device='cuda')
    indptr = torch.tensor([0, 100, 200, 300], device='cuda')
    clean = ts.scan_csr(src, gate, indptr)
    src[120, 3], src[130, 5], gate[140, 7] = math.nan, math.inf, math.nan
    xs, xg = src.requires_grad_(), gate.requires_grad_()
    out = ts.scan_csr(xs, xg, indptr)
    same = torch.ones(300, 40, dtype=torch.bool, device='cuda')
    same[120:200, 3] = same[130:200, 5] = same[140:200, 7] = False
    assert torch.equal(out[same], clean[same]) and not bool(out[~same].isfinite().any())
    gs, gg = torch.autograd.grad(out, (xs, xg), torch.ones_like(out))
    touched = torch.zeros_like(same)
    touched[100:200, [3, 5, 7]] = True
    assert bool(gs[~touched].isfinite().all()) and bool(gg[~touched].isfinite().all())


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('offset', [1, 2, 3, 4])
@pytest.mark.parametrize('K', [24, 7])
def test_scan_data_off_a_boundary(dtype, offset, K):
    """Inputs that begin anywhere in their storage, the first and the last value of it included; a gate wider than the data."""
    gen = torch.Generator().manual_seed(offset)
    E, ends = 300, [0, 120, 300]
    src, grad = rand(gen, E, K, dtype=dtype), rand(gen, E, K, dtype=dtype)
    gate = torch.sigmoid(rand(gen, E, K) + 2)

    def off(t):
        buf = torch.empty(t.numel() + offset, dtype=t.dtype, device='cuda')
        return buf[offset:].view(t.shape).copy_(t)

    for g in ([gate] if dtype == F32 else [gate, gate.to(dtype)]):
        h, before, _, mass, way = ref.scan(src.double(), g.double(), ends, None)
        dh, dg, _, dmass, dway, _, _ = ref.scan_backward(grad.double(), None, g.double(), before, ends)
        u = ref.unit(dtype)
        bound, dbound = u * (4 * way + 32 * mass), u * (4 * dway + 32 * dmass)
        xs, xg = off(src).requires_grad_(), off(g).requires_grad_()
        out = ts.scan_csr(xs, xg, torch.tensor(ends, device='cuda'))
        gs, gg = torch.autograd.grad(out, (xs, xg), off(grad))
        ref.assert_within(out, h, bound + ref.last_rounding(h, dtype), 'out')
        ref.assert_within(gs, dh, dbound + ref.last_rounding(dh, dtype), 'grad_src')
        rounded = ref.last_rounding(before, dtype) if g.dtype == dtype else 0
        err = dh.abs() * (torch.roll(bound, 1, 0) + rounded) + dbound * before.abs() + u * dg.abs()
        ref.assert_within(gg, dg, err + ref.last_rounding(dg, g.dtype), 'grad_gate')


def test_scan_many_empty_segments_and_a_long_stream():
    """Runs of empty segments around and inside tiles, and rows by the hundred thousand (several rounds of a cluster)."""
    gen = torch.Generator().manual_seed(12)
    lens = torch.randint(0, 3, (4000,), generator=gen) * (torch.rand(4000, generator=gen) < 0.05)
    lens[1000], lens[3000] = 70000, 40000
    ends = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    E = int(ends[-1])
    src, gate = torch.ones(E, 8, device='cuda'), torch.full((E, 8), 0.5, device='cuda')
    out, last = ts.scan_csr_state(src, gate, ends.cuda(), torch.full((4000, 8), 2.0, device='cuda'))
    # a fixed point: 0.5 * 2 + 1 = 2 exactly, whatever the segments are
    assert bool((out == 2).all()) and bool((last == 2).all())
    out = ts.scan_csr(src, torch.ones_like(gate), ends.cuda())
    # counts of the rows of each segment: whole numbers below 2^24, exact in any order
    row = torch.arange(E) - torch.repeat_interleave(ends[:-1], lens) + 1
    assert torch.equal(out.cpu(), row.float().unsqueeze(1).expand(E, 8))


def test_scan_runs_of_empty_segments():
    """Hundreds of thousands of empty segments at one row, at the first row and behind the last, forward and backward."""
    ends = torch.cat([torch.zeros(100001, dtype=torch.long), torch.tensor([37]), torch.full((300000,), 50), torch.tensor([51, 90, 90]),
                      torch.full((1000,), 130)])
    N, src, gate = ends.numel() - 1, torch.ones(140, 4, device='cuda').requires_grad_(), torch.ones(140, 4, device='cuda')
    out, last = ts.scan_csr_state(src, gate, ends.cuda())
    lens = ends[1:] - ends[:-1]
    row = torch.arange(130) - torch.repeat_interleave(ends[:-1], lens) + 1
    assert torch.equal(out[:130].cpu(), row.float().unsqueeze(1).expand(130, 4)) and not bool(out[130:].any())
    assert torch.equal(last[:, 0].cpu(), lens.float()) and last.shape == (N, 4)
    (g,) = torch.autograd.grad(out, src, torch.ones_like(out))
    behind = torch.repeat_interleave(ends[1:], lens) - torch.arange(130)  # rows from here to the segment's end
    assert torch.equal(g[:130].cpu(), behind.float().unsqueeze(1).expand(130, 4)) and not bool(g[130:].any())


def test_scan_empty_shapes():
    z = torch.zeros
    p = torch.tensor([0, 0, 0], device='cuda')
    state = torch.randn(2, 5, device='cuda', requires_grad=True)
    out, last = ts.scan_csr_state(z(0, 5, device='cuda'), z(0, 5, device='cuda'), p, state)
    assert out.shape == (0, 5) and torch.equal(last, state)
    g = torch.randn(2, 5, device='cuda')
    assert torch.equal(torch.autograd.grad(last, state, g)[0], g)
    assert ts.scan_csr(z(4, 0, device='cuda'), z(4, 0, device='cuda'), p).shape == (4, 0)
    out = ts.scan_csr(torch.ones(4, 3, device='cuda'), torch.ones(4, 3, device='cuda'), z(1, dtype=torch.long, device='cuda'))
    assert torch.equal(out, z(4, 3, device='cuda'))
    out, last = ts.scan_csr_state(torch.ones(4, 3, device='cuda'), torch.ones(4, 3, device='cuda'), p)
    assert torch.equal(out, z(4, 3, device='cuda')) and torch.equal(last, z(2, 3, device='cuda'))


@pytest.mark.parametrize('dtype,gdtype', [(F32, F32), (F64, F64), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize('n,heads,width', [(1, 1, 1), (3, 7, 1), (64, 128, 1), (5, 3, 33), (9, 4, 16), (2, 1, 4096)])
def test_step(n, heads, width, dtype, gdtype):
    gen = torch.Generator().manual_seed(n + heads)
    acc, u = F64 if dtype == F64 else F32, ref.unit(dtype)
    src, gate = rand(gen, n, heads, width, dtype=dtype), torch.rand(n, heads, 1, generator=gen).to(gdtype)
    state = rand(gen, n, heads, width, dtype=acc)
    pool = torch.zeros(n, 2, heads, width, dtype=acc, device='cuda')
    for s in (state.cuda(), pool[:, 1].copy_(state)):
        out = ts.scan_step(src.cuda(), gate.cuda(), s)
        want = gate.double() * state.double() + src.double()
        tol = 2 * u * ((gate * state).double().abs() + src.double().abs())
        ref.assert_within(s, want, tol, 'state')
        ref.assert_within(out, want, tol + ref.last_rounding(want, dtype), 'out')
    assert not bool(pool[:, 0].any())
    full, last = ts.scan_csr_state(src.cuda(), gate.cuda(), torch.arange(n + 1, device='cuda'), state.cuda())
    assert torch.equal(last, s) and torch.equal(full, out)


def test_step_compiles():
    state = torch.randn(4, 6, device='cuda')
    x, g = torch.randn(4, 6, device='cuda'), torch.rand(4, 6, device='cuda')
    want_state = g * state + x
    with torch.no_grad():
        out = torch.compile(lambda a, b, s: ts.scan_step(a, b, s) * 2, fullgraph=True)(x, g, state)
    assert torch.allclose(state, want_state, rtol=1e-6, atol=1e-6) and torch.allclose(out, 2 * want_state, rtol=1e-6, atol=1e-6)


def test_step_marks_the_state_as_changed():
    state, x = torch.ones(2, 3, device='cuda'), torch.ones(2, 3, device='cuda', requires_grad=True)
    y = (x * state).sum()
    with torch.no_grad():
        ts.scan_step(x, x, state)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


# ---- gradients by differences, second derivatives -----------------------------------------------------------------

def test_gradients_against_differences():
    gen = torch.Generator().manual_seed(8)
    d = lambda *s: rand(gen, *s, dtype=F64).cuda().requires_grad_()  # noqa: E731
    slot, indptr = (t.cuda() for t in plan(gen, 6, 3, 4))
    assert torch.autograd.gradcheck(lambda x, w: ts.expert_dispatch(x, slot, indptr, w), (d(6, 5), d(6, 3)))
    assert torch.autograd.gradcheck(lambda x, w: ts.expert_combine(x, slot, indptr, w), (d(18, 5), d(6, 3)))
    p = torch.tensor([1, 4, 4, 11], device='cuda')
    assert torch.autograd.gradcheck(lambda x, g, s: ts.scan_csr_state(x, g, p, s), (d(13, 2, 3), d(13, 2, 1), d(3, 2, 3)))
    assert torch.autograd.gradcheck(lambda x, g: ts.scan_csr(x, g, p), (d(13, 5), d(13, 5)))


def test_no_second_derivative():
    x = torch.randn(6, 4, device='cuda', requires_grad=True)
    slot, indptr = (t.cuda() for t in plan(torch.Generator().manual_seed(1), 6, 2, 3))
    w = torch.rand(6, 2, device='cuda', requires_grad=True)
    p = torch.tensor([0, 6], device='cuda')
    for out in (ts.expert_topk(x, 2)[0], ts.expert_dispatch(x, slot, indptr, w), ts.scan_csr(x, x, p)):
        (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match='no second derivative'):
            g.sum().backward()


def test_gradients_that_are_not_wanted():
    src, gate = torch.randn(20, 6, device='cuda'), torch.rand(20, 6, device='cuda')
    p = torch.tensor([0, 7, 20], device='cuda')
    state = torch.randn(2, 6, device='cuda')
    full = [t.clone().requires_grad_() for t in (src, gate, state)]
    ref_grads = torch.autograd.grad(ts.scan_csr(full[0], full[1], p, full[2]).square().sum(), full)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((src, gate, state))]
        (g,) = torch.autograd.grad(ts.scan_csr(args[0], args[1], p, args[2]).square().sum(), (args[i],))
        assert torch.equal(g, ref_grads[i])
    last = ts.scan_csr_state(*full[:2], p, full[2])[1]
    grads = torch.autograd.grad(last.sum(), full)  # nothing flows into the rows
    h = torch.autograd.grad(ts.scan_csr(*full[:2], p, full[2])[[6, 19]].sum(), full)
    for a, b in zip(grads, h):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    slot, indptr = (t.cuda() for t in plan(torch.Generator().manual_seed(1), 6, 2, 3))
    x, w = torch.randn(6, 4, device='cuda'), torch.rand(6, 2, device='cuda', requires_grad=True)
    assert torch.autograd.grad(ts.expert_dispatch(x, slot, indptr, w).sum(), w)[0].shape == (6, 2)
    assert torch.autograd.grad(ts.expert_combine(x.repeat(2, 1), slot, indptr, w).sum(), w)[0].shape == (6, 2)


# ---- together -----------------------------------------------------------------------------------------------------

def block(x, router, gate, indptr, E, k):
    """A recurrent layer over the sequences, then experts that are recurrences of their own over the tokens sent to them."""
    h = ts.scan_csr(x, gate, indptr)
    weight, index = ts.expert_topk(h.float() @ router, k)
    slot, order, experts = ts.expert_sort(index, E)
    rows = ts.expert_dispatch(h, slot, experts)
    rows = ts.scan_csr(rows, torch.sigmoid(rows.float() + 1).to(rows.dtype), experts)
    load = ts.segment_csr(torch.ones_like(rows[:, :1]), experts)
    return ts.expert_combine(rows, slot, experts, weight) + x, load, index


def block_plain(x, router, gate, ends, E, k, index):
    """The same in float64 on the CPU for the given choice, from elementary differentiable steps."""
    def walk(v, g, bounds):
        out = [torch.zeros_like(v[0])] * v.size(0)
        for lo, hi in zip(bounds[:-1], bounds[1:]):
            c = torch.zeros_like(v[0])
            for e in range(lo, hi):
                c = g[e] * c + v[e]
                out[e] = c
        return torch.stack(out)
    h = walk(x, gate, ends)
    logits = h @ router
    w = torch.softmax(logits.gather(1, index), 1)
    slot, order, indptr = ref.sort(index, E)
    rows = h[order // k]
    rows = walk(rows, torch.sigmoid(rows + 1), indptr.tolist())
    return (rows[slot.reshape(-1)].reshape(*index.shape, -1) * w.unsqueeze(-1)).sum(1) + x


def block_inputs(dtype):
    gen = torch.Generator().manual_seed(11)
    T, D, E, k = 60, 12, 5, 2
    x = rand(gen, T, D).mul(0.5)
    return x, rand(gen, D, E), torch.sigmoid(rand(gen, T, D)), [0, 20, 21, 60], E, k


def test_a_block_of_them():
    x, router, gate, ends, E, k = block_inputs(F32)
    leaves = [t.cuda().requires_grad_() for t in (x, router, gate)]
    out, load, index = block(*leaves, torch.tensor(ends, device='cuda'), E, k)
    assert int(load.sum()) == 60 * k
    plain = [t.double().requires_grad_() for t in (x, router, gate)]
    want = block_plain(*plain, ends, E, k, index.cpu())
    g = torch.randn(out.shape, generator=torch.Generator().manual_seed(1))
    got, exp = torch.autograd.grad(out, leaves, g.cuda()), torch.autograd.grad(want, plain, g.double())
    # a few hundred chained 32-bit roundings of values of order one
    for a, b, name in ((out, want, 'out'), (got[0], exp[0], 'x'), (got[1], exp[1], 'router'), (got[2], exp[2], 'gate')):
        ref.assert_within(a, b.detach(), 1000 * ref.unit(F32) * b.detach().abs().max().expand(b.shape), name)


def test_a_block_captured_and_replayed():
    x, router, gate, ends, E, k = block_inputs(F32)
    p = torch.tensor(ends, device='cuda')
    leaves = [t.cuda().requires_grad_() for t in (x, router, gate)]
    g = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).cuda()

    def both():
        out = block(*leaves, p, E, k)[0]
        # no eager graph of the leaves may live during a capture: their accumulation nodes would be on another stream
        return (out.detach(),) + torch.autograd.grad(out, leaves, g)

    eager = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs that are replayed in turn keep their workspaces apart
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both())
    for new in (leaves[0].detach().flip(0).contiguous(), leaves[0].detach().clone()):
        with torch.no_grad():
            leaves[0].copy_(new)
        want = both()
        for graph in graphs:
            graph.replay()
        for got in outs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(want, eager))


def test_streams_and_repeatability():
    """The same bits from every stream and every run."""
    gen = torch.Generator().manual_seed(4)
    src, gate = rand(gen, 5000, 64, dtype=BF16).cuda().requires_grad_(), torch.rand(5000, 64, generator=gen).cuda().requires_grad_()
    p = torch.tensor([0, 1700, 1701, 5000], device='cuda')
    index = torch.randint(0, 16, (5000, 4), generator=gen).cuda()

    def once():
        out = ts.scan_csr(src, gate, p)
        slot, order, ptr = ts.expert_sort(index, 16)
        rows = ts.expert_dispatch(out, slot, ptr)
        return (slot, rows) + torch.autograd.grad(rows, (src, gate), torch.ones_like(rows))

    want = once()
    torch.cuda.synchronize()
    for stream in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(stream):
            got = once()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_compile_fullgraph():
    gen = torch.Generator().manual_seed(9)
    x, router, gate, ends, E, k = block_inputs(F32)
    p = torch.tensor(ends, device='cuda')
    leaves = [t.cuda().requires_grad_() for t in (x, router, gate)]
    f = lambda a, b, c: block(a, b, c, p, E, k)[0]  # noqa: E731
    out = f(*leaves)
    got = torch.compile(f, fullgraph=True)(*leaves)
    g = rand(gen, *out.shape).cuda()
    for a, b in zip((got,) + torch.autograd.grad(got, leaves, g), (out,) + torch.autograd.grad(out, leaves, g)):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
