"""Plain 64-bit implementations of the packed-batch operators, and the error bounds their tests use.

Every bound counts roundings: u = 2^-24 (2^-53 for float64) for one operation in the accumulation type and eps / 2 of
the output's type for its last rounding, each times the sum of the magnitudes behind the value.
"""
import torch


def unit(dtype):
    """Half a step of the accumulation type."""
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def last_rounding(x, dtype):
    info = torch.finfo(dtype)
    return x.abs() * (info.eps / 2) + info.tiny * info.eps


def assert_within(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f'{what}: shape {tuple(got.shape)} instead of {tuple(want.shape)}'
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (f'{what}: {int(bad.sum())} of {bad.numel()} outside; worst error '
                                 f'{float((got - want).abs().max())}, there allowed {float(bound.flatten()[(got - want).abs().argmax()])}')


# ---- the recurrence ---------------------------------------------------------------------------------------------

def scan(src, gate, indptr, state):
    """src, gate [E, K] float64, indptr a list, state [N, K] or None -> (h, before, last, mass, way).

    mass: the same recurrence over magnitudes.  way: each magnitude times the steps it has come, so that a term that
    took d steps to its row (at most 4 roundings a step: gate product, carry product, two sums) is bounded by
    u (4 d + 32)."""
    N = len(indptr) - 1
    zero = torch.zeros_like(src)
    h, before, mass, way = zero.clone(), zero.clone(), zero.clone(), zero.clone()
    last = torch.zeros(N, src.size(1), dtype=torch.float64) if state is None else state.clone()
    for n in range(N):
        c = last[n].clone()
        m, w = c.abs(), torch.zeros_like(c)
        for e in range(indptr[n], indptr[n + 1]):
            g = gate[e].abs()
            before[e] = c
            c = gate[e] * c + src[e]
            w = g * (w + m)
            m = g * m + src[e].abs()
            h[e], mass[e], way[e] = c, m, w
        last[n] = c
    return h, before, last, mass, way


def scan_backward(grad, grad_last, gate, before, indptr):
    """-> (dh, dgate, dstate, mass of dh, way of dh)"""
    N = len(indptr) - 1
    zero = torch.zeros_like(grad)
    dh, mass, way = zero.clone(), zero.clone(), zero.clone()
    dstate = torch.zeros(N, grad.size(1), dtype=torch.float64) if grad_last is None else grad_last.clone()
    smass, sway = dstate.abs(), torch.zeros_like(dstate)
    for n in range(N):
        c, m, w = dstate[n].clone(), smass[n].clone(), sway[n].clone()
        for e in range(indptr[n + 1] - 1, indptr[n] - 1, -1):
            d = c + grad[e]
            m = m + grad[e].abs()
            dh[e], mass[e], way[e] = d, m, w
            g = gate[e].abs()
            w = g * (w + m)
            m = g * m
            c = gate[e] * d
        dstate[n], smass[n], sway[n] = c, m, w
    return dh, dh * before, dstate, mass, way, smass, sway


# ---- experts ------------------------------------------------------------------------------------------------------

def sort(index, experts):
    flat = index.reshape(-1).tolist()
    groups = [[] for _ in range(experts + 1)]
    for i, e in enumerate(flat):
        groups[e if 0 <= e < experts else experts].append(i)
    order = [i for g in groups for i in g]
    indptr = [0]
    for g in groups[:-1]:
        indptr.append(indptr[-1] + len(g))
    slot = [-1] * len(flat)
    for place, i in enumerate(order[:indptr[-1]]):
        slot[i] = place
    as_long = lambda v: torch.tensor(v, dtype=torch.long)  # noqa: E731
    return as_long(slot).reshape(index.shape), as_long(order), as_long(indptr)


def spread(few, slot, weight):
    """few [T, K], slot [T, k] -> [T * k, K]"""
    T, k = slot.shape
    many = torch.zeros(T * k, few.size(1), dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if slot[t, j] >= 0:
                many[slot[t, j]] = few[t] * (1 if weight is None else weight[t, j])
    return many


def fold(many, slot, weight):
    T, k = slot.shape
    few = torch.zeros(T, many.size(1), dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if slot[t, j] >= 0:
                few[t] += many[slot[t, j]] * (1 if weight is None else weight[t, j])
    return few


def dots(few, many, slot):
    T, k = slot.shape
    out = torch.zeros(T, k, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            if slot[t, j] >= 0:
                out[t, j] = (few[t] * many[slot[t, j]]).sum()
    return out


def topk(logits, k, normalize):
    """logits [T, E] float64 -> (weight, index); differentiable."""
    order = torch.sort(logits.detach(), dim=1, descending=True, stable=True)[1][:, :k]
    never = logits.detach().gather(1, order) == float('-inf')
    p = torch.softmax(logits, 1)
    w = p.gather(1, order).masked_fill(never, 0.0)
    if normalize:
        w = w / w.sum(1, keepdim=True)
    return w, order.masked_fill(never, -1)
