"""Cases of the packed-batch operators: the router's choice of experts, the sort of tokens by expert, the way of the
rows to the experts and back, and the gated linear recurrence over the sequences of a packed batch.

`run` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) or, where
`own` is true, through the package's own operators.  Both return the same outputs in the same layout.

A packed batch holds sequences one behind the other along the first dimension; `indptr` says where each begins.  A case
with `pad` has that many rows behind its last sequence, as a buffer of fixed size has.  `index[t, j]` names the j-th
expert of token t; negative numbers stand for padding tokens and choices that were dropped.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}
_BYTES = {'fp32': 4, 'fp16': 2, 'bf16': 2}

# No case may take more than the largest listed one: elements of the rows behind the experts, of a packed batch of the
# recurrence, of a router's logits, and entries of a sort.
_MOST_ROWS = 32768 * 8 * 2048
_MOST_SCAN = 65536 * 2048
_MOST_LOGITS = 65536 * 256
_MOST_ENTRIES = 262144 * 8


def listed():
    return [
        # the router of one decoding step: sixteen running requests
        dict(name='topk decode', op='topk', tokens=16, experts=64, k=6, dtype='bf16', normalize=True, masked=0, train=False),
        # the router of a training step over a packed batch, many fine-grained experts
        dict(name='topk train', op='topk', tokens=65536, experts=256, k=8, dtype='fp32', normalize=True, masked=3, train=True),
        # the sort of one decoding step
        dict(name='sort decode', op='sort', tokens=32, experts=128, k=8, dropped=0.0),
        # the sort of a large training batch: skewed load, some padding tokens
        dict(name='sort train', op='sort', tokens=262144, experts=256, k=8, dropped=0.02),
        # rows to the experts in one decoding step
        dict(name='dispatch decode', op='dispatch', tokens=8, experts=64, k=6, features=4096, dtype='bf16', weighted=False, dropped=0.0, train=False),
        # rows to the experts, forward and backward, of a training step
        dict(name='dispatch train', op='dispatch', tokens=32768, experts=128, k=8, features=2048, dtype='bf16', weighted=False, dropped=0.02, train=True),
        # rows back from few large experts, with the router's weights and their gradient
        dict(name='combine train', op='combine', tokens=32768, experts=16, k=2, features=4096, dtype='bf16', weighted=True, dropped=0.02, train=True),
        # the same in 32 bits with an odd row length and an odd number of tokens
        dict(name='combine odd', op='combine', tokens=5003, experts=23, k=3, features=1025, dtype='fp32', weighted=True, dropped=0.1, train=True),
        # a recurrent layer in training: ragged sequences, a gate of its own for every channel
        dict(name='scan train', op='scan', sequences=37, tokens=65536, heads=2048, width=1, dtype='bf16', gate='bf16', state=False, pad=500, train=True),
        # one long sequence, one gate for each head (shared by its 64 channels)
        dict(name='scan long', op='scan', sequences=1, tokens=131072, heads=8, width=64, dtype='fp32', gate='fp32', state=True, pad=0, train=True),
        # many short sequences that go on from states, an odd number of channels
        dict(name='scan short', op='scan', sequences=3001, tokens=60000, heads=333, width=1, dtype='fp16', gate='fp16', state=True, pad=0, train=True),
        # one decoding step of the recurrence: a token for each running sequence, states updated in place
        dict(name='step decode', op='step', sequences=128, heads=4096, width=1, dtype='bf16', gate='fp32'),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width_like(rng, low, high):
    """A row length: any number (odd ones among them), or a multiple of 2, 8 or 64."""
    n, of = _spread(rng, low, high), rng.choice((1, 1, 2, 8, 64, 64))
    return max(of, n // of * of) if n >= of else n


def draw(rng):
    op = rng.choice(('topk', 'sort', 'dispatch', 'combine', 'scan', 'scan', 'step'))
    dtype = rng.choice(('fp32', 'fp16', 'bf16', 'bf16'))
    train = rng.random() < 0.7
    if op == 'topk':
        experts = _spread(rng, 4, 512)
        k = rng.randint(1, min(experts, 10))
        return dict(op=op, tokens=_spread(rng, 1, min(65536, _MOST_LOGITS // experts)), experts=experts, k=k, dtype=dtype,
                    normalize=rng.random() < 0.6, masked=rng.choice((0, 0, experts // 8, experts - 1)), train=train)
    if op == 'sort':
        k = rng.randint(1, 10)
        return dict(op=op, tokens=_spread(rng, 1, _MOST_ENTRIES // k), experts=_spread(rng, 2, 512), k=k,
                    dropped=rng.choice((0.0, 0.05, 0.4)))
    if op in ('dispatch', 'combine'):
        k, features = rng.randint(1, 8), _width_like(rng, 32, 8192)
        most = _MOST_ROWS // (k * features * (2 if dtype == 'fp32' else 1) * 2)
        return dict(op=op, tokens=_spread(rng, 1, min(65536, most)), experts=_spread(rng, 4, 256), k=k, features=features,
                    dtype=dtype, weighted=op == 'combine' or rng.random() < 0.3, dropped=rng.choice((0.0, 0.05, 0.3)), train=train)
    if op == 'step':
        heads, width = _heads(rng)
        return dict(op=op, sequences=_spread(rng, 1, 1024), heads=heads, width=width, dtype=dtype, gate=rng.choice((dtype, 'fp32')))
    heads, width = _heads(rng)
    most = _MOST_SCAN // (heads * width * (4 if dtype == 'fp32' else 2))
    tokens = _spread(rng, 1, min(131072, most))
    return dict(op=op, sequences=_spread(rng, 1, max(1, min(4096, tokens // 2))), tokens=tokens, heads=heads, width=width,
                dtype=dtype, gate=rng.choice((dtype, dtype, 'fp32')), state=rng.random() < 0.5, pad=rng.choice((0, 0, 17, 200)), train=train)


def _heads(rng):
    """(gates a token has, channels that share one): a gate for every channel, or one for each head."""
    if rng.random() < 0.5:
        return _width_like(rng, 16, 4096), 1
    return _spread(rng, 1, 32), rng.choice((16, 32, 64, 64, 128, 24, 33))


# ---- inputs ------------------------------------------------------------------------------------------------------

def _choices(case, gen, dev):
    """[tokens, k] experts: k different ones for each token, drawn with a skewed load; dropped ones are -1."""
    T, E, k = case['tokens'], case['experts'], min(case['k'], case['experts'])
    load = -0.5 * torch.log1p(torch.arange(E, device=dev, dtype=torch.float32))
    index = torch.empty(T, k, dtype=torch.long, device=dev)
    for lo in range(0, T, 65536):
        noise = torch.rand(min(65536, T - lo), E, device=dev, generator=gen).clamp_min_(1e-9)
        index[lo:lo + 65536] = (load - torch.log(-torch.log(noise))).topk(k, dim=1).indices
    if case['dropped']:
        half = case['dropped'] / 2
        index[torch.rand(T, device=dev, generator=gen) < half] = -1
        index[torch.rand(T, k, device=dev, generator=gen) < half] = -1
    return index


def _lengths(case, seed):
    """Lengths of the sequences: log-normal, adding up to the case's tokens; where there are several some are empty."""
    S, T = case['sequences'], case['tokens']
    if S == 1:
        return [T]
    r = np.random.RandomState(seed % (1 << 31))
    part = np.exp(0.8 * r.randn(S)) * (r.rand(S) > 0.03)
    part[r.randint(S)] += 1e-3
    ends = np.floor(np.cumsum(part) / part.sum() * T + 0.5).astype(np.int64)
    ends[-1] = T
    return np.diff(np.concatenate([[0], ends])).tolist()


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, s = case['op'], dict(case)
    randn = lambda *shape: torch.randn(*shape, device=dev, generator=gen)  # noqa: E731
    if op == 'topk':
        dtype, T, E = _DTYPES[case['dtype']], case['tokens'], case['experts']
        logits = 1.5 * randn(T, E)
        if case['masked']:  # experts that a token may not use
            away = torch.rand(T, E, device=dev, generator=gen).argsort(dim=1)[:, :case['masked']]
            logits.scatter_(1, away, -math.inf)
        s['logits'] = logits.to(dtype).requires_grad_(case['train'])
        s['grad'] = randn(T, case['k'])
    elif op == 'sort':
        s['index'] = _choices(case, gen, dev)
    elif op in ('dispatch', 'combine'):
        dtype = _DTYPES[case['dtype']]
        index = _choices(case, gen, dev)
        T, k = index.shape
        s['slot'], s['order'], s['indptr'] = _sort_plain(index, case['experts'])
        weight = torch.rand(T, k, device=dev, generator=gen) + 0.05
        s['weight'] = (weight / weight.sum(1, keepdim=True)).requires_grad_(case['train']) if case['weighted'] else None
        few, many = randn(T, case['features']).to(dtype), randn(T * k, case['features']).to(dtype)
        s['x'], s['grad'] = (few, many) if op == 'dispatch' else (many, few)
        s['x'].requires_grad_(case['train'])
    else:
        dtype, gdtype, H, P = _DTYPES[case['dtype']], _DTYPES[case['gate']], case['heads'], case['width']
        rows = case['sequences'] if op == 'step' else case['tokens'] + case['pad']
        shape = (rows, H) if P == 1 else (rows, H, P)
        gates = (rows, H) if P == 1 else (rows, H, 1)
        s['src'] = randn(*shape).to(dtype)
        # decays from a few tokens to a few thousand, as such layers are initialised, moved by the token
        slow = torch.rand(H, device=dev, generator=gen) * 7 + 1
        s['gate'] = torch.sigmoid(slow.reshape((H,) if P == 1 else (H, 1)) + randn(*gates)).to(gdtype)
        if op == 'step':
            s['state'] = randn(case['sequences'], *shape[1:])
            return s
        lens = _lengths(case, seed)
        s['longest'] = max(lens)
        ends = np.concatenate([[0], np.cumsum(lens)])
        s['indptr'] = torch.tensor(ends, dtype=torch.long, device=dev)
        # the sequences that have a token, and their first and last one
        some = np.flatnonzero(np.diff(ends))
        s['some'], s['first'], s['end'] = (torch.tensor(v, device=dev) for v in (some, ends[some], ends[some + 1] - 1))
        s['state'] = randn(len(lens), *shape[1:]).requires_grad_(case['train']) if case['state'] else None
        s['grad'] = randn(*shape).to(dtype)
        s['grad_last'] = randn(len(lens), *shape[1:])
        s['src'].requires_grad_(case['train'])
        s['gate'].requires_grad_(case['train'])
    return s


# ---- the operators -----------------------------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import pytorch_scatter_b200 as ts
    op, train = s['op'], s.get('train', False)
    if op == 'topk':
        weight, index = ts.expert_topk(s['logits'], s['k'], s['normalize'])
        out = {'weight': weight, 'index': index}
        if train:
            out['grad_logits'], = torch.autograd.grad(weight, (s['logits'],), s['grad'])
        return out
    if op == 'sort':
        slot, order, indptr = ts.expert_sort(s['index'], s['experts'])
        return {'slot': slot, 'order': order, 'indptr': indptr}
    if op in ('dispatch', 'combine'):
        call = ts.expert_dispatch if op == 'dispatch' else ts.expert_combine
        out = {'out': call(s['x'], s['slot'], s['indptr'], s['weight'])}
        if train:
            leaves = (s['x'],) if s['weight'] is None else (s['x'], s['weight'])
            grads = torch.autograd.grad(out['out'], leaves, s['grad'])
            out.update(zip(('grad_x', 'grad_weight'), grads))
        return out
    if op == 'step':
        return {'out': ts.scan_step(s['src'], s['gate'], s['state']), 'state': s['state']}
    if s['state'] is None:
        out = {'out': ts.scan_csr(s['src'], s['gate'], s['indptr'])}
        if train:
            out['grad_src'], out['grad_gate'] = torch.autograd.grad(out['out'], (s['src'], s['gate']), s['grad'])
        return out
    res, last = ts.scan_csr_state(s['src'], s['gate'], s['indptr'], s['state'])
    out = {'out': res, 'last': last}
    if train:
        grads = torch.autograd.grad((res, last), (s['src'], s['gate'], s['state']), (s['grad'], s['grad_last']))
        out.update(zip(('grad_src', 'grad_gate', 'grad_state'), grads))
    return out


def _sort_plain(index, experts):
    flat = index.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, order = key.sort(stable=True)
    indptr = torch.searchsorted(key, torch.arange(experts + 1, device=key.device))
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    return torch.where(place < indptr[-1], place, -1).reshape(index.shape), order, indptr


def _gather_rows(many, slot):
    """[tokens, k, features] in 32 bits: the row of each entry, zeros for dropped ones."""
    return many[slot.clamp_min(0)].float() * (slot >= 0).unsqueeze(-1)


@torch.no_grad()
def _run_plain(s):
    op, train = s['op'], s.get('train', False)
    if op == 'topk':
        logits, k = s['logits'].float(), s['k']
        value, index = logits.sort(dim=1, descending=True, stable=True)
        value, index = value[:, :k], index[:, :k]
        index = torch.where(value == -math.inf, -1, index)
        prob = torch.exp(logits - logits.amax(1, keepdim=True))
        prob = prob / prob.sum(1, keepdim=True)
        weight = torch.where(index >= 0, prob.gather(1, index.clamp_min(0)), 0.0)
        total = weight.sum(1, keepdim=True)
        out = {'weight': weight / total if s['normalize'] else weight, 'index': index}
        if train:
            g = s['grad']
            if s['normalize']:
                at = out['weight'] * (g - (out['weight'] * g).sum(1, keepdim=True))
                grad = torch.zeros_like(logits)
            else:
                at = weight * g
                grad = -prob * at.sum(1, keepdim=True)
            grad.scatter_add_(1, index.clamp_min(0), torch.where(index >= 0, at, 0.0))
            out['grad_logits'] = grad.to(s['logits'].dtype)
        return out
    if op == 'sort':
        return dict(zip(('slot', 'order', 'indptr'), _sort_plain(s['index'], s['experts'])))
    if op in ('dispatch', 'combine'):
        slot, weight, dtype = s['slot'], s['weight'], s['x'].dtype
        few, many = (s['x'], s['grad']) if op == 'dispatch' else (s['grad'], s['x'])
        order, k = s['order'], slot.size(1)

        def spread():
            rows = few[order // k].float()
            if weight is not None:
                rows = rows * weight.reshape(-1)[order].unsqueeze(-1)
            behind = torch.arange(order.numel(), device=order.device) >= s['indptr'][-1]
            return rows.masked_fill(behind.unsqueeze(-1), 0).to(dtype)

        def fold():
            v = _gather_rows(many, slot)
            return (v.sum(1) if weight is None else (v * weight.unsqueeze(-1)).sum(1)).to(dtype)

        out = {'out': spread() if op == 'dispatch' else fold()}
        if train:
            out['grad_x'] = fold() if op == 'dispatch' else spread()
            if weight is not None:
                out['grad_weight'] = (_gather_rows(many, slot) * few.float().unsqueeze(1)).sum(-1)
        return out
    src, gate = s['src'].float(), s['gate'].float()
    if op == 'step':
        s['state'].copy_(gate * s['state'] + src)
        return {'out': s['state'].to(s['src'].dtype), 'state': s['state']}

    some, first, end, live = s['some'], s['first'], s['end'], s['tokens']
    state, dtype = s['state'], s['src'].dtype
    init = torch.zeros(some.numel(), *src.shape[1:], device=src.device) if state is None else state[some]
    carried = gate.clone()
    carried[live:] = 0
    carried[first] = 0  # a sequence takes nothing from the one before it
    begin = src.clone()
    begin[live:] = 0
    begin[first] += gate[first] * init
    h = _doubling(carried, begin, s['longest'])
    out = {'out': h.to(dtype)}
    if state is not None:
        last = state.detach().clone()
        last[some] = h[end]
        out['last'] = last
    if train:
        g = s['grad'].to(torch.float32, copy=True)
        g[live:] = 0
        if state is not None:
            g[end] += s['grad_last'][some]
        later = torch.zeros_like(carried)
        later[:-1] = carried[1:]
        dh = _doubling(later.flip(0), g.flip(0), s['longest']).flip(0)
        before = torch.zeros_like(h)
        before[1:] = h[:-1]
        before[first] = init
        dgate = dh * before
        dgate[live:] = 0
        out['grad_src'] = dh.to(dtype)
        out['grad_gate'] = (dgate.sum(-1, keepdim=True) if s['width'] > 1 else dgate).to(s['gate'].dtype)
        if state is not None:
            dstate = s['grad_last'].clone()
            dstate[some] = gate[first] * dh[first]
            out['grad_state'] = dstate
    return out


def _doubling(gate, value, longest):
    """h[t] = gate[t] * h[t-1] + value[t]: runs of twice the length from pairs of runs."""
    d = 1
    while d < longest:
        value = torch.cat([value[:d], torch.addcmul(value[d:], gate[d:], value[:-d])])
        gate = torch.cat([gate[:d], gate[d:] * gate[:-d]])
        d *= 2
    return value


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    op, train = case['op'], case.get('train', False)
    if op == 'sort':
        n = case['tokens'] * min(case['k'], case['experts'])
        return {'bytes': 24 * n + 8 * (case['experts'] + 1), 'flops': 0}
    b = _BYTES[case['dtype']]
    if op == 'topk':
        T, E, k = case['tokens'], case['experts'], case['k']
        return {'bytes': T * E * b * (2 if train else 1) + T * k * (12 + (4 if train else 0)), 'flops': T * E * (8 if train else 4)}
    if op in ('dispatch', 'combine'):
        T, k = case['tokens'], min(case['k'], case['experts'])
        few, many = T * case['features'], T * k * case['features'] * (1 - case['dropped'])
        small = 8 * T * k + (4 * T * k * (2 if train else 1) if case['weighted'] else 0)
        return {'bytes': (few + many) * b * (2 if train else 1) + small, 'flops': many * (4 if train else 1)}
    rows = case['sequences'] if op == 'step' else case['tokens']
    n, m = rows * case['heads'] * case['width'], rows * case['heads']
    g = _BYTES[case['gate']]
    if op == 'step':
        return {'bytes': n * (2 * b + 8) + m * g, 'flops': 2 * n}
    states = case['sequences'] * case['heads'] * case['width'] * 4 if case['state'] else 0
    return {'bytes': 2 * n * b + m * g + 2 * states + ((2 * n * b + m * g + 2 * states) if train else 0), 'flops': (6 if train else 2) * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    op, train = case['op'], case.get('train', False)
    if op == 'sort':
        return None
    if op == 'topk':
        x, k = s['logits'].double().cpu().numpy(), case['k']
        index = np.argsort(-x, axis=1, kind='stable')[:, :k]
        value = np.take_along_axis(x, index, 1)
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        w = np.take_along_axis(p, index, 1)
        if case['normalize']:
            w = w / w.sum(1, keepdims=True)
        out = {'weight': w, 'index': np.where(np.isneginf(value), -1, index)}
        if train:
            g = s['grad'].double().cpu().numpy()
            chosen = np.zeros(x.shape, bool)
            np.put_along_axis(chosen, index, True, 1)
            full = np.zeros(x.shape)
            np.put_along_axis(full, index, w * g, 1)
            # softmax over the chosen ones, or over all
            base = np.where(chosen, p, 0.0) / np.where(chosen, p, 0.0).sum(1, keepdims=True) if case['normalize'] else p
            out['grad_logits'] = full - base * full.sum(1, keepdims=True)
        return out
    if op in ('dispatch', 'combine'):
        few, many = (s['x'], s['grad']) if op == 'dispatch' else (s['grad'], s['x'])
        slot, k = s['slot'], s['slot'].size(1)
        spread = torch.zeros(many.shape, dtype=torch.float64, device=few.device)
        fold = torch.zeros(few.shape, dtype=torch.float64, device=few.device)
        dots = torch.zeros(slot.shape, dtype=torch.float64, device=few.device)
        for j in range(k):
            t = (slot[:, j] >= 0).nonzero()[:, 0]
            at = slot[t, j]
            w = 1.0 if s['weight'] is None else s['weight'][t, j].double().unsqueeze(1)
            spread.index_copy_(0, at, few[t].double() * w)
            v = many[at].double()
            fold.index_add_(0, t, v * w)
            if train and s['weight'] is not None:
                dots[t, j] = (v * few[t].double()).sum(1)
        out = {'out': spread if op == 'dispatch' else fold}
        if train:
            out['grad_x'] = fold if op == 'dispatch' else spread
            if s['weight'] is not None:
                out['grad_weight'] = dots
        return out
    src, gate = s['src'].detach().double(), s['gate'].detach().double()
    if op == 'step':
        h = gate * s['state'].double() + src
        return {'out': h, 'state': h}
    return _walk(s, src, gate, train)


def _walk(s, src, gate, train):
    """Token after token, all sequences that still have one at once."""
    indptr, S = s['indptr'], s['indptr'].numel() - 1
    lens, order = (indptr[1:] - indptr[:-1]).sort(descending=True)
    first = indptr[:-1][order]
    ascending = lens.flip(0).contiguous()
    left = (S - torch.searchsorted(ascending, torch.arange(s['longest'], device=lens.device), right=True)).tolist()
    start = torch.zeros(S, *src.shape[1:], dtype=torch.float64, device=src.device)
    if s['state'] is not None:
        start = s['state'].detach().double()[order]
    h, out, before = start.clone(), torch.zeros_like(src), torch.zeros_like(src)
    for t, n in enumerate(left):
        at = first[:n] + t
        before[at] = h[:n]
        h[:n] = gate[at] * h[:n] + src[at]
        out[at] = h[:n]
    back = torch.empty_like(order)
    back[order] = torch.arange(S, device=order.device)
    res = {'out': out}
    if s['state'] is not None:
        res['last'] = h[back]
    if train:
        g = s['grad'].double()
        d = torch.zeros_like(start) if s['state'] is None else s['grad_last'].double()[order]
        dsrc, dgate = torch.zeros_like(src), torch.zeros_like(gate)
        for t in range(len(left) - 1, -1, -1):
            n = left[t]
            at = first[:n] + t
            dh = d[:n] + g[at]
            dsrc[at] = dh
            dg = dh * before[at]
            dgate[at] = dg if dg.shape[1:] == gate.shape[1:] else dg.sum(-1, keepdim=True)
            d[:n] = gate[at] * dh
        res['grad_src'], res['grad_gate'] = dsrc, dgate
        if s['state'] is not None:
            res['grad_state'] = d[back]
    return res
