"""What is measured of the expert and gradient operators (diffusion_ccsp_amd.operators): rows sorted by expert and combined
back, the experts' products, the global gradient norm with clipping.

A case is a dict of plain values.  `run` computes one pass either in elementary torch operations in 32 bits (own = False) or
through the framework's entry points (own = True); `exact` computes the same in 64 bits."""
import math
import random

import torch

own = False

DEVICE = 'cuda:0'
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}


def listed():
    return [
        # one token of a served model on its way to 8 of 64 experts and back: nothing but latency
        dict(name='sort_one_token', op='sort', form='topk', tokens=1, k=8, experts=64, width=2048, dtype='bf16', grad=False, drop=0.0),
        # the training step of the denoiser on the benchmark batch: 2304 nodes, 20264 typed edges, both nodes' [geometry | pose] embeddings of every edge
        dict(name='sort_edges', op='sort', form='edges', tokens=2304, k=2, edges=20264, experts=13, width=512, dtype='fp32', grad=True, drop=0.0),
        # ragged in everything: an odd width (rows that start on odd 2-byte addresses), a tenth of the assignments dropped
        dict(name='sort_odd', op='sort', form='topk', tokens=4099, k=3, experts=13, width=1001, dtype='fp16', grad=True, drop=0.1),
        # a training step's share of a large routed layer
        dict(name='sort_top8_large', op='sort', form='topk', tokens=32768, k=8, experts=64, width=2048, dtype='bf16', grad=True, drop=0.0),
        # one token's eight experts: reads eight weight matrices for eight rows
        dict(name='linear_one_token', op='linear', rows=8, tail=0, experts=64, inp=2048, out=4096, dtype='bf16', act='silu', bias=False, grad=False, skew=0.0),
        # the type MLPs of the denoiser in its own precision: 13 types, [4H] -> [2H] at H = 256, training
        dict(name='linear_types', op='linear', rows=20264, tail=0, experts=13, inp=1024, out=512, dtype='fp32', act='silu', bias=True, grad=True, skew=0.5),
        # odd sizes: no row starts on 16 bytes, groups end inside tiles, dropped rows behind the last group
        dict(name='linear_odd', op='linear', rows=3001, tail=37, experts=7, inp=333, out=517, dtype='fp16', act='none', bias=True, grad=True, skew=0.5),
        # many small experts, some of them nearly empty
        dict(name='linear_many', op='linear', rows=8192, tail=0, experts=32, inp=2048, out=1408, dtype='bf16', act='silu', bias=False, grad=True, skew=1.0),
        # the products of a large routed layer's training step
        dict(name='linear_large', op='linear', rows=65536, tail=0, experts=16, inp=2048, out=4096, dtype='bf16', act='none', bias=True, grad=True, skew=0.3),
        # the parameters of the denoiser at H = 256 with its 13 type MLPs
        dict(name='clip_denoiser', op='clip', layout='denoiser', tensors=42, elements=0, dtype='fp32', align=64, ratio=0.5, seed=0),
        # many small tensors (adapters) of odd sizes, the clipped ones packed end to end: launch count decides
        dict(name='clip_adapters', op='clip', layout='generic', tensors=300, elements=400000, dtype='bf16', align=1, ratio=0.5, seed=1),
        # a rank's share of a large model, half of the tensors in 16 bits
        dict(name='clip_large', op='clip', layout='generic', tensors=391, elements=1000000000, dtype='mixed', align=64, ratio=0.25, seed=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['sort', 'sort', 'linear', 'linear', 'clip'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'sort':
        form = rng.choice(['topk', 'topk', 'edges'])
        width = _log(rng, 1, 4096)
        if rng.random() < 0.5 and width >= 64:
            width -= width % 64                                  # real widths are round as often as not
        most = min(262144, 32768 * 8 * 2048 * 2 // (width * BYTES[dtype]))
        if form == 'edges':
            edges = _log(rng, 1, most // 2)
            return dict(op='sort', form='edges', tokens=max(1, edges // rng.randint(1, 12)), k=2, edges=edges, experts=rng.randint(1, 30), width=width,
                        dtype=dtype, grad=rng.random() < 0.6, drop=rng.choice([0.0, 0.2]))
        experts = _log(rng, 2, 256)
        k = rng.randint(1, min(8, experts))
        return dict(op='sort', form='topk', tokens=max(1, _log(rng, 1, most) // k), k=k, experts=experts, width=width, dtype=dtype,
                    grad=rng.random() < 0.6, drop=rng.choice([0.0, 0.0, 0.3]))
    if op == 'linear':
        most = 65536 * 2048 * 4096 // (16 if dtype == 'fp32' else 1)
        inp, out = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.6:
            inp, out = max(16, inp - inp % 16), max(16, out - out % 16)
        experts = min(_log(rng, 1, 64), max(1, most // (inp * out)))
        return dict(op='linear', rows=_log(rng, 1, max(1, min(65536, most // (inp * out)))), tail=rng.choice([0, 0, 1, 100]), experts=experts, inp=inp, out=out,
                    dtype=dtype, act=rng.choice(['none', 'silu']), bias=rng.random() < 0.5, grad=rng.random() < 0.6, skew=rng.choice([0.0, 0.5, 1.5]))
    return dict(op='clip', layout='generic', tensors=_log(rng, 1, 800), elements=_log(rng, 1, 500000000), dtype=rng.choice(['fp32', 'bf16', 'fp16', 'mixed']),
                align=rng.choice([1, 64, 64]),
                ratio=rng.choice([0.1, 0.7, 3.0]), seed=rng.randint(0, 1 << 20))


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _sizes(case):
    """shapes of the gradients: the denoiser's own (hidden width 256, 13 types), or sizes spread over four decades, empty and odd ones among them"""
    if case['layout'] == 'denoiser':
        H, P, n = 256, 4, 13
        sh = [(H // 2, 2), (H // 2,), (H, H // 2), (H,), (H // 2, P), (H // 2,), (H, H // 2), (H,), (H // 2, H), (H // 2,), (P, H // 2), (P,),
              (4 * H, H), (4 * H,), (H, 4 * H), (H,)]
        return sh + [s for _ in range(n) for s in ((2 * H, 5 * H), (2 * H,))]
    r = random.Random(case['seed'])
    w = [math.exp(r.uniform(0.0, 9.0)) for _ in range(case['tensors'])]
    total = sum(w)
    sizes = [int(case['elements'] * v / total) for v in w]
    sizes[-1] += case['elements'] - sum(sizes)
    return [(n,) for n in sizes]


def _clip_dtypes(case, n):
    if case['dtype'] != 'mixed':
        return [DTYPES[case['dtype']]] * n
    return [torch.bfloat16 if i % 2 else torch.float32 for i in range(n)]


def _normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case['op'] == 'clip':
        sizes = _sizes(case)
        scale = random.Random(seed)
        grads = [_normal(s, gen, dt, 10.0 ** scale.uniform(-4, -1)) for s, dt in zip(sizes, _clip_dtypes(case, len(sizes)))]
        # the clipped gradients are views of one flat buffer per type, as a bucket of gradients is
        flat, place = {}, {}
        for g in grads:
            place[g.dtype] = place.get(g.dtype, 0) + -(-g.numel() // case['align']) * case['align']
        for dt, n in place.items():
            flat[str(dt)] = torch.zeros(n, dtype=dt, device=DEVICE)
        out, at = [], dict.fromkeys(place, 0)
        for g in grads:
            out.append(flat[str(g.dtype)][at[g.dtype]:at[g.dtype] + g.numel()].view(g.shape))
            at[g.dtype] += -(-g.numel() // case['align']) * case['align']
        total = math.sqrt(sum(float(g.float().pow(2).sum()) for g in grads)) if len(grads) <= 64 else math.sqrt(1e-3 * sum(g.numel() for g in grads))
        return dict(case=case, grads=grads, out=out, flat=flat, max_norm=max(case['ratio'] * total, 1e-6))
    dt = DTYPES[case['dtype']]
    E = case['experts']
    if case['op'] == 'sort':
        N, k, D = case['tokens'], case['k'], case['width']
        if case['form'] == 'edges':
            popular = torch.randn(E, generator=gen, device=DEVICE).mul(0.7).exp()
            kind = torch.multinomial(popular, case['edges'], replacement=True, generator=gen)
            if case['drop'] > 0:
                kind = torch.where(torch.rand(case['edges'], generator=gen, device=DEVICE) < case['drop'], torch.full_like(kind, -1), kind)
            expert = kind[:, None].expand(-1, 2).contiguous()
            token = torch.randint(0, N, (case['edges'], 2), generator=gen, device=DEVICE)
            degree = torch.bincount(token.reshape(-1), minlength=N).float()
            weight = degree.rsqrt()[token].contiguous()
        else:
            score = torch.randn(N, E, generator=gen, device=DEVICE) + 0.7 * torch.randn(E, generator=gen, device=DEVICE)
            top, expert = torch.topk(score, k, dim=1)
            token, weight = None, torch.softmax(top, dim=1)
            if case['drop'] > 0:
                expert = torch.where(torch.rand(N, k, generator=gen, device=DEVICE) < case['drop'], torch.full_like(expert, -1), expert)
        A = expert.numel()
        st = dict(case=case, expert=expert, token=token, weight=weight, x=_normal((N, D), gen, dt), ys=_normal((A, D), gen, dt))
        if case['grad']:
            st['g_xs'], st['g_y'] = _normal((A, D), gen, dt), _normal((N, D), gen, dt)
        return st
    R, tail, I, O = case['rows'], case['tail'], case['inp'], case['out']
    popular = (torch.randn(E, generator=gen, device=DEVICE) * case['skew']).exp()
    kind, _ = torch.sort(torch.multinomial(popular, R, replacement=True, generator=gen))
    counts = torch.bincount(kind, minlength=E)
    expert = torch.cat([kind, torch.full((tail,), -1, device=DEVICE, dtype=kind.dtype)])
    bound = 1.0 / math.sqrt(I)
    st = dict(case=case, expert=expert, counts=counts.tolist(), xs=_normal((R + tail, I), gen, dt),
              weight=((torch.rand(E, O, I, generator=gen, device=DEVICE) * 2 - 1) * bound).to(dt), bias=None)
    if tail:
        st['xs'][R:] = 0                                       # what sort_rows leaves behind the last group
    if case['bias']:
        st['bias'] = ((torch.rand(E, O, generator=gen, device=DEVICE) * 2 - 1) * bound).to(dt)
    if case['grad']:
        st['g_y'] = _normal((R + tail, O), gen, dt)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        if case['op'] == 'linear':
            from diffusion_ccsp_amd import operators
            st['plan'] = operators.route(st['expert'], case['experts'])          # made once a layer, used by every product in it
        if case.get('grad'):
            for name in ('x', 'ys', 'xs', 'weight', 'bias'):
                if st.get(name) is not None:
                    st[name].requires_grad_(True)
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state):
    op = state['case']['op']
    if own:
        return {'sort': _own_sort, 'linear': _own_linear, 'clip': _own_clip}[op](state)
    with torch.no_grad():
        return {'sort': _plain_sort, 'linear': _plain_linear, 'clip': _plain_clip}[op](state)


def _own_sort(st):
    from diffusion_ccsp_amd import operators
    case = st['case']
    plan = operators.route(st['expert'], case['experts'], tokens=st['token'], n_tokens=case['tokens'])
    xs = operators.sort_rows(st['x'], plan)
    y = operators.combine_rows(st['ys'], plan, st['weight'])
    out = dict(offsets=plan.offsets, rows=plan.rows, xs=xs, y=y)
    if case['grad']:
        out['d_x'], out['d_ys'], out['d_weight'] = torch.autograd.grad([xs, y], [st['x'], st['ys'], st['weight']], [st['g_xs'], st['g_y']])
        out['xs'], out['y'] = xs.detach(), y.detach()
    return out


def _own_linear(st):
    from diffusion_ccsp_amd import operators
    case = st['case']
    act = None if case['act'] == 'none' else case['act']
    y = operators.expert_linear(st['xs'], st['weight'], st['plan'], bias=st['bias'], activation=act)
    if not case['grad']:
        return dict(y=y)
    wrt = [t for t in (st['xs'], st['weight'], st['bias']) if t is not None]
    g = torch.autograd.grad(y, wrt, st['g_y'])
    return dict(zip(['y', 'd_xs', 'd_weight', 'd_bias'], (y.detach(),) + g))


def _own_clip(st):
    from diffusion_ccsp_amd import operators
    norm = operators.clip_global_norm(st['grads'], st['max_norm'], out=st['out'])
    return dict(norm=norm, grads=st['flat'])


def _order(st):
    """assignments in the order of their experts (the dropped ones behind), their rows, the experts' first rows"""
    case = st['case']
    E = case['experts']
    e = st['expert'].reshape(-1)
    key = torch.where((e >= 0) & (e < E), e, torch.full_like(e, E))
    order = torch.sort(key, stable=True)[1]
    rows = torch.empty_like(order)
    rows[order] = torch.arange(order.numel(), device=order.device)
    rows = torch.where(key < E, rows, torch.full_like(rows, -1))
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=order.device)
    offsets[1:] = torch.cumsum((key[:, None] == torch.arange(E, device=key.device)).sum(0), 0).to(torch.int32)
    token = st['token'].reshape(-1) if st['token'] is not None else torch.arange(key.numel(), device=key.device) // case['k']
    return order, rows.to(torch.int32), offsets, token, key < E


def _plain_sort(st):
    case, dt = st['case'], st['x'].dtype
    N = case['tokens']
    order, rows, offsets, token, active = _order(st)
    x, ys, w = st['x'].float(), st['ys'].float(), st['weight'].reshape(-1).float() * active
    live = active[order][:, None].float()
    tok = token[order]
    row = rows.clamp(min=0).long()
    y = torch.zeros(N, x.shape[1], device=x.device).index_add_(0, token, ys[row] * w[:, None])
    out = dict(offsets=offsets, rows=rows, xs=(x[tok] * live).to(dt), y=y.to(dt))
    if case['grad']:
        g_xs, g_y = st['g_xs'].float(), st['g_y'].float()
        out['d_x'] = torch.zeros_like(x).index_add_(0, token, g_xs[row] * active[:, None].float()).to(dt)
        out['d_ys'] = (g_y[tok] * w[order][:, None]).to(dt)
        out['d_weight'] = ((g_y[token] * ys[row]).sum(1) * active).reshape(st['weight'].shape)
    return out


def _plain_linear(st):
    case, dt = st['case'], st['xs'].dtype
    xs, O = st['xs'].float(), case['out']
    y = torch.zeros(xs.shape[0], O, device=xs.device)
    dxs, dw, db = torch.zeros_like(xs), torch.zeros(st['weight'].shape, device=xs.device), torch.zeros(case['experts'], O, device=xs.device)
    r0 = 0
    for e, n in enumerate(st['counts']):
        if n == 0:
            continue
        x, w = xs[r0:r0 + n], st['weight'][e].float()
        z = x @ w.t()
        if st['bias'] is not None:
            z = z + st['bias'][e].float()
        y[r0:r0 + n] = z * torch.sigmoid(z) if case['act'] == 'silu' else z
        if case['grad']:
            dz = st['g_y'][r0:r0 + n].float()
            if case['act'] == 'silu':
                s = torch.sigmoid(z)
                dz = dz * (s * (1 + z * (1 - s)))
            dxs[r0:r0 + n] = dz @ w
            dw[e] = dz.t() @ x
            db[e] = dz.sum(0)
        r0 += n
    if not case['grad']:
        return dict(y=y.to(dt))
    out = dict(y=y.to(dt), d_xs=dxs.to(dt), d_weight=dw.to(dt))
    if st['bias'] is not None:
        out['d_bias'] = db.to(dt)
    return out


def _plain_clip(st):
    # squares of 32-bit gradients leave 32 bits' range: summed in 64
    total = torch.zeros((), dtype=torch.float64, device=DEVICE)
    for g in st['grads']:
        total = total + (g.double() * g.double()).sum()
    norm = torch.sqrt(total)
    scale = torch.clamp(st['max_norm'] / (norm + 1e-6), max=1.0).float()
    for g, o in zip(st['grads'], st['out']):
        o.copy_(g.float() * scale)
    return dict(norm=norm.float(), grads=st['flat'])


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    st = _inputs(case, seed)
    if case['op'] == 'clip':
        norm = math.sqrt(sum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in st['grads']))
        c = min(1.0, st['max_norm'] / (norm + 1e-6))
        want, at = {k: torch.zeros(f.shape, dtype=torch.float64, device=DEVICE) for k, f in st['flat'].items()}, {}
        for g in st['grads']:
            key = str(g.dtype)
            lo = at.get(key, 0)
            want[key][lo:lo + g.numel()] = g.reshape(-1).double() * c
            at[key] = lo + (g.numel() + case['align'] - 1) // case['align'] * case['align']
        return dict(norm=torch.tensor(norm, dtype=torch.float64), grads=want)
    if case['op'] == 'sort':
        ids = st['expert'].reshape(-1).tolist()
        toks = st['token'].reshape(-1).tolist() if st['token'] is not None else [a // case['k'] for a in range(len(ids))]
        by = [[] for _ in range(case['experts'])]
        for a, e in enumerate(ids):
            if 0 <= e < case['experts']:
                by[e].append(a)
        flat = torch.tensor([a for b in by for a in b], dtype=torch.long, device=DEVICE)
        tok = torch.tensor(toks, dtype=torch.long, device=DEVICE)[flat]
        n = flat.numel()
        x, ys, w = st['x'].double(), st['ys'].double(), st['weight'].reshape(-1).double()
        xs = torch.zeros(len(ids), x.shape[1], dtype=torch.float64, device=DEVICE)
        xs[:n] = x[tok]
        y = torch.zeros_like(x).index_add_(0, tok, ys[:n] * w[flat][:, None])
        out = dict(offsets=None, rows=None, xs=xs, y=y)
        if case['grad']:
            g_xs, g_y = st['g_xs'].double(), st['g_y'].double()
            out['d_x'] = torch.zeros_like(x).index_add_(0, tok, g_xs[:n])
            out['d_ys'] = torch.zeros_like(xs)
            out['d_ys'][:n] = g_y[tok] * w[flat][:, None]
            dw = torch.zeros_like(w)
            dw[flat] = (g_y[tok] * ys[:n]).sum(1)
            out['d_weight'] = dw.reshape(st['weight'].shape)
        return out
    xs, W = st['xs'].double(), st['weight'].double()
    y = torch.zeros(xs.shape[0], case['out'], dtype=torch.float64, device=DEVICE)
    out = dict(y=y)
    if case['grad']:
        out['d_xs'], out['d_weight'] = torch.zeros_like(xs), torch.zeros_like(W)
        if st['bias'] is not None:
            out['d_bias'] = torch.zeros(case['experts'], case['out'], dtype=torch.float64, device=DEVICE)
    ends = torch.cumsum(torch.tensor(st['counts']), 0).tolist()
    for e, hi in enumerate(ends):
        rows = slice(ends[e - 1] if e else 0, hi)
        if rows.start == hi:
            continue
        z = torch.mm(xs[rows], W[e].t())
        if st['bias'] is not None:
            z += st['bias'][e].double()
        sig = 1.0 / (1.0 + torch.exp(-z))
        y[rows] = z * sig if case['act'] == 'silu' else z
        if case['grad']:
            g = st['g_y'][rows].double()
            if case['act'] == 'silu':
                g = g * (sig + z * sig * (1.0 - sig))
            out['d_xs'][rows] = torch.mm(g, W[e])
            out['d_weight'][e] = torch.mm(g.t(), xs[rows])
            if st['bias'] is not None:
                out['d_bias'][e] = g.sum(0)
    return out


def work(case):
    if case['op'] == 'clip':
        sizes = [math.prod(s) for s in _sizes(case)]
        b = sum(n * torch.empty((), dtype=dt).element_size() for n, dt in zip(sizes, _clip_dtypes(case, len(sizes))))
        return dict(bytes=2 * b, flops=3 * sum(sizes))
    s = BYTES[case['dtype']]
    if case['op'] == 'sort':
        N, D = case['tokens'], case['width']
        A = case['edges'] * 2 if case['form'] == 'edges' else N * case['k']
        byts, flops = s * D * 2 * (N + A) + A * (8 + 4 + 4), 2 * A * D
        if case['grad']:
            byts, flops = byts + s * D * 2 * (N + A) + 4 * A, flops + 4 * A * D
        return dict(bytes=byts, flops=flops)
    R, E, I, O = case['rows'], case['experts'], case['inp'], case['out']
    active = E * (1.0 - (1.0 - 1.0 / E) ** R)                    # experts that get a row, on average
    byts, flops = s * (R * I + active * O * I + R * O), 2 * R * I * O
    if case['grad']:
        byts, flops = byts + s * (R * I + R * O + E * O * I), 3 * flops
    return dict(bytes=int(byts), flops=flops)
