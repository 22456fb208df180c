"""The operators of diffusion_ccsp_amd.operators (include/ccsp_ops.h) against plain 64-bit restatements on the CPU.

Tolerances are bounds, worked out per element before the first run.  u(t) = finfo(t).eps / 2 is the relative error of one rounding to t.  A sum of n terms held in
32 bits is off by at most 2 n u(fp32) times the sum of the terms' magnitudes in any order (the 2 allows a matrix instruction whose inner adds
truncate); a result is rounded once to its type, plus half of that type's smallest step where it is subnormal."""
import ctypes
import math
import os
import re
import sys
import threading

import numpy as np
import pytest
import torch

from conftest import ROOT, worlds
from diffusion_ccsp_amd import CcspError, _ops
from diffusion_ccsp_amd import operators as ops

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
U32 = 2.0 ** -24


def u(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """half the smallest step of the type"""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def close(got, want, bound, what):
    got = got.detach().to(want.device).double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), '%s: %d of %d beyond the bound, worst %g over %g' % (
        what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float(torch.as_tensor(bound).expand_as(want)[bad].max()))


def plan_oracle(expert, E, token, N):
    """assignments by (expert, assignment) and by (token, assignment), in plain Python order"""
    e, t = expert.reshape(-1).tolist(), token.reshape(-1).tolist()
    act = [0 <= x < E and 0 <= y < N for x, y in zip(e, t)]
    by_expert = sorted((a for a in range(len(e)) if act[a]), key=lambda a: (e[a], a))
    by_token = sorted((a for a in range(len(e)) if act[a]), key=lambda a: (t[a], a))
    dropped = [a for a in range(len(e)) if not act[a]]
    return e, t, by_expert, by_token, dropped


def topk_tokens(expert):
    k = 1 if expert.dim() == 1 else expert.shape[1]
    return (torch.arange(expert.numel()) // max(k, 1)).reshape(expert.shape)


# ---- without a GPU: the library, the refusals ----------------------------------------------------------------------------

def test_library_exports_every_declared_symbol():
    text = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'ccsp_ops.h')).read(), flags=re.S)
    names = sorted(set(re.findall(r'\b(ccsp_ops_[a-z_0-9]+)\s*\(', text)))
    L = _ops.lib()
    assert len(names) == 14
    for n in names:
        assert hasattr(L, n), n
    assert L.ccsp_ops_version() // 1000 == _ops.OPS_ABI_MAJOR


def test_a_library_of_another_major_version_is_refused(monkeypatch):
    monkeypatch.setattr(_ops, '_lib', None)
    monkeypatch.setattr(_ops, 'OPS_ABI_MAJOR', _ops.OPS_ABI_MAJOR + 1)
    with pytest.raises(CcspError, match='ABI version'):
        _ops.lib()


def test_c_entries_refuse_before_any_launch():
    """every refusal below returns from the argument checks: no device is touched"""
    L = _ops.lib()
    ok = 64                                                       # (a non-null address that is never read)

    def refused(rc, word):
        assert rc != 0 and word in L.ccsp_ops_last_error().decode(), L.ccsp_ops_last_error()
    refused(L.ccsp_ops_route(ok, None, 16, 4, 2, 8, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), '32 or 64')
    refused(L.ccsp_ops_route(ok, None, 32, 5, 2, 8, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), 'tokens of 2 each')
    refused(L.ccsp_ops_route(ok, None, 32, 4, 2, 0, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), 'experts')
    refused(L.ccsp_ops_route(ok, None, 32, 4, 2, 1025, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), 'experts')
    refused(L.ccsp_ops_route(ok, None, 32, 4, 2, 8, 2, ok, ok, ok, ok, ok, None, None, ok, 3, None), 'workspace')
    refused(L.ccsp_ops_route(ok, ok, 32, 4, 0, 8, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), 'token_ptr')
    refused(L.ccsp_ops_route(None, None, 32, 4, 2, 8, 2, ok, ok, ok, ok, ok, None, None, ok, 1 << 20, None), 'null')
    assert L.ccsp_ops_route_workspace(-1, 4, 4, 0) == -1 and L.ccsp_ops_route_workspace((1 << 30) + 1, 4, 4, 0) == -1
    refused(L.ccsp_ops_rows_gather(7, 4, 4, ok, 4, ok, ok, ok, None, ok, None), 'type')
    refused(L.ccsp_ops_rows_gather(0, 4, 4, ok, 4, None, ok, ok, None, ok, None), 'null')
    refused(L.ccsp_ops_rows_gather(0, -1, 4, ok, 4, ok, ok, ok, None, ok, None), 'range')
    refused(L.ccsp_ops_rows_combine(1, 4, 8, 4, 2, None, None, ok, ok, 2, ok, 4, ok, None), 'weights')
    refused(L.ccsp_ops_rows_combine(1, 4, 8, 4, 2, None, None, None, None, 1, ok, 4, ok, None), 'null')
    refused(L.ccsp_ops_rows_combine(1, 4, 8, 4, 2, None, None, ok, None, 1, None, 4, ok, None), 'null')
    refused(L.ccsp_ops_rows_combine(1, 4, 7, 4, 2, None, None, ok, None, 1, ok, 4, ok, None), 'tokens of 2 each')
    refused(L.ccsp_ops_rows_combine(1, 4, 7, 4, 0, ok, None, ok, None, 1, ok, 4, ok, None), 'token_assign')
    refused(L.ccsp_ops_rows_back(1, 4, 4, ok, ok, ok, None, ok, 2, ok, 4, ok, 4, ok, ok, None), 'weights')
    refused(L.ccsp_ops_linear(0, 4, 4, 0, 4, ok, ok, 4, ok, None, 0, ok, None, None, 0, None), 'range')
    refused(L.ccsp_ops_linear(0, 4, 4, 4, 4, ok, ok, 4, ok, None, 5, ok, None, None, 0, None), 'activation')
    refused(L.ccsp_ops_linear(0, 4, 4, 4, 4, None, ok, 4, ok, None, 0, ok, None, None, 0, None), 'null')
    refused(L.ccsp_ops_linear(0, 4, 4, 4, 4, ok, ok, 4, None, None, 0, ok, None, None, 0, None), 'null')
    refused(L.ccsp_ops_linear(0, 4, 4, 5, 4, ok, ok, 5, ok, None, 0, ok, None, None, 0, None), 'workspace')
    refused(L.ccsp_ops_linear_back_input(0, 4, 4, 4, 4, ok, ok, 4, None, ok, None, 0, None), 'null')
    refused(L.ccsp_ops_linear_back_weight(0, 4, 4, 4, 4, ok, ok, 4, ok, 4, None, None, ok, 64, None), 'null')
    refused(L.ccsp_ops_linear_back_weight(0, 2, 2000, 4, 4, ok, ok, 4, ok, 4, ok, None, ok, 64, None), 'workspace')
    assert L.ccsp_ops_linear_workspace(2, 0, 2, 2000, 0, 4, ok, 4, ok, 4) == -1 and L.ccsp_ops_linear_workspace(3, 0, 2, 8, 4, 4, ok, 4, ok, 4) == -1
    assert L.ccsp_ops_linear_workspace(0, 0, 2, 8, 4, 4, ok, 4, ok, 4) == 0 and L.ccsp_ops_linear_workspace(0, 0, 2, 8, 4, 4, ok, 5, ok, 4) == 256
    refused(L.ccsp_ops_linear_silu_back(0, 4, 4, 4, ok, ok, 4, None, ok, None), 'null')
    sizes, types, ptrs = (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(0), (ctypes.c_void_p * 1)(64)
    refused(L.ccsp_ops_clip_norm(1, ptrs, ptrs, sizes, types, -1.0, ok, ok, ok, 64, None), 'negative')
    refused(L.ccsp_ops_clip_norm(1, ptrs, ptrs, sizes, types, 1.0, ok, None, ok, 64, None), 'factor')
    refused(L.ccsp_ops_clip_norm(1, ptrs, None, sizes, types, 1.0, ok, ok, ok, 8, None), 'workspace')
    types[0] = 9
    refused(L.ccsp_ops_clip_norm(1, ptrs, None, sizes, types, 1.0, ok, ok, ok, 64, None), 'type')
    assert L.ccsp_ops_norm_workspace(1, (ctypes.c_int64 * 1)(-4)) == -1


def test_cpu_tensors_are_refused():
    for call in (lambda: ops.route(torch.zeros(4, dtype=torch.int64), 2), lambda: ops.global_norm([torch.zeros(3)]),
                 lambda: ops.clip_global_norm([torch.zeros(3)], 1.0)):
        with pytest.raises(CcspError, match='no CPU fallback'):
            call()
    with pytest.raises(ValueError, match='no tensors'):
        ops.global_norm([])
    assert float(ops.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0


# ---- routes --------------------------------------------------------------------------------------------------------------

def ids(A, E, seed, drop, hot=False):
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(0, E, (A,), generator=g)
    if hot:
        e = torch.where(torch.rand(A, generator=g) < 0.9, torch.full_like(e, E // 2), e)
    if drop:
        far = torch.tensor([-1, E, E + 1000, -2 ** 31, 2 ** 31 - 1])
        e = torch.where(torch.rand(A, generator=g) < drop, far[torch.randint(0, 5, (A,), generator=g)], e)
    return e


def check_plan(plan, expert, E, token, N, listed):
    e, t, by_expert, by_token, dropped = plan_oracle(expert, E, token, N)
    A, n = len(e), len(by_expert)
    off, rows = plan.offsets.cpu().tolist(), plan.rows.cpu().tolist()
    counts = np.bincount([e[a] for a in by_expert], minlength=E) if n else np.zeros(E, int)
    assert off == [0] + np.cumsum(counts).tolist()
    want = [-1] * A
    for p, a in enumerate(by_expert):
        want[a] = p
    assert rows == want
    assert plan.assign.cpu().tolist() == by_expert + [~a for a in dropped]
    assert plan.row_token.cpu().tolist() == [t[a] for a in by_expert] + [-1] * (A - n)
    assert plan.counts.cpu().tolist() == counts.tolist()
    if listed:
        ptr = plan.token_ptr.cpu().tolist()
        per = np.bincount([t[a] for a in by_token], minlength=N) if n else np.zeros(N, int)
        assert ptr == [0] + np.cumsum(per).tolist()
        assert plan.token_assign.cpu().tolist()[:n] == by_token


@pytest.mark.gpu
@pytest.mark.parametrize('A,E,drop,hot', [(1, 1, 0, False), (1, 64, 0, False), (63, 3, 0.2, False), (64, 13, 0, False), (65, 1024, 0.1, False), (2049, 13, 0.3, True), (8191, 1024, 0, False),
                                          (8192, 7, 1.0, False), (8193, 7, 0.1, True), (40001, 1024, 0.2, False), (150000, 64, 0, True)])
@pytest.mark.parametrize('bits', [32, 64])
def test_route_top_k(device, A, E, drop, hot, bits):
    expert = ids(A, E, A + E, drop, hot)
    if bits == 64 and drop:
        expert[::17] = 2 ** 40 + 1                                # (low half in range)
    expert = expert.to(torch.int32 if bits == 32 else torch.int64)
    for k in (1, 3):
        ex = expert[:A - A % k].reshape(-1, k) if k > 1 else expert
        if ex.numel() == 0:
            continue
        plan = ops.route(ex.to(device), E)
        check_plan(plan, ex, E, topk_tokens(ex), ex.shape[0], False)


@pytest.mark.gpu
@pytest.mark.parametrize('A,E,N,drop', [(1, 1, 1, 0), (5, 2, 3, 0.5), (700, 13, 90, 0.1), (8192, 13, 1023, 0), (8000, 13, 1024, 0), (8192, 40, 16384, 0.2), (500, 3, 16385, 0), (500, 3, 70000, 0.1),
                                        (9001, 13, 4095, 0.1), (9001, 13, 4096, 0), (40528, 13, 2304, 0), (30000, 1024, 1, 0), (50000, 5, 300000, 0.3)])
@pytest.mark.parametrize('bits', [32, 64])
def test_route_listed_tokens(device, A, E, N, drop, bits):
    dt = torch.int32 if bits == 32 else torch.int64
    expert, token = ids(A, E, A, drop).to(dt), ids(A, N, A + 1, drop / 2).to(dt)
    plan = ops.route(expert.to(device), E, tokens=token.to(device), n_tokens=N)
    check_plan(plan, expert, E, token, N, True)


@pytest.mark.gpu
def test_route_of_nothing(device):
    none = torch.zeros((0, 2), dtype=torch.int64, device=device)
    plan = ops.route(none, 5)
    assert plan.offsets.cpu().tolist() == [0] * 6 and plan.n_rows == 0 and plan.n_tokens == 0
    plan = ops.route(none, 5, tokens=none, n_tokens=3)
    assert plan.offsets.cpu().tolist() == [0] * 6 and plan.token_ptr.cpu().tolist() == [0] * 4
    x = torch.randn(3, 4, device=device, requires_grad=True)
    w = torch.randn(5, 6, 4, device=device, requires_grad=True)
    b = torch.randn(5, 6, device=device, requires_grad=True)
    xs = ops.sort_rows(x, plan)
    y = ops.combine_rows(ops.expert_linear(xs, w, plan, b, 'silu'), plan)
    assert tuple(xs.shape) == (0, 4) and torch.equal(y, torch.zeros(3, 6, device=device))
    g = torch.autograd.grad(y.sum(), [x, w, b])
    assert all(float(t.abs().max()) == 0.0 for t in g)


@pytest.mark.gpu
def test_assignments_of_no_tokens(device):
    """listed tokens of an empty layer: everything is dropped, every result is there and zero"""
    expert, tokens = torch.zeros((6, 2), dtype=torch.int64, device=device), torch.zeros((6, 2), dtype=torch.int64, device=device)
    plan = ops.route(expert, 3, tokens=tokens, n_tokens=0)
    check_plan(plan, expert.cpu(), 3, tokens.cpu(), 0, True)
    for D in (0, 5, 256):
        x = torch.zeros((0, D), device=device, requires_grad=True)
        ys = torch.full((12, D), float('nan'), device=device, requires_grad=True)
        w = torch.ones((6, 2), device=device, requires_grad=True)
        xs, y = ops.sort_rows(x, plan), ops.combine_rows(ys, plan, w)
        assert tuple(y.shape) == (0, D) and float(xs.detach().abs().sum()) == 0.0
        for g in torch.autograd.grad([xs, y], [x, ys, w], [torch.ones_like(xs), torch.ones_like(y)]):
            assert float(g.abs().sum()) == 0.0


@pytest.mark.gpu
def test_offsets_past_32_bits(device):
    """more than 2^31 elements (and more than 2^32 bytes) before the rows that are looked at: the last ones"""
    R, D, I = 1100000, 2048, 64
    g = torch.Generator(device=device).manual_seed(0)
    expert = (torch.arange(R, device=device) % 3)[:, None]
    plan = ops.route(expert, 3)
    x = torch.randn(R, D, generator=g, device=device, dtype=torch.float16)
    xs = ops.sort_rows(x, plan)
    p = torch.arange(R - 5000, R, device=device)
    tok = plan.row_token[p].long()
    assert torch.equal(xs[p], x[tok])
    y = ops.combine_rows(xs, plan)
    assert torch.equal(y[-5000:], x[-5000:])
    del xs, y
    small = torch.randn(R, I, generator=g, device=device, dtype=torch.float16).requires_grad_()
    w = (torch.randn(3, D, I, generator=g, device=device) / 8).half().requires_grad_()
    z = ops.expert_linear(small, w, plan)
    d_small, d_w = torch.autograd.grad(z, [small, w], x)
    s64, w64, x64 = small.detach()[p].double(), w.detach()[2].double(), x[p].double()        # (the last rows are expert 2's)
    want = s64 @ w64.t()
    close(z[p], want, u(torch.float16) * want.abs() + 2 * (I + 1) * U32 * (s64.abs() @ w64.abs().t()) + tiny(torch.float16), 'y')
    want = x64 @ w64
    close(d_small[p], want, u(torch.float16) * want.abs() + 2 * (D + 1) * U32 * (x64.abs() @ w64.abs()) + tiny(torch.float16), 'd xs')
    r = slice(int(plan.offsets[2]), R)
    want, mag = torch.zeros(D, I, dtype=torch.float64, device=device), torch.zeros(D, I, dtype=torch.float64, device=device)
    for lo in range(r.start, R, 50000):
        a, b = x[lo:min(lo + 50000, R)].double(), small.detach()[lo:min(lo + 50000, R)].double()
        want += a.t() @ b
        mag += a.abs().t() @ b.abs()
    close(d_w[2], want, u(torch.float16) * want.abs() + 2 * (R - r.start + 1) * U32 * mag + tiny(torch.float16), 'd weight')


@pytest.mark.gpu
def test_route_refusals(device):
    e = torch.zeros((4, 2), dtype=torch.int64, device=device)
    with pytest.raises(TypeError, match='int32 or int64'):
        ops.route(e.float(), 3)
    with pytest.raises(ValueError, match='experts'):
        ops.route(e, 0)
    with pytest.raises(ValueError, match='experts'):
        ops.route(e, 1025)
    with pytest.raises(ValueError, match='N, k'):
        ops.route(e[None], 3)
    with pytest.raises(ValueError, match='5 tokens'):
        ops.route(e, 3, n_tokens=5)
    with pytest.raises(ValueError, match='n_tokens'):
        ops.route(e, 3, tokens=e)
    with pytest.raises(ValueError, match='differ'):
        ops.route(e, 3, tokens=e.int(), n_tokens=4)
    with pytest.raises(ValueError, match='no expert'):
        ops.route(e[:, :0], 3)
    plan = ops.route(e, 3)
    x = torch.zeros(4, 5, device=device)
    with pytest.raises(ValueError, match='one row per token'):
        ops.sort_rows(x[:3], plan)
    with pytest.raises(TypeError, match='float64'):
        ops.sort_rows(x.double(), plan)
    with pytest.raises(ValueError, match='one row per assignment'):
        ops.combine_rows(x, plan)
    ys = torch.zeros(8, 5, device=device)
    with pytest.raises(ValueError, match='weights'):
        ops.combine_rows(ys, plan, torch.zeros(8, device=device))
    with pytest.raises(TypeError, match='weights'):
        ops.combine_rows(ys, plan, torch.zeros(4, 2, device=device, dtype=torch.float16))
    w = torch.zeros(3, 6, 5, device=device)
    with pytest.raises(ValueError, match='weight must be'):
        ops.expert_linear(ys, w[:2], plan)
    with pytest.raises(ValueError, match='bias must be'):
        ops.expert_linear(ys, w, plan, bias=w[:, :, 0].t())
    with pytest.raises(TypeError, match='one type'):
        ops.expert_linear(ys, w.half(), plan)
    with pytest.raises(ValueError, match='activation'):
        ops.expert_linear(ys, w, plan, activation='relu')
    with pytest.raises(CcspError, match='no CPU fallback'):
        ops.sort_rows(x.cpu(), plan)


# ---- rows there and back -------------------------------------------------------------------------------------------------

def strided(t, how, device):
    """the same values in another memory layout: rows further apart than their width, starting off the allocation's alignment"""
    t = t.to(device)
    if how == 'plain':
        return t
    if how == 'expanded':                                         # every row the first one
        return t[:1].expand(t.shape)
    wide = torch.full((t.shape[0], t.shape[1] + 3), float('nan'), dtype=t.dtype, device=device)
    wide[:, 1:1 + t.shape[1]] = t
    if how == 'offset':
        return wide[:, 1:1 + t.shape[1]]
    return t.t().contiguous().t()                                 # 'columns': the last dimension is not contiguous


ROWS = [(1, 1, 1, 1), (1, 8, 64, 40), (7, 3, 4, 5), (40, 2, 13, 4), (130, 4, 8, 72), (33, 1, 3, 1001), (257, 8, 16, 256), (19, 5, 1024, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize('N,k,E,D', ROWS)
@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('form', ['topk', 'listed'])
@pytest.mark.parametrize('layout', ['plain', 'offset', 'columns'])
def test_sort_and_combine_with_gradients(device, N, k, E, D, dtype, form, layout):
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(N * 1000 + D)
    expert = ids(N * k, E, N + k, 0.25).reshape(N, k)
    token = topk_tokens(expert) if form == 'topk' else ids(N * k, N, 3 * N, 0.1).reshape(N, k)
    x, g_y = torch.randn(N, D, generator=g).to(dt), torch.randn(N, D, generator=g).to(dt)
    ys, g_xs = torch.randn(N * k, D, generator=g).to(dt), torch.randn(N * k, D, generator=g).to(dt)
    for wdt in (None, torch.float32, dt):
        w = None if wdt is None else torch.randn(N, k, generator=g).to(wdt)
        e, t, by_expert, by_token, dropped = plan_oracle(expert, E, token, N)
        n = len(by_expert)
        ys_, gxs_ = ys.clone(), g_xs.clone()
        ys_[n:] = float('nan')                                    # what lies behind the last active row reaches nothing
        gxs_[n:] = float('nan')
        plan = ops.route(expert.to(device), E, **({} if form == 'topk' else dict(tokens=token.to(device), n_tokens=N)))
        xd, yd = strided(x, layout, device).requires_grad_(), strided(ys_, layout, device).requires_grad_()
        wd = None if w is None else w.to(device).requires_grad_()
        xs = ops.sort_rows(xd, plan)
        y = ops.combine_rows(yd, plan, wd)
        wrt = [xd, yd] + ([] if wd is None else [wd])
        grads = torch.autograd.grad([xs, y], wrt, [strided(gxs_, layout, device), strided(g_y, layout, device)])
        tok = torch.tensor([t[a] for a in by_expert], dtype=torch.long)
        X, YS, GY, GX = x.double(), ys.double(), g_y.double(), g_xs.double()
        W = torch.ones(N * k, dtype=torch.float64) if w is None else w.double().reshape(-1)
        wr = W[torch.tensor(by_expert, dtype=torch.long)][:, None]
        want_xs = torch.zeros(N * k, D, dtype=torch.float64)
        want_xs[:n] = X[tok]
        assert torch.equal(xs.detach().cpu().double(), want_xs)
        want_y, mag = torch.zeros(N, D, dtype=torch.float64), torch.zeros(N, D, dtype=torch.float64)
        want_dx, mag_x = want_y.clone(), want_y.clone()
        deg = torch.zeros(N, 1, dtype=torch.float64)
        want_y.index_add_(0, tok, YS[:n] * wr)
        mag.index_add_(0, tok, (YS[:n] * wr).abs())
        want_dx.index_add_(0, tok, GX[:n])
        mag_x.index_add_(0, tok, GX[:n].abs())
        deg.index_add_(0, tok, torch.ones(n, 1, dtype=torch.float64))
        close(y, want_y, u(dt) * want_y.abs() + 2 * (deg + 1) * U32 * mag + tiny(dt), 'y')
        close(grads[0], want_dx, u(dt) * want_dx.abs() + 2 * (deg + 1) * U32 * mag_x + tiny(dt), 'd x')
        want_dys = torch.zeros(N * k, D, dtype=torch.float64)
        want_dys[:n] = GY[tok] * wr
        close(grads[1], want_dys, (u(dt) + 2 * U32) * want_dys.abs() + tiny(dt), 'd ys')
        if w is not None:
            want_dw, mag_w = torch.zeros(N * k, dtype=torch.float64), torch.zeros(N * k, dtype=torch.float64)
            at = torch.tensor(by_expert, dtype=torch.long)
            want_dw[at], mag_w[at] = (GY[tok] * YS[:n]).sum(1), (GY[tok] * YS[:n]).abs().sum(1)
            bound = u(wdt) * want_dw.abs() + 2 * D * U32 * mag_w + tiny(wdt)
            close(grads[2].reshape(-1), want_dw, bound, 'd weights')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_rows_larger_than_the_last_level_cache(device, dtype):
    """200 MB of rows and more, which are written past the cache; dropped rows among them"""
    dt, N, k, E = DTYPES[dtype], 16384, 8, 20
    D = 512 if dt == torch.float32 else 1024
    expert = ids(N * k, E, 1, 0.1).reshape(N, k).to(device)
    plan = ops.route(expert, E)
    g = torch.Generator(device=device).manual_seed(0)
    x, gy = torch.randn(N, D, generator=g, device=device).to(dt), torch.randn(N, D, generator=g, device=device).to(dt)
    ys, w = torch.randn(N * k, D, generator=g, device=device).to(dt).requires_grad_(), torch.randn(N, k, generator=g, device=device).requires_grad_()
    n = int(plan.offsets[-1])
    a = plan.assign[:n].long()
    xs = ops.sort_rows(x, plan)
    assert torch.equal(xs[:n], x[a // k]) and float(xs[n:].abs().max()) == 0.0 and 0 < n < N * k
    y = ops.combine_rows(ys, plan, w)
    d_ys, d_w = torch.autograd.grad(y, [ys, w], gy)
    W, G, Y = w.detach().reshape(-1)[a].double()[:, None], gy[a // k].double(), ys.detach()[:n].double()
    want = torch.zeros(N, D, dtype=torch.float64, device=device).index_add_(0, a // k, Y * W)
    mag = torch.zeros(N, D, dtype=torch.float64, device=device).index_add_(0, a // k, (Y * W).abs())
    close(y, want, u(dt) * want.abs() + 2 * (k + 1) * U32 * mag + tiny(dt), 'y')
    close(d_ys[:n], G * W, (u(dt) + 2 * U32) * (G * W).abs() + tiny(dt), 'd ys')
    assert float(d_ys[n:].abs().max()) == 0.0
    want_w, mag_w = torch.zeros(N * k, dtype=torch.float64, device=device), torch.zeros(N * k, dtype=torch.float64, device=device)
    want_w[a], mag_w[a] = (G * Y).sum(1), (G * Y).abs().sum(1)
    close(d_w.reshape(-1), want_w, 2 * (D + 1) * U32 * mag_w + tiny(torch.float32), 'd weights')


@pytest.mark.gpu
def test_rows_keep_infinities_and_nan_of_active_rows_only(device):
    expert = torch.tensor([[0, 1], [1, -1], [-1, -1]])
    plan = ops.route(expert.to(device), 2)
    ys = torch.tensor([[1.0, float('inf')], [2.0, 3.0], [float('nan'), -float('inf')], [float('nan')] * 2, [float('nan')] * 2, [float('nan')] * 2], device=device)
    w = torch.tensor([[1.0, 1.0], [1.0, float('nan')], [float('inf'), float('nan')]], device=device)
    y = ops.combine_rows(ys, plan, w)                            # rows: (0, 0) -> 0, (0, 1) -> 1, (1, 0) -> 2
    want = torch.tensor([[3.0, float('inf')], [float('nan'), -float('inf')], [0.0, 0.0]])
    assert torch.equal(torch.nan_to_num(y.cpu(), nan=-7.0), torch.nan_to_num(want, nan=-7.0))


# ---- products ------------------------------------------------------------------------------------------------------------

def linear_case(counts, tail, I, O, dt, seed):
    g = torch.Generator().manual_seed(seed)
    R, E = sum(counts), len(counts)
    expert = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((tail,), -1)]).long()
    b = 1.0 / math.sqrt(I)
    xs, gy = torch.randn(R + tail, I, generator=g).to(dt), torch.randn(R + tail, O, generator=g).to(dt)
    w, bias = ((torch.rand(E, O, I, generator=g) * 2 - 1) * b * 2).to(dt), (torch.rand(E, O, generator=g) * 2 - 1).to(dt)
    return expert, xs, w, bias, gy


def check_linear(device, counts, tail, I, O, dt, act, with_bias, layout='plain', seed=0, where='cpu'):
    """where: the device that works out the 64-bit reference (large cases: the GPU's own 64-bit products)"""
    expert, xs, w, bias, gy = linear_case(counts, tail, I, O, dt, seed)
    R, E = sum(counts), len(counts)
    xs_, gy_ = xs.clone(), gy.clone()
    xs_[R:], gy_[R:] = float('nan'), float('nan')                # what lies behind the last group reaches nothing
    plan = ops.route(expert.to(device), E)
    xd, wd = strided(xs_, layout, device).requires_grad_(), w.to(device).requires_grad_()
    bd = bias.to(device).requires_grad_() if with_bias else None
    y = ops.expert_linear(xd, wd, plan, bd, act)
    got = torch.autograd.grad(y, [t for t in (xd, wd, bd) if t is not None], strided(gy_, layout, device))
    with torch.no_grad():
        assert torch.equal(ops.expert_linear(xd, wd, plan, bd, act), y)          # (the form that keeps no pre-activation)
    lo = 0
    xs, w, bias, gy = (t.to(where) for t in (xs, w, bias, gy))
    zeros = lambda *s: torch.zeros(s, dtype=torch.float64, device=where)      # noqa: E731
    want_y, by, want_x, bx = zeros(R + tail, O), zeros(R + tail, O), zeros(R + tail, I), zeros(R + tail, I)
    want_w, bw, want_b, bb = zeros(E, O, I), zeros(E, O, I), zeros(E, O), zeros(E, O)
    for e, n in enumerate(counts):
        s = slice(lo, lo + n)
        lo += n
        X, W, G = xs[s].double(), w[e].double(), gy[s].double()
        z = X @ W.t() + (bias[e].double() if with_bias else 0.0)
        ez = 2 * (I + 1) * U32 * (X.abs() @ W.abs().t() + (bias[e].double().abs() if with_bias else 0.0))
        sg = torch.sigmoid(z)
        if act:
            # |silu'| <= 1.1, |silu''| <= 0.5; the exponential, sum and quotient of the sigmoid: a few units of 32 bits
            want_y[s], by[s] = z * sg, 1.1 * ez + 8 * U32 * (z.abs() + 1) + u(dt) * (z * sg).abs() + tiny(dt)
            slope = sg * (1 + z * (1 - sg))
            dz = G * slope
            # z is kept in the type: its rounding moves the slope by at most 0.5 u |z|; dz is rounded to the type
            edz = G.abs() * (0.5 * (u(dt) * z.abs() + ez + tiny(dt)) + 16 * U32 * (z.abs() + 1)) + u(dt) * dz.abs() + tiny(dt)
            edz = edz * (1 + u(dt))
        else:
            want_y[s], by[s] = z, ez + u(dt) * z.abs() + tiny(dt)
            dz, edz = G, torch.zeros_like(G)
        want_x[s] = dz @ W
        bx[s] = edz @ W.abs() + 2 * (O + 1) * U32 * ((dz.abs() + edz) @ W.abs()) + u(dt) * (want_x[s].abs() + edz @ W.abs()) + tiny(dt)
        want_w[e] = dz.t() @ X
        bw[e] = edz.t() @ X.abs() + 2 * (n + 1) * U32 * ((dz.abs() + edz).t() @ X.abs()) + u(dt) * (want_w[e].abs() + edz.t() @ X.abs()) + tiny(dt)
        want_b[e] = dz.sum(0)
        bb[e] = edz.sum(0) + 2 * (n + 1) * U32 * (dz.abs() + edz).sum(0) + u(dt) * (want_b[e].abs() + edz.sum(0)) + tiny(dt)
    close(y, want_y, by, 'y')
    close(got[0], want_x, bx, 'd xs')
    close(got[1], want_w, bw, 'd weight')
    if with_bias:
        close(got[2], want_b, bb, 'd bias')


LINEAR = [([1], 0, 1, 1), ([0, 3, 0], 1, 8, 8), ([1, 1, 1, 1], 0, 64, 40), ([5, 0, 130], 3, 64, 128), ([127, 129, 1], 0, 72, 136), ([40, 17, 200], 5, 33, 65), ([300, 0, 0, 21], 0, 256, 264),
          ([128, 256], 128, 128, 256), ([64, 70], 2, 13, 300), ([2, 0, 1], 0, 520, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize('counts,tail,I,O', LINEAR)
@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('act,with_bias', [(None, False), (None, True), ('silu', True), ('silu', False)])
def test_expert_linear_with_gradients(device, counts, tail, I, O, dtype, act, with_bias):
    check_linear(device, counts, tail, I, O, DTYPES[dtype], act, with_bias, seed=I + O)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('counts,tail,I,O', [([900, 0, 1100, 37], 5, 1032, 776), ([13000, 7001], 9, 2056, 4104), ([9000, 1, 0, 3999], 0, 2050, 4100)])
def test_expert_linear_in_its_larger_tiles(device, counts, tail, I, O, dtype):
    """enough rows and columns for the 128 x 128 and 256 x 256 tiles, groups and matrices that end inside one, rows that are not whole 16-byte pieces"""
    check_linear(device, counts, tail, I, O, DTYPES[dtype], 'silu', True, where=device)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('counts,tail,I,O', [([15000, 10001], 5, 72, 4104), ([30, 0, 1, 128] * 7, 0, 2056, 2048)])
def test_expert_linear_with_results_larger_than_the_last_level_cache(device, counts, tail, I, O, dtype):
    """205 MB of rows, 236 MB of weight gradients: they are written past the cache"""
    check_linear(device, counts, tail, I, O, DTYPES[dtype], 'silu', False, where=device)


@pytest.mark.gpu
@pytest.mark.parametrize('layout', ['offset', 'columns'])
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_expert_linear_on_strided_rows(device, layout, dtype):
    check_linear(device, [70, 3, 150], 4, 64, 96, DTYPES[dtype], 'silu', True, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_expert_linear_of_rows_that_are_one_row(device, dtype):
    """inputs and gradients broadcast over the rows: the same bits as their copies"""
    dt = DTYPES[dtype]
    expert, xs, w, bias, gy = linear_case([70, 0, 90], 2, 64, 96, dt, 4)
    plan = ops.route(expert.to(device), 3)
    out = []
    for how in ('expanded', 'plain'):
        x, g = strided(xs, 'expanded', device), strided(gy, 'expanded', device)
        if how == 'plain':
            x, g = x.contiguous(), g.contiguous()
        x, wd, bd = x.requires_grad_(), w.to(device).requires_grad_(), bias.to(device).requires_grad_()
        y = ops.expert_linear(x, wd, plan, bd)
        out.append([y.detach()] + list(torch.autograd.grad(y, [x, wd, bd], g)))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_expert_linear_of_many_experts(device, dtype):
    """more experts than a wave has lanes, most of them empty; a long group that ends inside a tile"""
    counts = [(3 * e) % 5 if e % 7 else 0 for e in range(201)]
    counts[150] = 700
    check_linear(device, counts, 9, 48, 56, DTYPES[dtype], None, True)


@pytest.mark.gpu
@pytest.mark.parametrize('counts', [[3000], [700, 1, 0, 1025, 512, 513], [2048, 1024, 1023, 4097, 0, 5], [1024, 1025, 1024, 1]])
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_expert_linear_with_rows_cut_into_segments(device, counts, dtype):
    """experts longer than a segment of the weight gradient, at its border, and without rows beside them"""
    need = _ops.lib().ccsp_ops_linear_workspace(2, _ops.TYPES[str(DTYPES[dtype])[6:]], len(counts), sum(counts), 24, 40, 64, 40, 64, 24)
    assert need > 0
    check_linear(device, counts, 3, 24, 40, DTYPES[dtype], 'silu', True)
    check_linear(device, counts, 0, 23, 41, DTYPES[dtype], None, True)


def test_segments_of_cut_experts_have_slots_of_their_own():
    """the slot rule of the weight gradient's partial sums (csrc/ops/ops_linear.h seg_slot), restated: no two share one, all lie in the workspace"""
    rng = np.random.default_rng(0)
    for _ in range(2000):
        l = int(rng.integers(1, 6))
        counts = rng.integers(0, int(rng.integers(1, 4 << l)) + 1, size=int(rng.integers(1, 12)))
        off = np.concatenate([[0], np.cumsum(counts)])
        used = []
        for e, n in enumerate(counts):
            if n > 1 << l:
                used += [2 * ((int(off[e]) >> l) + i) + (i > 0) for i in range((int(n) + (1 << l) - 1) >> l)]
        assert len(set(used)) == len(used) and all(0 <= s < 2 * ((int(off[-1]) >> l) + 1) for s in used), (l, counts)


@pytest.mark.gpu
def test_expert_linear_gradient_against_differences(device):
    """32-bit gradients against central differences of the 64-bit formula in random directions: the oracle's gradient is not taken on trust"""
    counts, I, O = [5, 0, 9], 12, 10
    expert, xs, w, bias, gy = linear_case(counts, 0, I, O, torch.float32, 3)
    plan = ops.route(expert.to(device), 3)
    leaves = [t.to(device).requires_grad_() for t in (xs, w, bias)]
    grads = torch.autograd.grad(ops.expert_linear(leaves[0], leaves[1], plan, leaves[2], 'silu'), leaves, gy.to(device))

    def f(x, W, b):
        z = torch.cat([x[:5] @ W[0].t() + b[0], x[5:] @ W[2].t() + b[2]])
        return float((z * torch.sigmoid(z) * gy.double()).sum())
    at = [t.double() for t in (xs, w, bias)]
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, dn = list(at), list(at)
        up[i], dn[i] = at[i] + h * d, at[i] - h * d
        num = (f(*up) - f(*dn)) / (2 * h)
        got = float((grads[i].cpu().double() * d).sum())
        # the difference quotient: h^2 / 6 times a third derivative of a few hundred, and the cancellation 1e-16 |f| / h
        assert abs(got - num) <= 1e-4 * float((grads[i].cpu().double() * d).abs().sum()) + 1e-6, i


@pytest.mark.gpu
def test_a_frozen_weight_or_input_gets_no_gradient(device):
    expert, xs, w, bias, gy = linear_case([4, 6], 0, 16, 24, torch.float32, 5)
    plan = ops.route(expert.to(device), 2)
    full = [t.to(device).requires_grad_() for t in (xs, w, bias)]
    want = torch.autograd.grad(ops.expert_linear(full[0], full[1], plan, full[2], 'silu'), full, gy.to(device))
    for i in range(3):
        part = [t.to(device).requires_grad_(j == i) for j, t in enumerate((xs, w, bias))]
        got = torch.autograd.grad(ops.expert_linear(part[0], part[1], plan, part[2], 'silu'), part[i], gy.to(device))[0]
        assert torch.equal(got, want[i])


@pytest.mark.gpu
@pytest.mark.parametrize('counts,I,O', [([40, 0, 90], 200, 136), ([900, 0, 1100, 37], 1032, 776), ([13000, 7001], 2056, 4104), ([3000, 5000], 300, 200)])
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_the_bias_gradient_alone_has_the_bits_it_has_beside_the_weights(device, counts, I, O, dtype):
    """over every size of tile, cut into segments and not"""
    expert = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).to(device)
    plan = ops.route(expert, len(counts))
    g = torch.Generator(device=device).manual_seed(8)
    xs, w, bias, gy = [torch.randn(*s, generator=g, device=device).to(DTYPES[dtype]) for s in ((sum(counts), I), (len(counts), O, I), (len(counts), O), (sum(counts), O))]
    bias.requires_grad_()
    alone, = torch.autograd.grad(ops.expert_linear(xs, w, plan, bias), bias, gy)
    w.requires_grad_()
    beside = torch.autograd.grad(ops.expert_linear(xs, w, plan, bias), (w, bias), gy)[1]
    assert torch.equal(alone, beside)


@pytest.mark.gpu
def test_a_gradient_of_a_gradient_is_refused(device):
    expert, leaves, E = layer_inputs(device, torch.float32)
    plan = ops.route(expert, E)
    x = leaves[0].requires_grad_()
    w = leaves[1].requires_grad_()
    rows = ops.sort_rows(x, plan)
    for y in (rows, ops.expert_linear(rows.detach().requires_grad_(), w, plan), ops.combine_rows(rows, plan, leaves[4].requires_grad_())):
        leaf = x if y is rows else w if y.shape[1] == w.shape[1] else leaves[4]
        g, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match='differentiable once'):
            g.sum().backward()


# ---- the global norm -----------------------------------------------------------------------------------------------------

def norm_oracle(ts, max_norm):
    n = math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))
    return n, min(1.0, max_norm / (n + 1e-6))


def check_clip(got_norm, got, ts, max_norm):
    n, c = norm_oracle(ts, max_norm)
    assert abs(float(got_norm) - n) <= 2 * U32 * n               # one rounding to 32 bits, and 64-bit sums
    for i, (a, t) in enumerate(zip(got, ts)):
        want = t.double() * c
        close(a, want, (u(t.dtype) + 4 * U32) * want.abs() + tiny(t.dtype), 'tensor %d' % i)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES) + ['mixed'])
@pytest.mark.parametrize('max_norm', [0.0, 0.7, 1e9, math.inf])
def test_clip_global_norm(device, dtype, max_norm):
    g = torch.Generator().manual_seed(5)
    sizes = [(1,), (0,), (3, 5), (16384,), (16385,), (0, 7), (7,), (100003,), (2, 3, 4), (40000,)]
    dts = list(DTYPES.values())
    ts = [(torch.randn(s, generator=g) * 10.0 ** (i % 3 - 1)).to(dts[i % 3] if dtype == 'mixed' else DTYPES[dtype]) for i, s in enumerate(sizes)]
    dev = [t.to(device) for t in ts]
    assert abs(float(ops.global_norm(dev)) - norm_oracle(ts, 1.0)[0]) <= 2 * U32 * norm_oracle(ts, 1.0)[0]
    out = [torch.full_like(t, 7.0) for t in dev]
    check_clip(ops.clip_global_norm(dev, max_norm, out=out), out, ts, max_norm)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, ts))
    check_clip(ops.clip_global_norm(dev, max_norm), dev, ts, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_clip_of_many_unaligned_tensors(device, dtype):
    """more tensors than a launch's table holds, each starting anywhere in one buffer; the gaps between them stay"""
    dt = DTYPES[dtype]
    g = torch.Generator().manual_seed(2)
    sizes = [int(v) for v in torch.randint(0, 90, (450,), generator=g)]
    host = torch.randn(sum(sizes) + len(sizes), generator=g).to(dt)
    buf, out = host.to(device), torch.full((sum(sizes) + 2 * len(sizes),), 7.0, dtype=dt, device=device)
    src, dst, cpu, at, ot = [], [], [], 0, 0
    for i, n in enumerate(sizes):
        src.append(buf[at:at + n]); cpu.append(host[at:at + n]); dst.append(out[ot:ot + n])
        at += n + i % 2
        ot += n + i % 3
    check_clip(ops.clip_global_norm(src, 2.5, out=dst), dst, cpu, 2.5)
    assert torch.equal(buf.cpu(), host)
    keep = torch.ones(out.numel(), dtype=torch.bool)
    ot = 0
    for i, n in enumerate(sizes):
        keep[ot:ot + n] = False
        ot += n + i % 3
    assert bool((out.cpu()[keep] == 7.0).all())


@pytest.mark.gpu
def test_norm_range_and_values_that_are_not_finite(device):
    big = torch.full((1000,), 1e30, device=device)
    assert abs(float(ops.global_norm([big])) / (1e30 * math.sqrt(1000.0)) - 1) < 1e-6
    small = torch.full((1000,), 1e-30, device=device)
    assert abs(float(ops.global_norm([small])) / (1e-30 * math.sqrt(1000.0)) - 1) < 1e-6
    zero = torch.zeros(5, device=device)
    assert float(ops.clip_global_norm([zero], 1.0)) == 0.0 and float(zero.abs().max()) == 0.0
    a = torch.tensor([1.0, math.inf], device=device)
    assert math.isinf(float(ops.clip_global_norm([a], 1.0)))
    assert float(a[0]) == 0.0 and math.isnan(float(a[1]))
    b = torch.tensor([1.0, math.nan], device=device)
    assert math.isnan(float(ops.clip_global_norm([b], 1.0))) and bool(torch.isnan(b).all())


@pytest.mark.gpu
def test_clip_grad_norm_of_parameters(device):
    g = torch.Generator().manual_seed(9)
    ps = [torch.nn.Parameter(torch.zeros(6, 10, device=device)) for _ in range(3)] + [torch.nn.Parameter(torch.zeros(2, device=device))]
    host = [torch.randn(6, 10, generator=g) for _ in range(3)]
    for p, h in zip(ps, host):
        p.grad = h.to(device)
    ps[1].grad = host[1].to(device).t().contiguous().t()         # a gradient with another memory order
    v = ps[0].grad._version
    norm = ops.clip_grad_norm_(iter(ps + [ps[0]]), 0.5)          # without a gradient: skipped; twice: once
    check_clip(norm, [p.grad for p in ps[:3]], host, 0.5)
    assert ps[0].grad._version > v and ps[3].grad is None
    with pytest.raises(ValueError, match='twice'):
        ops.clip_global_norm([ps[0].grad, ps[0].grad], 1.0)
    a, b = torch.ones(8, device=device), torch.ones(8, device=device)
    for grads, out in (([a[:5], a[4:]], None), ([a, b], [b, a]), ([a], [a.clone()[1:].new_zeros(8)]), ([a[:4], b[:4]], [a[2:6], b[:4]]), ([a[:4], a[4:]], [b[4:], b[:4]])):
        if out is None or out[0].data_ptr() in (b.data_ptr(), a[2:].data_ptr()):
            with pytest.raises(ValueError, match='lies on another'):
                ops.clip_global_norm(grads, 1.0, out=out)
        else:
            ops.clip_global_norm(grads, 1.0, out=out)
    with pytest.raises(ValueError, match='negative'):
        ops.clip_global_norm([ps[0].grad], -1.0)
    with pytest.raises(ValueError, match='negative'):
        ops.clip_global_norm([ps[0].grad], math.nan)
    with pytest.raises(ValueError, match='same type and shape'):
        ops.clip_global_norm([ps[0].grad], 1.0, out=[ps[0].grad[:2]])
    with pytest.raises(TypeError, match='float64'):
        ops.global_norm([ps[0].grad.double()])
    with pytest.raises(TypeError, match='sparse'):
        ops.global_norm([ps[0].grad.to_sparse()])


# ---- together, as they are used ------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_clip_of_gradients_between_each_others_elements(device):
    """strided views without a common element are clipped in place, whatever lies between their elements"""
    x = torch.randn(40, 6, generator=torch.Generator().manual_seed(3))
    y = x.to(device)
    host = [x[:, ::2].clone(), x[:, 1].clone(), x[:, 3::2].clone()]
    got = [y[:, ::2], y[:, 1], y[:, 3::2]]
    check_clip(ops.clip_global_norm(got, 0.5), got, host, 0.5)
    with pytest.raises(ValueError, match='twice'):
        ops.clip_global_norm([got[0], y[:, ::2]], 0.5)


def layer(x, plan, w1, b1, w2, weights):
    h = ops.expert_linear(ops.sort_rows(x, plan), w1, plan, b1, 'silu')
    return ops.combine_rows(ops.expert_linear(h, w2, plan), plan, weights)


def layer_inputs(device, dt, N=50, k=2, E=6, D=32, H=48, seed=0):
    g = torch.Generator().manual_seed(seed)
    expert = ids(N * k, E, seed, 0.1).reshape(N, k).to(device)
    mk = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(device, dt)     # noqa: E731
    return expert, [mk(N, D), mk(E, H, D), mk(E, H), mk(E, D, H), torch.rand(N, k, generator=g).to(device)], E


@pytest.mark.gpu
def test_a_routed_layer_trains_like_its_plain_form(device):
    """route, sort, two products, combine, backward, clip against torch's 64-bit autograd of the same layer.  Each of the six operators in a row adds at most some
    (width + 2) units of 32 bits of its terms' magnitude: 1e-4 of the largest entry leaves an order of magnitude"""
    expert, leaves, E = layer_inputs(device, torch.float32)
    for t in leaves:
        t.requires_grad_()
    plan = ops.route(expert, E)
    y = layer(leaves[0], plan, *leaves[1:])
    y.square().sum().backward()
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    x, w1, b1, w2, wt = ref
    want = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64)
    rows = []
    for n in range(expert.shape[0]):
        acc = torch.zeros(w2.shape[1], dtype=torch.float64)
        for j in range(expert.shape[1]):
            e = int(expert[n, j])
            if 0 <= e < E:
                acc = acc + wt[n, j] * (w2[e] @ torch.nn.functional.silu(w1[e] @ x[n] + b1[e]))
        rows.append(acc)
    want = torch.stack(rows)
    want.square().sum().backward()
    assert float((y.detach().cpu().double() - want.detach()).abs().max()) <= 1e-4 * float(want.detach().abs().max())
    for t, r in zip(leaves, ref):
        assert float((t.grad.cpu().double() - r.grad).abs().max()) <= 1e-4 * float(r.grad.abs().max())
    norm = ops.clip_grad_norm_(leaves, 0.1)
    want_norm = math.sqrt(sum(float((r.grad ** 2).sum()) for r in ref))
    assert abs(float(norm) - want_norm) <= 1e-4 * want_norm
    assert abs(float(ops.global_norm([t.grad for t in leaves])) - 0.1) <= 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_the_same_bits_every_time_and_on_any_stream(device, dtype):
    expert, leaves, E = layer_inputs(device, DTYPES[dtype], N=700, k=4, E=13, D=64, H=96)

    def once():
        ls = [t.detach().clone().requires_grad_() for t in leaves]
        plan = ops.route(expert, E)
        y = layer(ls[0], plan, *ls[1:])
        return [y.detach()] + list(torch.autograd.grad(y, ls, torch.ones_like(y)))
    want = once()
    torch.cuda.synchronize()
    results = {}

    def worker(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            results[i] = [once() for _ in range(3)]
        s.synchronize()
    threads = [threading.Thread(target=worker, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        for got in results[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_captured_and_replayed(device):
    """forward, backward and clipping in one graph; every replay, on new inputs and with eager work between, equals the eager result"""
    expert, leaves, E = layer_inputs(device, torch.float32, N=300, k=3, E=7, D=40, H=56)
    static = [t.clone().requires_grad_() for t in leaves]
    ids_in = expert.clone()

    def step():
        plan = ops.route(ids_in, E)
        y = layer(static[0], plan, *static[1:])
        grads = torch.autograd.grad(y, static, torch.ones_like(y))
        out = [torch.empty_like(t) for t in grads]
        norm = ops.clip_global_norm(grads, 0.25, out=out)
        return [plan.offsets, y.detach(), norm] + out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        ex, new, _ = layer_inputs(device, torch.float32, N=300, k=3, E=7, D=40, H=56, seed=seed + 10)
        with torch.no_grad():
            ids_in.copy_(ex)
            for s, t in zip(static, new):
                s.copy_(t)
        graph.replay()
        got = [t.detach().clone() for t in captured]
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


@pytest.mark.gpu
def test_two_graphs_do_not_share_workspaces(device):
    """two captured routes replayed on two streams at once: each has its own memory"""
    graphs = []
    for seed in range(2):
        expert = ids(30000, 20, seed, 0.1).to(device)
        ops.route(expert, 20)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan = ops.route(expert, 20)
        graphs.append((g, plan, ops.route(expert, 20), torch.cuda.Stream(), expert))    # (a graph reads its inputs where they were: they live on)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, _, _, s, _ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, plan, want, _, _ in graphs:
            assert torch.equal(plan.rows, want.rows) and torch.equal(plan.assign, want.assign) and torch.equal(plan.offsets, want.offsets)


@pytest.mark.gpu
def test_the_training_command_on_operators_equals_its_plain_form(device, monkeypatch):
    """tools/train_gpu.py: loss and gradients of the denoiser on the operators against its loop over the types, both in 32 bits on the GPU.  A gradient entry is a sum
    of at most some thousand rounded terms down a chain of seven layers: 2e-4 of the largest entry of its tensor is an order above the 32-bit spread"""
    monkeypatch.setenv('TRAIN_DEVICE', 'cuda:0')
    monkeypatch.setenv('TRAIN_HIDDEN', '64')
    monkeypatch.setenv('TRAIN_OPERATORS', '1')
    monkeypatch.syspath_prepend(os.path.join(ROOT, 'tools'))
    monkeypatch.delitem(sys.modules, 'train_gpu', raising=False)
    import train_gpu as tg
    assert tg.USE_OPERATORS
    rng = np.random.default_rng(4)
    worlds_ = [worlds.sample_qualitative_world(rng, int(rng.integers(2, 9))) for _ in range(24)]
    batch = worlds.collate([worlds.encode_qualitative(w['nodes'], w['constraints']) for w in worlds_])
    torch.manual_seed(1)
    net = tg.Denoiser().to(device)
    sa, sb = tg.schedule_tables()
    b = tg.to_dev(batch)
    noise, t = torch.randn(batch.x.shape[0], 4, device=device), torch.tensor([300], device=device)
    results = []
    for form in ('operators', 'operators', 'plain'):
        bb = dict(b, nodes=None) if form == 'plain' else b
        net.zero_grad(set_to_none=True)
        loss = tg.loss_on(net, bb, t, noise, sa, sb)
        loss.backward()
        results.append((loss.detach(), {n: None if p.grad is None else p.grad.clone() for n, p in net.named_parameters()}))
    (l0, g0), (l1, g1), (l2, g2) = results
    assert abs(float(l0) - float(l2)) <= 1e-5 * float(l2)
    for name in g0:
        # a type without edges: no gradient from the loop, zeros from its group
        want = torch.zeros_like(g0[name]) if g2[name] is None else g2[name]
        assert float((g0[name] - want).abs().max()) <= 2e-4 * max(float(want.abs().max()), 1e-6), name
    norm = ops.clip_grad_norm_(net.parameters(), 0.01)
    total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in g2.values() if g is not None))
    assert abs(float(norm) - total) <= 1e-3 * total
    monkeypatch.delitem(sys.modules, 'train_gpu', raising=False)


# ---- values past a 16-bit type's range -----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize('O', [24, 25])
@pytest.mark.parametrize('counts', [[5, 0, 9], [9000, 1, 0, 3999]])
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_silu_gradient_of_pre_activations_past_the_types_range(device, counts, O, dtype):
    """Pre-activations that are finite in 32 bits and infinite in the rows' type, of both signs: the slope there is 0 or 1.  All values are powers of two or short sums of
    them.  Columns 0 and 1 make the large pre-activation, which lies 0.1 % and more past the type's largest value: what the sigmoid leaves of it is 0 on the
    negative side, 1 on the other, in 32 and 64 bits alike.  The other columns are zero, so every product below is one term and exact up to its own rounding"""
    dt, I, E = DTYPES[dtype], 16, len(counts)
    g = torch.Generator().manual_seed(2)
    R = sum(counts)
    a, b = (1024.0, 72.0) if dt == torch.float16 else (2.0 ** 64, 2.0 ** 63 * 1.9921875)
    x = torch.zeros(R, I, dtype=dt)
    x[:, 0], x[:, 1], x[:, 2] = a, a, torch.randint(1, 4, (R,), generator=g).to(dt)
    w = torch.zeros(E, O, I, dtype=dt)
    w[:, 3, 0], w[:, 3, 1] = -b, -b * 2.0 ** -8                   # 2^127 * 1.9999 is past bfloat16, inside float32; -74016 past float16
    w[:, 5] = -w[:, 3]
    w[:, 7, 2] = 1.0                                              # an ordinary one beside them
    gy = (torch.randint(0, 2, (R, O), generator=g) * 2 - 1).to(dt) * 2.0 ** -6
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts))
    plan = ops.route(expert.to(device), E)
    xd, wd, bd = x.to(device).requires_grad_(), w.to(device).requires_grad_(), torch.zeros(E, O, dtype=dt, device=device, requires_grad=True)
    y = ops.expert_linear(xd, wd, plan, bd, 'silu')
    d_x, d_w, d_b = torch.autograd.grad(y, (xd, wd, bd), gy.to(device))
    z = torch.stack([x[p].double() @ w[e].double().t() for p, e in enumerate(expert.tolist()[:4])])
    assert (dt == torch.float32) == bool(torch.isfinite(z.to(dt)).all()) and bool(torch.isfinite(z.float()).all())
    Z = torch.zeros(R, O, dtype=torch.float64)
    Z[:, 3], Z[:, 5], Z[:, 7] = z[0, 3], z[0, 5], x[:, 2].double()
    s = torch.sigmoid(Z)
    got = y.detach().cpu()
    assert float(got[:, 3].abs().max()) == 0.0 and torch.equal(got[:, 5].double(), Z[:, 5].to(dt).double())
    slope = s * (1 + Z * (1 - s))
    assert float(slope[:, 3].abs().max()) == 0.0 and float((slope[:, 5] - 1).abs().max()) == 0.0
    dz = gy.double() * slope
    edz = (u(dt) + 64 * U32) * dz.abs() + tiny(dt)                # (z of column 7 is a whole number, exact; the sigmoid's few units of 32 bits, times 1 + |z|)
    bound = lambda want, e: e + (u(dt) + 2 * U32) * want.abs() + tiny(dt)      # noqa: E731
    We = w.double()[0]                                            # (every expert has the same)
    want = dz @ We
    close(d_x, want, bound(want, edz @ We.abs() + 2 * (O + 1) * U32 * (dz.abs() @ We.abs())), 'd xs')
    lo = 0
    for e, n in enumerate(counts):
        D, ED, X = dz[lo:lo + n], edz[lo:lo + n], x[lo:lo + n].double()
        lo += n
        want = D.t() @ X
        close(d_w[e], want, bound(want, ED.t() @ X.abs() + 2 * (n + 1) * U32 * (D.abs().t() @ X.abs())), 'd weight')
        want = D.sum(0)
        close(d_b[e], want, bound(want, ED.sum(0) + 2 * (n + 1) * U32 * D.abs().sum(0)), 'd bias')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_silu_of_infinite_pre_activations_is_the_formulas(device, dtype):
    """inputs that are infinite themselves: z sigmoid(z) and its slope as the formula gives them, inf or NaN, and nothing of it in other rows"""
    dt = DTYPES[dtype]
    x = torch.zeros(3, 8, dtype=dt, device=device)
    x[0, 0], x[1, 0], x[2, 1] = math.inf, -math.inf, 1.0
    w = torch.zeros(1, 8, 8, dtype=dt, device=device)
    w[0, :, 0] = 1.0
    plan = ops.route(torch.zeros(3, dtype=torch.int64, device=device), 1)
    x.requires_grad_()
    y = ops.expert_linear(x, w, plan, None, 'silu')
    d_x, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert bool((y[0] == math.inf).all()) and bool(y[1].isnan().all()) and bool((y[2] == 0).all())
    assert bool(d_x[:2, 0].isnan().all()) and bool((d_x[2, 0] == 4.0).all())      # eight slopes of a half


# ---- addresses that are not there ----------------------------------------------------------------------------------------

def test_the_weights_gradient_without_rows_to_read_is_refused():
    L = _ops.lib()
    ok = 64                                                       # (never read)
    assert L.ccsp_ops_rows_back(1, 4, 4, ok, ok, ok, None, None, 1, ok, 4, None, 4, ok, ok, None) != 0
    assert 'null' in L.ccsp_ops_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize('width', [5, 400])
@pytest.mark.parametrize('dtype', list(DTYPES))
def test_rows_of_no_tokens_are_zeros(device, dtype, width):
    """a source without an address has no rows: zeros, and no access, also where a plan says that there are some"""
    dt, code, L = DTYPES[dtype], _ops.TYPES[str(DTYPES[dtype])[6:]], _ops.lib()
    expert = torch.tensor([[1, 0], [0, -1], [2, 2]], device=device)
    plan = ops.route(expert, 3)
    place = torch.empty(6, dtype=torch.int32, device=device)
    rows, assign = plan.rows.cpu().tolist(), plan.assign.cpu().tolist()
    host = [0] * 6
    for p, a in enumerate(assign):
        host[a if a >= 0 else ~a] = p if a >= 0 else ~p
    assert [p if p >= 0 else -1 for p in host] == rows
    place.copy_(torch.tensor(host))
    stream = torch.cuda.current_stream().cuda_stream
    out = torch.full((6, width), 7.0, dtype=dt, device=device)
    parts = (plan.row_token.data_ptr(), plan.assign.data_ptr(), place.data_ptr(), None)
    assert L.ccsp_ops_rows_gather(code, 6, width, None, width, *parts, out.data_ptr(), stream) == 0
    assert float(out.abs().max()) == 0.0
    ys, w = torch.ones(6, width, dtype=dt, device=device), torch.ones(6, device=device)
    out.fill_(7.0)
    d_w = torch.full((6,), 7.0, device=device)
    assert L.ccsp_ops_rows_back(code, 6, width, *parts, w.data_ptr(), 0, None, width, ys.data_ptr(), width, out.data_ptr(), d_w.data_ptr(), stream) == 0
    assert float(out.abs().max()) == 0.0 and float(d_w.abs().max()) == 0.0


# ---- calls that would lose something without a word ----------------------------------------------------------------------

def test_the_norm_of_dual_numbers_is_refused():
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(3), torch.ones(3))
        for call in (lambda: ops.global_norm([dual]), lambda: ops.clip_global_norm([dual], 1.0), lambda: ops.global_norm([dual[:2]])):
            with pytest.raises(CcspError, match='forward-mode'):
                call()


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused(device):
    import torch.autograd.forward_ad as forward_ad
    expert, (x, w, b, w2, weights), E = layer_inputs(device, torch.float32)
    plan = ops.route(expert, E)
    xs = ops.sort_rows(x, plan)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))      # noqa: E731
        for call in (lambda: ops.sort_rows(dual(x), plan), lambda: ops.combine_rows(dual(xs), plan, weights), lambda: ops.combine_rows(xs, plan, dual(weights)),
                     lambda: ops.expert_linear(dual(xs), w, plan, b), lambda: ops.expert_linear(xs, dual(w), plan, b), lambda: ops.expert_linear(xs, w, plan, dual(b)),
                     lambda: ops.sort_rows(dual(x.clone().requires_grad_()), plan), lambda: ops.sort_rows(dual(x)[:, 1:], plan), lambda: ops.clip_global_norm([x, dual(b)], 1.0),
                     lambda: ops.clip_global_norm([x], 1.0, out=[dual(x)])):
            with pytest.raises(CcspError, match='forward-mode'):
                call()
        assert torch.equal(ops.sort_rows(x, plan), xs)            # (a tensor without a tangent is what it was)


def tracers():
    from torch.fx.experimental.proxy_tensor import make_fx
    return [lambda f, t: torch.jit.trace(f, t, check_trace=False), lambda f, t: make_fx(f)(t), lambda f, t: make_fx(f, tracing_mode='real', pre_dispatch=True)(t)]


@pytest.mark.parametrize('which', range(3))
def test_a_trace_of_an_operator_is_refused(which):
    with pytest.raises(CcspError, match='recorded'):
        tracers()[which](lambda t: ops.global_norm([t]), torch.ones(3))
    with pytest.raises(CcspError, match='no CPU fallback'):      # (and it is over with the trace)
        ops.global_norm([torch.ones(3)])


@pytest.mark.gpu
@pytest.mark.parametrize('which', range(3))
def test_traces_of_all_operators_are_refused(device, which):
    expert, (x, w, b, w2, weights), E = layer_inputs(device, torch.float32)
    plan = ops.route(expert, E)
    xs = ops.sort_rows(x, plan)
    for f, t in ((lambda t: ops.route(t, E).offsets, expert), (lambda t: ops.sort_rows(t, plan), x), (lambda t: ops.combine_rows(xs, plan, t), weights), (lambda t: ops.expert_linear(xs, t, plan), w),
                 (lambda t: ops.clip_global_norm([t], 1.0), x.clone())):
        with pytest.raises(CcspError, match='recorded'):
            tracers()[which](f, t)
    assert torch.equal(ops.sort_rows(x, plan), xs)


@pytest.mark.gpu
def test_gradients_of_a_trace_or_with_a_tangent_are_refused(device):
    """the forward before, the backward pass inside"""
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    expert, leaves, E = layer_inputs(device, torch.float32)
    x, w, b, w2, weights = [t.requires_grad_() for t in leaves]
    plan = ops.route(expert, E)
    xs = ops.sort_rows(x, plan)
    for y, leaf in ((xs, x), (ops.expert_linear(xs.detach(), w, plan, b), w), (ops.combine_rows(xs.detach(), plan, weights), weights)):
        g = torch.ones_like(y)
        want, = torch.autograd.grad(y, leaf, g, retain_graph=True)
        with pytest.raises(RuntimeError, match='recorded'):
            make_fx(lambda t: torch.autograd.grad(y, leaf, t, retain_graph=True)[0])(g)      # noqa: B023
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(g, torch.ones_like(g)), retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, leaf, g)[0], want)


class Wrapper(torch.Tensor):
    """a tensor without memory that says it is on the GPU"""
    @staticmethod
    def __new__(cls, like, device='cuda:0'):
        return torch.Tensor._make_wrapper_subclass(cls, like.shape, dtype=like.dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


def test_tensors_that_wrap_others_are_refused():
    for call in (lambda t: ops.global_norm([t]), lambda t: ops.clip_global_norm([t], 1.0), lambda t: ops.route(t, 3)):
        with pytest.raises(TypeError, match='wraps others'):
            call(Wrapper(torch.ones(4, dtype=torch.float32)))
    with pytest.raises(TypeError, match='wraps others'):
        torch.func.vmap(lambda t: ops.global_norm([t]))(torch.ones(2, 3))
    with pytest.raises(TypeError, match='sparse'):
        ops.global_norm([torch.ones(3).to_sparse()])


@pytest.mark.gpu
def test_every_operand_that_wraps_others_is_refused(device):
    """(the checks are the host's: nothing is launched)"""
    expert, (x, w, b, w2, weights), E = layer_inputs(device, torch.float32)
    plan = ops.route(expert, E)
    xs = ops.sort_rows(x, plan)
    for call in (lambda: ops.route(Wrapper(expert), E), lambda: ops.route(expert, E, Wrapper(expert), 50), lambda: ops.sort_rows(Wrapper(x), plan), lambda: ops.combine_rows(Wrapper(xs), plan),
                 lambda: ops.combine_rows(xs, plan, Wrapper(weights)), lambda: ops.expert_linear(Wrapper(xs), w, plan, b), lambda: ops.expert_linear(xs, Wrapper(w), plan, b),
                 lambda: ops.expert_linear(xs, w, plan, Wrapper(b)), lambda: ops.clip_global_norm([x, Wrapper(x)], 1.0), lambda: ops.clip_global_norm([x], 1.0, out=[Wrapper(x)]),
                 lambda: torch.func.vmap(lambda t: ops.sort_rows(t, plan))(x[None]),
                 lambda: torch.func.grad(lambda t: ops.sort_rows(t, plan).sum())(x), lambda: ops.sort_rows(x.to_sparse(), plan)):
        with pytest.raises(TypeError, match='wraps others|sparse'):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize('D', [1, 24])
def test_negative_views_and_zeros_without_memory(device, D):
    """what torch keeps as a flag on a tensor (the imaginary part of a conjugate; gradients that are zero): the operators see the values"""
    expert = ids(40, 5, 1, 0.2).reshape(20, 2).to(device)
    neg, zero = torch._neg_view, torch._efficientzerotensor((20, D), device=device)
    g = torch.Generator(device=device).manual_seed(0)
    x, ys, weights = [torch.randn(*s, generator=g, device=device) for s in ((20, D), (40, D), (20, 2))]
    w, b = torch.randn(5, 3, D, generator=g, device=device), torch.randn(5, 3, generator=g, device=device)
    assert x.is_contiguous() and neg(x).is_neg() and zero._is_zerotensor()
    plan = ops.route(expert, 5)
    assert torch.equal(ops.route(neg(-expert), 5).rows, plan.rows)
    assert torch.equal(ops.route(expert, 5, neg(-expert), 20).row_token, ops.route(expert, 5, expert, 20).row_token)
    assert torch.equal(ops.sort_rows(neg(x), plan), ops.sort_rows(-x, plan))
    assert float(ops.sort_rows(zero, plan).abs().max()) == 0.0
    assert torch.equal(ops.combine_rows(neg(ys), plan, neg(weights)), ops.combine_rows(-ys, plan, -weights))
    assert torch.equal(ops.expert_linear(neg(ys), neg(w), plan, neg(b)), ops.expert_linear(-ys, -w, plan, -b))
    leaves = [t.clone().requires_grad_() for t in (x, ys, weights, w, b)]
    outs = [ops.sort_rows(leaves[0], plan), ops.combine_rows(leaves[1], plan, leaves[2]), ops.combine_rows(leaves[1], plan), ops.expert_linear(leaves[1], leaves[3], plan, leaves[4], 'silu')]
    for y, at in zip(outs, ([0], [1, 2], [1], [1, 3, 4])):
        gy = torch.randn(y.shape, generator=g, device=device)
        for lazy, plain in ((neg(gy), -gy), (torch._efficientzerotensor(y.shape, device=device), torch.zeros_like(gy))):
            got, want = [torch.autograd.grad(y, [leaves[i] for i in at], t, retain_graph=True) for t in (lazy, plain)]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    a, out = torch.ones(4, D, device=device), [torch.empty(4, D, device=device), torch.empty(20, D, device=device)]
    norm = ops.clip_global_norm([neg(a), zero], 0.5, out=out)
    assert abs(float(norm) - math.sqrt(4 * D)) < 1e-5 and float(out[1].abs().max()) == 0.0
    assert float((out[0] + 0.5 / math.sqrt(4 * D)).abs().max()) < 1e-6 and float((a - 1).abs().max()) == 0.0
    assert abs(float(ops.global_norm([zero, neg(a)])) - math.sqrt(4 * D)) < 1e-5
    ops.clip_global_norm([neg(a)], 0.5)
    assert float((a - 0.5 / math.sqrt(4 * D)).abs().max()) < 1e-6
    with pytest.raises(ValueError, match='without memory'):
        ops.clip_global_norm([a, zero], 0.1)
    with pytest.raises(ValueError, match='contiguous'):
        ops.clip_global_norm([a], 0.1, out=[neg(a.clone())])
    assert float((a - 0.5 / math.sqrt(4 * D)).abs().max()) < 1e-6      # (refused before anything is written)


@pytest.mark.gpu
def test_expanded_gradients_are_refused_in_place_before_anything_is_scaled(device):
    a, e = torch.ones(4, device=device), torch.ones(1, device=device).expand(5)
    for grads in ([a, e], [e, a], [a, torch.ones(2, 1, device=device).expand(2, 3)]):
        with pytest.raises(ValueError, match='share memory'):
            ops.clip_global_norm(grads, 0.5)
    p = torch.nn.Parameter(torch.zeros(5, device=device))
    p.grad = e
    with pytest.raises(ValueError, match='share memory'):
        ops.clip_grad_norm_([p], 0.5)
    assert float((a - 1).abs().max()) == 0.0 and float(e[0]) == 1.0
    none = torch.ones(1, device=device).expand(0)
    out = [torch.empty(4, device=device), torch.empty(5, device=device), torch.empty(0, device=device)]
    assert float(ops.clip_global_norm([a, e, none], 1.5, out=out)) == 3.0 == float(ops.global_norm([a, e]))      # (every element counts)
    assert float((out[0] - 0.5).abs().max()) < 1e-6 and float((out[1] - 0.5).abs().max()) < 1e-6
    assert float(ops.clip_global_norm([a, none], 1.0)) == 2.0 and float((a - 0.5).abs().max()) < 1e-6


# ---- the training command ------------------------------------------------------------------------------------------------

def check_absent_types(monkeypatch, dev, operators_on):
    monkeypatch.setenv('TRAIN_DEVICE', dev)
    monkeypatch.setenv('TRAIN_HIDDEN', '64')
    monkeypatch.setenv('TRAIN_OPERATORS', operators_on)
    monkeypatch.syspath_prepend(os.path.join(ROOT, 'tools'))
    monkeypatch.delitem(sys.modules, 'train_gpu', raising=False)
    import train_gpu as tg
    assert tg.USE_OPERATORS == (operators_on == '1')
    rng = np.random.default_rng(4)
    ws = [worlds.sample_qualitative_world(rng, int(rng.integers(2, 9))) for _ in range(24)]
    batch = worlds.collate([worlds.encode_qualitative(w['nodes'], w['constraints']) for w in ws])
    kinds = np.asarray(batch.edge_attr).reshape(-1).astype(int)
    gone = int(np.bincount(kinds[kinds >= 0]).argmax())           # a type that the first batch has
    torch.manual_seed(1)
    net = tg.Denoiser().to(dev)
    opt = torch.optim.Adam(net.parameters(), lr=5e-4)
    sa, sb = tg.schedule_tables()
    noise, t = torch.randn(batch.x.shape[0], 4, device=dev), torch.tensor([300], device=dev)
    tg.train_step(net, opt, tg.to_dev(batch), t, noise, sa, sb)
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    moment = opt.state[net.mlps[gone][0].weight]['exp_avg'].clone()
    assert float(moment.abs().max()) > 0.0
    keep = kinds != gone
    batch.edge_attr, batch.edge_index = batch.edge_attr[keep], batch.edge_index[:, keep]
    b = tg.to_dev(batch)
    assert gone in b['absent']
    assert bool(torch.isfinite(tg.train_step(net, opt, b, t, noise, sa, sb)))
    for i, mlp in enumerate(net.mlps):
        for n, p in mlp.named_parameters():
            assert torch.equal(p.detach(), before['mlps.%d.%s' % (i, n)]) == (i in b['absent']), (i, n)
    assert torch.equal(opt.state[net.mlps[gone][0].weight]['exp_avg'], moment)
    monkeypatch.delitem(sys.modules, 'train_gpu', raising=False)


def test_a_type_without_edges_is_not_trained(monkeypatch):
    """its weights and moments stay as they are, as where its MLP is not called at all"""
    check_absent_types(monkeypatch, 'cpu', '0')


@pytest.mark.gpu
@pytest.mark.parametrize('operators_on', ['0', '1'])
def test_a_type_without_edges_is_not_trained_on_the_gpu(device, monkeypatch, operators_on):
    check_absent_types(monkeypatch, 'cuda:0', operators_on)

# ---- every tile of the products ------------------------------------------------------------------------------------------

def most_tiles(R, E, l):
    return (R >> l) + min(R, E + 1)


def prod_tile(weight, R, E, M, N):
    """the rule of csrc/ops/ops_linear.h prod_tile for 16 bits, restated"""
    tiles = lambda l: (E * -(-M >> l) if weight else most_tiles(R, E, l)) * -(-N >> l)      # noqa: E731
    big = tiles(8)
    if (big >= 256 and R >= 1024 * E) if weight else (big >= 1024 or (big >= 512 and R >= 1024 * E)):
        return 256
    return 128 if tiles(7) >= 512 else 64


def seg_log2(R, E, M, N):
    """the rule of seg_log2_for for 16 bits, restated; 31: uncut"""
    tile = prod_tile(True, R, E, M, N)
    tiles = -(-M // tile) * -(-N // tile)
    if tile == 256 or tiles >= 128:
        return 31
    l = 10
    while l < 30 and (2 << l) <= R * tiles // 1024:
        l += 1
    return 31 if 1 << l >= R else l


# counts, tail, inputs, outputs, tiles of the forward, the input gradient and the weight gradient, the weight gradient's segment
TILES = [([3000, 1024, 0, 1025, 951], 3, 1240, 1288, 128, 128, 128, 10),             # an expert longer than a segment, at its border, without rows
         ([3000, 1024, 0, 1025, 951], 3, 1237, 1285, 128, 128, 128, 10),             # results without whole pieces
         ([900, 0, 3, 1, 50], 0, 1240, 1288, 64, 64, 128, 31),                       # few rows: uncut
         ([4000, 1, 0, 3000], 5, 1400, 1416, 128, 128, 128, 31),                     # enough tiles: uncut
         ([4000, 1, 0, 3000], 5, 1401, 1419, 128, 128, 128, 31),
         ([9000, 1, 0, 3999], 2, 264, 4099, 256, 64, 64, 31),                        # 256 x 256 without whole pieces, forward
         ([9000, 1, 0, 3999], 2, 4099, 264, 64, 256, 64, 31),                        # and input gradient
         ([9000, 1, 0, 3999], 0, 2049, 4099, 256, 128, 256, 31)]                     # and weight gradient


@pytest.mark.parametrize('case', TILES, ids=str)
def test_the_cases_below_reach_the_tiles_that_they_name(case):
    """by the rules restated above; the rules' own lines and, for the segments, the workspace say that they are still the library's"""
    counts, tail, I, O, forward, back_input, back_weight, seg = case
    R, E = sum(counts) + tail, len(counts)
    assert prod_tile(False, R, E, O, O) == forward and prod_tile(False, R, E, O, I) == back_input
    assert prod_tile(True, R, E, O, I) == back_weight and seg_log2(R, E, O, I) == seg
    text = open(os.path.join(ROOT, 'diffusion-ccsp_amd', 'csrc', 'ops', 'ops_linear.h')).read()
    for line in ('inline long most_tiles(long R, long E, int l) { const long g = R < E + 1 ? R : E + 1; return (R >> l) + g; }',
                 'return (weight ? E * cdiv(M, 1l << l) : most_tiles(R, E, l)) * cdiv(N, 1l << l);',
                 'if (weight ? big >= 256 && R >= 1024 * E : big >= 1024 || (big >= 512 && R >= 1024 * E)) return TILE_256;',
                 'return prod_tiles(weight, R, E, M, N, 7) >= 512 ? TILE_128 : TILE_64;',
                 'prod_tile<T>(PROD == PROD_WEIGHT, p.R, p.E, out, PROD == PROD_FORWARD ? out : inp)'):
        assert line in text, line
    padded = lambda n: -(-n // 8) * 8      # noqa: E731
    need = sum(-(-R * padded(n) * 2 // 256) * 256 for n in (I, O) if n % 8)
    if seg != 31:
        need += 2 * ((R >> seg) + 1) * ((O * I + O + 3) // 4 * 4) * 4
    assert _ops.lib().ccsp_ops_linear_workspace(2, 1, E, R, I, O, 64, O, 64, I) == need


@pytest.mark.gpu
@pytest.mark.parametrize('case', TILES, ids=str)
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('act', [None, 'silu'])
def test_expert_linear_in_every_tile_with_gradients(device, case, dtype, act):
    counts, tail, I, O = case[:4]
    check_linear(device, counts, tail, I, O, DTYPES[dtype], act, True, where=device)


@pytest.mark.gpu
@pytest.mark.parametrize('case', TILES, ids=str)
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
def test_the_bias_gradient_alone_in_every_tile(device, case, dtype):
    """the bits that it has beside the weights' gradient, where a tile of 128 x 128 makes it too"""
    counts, tail, I, O = case[:4]
    expert = torch.cat([torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)), torch.full((tail,), -1)]).to(device)
    plan = ops.route(expert, len(counts))
    g = torch.Generator(device=device).manual_seed(8)
    xs, w, bias, gy = [torch.randn(*s, generator=g, device=device).to(DTYPES[dtype]) for s in ((len(expert), I), (len(counts), O, I), (len(counts), O), (len(expert), O))]
    bias.requires_grad_()
    alone, = torch.autograd.grad(ops.expert_linear(xs, w, plan, bias), bias, gy)
    w.requires_grad_()
    beside = torch.autograd.grad(ops.expert_linear(xs, w, plan, bias), (w, bias), gy)[1]
    assert torch.equal(alone, beside)


# ---- loading -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('which', ['lib', 'torch_ops'])
def test_first_calls_from_several_threads_load_once(monkeypatch, which):
    """each loader waits until the others had time to come in too"""
    import time
    loads, name = [], {'lib': '_lib', 'torch_ops': '_torch'}[which]

    def ensure():
        loads.append(threading.get_ident())
        time.sleep(0.2)
    monkeypatch.setattr(_ops, '_ensure', ensure)
    monkeypatch.setattr(_ops, name, None)
    if which == 'torch_ops':
        class Loader:
            def __init__(self, *args):
                pass

            def create_module(self, spec):
                return None

            def exec_module(self, m):
                m.version, m.set_error = (lambda: 1000 * _ops.OPS_ABI_MAJOR), (lambda e: None)
        monkeypatch.setattr(_ops.importlib.machinery, 'ExtensionFileLoader', Loader)
    got, gate = [], threading.Barrier(4)

    def first():
        gate.wait()
        got.append(getattr(_ops, which)())
    threads = [threading.Thread(target=first) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(loads) == 1 and len(got) == 4 and all(g is got[0] for g in got)

# ---- streams -------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_a_plan_recorded_on_another_stream_outlives_its_name(device):
    """the owner of a plan that another stream still reads records it there, as any tensor: its memory is not given away before"""
    expert = ids(60000, 20, 3, 0.1).to(device)
    x = torch.randn(60000, 64, device=device)
    want = ops.sort_rows(x, ops.route(expert, 20))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    plan = ops.route(expert, 20)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(20):
            got = ops.sort_rows(x, plan)
    size = plan.offsets.untyped_storage().nbytes()
    plan.offsets.record_stream(s)
    del plan
    for _ in range(4):                                            # (on the plan's own stream, while the other may still be at work)
        torch.full((size // 4,), -1, dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---- subclasses with memory ----------------------------------------------------------------------------------------------

class Counted(torch.Tensor):
    """a subclass with its own dispatch whose memory is its values"""
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        strip = lambda t: t.as_subclass(torch.Tensor) if isinstance(t, Counted) else t      # noqa: E731
        return func(*[strip(a) for a in args], **(kwargs or {}))


@pytest.mark.gpu
def test_a_subclass_with_memory_is_read_as_its_values(device):
    expert, (x, w, b, w2, weights), E = layer_inputs(device, torch.float32)
    plan = ops.route(expert, E)
    sub = torch.Tensor._make_subclass(Counted, x)
    assert type(sub) is Counted and sub.data_ptr() == x.data_ptr()
    assert torch.equal(ops.sort_rows(sub, plan), ops.sort_rows(x, plan))
    assert float(ops.global_norm([sub])) == float(ops.global_norm([x]))


def test_fake_tensors_are_refused():
    """tensors that say they are on the GPU and have no memory there"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True):
        t = torch.empty(4, device='cuda:0')
    with pytest.raises(TypeError, match='wraps others'):
        ops.global_norm([t])
