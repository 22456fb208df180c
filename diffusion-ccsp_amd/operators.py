"""Operators for training and serving routed layers on the GPU, in the framework's own HIP kernels (include/ccsp_ops.h):

    plan = route(expert, n_experts)                  assignments sorted by expert (token n's k experts: expert [N, k])
    plan = route(expert, n_experts, tokens, n)       the same with an explicit token for every assignment
    xs   = sort_rows(x, plan)                        x [N, D] -> rows in their experts' order [A, D]
    ys   = expert_linear(xs, weight, plan, bias, activation='silu')      one product per expert, [E, O, I]
    y    = combine_rows(ys, plan, weights)           back to the tokens with the assignments' weights
    norm = clip_grad_norm_(parameters, max_norm)     the global gradient norm, gradients clipped in place

The denoiser is such a layer: an edge of type e sends its two nodes through the MLP of type e and adds the results onto them with the weight
1 / sqrt(degree) (networks/denoise_fn.py:313-389, :508-523); tools/train_gpu.py trains it with these operators.

Tensors live on one GPU, rows in float32, bfloat16 or float16; sums are held in 32 bits and rounded once.  Work goes to the current stream of the tensors'
device, nothing waits for it, and a call may be captured into a graph.  The gradients of sort_rows, combine_rows and expert_linear come through
torch.autograd (first order).  Every operator gives the same bits for the same inputs.
"""
from array import array

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _ops
from ._lib import CcspError

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATION = {None: 0, 'silu': 1}


def _on_gpu(who, *tensors):
    """the one device of the tensors (None entries skipped)"""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError('%s: expected a tensor, got %s' % (who, type(t).__name__))
        if not t.is_cuda:
            raise CcspError('%s: tensors must be on a GPU (got %s); there is no CPU fallback' % (who, t.device))
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError('%s: tensors on %s and %s' % (who, dev, t.device))
    return dev


def _run(dev, fn, *args):
    """one library call on the device's current stream"""
    if torch.cuda.current_device() == dev.index:
        _ops.check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))
    else:
        with torch.cuda.device(dev):
            _ops.check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))


def _rows(t):
    """a matrix the kernels can read: last dimension contiguous, rows at any non-negative distance"""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _float_rows(who, name, t, n, what):
    if t.dim() != 2 or t.shape[0] != n:
        raise ValueError('%s: %s must be [%d, width] (%s), got %s' % (who, name, n, what, tuple(t.shape)))
    if t.dtype not in _TYPE:
        raise TypeError('%s: %s of type %s; supported are float32, bfloat16 and float16' % (who, name, t.dtype))


class ExpertPlan(object):
    """What route() leaves on the device; all int32, made without waiting for the GPU.

    offsets [E + 1]   first row of every expert; offsets[E] = active rows
    rows [A]          row of every assignment, -1 if dropped
    assign [A]        assignment of every row; behind the last active row ~a of the dropped ones
    row_token [A]     token of every row, -1 behind the last active row
    shape             shape of the expert ids: the shape of combine_rows' weights"""
    __slots__ = ('n_experts', 'n_tokens', 'n_rows', 'k', 'shape', 'device', 'offsets', 'rows', 'assign', 'row_token', 'token_ptr', 'token_assign')

    @property
    def counts(self):
        """rows of every expert [E]"""
        return self.offsets[1:] - self.offsets[:-1]


def route(expert, n_experts, tokens=None, n_tokens=None):
    """Sorts assignments by expert.  expert: int32 / int64 ids in [0, n_experts), [N] or [N, k]: assignment (n, j) belongs to token n.  With `tokens` (the shape and type of
    `expert`) assignment a belongs to token tokens[a] of n_tokens: the typed edges of a graph, each node of an edge one assignment.  An
    assignment whose expert or token is out of range is dropped (the convention is -1), like the edges that match no constraint type."""
    dev = _on_gpu('route', expert, tokens)
    if expert.dtype not in (torch.int32, torch.int64):
        raise TypeError('route: expert ids must be int32 or int64, got %s' % expert.dtype)
    if not 1 <= n_experts <= _ops.MAX_EXPERTS:
        raise ValueError('route: %d experts, supported are 1 to %d' % (n_experts, _ops.MAX_EXPERTS))
    if tokens is None:
        if expert.dim() not in (1, 2):
            raise ValueError('route: expert ids must be [N] or [N, k], got %s' % (tuple(expert.shape),))
        if n_tokens is not None and n_tokens != expert.shape[0]:
            raise ValueError('route: %d tokens, but expert ids of %d' % (n_tokens, expert.shape[0]))
        n_tokens, k = expert.shape[0], 1 if expert.dim() == 1 else expert.shape[1]
        if k == 0:
            raise ValueError('route: no expert per token')
    else:
        if tokens.shape != expert.shape or tokens.dtype != expert.dtype:
            raise ValueError('route: tokens %s %s and expert ids %s %s differ' % (tokens.dtype, tuple(tokens.shape), expert.dtype, tuple(expert.shape)))
        if n_tokens is None or n_tokens < 0:
            raise ValueError('route: tokens need n_tokens')
        tokens, k = tokens.contiguous(), 0
    expert = expert.contiguous()
    p, A = ExpertPlan(), expert.numel()
    p.n_experts, p.n_tokens, p.n_rows, p.k, p.shape, p.device = n_experts, n_tokens, A, k, expert.shape, dev
    L = _ops.lib()
    need = L.ccsp_ops_route_workspace(A, n_experts, n_tokens, tokens is not None)
    if need < 0:
        raise ValueError('route: %d assignments of %d tokens are out of range' % (A, n_tokens))
    with torch.no_grad():
        p.offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
        p.rows, p.assign, p.row_token = torch.empty((3, A), dtype=torch.int32, device=dev).unbind(0)
        p.token_ptr = p.token_assign = None
        if tokens is not None:
            p.token_ptr = torch.empty(n_tokens + 1, dtype=torch.int32, device=dev)
            p.token_assign = torch.empty(A, dtype=torch.int32, device=dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _run(dev, L.ccsp_ops_route, expert.data_ptr(), None if tokens is None else tokens.data_ptr(), expert.element_size() * 8, A, k, n_experts, n_tokens, p.offsets.data_ptr(),
         p.rows.data_ptr(), p.assign.data_ptr(), p.row_token.data_ptr(), None if tokens is None else p.token_ptr.data_ptr(), None if tokens is None else p.token_assign.data_ptr(),
         ws.data_ptr(), need)
    return p


def _gather(src, plan):
    src = _rows(src)
    out = torch.empty((plan.n_rows, src.shape[1]), dtype=src.dtype, device=src.device)
    _run(src.device, _ops.lib().ccsp_ops_rows_gather, _TYPE[src.dtype], plan.n_rows, src.shape[1], src.data_ptr(), src.stride(0), plan.row_token.data_ptr(), out.data_ptr())
    return out


def _combine(src, plan, weights):
    src = _rows(src)
    out = torch.empty((plan.n_tokens, src.shape[1]), dtype=src.dtype, device=src.device)
    listed = plan.token_ptr is not None
    _run(src.device, _ops.lib().ccsp_ops_rows_combine, _TYPE[src.dtype], plan.n_tokens, src.shape[1], plan.k, plan.token_ptr.data_ptr() if listed else None,
         plan.token_assign.data_ptr() if listed else None, plan.rows.data_ptr(), None if weights is None else weights.data_ptr(), 0 if weights is None else _TYPE[weights.dtype],
         src.data_ptr(), src.stride(0), out.data_ptr())
    return out


class _SortRows(Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        return _gather(x, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return _combine(g, ctx.plan, None), None


class _CombineRows(Function):
    @staticmethod
    def forward(ctx, ys, weights, plan):
        ctx.plan = plan
        ctx.save_for_backward(ys if weights is not None and ctx.needs_input_grad[1] else None, weights)
        return _combine(ys, plan, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        plan, (ys, weights) = ctx.plan, ctx.saved_tensors
        if weights is None:
            return _gather(g, plan), None, None
        want_ys, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        g = _rows(g)
        ys = _rows(ys) if want_w else None
        d_ys = torch.empty((plan.n_rows, g.shape[1]), dtype=g.dtype, device=g.device) if want_ys else None
        d_w = torch.empty_like(weights, memory_format=torch.contiguous_format) if want_w else None
        _run(g.device, _ops.lib().ccsp_ops_rows_back, _TYPE[g.dtype], plan.n_rows, g.shape[1], plan.assign.data_ptr(), plan.row_token.data_ptr(), weights.data_ptr(), _TYPE[weights.dtype],
             g.data_ptr(), g.stride(0), ys.data_ptr() if want_w else None, ys.stride(0) if want_w else 0, d_ys.data_ptr() if want_ys else None, d_w.data_ptr() if want_w else None)
        return d_ys, d_w, None


def sort_rows(x, plan):
    """x [n_tokens, D] -> the rows of the plan's assignments in their experts' order [n_rows, D], zeros behind the last active row.  Gradient: every
    token's rows summed in the order of its assignments."""
    _on_gpu('sort_rows', x, plan.offsets)
    _float_rows('sort_rows', 'x', x, plan.n_tokens, 'one row per token')
    return _SortRows.apply(x, plan)


def combine_rows(ys, plan, weights=None):
    """y[n] = sum over token n's active assignments a, in their order, of weights[a] * ys[row of a]: [n_rows, D] -> [n_tokens, D]; zeros for a token without any.
    weights: the shape of the expert ids, float32 or the rows' type; None = 1.  Gradients for ys and weights."""
    _on_gpu('combine_rows', ys, weights, plan.offsets)
    _float_rows('combine_rows', 'ys', ys, plan.n_rows, 'one row per assignment')
    if weights is not None:
        if weights.shape != plan.shape:
            raise ValueError('combine_rows: weights %s for expert ids %s' % (tuple(weights.shape), tuple(plan.shape)))
        if weights.dtype not in (torch.float32, ys.dtype):
            raise TypeError('combine_rows: weights of type %s for rows of type %s; supported are float32 and the rows\' type' % (weights.dtype, ys.dtype))
        weights = weights.contiguous()
    return _CombineRows.apply(ys, weights, plan)


def _linear_space(product, code, E, plan, I, O, a, b):
    """(address, bytes, the tensor that holds them) of a product's workspace; a, b: its operands"""
    need = _ops.lib().ccsp_ops_linear_workspace(product, code, E, plan.n_rows, I, O, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(-2))
    if need < 0:
        raise ValueError('expert_linear: %d rows, %d -> %d of %d experts are out of range' % (plan.n_rows, I, O, E))
    if need == 0:
        return None, 0, None
    ws = torch.empty(need, dtype=torch.uint8, device=a.device)
    return ws.data_ptr(), need, ws


class _ExpertLinear(Function):
    @staticmethod
    def forward(ctx, xs, weight, bias, plan, act):
        x = _rows(xs)
        E, O, I = weight.shape
        code = _TYPE[x.dtype]
        y = torch.empty((plan.n_rows, O), dtype=x.dtype, device=x.device)
        z = torch.empty_like(y) if act and any(ctx.needs_input_grad) else None
        at, need, ws = _linear_space(0, code, E, plan, I, O, x, weight)
        _run(x.device, _ops.lib().ccsp_ops_linear, code, E, plan.n_rows, I, O, plan.offsets.data_ptr(), x.data_ptr(), x.stride(0), weight.data_ptr(),
             None if bias is None else bias.data_ptr(), act, y.data_ptr(), None if z is None else z.data_ptr(), at, need)
        ctx.plan, ctx.act = plan, act
        ctx.save_for_backward(x if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else None, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        plan, L = ctx.plan, _ops.lib()
        x, weight, z = ctx.saved_tensors
        E, O, I = weight.shape
        dev, code, off = g.device, _TYPE[g.dtype], plan.offsets.data_ptr()
        g = _rows(g)
        if ctx.act:
            dz = torch.empty((plan.n_rows, O), dtype=g.dtype, device=dev)
            _run(dev, L.ccsp_ops_linear_silu_back, code, E, plan.n_rows, O, off, g.data_ptr(), g.stride(0), z.data_ptr(), dz.data_ptr())
        else:
            dz = g
        d_x = d_w = d_b = None
        if ctx.needs_input_grad[0]:
            d_x = torch.empty((plan.n_rows, I), dtype=g.dtype, device=dev)
            at, need, ws = _linear_space(1, code, E, plan, I, O, dz, weight)
            _run(dev, L.ccsp_ops_linear_back_input, code, E, plan.n_rows, I, O, off, dz.data_ptr(), dz.stride(0), weight.data_ptr(), d_x.data_ptr(), at, need)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            if ctx.needs_input_grad[1]:
                d_w = torch.empty((E, O, I), dtype=g.dtype, device=dev)
            if ctx.needs_input_grad[2]:
                d_b = torch.empty((E, O), dtype=g.dtype, device=dev)
            at, need, ws = _linear_space(2, code, E, plan, I, O, dz, x)
            _run(dev, L.ccsp_ops_linear_back_weight, code, E, plan.n_rows, I, O, off, dz.data_ptr(), dz.stride(0), x.data_ptr(), x.stride(0),
                 None if d_w is None else d_w.data_ptr(), None if d_b is None else d_b.data_ptr(), at, need)
        return d_x, d_w, d_b, None, None


def expert_linear(xs, weight, plan, bias=None, activation=None):
    """The experts' products: rows of expert e become act(xs weight[e]^T + bias[e]); xs [n_rows, I] in the plan's order, weight [E, O, I], bias [E, O], all of one type;
    zeros behind the last active row.  activation: None or 'silu'.  Gradients for xs, weight and bias."""
    _on_gpu('expert_linear', xs, weight, bias, plan.offsets)
    _float_rows('expert_linear', 'xs', xs, plan.n_rows, 'one row per assignment')
    if activation not in _ACTIVATION:
        raise ValueError('expert_linear: activation %r; supported are None and \'silu\'' % (activation,))
    if weight.dim() != 3 or weight.shape[0] != plan.n_experts or weight.shape[2] != xs.shape[1] or 0 in weight.shape:
        raise ValueError('expert_linear: weight must be [%d, out, %d], got %s' % (plan.n_experts, xs.shape[1], tuple(weight.shape)))
    if bias is not None and tuple(bias.shape) != tuple(weight.shape[:2]):
        raise ValueError('expert_linear: bias must be [%d, %d], got %s' % (weight.shape[0], weight.shape[1], tuple(bias.shape)))
    if weight.dtype != xs.dtype or (bias is not None and bias.dtype != xs.dtype):
        raise TypeError('expert_linear: xs, weight and bias must have one type, got %s' % ', '.join(str(t.dtype) for t in (xs, weight, bias) if t is not None))
    return _ExpertLinear.apply(xs, weight.contiguous(), None if bias is None else bias.contiguous(), plan, _ACTIVATION[activation])


def _clip(who, tensors, max_norm, out):
    """norm of the tensors; out None: the norm alone, else the clipped tensors go there (out is tensors: in place)"""
    src = [t for t in tensors]
    if not src:
        raise ValueError('%s: no tensors' % who)
    dev = _on_gpu(who, *src) if out is None or out is tensors else _on_gpu(who, *src, *out)
    for t in src:
        if t.dtype not in _TYPE or t.layout != torch.strided:
            raise TypeError('%s: a tensor of type %s, %s; supported are dense float32, bfloat16 and float16' % (who, t.dtype, t.layout))
    dst = back = None
    flat = [t if t.is_contiguous() else t.contiguous() for t in src]
    if out is not None:
        if out is tensors:
            dst = flat                                           # (a tensor with gaps is clipped in its contiguous copy, then copied back)
            back = [(t, c) for t, c in zip(src, flat) if c is not t]
        else:
            dst = list(out)
            if len(dst) != len(src) or any(o.dtype != t.dtype or o.shape != t.shape for o, t in zip(dst, src)):
                raise ValueError('%s: out must hold one tensor of the same type and shape per gradient' % who)
            if not all(o.is_contiguous() for o in dst):
                raise ValueError('%s: out must be contiguous' % who)
        if not max_norm >= 0:
            raise ValueError('%s: max_norm %r must not be negative' % (who, max_norm))
    n = len(src)
    ptr_in, sizes = array('Q', [t.data_ptr() for t in flat]), array('q', [t.numel() for t in flat])
    types = array('i', [_TYPE[t.dtype] for t in flat])
    ptr_out = None
    if dst is not None:
        ptr_out = array('Q', [t.data_ptr() for t in dst])
        used = [p for p, m in zip(ptr_out, sizes) if m]
        if len(set(used)) != len(used):
            raise ValueError('%s: a tensor to write appears twice' % who)
    L = _ops.lib()
    a_sizes = sizes.buffer_info()[0]
    need = L.ccsp_ops_norm_workspace(n, a_sizes)
    with torch.no_grad():
        res = torch.empty(2, dtype=torch.float32, device=dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _run(dev, L.ccsp_ops_clip_norm, n, ptr_in.buffer_info()[0], None if dst is None else ptr_out.buffer_info()[0], a_sizes, types.buffer_info()[0],
             0.0 if out is None else float(max_norm), res.data_ptr(), res.data_ptr() + 4, ws.data_ptr(), need)
        for t, c in back or ():
            t.copy_(c)
        if dst is not None:
            written = [t for t in dst if not t.is_inference()]
            if written:
                torch.autograd.graph.increment_version(written)
    return res[0]


def global_norm(tensors):
    """sqrt of the sum of squares over all elements of all tensors, a float32 scalar on their device; squares and sums in 64 bits.  Not differentiable."""
    return _clip('global_norm', list(tensors), None, None)


def clip_global_norm(grads, max_norm, out=None):
    """Scales the tensors by min(1, max_norm / (norm + 1e-6)), norm their global norm before scaling, which is returned (a float32 scalar on the device;
    nothing waits for it).  In place, or into `out`: contiguous tensors of the same types and shapes, each the same memory as its gradient or disjoint from
    all.  Types may differ from tensor to tensor.  A norm that is not finite gives what the formula gives: factor 0 for infinity, NaN for NaN."""
    grads = list(grads)
    return _clip('clip_global_norm', grads, max_norm, grads if out is None else out)


def clip_grad_norm_(parameters, max_norm):
    """clip_global_norm in place on the gradients of `parameters` (a tensor or an iterable; those without a gradient are skipped, one that appears twice counts
    once).  Returns the norm before clipping, a float32 scalar on the device; 0 on the CPU if nothing has a gradient."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    seen, grads = set(), []
    for p in parameters:
        if p.grad is not None and id(p) not in seen:
            seen.add(id(p))
            grads.append(p.grad)
    if not grads:
        return torch.zeros(())
    return _clip('clip_grad_norm_', grads, max_norm, grads)
