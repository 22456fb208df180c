"""Operators for training and serving routed layers on the GPU, in the framework's own HIP kernels (include/ccsp_ops.h):

    plan = route(expert, n_experts)                  assignments sorted by expert (token n's k experts: expert [N, k])
    plan = route(expert, n_experts, tokens, n)       the same with an explicit token for every assignment
    xs   = sort_rows(x, plan)                        x [N, D] -> rows in their experts' order [A, D]
    ys   = expert_linear(xs, weight, plan, bias, activation='silu')      one product per expert, [E, O, I]
    y    = combine_rows(ys, plan, weights)           back to the tokens with the assignments' weights
    norm = clip_grad_norm_(parameters, max_norm)     the global gradient norm, gradients clipped in place

The denoiser is such a layer: an edge of type e sends its two nodes through the MLP of type e and adds the results onto them with the weight
1 / sqrt(degree) (networks/denoise_fn.py:313-389, :508-523); tools/train_gpu.py trains it with these operators.

Tensors live on one GPU, rows in float32, bfloat16 or float16; sums are held in 32 bits and each result is rounded once.  expert_linear with an activation
keeps two values between its forward and its backward in the rows' type as well: the pre-activation, and the gradient of it that the matrix instructions take (in
float16 one beyond 65504 is infinite, like any result).

Work goes to the current stream of the tensors' device and nothing waits for it.  A plan or tensor that another stream uses is recorded there by its owner, as
everywhere in torch (plan.offsets.record_stream).  A call may be captured into a graph; a backward pass through torch.autograd.grad, as nothing may be left to do
on the leaves' own stream, and with no autograd graph from outside of the capture alive on the same leaves, whose stream torch would join with the capture.
torch.jit.trace and make_fx record torch's own operations only: an operator raises under them, and for tensors that wrap others.

The gradients of sort_rows, combine_rows and expert_linear come through torch.autograd, first order and in reverse (forward-mode derivatives raise).  Every
operator gives the same bits for the same inputs.
"""
import torch

from . import _ops


def __getattr__(name):
    if name == 'ExpertPlan':                      # the class of route()'s results
        return _ops.torch_ops().ExpertPlan
    raise AttributeError(name)


def route(expert, n_experts, tokens=None, n_tokens=None):
    """Sorts assignments by expert.  expert: int32 / int64 ids in [0, n_experts), [N] or [N, k]: assignment (n, j) belongs to token n.  With `tokens` (the shape and type of
    `expert`) assignment a belongs to token tokens[a] of n_tokens: the typed edges of a graph, each node of an edge one assignment.  An
    assignment whose expert or token is out of range is dropped (the convention is -1), like the edges that match no constraint type.
    Returns an ExpertPlan: offsets, rows, assign, row_token, counts (int32, on the device)."""
    return _ops.torch_ops().route(expert, n_experts, tokens, n_tokens)


def sort_rows(x, plan):
    """x [n_tokens, D] -> the rows of the plan's assignments in their experts' order [n_rows, D], zeros behind the last active row.  Gradient: every
    token's rows summed in the order of its assignments."""
    return _ops.torch_ops().sort_rows(x, plan)


def combine_rows(ys, plan, weights=None):
    """y[n] = sum over token n's active assignments a, in their order, of weights[a] * ys[row of a]: [n_rows, D] -> [n_tokens, D]; zeros for a token without any.
    weights: the shape of the expert ids, float32 or the rows' type; None = 1.  Gradients for ys and weights."""
    return _ops.torch_ops().combine_rows(ys, plan, weights)


def expert_linear(xs, weight, plan, bias=None, activation=None):
    """The experts' products: rows of expert e become act(xs weight[e]^T + bias[e]); xs [n_rows, I] in the plan's order, weight [E, O, I], bias [E, O], all of one type;
    zeros behind the last active row.  activation: None or 'silu'.  Gradients for xs, weight and bias."""
    return _ops.torch_ops().expert_linear(xs, weight, plan, bias, activation)


def global_norm(tensors):
    """sqrt of the sum of squares over all elements of all tensors, a float32 scalar on their device; squares and sums in 64 bits.  Not differentiable."""
    return _ops.torch_ops().clip('global_norm', list(tensors), None, None)


def clip_global_norm(grads, max_norm, out=None):
    """Scales the tensors by min(1, max_norm / (norm + 1e-6)), norm their global norm before scaling, which is returned (a float32 scalar on the device;
    nothing waits for it).  In place (gradients that are not expanded), or into `out`: contiguous tensors of the same types and shapes, each the same memory as its gradient or disjoint from
    all (checked).  Types may differ from tensor to tensor.  A norm that is not finite gives what the formula gives: factor 0 for infinity, NaN for NaN."""
    return _ops.torch_ops().clip('clip_global_norm', list(grads), float(max_norm), out if out is None else list(out))


def clip_grad_norm_(parameters, max_norm):
    """clip_global_norm in place on the gradients of `parameters` (a tensor or an iterable; those without a gradient are skipped, one that appears twice counts
    once).  Returns the norm before clipping, a float32 scalar on the device; 0 on the CPU if nothing has a gradient."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in dict.fromkeys(parameters) if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return _ops.torch_ops().clip('clip_grad_norm_', grads, float(max_norm), None)
