"""Rows sorted by expert and back (no counterpart in the reference): the learned form of its quadrant lists.

A router names top_k experts for every row (token).  `expert_plan` sorts those choices, `expert_dispatch` copies the rows
into expert order, the experts work on consecutive rows, and `expert_combine` adds their results back with
the router's weights:

    plan = expert_plan(index, n_experts)               # index int32 [T, k]; -1 = dropped
    rows = expert_dispatch(x, plan)                    # [T * k, C], expert e at plan.offsets[e]:plan.offsets[e + 1]
    ...                                                # e.g. mxfp4_expert_dense
    out = expert_combine(rows, weights, plan)          # weights float32 [T, k]

Unlike the index plans of the city graphs nothing here synchronises or is cached: a router chooses
anew at every step, and everything can be captured into a HIP graph.  Like the rest of the package the functions record no
autograd graph: a training step calls the gradients, `expert_combine_grad` and `expert_dispatch_grad`, itself (or from
an autograd.Function of its own); a tensor that requires a gradient, or carries a forward-mode tangent, is refused rather
than dropped from the graph.
Tensors may be strided (they are then copied first); all of them on one GPU, whose current stream the work goes to.
"""
import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import launch

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def dtype_code(t, what):
    code = DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f'{what} must be float32, bfloat16 or float16, got {t.dtype}')
    return code


def checked(t, what, device=None, dtype=None, shape=None):
    """t as a packed tensor, or a TypeError / ValueError that says what is wrong with it."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TypeError(f'{what} must be a CUDA tensor')
    if device is not None and t.device != device:
        raise ValueError(f'{what} is on {t.device}, the other tensors are on {device}')
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f'{what} must be {dtype}, got {t.dtype}')
    if shape is not None and t.shape != shape:
        raise ValueError(f'{what} must have the shape {tuple(shape)}, got {tuple(t.shape)}')
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{what} requires a gradient: this call records no autograd graph (detach it, or call under '
                         'torch.no_grad() and use the _grad functions)')
    if getattr(forward_ad, '_current_level', 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f'{what} carries a tangent, which this call would drop (take forward_ad.unpack_dual({what}).primal)')
    return t if t.is_contiguous() else t.contiguous()


class ExpertPlan:
    """offsets int32 [n_experts + 1] (rows of each expert), order int32 [T * k] (flat position t * k + j of each
    row, -1 behind the last) and slot int32 [T, k] (row of each choice, -1 = dropped).  Usually from expert_plan; parts
    that a program has from elsewhere must be packed int32 tensors of these shapes on one GPU.  Their values are
    taken into range by the kernels: wrong ones give wrong rows."""

    def __init__(self, offsets, order, slot, n_experts):
        parts = (offsets, 'offsets'), (order, 'order'), (slot, 'slot')
        for t, what in parts:
            if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32):
                raise TypeError(f'{what} must be an int32 CUDA tensor')
        n_experts = int(n_experts)
        if n_experts < 1 or slot.dim() != 2 or slot.shape[1] < 1:
            raise ValueError(f'a plan is of one expert or more and slot is [T, k] with k >= 1, got {n_experts} and {tuple(slot.shape)}')
        for (t, what), shape in zip(parts, ((n_experts + 1,), (slot.numel(),), slot.shape)):
            if t.shape != shape or not t.is_contiguous() or t.device != slot.device:
                raise ValueError(f'{what} must be packed {tuple(shape)} on {slot.device}, got {tuple(t.shape)} on {t.device}')
        if not slot.is_cuda:
            raise TypeError('the parts of a plan must be CUDA tensors')
        self._take(offsets, order, slot, n_experts)

    def _take(self, offsets, order, slot, n_experts):
        self.offsets, self.order, self.slot = offsets, order, slot
        self.n_experts = n_experts
        self.shape = slot.shape
        self.n_tokens, self.top_k = self.shape
        self.n_rows = self.n_tokens * self.top_k
        self.device = slot.device
        return self


def expert_plan(expert_index, n_experts):
    """The order of the choices expert_index int32 [T, k]; a value outside 0 .. n_experts - 1 drops the choice."""
    index = checked(expert_index, 'expert_index', None, torch.int32)
    if index.dim() != 2 or index.shape[1] < 1:
        raise ValueError(f'expert_index must be [T, k] with k >= 1, got {tuple(index.shape)}')
    n_experts = int(n_experts)
    t, k = index.shape
    dev = index.device
    offsets = index.new_empty(max(0, min(n_experts, _lib.MAX_EXPERTS)) + 1)       # the library refuses other numbers
    order = index.new_empty(t * k)
    slot = torch.empty_like(index)
    nbytes = _lib.lib.gunet_expert_sort_workspace_bytes(t, k, n_experts)
    scratch = index.new_empty(nbytes // 4) if nbytes else None
    launch('gunet_expert_sort', dev, index.data_ptr(), t, k, n_experts, offsets.data_ptr(), order.data_ptr(), slot.data_ptr(),
           scratch.data_ptr() if nbytes else None, nbytes)
    return ExpertPlan.__new__(ExpertPlan)._take(offsets, order, slot, n_experts)      # what __init__ checks holds by construction


def check_plan(plan):
    """Its parts go to the kernels as addresses: what an ExpertPlan holds is checked, what another object holds is not."""
    if not isinstance(plan, ExpertPlan):
        raise TypeError(f'plan must be an ExpertPlan, got {type(plan).__name__}')


def _width(t, what, rows):
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f'{what} must be [{rows}, width], got {tuple(t.shape)}')
    return t.shape[1]


def expert_dispatch(x, plan):
    """x [T, C] -> rows [T * k, C] in expert order (zeros behind the last expert's)."""
    check_plan(plan)
    x = checked(x, 'x', plan.device)
    width = _width(x, 'x', plan.n_tokens)
    code = dtype_code(x, 'x')
    rows = x.new_empty((plan.n_rows, width))
    launch('gunet_expert_dispatch', plan.device, x.data_ptr(), code, plan.offsets.data_ptr(), plan.slot.data_ptr(), plan.n_tokens,
           plan.top_k, plan.n_experts, width, rows.data_ptr())
    return rows


def expert_dispatch_grad(grad_rows, plan):
    """Gradient of expert_dispatch: grad_rows [T * k, C] -> grad_x [T, C]."""
    check_plan(plan)
    g = checked(grad_rows, 'grad_rows', plan.device)
    width = _width(g, 'grad_rows', plan.n_rows)
    code = dtype_code(g, 'grad_rows')
    grad_x = g.new_empty((plan.n_tokens, width))
    launch('gunet_expert_dispatch_grad', plan.device, g.data_ptr(), code, plan.slot.data_ptr(), plan.n_tokens, plan.top_k, width,
           grad_x.data_ptr())
    return grad_x


def expert_combine(rows, weights, plan):
    """out[t] = sum_j weights[t, j] * rows[slot[t, j]]: rows [T * k, C], weights float32 [T, k] -> [T, C]."""
    check_plan(plan)
    rows = checked(rows, 'rows', plan.device)
    width = _width(rows, 'rows', plan.n_rows)
    code = dtype_code(rows, 'rows')
    w = checked(weights, 'weights', plan.device, torch.float32, plan.shape)
    out = rows.new_empty((plan.n_tokens, width))
    launch('gunet_expert_combine', plan.device, rows.data_ptr(), code, w.data_ptr(), plan.slot.data_ptr(), plan.n_tokens, plan.top_k,
           width, out.data_ptr())
    return out


def expert_combine_grad(grad_out, rows, weights, plan):
    """Gradients of expert_combine: (grad_rows [T * k, C] in the type of rows, grad_weights float32 [T, k])."""
    check_plan(plan)
    rows = checked(rows, 'rows', plan.device)
    width = _width(rows, 'rows', plan.n_rows)
    code = dtype_code(rows, 'rows')
    g = checked(grad_out, 'grad_out', plan.device, rows.dtype, (plan.n_tokens, width))
    w = checked(weights, 'weights', plan.device, torch.float32, plan.shape)
    grad_rows = torch.empty_like(rows)
    grad_weights = torch.empty_like(w)
    launch('gunet_expert_combine_grad', plan.device, g.data_ptr(), rows.data_ptr(), code, w.data_ptr(), plan.offsets.data_ptr(),
           plan.slot.data_ptr(), plan.n_tokens, plan.top_k, plan.n_experts, width, grad_rows.data_ptr(), grad_weights.data_ptr())
    return grad_rows, grad_weights
