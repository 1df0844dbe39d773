"""Dense on microscaled 4-bit weights (no counterpart in the reference).

    w4 = mxfp4_quantize(kernel.t())                    # [n_out, k], once
    y = mxfp4_dense(x, w4, bias, 'relu')               # x is quantised on the way in

or, for a layer that exists already, `Mxfp4Dense.from_dense(dense)`.  Weights of several experts are one tensor [E, n_out, k],
used by mxfp4_expert_dense on the rows that an expert_plan has sorted.  The format is OCP MXFP4: blocks of 32 columns
share a power of two, elements are +-0, .5, 1, 1.5, 2, 3, 4, 6 (include/gunet_hip.h has every rule).  x is rounded to 4 bits as well as the weights: on normal data a result is off by 0.16 of the
results' root mean square, 70 times the bf16 matmul mode's 0.0024, so a network has to be made for it.  For serving: no
gradients (a tensor that requires one or carries a tangent is refused), nothing synchronises, everything can be captured into a HIP graph.
"""
import torch

from .. import _lib
from .._lib import launch
from .expert_ops import DTYPES, check_plan, checked, dtype_code
from .hybrid_gnn import _activation_code

BLOCK = 32


class Mxfp4Tensor:
    """A 4-bit matrix [rows, k] or stack of matrices [groups, rows, k]: codes uint8 [groups, rows, blocks, 16] and scales uint8
    [groups, ceil(blocks / 8), rows, 8], the layout of include/gunet_hip.h."""

    def __init__(self, codes, scales, shape):
        self.shape = tuple(shape)
        want = self._layout(self.shape)
        for t, what, size in ((codes, 'codes', want[0]), (scales, 'scales', want[1])):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.uint8):
                raise TypeError(f'{what} must be a uint8 CUDA tensor')
            if t.shape != size or not t.is_contiguous() or t.data_ptr() % 16 or t.device != codes.device:
                raise ValueError(f'{what} must be packed {size} on 16 bytes, on one device, got {tuple(t.shape)} on {t.device}')
        self.codes, self.scales = codes, scales
        self.groups, self.rows, self.k = ((1,) + self.shape)[-3:]
        self.device = codes.device

    @staticmethod
    def _layout(shape):
        if len(shape) not in (2, 3) or shape[-1] < 1:
            raise ValueError(f'a 4-bit tensor is [rows, k] or [groups, rows, k] with k >= 1, got {tuple(shape)}')
        groups, rows, k = ((1,) + tuple(shape))[-3:]
        blocks = -(-k // BLOCK)
        return (groups, rows, blocks, 16), (groups, -(-blocks // 8), rows, 8)

    @classmethod
    def empty(cls, shape, device):
        """Room for a tensor of that shape, contents undefined."""
        codes, scales = cls._layout(shape)
        t = cls.__new__(cls)                    # what __init__ checks holds by construction
        t.codes = torch.empty(codes, dtype=torch.uint8, device=device)
        t.scales = t.codes.new_empty(scales)
        t.shape = tuple(shape)
        t.groups, t.rows, t.k = codes[0], codes[1], t.shape[-1]
        t.device = t.codes.device
        return t

    @classmethod
    def from_codes(cls, codes, scales, k):
        """From the row-major form that checkpoints hold: codes uint8 [.., rows, blocks * 16] (two columns a byte, the even one in the
        low four bits), scales uint8 [.., rows, blocks] (exponent + 127), blocks = ceil(k / 32)."""
        codes, scales = checked(codes, 'codes', dtype=torch.uint8), checked(scales, 'scales', dtype=torch.uint8)
        blocks = -(-int(k) // BLOCK)
        if codes.dim() not in (2, 3) or k < 1 or codes.shape[-1] != blocks * 16:
            raise ValueError(f'codes must be [.., rows, {blocks * 16}] for k = {k}, got {tuple(codes.shape)}')
        if tuple(scales.shape) != tuple(codes.shape[:-1]) + (blocks,) or scales.device != codes.device:
            raise ValueError(f'scales must be {tuple(codes.shape[:-1]) + (blocks,)} on {codes.device}, got {tuple(scales.shape)} on {scales.device}')
        t = cls.empty(codes.shape[:-1] + (int(k),), codes.device)
        t.codes.copy_(codes.view(t.codes.shape))
        if k % BLOCK:                                   # columns behind k: zeros, whatever the padding held
            used = k % BLOCK
            t.codes[:, :, -1, (used + 1) // 2:] = 0
            if used % 2:
                t.codes[:, :, -1, used // 2] &= 15
        t.scales.zero_()
        grouped = torch.nn.functional.pad(scales.view(t.groups, t.rows, blocks), (0, -blocks % 8))
        t.scales.copy_(grouped.view(t.groups, t.rows, -1, 8).transpose(1, 2))
        return t


def mxfp4_quantize(x):
    """x float32 / bfloat16 / float16 [rows, k] or [groups, rows, k] -> Mxfp4Tensor."""
    x = checked(x, 'x')
    code = dtype_code(x, 'x')
    t = Mxfp4Tensor.empty(x.shape, x.device)
    launch('gunet_mxfp4_quantize', t.device, x.data_ptr(), code, t.groups, t.rows, t.k, t.codes.data_ptr(), t.scales.data_ptr())
    return t


def mxfp4_dequantize(t, dtype=torch.float32):
    """The values of an Mxfp4Tensor (float16 may overflow or lose the smallest ones)."""
    if not isinstance(t, Mxfp4Tensor):
        raise TypeError('t must be an Mxfp4Tensor')
    if dtype not in DTYPES:
        raise TypeError(f'dtype must be float32, bfloat16 or float16, got {dtype}')
    out = torch.empty(t.shape, dtype=dtype, device=t.device)
    launch('gunet_mxfp4_dequantize', t.device, t.codes.data_ptr(), t.scales.data_ptr(), t.groups, t.rows, t.k, out.data_ptr(),
           DTYPES[dtype])
    return out


def _operands(x, w, bias, activation, out_dtype, groups_shape):
    if not isinstance(w, Mxfp4Tensor):
        raise TypeError('w must be an Mxfp4Tensor')
    x = checked(x, 'x', w.device)
    code = dtype_code(x, 'x')
    if x.dim() < 1 or x.shape[-1] != w.k:
        raise ValueError(f'x has {x.shape[-1] if x.dim() else 0} columns, w has {w.k}')
    if bias is not None:
        bias = checked(bias, 'bias', w.device, torch.float32, groups_shape + (w.rows,))
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in DTYPES:
        raise TypeError(f'out_dtype must be float32, bfloat16 or float16, got {out_dtype}')
    return x, code, bias, _activation_code(activation), out_dtype


def mxfp4_dense(x, w, bias=None, activation=None, out_dtype=None):
    """act(q(x) @ w^T + bias): x [.., k] float32 / bfloat16 / float16, w Mxfp4Tensor [n_out, k], bias float32 [n_out];
    the result [.., n_out] has x's type unless out_dtype names another.  Activations as for Dense."""
    x, code, bias, act, out_dtype = _operands(x, w, bias, activation, out_dtype, ())
    if len(w.shape) != 2:
        raise ValueError(f'w must be [n_out, k], got {w.shape} (mxfp4_expert_dense takes stacks)')
    rows = x.numel() // w.k
    out = x.new_empty(x.shape[:-1] + (w.rows,), dtype=out_dtype)
    nbytes = _lib.lib.gunet_mxfp4_dense_workspace_bytes(rows, w.k)
    scratch = w.codes.new_empty(nbytes) if nbytes else None
    launch('gunet_mxfp4_dense_forward', w.device, x.data_ptr(), code, rows, w.k, w.codes.data_ptr(), w.scales.data_ptr(),
           bias.data_ptr() if bias is not None else None, w.rows, act, out.data_ptr(), DTYPES[out_dtype],
           scratch.data_ptr() if nbytes else None, nbytes)
    return out


def mxfp4_expert_dense(x, w, plan, bias=None, activation=None, out_dtype=None, sorted_rows=False):
    """The experts' Dense layers on the rows of an ExpertPlan: w Mxfp4Tensor [E, n_out, k], bias float32 [E, n_out].
    x [T, k] holds the tokens (each row is dispatched in its 4-bit form), or with sorted_rows=True
    x [T * top_k, k] rows in expert order.  Returns [T * top_k, n_out] in expert order, zeros behind the last expert's rows."""
    check_plan(plan)
    x, code, bias, act, out_dtype = _operands(x, w, bias, activation, out_dtype, (getattr(w, 'groups', 0),))
    if len(w.shape) != 3 or w.groups != plan.n_experts:
        raise ValueError(f'w must be [{plan.n_experts}, n_out, k], got {w.shape}')
    if plan.device != x.device:
        raise ValueError(f'the plan is on {plan.device}, x is on {x.device}')
    want = plan.n_rows if sorted_rows else plan.n_tokens
    if x.dim() != 2 or x.shape[0] != want:
        raise ValueError(f'x must be [{want}, {w.k}], got {tuple(x.shape)}')
    out = x.new_empty((plan.n_rows, w.rows), dtype=out_dtype)
    nbytes = _lib.lib.gunet_mxfp4_expert_dense_workspace_bytes(plan.n_rows, w.k)
    scratch = w.codes.new_empty(nbytes)
    launch('gunet_mxfp4_expert_dense_forward', w.device, x.data_ptr(), code, plan.offsets.data_ptr(),
           None if sorted_rows else plan.slot.data_ptr(), plan.n_tokens, plan.top_k, plan.n_experts, w.k, w.codes.data_ptr(),
           w.scales.data_ptr(), bias.data_ptr() if bias is not None else None, w.rows, act, out.data_ptr(), DTYPES[out_dtype],
           scratch.data_ptr(), nbytes)
    return out


class Mxfp4Dense:
    """A Dense layer served from 4-bit weights: the same call, y = activation(x @ kernel + bias).  It can stand for in_layer or out_model
    of a GraphUNet that has its weights, which then walks its layers one by one; loading and listing weights is the Dense layer's."""

    def __init__(self, units, weights, bias=None, activation=None):
        if not isinstance(weights, Mxfp4Tensor) or len(weights.shape) != 2 or weights.rows != units:
            raise ValueError(f'weights must be an Mxfp4Tensor [{units}, in]')
        self.units, self.weights, self.bias, self.activation = units, weights, bias, activation
        _activation_code(activation)

    @classmethod
    def from_dense(cls, dense):
        """From a hybrid_gnn.Dense that holds its weights: the kernel [in, units] is transposed and quantised, the
        bias stays float32."""
        if dense.kernel is None:
            raise ValueError('the Dense layer has no weights yet')
        bias = dense.bias.detach().clone() if dense.bias is not None else None
        return cls(dense.units, mxfp4_quantize(dense.kernel.detach().t()), bias, dense.activation)

    def __call__(self, x, activation=Ellipsis):
        """activation overrides the layer's own for this call, as in Dense."""
        return mxfp4_dense(x, self.weights, self.bias, self.activation if activation is Ellipsis else activation)
