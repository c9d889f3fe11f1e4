"""Products grouped by agent (or expert) with ragged row counts: one dense layer of many networks in one launch
(libmpe_hip.so: mpe_grouped_linear, mpe_grouped_linear_backward; no counterpart in the reference, whose
learners evaluate one network at a time, maddpg/maddpg/trainer/maddpg.py:161-196).

    y = grouped_linear(x, weight, ends, bias=None, relu=False)       # y[r] = act(x[r] @ weight[g].T + bias[g])

``x``: ``[rows, k]``; ``weight``: ``[groups, n, k]`` (``torch.nn.Linear``'s layout, stacked); ``bias``: ``[groups, n]``;
``ends``: ``[groups]`` int32 or int64 on the same GPU: group ``g`` owns rows ``ends[g - 1] .. ends[g] - 1``
(``group_ends(sizes, device)`` makes it from row counts).  The kernels read ``ends`` from device memory, so a captured
launch follows what the tensor holds at replay and nothing is copied to the host; whatever it holds, it is read as its
running maximum clamped to ``[0, rows]``.  Groups may be empty.  float32, bfloat16 and float16, all arrays alike;
sums are in 32 bits, each result is rounded once.  1 <= groups <= 1024; rows and n * k below 2**31.

Rows of ``x`` may have any stride; an ``x`` whose columns are not adjacent is copied first (also a ``weight`` or ``bias``
that is not contiguous).  ``grouped_linear`` is differentiable (once) in ``x``, ``weight`` and ``bias``;
``grouped_linear_backward`` is the same backward pass as a plain call.  The sums run in a fixed order: the same inputs
give the same bits."""
import torch

from . import _hip

_DTYPES = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16, torch.float16: _hip.F16}
MAX_GROUPS = 1024


def group_ends(sizes, device='cuda'):
    """The ``ends`` tensor of consecutive groups with these row counts."""
    ends, total = [], 0
    for s in sizes:
        if int(s) != s or s < 0:
            raise ValueError('group sizes are whole numbers >= 0, got %r' % (s,))
        total += int(s)
        ends.append(total)
    if not 1 <= len(ends) <= MAX_GROUPS:
        raise ValueError('%d groups: 1 to %d are supported' % (len(ends), MAX_GROUPS))
    if total >= 1 << 31:
        raise ValueError('%d rows: below 2**31 are supported' % total)
    return torch.tensor(ends, dtype=torch.int32, device=device)


def _rows_of(t, name, shape=None, like=None):
    """A 2-d tensor the kernels take: adjacent columns, rows that do not overlap (a copy if need be); its row stride."""
    if t.dim() != 2 or (shape is not None and tuple(t.shape) != tuple(shape)):
        raise ValueError('%s: expected %s, got shape %s' % (name, 'a matrix' if shape is None else list(shape), list(t.shape)))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError('%s is %s on %s, not %s on %s' % (name, t.dtype, t.device, like.dtype, like.device))
    rows, cols = t.shape
    if not ((cols <= 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= cols)):
        t = t.contiguous()
    return t, (cols if rows <= 1 else t.stride(0))


def _check(x, weight, ends, bias=None):
    if not (torch.is_tensor(x) and torch.is_tensor(weight) and torch.is_tensor(ends)):
        raise TypeError('x, weight and ends are tensors')
    if x.device.type != 'cuda':
        raise RuntimeError('marl_amd.grouped works on GPU tensors (no CPU fallback)')
    if x.dtype not in _DTYPES:
        raise TypeError('marl_amd.grouped supports float32, bfloat16 and float16, got %r' % (x.dtype,))
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1]:
        raise ValueError('x [rows, k] and weight [groups, n, k] do not fit: %s, %s' % (list(x.shape), list(weight.shape)))
    g, n, k = weight.shape
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError('%s is %s on %s, not %s on %s' % (name, t.dtype, t.device, x.dtype, x.device))
    if bias is not None and tuple(bias.shape) != (g, n):
        raise ValueError('bias: expected %s, got shape %s' % ([g, n], list(bias.shape)))
    if not 1 <= g <= MAX_GROUPS or n < 1 or k < 1:
        raise ValueError('weight %s: 1 to %d groups of at least 1 x 1 are supported' % (list(weight.shape), MAX_GROUPS))
    if x.shape[0] >= 1 << 31 or n * k >= 1 << 31:
        raise ValueError('rows and n * k are below 2**31')
    if ends.dtype not in (torch.int32, torch.int64) or tuple(ends.shape) != (g,) or ends.device != x.device:
        raise ValueError('ends: expected int32 or int64 [%d] on %s, got %s %s on %s'
                         % (g, x.device, ends.dtype, list(ends.shape), ends.device))


def _desc(x, weight, ends):
    g, n, k = weight.shape
    return _hip.GroupedDesc(ends=ends.data_ptr(), rows=x.shape[0], groups=g, n=n, k=k, dtype=_DTYPES[x.dtype],
                            ends64=ends.dtype == torch.int64)


def _overlap(a, b):
    """Whether the byte ranges of two tensors meet."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _forward(x, weight, ends, bias, relu, out):
    _check(x, weight, ends, bias)
    x, ld_x = _rows_of(x, 'x')
    weight, ends = weight.contiguous(), ends.contiguous()
    bias = None if bias is None else bias.contiguous()
    rows, n = x.shape[0], weight.shape[1]
    own = out is None
    if own:
        out, ld_y = torch.empty(rows, n, dtype=x.dtype, device=x.device), n
    else:
        y, ld_y = _rows_of(out, 'out', (rows, n), x)
        if y is not out:
            raise ValueError('out: its columns must be adjacent and its rows must not overlap')
        if any(_overlap(out, t) for t in (x, weight, bias, ends)):
            raise ValueError('out overlaps an input')
    with _hip.on_device(x.device):
        _hip.check(_hip.lib.mpe_grouped_linear(_desc(x, weight, ends), x.data_ptr(), ld_x, weight.data_ptr(), _hip.ptr(bias),
                                               out.data_ptr(), ld_y, int(relu), int(own), _hip.stream_of(x.device)),
                   'mpe_grouped_linear')
    return out


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ends, bias, relu):
        y = _forward(x, weight, ends, bias, relu, None)
        ctx.save_for_backward(x, weight, ends, y if relu else None)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, ends, y = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx, dw, db = grouped_linear_backward(grad, x, weight, ends, y=y, need_dx=want[0], need_dweight=want[1], need_dbias=want[3])
        return dx, dw, None, db, None


def grouped_linear(x, weight, ends, bias=None, relu=False, out=None):
    """``y[r] = act(x[r] @ weight[g].T + bias[g])`` for the rows ``r`` of every group ``g`` (module docstring).  Rows behind
    the last group: zeros, or with ``out`` (``[rows, n]``, adjacent columns, no overlap with an input) left as they were."""
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in (x, weight, bias)):
        if out is not None:
            raise RuntimeError('grouped_linear(out=...) does not support automatic differentiation')
        return _GroupedLinear.apply(x, weight, ends, bias, bool(relu))
    return _forward(x, weight, ends, bias, bool(relu), out)


@torch.no_grad()
def grouped_linear_backward(grad, x, weight, ends, y=None, need_dx=True, need_dweight=True, need_dbias=True):
    """``(dx, dweight, dbias)`` of ``grouped_linear`` for the gradient ``grad`` ``[rows, n]`` of its result; ``y``: the
    result itself where it was made with ``relu=True`` (``grad`` counts where ``y`` is not <= 0).  An entry that is not needed
    is None.  ``dx`` is zero in rows of no group, ``dweight`` / ``dbias`` are zero for groups without rows."""
    _check(x, weight, ends)
    shape, want_dweight = (x.shape[0], weight.shape[1]), need_dweight
    grad, ld_g = _rows_of(grad, 'grad', shape, x)
    ld_y = 0
    if y is not None:
        y, ld_y = _rows_of(y, 'y', shape, x)
    ends = ends.contiguous()
    need_dweight = need_dweight or need_dbias
    desc, dx, dw, db = _desc(x, weight, ends), None, None, None
    ld_x = 0
    if need_dx:
        weight = weight.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if need_dweight:
        x, ld_x = _rows_of(x, 'x')
        dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
        db = torch.empty(weight.shape[:2], dtype=x.dtype, device=x.device) if need_dbias else None
    need = _hip.lib.mpe_grouped_backward_workspace(desc, y is not None, need_dweight)
    _hip.check(min(need, 0), 'mpe_grouped_backward_workspace')
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    with _hip.on_device(x.device):
        _hip.check(_hip.lib.mpe_grouped_linear_backward(
            desc, grad.data_ptr(), ld_g, _hip.ptr(y), ld_y, x.data_ptr(), ld_x, weight.data_ptr(), _hip.ptr(dx), x.shape[1], 1,
            _hip.ptr(dw), _hip.ptr(db), _hip.ptr(ws), need, _hip.stream_of(x.device)), 'mpe_grouped_linear_backward')
    return dx, dw if want_dweight else None, db
