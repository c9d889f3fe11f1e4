"""Products grouped by agent (or expert) with ragged row counts: one dense layer of many networks in one launch
(libmpe_hip.so: mpe_grouped_linear, mpe_grouped_linear_backward; no counterpart in the reference, whose
learners evaluate one network at a time, maddpg/maddpg/trainer/maddpg.py:161-196).

    y = grouped_linear(x, weight, ends, bias=None, relu=False)       # y[r] = act(x[r] @ weight[g].T + bias[g])

``x``: ``[rows, k]``; ``weight``: ``[groups, n, k]`` (``torch.nn.Linear``'s layout, stacked); ``bias``: ``[groups, n]``;
``ends``: ``[groups]`` int32 or int64 on the same GPU: group ``g`` owns rows ``ends[g - 1] .. ends[g] - 1``
(``group_ends(sizes, device)`` makes it from row counts).  The kernels read ``ends`` from device memory, so a captured
launch follows what the tensor holds at replay and nothing is copied to the host; whatever it holds, it is read as its
running maximum clamped to ``[0, rows]``.  Groups may be empty.  float32, bfloat16 and float16, all arrays alike;
sums are in 32 bits, each result is rounded once.  1 <= groups <= 1024; n and k up to 2**20, rows and n * k
below 2**31; more than 2**23 - 8 tiles of 64 x 64 results are refused.

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


def _rows_of(t):
    """A matrix the kernels take -- adjacent columns, rows that do not overlap -- as it is or as a copy; its row stride."""
    rows, cols = t.shape
    if t.is_contiguous():
        return t, cols
    if not ((cols <= 1 or t.stride(1) == 1) and (rows <= 1 or t.stride(0) >= cols)):
        return t.contiguous(), cols
    return t, (cols if rows <= 1 else t.stride(0))


def _matrix(t, name, rows, cols, like):
    """Checks an argument that belongs to ``like``'s rows."""
    if not torch.is_tensor(t) or t.dtype is not like.dtype or t.get_device() != like.get_device():
        raise ValueError('%s: expected %s on %s, got %s' % (name, like.dtype, like.device,
                                                            '%s on %s' % (t.dtype, t.device) if torch.is_tensor(t) else type(t)))
    if tuple(t.shape) != (rows, cols):
        raise ValueError('%s: expected %s, got shape %s' % (name, [rows, cols], list(t.shape)))


def _refuse(x, weight, ends, bias):
    """Says what is wrong with arguments that ``_check`` does not take."""
    if not (torch.is_tensor(x) and torch.is_tensor(weight) and torch.is_tensor(ends) and (bias is None or torch.is_tensor(bias))):
        raise TypeError('x, weight, ends and bias are tensors')
    if x.device.type != 'cuda':
        raise RuntimeError('marl_amd.grouped works on GPU tensors (no CPU fallback)')
    if x.dtype not in _DTYPES:
        raise TypeError('marl_amd.grouped supports float32, bfloat16 and float16, got %r' % (x.dtype,))
    if x.dim() != 2 or weight.dim() != 3 or weight.shape[2] != x.shape[1]:
        raise ValueError('x [rows, k] and weight [groups, n, k] do not fit: %s, %s' % (list(x.shape), list(weight.shape)))
    for t, name in ((weight, 'weight'), (bias, 'bias')):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError('%s is %s on %s, not %s on %s' % (name, t.dtype, t.device, x.dtype, x.device))
    g, n, k = weight.shape
    if bias is not None and tuple(bias.shape) != (g, n):
        raise ValueError('bias: expected %s, got shape %s' % ([g, n], list(bias.shape)))
    if not 1 <= g <= MAX_GROUPS or n < 1 or k < 1:
        raise ValueError('weight %s: 1 to %d groups of at least 1 x 1 are supported' % (list(weight.shape), MAX_GROUPS))
    if ends.dtype not in (torch.int32, torch.int64) or tuple(ends.shape) != (g,) or ends.device != x.device:
        raise ValueError('ends: expected int32 or int64 [%d] on %s, got %s %s on %s'
                         % (g, x.device, ends.dtype, list(ends.shape), ends.device))
    raise ValueError('n and k are up to 2**20, rows and n * k below 2**31')


def _check(x, weight, ends, bias=None):
    """The sizes' descriptor and the GPU's index; ``ends`` has to outlive the call."""
    try:
        (rows, k), (g, n, wk), (ge,) = x.shape, weight.shape, ends.shape
        dtype, index, e64 = x.dtype, x.get_device(), ends.dtype is torch.int64
        ok = (index >= 0 and dtype in _DTYPES and weight.dtype is dtype and weight.get_device() == index and wk == k and ge == g
              and ends.get_device() == index and (e64 or ends.dtype is torch.int32) and 1 <= g <= MAX_GROUPS and n >= 1 and k >= 1
              and rows < 1 << 31 and n * k < 1 << 31 and n <= 1 << 20 and k <= 1 << 20
              and (bias is None or (bias.dtype is dtype and bias.get_device() == index and bias.shape == (g, n))))
    except (ValueError, AttributeError, TypeError):
        ok = False
    if not ok:
        _refuse(x, weight, ends, bias)
    return _hip.GroupedDesc(ends.data_ptr(), rows, g, n, k, _DTYPES[dtype], e64, 0), index, rows, n, k


def _overlap(a, b):
    """Whether the byte ranges of two tensors meet."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((s - 1) * st for s, st in zip(t.shape, t.stride())) + 1) * t.element_size()
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _scratch(x, need):
    """``need`` bytes of this call's own (from torch's allocator, so on this stream or of this recording)."""
    _hip.check(min(need, 0), 'workspace')
    return x.new_empty((need + 3) // 4, dtype=torch.float32)


def _forward(x, weight, ends, bias, relu, out):
    if torch.is_tensor(ends) and not ends.is_contiguous():
        ends = ends.contiguous()
    desc, index, rows, n, _ = _check(x, weight, ends, bias)
    x, ld_x = _rows_of(x)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    own = out is None
    if own:
        out, ld_y = x.new_empty((rows, n)), n
    else:
        _matrix(out, 'out', rows, n, x)
        y, ld_y = _rows_of(out)
        if y is not out:
            raise ValueError('out: its columns must be adjacent and its rows must not overlap')
        if any(_overlap(out, t) for t in (x, weight, bias, ends)):
            raise ValueError('out overlaps an input')
    px, pw, ws = x.data_ptr(), weight.data_ptr(), None
    need = _hip.lib.mpe_grouped_linear_workspace(desc, px, ld_x, pw)
    if need:
        ws = _scratch(x, need)
    _hip.check(_hip.launch(index, _hip.lib.mpe_grouped_linear, desc, px, ld_x, pw, None if bias is None else bias.data_ptr(),
                           out.data_ptr(), ld_y, relu, own, _hip.ptr(ws), need), 'mpe_grouped_linear')
    if not own and not out.is_inference():
        torch.autograd.graph.increment_version(out)          # what autograd saved of it before is no longer there
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
    if torch.is_grad_enabled() and any([torch.is_tensor(t) and t.requires_grad for t in (x, weight, bias, out)]):
        if out is not None:
            raise RuntimeError('grouped_linear(out=...) does not support automatic differentiation')
        return _GroupedLinear.apply(x, weight, ends, bias, bool(relu))
    return _forward(x, weight, ends, bias, bool(relu), out)


def grouped_linear_backward(grad, x, weight, ends, y=None, need_dx=True, need_dweight=True, need_dbias=True):
    """``(dx, dweight, dbias)`` of ``grouped_linear`` for the gradient ``grad`` ``[rows, n]`` of its result; ``y``: the
    result itself where it was made with ``relu=True`` (``grad`` counts where ``y`` is not <= 0).  An entry that is not needed
    is None.  ``dx`` is zero in rows of no group, ``dweight`` / ``dbias`` are zero for groups without rows.  ``dbias`` comes with
    ``dweight``: alone it costs the same.  Groups may have any rows, but dweight's work is split for groups of the mean size: one
    group with most of the rows is slow (``dw_splits`` in mpe_grouped.hip has figures)."""
    if torch.is_tensor(ends) and not ends.is_contiguous():
        ends = ends.contiguous()
    desc, index, rows, n, k = _check(x, weight, ends)
    _matrix(grad, 'grad', rows, n, x)
    grad, ld_g = _rows_of(grad)
    ld_x = ld_y = 0
    if y is not None:
        _matrix(y, 'y', rows, n, x)
        y, ld_y = _rows_of(y)
    both = need_dweight or need_dbias
    dx = dw = db = ws = None
    if need_dx:
        if not weight.is_contiguous():
            weight = weight.contiguous()
        dx = x.new_empty((rows, k))
    if both:
        x, ld_x = _rows_of(x)
        dw = x.new_empty(weight.shape)
        db = x.new_empty(weight.shape[:2]) if need_dbias else None
    pg, py, px, pw = grad.data_ptr(), _hip.ptr(y), x.data_ptr(), weight.data_ptr()
    need = _hip.lib.mpe_grouped_backward_workspace(desc, pg, ld_g, py, ld_y, px, ld_x, pw, need_dx, both)
    if need:
        ws = _scratch(x, need)
    _hip.check(_hip.launch(index, _hip.lib.mpe_grouped_linear_backward, desc, pg, ld_g, py, ld_y, px, ld_x, pw, _hip.ptr(dx), k, 1, _hip.ptr(dw), _hip.ptr(db), _hip.ptr(ws), need),
               'mpe_grouped_linear_backward')
    return dx, dw if need_dweight else None, db
