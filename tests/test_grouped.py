"""marl_amd.grouped: products grouped by agent with ragged row counts against plain 64-bit products, forward and backward."""
import ctypes as C

import pytest
import torch

from marl_amd import _hip, grouped

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative


# ---- refusals (no GPU needed) --------------------------------------------------------------------------------------------
def test_group_ends_checks_its_sizes():
    assert grouped.group_ends([3, 0, 2], device='cpu').tolist() == [3, 3, 5]
    for bad in ([], [1, -1], [1.5], [1] * 1025, [1 << 30, 1 << 30]):
        with pytest.raises(ValueError):
            grouped.group_ends(bad, device='cpu')


def test_cpu_tensors_are_refused():
    x, w, e = torch.zeros(4, 3), torch.zeros(2, 5, 3), torch.tensor([2, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        grouped.grouped_linear(x, w, e)
    with pytest.raises(RuntimeError):
        grouped.grouped_linear_backward(torch.zeros(4, 5), x, w, e)


def _desc(**kw):
    d = dict(ends=4096, rows=4, groups=2, n=5, k=3, dtype=_hip.F32, ends64=0)
    d.update(kw)
    return _hip.GroupedDesc(**d)


@pytest.mark.parametrize('change,code', [
    (dict(ends=None), -1), (dict(dtype=3), -5), (dict(groups=0), -6), (dict(groups=1025), -6), (dict(n=0), -6), (dict(k=0), -6),
    (dict(rows=-1), -6), (dict(rows=1 << 31), -6), (dict(n=1 << 16, k=1 << 15), -6), (dict(n=(1 << 20) + 1), -6), (dict(k=(1 << 20) + 1), -6), (dict(ends=4098), -4),
    (dict(ends=4100, ends64=1), -4), (dict(ends64=2), -6)])
def test_c_abi_refuses_bad_descriptors(change, code):
    """Nothing is launched: the pointers are never read."""
    d, p = _desc(**change), 1 << 20
    assert _hip.lib.mpe_grouped_linear(d, p, 3, p, None, p, 5, 0, 0, None, 0, None) == code
    assert _hip.lib.mpe_grouped_linear_workspace(d, p, 3, p) == code
    assert _hip.lib.mpe_grouped_backward_workspace(d, p, 5, None, 0, p, 3, p, 1, 1) == code
    assert _hip.lib.mpe_grouped_linear_backward(d, p, 5, None, 0, p, 3, p, p, 3, 0, p, p, None, 0, None) == code


def test_c_abi_refuses_bad_arrays():
    L, d, p = _hip.lib, _desc(), 1 << 20
    assert L.mpe_grouped_linear(None, p, 3, p, None, p, 5, 0, 0, None, 0, None) == -1
    assert L.mpe_grouped_linear(d, None, 3, p, None, p, 5, 0, 0, None, 0, None) == -1
    assert L.mpe_grouped_linear(d, p, 2, p, None, p, 5, 0, 0, None, 0, None) == -6
    assert L.mpe_grouped_linear(d, p, 3, p, None, p, 4, 0, 0, None, 0, None) == -6
    assert L.mpe_grouped_linear(d, p, 3, p, None, p, 5, 2, 0, None, 0, None) == -6
    assert L.mpe_grouped_linear(d, p, 3, p, None, p, 5, 0, 2, None, 0, None) == -6
    assert L.mpe_grouped_linear(d, p + 2, 3, p, None, p, 5, 0, 0, None, 0, None) == -4
    assert L.mpe_grouped_linear(d, p, 3, p, p + 1, p, 5, 0, 0, None, 0, None) == -4
    ok = dict(dy=p, ld_dy=5, y=None, ld_y=0, x=p, ld_x=3, w=p, dx=p, ld_dx=3, zero=0, dw=p, db=p, ws=None, size=0)

    def back(desc=d, **kw):
        return L.mpe_grouped_linear_backward(desc, *dict(ok, **kw).values(), None)
    for kw, code in ((dict(dy=None), -1), (dict(x=None), -1), (dict(w=None), -1), (dict(dw=None), -1), (dict(ld_dy=4), -6),
                     (dict(y=p, ld_y=4), -6), (dict(ld_x=2), -6), (dict(ld_dx=2), -6), (dict(zero=2), -6), (dict(dy=p + 1), -4),
                     (dict(y=p + 2, ld_y=5), -4), (dict(x=p + 2), -4), (dict(w=p + 2), -4), (dict(dx=p + 2), -4), (dict(dw=p + 2), -4),
                     (dict(db=p + 2), -4), (dict(ws=p + 8), -4)):
        assert back(**kw) == code, kw
    def size(desc=d, y=None, dx=1, dw=1):
        return L.mpe_grouped_backward_workspace(desc, p, 5, y, 5, p, 3, p, dx, dw)
    assert size(dx=2) == -6 and size(dw=-1) == -6 and size() == 0 and size(y=p) == 0
    wide = _desc(dtype=_hip.BF16, rows=1 << 14, n=1001, k=1024)    # y beside large products: dy masked, in rows of whole chunks
    assert size(wide, y=p, dw=0) == (1 << 14) * 1008 * 2
    big = _desc(rows=1 << 20)                                     # rows split over workgroups: partial sums need an array
    need = size(big)
    assert need > 0 and size(big, dw=0) == 0
    assert back(big, ws=None, size=need) == -1
    assert back(big, ws=p, size=need - 1) == -7
    far = 1 << 24                                                 # rows so far apart that they are packed into scratch first
    need = L.mpe_grouped_linear_workspace(d, p, far, p)
    assert need == 4 * 4 * 4 and L.mpe_grouped_linear_workspace(d, p, 3, p) == 0
    assert L.mpe_grouped_linear(d, p, far, p, None, p, 5, 0, 0, None, need, None) == -1
    assert L.mpe_grouped_linear(d, p, far, p, None, p, 5, 0, 0, p, need - 1, None) == -7
    assert L.mpe_grouped_linear(d, p, far, p, None, p, 5, 0, 0, p + 8, need, None) == -4
    many = _desc(rows=(1 << 31) - 1, n=64, k=16)                  # more tiles than one launch may have
    assert L.mpe_grouped_linear(many, p, 16, p, None, p, 64, 0, 0, None, 0, None) == -6
    assert L.mpe_grouped_linear_backward(many, p, 64, None, 0, p, 16, p, p, 16, 0, None, None, None, 0, None) == -6
    assert C.sizeof(_hip.GroupedDesc) == 40


# ---- against 64 bits -----------------------------------------------------------------------------------------------------
def _case(sizes, k, n, dtype, tail=0, seed=0, device='cuda'):
    g = torch.Generator().manual_seed(seed)
    t = sum(sizes) + tail
    mk = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)     # noqa: E731
    return (mk(t, k), (mk(len(sizes), n, k).float() * k ** -0.5).to(dtype), mk(len(sizes), n), mk(t, n),
            grouped.group_ends(sizes, device))


def _reference(x, w, b, grad, sizes, relu, y_saved=None):
    """(y, dx, dw, db) in 64 bits, and for each the sum of the absolute values of its terms."""
    x, w, b, grad = x.double(), w.double(), b.double(), grad.double()
    y, dx = torch.zeros(grad.shape, dtype=torch.float64, device=x.device), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    ya, dxa, dwa, dba = (torch.zeros_like(t) for t in (y, dx, dw, db))
    r = 0
    for g, s in enumerate(sizes):
        p = slice(r, r + s)
        r += s
        y[p], ya[p] = x[p] @ w[g].t().contiguous() + b[g], x[p].abs() @ w[g].abs().t().contiguous() + b[g].abs()
        if relu:
            y[p] = y[p].clamp(min=0)
        d = grad[p] if y_saved is None else grad[p] * (y_saved[p].double() > 0)
        dx[p], dxa[p] = d @ w[g], d.abs() @ w[g].abs()
        dw[g], dwa[g] = d.t().contiguous() @ x[p], d.abs().t().contiguous() @ x[p].abs()
        db[g], dba[g] = d.sum(0), d.abs().sum(0)
    return (y, dx, dw, db), (ya, dxa, dwa, dba)


def _close(got, want, terms, count, dtype, what):
    """Sum of ``count`` products in f32, any order: each product and addition is off by at most 2^-23 of a partial sum, which
    is at most the sum of the terms' absolute values (2^-23, not 2^-24: the matrix unit may cut off what it aligns); then one
    rounding to the type (half a step; f16 below its normal range: half of 2^-24)."""
    tol = (count + 2) * 2.0 ** -23 * terms + HALF[dtype] * want.abs() * (1 + 1e-3) + (2.0 ** -25 if dtype == torch.float16 else 0)
    bad = (got.double() - want).abs() > tol
    assert got.dtype == dtype and not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


SHAPES = [
    ([1], 1, 1), ([5], 3, 2), ([0, 1, 0], 7, 9), ([3, 0, 64, 65, 1], 16, 64), ([63, 64, 65], 33, 65), ([256] * 4, 64, 64),
    ([1000, 1, 0, 500], 226, 64), ([128, 129], 64, 5), ([17, 300, 3], 333, 517), ([200, 0, 56], 512, 256), ([0, 0], 8, 8),
    ([2500], 130, 40), ([1] * 70, 20, 24), ([700, 900], 128, 136), ([1, 2, 1, 0, 3], 1024, 520),
    ([900, 0, 1300, 760], 512, 2048), ([4100, 5001], 2048, 264), ([3000, 2200], 130, 2050), ([1500] * 6, 1032, 1024),
    ([700, 0, 1300, 399, 1111, 2600, 520, 1501], 264, 2056), ([33, 0, 64, 1] * 4, 1000, 1032),
    ([1024, 1500, 3, 900, 0, 2048, 1111, 130, 1793, 640, 1280, 385, 2200, 1029, 1337, 1020], 1032, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('relu', [False, True], ids=['linear', 'relu'])
@pytest.mark.parametrize('sizes,k,n', SHAPES, ids=['%dx%d_%d_%d' % (len(s), sum(s), k, n) for s, k, n in SHAPES])
def test_forward_and_backward(sizes, k, n, relu, dtype):
    x, w, b, grad, ends = _case(sizes, k, n, dtype)
    y = grouped.grouped_linear(x, w, ends, bias=b, relu=relu)
    dx, dw, db = grouped.grouped_linear_backward(grad, x, w, ends, y=y if relu else None)
    want, terms = _reference(x, w, b, grad, sizes, relu, y if relu else None)
    most = max(sizes)
    for got, ref, ab, count, what in zip((y, dx, dw, db), want, terms, (k + 1, n, most, most), ('y', 'dx', 'dw', 'db')):
        _close(got, ref, ab, count, dtype, what)
    for g, s in enumerate(sizes):
        if s == 0:
            assert not dw[g].any() and not db[g].any()
    y0 = grouped.grouped_linear(x, w, ends, relu=relu)                       # no bias
    ref0, terms0 = _reference(x, w, torch.zeros_like(b), grad, sizes, relu)
    _close(y0, ref0[0], terms0[0], k, dtype, 'y without bias')


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_strides_alignment_and_rows_of_no_group(dtype):
    """Row strides that are no multiple of anything, bases in the middle of a 16-byte word, columns that are not adjacent,
    int64 ends; rows behind the last group are zeros, or left as they were in ``out``."""
    sizes, k, n, tail = [70, 0, 131, 9], 45, 77, 100
    x, w, b, grad, ends = _case(sizes, k, n, dtype, tail=tail)
    want, terms = _reference(x, w, b, grad, sizes, False)
    t, live = x.shape[0], sum(sizes)
    xs = torch.full((t, k + 6), 7.0, dtype=dtype, device='cuda')[:, 3:3 + k]
    xs.copy_(x)
    gs = torch.full((t, n + 4), 7.0, dtype=dtype, device='cuda')[:, 1:1 + n]
    gs.copy_(grad)
    ws = torch.empty(w.numel() + 1, dtype=dtype, device='cuda')[1:].view(w.shape).copy_(w)
    for xx, ww, gg in ((xs, ws, gs), (x.t().contiguous().t(), w.transpose(0, 1).contiguous().transpose(0, 1), grad.t().contiguous().t())):
        y = grouped.grouped_linear(xx, ww, ends.long(), bias=b)
        dx, dw, db = grouped.grouped_linear_backward(gg, xx, ww, ends.long())
        for got, ref, ab, count, what in zip((y, dx, dw, db), want, terms, (k + 1, n, 131, 131), ('y', 'dx', 'dw', 'db')):
            _close(got, ref, ab, count, dtype, what)
        assert not y[live:].any() and not dx[live:].any()
    out = torch.full((t, n + 3), 5.0, dtype=dtype, device='cuda')
    assert grouped.grouped_linear(xs, ws, ends, bias=b, out=out[:, 2:2 + n]).data_ptr() == out[:, 2:].data_ptr()
    _close(out[:live, 2:2 + n], want[0][:live], terms[0][:live], k + 1, dtype, 'out')
    assert (out[live:] == 5).all() and (out[:, :2] == 5).all() and (out[:, 2 + n:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('k,n', [(64, 768), (768, 64)])
def test_more_groups_than_lanes_with_whole_and_partial_tiles_and_a_tail(k, n, dtype):
    """70 groups of one to three whole tiles and a rest of any size, empty ones between, rows of no group behind them."""
    sizes, tail = [0 if i % 17 == 5 else 256 * (1 + i % 3) + i * 29 % 256 for i in range(70)], 300
    x, w, b, grad, ends = _case(sizes, k, n, dtype, tail=tail)
    live = sum(sizes)
    y = grouped.grouped_linear(x, w, ends, bias=b, relu=True)
    got = (y,) + grouped.grouped_linear_backward(grad, x, w, ends, y=y)
    want, terms = _reference(x, w, b, grad, sizes, True, y)
    for o, ref, ab, count, what in zip(got, want, terms, (k + 1, n, max(sizes), max(sizes)), ('y', 'dx', 'dw', 'db')):
        _close(o, ref, ab, count, dtype, what)
    assert not y[live:].any() and not got[1][live:].any()
    out = torch.full((live + tail, n), 5.0, dtype=dtype, device='cuda')
    grouped.grouped_linear(x, w, ends, bias=b, relu=True, out=out)
    assert torch.equal(out[:live], y[:live]) and (out[live:] == 5).all()


@pytest.mark.gpu
def test_ends_outside_the_rows_are_clamped():
    """Running maximum, clamped to [0, rows]: decreasing, negative and far too large entries touch nothing they should not."""
    x, w, b, grad, _ = _case([50, 30, 20, 10], 24, 40, torch.float32)
    ends = torch.tensor([-7, 60, 40, 1 << 30], dtype=torch.int32, device='cuda')
    sizes = [0, 60, 0, 50]
    y = grouped.grouped_linear(x, w, ends, bias=b)
    got = (y,) + grouped.grouped_linear_backward(grad, x, w, ends)
    want, terms = _reference(x, w, b, grad, sizes, False)
    for o, ref, ab, count, what in zip(got, want, terms, (25, 40, 60, 60), ('y', 'dx', 'dw', 'db')):
        _close(o, ref, ab, count, torch.float32, what)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
def test_infinities_and_nan_stay_in_their_rows(dtype):
    sizes, k, n = [40, 33], 70, 50
    x, w, b, grad, ends = _case(sizes, k, n, dtype)
    clean = grouped.grouped_linear(x, w, ends, bias=b, relu=True)
    x[39, 69], x[40, 0] = float('inf'), float('nan')                # the last row of group 0, the first of group 1
    y = grouped.grouped_linear(x, w, ends, bias=b, relu=True)
    rest = [i for i in range(73) if i not in (39, 40)]
    assert torch.equal(y[rest], clean[rest])
    assert y[40].isnan().all()                                      # relu keeps NaN
    plus = w[0, :, 69] > 0
    assert (y[39][plus] == float('inf')).all() and (y[39][~plus] == 0).all()
    dx, dw, db = grouped.grouped_linear_backward(grad, x, w, ends, y=y)
    assert torch.isfinite(dx).all() and torch.isfinite(dw[0][:, :69]).all() and torch.isfinite(db).all()
    assert dw[1][:, 0].isnan().all() and torch.isfinite(dw[1][:, 1:]).all()


@pytest.mark.gpu
def test_autograd_matches_the_formula_and_differences():
    sizes, k, n = [9, 0, 14], 6, 7
    x, w, b, grad, ends = _case(sizes, k, n, torch.float32)
    for t in (x, w, b):
        t.requires_grad_()
    y = grouped.grouped_linear(x, w, ends, bias=b, relu=True)
    (y * grad).sum().backward()
    plain = grouped.grouped_linear_backward(grad, x.detach(), w.detach(), ends, y=y.detach())
    for t, p in zip((x, w, b), plain):
        assert torch.equal(t.grad, p)

    def loss(xx, ww, bb):                                           # the formula in 64 bits
        return float((_reference(xx, ww, bb, grad, sizes, True)[0][0] * grad.double()).sum())
    h = 1e-6
    for pos, (t, gr) in enumerate(((x, x.grad), (w, w.grad), (b, b.grad))):
        flat, r = t.detach().double().flatten(), torch.Generator().manual_seed(pos)
        for i in torch.randperm(flat.numel(), generator=r)[:12].tolist():
            args = [x.detach().double(), w.detach().double(), b.detach().double()]
            up, dn = flat.clone(), flat.clone()
            up[i] += h
            dn[i] -= h
            args[pos] = up.view(t.shape)
            hi = loss(*args)
            args[pos] = dn.view(t.shape)
            lo = loss(*args)
            # central difference of a piecewise linear function, 64 bits: rounding ~1e-15 / h; the f32 gradient: < 1e-5
            assert abs((hi - lo) / (2 * h) - float(gr.flatten()[i])) < 2e-5, (pos, i)
    only_w = torch.autograd.grad(grouped.grouped_linear(x.detach(), w, ends).sum(), w)[0]
    assert only_w.shape == w.shape
    with pytest.raises(RuntimeError):                               # out= has no gradient
        grouped.grouped_linear(x, w, ends, out=torch.empty(23, n, device='cuda'))


@pytest.mark.gpu
def test_expanded_gradient_and_shared_weight():
    """``sum().backward()`` hands a stride-0 gradient; one weight shared by every group gets the sum of their gradients."""
    sizes, k, n = [5, 8], 6, 4
    x, w, b, _, ends = _case(sizes, k, n, torch.float32)
    shared = w[:1].clone().requires_grad_()
    grouped.grouped_linear(x, shared.expand(2, n, k), ends).sum().backward()
    want = x.double().sum(0).expand(n, k)
    assert (shared.grad[0].double() - want).abs().max() < 13 * 2.0 ** -22 * x.double().abs().sum(0).max()


@pytest.mark.gpu
def test_results_repeat_and_follow_a_graph():
    """The same bits on every call, eager or replayed; a replay reads what `ends` and the arrays hold then; another stream."""
    sizes, k, n = [300, 500, 200], 96, 80
    x, w, b, grad, ends = _case(sizes, k, n, torch.float32)

    def both():
        y = grouped.grouped_linear(x, w, ends, bias=b, relu=True)
        return (y,) + grouped.grouped_linear_backward(grad, x, w, ends, y=y)
    eager = [t.clone() for t in both()]
    assert all(torch.equal(a, c) for a, c in zip(eager, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(eager, other))
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):                                              # two graphs: each has its own scratch memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode='thread_local'):
            out = both()
        graphs.append((g, out))
    for step in range(3):
        ends.copy_(grouped.group_ends([[300, 500, 200], [0, 700, 300], [1000, 0, 0]][step]))
        x.mul_(1.25)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        want = both()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want)), step


@pytest.mark.gpu
def test_arguments_are_checked():
    x, w, b, grad, ends = _case([3, 4], 6, 5, torch.float32)
    ok = dict(x=x, weight=w, ends=ends, bias=b)
    bad = [dict(x=x.double()), dict(x=x.half()), dict(x=x[:, :5]), dict(x=x[0]), dict(weight=w[0]), dict(weight=w.bfloat16()),
           dict(bias=b[:, :4]), dict(bias=b.half()), dict(bias=b.cpu()), dict(ends=ends[:1]), dict(ends=ends.float()),
           dict(ends=ends.cpu()), dict(ends=[3, 7]), dict(weight=w[:, :0]), dict(weight=w[:, :, :0], x=x[:, :0]),
           dict(weight=w.expand(2, 5, 6)[:0], bias=None, ends=ends[:0]), dict(out=x), dict(out=torch.empty(7, 4, device='cuda')),
           dict(out=torch.empty(7, 5, device='cuda').half()), dict(out=torch.empty(5, 7, device='cuda').t())]
    for change in bad:
        with pytest.raises((TypeError, ValueError)):
            grouped.grouped_linear(**dict(ok, **change))
    sq = torch.zeros(7, 7, device='cuda')
    with pytest.raises(ValueError):                                 # the result would overwrite what it reads
        grouped.grouped_linear(sq[:, :6], w, ends, out=sq[:, 2:])
    for kw in (dict(grad=grad[:, :4]), dict(grad=grad.half()), dict(y=grad[:3])):
        with pytest.raises(ValueError):
            grouped.grouped_linear_backward(**dict(dict(grad=grad, x=x, weight=w, ends=ends), **kw))
    empty = grouped.grouped_linear(x[:0], w, ends, bias=b)
    assert empty.shape == (0, 5)
    dx, dw, db = grouped.grouped_linear_backward(grad[:0], x[:0], w, ends)
    assert dx.shape == (0, 6) and not dw.any() and not db.any()
    dx, dw, db = grouped.grouped_linear_backward(grad, x, w, ends, need_dx=False, need_dbias=False)
    assert dx is None and db is None and dw.shape == w.shape


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('at', [0, 1, 2, 3])
def test_every_alignment_of_odd_widths_and_the_arrays_last_elements(dtype, at):
    """Odd and even widths at every 2-byte place; the arrays end where their memory's used part does (NaN behind and before),
    and the last element of each counts."""
    for sizes, k, n in (([7, 66], 9, 11), ([130, 1], 65, 67), ([5, 60], 71, 130), ([3], 1, 1), ([64, 3], 130, 5), ([300, 2], 129, 131)):
        x, w, b, grad, ends = _case(sizes, k, n, dtype, seed=at)

        def place(t):
            flat = torch.full((t.numel() + at + 64,), float('nan'), dtype=dtype, device='cuda')
            return flat[at:at + t.numel()].view(t.shape).copy_(t)
        x, w, b, grad = (place(t) for t in (x, w, b, grad))
        for t in (x, w, grad):
            t.view(-1)[-1] = 30.0
        y = grouped.grouped_linear(x, w, ends, bias=b)
        got = (y,) + grouped.grouped_linear_backward(grad, x, w, ends)
        want, terms = _reference(x, w, b, grad, sizes, False)
        most = max(sizes)
        for o, ref, ab, count, what in zip(got, want, terms, (k + 1, n, most, most), ('y', 'dx', 'dw', 'db')):
            _close(o, ref, ab, count, dtype, (what, sizes, k, n))
        relu = place(torch.randn(grad.shape, device='cuda').to(dtype))
        got = grouped.grouped_linear_backward(grad, x, w, ends, y=relu)
        want, terms = _reference(x, w, b, grad, sizes, False, relu)
        for o, ref, ab, count, what in zip(got, want[1:], terms[1:], (n, most, most), ('dx', 'dw', 'db')):
            _close(o, ref, ab, count, dtype, (what, sizes, k, n, 'masked'))


@pytest.mark.gpu
def test_rows_that_lie_far_apart_are_packed_first():
    """A row stride beyond what a tile's copies reach (2^23 bytes): the same result as from adjacent rows."""
    sizes, k, n = [3, 4], 70, 40
    x, w, b, grad, ends = _case(sizes, k, n, torch.float32)
    far = torch.zeros(7 << 21, device='cuda').view(7, 1 << 21)
    xs, gs = far[:, 5:5 + k], far[:, 1000:1000 + n]
    xs.copy_(x)
    gs.copy_(grad)
    assert torch.equal(grouped.grouped_linear(xs, w, ends, bias=b), grouped.grouped_linear(x, w, ends, bias=b))
    for got, want in zip(grouped.grouped_linear_backward(gs, xs, w, ends), grouped.grouped_linear_backward(grad, x, w, ends)):
        assert torch.equal(got, want)
    y = torch.randn(7, n, device='cuda')
    ys, near = far[:, 9000:9000 + n], torch.full((7, n + 5), float('nan'), device='cuda')[:, 2:2 + n]
    ys.copy_(y)
    near.copy_(y)
    plain = grouped.grouped_linear_backward(grad, x, w, ends, y=y)      # masked as they are read: y with strides of its own
    for gg, yy in ((grad, near), (grad, ys), (gs, y), (gs, ys)):
        for got, want in zip(grouped.grouped_linear_backward(gg, xs, w, ends, y=yy), plain):
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31 (x) and 2^32 bytes: the last rows equal those of a call of their own."""
    t, k, n = (1 << 20) + 77, 2080, 8
    x = torch.zeros(t, k, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(1)
    x[-300:] = torch.randn(300, k, generator=g, device='cuda').bfloat16()
    w = torch.randn(2, n, k, generator=g, device='cuda').bfloat16()
    ends = torch.tensor([t - 200, t], dtype=torch.int64, device='cuda')
    y = grouped.grouped_linear(x, w, ends)
    small = grouped.grouped_linear(x[-300:], w, ends - (t - 300))
    assert torch.equal(y[-300:], small) and not y[:-300].any()
    grad = torch.zeros(t, n, dtype=torch.bfloat16, device='cuda')
    grad[-300:] = torch.randn(300, n, generator=g, device='cuda').bfloat16()
    dx, dw, db = grouped.grouped_linear_backward(grad, x, w, ends)
    sx, sw, sb = grouped.grouped_linear_backward(grad[-300:], x[-300:], w, ends - (t - 300))
    assert torch.equal(dx[-300:], sx) and not dx[:-300].any()
    want, terms = _reference(x[-300:], w, torch.zeros(2, n, device='cuda'), grad[-300:], [100, 200], False)
    for got, ref, ab, what in ((dw, want[2], terms[2], 'dw'), (db, want[3], terms[3], 'db')):
        _close(got, ref, ab, 200, torch.bfloat16, what)


def _same(got, want, terms, count, dtype, what):
    """Where the definition in 64 bits gives an infinity or NaN the result is the same, elsewhere it is close."""
    odd = ~torch.isfinite(want)
    assert torch.equal(got.double()[odd].nan_to_num(0.5), want[odd].nan_to_num(0.5)), what
    _close(torch.where(odd, 0, got), torch.where(odd, 0, want), torch.where(odd, 0, terms), count, dtype, what)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('sizes,k,n', [([40, 33], 71, 51), ([3], 1, 1), ([5, 60], 70, 131), ([64, 3], 131, 8), ([600, 505], 301, 67),
                                       ([300, 200, 100, 500], 1025, 1025), ([4000, 4192], 131, 1025), ([2000, 2100], 1025, 131)])
def test_infinities_opposite_an_arrays_last_element(sizes, k, n, dtype):
    """Odd widths, every tile: an infinity that meets x's, dy's or weight's last element in forward, dx or dweight gives what
    the sum gives, plus or minus infinity, and relu turns the latter into zero."""
    t, last = sum(sizes), len(sizes) - 1
    for case in range(5):
        x, w, b, grad, ends = _case(sizes, k, n, dtype, seed=case)
        if n > 1 or case == 2:
            r = t - 1 - (case + 1) % min(3, sizes[-1])
            if case == 0:
                x[r, k - 1] = float('inf')                           # forward: opposite weight's last
            elif case == 1:
                w[last, n // 2, k - 1] = float('-inf')               # forward: opposite x's last (and of weight's last column)
            elif case == 2:
                w[last, n - 1, k // 2] = float('inf')                # dx: opposite dy's last
            elif case == 3:
                grad[r, n - 1] = float('-inf')                       # dx: opposite weight's last; dweight
                grad[t - 1, 0] = float('inf')                        # dweight: opposite x's last
            else:
                x[t - 1, 0] = float('inf')                           # dweight: opposite dy's last
        y_saved = torch.randn(t, n, generator=torch.Generator().manual_seed(case)).to(dtype).cuda()
        for y in (None, y_saved):
            got = (grouped.grouped_linear(x, w, ends, bias=b, relu=y is not None),) + grouped.grouped_linear_backward(grad, x, w, ends, y=y)
            want, terms = _reference_with_infinities(x, w, b, grad, sizes, y)
            most = max(sizes)
            for o, ref, ab, count, what in zip(got, want, terms, (k + 1, n, most, most), ('y', 'dx', 'dw', 'db')):
                _same(o, ref, ab, count, dtype, (what, case, y is None))


def _reference_with_infinities(x, w, b, grad, sizes, y_saved):
    """``_reference`` with a gradient that is selected, not multiplied, by the mask, and a relu that keeps NaN; products on the
    CPU, plain sums of products."""
    x, w, b, grad = (t.double().cpu() for t in (x, w, b, grad))
    if y_saved is not None:
        grad = torch.where(y_saved.cpu() <= 0, 0.0, grad)
    (y, dx, dw, db), terms = _reference(x, w, b, grad, sizes, False)
    if y_saved is not None:
        y = torch.where(y < 0, 0.0, y)
    return [t.cuda() for t in (y, dx, dw, db)], [t.cuda() for t in terms]


@pytest.mark.gpu
def test_autograd_notices_a_write_to_out():
    """A buffer that autograd saved and a later call overwrites raises in the backward pass; an ``out`` that requires grad is
    refused, outside ``no_grad``."""
    x, w, b, grad, ends = _case([3, 4], 6, 5, torch.float32)
    out = torch.zeros(7, 5, device='cuda')
    scale = torch.ones(7, 5, device='cuda', requires_grad=True)
    loss = (out * scale).sum()                                      # saves out
    assert grouped.grouped_linear(x, w, ends, bias=b, out=out) is out
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    grows = torch.zeros(7, 5, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='automatic differentiation'):
        grouped.grouped_linear(x, w, ends, bias=b, out=grows)
    assert not grows.any()
    with torch.no_grad():
        grouped.grouped_linear(x, w, ends, bias=b, out=grows)
    with torch.inference_mode():
        again = grouped.grouped_linear(x, w, ends, bias=b, out=torch.empty(7, 5, device='cuda'))
    assert torch.equal(grows, out) and torch.equal(again, out)


@pytest.mark.parametrize('dtype,size', [(_hip.F32, 4), (_hip.BF16, 2), (_hip.F16, 2)])
def test_what_is_packed_into_scratch(dtype, size):
    """Rows that lie further apart than 2^23 bytes less 100, and nothing else: the widest weight is read where it lies."""
    L, p, far = _hip.lib, 1 << 20, (1 << 23) // size
    d, wide = _desc(dtype=dtype), _desc(dtype=dtype, n=2047, k=1 << 20, groups=4)
    for ld, packed in ((3, False), (far - 100, False), (far, True)):
        assert (L.mpe_grouped_linear_workspace(d, p, ld, p) > 0) == packed
        assert (L.mpe_grouped_backward_workspace(d, p, 5, None, 0, p, ld, p, 1, 1) > 0) == packed
        assert (L.mpe_grouped_backward_workspace(d, p, ld + 5, None, 0, p, 3, p, 1, 0) > 0) == packed
        assert (L.mpe_grouped_backward_workspace(d, p, 5, p, ld + 5, p, 3, p, 1, 0) > 0) == packed
        assert L.mpe_grouped_backward_workspace(d, p, 5, None, 0, p, ld, p, 1, 0) == 0       # x is not read
    assert L.mpe_grouped_linear_workspace(wide, p, 1 << 20, p) == 0
    assert L.mpe_grouped_backward_workspace(wide, p, 2047, None, 0, p, 1 << 20, p, 1, 0) == 0


@pytest.mark.parametrize('version,says', [(_hip.ABI_VERSION, 'lacks a function'), (_hip.ABI_VERSION - 1, 'ABI %d != expected' % (_hip.ABI_VERSION - 1))])
def test_an_older_library_is_refused_in_words(version, says, tmp_path):
    """One of the same ABI without the later functions, and one of an older ABI, which is told first."""
    import os
    import shutil
    import subprocess
    import sys
    if shutil.which('gcc') is None:
        pytest.skip('no C compiler')
    (tmp_path / 'old.c').write_text('int mpe_abi_version(void) { return %d; }' % version)
    subprocess.run(['gcc', '-shared', '-fPIC', '-o', str(tmp_path / 'old.so'), str(tmp_path / 'old.c')], check=True)
    root = os.path.dirname(os.path.dirname(os.path.abspath(_hip.__file__)))
    run = subprocess.run([sys.executable, '-c', 'import marl_amd._hip'], cwd=root, capture_output=True, text=True,
                         env=dict(os.environ, MARL_AMD_LIB=str(tmp_path / 'old.so')))
    assert run.returncode == 1 and 'ImportError' in run.stderr and says in run.stderr
