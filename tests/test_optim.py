"""marl_amd.optim.AdamW: one step over many tensors against the formulas in 64 bits, and its 8-bit moments against a
restatement in numpy's float32, bit for bit."""
import copy
import ctypes as C
import math
import pickle

import numpy as np
import pytest
import torch

from marl_amd import _hip, optim

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ---- refusals (no GPU needed) --------------------------------------------------------------------------------------------
def test_cpu_parameters_and_bad_settings_are_refused():
    with pytest.raises(RuntimeError):
        optim.AdamW([torch.zeros(3)])
    with pytest.raises(ValueError):
        optim.AdamW([torch.zeros(3)], state_bits=16)
    with pytest.raises(ValueError):
        optim.AdamW([])
    with pytest.raises(ValueError):
        optim.dequantize(torch.zeros(128), torch.zeros(1, dtype=torch.int16), True)
    with pytest.raises(RuntimeError):
        optim.dequantize(torch.zeros(128, dtype=torch.uint8), torch.zeros(1, dtype=torch.int16), True)


def _args(**kw):
    d = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, max_norm=0.0, polyak=0.99, step=1, dtype=_hip.F32,
             state_bits=32)
    d.update(kw)
    return _hip.AdamArgs(**d)


def _table(**kw):
    p = 1 << 20
    d = dict(param=p, exp_avg=p, exp_avg_sq=p, exp_avg_base=p, exp_avg_sq_base=p, count=300)
    d.update(kw)
    return (_hip.AdamTensor * 1)(_hip.AdamTensor(**d))


def test_c_abi_refuses_bad_arguments():
    """Nothing is launched: the pointers are never read."""
    L, p, inf, nan = _hip.lib, 1 << 20, float('inf'), float('nan')
    assert L.mpe_adamw_plan(1, _table(count=1 << 37), _hip.F32, 32, None, 0) == -6     # more work items than a launch may have
    assert L.mpe_adamw_moments(p, p, p, p, p, p, 1 << 36, _hip.F32, None) == -6
    grads = (C.c_void_p * 1)(p)
    for change, code in ((dict(lr=-1.0), -6), (dict(lr=nan), -6), (dict(lr=inf), -6), (dict(beta1=1.0), -6), (dict(beta2=-0.1), -6),
                         (dict(eps=-1.0), -6), (dict(eps=nan), -6), (dict(weight_decay=-1.0), -6), (dict(polyak=1.1), -6),
                         (dict(max_norm=-1.0), -6), (dict(max_norm=inf), -6), (dict(step=0), -6), (dict(dtype=7), -5),
                         (dict(state_bits=16), -5), (dict(clock=p + 4, step=0), -4)):
        assert L.mpe_adamw_step(_args(**change), 1, _table(), p, grads, None) == code, change
    for change, code in ((dict(param=None), -1), (dict(exp_avg=None), -1), (dict(exp_avg_sq=None), -1), (dict(count=-1), -6),
                         (dict(param=p + 2), -4), (dict(target=p + 1), -4), (dict(exp_avg=p + 4), -4), (dict(exp_avg_sq=p + 8), -4)):
        assert L.mpe_adamw_step(_args(), 1, _table(**change), p, grads, None) == code, change
        assert L.mpe_adamw_plan(1, _table(**change), _hip.F32, 32, None, 0) == code, change
    assert L.mpe_adamw_step(_args(state_bits=8), 1, _table(exp_avg_base=None), p, grads, None) == -1
    assert L.mpe_adamw_step(_args(state_bits=8), 1, _table(exp_avg_sq_base=p + 1), p, grads, None) == -4
    assert L.mpe_adamw_step(_args(), 1, _table(), p, (C.c_void_p * 1)(p + 2), None) == -4
    assert L.mpe_adamw_step(_args(), 1, _table(), p + 4, grads, None) == -4
    assert L.mpe_adamw_step(None, 1, _table(), p, grads, None) == -1
    assert L.mpe_adamw_step(_args(), 1, _table(), None, grads, None) == -1
    assert L.mpe_adamw_step(_args(), 1, None, p, grads, None) == -1
    assert L.mpe_adamw_step(_args(), 1, _table(), p, None, None) == -1
    assert L.mpe_adamw_step(_args(), 0, _table(), p, grads, None) == -6
    need = L.mpe_adamw_plan(1, _table(), _hip.F32, 32, None, 0)
    blob = torch.empty(need, dtype=torch.uint8)
    assert need > 0 and L.mpe_adamw_plan(1, _table(), _hip.F32, 32, blob.data_ptr(), need) == need
    assert L.mpe_adamw_plan(1, _table(), _hip.F32, 32, blob.data_ptr(), need - 1) == -7
    for count in (100, -128):
        assert L.mpe_adamw_moments(p, p, p, p, p, p, count, 0, None) == -6
    assert L.mpe_adamw_moments(p, p, p, p, p, p, 128, 2, None) == -5
    for bad in ((None, p, p, p, p, p), (p, None, p, p, p, p), (p, p, None, p, p, p), (p, p, p, None, p, p), (p, p, p, p, None, None)):
        assert L.mpe_adamw_moments(*bad, 128, 0, None) == -1
    for bad in ((p + 4, p, p, p, p, p), (p, p + 1, p, p, p, p), (p, p, p + 4, p, p, p), (p, p, p, p, p + 2, p), (p, p, p, p, p, p + 1)):
        assert L.mpe_adamw_moments(*bad, 128, 0, None) == -4
    assert C.sizeof(_hip.AdamTensor) == 56 and C.sizeof(_hip.AdamArgs) == 96


# ---- the 8-bit moments in numpy ------------------------------------------------------------------------------------------
def _mix(h):
    h = h ^ (h >> np.uint32(16))
    h = h * np.uint32(0x85EBCA6B)
    h = h ^ (h >> np.uint32(13))
    h = h * np.uint32(0xC2B2AE35)
    return h ^ (h >> np.uint32(16))


def _random_bits(seed, step, tensor, index):
    with np.errstate(over='ignore'):
        k = _mix(np.array([(seed + step * 0x9E3779B9) & 0xFFFFFFFF], dtype=np.uint32)) ^ np.uint32(seed >> 32)
        k = _mix(k + np.uint32((tensor * 0x85EBCA77) & 0xFFFFFFFF))
        return _mix(index.astype(np.uint32) ^ (k + (index >> 32).astype(np.uint32) * np.uint32(0x9E3779B1)))


def _encode(x, rnd, signed):
    top = 127 if signed else 255
    pad = -x.size % 128
    bits = np.pad(x.view(np.uint32) & np.uint32(0x7FFFFFFF), (0, pad)).astype(np.int64)
    neg = np.pad(x.view(np.uint32) >> np.uint32(31), (0, pad)).astype(np.int64)
    rnd = np.pad(rnd.astype(np.int64), (0, pad))
    base = np.maximum((bits.reshape(-1, 128).max(1) >> 20) + 1 - top, 0)
    code = np.maximum((np.minimum(bits + rnd, 0x7FFFFFFF) >> 20) - np.repeat(base, 128), 0)
    code = code | neg << 7 if signed else np.maximum(code, bits > 0)
    return code[:x.size].astype(np.uint8), base.astype(np.int16)


def _decode(code, base, signed):
    mag = (code & 127 if signed else code).astype(np.int64)
    b = np.repeat(base.astype(np.int64), 128)[:code.size]
    x = np.where(mag > 0, (mag + b) << 20, 0).astype(np.uint32).view(np.float32)
    return np.where(code > 127, -x, x).astype(np.float32) if signed else x


def _step8(code_m, base_m, code_v, base_v, g, scale, step, seed, tensor, index, b1=0.9, b2=0.999):
    f = np.float32
    gc = g * f(scale)
    m = _decode(code_m, base_m, True) * f(b1) + gc * f(1 - b1)
    v = _decode(code_v, base_v, False) * f(b2) + (gc * gc) * f(1 - b2)
    r = _random_bits(seed, step, tensor, index)
    return _encode(m, (r >> np.uint32(16)) << np.uint32(4), True) + _encode(v, (r & np.uint32(0xFFFF)) << np.uint32(4), False) + (m, v)


def test_the_restated_code_holds_what_the_text_says():
    """Every code's value survives the round trip; rounding errs by less than an eighth of a binade, zero on average."""
    r = np.random.RandomState(0)
    x = (r.standard_normal(128 * 64) * np.exp(r.standard_normal(128 * 64))).astype(np.float32)
    rnd = r.randint(0, 1 << 16, x.size).astype(np.uint32) << np.uint32(4)
    for signed, y in ((True, x), (False, x * x)):
        code, base = _encode(y, rnd, signed)
        held = _decode(code, base, signed)
        big = np.abs(y) > np.repeat(np.abs(y).reshape(-1, 128).max(1), 128) * 2.0 ** -14
        assert (np.abs(held - y)[big] <= np.abs(y)[big] / 8).all()
        # mean error of n roundings, each below 1/8 with zero mean: 5 sigma of a uniform-like error
        assert abs(float(np.mean((held - y)[big] / y[big]))) < 5 * 0.125 / math.sqrt(int(big.sum()))
        again, base2 = _encode(held, np.zeros_like(rnd), signed)
        assert np.array_equal(_decode(again, base2, signed)[big], held[big])
    code, base = _encode(np.array([1.0, 1e-20, 0.0], dtype=np.float32), np.zeros(3, np.uint32), False)
    assert code.tolist()[1:] == [1, 0]                                 # v > 0 is never held as zero


# ---- steps against 64 bits -----------------------------------------------------------------------------------------------
SIZES = [(1,), (7,), (128,), (129, 3), (64, 64), (5,), (8192,), (8193,), (0,), (300, 100), (64,), (31, 17)]


def _tensors(sizes, dtype, seed, scale=1.0, offset=0):
    """Tensors in one array, ``offset`` elements apart: bases of every alignment."""
    g = torch.Generator().manual_seed(seed)
    out, flat = [], torch.zeros(sum(math.prod(s) + offset for s in sizes) + offset, dtype=dtype, device='cuda')
    at = offset
    for s in sizes:
        c = math.prod(s)
        t = flat[at:at + c].view(s)
        t.copy_(torch.randn(s, generator=g) * scale)
        out.append(t)
        at += c + offset
    return out


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16], ids=['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('clip,target,offset', [(None, False, 0), (0.5, True, 1), (3.0, False, 3), (None, True, 5)])
def test_steps_follow_the_formulas(bits, dtype, clip, target, offset):
    """Three steps.  32 bits: m and v to 4 roundings of f32; the parameter to its own rounding and those of the step.
    8 bits: the codes equal numpy's float32 restatement; the parameter follows from the moments before they are rounded."""
    lr, b1, b2, eps, wd, rho, seed = 1e-2, 0.9, 0.999, 1e-8, 0.1, 0.9, (5 << 32) + 77
    ps = _tensors(SIZES, dtype, 1, 0.3, offset)
    ts = _tensors(SIZES, dtype, 2, 0.3, offset) if target else None
    opt = optim.AdamW(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, max_norm=clip, targets=ts,
                      polyak=rho, seed=seed)
    e, h = 2.0 ** -24, HALF[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0               # half a step under f16's normal range
    for step in range(1, 4):
        gs = _tensors(SIZES, dtype, 10 + step, 0.05, offset)
        before = [(p.double().flatten(), None if not target else t.double().flatten(), {k: v.clone() for k, v in opt.state[p].items()})
                  for p, t in zip(ps, ts or ps)]
        for p, g in zip(ps, gs):
            p.grad = g
        opt.step()
        assert opt.step_count == step
        for j, (p, g, (p0, t0, st)) in enumerate(zip(ps, gs, before)):
            if p.numel() == 0:
                continue
            gd = g.double().flatten()
            norm = float(gd.norm())
            s32 = np.float32(clip) / max(np.float32(norm), np.float32(clip)) if clip else np.float32(1)
            gc = gd * float(s32)
            if bits == 32:
                m0, v0 = st['exp_avg'].double().flatten(), st['exp_avg_sq'].double().flatten()
            else:
                cm, bm, cv, bv = (st[k].cpu().numpy().ravel() for k in ('exp_avg', 'exp_avg_base', 'exp_avg_sq', 'exp_avg_sq_base'))
                want = _step8(cm, bm, cv, bv, g.float().flatten().cpu().numpy(), s32, step, seed, j, np.arange(p.numel()))
                for k, w in zip(('exp_avg', 'exp_avg_base', 'exp_avg_sq', 'exp_avg_sq_base'), want):
                    assert np.array_equal(opt.state[p][k].cpu().numpy().ravel(), w), (j, k)
                m0 = torch.from_numpy(_decode(cm, bm, True)).double().cuda()
                v0 = torch.from_numpy(_decode(cv, bv, False)).double().cuda()
            m, v = b1 * m0 + (1 - b1) * gc, b2 * v0 + (1 - b2) * gc * gc
            dm = 4 * e * (b1 * m0.abs() + (1 - b1) * gc.abs())       # g scale, two products, one sum, the factors' own rounding
            dv = 6 * e * v
            if bits == 32:
                assert bool(((opt.state[p]['exp_avg'].double().flatten() - m).abs() <= dm + 1e-44).all())
                assert bool(((opt.state[p]['exp_avg_sq'].double().flatten() - v).abs() <= dv + 1e-44).all())
            denom = (v / (1 - b2 ** step)).sqrt() + eps
            upd = lr / (1 - b1 ** step) * m / denom
            pn = p0 * (1 - lr * wd) - upd
            # m off by dm, denom by half of v's error and its own four roundings; quotient, two products, one sum
            dp = lr / (1 - b1 ** step) * dm / denom + 12 * e * upd.abs() + 3 * e * p0.abs()
            tol = dp + h * (pn.abs() + dp) * (1 + 1e-3) + tiny
            assert bool(((p.double().flatten() - pn).abs() <= tol).all()), (j, step)
            if target:
                tn = rho * t0 + (1 - rho) * p.double().flatten()
                tol = 4 * e * (t0.abs() + p.double().flatten().abs()) + h * tn.abs() * (1 + 1e-3) + tiny
                assert bool(((ts[j].double().flatten() - tn).abs() <= tol).all()), (j, step)
    if offset:                                                         # what lies between the tensors is still zero
        flat = ps[0]._base
        used = torch.zeros(flat.numel(), dtype=torch.bool, device='cuda')
        for p in ps:
            o = (p.data_ptr() - flat.data_ptr()) // p.element_size()
            used[o:o + p.numel()] = True
        assert not flat[~used].any()


@pytest.mark.gpu
def test_one_step_matches_torch_adam_at_zero_decay():
    """weight_decay = 0: the learner's Adam (torch's, whose eps stands outside the corrected root as here)."""
    torch.manual_seed(0)
    a = [torch.randn(s, device='cuda') for s in SIZES]
    b = [t.clone() for t in a]
    for x in a + b:
        x.requires_grad_()
    mine, ref = optim.AdamW(a, lr=1e-2, weight_decay=0.0), torch.optim.Adam(b, lr=1e-2)
    for k in range(5):
        for x, y in zip(a, b):
            x.grad = torch.randn(x.shape, device='cuda')
            y.grad = x.grad.clone()
        mine.step()
        ref.step()
    for x, y in zip(a, b):                                             # five steps of at most ~1e-2, each to a few 2^-24
        assert torch.allclose(x, y, rtol=1e-6, atol=5 * 1e-2 * 20 * 2.0 ** -24)


@pytest.mark.gpu
def test_more_tensors_than_one_launch_holds_and_missing_gradients():
    """1 000 variables (three launches), every third without a gradient: value and moments stay, the target still follows."""
    sizes = [(1 + (i * 37) % 300,) for i in range(999)] + [(20000,)]
    ps, ts = _tensors(sizes, torch.float32, 1), _tensors(sizes, torch.float32, 2)
    gs = _tensors(sizes, torch.float32, 3)
    p0, t0 = [p.clone() for p in ps], [t.clone() for t in ts]
    opt = optim.AdamW(ps, lr=0.1, weight_decay=0.0, max_norm=0.5, targets=ts, polyak=0.75)
    for i, (p, g) in enumerate(zip(ps, gs)):
        p.grad = g if i % 3 else None
    opt.step()
    for i, p in enumerate(ps):
        if i % 3 == 0:
            assert torch.equal(p, p0[i]) and not opt.state[p]['exp_avg'].any()
        else:                   # the first step: m / (1 - b1) = g', sqrt(v / (1 - b2)) = |g'|, so lr g' / (|g'| + eps): with
            live = gs[i].abs() > 1e-3                                 # 20 000 elements clipped to 0.5, |g'| is down to 3.5e-6
            gc = gs[i].double() * (0.5 / max(0.5, float(gs[i].double().norm())))
            assert torch.allclose((p0[i] - p)[live].double(), (0.1 * gc / (gc.abs() + 1e-8))[live], rtol=1e-5, atol=1e-6)
        assert torch.allclose(ts[i], 0.75 * t0[i] + 0.25 * p, rtol=1e-6, atol=1e-6)


@pytest.mark.gpu
def test_eight_bit_moments_are_right_on_average():
    """1 500 steps of unit normal gradients: the mean of the held v over 16 384 elements follows the exact average.  One
    element's v walks by 25 % (an eighth of a binade with probability 0.8 % a step, forgotten at 0.1 % a step); the mean
    over 16 384 of them by 0.2 %, ten times which is allowed."""
    p = torch.zeros(16384, device='cuda')
    opt = optim.AdamW([p], lr=0.0, state_bits=8, seed=3)
    g = torch.Generator(device='cuda').manual_seed(0)
    v = torch.zeros(16384, device='cuda', dtype=torch.float64)
    m = torch.zeros_like(v)
    for _ in range(1500):
        p.grad = torch.randn(16384, generator=g, device='cuda')
        opt.step()
        v = 0.999 * v + 0.001 * p.grad.double() ** 2
        m = 0.9 * m + 0.1 * p.grad.double()
    hm, hv = opt.moments()[0]
    assert abs(float(hv.double().mean() / v.mean()) - 1) < 0.02
    # m: rounding noise of at most 1/8 of |m| a step, remembered 5 steps (variance 1 / (1 - 0.81)), zero on average
    assert abs(float((hm.double() - m).mean())) < 10 * 0.125 * float(m.abs().mean()) * math.sqrt(5.3) / 128
    assert float((hm.double() - m).abs().mean()) < 0.3 * float(m.abs().mean())
    assert torch.equal(opt.moments(torch.bfloat16)[0][0].float(), hm)     # bfloat16 holds the values
    flat = opt.buffers()[0]
    assert torch.equal(optim.dequantize(flat['exp_avg'], flat['exp_avg_base'], True), hm)
    assert torch.equal(optim.dequantize(flat['exp_avg_sq'], flat['exp_avg_sq_base'], False, torch.bfloat16).float(), hv)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_captured_steps_equal_eager_steps(bits):
    """capturable: the step count lives on the device; replays between eager steps and other work, all equal to eager ones."""
    def make():
        ps, ts = _tensors(SIZES, torch.float32, 1), _tensors(SIZES, torch.float32, 2)
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, ts
    (pa, ta), (pb, tb) = make(), make()
    kw = dict(lr=1e-2, state_bits=bits, max_norm=0.5, seed=9)
    a, b = optim.AdamW(pa, targets=ta, **kw), optim.AdamW(pb, targets=tb, capturable=True, **kw)
    grads = [_tensors(SIZES, torch.float32, 20 + k) for k in range(5)]

    def load(ps, k):
        for p, g in zip(ps, grads[k]):
            p.grad.copy_(g)
    for k in range(2):
        load(pa, k)
        a.step()
    load(pb, 0)
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode='thread_local'):
        b.step()
    assert b.step_count == 1                                          # a recording executes nothing
    load(pb, 1)
    graph.replay()
    for k in range(2, 5):
        load(pa, k)
        a.step()
        load(pb, k)
        if k == 3:
            b.step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert a.step_count == b.step_count == k + 1
        for x, y in zip(pa + ta, pb + tb):
            # the device's pow and the host's may differ in a last place of 64 bits: one rounding of each factor
            assert torch.allclose(x, y, rtol=2.0 ** -21, atol=1e-2 * 2.0 ** -20)
        for x, y in zip(a.buffers()[0].values(), b.buffers()[0].values()):
            assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_state_dict_continues_a_run(bits):
    sizes = [(40, 9), (3,)]
    pa, pb = _tensors(sizes, torch.float32, 1), _tensors(sizes, torch.float32, 1)
    a = optim.AdamW([dict(params=pa[:1], lr=0.1), dict(params=pa[1:])], state_bits=bits, seed=4)

    def go(ps, opt, k):
        for p, g in zip(ps, _tensors(sizes, torch.float32, 30 + k)):
            p.grad = g
        opt.step()
    for k in range(3):
        go(pa, a, k)
    saved = a.state_dict()
    for x, y in zip(pb, pa):
        x.copy_(y)
    b = optim.AdamW([dict(params=pb[:1]), dict(params=pb[1:])], state_bits=bits, seed=4, capturable=bits == 8)
    held = b.buffers()[0]['exp_avg'].data_ptr()
    b.load_state_dict(saved)
    assert b.step_count == 3 and b.param_groups[0]['lr'] == 0.1 and b.buffers()[0]['exp_avg'].data_ptr() == held
    for k in range(3, 5):
        go(pa, a, k)
        go(pb, b, k)
    for x, y in zip(pa, pb):
        assert torch.allclose(x, y, rtol=2.0 ** -21, atol=1e-1 * 2.0 ** -20)
    for ga, gb in zip(a.buffers(), b.buffers()):
        assert all(torch.equal(ga[k], gb[k]) for k in ga)
    for bad in (optim.AdamW(pb, state_bits=bits), optim.AdamW([dict(params=pb[:1]), dict(params=pb[1:])], state_bits=40 - bits)):
        with pytest.raises(ValueError):
            bad.load_state_dict(saved)


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_values_that_are_not_finite(bits):
    """An infinite or NaN gradient reaches its element (8 bits: its block of 128) and nothing else; with a clip its variable."""
    sizes = [(400,), (300,)]
    ps = _tensors(sizes, torch.float32, 1)
    gs = _tensors(sizes, torch.float32, 2)
    clean = [p.clone() for p in ps]
    ref = optim.AdamW(clean, lr=0.1, state_bits=bits)
    for p, g in zip(clean, gs):
        p.grad = g.clone()
    ref.step()
    gs[0][130], gs[0][140] = float('inf'), float('nan')
    opt = optim.AdamW(ps, lr=0.1, state_bits=bits)
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    rest = [i for i in range(400) if i not in (130, 140)]
    assert torch.equal(ps[0][rest], clean[0][rest]) and torch.equal(ps[1], clean[1]) and ps[0][[130, 140]].isnan().all()
    m, v = opt.moments()[0]
    rm, rv = ref.moments()[0]
    out = [i for i in range(512 + 384) if not 128 <= i < 256]
    assert torch.equal(m[out], rm[out]) and torch.equal(v[out], rv[out])
    assert m[140].isnan() and v[140].isnan() and v[130] == float('inf')
    clipped = optim.AdamW(ps, lr=0.1, state_bits=bits, max_norm=1.0)
    before = ps[1].clone()
    clipped.step()
    assert ps[0].isnan().all() and torch.isfinite(ps[1]).all() and not torch.equal(ps[1], before)


@pytest.mark.gpu
def test_zero_gradients_and_zero_moments():
    p = torch.randn(1000, device='cuda')
    for bits in (8, 32):
        x = p.clone()
        x.grad = torch.zeros_like(x)
        opt = optim.AdamW([x], lr=0.1, weight_decay=0.0, state_bits=bits, max_norm=0.5)
        opt.step()
        assert torch.equal(x, p) and not any(t.any() for t in opt.buffers()[0].values())


@pytest.mark.gpu
def test_groups_streams_versions_and_moved_parameters():
    """Groups of different types and settings; a scheduler; a step on another stream; autograd notices the write; a
    parameter whose storage was replaced is followed."""
    a, b = torch.nn.Parameter(torch.ones(300, device='cuda')), torch.nn.Parameter(torch.ones(40, device='cuda').bfloat16())
    opt = optim.AdamW([dict(params=[a], lr=0.5), dict(params=[b], weight_decay=0.0, max_norm=1.0)], lr=0.25, weight_decay=0.0)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    a.grad, b.grad = torch.ones_like(a), -torch.ones_like(b)
    kept = (a * a).sum()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    sched.step()
    assert torch.allclose(a, torch.full_like(a, 0.5)) and torch.allclose(b.float(), torch.full((40,), 1.25, device='cuda'))
    with pytest.raises(RuntimeError):                                  # a changed behind the saved product
        kept.backward()
    a.data = a.data.clone()
    a.grad = torch.ones(10, 30, device='cuda').t().reshape(300)
    opt.step()
    assert torch.allclose(a, torch.full_like(a, 0.25), atol=1e-6)
    a.grad = None
    loss = opt.step(lambda: torch.tensor(3.0))
    assert float(loss) == 3.0
    a.data = torch.ones(600, device='cuda')[::2]
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.gpu
def test_parameters_that_change_size_are_refused():
    """Host checks: no kernel reads behind a parameter, gradient or target that is smaller than it was."""
    def fresh():
        p, t = torch.nn.Parameter(torch.ones(40, device='cuda')), torch.ones(40, device='cuda')
        p.grad = torch.ones_like(p)
        return p, t, optim.AdamW([p], targets=[t])
    p, t, opt = fresh()
    p.data = p.data[:10]                                               # the same address
    with pytest.raises(RuntimeError):                                  # torch's own check
        p.grad = torch.ones(40, device='cuda')
    p.grad = torch.ones(10, device='cuda')
    with pytest.raises(ValueError):
        opt.step()
    p, t, opt = fresh()
    p.data = torch.ones(10, device='cuda')
    with pytest.raises(ValueError):
        opt.step()
    p, t, opt = fresh()
    t.data = torch.ones(10, device='cuda')
    with pytest.raises(ValueError):
        opt.step()
    assert (p == 1).all() and opt.step_count == 0


@pytest.mark.gpu
def test_recording_without_capturable_and_copies_are_refused():
    p = torch.nn.Parameter(torch.ones(40, device='cuda'))
    p.grad = torch.ones_like(p)
    opt = optim.AdamW([p])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode='thread_local'):
        with pytest.raises(RuntimeError):
            opt.step()
        p.grad.mul_(1.0)
    torch.cuda.synchronize()
    assert (p == 1).all() and opt.step_count == 0
    for copies in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError):
            copies(opt)


@pytest.mark.gpu
def test_arguments_are_checked():
    p = torch.zeros(8, 4, device='cuda')
    for kw in (dict(lr=-1), dict(lr=float('inf')), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1), dict(weight_decay=-1),
               dict(max_norm=0.0), dict(max_norm=float('inf')), dict(polyak=2.0), dict(targets=[]), dict(targets=[torch.zeros(4, 8, device='cuda')]),
               dict(targets=[p]), dict(targets=[torch.zeros(8, 4, device='cuda').half()])):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    for bad in ([p.t()], [p, p[:2].clone().half()], [p, p[1:]], [dict(params=[])]):
        with pytest.raises(ValueError):
            optim.AdamW(bad)
    for bad in ([p.double()], [3.0]):
        with pytest.raises(TypeError):
            optim.AdamW(bad)
    with pytest.raises(ValueError):
        optim.AdamW([dict(params=[p])], targets=[p.clone()])
    opt = optim.AdamW([p])
    p.grad = torch.ones_like(p)
    opt.param_groups[0]['lr'] = -1.0
    with pytest.raises(ValueError):
        opt.step()
    with pytest.raises(ValueError):
        opt.step_count = -1
    with pytest.raises(TypeError):
        opt.moments(torch.bfloat16)
    with pytest.raises(TypeError):
        optim.dequantize(torch.zeros(128, dtype=torch.uint8, device='cuda'), torch.zeros(1, dtype=torch.int16, device='cuda'), True, torch.float16)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A variable of more than 2^31 elements (its byte offsets pass 2^32): the last elements' step, 8-bit codes and target."""
    n, last = (1 << 31) + 300, 1000
    p = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(0)
    p.grad[-last:] = torch.randn(last, generator=g, device='cuda').bfloat16()
    opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, state_bits=8, seed=11)
    opt.step()
    first = n - last
    lo = first // 128 * 128
    gn = p.grad[lo:].float().cpu().numpy()
    z, zb = np.zeros(gn.size, np.uint8), np.zeros(-(-gn.size // 128), np.int16)
    want = _step8(z, zb, z, zb, gn, 1.0, 1, 11, 0, np.arange(lo, n))
    st = opt.state[p]
    for k, w in zip(('exp_avg', 'exp_avg_base', 'exp_avg_sq', 'exp_avg_sq_base'), want):
        got = st[k][lo // 128:] if k.endswith('base') else st[k][lo:]
        assert np.array_equal(got.cpu().numpy(), w), k
    assert not p[:first].any() and not st['exp_avg'][:lo].any()
    live = p.grad[first:].float().abs() > 1e-3
    assert torch.allclose(p[first:].float()[live], -0.5 * p.grad[first:].float().sign()[live], rtol=2.0 ** -7)


# ---- gradients of another type or device ---------------------------------------------------------------------------------
OTHER_TYPES = [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16), (torch.float32, torch.float64)]


def _with_gradient(dtype, grad_dtype, device):
    """Two parameters, the second with a gradient of another type: torch's own way, ``grad_dtype``."""
    ps = [torch.nn.Parameter(torch.ones(300, dtype=dtype, device=device)) for _ in range(2)]
    ps[0].grad = torch.ones(300, dtype=dtype, device=device)
    ps[1].grad_dtype = grad_dtype
    ps[1].grad = torch.ones(300, dtype=grad_dtype, device=device)
    return ps


@pytest.mark.parametrize('first', [True, False], ids=['all', 'one_missing'])
@pytest.mark.parametrize('dtype,grad_dtype', OTHER_TYPES)
def test_the_host_refuses_gradients_of_another_type(dtype, grad_dtype, first):
    """The check itself, on the CPU: what it lets through is read as the parameter's type."""
    ps = _with_gradient(dtype, grad_dtype, 'cpu')
    plan = optim._Plan(ps, None, 32)
    if not first:
        ps[0].grad = None
    with pytest.raises(ValueError):
        optim.AdamW._gradients(None, plan)
    ps[1].grad = None
    ps[1].grad_dtype = dtype
    ps[1].grad = torch.ones(300, dtype=dtype)
    assert optim.AdamW._gradients(None, plan)[1] is ps[1].grad
    plan.like = plan.like[0], {0}                                      # parameters on a GPU, gradients that are not
    with pytest.raises(ValueError):
        optim.AdamW._gradients(None, plan)
    ps[0].grad = ps[1].grad = None
    assert optim.AdamW._gradients(None, plan) == [None, None]


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,grad_dtype', OTHER_TYPES)
def test_a_step_with_gradients_of_another_type_is_refused(dtype, grad_dtype, bits):
    ps = _with_gradient(dtype, grad_dtype, 'cuda')
    opt = optim.AdamW(ps, lr=0.5, state_bits=bits)
    with pytest.raises(ValueError):
        opt.step()
    assert all((p == 1).all() for p in ps) and opt.step_count == 0 and not any(t.any() for t in opt.buffers()[0].values())
    ps[1].grad = None
    ps[1].grad_dtype = dtype
    ps[1].grad = torch.ones(300, dtype=dtype, device='cuda')
    opt.step()
    assert opt.step_count == 1 and all((p < 1).all() for p in ps)


@pytest.mark.gpu
@pytest.mark.parametrize('capturable', [False, True], ids=['host', 'device'])
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_subnormal_second_moments_without_eps(dtype, bits, capturable):
    """eps = 0: the first step is lr sign(g) however small g is.  g = 2e-20: g^2 = 4e-40 and v = g^2 / 1000 are subnormal, v holds
    285 of the smallest steps, so sqrt(v) is right to half of 1 / 285 / 2 (0.1 %); the parameter to its own rounding."""
    g = torch.full((700,), 2e-20, dtype=dtype, device='cuda')
    g[::2].neg_()
    p = torch.zeros(700, dtype=dtype, device='cuda')
    p.grad = g
    opt = optim.AdamW([p], lr=0.5, eps=0.0, weight_decay=0.0, state_bits=bits, capturable=capturable)
    opt.step()
    assert torch.allclose(p.double(), -0.5 * g.double().sign(), rtol=2e-3 + HALF[dtype], atol=0)
    assert (opt.moments()[0][1][:700] > 0).all()


# ---- the clip at the ends of 32 bits -------------------------------------------------------------------------------------
@pytest.mark.parametrize('max_norm', [1e39, 1e-39, 1e-50])
def test_a_clip_that_float32_does_not_hold_is_refused(max_norm):
    """As float32 these are infinity, subnormal and zero."""
    p = 1 << 20
    assert _hip.lib.mpe_adamw_step(_args(max_norm=max_norm), 1, _table(), p, (C.c_void_p * 1)(p), None) == -6
    group = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, polyak=0.99, max_norm=max_norm)
    with pytest.raises(ValueError):
        optim.AdamW._check_group(group)
    for good in (None, 2.0 ** -126, 3.4028234663852886e38):
        optim.AdamW._check_group(dict(group, max_norm=good))


@pytest.mark.gpu
@pytest.mark.parametrize('count', [4, 8192, 20000])
def test_a_norm_beyond_float32_is_clipped(count):
    """Finite gradients whose norm is not a float32: g' = g max_norm / |g| (the factor, 1e-41 at least, has 12 bits)."""
    g = torch.full((count,), 3e38, device='cuda')
    g[::2].neg_()
    p = torch.zeros(count, device='cuda')
    p.grad = g
    opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, max_norm=0.5)
    opt.step()
    want = 0.1 * 0.5 * g.double() / g.double().norm()
    assert torch.allclose(opt.moments()[0][0][:count].double(), want, rtol=2.0 ** -10, atol=0)
    assert torch.allclose(p.double(), -0.5 * g.double().sign(), rtol=2.0 ** -10, atol=0)


@pytest.mark.gpu
def test_versions_move_where_something_is_written():
    """A parameter without a gradient is not written: a graph that saved it still runs; its target is.  Parameters and targets
    made in inference mode, which have no version, are stepped like others."""
    a, b = (torch.nn.Parameter(torch.ones(30, device='cuda')) for _ in range(2))
    ta, tb = torch.zeros(30, device='cuda'), torch.zeros(30, device='cuda')
    opt = optim.AdamW([a, b], lr=0.5, weight_decay=0.0, targets=[ta, tb])
    kept = (a * a).sum()
    seen = [t._version for t in (a, b, ta, tb)]
    b.grad = torch.ones(30, device='cuda')
    opt.step()
    assert [t._version - v for t, v in zip((a, b, ta, tb), seen)] == [0, 1, 1, 1]
    kept.backward()
    assert (a.grad == 2).all()
    with torch.inference_mode():
        p, t = torch.ones(30, device='cuda'), torch.zeros(30, device='cuda')
        p.grad = torch.ones(30, device='cuda')
        opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, targets=[t])
        opt.step()
        opt.step()
        assert opt.step_count == 2 and torch.allclose(p, torch.zeros(30, device='cuda'), atol=1e-6) and (t > 0).all()


# ---- the plan's memory ---------------------------------------------------------------------------------------------------
def test_the_plan_stays_where_it_is_when_parameters_move():
    """On the CPU: what a recording or a step under way reads is not given back while the optimizer lives."""
    p, t = torch.nn.Parameter(torch.ones(300)), torch.ones(300)
    plan = optim._Plan([p], [t], 8)
    at, held = plan.plan_ptr, plan.plan.clone()
    hold = [p.data, t.data]
    p.data, t.data = p.data.clone(), t.data.clone()
    assert plan.pointers() != plan.ptrs
    plan.build()
    assert plan.plan_ptr == plan.plan.data_ptr() == at and not torch.equal(plan.plan, held) and plan.pointers() == plan.ptrs
    del hold


@pytest.mark.gpu
def test_recordings_follow_parameters_that_moved():
    """After an eager step that found the parameters elsewhere, replays step them there, like the eager run."""
    def make():
        p = torch.nn.Parameter(torch.full((9000,), 2.0, device='cuda'))
        p.grad = torch.linspace(-1, 1, 9000, device='cuda')
        return p, optim.AdamW([p], lr=0.1, max_norm=0.5, capturable=True)
    (a, oa), (b, ob) = make(), make()
    for _ in range(5):
        oa.step()
    ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode='thread_local'):
        ob.step()
    graph.replay()
    old = b.data
    b.data = b.data.clone()
    ob.step()
    left = old.clone()
    junk = [torch.full_like(ob._plans[0].plan, 255) for _ in range(4)]
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(old, left) and torch.equal(a, b) and oa.step_count == ob.step_count == 5
    del junk


@pytest.mark.gpu
@pytest.mark.parametrize('capturable', [False, True])
def test_an_optimizer_that_goes_while_another_stream_steps(capturable):
    """Steps queued on a side stream behind other work; the optimizer is dropped and its memory asked for and written on the
    main stream at once: the steps still read their own."""
    n = 1 << 20
    p = torch.nn.Parameter(torch.zeros(n, device='cuda'))
    p.grad = torch.ones(n, device='cuda')
    opt = optim.AdamW([p], lr=0.125, weight_decay=0.0, capturable=capturable)
    sizes = [(t.numel(), t.dtype) for t in list(opt.buffers()[0].values()) + [opt._plans[0].plan]]
    busy = torch.randn(4096, 4096, device='cuda')
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-2
        for _ in range(3):
            opt.step()
    del opt
    junk = [torch.full((c,), 77, dtype=dt, device='cuda') for c, dt in sizes for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.allclose(p, torch.full_like(p, -0.375), rtol=1e-5)
    del junk


@pytest.mark.gpu
def test_a_group_that_could_not_be_added_is_not_there(monkeypatch):
    """A failure on the way (memory, say) leaves no group that later steps pass over in silence."""
    a, b = (torch.nn.Parameter(torch.ones(30, device='cuda')) for _ in range(2))
    opt = optim.AdamW([a], lr=0.5)
    with monkeypatch.context() as m:
        m.setattr(optim._Plan, 'build', lambda self: (_ for _ in ()).throw(MemoryError()))
        with pytest.raises(MemoryError):
            opt.add_param_group(dict(params=[b]))
    assert len(opt.param_groups) == 1 and b not in opt.state
    opt.add_param_group(dict(params=[b]))
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[b]))              # torch's own check: already in a group
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    assert (a < 1).all() and (b < 1).all() and len(opt.buffers()) == len(opt.param_groups) == 2


@pytest.mark.gpu
@pytest.mark.parametrize('capturable', [False, True])
def test_a_resumed_run_keeps_its_seed(capturable):
    """8-bit moments: a run continued by an optimizer of another seed rounds as the first one would have."""
    p, q = (torch.nn.Parameter(torch.ones(5000, device='cuda')) for _ in range(2))
    a, b = optim.AdamW([p], state_bits=8, seed=(3 << 40) + 4), optim.AdamW([q], state_bits=8, seed=9, capturable=capturable)

    def go(x, opt, k):
        x.grad = torch.randn(5000, generator=torch.Generator(device='cuda').manual_seed(k), device='cuda')
        opt.step()
    for k in range(2):
        go(p, a, k)
    q.data.copy_(p.data)
    b.load_state_dict(a.state_dict())
    for k in range(2, 4):
        go(p, a, k)
        go(q, b, k)
    assert all(torch.equal(x, b.buffers()[0][k]) for k, x in a.buffers()[0].items())
    old = a.state_dict()
    for g in old['param_groups']:
        del g['seed']                                        # as before the seed was held
    b.load_state_dict(old)
    assert b.param_groups[0]['seed'] == (3 << 40) + 4


@pytest.mark.gpu
def test_load_hooks_run():
    p = torch.nn.Parameter(torch.ones(300, device='cuda'))
    p.grad = torch.ones_like(p)
    opt, seen = optim.AdamW([p], lr=0.5), []
    opt.step()
    saved = opt.state_dict()

    def halve(o, d):
        seen.append('halve')
        return dict(d, param_groups=[dict(g, lr=g['lr'] / 2) for g in d['param_groups']])
    opt.register_load_state_dict_pre_hook(halve)
    opt.register_load_state_dict_pre_hook(lambda o, d: seen.append('first'), prepend=True)
    opt.register_load_state_dict_post_hook(lambda o: seen.append((o is opt, o.param_groups[0]['lr'])))
    gone = opt.register_load_state_dict_post_hook(lambda o: seen.append('gone'))
    gone.remove()
    opt.load_state_dict(saved)
    assert seen == ['first', 'halve', (True, 0.25)] and saved['param_groups'][0]['lr'] == 0.5


@pytest.mark.gpu
def test_views_of_one_array_move_its_version():
    """Parameters that are views of one array share its version: autograd notices a step through any of them and through it."""
    flat, lone = torch.ones(300, device='cuda'), torch.nn.Parameter(torch.ones(30, device='cuda'))
    ps = [flat[:100], flat[128:200], flat[200:300].view(10, 10), lone]
    opt = optim.AdamW(ps, lr=0.5, targets=[p.detach().clone() for p in ps])
    scale = torch.ones(300, device='cuda', requires_grad=True)
    for saved in (lambda: (flat * scale).sum(), lambda: (ps[1] * scale[:72]).sum(), lambda: (ps[2].view(-1) * scale[:100]).sum(),
                  lambda: (lone * lone).sum()):
        loss = saved()
        seen = [p._version for p in ps]
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        assert all(p._version > v for p, v in zip(ps, seen))
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
