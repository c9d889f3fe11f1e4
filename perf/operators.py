"""Cases that measure the learner's operators: products grouped by agent with ragged row counts (forward and
backward) and the AdamW step over many tensors (moments in 32 or in 8 bits).

``own = False``: ``run`` computes them from elementary torch operations in 32 bits; ``own = True``: it calls
``marl_amd.grouped`` / ``marl_amd.optim``.  ``exact`` is the definition in 64 bits, written apart from both."""
import math

import numpy as np
import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BETA1, BETA2, EPS, LR, DECAY, POLYAK, MAX_NORM = 0.9, 0.999, 1e-8, 1e-2, 1e-2, 0.99, 0.5
BLOCK = 128                   # elements of a tensor that share the exponent base of their 8-bit moments
M32 = 0xFFFFFFFF


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # first layer of simple_tag's four actors on the learners' batch of 1 024: the smallest call, all latency
        {'name': 'forward f32 actors', 'op': 'forward', 'dtype': 'f32', 'groups': 4, 'rows': 4096, 'k': 16, 'n': 64, 'relu': True, 'even': True},
        # a handful of rows over sixteen networks of a wide policy (single steps of a few envs; most networks idle): weight bytes
        {'name': 'forward bf16 few rows', 'op': 'forward', 'dtype': 'bf16', 'groups': 16, 'rows': 13, 'k': 1024, 'n': 2048, 'relu': True, 'even': False},
        # nothing a multiple of anything: seven policies of unlike populations
        {'name': 'forward f16 odd', 'op': 'forward', 'dtype': 'f16', 'groups': 7, 'rows': 5003, 'k': 333, 'n': 517, 'relu': False, 'even': False},
        # scaled tag (48 + 16 agents, 32 landmarks): first layer of its 64 critics, all observations and actions (14 752) of 1 024 transitions each
        {'name': 'forward f32 scaled critics', 'op': 'forward', 'dtype': 'f32', 'groups': 64, 'rows': 65536, 'k': 14752, 'n': 64, 'relu': True, 'even': True},
        # wide networks on many rows: arithmetic
        {'name': 'forward bf16 wide', 'op': 'forward', 'dtype': 'bf16', 'groups': 32, 'rows': 32768, 'k': 2048, 'n': 2048, 'relu': True, 'even': False},
        # backward of the hidden layer of simple_tag's four learners: latency
        {'name': 'backward f32 hidden', 'op': 'backward', 'dtype': 'f32', 'groups': 4, 'rows': 4096, 'k': 64, 'n': 64, 'relu': True, 'even': True},
        # backward of the first layer of scaled tag's 64 actors (226 observations) on unlike batches
        {'name': 'backward f32 scaled actors', 'op': 'backward', 'dtype': 'f32', 'groups': 64, 'rows': 60001, 'k': 226, 'n': 64, 'relu': True, 'even': False},
        # backward of wide networks: arithmetic
        {'name': 'backward bf16 wide', 'op': 'backward', 'dtype': 'bf16', 'groups': 16, 'rows': 16384, 'k': 1024, 'n': 1024, 'relu': True, 'even': False},
        # every actor and critic of simple_tag's four learners: 48 variables, clipped each, with their targets: latency
        {'name': 'adamw32 f32 learners', 'op': 'adamw', 'dtype': 'f32', 'bits': 32, 'agents': 4, 'obs': 16, 'hidden': 64, 'joint': 84, 'clip': True, 'target': True},
        # the same of scaled tag's 64 learners: 768 variables, 64 million values
        {'name': 'adamw32 f32 scaled learners', 'op': 'adamw', 'dtype': 'f32', 'bits': 32, 'agents': 64, 'obs': 226, 'hidden': 64, 'joint': 14752, 'clip': True, 'target': True},
        # the small learners with moments in 8 bits
        {'name': 'adamw8 f32 learners', 'op': 'adamw', 'dtype': 'f32', 'bits': 8, 'agents': 5, 'obs': 34, 'hidden': 128, 'joint': 197, 'clip': True, 'target': True},
        # wide learners in bfloat16 with moments in 8 bits, no targets: bytes
        {'name': 'adamw8 bf16 wide learners', 'op': 'adamw', 'dtype': 'bf16', 'bits': 8, 'agents': 16, 'obs': 1024, 'hidden': 2048, 'joint': 4096, 'clip': False, 'target': False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        op = rng.choice(['forward', 'backward'])
        dtype = rng.choice(['f32', 'bf16', 'f16'])
        groups, k, n = _log(rng, 1, 64), _log(rng, 9, 2048), _log(rng, 5, 2048)
        most = 65536 if dtype == 'f32' else 32768
        rows = _log(rng, 1, most)
        while rows * k * n * (2 if op == 'backward' else 1) > 5e10:      # about the largest listed f32 product
            rows = rows // 2 + 1
        return {'op': op, 'dtype': dtype, 'groups': groups, 'rows': rows, 'k': k, 'n': n, 'relu': rng.random() < 0.6,
                'even': False}
    hidden = _log(rng, 17, 1024)
    agents, obs = _log(rng, 1, 32), _log(rng, 4, 512)
    return {'op': 'adamw', 'dtype': rng.choice(['f32', 'bf16', 'f16']), 'bits': rng.choice([8, 32]), 'agents': agents, 'obs': obs,
            'hidden': hidden, 'joint': min(_log(rng, 16, 8192), agents * (obs + 5)) + 1, 'clip': rng.random() < 0.6,
            'target': rng.random() < 0.6}


def _shapes(case):
    """Variables of every agent's actor and critic: two hidden layers, five actions, one value."""
    h, out = case['hidden'], []
    for a in range(case['agents']):
        for d, o in ((case['obs'] - a % 3, 5), (case['joint'], 1)):          # agents observe unlike numbers of entities
            out += [(h, d), (h,), (h, h), (h,), (o, h), (o,)]
    return out


def work(case):
    size = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'adamw':
        count = sum(math.prod(s) for s in _shapes(case))
        moments = 16 if case['bits'] == 32 else 4 + 8 / BLOCK
        # parameter and target read and written, gradient read, two moments read and written
        return {'bytes': count * (3 * size + moments + (2 * size if case['target'] else 0)), 'flops': count * 18}
    g, t, k, n = case['groups'], case['rows'], case['k'], case['n']
    used = min(g, t)                                     # a network without rows is not read in the forward pass
    if case['op'] == 'forward':
        return {'bytes': size * (t * k + used * n * (k + 1) + t * n), 'flops': 2 * t * k * n}
    # grad, the saved output (its sign), x and weight read; dx, dweight, dbias written
    return {'bytes': size * (t * n * (2 if case['relu'] else 1) + 2 * t * k + used * n * k + g * n * (k + 1)), 'flops': 4 * t * k * n}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _sizes(case, seed):
    """Rows of each group: even, or drawn (some groups empty when rows are few, unlike by up to about eight otherwise)."""
    g, t = case['groups'], case['rows']
    if case['even']:
        return [t // g] * g
    r = np.random.RandomState(seed % (1 << 31))
    share = r.uniform(0.25, 2.0, g)
    return [int(v) for v in r.multinomial(t, share / share.sum())]


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, dtype=dtype):
        return torch.randn(*shape, generator=gen, device='cuda', dtype=dtype).mul_(scale)

    if case['op'] != 'adamw':
        sizes = _sizes(case, seed)
        g, t, k, n = case['groups'], case['rows'], case['k'], case['n']
        s = {'case': case, 'sizes': sizes,
             'ends': torch.tensor(np.cumsum(sizes), dtype=torch.int32, device='cuda'),
             'x': normal(t, k), 'weight': normal(g, n, k, scale=k ** -0.5)}
        if case['op'] == 'forward':
            s['bias'] = normal(g, n, scale=0.1)
        else:                                            # what the forward pass saved, and the loss's gradient
            s['y'] = normal(t, n).clamp_(min=0) if case['relu'] else None
            s['grad'] = normal(t, n, scale=0.1)
        return s
    shapes = _shapes(case)
    counts = [math.prod(s) for s in shapes]
    blocks = [-(-c // BLOCK) for c in counts]            # every variable starts at a multiple of BLOCK of the flat arrays
    first = np.concatenate([[0], np.cumsum(blocks)])
    total = int(first[-1]) * BLOCK
    of_block = torch.repeat_interleave(torch.arange(len(counts), device='cuda'), torch.tensor(blocks, device='cuda'))
    within = ((torch.arange(total // BLOCK, device='cuda') - torch.tensor(first[:-1], device='cuda')[of_block])[:, None] * BLOCK
              + torch.arange(BLOCK, device='cuda')).reshape(-1)
    live = within < torch.tensor(counts, device='cuda')[of_block].repeat_interleave(BLOCK)
    # gradients of unlike size from variable to variable (some above the clip, some below) and within one
    scale = torch.exp(torch.randn(len(counts), generator=gen, device='cuda') * 1.5 - 4.0)[of_block].repeat_interleave(BLOCK)
    scale *= torch.exp(torch.randn(total, generator=gen, device='cuda') * 0.7)
    grad = normal(total, dtype=torch.float32) * scale * live
    m = (0.2 * normal(total, dtype=torch.float32) * scale * live)
    v = (scale.square() * torch.rand(total, generator=gen, device='cuda') * live)
    s = {'case': case, 'shapes': shapes, 'counts': counts, 'first': first, 'of_block': of_block, 'within': within,
         'step': 400, 'seed': int(seed) & 0x7FFFFFFF, 'param': (normal(total, scale=0.1, dtype=torch.float32) * live).to(dtype),
         'grad': grad.to(dtype)}
    s['target'] = (normal(total, scale=0.1, dtype=torch.float32) * live).to(dtype) if case['target'] else None
    if case['bits'] == 8:
        half = torch.full((total,), 1 << 19, dtype=torch.int64, device='cuda')
        s['m'], s['m_base'] = _encode(m, half, True)
        s['v'], s['v_base'] = _encode(v, half, False)
    else:
        s['m'], s['v'] = m, v
    if own:
        from marl_amd.optim import AdamW
        span = [(int(f) * BLOCK, c, sh) for f, c, sh in zip(first, counts, shapes)]
        views = lambda flat: [flat[o:o + c].view(sh) for o, c, sh in span]   # noqa: E731
        params = views(s['param'])
        for p, gr in zip(params, views(s['grad'])):
            p.grad = gr
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case['bits'],
                    max_norm=MAX_NORM if case['clip'] else None, targets=views(s['target']) if case['target'] else None,
                    polyak=POLYAK, seed=s['seed'])
        opt.step_count = s['step']
        flat = opt.buffers()[0]
        for name, key in (('exp_avg', 'm'), ('exp_avg_sq', 'v'), ('exp_avg_base', 'm_base'), ('exp_avg_sq_base', 'v_base')):
            if key in s:
                flat[name].copy_(s.pop(key))
        s['opt'] = opt
    return s


# ---- 8-bit moments: the leading 12 bits of a float (sign apart), counted from a base that a block of 128 shares ---------
def _encode(x, rnd, signed):
    """``rnd``: 20 random bits an element; added below the kept bits, they round up with the probability of the rest."""
    top = 127 if signed else 255
    bits = (x.view(torch.int32) & 0x7FFFFFFF).to(torch.int64)
    base = ((bits >> 20).view(-1, BLOCK).amax(1) + 1 - top).clamp_(min=0)
    code = (torch.clamp(bits + rnd, max=0x7FFFFFFF) >> 20) - base.repeat_interleave(BLOCK)
    code = code.clamp_(min=0) if signed else torch.maximum(code, (bits > 0).to(torch.int64))
    if signed:
        code = code | ((x.view(torch.int32) < 0).to(torch.int64) << 7)
    return code.to(torch.uint8), base.to(torch.int16)


def _decode(code, base, signed):
    c = code.to(torch.int32)
    mag = c & 127 if signed else c
    x = torch.where(mag > 0, (mag + base.to(torch.int32).repeat_interleave(BLOCK)) << 20, 0).view(torch.float32)
    return torch.where(c > 127, -x, x) if signed else x


def _mix(h):
    """The 32-bit finaliser of MurmurHash3 (A. Appleby, public domain)."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & M32
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & M32
    return h ^ (h >> 16)


def _random(s):
    """32 random bits an element, of the run's seed, the step, the variable and the element's place in it."""
    t = torch.tensor(s['step'], dtype=torch.int64, device='cuda')
    key = _mix((_mix((s['seed'] + t * 0x9E3779B9) & M32) + torch.arange(len(s['counts']), device='cuda') * 0x85EBCA77) & M32)
    return _mix(s['within'] ^ key[s['of_block']].repeat_interleave(BLOCK))


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _products(a, b, sizes, even):
    """a[rows of g] @ b[g] in 32 bits: one batched product for equal groups, one product a group otherwise."""
    a, b = a.float(), b.float()
    if even:
        return torch.bmm(a.view(len(sizes), -1, a.shape[1]), b).view(a.shape[0], -1)
    return torch.cat([p @ q for p, q in zip(a.split(sizes), b)])


def _plain_forward(s):
    even, sizes = s['case']['even'], s['sizes']
    y = _products(s['x'], s['weight'].float().transpose(1, 2).contiguous(), sizes, even)
    y += s['bias'].float().repeat_interleave(torch.diff(s['ends'], prepend=s['ends'].new_zeros(1)), 0, output_size=y.shape[0])
    if s['case']['relu']:
        y = torch.clamp(y, min=0)
    return {'y': y.to(s['x'].dtype)}


def _plain_backward(s):
    even, sizes, dtype = s['case']['even'], s['sizes'], s['x'].dtype
    d, x = s['grad'].float(), s['x'].float()
    if s['case']['relu']:
        d = d * (s['y'] > 0)
    dx = _products(d, s['weight'], sizes, even)
    if even:
        d3 = d.view(len(sizes), -1, d.shape[1])
        dw, db = torch.bmm(d3.transpose(1, 2).contiguous(), x.view(len(sizes), -1, x.shape[1])), d3.sum(1)
    else:
        pairs = list(zip(d.split(sizes), x.split(sizes)))
        dw, db = torch.stack([p.t() @ q for p, q in pairs]), torch.stack([p.sum(0) for p, _ in pairs])
    return {'dx': dx.to(dtype), 'dweight': dw.to(dtype), 'dbias': db.to(dtype)}


def _plain_adamw(s):
    case = s['case']
    s['step'] += 1
    g = s['grad'].float()
    if case['clip']:                                     # each variable's gradient to a norm of at most MAX_NORM
        squares = g.double().square().view(-1, BLOCK).sum(1)
        norm = torch.zeros(len(s['counts']), dtype=torch.float64, device='cuda').index_add_(0, s['of_block'], squares).sqrt().float()
        g = g * (MAX_NORM / torch.clamp(norm, min=MAX_NORM))[s['of_block']].repeat_interleave(BLOCK)
    m = _decode(s['m'], s['m_base'], True) if case['bits'] == 8 else s['m']
    v = _decode(s['v'], s['v_base'], False) if case['bits'] == 8 else s['v']
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    denom = v.sqrt() * (1 / math.sqrt(1 - BETA2 ** s['step'])) + EPS
    p = s['param'].float() * (1 - LR * DECAY) - (m / denom) * (LR / (1 - BETA1 ** s['step']))
    s['param'].copy_(p)
    out = {'param': s['param']}
    if case['target']:
        s['target'].copy_(s['target'].float() * POLYAK + s['param'].float() * (1 - POLYAK))
        out['target'] = s['target']
    if case['bits'] == 8:
        r = _random(s)
        s['m'], s['m_base'] = _encode(m, (r >> 16) << 4, True)
        s['v'], s['v_base'] = _encode(v, (r & 0xFFFF) << 4, False)
        # four significant bits: bfloat16 holds every value an 8-bit moment can stand for
        out['exp_avg'] = _decode(s['m'], s['m_base'], True).bfloat16()
        out['exp_avg_sq'] = _decode(s['v'], s['v_base'], False).bfloat16()
    else:
        s['m'], s['v'] = m, v
        out['exp_avg'], out['exp_avg_sq'] = m, v
    return out


def run(s):
    case = s['case']
    if not own:
        return {'forward': _plain_forward, 'backward': _plain_backward, 'adamw': _plain_adamw}[case['op']](s)
    if case['op'] == 'adamw':
        s['opt'].step()
        out = {'param': s['param']}
        if case['target']:
            out['target'] = s['target']
        out['exp_avg'], out['exp_avg_sq'] = s['opt'].moments(torch.bfloat16 if case['bits'] == 8 else torch.float32)[0]
        return out
    from marl_amd.grouped import grouped_linear, grouped_linear_backward
    if case['op'] == 'forward':
        return {'y': grouped_linear(s['x'], s['weight'], s['ends'], bias=s['bias'], relu=case['relu'])}
    dx, dw, db = grouped_linear_backward(s['grad'], s['x'], s['weight'], s['ends'], y=s['y'])
    return {'dx': dx, 'dweight': dw, 'dbias': db}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'forward': _exact_forward, 'backward': _exact_backward, 'adamw': _exact_adamw}[case['op']](s)


def _exact_forward(s):
    """Group by group, as the formula is written."""
    x, w, b = s['x'], s['weight'], s['bias']
    y = torch.empty(x.shape[0], w.shape[1], dtype=torch.float64, device=x.device)
    at = [0] + list(np.cumsum(s['sizes']))
    for i in range(len(s['sizes'])):
        z = torch.addmm(b[i].double(), x[at[i]:at[i + 1]].double(), w[i].double().t())
        y[at[i]:at[i + 1]] = torch.where(z > 0, z, 0.0) if s['case']['relu'] else z
    return {'y': y}


def _exact_backward(s):
    x, w = s['x'], s['weight']
    at = [0] + list(np.cumsum(s['sizes']))
    dx, dw = torch.empty(x.shape, dtype=torch.float64, device=x.device), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    db = torch.zeros(w.shape[:2], dtype=torch.float64, device=x.device)
    for i in range(len(s['sizes'])):
        part = slice(at[i], at[i + 1])
        d = s['grad'][part].double()
        if s['case']['relu']:
            d = torch.where(s['y'][part] > 0, d, 0.0)
        dx[part] = torch.mm(d, w[i].double())
        dw[i] = torch.mm(d.t().contiguous(), x[part].double())
        db[i] = d.sum(0)
    return {'dx': dx, 'dweight': dw, 'dbias': db}


def _exact_moment(codes, base, signed):
    """Value of a code c > 0 over the base b: the float whose leading 12 bits (sign apart) count c + b."""
    c = codes.to(torch.int64)
    mag = torch.remainder(c, 128) if signed else c
    n = mag + base.to(torch.int64).repeat_interleave(BLOCK)
    e, f = torch.div(n, 8, rounding_mode='floor'), torch.remainder(n, 8).double()
    val = torch.where(e > 0, torch.exp2(e.double() - 127) * (1 + f / 8), f / 8 * 2.0 ** -126)
    val = torch.where(mag > 0, val, 0.0)
    return torch.where(c >= 128, -val, val) if signed else val


def _exact_held(x, u, signed):
    """``x`` rounded to a value that an 8-bit code can hold: to the eighth of a binade below or, where the rest exceeds
    1 - u, above; what lies under the block's range is zero (first moment) or the smallest value (second)."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.clamp(a, min=2.0 ** -126)))
    e = torch.where(a < torch.exp2(e), e - 1, e).clamp(min=-126)
    n8 = a / torch.exp2(e) * 8                                       # 8 .. 16 (below 8: subnormal)
    n = torch.floor(n8 + u) + (e + 126) * 8                          # eighths counted from zero
    whole = torch.floor(n8) + (e + 126) * 8
    base = (whole.view(-1, BLOCK).amax(1) + 1 - (127 if signed else 255)).clamp(min=0).repeat_interleave(BLOCK)
    low = torch.zeros_like(n) if signed else base + 1
    n = torch.where(n > base, n, low)
    q, f = torch.floor(n / 8), torch.remainder(n, 8)
    val = torch.where(q > 0, torch.exp2(q - 127) * (1 + f / 8), f / 8 * 2.0 ** -126)
    return torch.where(a > 0, val * torch.sign(x), 0.0)


def _exact_adamw(s):
    case, t = s['case'], s['step'] + 1
    eight = case['bits'] == 8
    at = [int(f) * BLOCK for f in s['first']]
    g = s['grad'].double()
    if case['clip']:
        for i in range(len(s['counts'])):
            norm = float(torch.linalg.vector_norm(g[at[i]:at[i + 1]]))
            if norm > MAX_NORM:
                g[at[i]:at[i + 1]] *= MAX_NORM / norm
    m = _exact_moment(s['m'], s['m_base'], True) if eight else s['m'].double()
    v = _exact_moment(s['v'], s['v_base'], False) if eight else s['v'].double()
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g.square(), v, BETA2)
    mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = s['param'].double()
    p = p - LR * (DECAY * p + mhat / (vhat.sqrt() + EPS))
    out = {'param': p}
    if case['target']:
        held = p.to(s['param'].dtype).double()                       # the target follows the parameter as it is stored
        out['target'] = POLYAK * s['target'].double() + (1 - POLYAK) * held
    if eight:
        s['step'] = t
        r = _random(s)
        m = _exact_held(m, torch.div(r, 1 << 16, rounding_mode='floor').double() / 65536, True)
        v = _exact_held(v, torch.remainder(r, 1 << 16).double() / 65536, False)
    out['exp_avg'], out['exp_avg_sq'] = m, v
    return out
