"""AdamW over many tensors in one or a few launches, with moments in 32 or in 8 bits (libmpe_hip.so: mpe_adamw_step).

What a learner's update does behind its backward pass -- clip every variable's gradient to a norm (tf_util.py:137-149), Adam
(maddpg/maddpg/trainer/maddpg.py:130-145), polyak step of the target networks (maddpg.py:20-26) -- is one pass over the
variables' memory here:

    g' = g * max_norm / max(|g|, max_norm)                                                  (max_norm given)
    m  = b1 m + (1 - b1) g';   v = b2 v + (1 - b2) g'^2
    p  = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
    target = polyak target + (1 - polyak) p                                                 (targets given)

Parameters are float32, bfloat16 or float16 (one type a group; targets and gradients alike, others are refused); the arithmetic is in
32 bits, the norms in 64, and p is rounded once.  (Of 16-bit parameters with 8-bit moments the root and the quotient are to one last
place of 32 bits, elsewhere correctly rounded.)  ``state_bits=32`` holds the moments in float32; ``state_bits=8`` in one byte
each, plus one int16 for 128 of them: a logarithmic code (eighths of a binade; m 16 binades and a sign, v 32 binades) below
the largest element of its block, rounded stochastically from (seed, step, tensor, element), so that a moment is right on
average and a run repeats bit for bit.  A gradient that is not finite makes its element (32 bits) or its block of 128
(8 bits) useless, as it does any Adam; with ``max_norm`` its whole variable, whose norm it is part of."""
import collections
import ctypes as C
from operator import attrgetter

import torch
from torch.utils.hooks import RemovableHandle

from . import _hip

BLOCK = 128                       # elements that share the base of their 8-bit moments; every variable starts a new one
_DTYPES = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16, torch.float16: _hip.F16}
_dtype = attrgetter('dtype')
_F32 = torch.finfo(torch.float32)
_SEED = 0xFFFFFFFFFFFFFFFF


def dequantize(codes, base, signed, dtype=torch.float32):
    """The values that 8-bit moments stand for: ``codes`` (uint8, a multiple of 128), ``base`` (int16, one per 128);
    ``signed``: first moments.  float32 and bfloat16 hold them exactly."""
    if codes.dtype != torch.uint8 or base.dtype != torch.int16 or codes.numel() != base.numel() * BLOCK:
        raise ValueError('dequantize: uint8 codes with one int16 base per %d expected' % BLOCK)
    if codes.device.type != 'cuda' or base.device != codes.device:
        raise RuntimeError('dequantize works on GPU tensors (no CPU fallback)')
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError('dequantize returns float32 or bfloat16, not %r' % (dtype,))
    codes, base = codes.contiguous(), base.contiguous()
    out = torch.empty(codes.numel(), dtype=dtype, device=codes.device)
    pair, none = (codes.data_ptr(), base.data_ptr()), (None, None)
    _hip.check(_hip.launch(codes.get_device(), _hip.lib.mpe_adamw_moments, *(pair + none if signed else none + pair),
                           *((out.data_ptr(), None) if signed else (None, out.data_ptr())), codes.numel(), _DTYPES[dtype]),
               'mpe_adamw_moments')
    return out


def _encode(x, signed):
    """Moments in 32 bits as codes and bases of 8 (rounded to nearest; a step rounds as the kernel does): ``x`` float32, flat."""
    x = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK))
    top, bits = 127 if signed else 255, (x.view(torch.int32) & 0x7FFFFFFF).to(torch.int64)
    base = ((bits >> 20).view(-1, BLOCK).amax(1) + 1 - top).clamp_(min=0)
    code = (torch.clamp(bits + (1 << 19), max=0x7FFFFFFF) >> 20) - base.repeat_interleave(BLOCK)
    code = code.clamp_(min=0) | (x < 0).to(torch.int64) << 7 if signed else torch.maximum(code, (bits > 0).to(torch.int64))
    return code.to(torch.uint8), base.to(torch.int16)


def _families(tensors):
    """One of every family of views: they share the version that autograd looks at."""
    bases = [t if t._base is None else t._base for t in tensors]
    return list({id(b): t for b, t in zip(bases, tensors)}.values())


class _Plan(object):
    """One parameter group: its flat moments and what the kernels read about its variables."""

    def __init__(self, params, targets, state_bits):
        p0 = params[0]
        self.params, self.targets, self.bits = list(params), targets, state_bits
        self.device, self.dtype = p0.device, p0.dtype
        self.like = ({p0.dtype}, {p0.get_device()})           # of every gradient
        self.tracked = [not p.is_inference() for p in self.params]     # tensors of inference mode have no version
        self.moved = [t for t in self.targets or [] if not t.is_inference()]
        self.written = _families([p for p, on in zip(self.params, self.tracked) if on] + self.moved)
        self.counts = [p.numel() for p in self.params]
        self.first, total = [], 0
        for c in self.counts:                       # every variable starts at a multiple of BLOCK
            self.first.append(total)
            total += -(-c // BLOCK) * BLOCK
        dev = self.device
        if state_bits == 8:
            self.flat = {'exp_avg': torch.zeros(total, dtype=torch.uint8, device=dev),
                         'exp_avg_base': torch.zeros(total // BLOCK, dtype=torch.int16, device=dev),
                         'exp_avg_sq': torch.zeros(total, dtype=torch.uint8, device=dev),
                         'exp_avg_sq_base': torch.zeros(total // BLOCK, dtype=torch.int16, device=dev)}
        else:
            self.flat = {'exp_avg': torch.zeros(total, dtype=torch.float32, device=dev),
                         'exp_avg_sq': torch.zeros(total, dtype=torch.float32, device=dev)}
        self.grads = (C.c_void_p * len(self.params))()
        self.plan, self.streams = None, set()
        self.build()

    def views(self, j):
        """The moments of variable j, as views of the flat arrays."""
        o, c, out = self.first[j], self.counts[j], {}
        for name, t in self.flat.items():
            if name.endswith('_base'):
                out[name] = t[o // BLOCK:-(-(o + c) // BLOCK)]
            else:
                out[name] = t[o:o + c].view(self.params[j].shape)
        return out

    def set_moments(self, j, exp_avg, exp_avg_sq):
        """Variable j's moments from float32 values of its shape."""
        for name, value in (('exp_avg', exp_avg), ('exp_avg_sq', exp_avg_sq)):
            have, value = self.views(j), value.to(self.device, torch.float32)
            if self.bits == 32:
                have[name].copy_(value)
            else:
                code, base = _encode(value.reshape(-1), name == 'exp_avg')
                have[name].view(-1).copy_(code[:self.counts[j]])
                have[name + '_base'].copy_(base)

    def build(self):
        """The host table of pointers and its device plan."""
        for t in self.params + (self.targets or []):
            if not t.is_contiguous() or t.dtype != self.dtype or t.device != self.device:
                raise ValueError('AdamW: parameters and targets are contiguous and keep their type and device')
        n = len(self.params)
        if any(t.numel() != self.counts[j % n] for j, t in enumerate(self.params + (self.targets or []))):
            raise ValueError('AdamW: parameters and targets keep their size')
        self.table = (_hip.AdamTensor * n)()
        for j, p in enumerate(self.params):
            o = self.first[j]
            at = {k: t.data_ptr() + (o // BLOCK if k.endswith('_base') else o) * t.element_size() for k, t in self.flat.items()}
            self.table[j] = _hip.AdamTensor(param=p.data_ptr(), count=self.counts[j],
                                            target=None if self.targets is None else self.targets[j].data_ptr(), **at)
        code = _DTYPES[self.dtype]
        size = _hip.lib.mpe_adamw_plan(n, self.table, code, self.bits, None, 0)
        _hip.check(min(size, 0), 'mpe_adamw_plan')
        blob = torch.empty(size, dtype=torch.uint8)
        _hip.check(min(_hip.lib.mpe_adamw_plan(n, self.table, code, self.bits, blob.data_ptr(), size), 0), 'mpe_adamw_plan')
        if self.plan is None:                       # written again in place: a recording keeps reading this array
            self.plan = torch.empty(size, dtype=torch.uint8, device=self.device)
            self.plan_ptr = self.plan.data_ptr()
        self.plan.copy_(blob)
        self.ptrs = self.pointers()

    def use_on(self, raw):
        """Before the first eager step on a stream: what the plan owns is not handed to others until that stream is through."""
        for t in [self.plan] + list(self.flat.values()):
            t.record_stream(torch.cuda.current_stream(self.device))
        self.streams.add(raw)

    def pointers(self):
        return list(map(torch.Tensor.data_ptr, self.params if self.targets is None else self.params + self.targets))


class AdamW(torch.optim.Optimizer):
    """``torch.optim.Optimizer`` with ``step()`` as above (parameter groups and learning-rate schedulers work as usual).

    ``targets``: tensors like the parameters, in their order (of a parameter group: its ``'targets'`` entry), that follow
    them by ``polyak``; ``max_norm``: clip of each variable's gradient on its own; ``seed``: of the 8-bit rounding.
    ``capturable=True`` keeps the step count on the device, so that ``step()`` can be recorded in a HIP graph: every replay
    is one more step, with the learning rate and the other settings of the recording.  Gradients are read where they lie:
    a recording reads the same addresses again, so let them stay (``zero_grad(set_to_none=False)``), and keep the optimizer.

    A parameter without a gradient keeps its value and moments (its target still moves); the step count is the group's.
    ``state_dict`` / ``load_state_dict`` hold the moments as they are stored, the step counts and the seed: a run that is
    resumed repeats bit for bit."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=None,
                 targets=None, polyak=0.99, seed=0, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError('state_bits: 8 or 32, got %r' % (state_bits,))
        params = list(params)
        if targets is not None:
            if params and isinstance(params[0], dict):
                raise ValueError("targets: give each parameter group its own 'targets'")
            params = [dict(params=params, targets=list(targets))]
        self._bits, self._capturable = state_bits, bool(capturable)
        self._plans, self._clocks = [], []
        self._before_load, self._after_load = collections.OrderedDict(), collections.OrderedDict()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm,
                                      polyak=polyak, step=0, seed=int(seed) & _SEED))

    # -- construction ------------------------------------------------------------------------------------------------------
    @staticmethod
    def _check_group(g):
        b1, b2 = g['betas']
        if not (0 <= g['lr'] < float('inf')) or not 0 <= b1 < 1 or not 0 <= b2 < 1 or not g['eps'] >= 0 \
                or not g['weight_decay'] >= 0 or not 0 <= g['polyak'] <= 1:
            raise ValueError('AdamW: lr %r, betas %r, eps %r, weight_decay %r, polyak %r' % (
                g['lr'], g['betas'], g['eps'], g['weight_decay'], g['polyak']))
        if g['max_norm'] is not None and not _F32.tiny <= g['max_norm'] <= _F32.max:
            raise ValueError('AdamW: max_norm is positive and finite (a normal float32), or None, got %r' % (g['max_norm'],))

    def add_param_group(self, group):
        group = dict(group)
        targets = group.pop('targets', None)
        if torch.is_tensor(group.get('params')):
            group['params'] = [group['params']]
        params = group['params'] = list(group.get('params', ()))
        if not params:
            raise ValueError('AdamW: an empty parameter group')
        if targets is not None:
            targets = list(targets)
            if len(targets) != len(params):
                raise ValueError('AdamW: %d targets for %d parameters' % (len(targets), len(params)))
        p0 = params[0]
        for t in params + (targets or []):
            if not torch.is_tensor(t):
                raise TypeError('AdamW: parameters and targets are tensors, got %r' % (type(t),))
            if t.device.type != 'cuda':
                raise RuntimeError('marl_amd.optim.AdamW works on GPU tensors (no CPU fallback)')
            if t.dtype not in _DTYPES:
                raise TypeError('AdamW supports float32, bfloat16 and float16 parameters, got %r' % (t.dtype,))
            if t.dtype != p0.dtype or t.device != p0.device:
                raise ValueError('AdamW: the tensors of a parameter group share type and device')
            if not t.is_contiguous():
                raise ValueError('AdamW: parameters and targets are contiguous')
        if targets is not None and any(t.shape != p.shape for t, p in zip(targets, params)):
            raise ValueError('AdamW: a target has the shape of its parameter')
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in params + (targets or []) if t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError('AdamW: two of the tensors share memory')
        for key, value in self.defaults.items():
            group.setdefault(key, value)
        self._check_group(group)
        plan = _Plan(params, targets, self._bits)       # may fail: before the group is there
        clock = torch.zeros(4, dtype=torch.int64, device=plan.device) if self._capturable else None
        super().add_param_group(group)
        self._plans.append(plan)
        self._clocks.append(clock)
        for j, p in enumerate(params):
            self.state[p] = plan.views(j)

    # -- step count --------------------------------------------------------------------------------------------------------
    @property
    def step_count(self):
        """Steps taken (of the first parameter group; reads the device where it is kept there)."""
        return self._steps(0)

    @step_count.setter
    def step_count(self, value):
        for i in range(len(self._plans)):
            self._set_steps(i, value)

    def _steps(self, i):
        return int(self._clocks[i][0]) if self._clocks[i] is not None else self.param_groups[i]['step']

    def _set_steps(self, i, value):
        if int(value) < 0:
            raise ValueError('AdamW: a step count is >= 0, got %r' % (value,))
        self.param_groups[i]['step'] = int(value)
        if self._clocks[i] is not None:
            self._clocks[i][0] = int(value)

    # -- the step ----------------------------------------------------------------------------------------------------------
    def _gradients(self, plan):
        """Fills the plan's pointers; returns what must outlive the launch (``plan.whole``: no gradient is missing).  torch lets a gradient differ from its parameter in
        type (``grad_dtype``) and, through ``.data``, in everything else: the kernels read it as the parameter's."""
        grads = live = [p.grad for p in plan.params]
        try:
            plain = all(map(torch.Tensor.is_contiguous, grads))
        except TypeError:                                         # a None
            plain = False
        if not plain:
            grads = [None if g is None else g.contiguous() for g in grads]
            live = [g for g in grads if g is not None]
            sizes = [c if g is None else g.numel() for g, c in zip(grads, plan.counts)]
            pointers = [None if g is None else g.data_ptr() for g in grads]
        else:
            sizes, pointers = list(map(torch.Tensor.numel, grads)), list(map(torch.Tensor.data_ptr, grads))
        if live and (set(map(_dtype, live)), set(map(torch.Tensor.get_device, live))) != plan.like:
            raise ValueError('AdamW: gradients are %s on %s, as their parameters are' % (plan.dtype, plan.device))
        if sizes != plan.counts:
            raise ValueError('AdamW: a gradient is not of the size that its parameter had')
        plan.grads[:] = pointers
        plan.whole = len(live) == len(grads)
        return grads

    @torch.no_grad()
    def step(self, closure=None):
        """One step of every parameter group, on the current stream of its device."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if not self._capturable and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('AdamW: step() is recorded with capturable=True only (every replay is one more step)')
        index0 = 0
        for i, (group, plan) in enumerate(zip(self.param_groups, self._plans)):
            self._check_group(group)
            if plan.pointers() != plan.ptrs:                      # a parameter's storage was replaced
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError('AdamW: a parameter moved since the last step; take one step before recording')
                plan.build()
            keep = self._gradients(plan)
            clock = self._clocks[i]
            raw = torch._C._cuda_getCurrentRawStream(plan.device.index)
            if raw not in plan.streams and not torch.cuda.is_current_stream_capturing():
                plan.use_on(raw)
                if clock is not None:
                    clock.record_stream(torch.cuda.current_stream(plan.device))
            args = _hip.AdamArgs(group['lr'], *group['betas'], group['eps'], group['weight_decay'], group['max_norm'] or 0.0,
                                 group['polyak'], group['step'] + 1, _hip.ptr(clock), int(group['seed']) & _SEED, index0, _DTYPES[plan.dtype],
                                 self._bits)
            _hip.check(_hip.launch(plan.device.index, _hip.lib.mpe_adamw_step, args, len(plan.params), plan.table,
                                   plan.plan_ptr, plan.grads), 'mpe_adamw_step')
            if clock is None:
                group['step'] += 1
            index0 += len(plan.params)
            torch.autograd.graph.increment_version(plan.written if plan.whole else plan.moved + [
                p for p, g, on in zip(plan.params, keep, plan.tracked) if g is not None and on])
            del keep
        return loss

    # -- the moments -------------------------------------------------------------------------------------------------------
    def buffers(self):
        """For every parameter group the flat arrays that hold its moments (``exp_avg``, ``exp_avg_sq``, and with 8 bits
        their ``_base``): variables in order, each from a multiple of 128 on, zeros in between."""
        return [dict(plan.flat) for plan in self._plans]

    def moments(self, dtype=torch.float32):
        """For every parameter group its flat ``(exp_avg, exp_avg_sq)`` as values (laid out as in ``buffers``): the arrays
        themselves with ``state_bits=32``, what the codes stand for with 8."""
        if self._bits == 32:
            if dtype != torch.float32:
                raise TypeError('32-bit moments are float32')
            return [(plan.flat['exp_avg'], plan.flat['exp_avg_sq']) for plan in self._plans]
        if dtype not in (torch.float32, torch.bfloat16):
            raise TypeError('8-bit moments are given in float32 or bfloat16, not %r' % (dtype,))
        out = []
        for plan in self._plans:
            f = plan.flat
            m, v = torch.empty_like(f['exp_avg'], dtype=dtype), torch.empty_like(f['exp_avg_sq'], dtype=dtype)
            _hip.check(_hip.launch(plan.device.index, _hip.lib.mpe_adamw_moments, f['exp_avg'].data_ptr(),
                                   f['exp_avg_base'].data_ptr(), f['exp_avg_sq'].data_ptr(), f['exp_avg_sq_base'].data_ptr(),
                                   m.data_ptr(), v.data_ptr(), m.numel(), _DTYPES[dtype]), 'mpe_adamw_moments')
            out.append((m, v))
        return out

    def __getstate__(self):
        raise TypeError('AdamW is not copied or pickled: build another one and load this one\'s state_dict()')

    def state_dict(self):
        for i in range(len(self._plans)):
            self.param_groups[i]['step'] = self._steps(i)
        return super().state_dict()

    def fits(self, state_dict):
        """Raises where ``load_state_dict`` would refuse this one; the pairs of arrays to copy."""
        groups = state_dict['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in self.param_groups]:
            raise ValueError('AdamW: the state dict has other parameter groups')
        todo = []
        for plan, saved in zip(self._plans, groups):
            for j, key in enumerate(saved['params']):
                have, got = plan.views(j), state_dict['state'].get(key)
                if got is None or set(got) != set(have) or any(
                        got[k].shape != have[k].shape or got[k].dtype != have[k].dtype for k in have):
                    raise ValueError('AdamW: the moments of parameter %r have other names, shapes or types' % (key,))
                todo += [(have[k], got[k]) for k in have]
        for saved in groups:
            self._check_group(saved)
        return todo

    def load_state_dict(self, state_dict):
        """Settings, step counts and moments of an optimizer with the same groups, shapes and ``state_bits``; the moments are
        copied into this optimizer's arrays, which stay where they are."""
        state_dict = dict(state_dict)
        for hook in list(self._before_load.values()):
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        todo = self.fits(state_dict)
        groups = state_dict['param_groups']
        for dst, src in todo:
            dst.copy_(src)
        for i, (group, saved) in enumerate(zip(self.param_groups, groups)):
            group.update({k: v for k, v in saved.items() if k != 'params'})
            self._set_steps(i, saved['step'])
        for hook in list(self._after_load.values()):
            hook(self)

    @staticmethod
    def _add_hook(hooks, hook, prepend):
        handle = RemovableHandle(hooks)
        hooks[handle.id] = hook
        if prepend:
            hooks.move_to_end(handle.id, last=False)
        return handle

    def register_load_state_dict_pre_hook(self, hook, prepend=False):
        """As ``torch.optim.Optimizer``'s: ``hook(optimizer, state_dict)`` before ``load_state_dict``, which takes what it returns."""
        return self._add_hook(self._before_load, hook, prepend)

    def register_load_state_dict_post_hook(self, hook, prepend=False):
        """As ``torch.optim.Optimizer``'s: ``hook(optimizer)`` behind ``load_state_dict``."""
        return self._add_hook(self._after_load, hook, prepend)
