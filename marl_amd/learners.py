"""Every learner's update in one pass: the networks of all agents stacked, their dense layers as grouped products
(``marl_amd.grouped``), their variables stepped together (``marl_amd.optim``).

``MADDPGAgentTrainer.update`` (maddpg/maddpg/trainer/maddpg.py:161-196) evaluates n + 3 small networks per learner one after
the other, ~150 launches each, n learners in turn.  ``Learners(trainers)`` does the same arithmetic for all of them at once:
3 grouped layers for all agents' target actions, 3 + 3 for all critics, and so on, and one AdamW step per kind of network.  What is
left per trainer is data movement: the gather of its batch, its columns of the critics' inputs, its packed acting weights.  One
update is 153 launches for 4 learners, 201 for 5 (of two action spaces), 254 for 8.

One difference from the loop over trainers: every learner's targets come from the target networks as they were before this
update.  In the loop learner i already sees the target policies of learners < i moved by their polyak step of 1 %.

The trainers' networks become views of the stacked arrays (weights of narrower agents are padded with zeros, which stay
zero), so acting, ``act_all`` and the trainers' own methods go on as before (an update finds and refuses networks that were
taken out of the stacks since, as a second ``Learners`` of the same trainers does); the step is AdamW with ``weight_decay`` 0 unless
given, which is the trainers' Adam.  Moments live here (``Learners.p_opt`` / ``.q_opt``; they begin as the trainers' own, in 8 bits
rounded), not in the trainers' ``p_opt`` / ``q_opt``, which stay as they were: use one or the other
(a second ``Learners`` of the same trainers goes on where the first was with its ``state_dict``),
and save a run with ``Learners.state_dict`` (the trainers' optimizers no longer hold what a resumed run needs)."""
import torch
from torch import nn

from . import maddpg
from .grouped import grouped_linear, grouped_linear_backward, group_ends
from .optim import AdamW


NETS = ('p', 'q', 'target_p', 'target_q')          # a trainer's networks
OPTS = ('p_opt', 'q_opt')


def _linears(net):
    lin = list(net[::2]) if isinstance(net, nn.Sequential) and len(net) == 5 else []
    if len(lin) != 3 or not all(isinstance(m, nn.Linear) and m.bias is not None for m in lin) or not all(isinstance(m, nn.ReLU) for m in net[1::2]):
        raise NotImplementedError('Learners: networks of two hidden ReLU layers (maddpg.mlp_model) are supported')
    return lin


class _Stack(object):
    """n networks of one shape up to their input and output widths: weights [n, out, in], biases [n, out] per layer."""

    def __init__(self, nets):
        layers = list(zip(*[_linears(net) for net in nets]))
        if any(len({m.out_features for m in layer}) != 1 for layer in layers[:2]):
            raise NotImplementedError('Learners: networks of one hidden width are supported')
        self.w, self.b, self.n, self.nets = [], [], len(nets), list(nets)
        for k, layer in enumerate(layers):
            w0 = layer[0].weight
            if any(m.weight.dtype != torch.float32 or m.weight.device != w0.device for m in layer):
                raise TypeError('Learners: float32 networks on one GPU are supported')
            wide = max(m.in_features for m in layer)
            wide = -(-wide // 4) * 4 if k == 0 else wide       # 16-byte rows
            w = torch.zeros(self.n, max(m.out_features for m in layer), wide, device=w0.device)
            b = torch.zeros(w.shape[:2], device=w0.device)
            for i, m in enumerate(layer):
                with torch.no_grad():
                    w[i, :m.out_features, :m.in_features] = m.weight
                    b[i, :m.out_features] = m.bias
                m.weight.data = w[i, :m.out_features, :m.in_features]
                m.bias.data = b[i, :m.out_features]
            self.w.append(w)
            self.b.append(b)
        self.params = [t for net in nets for t in net.parameters()]
        self.at = [t.data_ptr() for t in self.params]

    def check(self, nets):
        """The networks' variables are still this stack's memory."""
        if any(a is not b for a, b in zip(nets, self.nets)) or list(map(torch.Tensor.data_ptr, self.params)) != self.at:
            raise RuntimeError('Learners: a network was replaced or its variables moved (.to(), .data, other Learners): build Learners anew')

    def written(self):
        """The networks' variables share the stacks' memory, not their versions: graphs that saved them are told of a step here."""
        torch.autograd.graph.increment_version(self.params)

    def variables(self):
        """Every network's variables, each a contiguous tensor of its own (clipping is per variable)."""
        return [t[i] for w, b in zip(self.w, self.b) for t in (w, b) for i in range(self.n)]

    def forward(self, x, ends):
        h1 = grouped_linear(x, self.w[0], ends, bias=self.b[0], relu=True)
        h2 = grouped_linear(h1, self.w[1], ends, bias=self.b[1], relu=True)
        return x, h1, h2, grouped_linear(h2, self.w[2], ends, bias=self.b[2])

    def gradients(self, acts, dout, ends):
        """The variables' gradients, stacked like them: [dw0, db0, dw1, db1, dw2, db2]."""
        x, h1, h2, _ = acts
        d2, dw2, db2 = grouped_linear_backward(dout, h2, self.w[2], ends)
        d1, dw1, db1 = grouped_linear_backward(d2, h1, self.w[1], ends, y=h2)
        _, dw0, db0 = grouped_linear_backward(d1, x, self.w[0], ends, y=h1, need_dx=False)
        return [dw0, db0, dw1, db1, dw2, db2]

    def to_columns(self, acts, dout, ends, w0_columns):
        """The gradient with respect to some input columns, given the first layer's weights of those columns."""
        x, h1, h2, _ = acts
        only = dict(need_dweight=False, need_dbias=False)
        d2 = grouped_linear_backward(dout, h2, self.w[2], ends, **only)[0]
        d1 = grouped_linear_backward(d2, h1, self.w[1], ends, y=h2, **only)[0]
        cols = d1.new_empty(d1.shape[0], w0_columns.shape[2])   # stands for x: only its shape counts
        return grouped_linear_backward(d1, cols, w0_columns, ends, y=h1, **only)[0]


class Learners(object):
    """All trainers' updates at once.  ``state_bits``: of the Adam moments (8 or 32)."""

    def __init__(self, trainers, weight_decay=0.0, state_bits=32, seed=0):
        self.trainers = list(trainers)
        t0 = self.trainers[0]
        n = self.n = len(self.trainers)
        if n != t0.n or [tr.agent_index for tr in self.trainers] != list(range(n)):
            raise ValueError('Learners: one trainer for every agent, in order')
        if len({(tr.local_q_func, tr.args.batch_size, tr.args.lr, tr.args.gamma, tr.grad_norm_clipping, str(tr.device))
                for tr in self.trainers}) != 1:
            raise NotImplementedError('Learners: trainers that share local_q_func, batch size, lr, gamma, clipping and device')
        steps = {}
        for kind in 'pq':
            taken = {int(getattr(tr, kind + '_opt').state.get(t, {}).get('step', 0))
                     for tr in self.trainers for t in getattr(tr, kind).parameters()}
            if len(taken) != 1:
                raise ValueError('Learners: the trainers have taken unlike numbers of steps: %s' % sorted(taken))
            steps[kind] = taken.pop()
        self.device, self.batch, self.gamma, self.local = t0.device, t0.args.batch_size, t0.args.gamma, t0.local_q_func
        self.sizes = t0.sizes_n
        self.acts = [sum(s) for s in self.sizes]
        self.p, self.target_p = _Stack([tr.p for tr in self.trainers]), _Stack([tr.target_p for tr in self.trainers])
        self.q, self.target_q = _Stack([tr.q for tr in self.trainers]), _Stack([tr.target_q for tr in self.trainers])
        kw = dict(lr=t0.args.lr, eps=1e-8, weight_decay=weight_decay, state_bits=state_bits, max_norm=t0.grad_norm_clipping,
                  polyak=1.0 - 1e-2, capturable=True)
        self.p_opt = AdamW(self.p.variables(), targets=self.target_p.variables(), seed=2 * seed, **kw)
        self.q_opt = AdamW(self.q.variables(), targets=self.target_q.variables(), seed=2 * seed + 1, **kw)
        self._adopt(steps['p'], [tr.p_opt for tr in self.trainers], self.p, self.p_opt)
        self._adopt(steps['q'], [tr.q_opt for tr in self.trainers], self.q, self.q_opt)
        b = self.batch
        self.ends = group_ends([b] * n, self.device)            # learner i's batch: rows i b .. (i + 1) b
        self.ends_all = group_ends([n * b] * n, self.device)    # agent j's observations of every learner's batch
        # columns of the critics' inputs that hold learner i's own action, and of the actors' outputs that exist
        obs = [tr.p[0].in_features for tr in self.trainers]
        first = self.first = [(obs[i] if self.local else sum(obs) + sum(self.acts[:i])) for i in range(n)]
        most = max(self.acts)
        self.cols = torch.tensor([[f + min(c, a - 1) for c in range(most)] for f, a in zip(first, self.acts)], device=self.device)
        self.real = torch.tensor([[float(c < a) for c in range(most)] for a in self.acts], device=self.device)
        self.alike = {}                                         # agents of one action space are sampled together
        for i, s in enumerate(self.sizes):
            self.alike.setdefault(tuple(s), []).append(i)
        self.alike = [(list(s), torch.tensor(who, device=self.device)) for s, who in self.alike.items()]

    @staticmethod
    def _adopt(steps, opts, stack, opt):
        """The step count and the moments of the trainers' own optimizers."""
        if steps == 0:
            return
        states = [[o.state[t] for t in net.parameters()] for o, net in zip(opts, stack.nets)]
        opt.step_count = steps
        shapes = [p.shape for p in opt.param_groups[0]['params']]
        for j, shape in enumerate(shapes):                      # variables as stacked: by layer, weight then bias, every network
            st = states[j % stack.n][j // stack.n]
            whole = []
            for key in ('exp_avg', 'exp_avg_sq'):
                whole.append(torch.zeros(shape, device=st[key].device))
                whole[-1][tuple(slice(c) for c in st[key].shape)] = st[key]
            opt._plans[0].set_moments(j, *whole)

    def _sample(self, logits):
        """Every agent's soft sample of its [rows, most] logits [n, rows, most]; columns it does not have are zero."""
        out = torch.zeros_like(logits)
        for s, who in self.alike:
            out[who, :, :sum(s)] = maddpg.soft_sample(logits[who][:, :, :sum(s)], s)
        return out

    def _softmax_backward(self, sample, grad):
        """Through ``_sample``: d = s (g - sum over the sub-space of s g)."""
        out = torch.zeros_like(grad)
        for s, who in self.alike:
            sg, at = sample[who] * grad[who], 0
            for width in s:
                part = slice(at, at + width)
                out[who, :, part] = sg[:, :, part] - sample[who][:, :, part] * sg[:, :, part].sum(-1, keepdim=True)
                at += width
        return out

    @staticmethod
    def _wide(parts, width):
        """The tensors side by side, filled up with zero columns."""
        have = sum(p.shape[1] for p in parts)
        if have < width:
            parts = list(parts) + [parts[0].new_zeros(parts[0].shape[0], width - have)]
        return torch.cat(parts, dim=1)

    def _rows(self, t, i):
        return t[i * self.batch:(i + 1) * self.batch]

    def _critic_input(self, obs_n, act_n, stack):
        width = stack.w[0].shape[2]
        if self.local:                                          # maddpg.py:51-52,86-87
            return torch.cat([self._wide([self._rows(obs_n[i], i), self._rows(act_n[i], i)], width) for i in range(self.n)])
        return self._wide(list(obs_n) + list(act_n), width)

    def state_dict(self):
        """What a run needs to go on, copied: the networks (of every trainer, unpadded), the moments, step counts and settings.
        (The trainers' networks lie in shared arrays: ``torch.save`` of one's own ``state_dict`` writes all of them.)"""
        nets = {name: [{k: v.detach().clone() for k, v in net.state_dict().items()} for net in getattr(self, name).nets]
                for name in NETS}
        out = {'networks': nets}
        for name in OPTS:
            d = getattr(self, name).state_dict()
            out[name] = dict(d, state={j: {k: v.clone() for k, v in st.items()} for j, st in d['state'].items()})
        return out

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Takes over a ``state_dict`` of Learners with the same networks and ``state_bits``; the arrays stay where they are, so
        a recording goes on with them."""
        self.check()
        have = {name: [net.state_dict() for net in getattr(self, name).nets] for name in NETS}
        for name in NETS:
            got = state_dict['networks'][name]
            if [{k: v.shape for k, v in d.items()} for d in got] != [{k: v.shape for k, v in d.items()} for d in have[name]]:
                raise ValueError('Learners: the state dict is of other networks (%s)' % name)
        for name in OPTS:                                       # all of it or nothing
            getattr(self, name).fits(state_dict[name])
        for name in OPTS:
            getattr(self, name).load_state_dict(state_dict[name])
        for name in NETS:
            for mine, got in zip(have[name], state_dict['networks'][name]):
                for k, v in mine.items():
                    v.copy_(got[k])
        self._repack()

    def written(self):
        """For autograd: every network was written."""
        for name in NETS:
            getattr(self, name).written()

    def _repack(self):
        for tr in self.trainers:                                # refilled in place: recorded acting steps read it
            if tr._packed is not None:
                maddpg.pack_actor(tr.p, out=tr._packed)

    def check(self):
        """Raises where a trainer's networks are no longer the ones that are updated here."""
        for name in NETS:
            getattr(self, name).check([getattr(tr, name) for tr in self.trainers])

    def draw(self):
        """Every learner's batch indices, [n, batch]."""
        return torch.stack([tr.replay_buffer.make_index(self.batch) for tr in self.trainers])

    def due(self, t):
        """Whether the trainers' two gates are open (maddpg.py:162-164)."""
        return t % 100 == 0 and all(len(tr.replay_buffer) >= tr.max_replay_buffer_len for tr in self.trainers)

    def update(self, t):
        """``[tr.update(trainers, t) for tr in trainers]`` at once: every trainer's [q_loss, p_loss, mean(target_q), mean(rew),
        mean(target_q_next), std(target_q)] as device scalars, or None when no update is due."""
        if not self.due(t):
            return None
        index = self.draw()
        for tr, idx in zip(self.trainers, index):
            tr.replay_sample_index = idx
        return self.update_from_index(index)

    @torch.no_grad()
    def update_from_index(self, index):
        """The update for the batches ``index`` [n, batch] (device int64), behind its gates."""
        n, b = self.n, self.batch
        if tuple(index.shape) != (n, b):
            raise ValueError('Learners: index is [%d, %d], got %s' % (n, b, list(index.shape)))
        self.check()
        flat = index.reshape(-1)
        obs_n, act_n, rew_n, next_n, done_n = zip(*[tr.replay_buffer.sample_index(flat) for tr in self.trainers])   # maddpg.py:173-177
        rew = torch.cat([self._rows(r, i) for i, r in enumerate(rew_n)])
        done = torch.cat([self._rows(d, i) for i, d in enumerate(done_n)])
        wide_p = self.p.w[0].shape[2]

        # targets (maddpg.py:181-187): every agent's target action for every learner's batch, then every learner's critic
        logits = self.target_p.forward(torch.cat([self._wide([o], wide_p) for o in next_n]), self.ends_all)[3]
        sample = self._sample(logits.view(n, n * b, -1))
        act_next = [sample[j, :, :a] for j, a in enumerate(self.acts)]
        target_next = self.target_q.forward(self._critic_input(next_n, act_next, self.target_q), self.ends)[3][:, 0]
        target = rew + self.gamma * (1.0 - done) * target_next

        # q_train (maddpg.py:75-110): mean squared Bellman error
        x = self._critic_input(obs_n, act_n, self.q)
        acts = self.q.forward(x, self.ends)
        err = acts[3][:, 0] - target
        q_loss = err.square().view(n, b).mean(1)
        self._step(self.q_opt, self.q.gradients(acts, (err * (2.0 / b)).unsqueeze(1), self.ends))

        # p_train (maddpg.py:28-73): -mean Q with the learner's own action replaced by a fresh sample, + 1e-3 mean(logits^2)
        own_obs = torch.cat([self._wide([self._rows(o, i)], wide_p) for i, o in enumerate(obs_n)])
        pol = self.p.forward(own_obs, self.ends)
        logits = pol[3].view(n, b, -1)
        sample = self._sample(logits)
        x2 = x.view(n, b, -1).clone()
        for i, a in enumerate(self.acts):
            x2[i, :, self.first[i]:self.first[i] + a] = sample[i, :, :a]
        acts = self.q.forward(x2.view(n * b, -1), self.ends)
        w_own = self.q.w[0].gather(2, self.cols.unsqueeze(1).expand(-1, self.q.w[0].shape[1], -1))
        dq = torch.full((n * b, 1), -1.0 / b, device=self.device)
        da = self.q.to_columns(acts, dq, self.ends, w_own).view(n, b, -1) * self.real.unsqueeze(1)
        width = self.real.sum(1).view(n, 1, 1)
        dlogits = self._softmax_backward(sample, da) + logits * self.real.unsqueeze(1) * (2e-3 / b / width)
        p_loss = -acts[3].view(n, b).mean(1) + 1e-3 * (logits.square() * self.real.unsqueeze(1)).sum((1, 2)) / (b * width.view(n))
        self._step(self.p_opt, self.p.gradients(pol, dlogits.reshape(n * b, -1), self.ends))
        self._repack()
        self.written()

        tq, tn = target.view(n, b), target_next.view(n, b)
        stats = torch.stack([q_loss, p_loss, tq.mean(1), rew.view(n, b).mean(1), tn.mean(1), tq.std(1, unbiased=False)], 1)
        return [list(row) for row in stats]

    @staticmethod
    def _step(opt, grads):
        flat = [g[i] for g in grads for i in range(g.shape[0])]
        for p, g in zip(opt.param_groups[0]['params'], flat):
            p.grad = g
        opt.step()
        for p in opt.param_groups[0]['params']:
            p.grad = None
