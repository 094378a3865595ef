"""What is measured of the sequence and loss operators that also take 16-bit storage:

* the gated linear recurrence (ops.linear_rnn: training, forward and backward; ops.linear_rnn_step: one decoding step),
* the losses of projected logits that never form the (rows, vocabulary) array: softmax cross-entropy on 16-bit tensors
  (ops.proj_ce) and distillation from a teacher's top logits beside it (ops.proj_distill).

`own` false: plain torch formulas in 32 bits.  `own` true: the framework's operators, called as a training loop or a
decoding loop calls them."""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
PAD = 0


@functools.lru_cache(maxsize=None)
def _ops():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'coupled-vae_amd'))
    from cvae_amd import _lib, ops
    _lib.init()
    return ops


# ------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # a decoder layer of the Yelp text model in place of its LSTM (batch 32, hidden 512): right-padded sentences
        dict(name='rnn_yelp_f32', op='rnn', T=110, B=32, H=512, gates=3, dtype='f32', reverse=False, shortest=20),
        # the backward direction of an encoder, sizes that are no multiple of anything, without an output gate
        dict(name='rnn_odd_reverse_f16', op='rnn', T=1001, B=3, H=203, gates=2, dtype='f16', reverse=True, shortest=1),
        # few long documents: the work of one channel is long, the channels are few
        dict(name='rnn_long_bf16', op='rnn', T=8192, B=2, H=1000, gates=3, dtype='bf16', reverse=False, shortest=6000),
        # the largest: the scale-up decoder's hidden size over long rows
        dict(name='rnn_scaleup_bf16', op='rnn', T=2000, B=32, H=2048, gates=3, dtype='bf16', reverse=False,
             shortest=1000),
        # one token of interactive generation, and one token of a large serving batch
        dict(name='step_small_f32', op='step', B=4, H=512, gates=3, dtype='f32'),
        dict(name='step_batch_bf16', op='step', B=512, H=2048, gates=3, dtype='bf16'),
        # one training step's loss of the PTB text model held in 16 bits
        dict(name='ce_ptb_bf16', op='ce', B=32, T=45, E=200, V=10002, dtype='bf16', shortest=8),
        # a wide model over the scale-up vocabulary: the largest products
        dict(name='ce_wide_bf16', op='ce', B=16, T=256, E=1024, V=50000, dtype='bf16', shortest=200),
        # a handful of tokens, odd sizes everywhere
        dict(name='kd_small_odd_f16', op='kd', B=5, T=7, E=75, V=1003, K=5, tau=1.5, dtype='f16', shortest=1),
        # distillation of the Yelp model from the top 32 logits of a larger teacher, in the framework's own 32 bits
        dict(name='kd_yelp_f32', op='kd', B=32, T=110, E=200, V=20000, K=32, tau=2.0, dtype='f32', shortest=20),
        # the same in 16 bits at the scale-up vocabulary and batch
        dict(name='kd_scaleup_bf16', op='kd', B=64, T=120, E=200, V=50000, K=64, tau=2.0, dtype='bf16', shortest=30),
    ]


RNN_MOST = 2000 * 32 * 2048         # elements of one gate in the largest listed recurrence
LOSS_MOST = 16 * 256 * 1024 * 50000   # rows x width x vocabulary of the largest listed loss


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.499)))))))


def draw(rng):
    op = rng.choice(['rnn', 'rnn', 'step', 'ce', 'kd', 'kd'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'step':
        return dict(op=op, B=_log_int(rng, 1, 512), H=_log_int(rng, 33, 2048), gates=rng.choice([2, 3]), dtype=dtype)
    if op == 'rnn':
        B, H = _log_int(rng, 1, 64), _log_int(rng, 33, 2048)
        most = min(8192, RNN_MOST // ((2 if dtype == 'f32' else 1) * B * H))
        T = _log_int(rng, 1, most)
        return dict(op=op, T=T, B=B, H=H, gates=rng.choice([2, 3]), dtype=dtype, reverse=rng.random() < 0.4,
                    shortest=rng.randint(1, T))
    if op == 'ce':
        dtype = rng.choice(['bf16', 'f16'])
    E, V, B = _log_int(rng, 24, 1024), _log_int(rng, 500, 50000), _log_int(rng, 1, 64)
    most = min(400, LOSS_MOST // ((3 if dtype == 'f32' else 1) * (2 if op == 'kd' else 1) * E * V * B))
    T = _log_int(rng, 1, max(1, most))
    case = dict(op=op, B=B, T=T, E=E, V=V, dtype=dtype, shortest=rng.randint(1, T))
    if op == 'kd':
        case.update(K=_log_int(rng, 1, 64), tau=rng.choice([1.0, 1.5, 2.0, 4.0]))
    return case


def _lengths(case):
    """B row lengths, evenly spread from the longest (T) to the shortest."""
    T, B, lo = case['T'], case['B'], case['shortest']
    return [T - (T - lo) * i // max(1, B - 1) for i in range(B)]


# ------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    dt = DTYPES[case['dtype']]
    st = dict(case=case)
    if case['op'] == 'step':
        B, H, G = case['B'], case['H'], case['gates']
        st.update(u=rnd(B, G * H).to(dt), h=torch.tanh(rnd(B, H)))
        return st
    T, B = case['T'], case['B']
    length = torch.tensor(_lengths(case), device=dev)[torch.randperm(B, generator=g, device=dev)]
    if case['op'] == 'rnn':
        H, G = case['H'], case['gates']
        u = rnd(T, B, G * H)
        u[:, :, :H] += 2.0               # forget gates that keep most of the state, as trained ones do
        st.update(u=u.to(dt), h0=torch.tanh(rnd(B, H)), length=length, dy=rnd(T, B, H).to(dt), dlast=rnd(B, H))
        return st
    E, V = case['E'], case['V']
    st['final'] = torch.tanh(rnd(T, B, E)).to(dt)
    st['W'] = (rnd(V, E) * (1.5 / math.sqrt(E))).to(dt)
    st['b'] = (rnd(V) * 0.1).to(dt)
    eos = torch.randint(1, V, (B, T), generator=g, device=dev)
    st['eos'] = torch.where(torch.arange(T, device=dev)[None] < length[:, None], eos, PAD)
    st['g_hard'] = torch.rand(B, generator=g, device=dev) / B
    if case['op'] == 'kd':
        K = case['K']
        step = max(1, V // K)
        # K different ids a position, the teacher's logits falling; some rows list fewer entries than K (-inf)
        ids = torch.randint(0, V, (B, T, 1), generator=g, device=dev) + torch.arange(K, device=dev) * step
        st['ids'] = ids % V
        top = torch.sort(rnd(B, T, K) * 3.0, dim=2, descending=True)[0]
        few = torch.randint(1, 4 * K, (B, T, 1), generator=g, device=dev)
        st['teacher'] = torch.where(torch.arange(K, device=dev) < few, top, float('-inf'))
        st['g_soft'] = torch.rand(B, generator=g, device=dev) / B
    return st


# ------------------------------------------------------------------------------------------------------ plain forms
def _scan(a, x):
    """y[t] = a[t] y[t-1] + x[t] along dim 0 from y = 0, by doubling: after a round every entry covers twice the steps."""
    d = 1
    while d < a.shape[0]:
        x = torch.cat([x[:d], x[d:] + a[d:] * x[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return x


def _gates(u, H):
    u = u.float()
    z, n = torch.sigmoid(u[..., :H]), torch.tanh(u[..., H:2 * H])
    o = torch.sigmoid(u[..., 2 * H:]) if u.shape[-1] == 3 * H else torch.ones_like(z)
    return z, n, o


def _step_plain(st):
    H = st['case']['H']
    z, n, o = _gates(st['u'], H)
    h = z * st['h'] + (1 - z) * n
    return dict(y=(o * h).to(st['u'].dtype), h=h)


def _rnn_plain(st):
    case, u, h0 = st['case'], st['u'], st['h0']
    T, H, G = case['T'], case['H'], case['gates']
    # every row in the order that it is walked in; a reversed row starts at its own last token
    live = (torch.arange(T, device=u.device)[:, None] < st['length'][None])[..., None]
    u, dy = (u.flip(0), st['dy'].flip(0)) if case['reverse'] else (u, st['dy'])
    live = live.flip(0) if case['reverse'] else live
    z, n, o = _gates(u, H)
    dy = dy.float() * live
    a = torch.where(live, z, 1.0)
    x = torch.where(live, (1 - z) * n, 0.0)
    x = torch.cat([x[:1] + a[:1] * h0, x[1:]])
    h = _scan(a, x)
    prev = torch.cat([h0[None], h[:-1]])
    y = torch.where(live, o * h, 0.0)
    # delta[t] = dL/dh[t]: what leaves through y[t], and what comes back from the next step
    late = torch.cat([dy[:-1] * o[:-1], dy[-1:] * o[-1:] + st['dlast']])
    back = torch.cat([torch.ones_like(a[:1]), a.flip(0)[:-1]])
    delta = _scan(back, late.flip(0)).flip(0)
    du = [delta * (prev - n) * z * (1 - z), delta * (1 - z) * (1 - n * n)]
    du = torch.cat(du + [dy * h * o * (1 - o)] if G == 3 else du, 2) * live
    dh0 = a[0] * delta[0]
    if case['reverse']:
        y, du = y.flip(0), du.flip(0)
    return dict(y=y.to(u.dtype), h_last=h[-1], du=du.to(u.dtype), dh0=dh0)


def _lse(x):
    m = x.max(1, keepdim=True)[0]
    return (m + torch.log(torch.exp(x - m).sum(1, keepdim=True)))


def _loss_plain(st):
    case, dt = st['case'], st['final'].dtype
    T, B, E = st['final'].shape
    x, W = st['final'].float().reshape(T * B, E), st['W'].float()
    tgt = st['eos'].t().reshape(T * B, 1)
    live = (tgt != PAD).float()
    logits = x @ W.t() + st['b'].float()
    lse = _lse(logits)
    hard = ((lse - logits.gather(1, tgt)) * live).reshape(T, B).sum(0)
    gh = st['g_hard'].repeat(T)[:, None] * live
    d = gh * torch.exp(logits - lse)
    d.scatter_add_(1, tgt, -gh)
    out = dict(hard=hard)
    if case['op'] == 'kd':
        K, tau = case['K'], case['tau']
        ids = st['ids'].transpose(0, 1).reshape(T * B, K)
        t = st['teacher'].transpose(0, 1).reshape(T * B, K) / tau
        lp = t - _lse(t)
        p = torch.exp(lp)
        s = logits / tau
        lse_s = _lse(s)
        term = torch.where(p > 0, p * (torch.where(p > 0, lp, 0.0) - s.gather(1, ids) + lse_s), 0.0)
        out['soft'] = (tau * tau * term.sum(1, keepdim=True) * live).reshape(T, B).sum(0)
        gs = st['g_soft'].repeat(T)[:, None] * live * tau
        d += gs * torch.exp(s - lse_s)
        d.scatter_add_(1, ids, -gs * p)
    out.update(dfinal=(d @ W).reshape(T, B, E).to(dt), dW=(d.t() @ x).to(dt), db=d.sum(0).to(dt))
    return out


# ------------------------------------------------------------------------------------------------------ one pass
def run(st):
    op = st['case']['op']
    if not own:
        return {'step': _step_plain, 'rnn': _rnn_plain, 'ce': _loss_plain, 'kd': _loss_plain}[op](st)
    ops, case = _ops(), st['case']
    if op == 'step':
        y, h = ops.linear_rnn_step(st['u'], case['gates'], st['h'])
        return dict(y=y, h=h)
    if op == 'rnn':
        u, h0 = st['u'].detach().requires_grad_(), st['h0'].detach().requires_grad_()
        y, last = ops.linear_rnn(u, case['gates'], h0=h0, length=st['length'], reverse=case['reverse'])
        du, dh0 = torch.autograd.grad([y, last], [u, h0], [st['dy'], st['dlast']])
        return dict(y=y.detach(), h_last=last.detach(), du=du, dh0=dh0)
    leaves = [st[k].detach().requires_grad_() for k in ('final', 'W', 'b')]
    if op == 'ce':
        hard = ops.proj_ce(*leaves, st['eos'], PAD)
        grads = torch.autograd.grad([hard], leaves, [st['g_hard']])
        out = dict(hard=hard.detach())
    else:
        hard, soft = ops.proj_distill(*leaves, st['eos'], PAD, st['ids'], st['teacher'], case['tau'])
        grads = torch.autograd.grad([hard, soft], leaves, [st['g_hard'], st['g_soft']])
        out = dict(hard=hard.detach(), soft=soft.detach())
    out.update(zip(('dfinal', 'dW', 'db'), grads))
    return out


# ------------------------------------------------------------------------------------------------------ what it takes
def work(case):
    w = 4 if case['dtype'] == 'f32' else 2
    if case['op'] == 'step':
        n, G = case['B'] * case['H'], case['gates']
        return dict(bytes=n * ((G + 1) * w + 8), flops=n * (10 * G + 5))
    tokens = sum(_lengths(case))
    if case['op'] == 'rnn':
        B, H, G = case['B'], case['H'], case['gates']
        full = case['T'] * B * H
        return dict(bytes=tokens * H * (G + 1) * w + full * (G + 1) * w + 16 * B * H, flops=tokens * H * (20 * G + 20))
    E, V, N = case['E'], case['V'], case['B'] * case['T']
    size = (2 * V * (E + 1) + (tokens + N) * E) * w + 8 * N + 8 * case['B']
    return dict(bytes=size + tokens * 12 * case.get('K', 0), flops=6 * tokens * E * V)


# ------------------------------------------------------------------------------------------------------ 64 bits
def _exact_rnn(st):
    case = st['case']
    H, T, B = case['H'], case['T'], case['B']
    u, dy, h0 = st['u'].double(), st['dy'].double(), st['h0'].double()
    one = torch.ones((), dtype=torch.float64, device=u.device)
    alive = [st['length'] > t for t in range(T)]
    order = list(range(T - 1, -1, -1) if case['reverse'] else range(T))
    f = 1 / (1 + torch.exp(-u[:, :, :H]))
    c = torch.tanh(u[:, :, H:2 * H])
    o = 1 / (1 + torch.exp(-u[:, :, 2 * H:])) if case['gates'] == 3 else one.expand(T, B, H)
    y, du, states, h = torch.zeros_like(dy), torch.zeros_like(u), {}, h0
    for t in order:
        m = alive[t][:, None]
        states[t] = h
        h = torch.where(m, f[t] * h + (1 - f[t]) * c[t], h)
        y[t] = torch.where(m, o[t] * h, 0)
    last, back = h, st['dlast'].double()
    for t in reversed(order):
        m = alive[t][:, None]
        before = states.pop(t)
        h = f[t] * before + (1 - f[t]) * c[t]
        g = back + dy[t] * o[t]
        parts = [g * (before - c[t]) * f[t] * (1 - f[t]), g * (1 - f[t]) * (1 - c[t] ** 2)]
        if case['gates'] == 3:
            parts.append(dy[t] * h * o[t] * (1 - o[t]))
        du[t] = torch.where(m, torch.cat(parts, 1), 0)
        back = torch.where(m, g * f[t], back)
    return dict(y=y, h_last=last, du=du, dh0=back)


def _exact_loss(st):
    case = st['case']
    dev = st['eos'].device
    leaves = [st[k].double().requires_grad_() for k in ('final', 'W', 'b')]
    sent, pos = torch.nonzero(st['eos'] != PAD, as_tuple=True)
    logits = torch.nn.functional.linear(leaves[0][pos, sent], leaves[1], leaves[2])
    row = -torch.log_softmax(logits, 1)[torch.arange(len(sent), device=dev), st['eos'][sent, pos]]
    out = dict(hard=torch.zeros(case['B'], dtype=torch.float64, device=dev).index_add(0, sent, row))
    back = [st['g_hard'].double()]
    if case['op'] == 'kd':
        tau = case['tau']
        p = torch.softmax(st['teacher'][sent, pos].double() / tau, 1)
        lq = torch.log_softmax(logits / tau, 1).gather(1, st['ids'][sent, pos])
        row = tau ** 2 * (torch.special.xlogy(p, p) - p * lq).sum(1)
        out['soft'] = torch.zeros_like(out['hard']).index_add(0, sent, row)
        back.append(st['g_soft'].double())
    grads = torch.autograd.grad(list(out.values()), leaves, back)
    out = {k: v.detach() for k, v in out.items()}
    out.update(zip(('dfinal', 'dW', 'db'), grads))
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'step':
        H, u = case['H'], st['u'].double()
        f = 1 / (1 + torch.exp(-u[:, :H]))
        h = torch.lerp(torch.tanh(u[:, H:2 * H]), st['h'].double(), f)
        y = h / (1 + torch.exp(-u[:, 2 * H:])) if case['gates'] == 3 else h.clone()
        return dict(y=y, h=h)
    return _exact_rnn(st) if case['op'] == 'rnn' else _exact_loss(st)
