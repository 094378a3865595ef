"""Losses of projected logits (ops.proj_distill, ops.proj_ce on 16-bit tensors) against float64 formulas.

Tolerances, u = 2^-24, carried through the formulas in float64 beside the values:
 * a logit: fp32 operands are hi + lo fp16 planes.  fp16 has 11 significant bits, so half a step is 2^-11 of the value
   (1 + 2^-11 lies midway between two neighbours): |lo| <= 2^-11 |x|, rounded by 2^-11 of itself: 2^-22 = 4 u, for each
   operand, and lo.lo, which is dropped, is 2^-22 of the product: 12 u |x w|.  16-bit operands are exact.  E products
   added in fp32: (E + 20) u sum |x w| covers both, and the bias;
 * a normaliser: its logits' error, V / 4 + 64 additions in a row, base-2 logits (|lse| + |S| rounded a few times);
 * an entry of d loss / d S = g q: |g q| (error of its exponent) and the rounding of its storage, half a step as above:
   2^-11 (bf16: one plane) or 2^-22 (fp32 and fp16: two) of it, and of its row's |g| half of fp16's smallest, 2^-25, over the 2^13 that it
   is stored times, for a row's power of two up to twice |g|: 2^-37;
 * a gradient: those entries times the operand (12 u as for a logit), N or V additions in fp32, half a step of the output
   type.
Worst cases added up are far from what happens, so fp32 results are also held in norm to root-mean-square growth."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
PAD = 0


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'GPU tests need an MI355X'
    from cvae_amd import _lib
    _lib.init(0)
    return torch.device('cuda:0')


def inputs(T, R, B, E, V, K, dtype, seed, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    a = dict(final=torch.tanh(torch.randn(T, R, E, generator=g)), W=torch.randn(V, E, generator=g) * scale / math.sqrt(E),
             b=torch.randn(V, generator=g) * 0.2)
    a = {k: v.to(DT[dtype]) for k, v in a.items()}
    eos = torch.randint(1, max(V, 2), (B, T), generator=g)
    length = torch.randint(0, T + 1, (B,), generator=g)
    length[0] = T
    a['eos'] = torch.where(torch.arange(T)[None] < length[:, None], eos, PAD)
    a['gh'] = torch.randn(R, generator=g)
    if K:
        a['ids'] = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(B * T)]).reshape(B, T, K)
        a['top'] = torch.randn(B, T, K, generator=g) * 3
        a['gs'] = torch.randn(R, generator=g)
    return a


def oracle(a, tau, tgt=None):
    """{name: (value, bound)} in float64 on the CPU."""
    x0, W, b = (a[k].detach().double().cpu() for k in ('final', 'W', 'b'))
    T, R, E = x0.shape
    V = W.shape[0]
    B = a['eos'].shape[0]
    np1 = a['final'].dtype == torch.bfloat16                              # one plane of P, else two
    if tgt is None:
        tgt = a['eos'].cpu().t().repeat(1, R // B)                        # (T,R), row r reads sentence r % B
    live = tgt != PAD
    x = x0.reshape(T * R, E)[live.reshape(-1)]
    t = tgt.reshape(-1)[live.reshape(-1)]
    sent = torch.arange(R).repeat(T)[live.reshape(-1)]
    N = len(t)
    S = x @ W.t() + b
    eS = (E + 20) * U * (x.abs() @ W.abs().t() + torch.where(b.isfinite(), b.abs(), 0.0))
    inside = (t >= 0) & (t < V)
    t0 = t.clamp(0, V - 1)
    onehot = torch.zeros_like(S)
    if N:
        onehot[torch.arange(N), t0] = inside.double()
    Sf = torch.where(S.isfinite(), S.abs(), 0.0)

    def lse_of(Z, eZ):
        L = torch.logsumexp(Z, 1)
        q = torch.exp(Z - L[:, None])
        return L, q, eZ.amax(1) + (V / 4 + 64) * U + 8 * U * (L.abs() + Sf.amax(1)) if N else (L, q, torch.zeros(0))
    if N == 0:
        zero = lambda *s: (torch.zeros(*s, dtype=torch.float64), torch.zeros(*s, dtype=torch.float64))
        out = dict(hard=zero(R), dfinal=zero(T, R, E), dW=zero(V, E), db=zero(V))
        if 'ids' in a:
            out['soft'] = zero(R)
        return out
    L, q, eL = lse_of(S, eS)
    St = torch.where(inside, S.gather(1, t0[:, None])[:, 0], 0.0)
    hard = L - St
    ehard = eL + torch.where(inside, eS.gather(1, t0[:, None])[:, 0], 0.0) + 8 * U * (L.abs() + St.abs())
    add = lambda v: torch.zeros(R, dtype=torch.float64).index_add(0, sent, v)
    out = dict(hard=(add(hard), add(ehard) + T * U * add(hard.abs())))
    gh = a['gh'].double()[sent][:, None]
    P = gh * (q - onehot)
    eP = gh.abs() * q * (eS + eL[:, None] + 16 * U * (1 + Sf + L.abs()[:, None]))
    mag = gh.abs()
    if 'ids' in a:
        row = torch.nonzero(live)                                         # (t, r)
        ids = a['ids'].cpu()[row[:, 1] % B, row[:, 0]]
        top = a['top'].double().cpu()[row[:, 1] % B, row[:, 0]]
        ok = (ids >= 0) & (ids < V)
        top = torch.where(ok, top, float('-inf')) / tau
        some = (top > float('-inf')).any(1)
        p = torch.where(some[:, None], torch.softmax(torch.where(some[:, None], top, 0.0), 1), 0.0)
        id0 = ids.clamp(0, V - 1)
        Lt, qt, eLt = lse_of(S / tau, eS / tau)
        term = torch.special.xlogy(p, p) - torch.where(p > 0, p * (S.gather(1, id0) / tau - Lt[:, None]), 0.0)
        eterm = p * (eS.gather(1, id0) / tau + eLt[:, None] + 40 * U * (1 + Sf.gather(1, id0) / tau + Lt.abs()[:, None] +
                                                                    torch.where(p > 0, torch.log(p).abs(), 0.0)))
        soft, esoft = tau ** 2 * term.sum(1), tau ** 2 * (eterm.sum(1) + 16 * U * term.abs().sum(1))
        out['soft'] = (add(soft), add(esoft) + T * U * add(soft.abs()))
        gs = a['gs'].double()[sent][:, None] * tau
        share = torch.zeros_like(S).scatter_add_(1, id0, torch.where(ok, p, 0.0))
        P = P + gs * (some[:, None] * qt - share)
        eP = eP + gs.abs() * (some[:, None] * qt * (eS / tau + eLt[:, None] + 16 * U * (1 + Sf / tau + Lt.abs()[:, None])) + 40 * U * share)
        mag = mag + gs.abs()
    eP = eP + (2.0 ** -11 if np1 else 2.0 ** -22) * P.abs() + 2.0 ** -37 * mag + 8 * U * P.abs()
    dx, edx = P @ W, eP @ W.abs() + (V + 28) * U * (P.abs() @ W.abs())
    full = lambda v: torch.zeros(T * R, E, dtype=torch.float64).index_copy(0, torch.nonzero(live.reshape(-1))[:, 0], v).reshape(T, R, E)
    out['dfinal'] = (full(dx), full(edx))
    gmax = mag.max()
    out['dW'] = (P.t() @ x, eP.t() @ x.abs() + (N + 28) * U * (P.abs().t() @ x.abs()) + 2.0 ** -37 * gmax * x.abs().max() * (P.abs() / mag.clamp_min(1e-300)).sum(0)[:, None])
    out['db'] = (P.sum(0), eP.sum(0) + (N + 28) * U * P.abs().sum(0))
    return out


def check(got, want, name, E, V, N):
    value, bound = want
    a = got.detach().double().cpu()
    assert a.shape == value.shape, name
    assert bool(torch.isfinite(a).all()), name
    fi = torch.finfo(got.dtype)
    tol = bound * 1.01 + fi.eps / 2 * (value.abs() + bound) + (fi.tiny * fi.eps if got.dtype != torch.float32 else 1e-37)
    over = (a - value).abs() > tol
    assert not bool(over.any()), '%s: %d of %d outside, worst %.3g over %.3g' % (
        name, int(over.sum()), over.numel(), float((a - value).abs()[over].max()), float(tol[over].max()))
    if got.dtype == torch.float32 and float(value.norm()) > 0:
        rms = (math.sqrt(E) + math.sqrt(max(V, N)) + 64) * U
        size = float((value.abs() + bound / ((max(E, V, N) + 16) * U) * 0.02).norm())
        assert float((a - value).norm()) <= 2 * rms * size, (name, float((a - value).norm()) / float(value.norm()))


def run(dev, a, tau, ops_name='distill'):
    from cvae_amd import ops
    leaves = [a[k].to(dev).detach().requires_grad_() for k in ('final', 'W', 'b')]
    eos = a['eos'].to(dev)
    if 'ids' in a:
        hard, soft = ops.proj_distill(*leaves, eos, PAD, a['ids'].to(dev), a['top'].to(dev), tau)
        grads = torch.autograd.grad([hard, soft], leaves, [a['gh'].to(dev), a['gs'].to(dev)])
        out = dict(hard=hard, soft=soft)
    else:
        hard = (ops.proj_ce if ops_name == 'distill' else ops.proj_ce_sorted)(*leaves, eos, PAD)
        grads = torch.autograd.grad([hard], leaves, [a['gh'].to(dev)])
        out = dict(hard=hard)
    out.update(zip(('dfinal', 'dW', 'db'), grads))
    return out


def compare(dev, a, tau, **kw):
    got, want = run(dev, a, tau, **kw), oracle(a, tau)
    T, R, E = a['final'].shape
    for k in got:
        check(got[k], want[k], k, E, a['W'].shape[0], T * R)
    return got


# one token, one word; odd everything; widths around the image's 64 and the tile's 128 columns; vocabularies around a tile;
# more than one tile of rows; more splits than tiles
SIZES = [(1, 1, 1, 1, 1, 1), (3, 2, 2, 8, 5, 5), (7, 5, 5, 75, 1003, 5), (4, 3, 3, 63, 127, 2), (4, 3, 3, 64, 128, 16),
         (5, 2, 2, 127, 129, 3), (2, 4, 2, 128, 300, 7), (3, 3, 3, 200, 513, 33), (11, 14, 7, 37, 260, 64),
         (30, 12, 12, 201, 1500, 4), (2, 1, 1, 513, 400, 9), (3, 2, 2, 24, 1030, 1024), (2, 2, 2, 300, 640, 130)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('tau', [1.0, 2.5])
@pytest.mark.parametrize('size', SIZES)
def test_distillation(dev, size, tau, dtype):
    compare(dev, inputs(*size, dtype, sum(size)), tau)


# the last tile of E around what its waves share differently (96, 224 columns, and one more for the bias), alone and behind
# whole tiles; a vocabulary whose tiles leave part of the chip free
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('size', [(20, 7, 7, 95, 900, 3), (20, 7, 7, 96, 900, 3), (20, 7, 7, 223, 900, 2), (20, 7, 7, 224, 900, 2),
                                  (9, 4, 4, 225, 700, 2), (9, 4, 4, 352, 700, 2), (9, 4, 4, 480, 700, 2),
                                  (32, 8, 8, 200, 20000, 4)])
def test_partly_filled_tiles(dev, size, dtype):
    compare(dev, inputs(*size, dtype, sum(size)), 2.0)


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
@pytest.mark.parametrize('size', SIZES)
def test_cross_entropy_16_bit(dev, size, dtype):
    compare(dev, inputs(*size[:5], 0, dtype, sum(size)), 1.0)


def test_cross_entropy_sorted_rows(dev):
    """Sentence-major rows r = b K + k: targets of sentence r / K."""
    T, R, B, E, V = 6, 12, 4, 40, 333
    a = inputs(T, R, B, E, V, 0, 'bf16', 3)
    tgt = a['eos'].t().repeat_interleave(R // B, dim=1)
    got, want = run(dev, a, 1.0, ops_name='sorted'), oracle(a, 1.0, tgt)
    for k in got:
        check(got[k], want[k], k, E, V, T * R)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_absent_repeated_and_shared_entries(dev, dtype):
    """Ids outside the vocabulary, logits of -inf and of the type's lowest value, rows with no entry at all, one id listed
    several times, the target among the teacher's entries, a target outside the vocabulary."""
    T, B, E, V, K = 6, 4, 48, 200, 6
    a = inputs(T, B, B, E, V, K, dtype, 8)
    a['eos'][1, 0], a['eos'][2, 0] = V + 5, -7
    a['eos'][0] = torch.arange(1, T + 1)
    a['eos'][3, 2:] = PAD
    a['eos'][3, 1] = 5
    a['ids'][0, :, 1] = a['eos'][0]                       # the target is an entry
    a['ids'][0, 1, :] = 17                                # one id, K times
    a['ids'][0, 2, 3:] = a['ids'][0, 2, 0]
    a['ids'][0, 3, :2] = torch.tensor([-1, V])
    a['ids'][1, 0, :] = V + 100
    a['top'][0, 4, 2:] = float('-inf')
    a['top'][0, 5, :] = float('-inf')
    a['top'][2, 0, 1:] = torch.finfo(torch.float32).min
    a['top'][3, 0, 3] = 1e4
    compare(dev, a, 2.0)
    compare(dev, a, 1.0)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_garbage_in_dropped_rows(dev, dtype):
    """NaN, infinities and huge numbers behind a sentence's end -- states, teacher, gradients of empty sentences -- reach
    nothing, not even the scale of the others."""
    T, B, E, V, K = 5, 4, 33, 150, 4
    a = inputs(T, B, B, E, V, K, dtype, 9)
    a['eos'][1, 2:] = PAD
    a['eos'][2] = PAD
    want = oracle(a, 2.0)
    dead = a['eos'].t() == PAD
    big = 6e4 if dtype == 'f16' else 1e30
    for junk in (float('nan'), float('inf'), big):
        b = {k: v.clone() for k, v in a.items()}
        b['final'][dead] = junk
        b['top'][a['eos'] == PAD] = junk
        b['ids'][a['eos'] == PAD] = 1 << 40
        b['gh'][2] = b['gs'][2] = junk if junk == big else 1e30
        got = run(dev, b, 2.0)
        for k in got:
            check(got[k], want[k], k, E, V, T * B)
        assert not bool(got['dfinal'][dead.to(dev)].any())


@pytest.mark.parametrize('K', [0, 3])
def test_nothing_live(dev, K):
    a = inputs(4, 3, 3, 20, 90, K, 'bf16', 1)
    a['eos'][:] = PAD
    got = run(dev, a, 2.0)
    for k, v in got.items():
        assert not bool(v.any()), k


def test_no_rows(dev):
    from cvae_amd import ops
    W, b = torch.randn(7, 4, device=dev).bfloat16().requires_grad_(), torch.zeros(7, device=dev).bfloat16()
    for T, R in ((0, 2), (3, 0)):
        final = torch.zeros(T, R, 4, device=dev).bfloat16()
        eos = torch.zeros(2, T, dtype=torch.int64, device=dev)
        hard = ops.proj_ce(final, W, b, eos, PAD)
        assert hard.shape == (R,) and not bool(hard.any())
        dW, = torch.autograd.grad([hard], [W], [torch.ones_like(hard)])
        assert not bool(dW.any())


def test_words_masked_by_their_bias(dev):
    """A bias of -inf takes words out of the vocabulary; a confident row (its softmax nearly one-hot); tiny and huge scales."""
    T, B, E, V, K = 3, 2, 16, 300, 3
    for dtype in ('f32', 'bf16'):
        a = inputs(T, B, B, E, V, K, dtype, 4)
        a['b'][200:] = float('-inf')
        a['eos'] = a['eos'] % 199 + 1
        a['ids'] = a['ids'] % 200
        got, want = run(dev, a, 2.0), oracle(a, 2.0)
        for k in got:
            check(got[k], want[k], k, E, V, T * B)
    a = inputs(T, B, B, E, V, K, 'f32', 5, scale=12.0)
    compare(dev, a, 2.0)
    for s in (2.0 ** -40, 2.0 ** 30):
        b = dict(a, final=a['final'] * s, W=a['W'] / s / 8)
        compare(dev, b, 2.0)


def test_strides_alignment_and_broadcast_upstream(dev):
    from cvae_amd import ops
    T, B, E, V, K = 5, 3, 24, 140, 4
    a = inputs(T, B, B, E, V, K, 'bf16', 6)
    a['gh'], a['gs'] = torch.full((B,), 0.25), torch.full((B,), 0.25)
    want = oracle(a, 1.5)
    store = torch.empty(V * E + 1, dtype=torch.bfloat16, device=dev)     # weights on an odd 2-byte address
    W = store[1:].view(V, E)
    W.copy_(a['W'])
    final = a['final'].to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    ids = a['ids'].to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    leaves = [final.requires_grad_(), W.requires_grad_(), a['b'].to(dev).requires_grad_()]
    hard, soft = ops.proj_distill(*leaves, a['eos'].to(dev), PAD, ids, a['top'].to(dev), 1.5)
    grads = torch.autograd.grad(0.25 * (hard.sum() + soft.sum()), leaves)
    got = dict(hard=hard, soft=soft, dfinal=grads[0], dW=grads[1], db=grads[2])
    for k in got:
        check(got[k], want[k], k, E, V, T * B)


def test_one_loss_alone_and_a_second_backward(dev):
    from cvae_amd import ops
    a = inputs(6, 4, 4, 40, 210, 5, 'f32', 7)
    leaves = [a[k].to(dev).requires_grad_() for k in ('final', 'W', 'b')]
    hard, soft = ops.proj_distill(*leaves, a['eos'].to(dev), PAD, a['ids'].to(dev), a['top'].to(dev), 2.0)
    for which, g in ((hard, 'gh'), (soft, 'gs')):
        only = dict(a)
        only['gh' if g == 'gs' else 'gs'] = torch.zeros(4)
        want = oracle(only, 2.0)
        for _ in range(2):
            grads = torch.autograd.grad([which], leaves, [a[g].to(dev)], retain_graph=True)
            for k, v in zip(('dfinal', 'dW', 'db'), grads):
                check(v, want[k], k, 40, 210, 24)


def test_only_the_gradients_that_are_wanted(dev):
    """Frozen weights, or a frozen decoder: the other gradients do not change."""
    from cvae_amd import ops
    a = inputs(6, 5, 5, 72, 900, 4, 'f32', 17)
    full = run(dev, a, 2.0)
    for wanted in (('final',), ('W', 'b'), ('W',), ('b', 'final')):
        leaves = {k: a[k].to(dev).requires_grad_(k in wanted) for k in ('final', 'W', 'b')}
        hard, soft = ops.proj_distill(*leaves.values(), a['eos'].to(dev), PAD, a['ids'].to(dev), a['top'].to(dev), 2.0)
        grads = torch.autograd.grad([hard, soft], [leaves[k] for k in wanted], [a['gh'].to(dev), a['gs'].to(dev)])
        for k, v in zip(wanted, grads):
            assert torch.equal(v, full['d' + k]), (wanted, k)


def test_a_teacher_that_is_not_a_number(dev):
    """A NaN among a row's teacher logits makes its sentence's soft loss NaN, and only that."""
    from cvae_amd import ops
    a = inputs(4, 3, 3, 16, 60, 4, 'f32', 18)
    a['eos'] = torch.where(a['eos'] == PAD, 3, a['eos'])
    a['top'][1, 2, 3] = float('nan')
    args = [a[k].to(dev) for k in ('final', 'W', 'b')]
    hard, soft = ops.proj_distill(*args, a['eos'].to(dev), PAD, a['ids'].to(dev), a['top'].to(dev), 2.0)
    assert bool(torch.isfinite(hard).all()) and torch.isnan(soft).tolist() == [False, True, False]


def test_gradient_against_differences(dev):
    """fp32, along one direction of W, b and final: the quotient of differences and the gradient agree within the e^2 term
    (measured by halving e) and the noise of the losses themselves (their derived bounds over e)."""
    from cvae_amd import ops
    T, B, E, V, K = 5, 3, 20, 90, 4
    a = inputs(T, B, B, E, V, K, 'f32', 12)
    got, bounds = run(dev, a, 2.0), oracle(a, 2.0)
    g = torch.Generator().manual_seed(2)
    d = {k: torch.randn(a[k].shape, generator=g) for k in ('final', 'W', 'b')}
    slope = sum(float((got['d' + k].double().cpu() * d[k]).sum()) for k in d)

    def loss(e):
        x = [(a[k] + e * d[k]).to(dev) for k in d]
        hard, soft = ops.proj_distill(*x, a['eos'].to(dev), PAD, a['ids'].to(dev), a['top'].to(dev), 2.0)
        return float((hard.double().cpu() * a['gh']).sum() + (soft.double().cpu() * a['gs']).sum())
    noise = float((bounds['hard'][1] * a['gh'].abs()).sum() + (bounds['soft'][1] * a['gs'].abs()).sum())
    quot = {e: (loss(e) - loss(-e)) / (2 * e) for e in (2e-2, 1e-2)}
    assert abs(quot[1e-2] - slope) <= abs(quot[2e-2] - quot[1e-2]) + 2 * noise / 1e-2 + 1e-4 * abs(slope)


def test_large_vocabulary_in_pieces(dev, monkeypatch):
    """Rows and words enough that the gradient is formed in more than one piece of the vocabulary (they are held to
    400 MiB), on a case whose float64 formulas still run on the GPU: N = 2600 rows, V = 45000, in fp16 storage."""
    from cvae_amd import _lib
    T, B, E, V, K = 65, 40, 24, 45000, 3
    assert 4 * 2816 * V > 400 << 20
    a = inputs(T, B, B, E, V, K, 'f16', 13)
    a['eos'] = torch.where(a['eos'] == PAD, 3, a['eos'])
    got = run(dev, a, 2.0)
    x, W, b = (a[k].to(dev).double().requires_grad_() for k in ('final', 'W', 'b'))
    logits = x @ W.t() + b
    tgt, ids = a['eos'].to(dev).t(), a['ids'].to(dev).transpose(0, 1)
    lq = torch.log_softmax(logits, 2)
    hard = -lq.gather(2, tgt[..., None])[..., 0].sum(0)
    p = torch.softmax(a['top'].to(dev).double().transpose(0, 1) / 2.0, 2)
    soft = (4.0 * (p * (torch.log(p) - torch.log_softmax(logits / 2.0, 2).gather(2, ids))).sum(2)).sum(0)
    want = dict(zip(('dfinal', 'dW', 'db'), torch.autograd.grad([hard, soft], [x, W, b], [a['gh'].to(dev).double(), a['gs'].to(dev).double()])))
    want.update(hard=hard, soft=soft)
    for k in got:
        # the rounding of the fp16 output, root mean square 2^-11 / sqrt(3) at most, and far smaller ones: under 2^-11;
        # fp32 losses: their logits' error, under 1e-6
        rel = float((got[k].detach().double() - want[k].detach()).norm() / want[k].detach().norm())
        assert rel < (1e-6 if k in ('hard', 'soft') else 2.0 ** -11), (k, rel)


def test_other_stream_and_repeatable(dev):
    a = inputs(30, 12, 12, 75, 1003, 6, 'bf16', 14)
    first = run(dev, a, 2.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(dev, a, 2.0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in first:
        assert torch.equal(first[k], again[k]), k


def test_captured_and_replayed(dev):
    """A training step's loss and gradients in one graph, replayed on new inputs with another number of live rows."""
    from cvae_amd import ops
    T, B, E, V, K = 12, 6, 40, 700, 5
    cur = {k: v.to(dev) for k, v in inputs(T, B, B, E, V, K, 'bf16', 1).items()}

    def work():
        leaves = [cur[k].detach().requires_grad_() for k in ('final', 'W', 'b')]
        hard, soft = ops.proj_distill(*leaves, cur['eos'], PAD, cur['ids'], cur['top'], 2.0)
        ce = ops.proj_ce(*leaves, cur['eos'], PAD)
        grads = torch.autograd.grad([hard, soft], leaves, [cur['gh'], cur['gs']])
        return [t.detach() for t in (hard, soft, ce, *grads)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (31, 32, 33, 34):
        new = inputs(T, B, B, E, V, K, 'bf16', seed)
        if seed == 33:
            new['eos'][:] = PAD
        for k in cur:
            cur[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, work()):
            assert torch.equal(x, y), seed


def test_a_text_decoder_of_the_new_operators(dev):
    """Embedded tokens -> gated linear recurrence -> cross-entropy and distillation, 16-bit, forward and backward together,
    against float64 autograd of the same model on the same (rounded) intermediate values."""
    from cvae_amd import ops
    T, B, H, V, K = 20, 6, 64, 500, 8
    g = torch.Generator().manual_seed(3)
    a = inputs(T, B, B, H, V, K, 'bf16', 15)
    u = (torch.randn(T, B, 3 * H, generator=g)).bfloat16().to(dev).requires_grad_()
    h0 = torch.randn(B, H, generator=g).to(dev).requires_grad_()
    W, b = a['W'].to(dev).requires_grad_(), a['b'].to(dev).requires_grad_()
    length = (a['eos'] != PAD).sum(1).to(dev)
    y, _ = ops.linear_rnn(u, 3, h0=h0, length=length)
    hard, soft = ops.proj_distill(y, W, b, a['eos'].to(dev), PAD, a['ids'].to(dev), a['top'].to(dev), 2.0)
    tot, _ = ops.loss_assemble([hard, soft], [0.5, 0.5])
    grads = torch.autograd.grad(tot, [u, h0, W, b])
    a['final'] = y.detach().cpu()                          # the loss is compared on the states it was given
    a['gh'] = a['gs'] = torch.full((B,), 0.5 / B)
    want = oracle(a, 2.0)
    check(hard, want['hard'], 'hard', H, V, T * B)
    check(soft, want['soft'], 'soft', H, V, T * B)
    check(grads[2], want['dW'], 'dW', H, V, T * B)
    check(grads[3], want['db'], 'db', H, V, T * B)
    # the recurrence's gradient, from the gradient of its output rounded to bf16 as autograd hands it over
    from test_gpu_linear_rnn import check as check_rnn, oracle as oracle_rnn
    dy = run(dev, a, 2.0)['dfinal']
    rnn = oracle_rnn(u, 3, h0, length, False, dy, torch.zeros(B, H))
    check_rnn(y, rnn['y'], 'y')
    check_rnn(grads[0], rnn['du'], 'du')
    check_rnn(grads[1], rnn['dh0'], 'dh0')


def test_most_rows_that_a_backward_pass_takes(dev):
    """2^22 rows of which 300 are live: offsets inside a tile of P pass 2^31 bytes.  The same 300 rows alone give the same bits."""
    from cvae_amd import ops
    T, R, E, V, K, n = 2048, 2048, 75, 250, 3, 300
    g = torch.Generator().manual_seed(4)
    small = inputs(1, n, n, E, V, K, 'f16', 41)
    small['eos'] = torch.randint(1, V, (n, 1), generator=g)
    big = dict(small, final=torch.zeros(T, R, E, dtype=torch.float16), eos=torch.full((R, T), PAD), gh=torch.zeros(R), gs=torch.zeros(R),
               ids=torch.zeros(R, T, K, dtype=torch.int64), top=torch.zeros(R, T, K))
    big['final'][T - 1, :n] = small['final'][0]
    for k in ('gh', 'gs'):
        big[k][:n] = small[k]
    for k in ('eos', 'ids', 'top'):
        big[k][:n, T - 1] = small[k][:, 0]
    want, got = run(dev, small, 2.0), run(dev, big, 2.0)
    for k in ('hard', 'soft'):
        assert torch.equal(got[k][:n], want[k]) and not got[k][n:].any(), k
    for k in ('dW', 'db'):
        assert torch.equal(got[k], want[k]), k
    assert torch.equal(got['dfinal'][T - 1, :n], want['dfinal'][0])
    assert not got['dfinal'][T - 1, n:].any() and not got['dfinal'][:T - 1].any()


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('E,V', [(20, 90), (200, 20000), (300, 700)])
def test_nothing_live_of_every_type(dev, E, V, dtype):
    """A batch of padding alone, by storage type and width: the number of live rows is known on the device only."""
    a = inputs(4, 3, 3, E, V, 3, dtype, 1)
    a['eos'][:] = PAD
    got = run(dev, a, 2.0)
    for k, v in got.items():
        assert not bool(v.any()), k


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('E,V', [(16, 300), (224, 300)])
def test_states_up_to_the_largest_float(dev, E, V, dtype):
    """A column of 2^127 that no word weighs, beside states near 2^95 and weights near 2^-95.  The images scale by 2^-114 and keep
    2^-25 of what is then the unit: a logit is off by 2^89 sum |w| at most, a loss and its logit's share in lse by twice that."""
    T, B, K, tau = 3, 2, 3, 2.0
    a = inputs(T, B, B, E, V, K, dtype, 21)
    a['eos'] = a['eos'] % (V - 1) + 1
    a['final'], a['W'] = a['final'] * 2.0 ** 95, a['W'] * 2.0 ** -95
    a['final'][:, :, 0], a['W'][:, 0] = 2.0 ** 127, 0.0
    a['gh'], a['gs'] = a['gh'] * 0.01, a['gs'] * 0.01                  # (dW's first column stays below the largest float)
    got, want = run(dev, a, tau), oracle(a, tau)
    off = 2 * 2.0 ** 89 * float(a['W'].double().abs().sum(1).max())
    for k, f in (('hard', 1.0), ('soft', tau)):                        # soft: tau^2 times a difference of logits over tau
        value, bound = want[k]
        assert bool(((got[k].detach().double().cpu() - value).abs() <= bound + f * T * off).all()), k
    for k, v in got.items():
        assert bool(torch.isfinite(v).all()), k


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('E', [24, 200, 224])
@pytest.mark.parametrize('tau', [2.0, 1.3])
def test_no_word_has_more_than_the_whole(dev, tau, E, dtype):
    """Logits so large that their rounding is more than what tells the best word from the normaliser: lse >= S[target] all the
    same, so no loss is negative, and no gradient outgrows its upstream one."""
    T, B, V, K = 4, 16, 300, 3
    for scale in (1e3, 1e4) if dtype == 'f16' else (1e3, 1e7, 1e12):
        a = inputs(T, B, B, E, V, K, dtype, 22, scale=scale)
        best = (a['final'].double() @ a['W'].double().t() + a['b'].double()).argmax(2).t().contiguous()     # (B,T)
        best[B // 2:] = (best[B // 2:] + 31) % V                       # half of the rows pick other words
        best = torch.where(best == PAD, 1, best)
        a['eos'] = best
        a['ids'][:, :, 0] = best
        a['ids'][:, :, 1:] = (best[..., None] + torch.tensor([7, 19])) % V
        got = run(dev, a, tau)
        assert bool((got['hard'] >= 0).all()) and bool((got['soft'] >= 0).all()), (scale, got['hard'].min(), got['soft'].min())
        for k, v in got.items():
            assert bool(torch.isfinite(v).all()), (scale, k)
        # |db| of a word: its rows' (|gh| + tau |gs|), to the sum's rounding
        most = T * (a['gh'].abs() + tau * a['gs'].abs()).sum()
        assert float(got['db'].float().abs().max()) <= float(most) * 1.01, scale


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('K', [0, 3])
def test_flat_batch_of_many_sentences(dev, K, dtype):
    """T = 1: as many sentences as rows, whose upstream gradients span 2^30; what an empty one carries counts nowhere."""
    T, R, E, V = 1, 3001, 24, 60
    if dtype == 'f32' and not K:
        K = 1                                                            # (fp32 without a teacher has kernels of its own)
    a = inputs(T, R, R, E, V, K, dtype, 23)
    a['eos'] = torch.where(torch.arange(R)[:, None] % 7 == 3, PAD, a['eos'].clamp_min(1))
    for k in ('gh', 'gs') if K else ('gh',):
        a[k] = a[k] * 2.0 ** -(torch.arange(R) % 31)
    want = oracle(a, 2.0)
    dead = a['eos'][:, 0] == PAD
    for k in ('gh', 'gs') if K else ('gh',):
        a[k] = torch.where(dead, 1e30, a[k])
    got = run(dev, a, 2.0)
    for k in got:
        check(got[k], want[k], k, E, V, T * R)


def test_more_rows_than_their_counts_are_added_up_in_every_block(dev):
    """525 066 rows, a third of them dropped at random, against the formulas in float64 on the GPU: every live row keeps its place
    in the compact order.  Tolerances as in `oracle`, with |x| <= 1 and the largest sums of |w|."""
    from cvae_amd import ops
    R, E, V = 525066, 8, 20
    g = torch.Generator(device=dev).manual_seed(5)
    final = torch.tanh(torch.randn(1, R, E, generator=g, device=dev)).bfloat16().requires_grad_()
    W = torch.randn(V, E, generator=g, device=dev).bfloat16().requires_grad_()
    b = (torch.randn(V, generator=g, device=dev) * 0.2).bfloat16().requires_grad_()
    eos = torch.randint(1, V, (R, 1), generator=g, device=dev)
    eos = torch.where(torch.rand(R, 1, generator=g, device=dev) < 1 / 3, PAD, eos)
    gh = torch.randn(R, generator=g, device=dev)
    hard = ops.proj_ce(final, W, b, eos, PAD)
    dX, dW, db = torch.autograd.grad([hard], [final, W, b], [gh])
    x, w, tgt = final.detach()[0].double(), W.detach().double(), eos[:, 0]
    live = (tgt != PAD).double()
    S = (x[:, None, :] * w[None]).sum(2) + b.detach().double()
    lq = S - torch.logsumexp(S, 1, keepdim=True)
    eS = (E + 20) * U * float(w.abs().sum(1).max() + b.detach().abs().max())
    e1 = 2 * eS + (V / 4 + 80) * U * (1 + float(S.abs().max()))          # of a loss, and of the exponent of a softmax
    want = -lq.gather(1, tgt[:, None])[:, 0] * live
    assert float((hard.detach().double() - want).abs().max()) <= e1
    P = (torch.exp(lq) - torch.nn.functional.one_hot(tgt, V)) * (gh.double() * live)[:, None]
    eP = (e1 + 2.0 ** -11) * P.abs() + e1 * (gh.double() * live).abs()[:, None] * torch.exp(lq) + 2.0 ** -37 * gh.double().abs()[:, None] * live[:, None]
    half = 2.0 ** -8
    for got, value, bound in ((dX[0], (P[:, :, None] * w[None]).sum(1), (eP[:, :, None] * w[None].abs()).sum(1)),
                              (db, P.sum(0), eP.sum(0) + R * U * P.abs().sum(0)),
                              (dW, torch.stack([(P[:, v:v + 1] * x).sum(0) for v in range(V)]),
                               torch.stack([((eP + R * U * P.abs())[:, v:v + 1] * x.abs()).sum(0) for v in range(V)]))):
        tol = 1.01 * bound + 40 * U * bound + half * (value.abs() + bound) + 1e-30
        assert bool(((got.double() - value).abs() <= tol).all())
    assert not bool(dX[0][tgt == PAD].any())


def test_gradients_of_the_weights_do_not_lose_bits_with_the_rows(dev):
    """fp32, 131072 rows: the sums over the rows are chains of 768 rows, joined by one of 171, and random roundings grow with the
    root of a chain's length: sqrt(768) + sqrt(171) units, and 12 for the operands' 22 bits as in `oracle`.  (One chain of all of
    them: 362 units, of which 83 were seen.)"""
    from cvae_amd import ops
    R, E, V, K, tau = 131072, 24, 60, 2, 2.0
    g = torch.Generator(device=dev).manual_seed(6)
    final = torch.tanh(torch.randn(1, R, E, generator=g, device=dev)).requires_grad_()
    W = (torch.randn(V, E, generator=g, device=dev) * 0.3).requires_grad_()
    b = (torch.randn(V, generator=g, device=dev) * 0.2).requires_grad_()
    eos = torch.randint(1, V, (R, 1), generator=g, device=dev)
    ids = torch.stack([torch.randint(0, V // 2, (R, 1), generator=g, device=dev), torch.randint(V // 2, V, (R, 1), generator=g, device=dev)], 2)
    top = torch.randn(R, 1, K, generator=g, device=dev)
    gh, gs = (torch.rand(R, generator=g, device=dev) + 0.5 for _ in range(2))
    hard, soft = ops.proj_distill(final, W, b, eos, PAD, ids, top, tau)
    dW, db = torch.autograd.grad([hard, soft], [W, b], [gh, gs])
    x, w = final.detach()[0].double(), W.detach().double()
    S = (x[:, None, :] * w[None]).sum(2) + b.detach().double()
    P = torch.softmax(S, 1) * gh.double()[:, None] + torch.softmax(S / tau, 1) * (gs.double() * tau)[:, None]
    P.scatter_add_(1, eos, -gh.double()[:, None])
    P.scatter_add_(1, ids[:, 0], -torch.softmax(top[:, 0].double() / tau, 1) * (gs.double() * tau)[:, None])
    units = math.sqrt(768) + math.sqrt(171) + 12
    for name, got, value in (('dW', dW, torch.stack([(P[:, v:v + 1] * x).sum(0) for v in range(V)])), ('db', db, P.sum(0))):
        off = float((got.double() - value).norm() / value.norm()) / U
        assert off <= units, (name, off)


# Wide rows over more than a tile everywhere: an odd and an even number of stages in one plane (300: 5, 330: 6, 513: 9) and in two
# (10, 11, 17), more than eight tiles of rows, several tiles of words to a range, several ranges to an XCD
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('E,V,K', [(300, 20000, 3), (330, 9001, 3), (513, 9001, 3), (513, 12000, 0)])
def test_wide_rows_over_many_tiles(dev, E, V, K, dtype):
    if dtype == 'f32' and not K:
        K = 2
    T, R = 18, 70
    a = inputs(T, R, R, E, V, K, dtype, E + V)
    a['eos'] = torch.where(a['eos'] == PAD, 3, a['eos'])
    a['eos'][5, 7:] = PAD
    assert int((a['eos'] != PAD).sum()) > 8 * 128
    compare(dev, a, 2.0)


# (words: an odd number of blocks of 256, so that two ranges of P are not equally long)
@pytest.mark.parametrize('dtype,T,R,E,V', [('f32', 64, 80, 300, 24700), ('f32', 64, 80, 200, 24700), ('bf16', 64, 128, 300, 25800),
                                           ('bf16', 64, 128, 120, 25800), ('f16', 64, 80, 513, 24700), ('f16', 64, 80, 200, 24700)])
def test_ranges_of_unequal_length(dev, dtype, T, R, E, V):
    """Two ranges of the vocabulary, the last one shorter, against float64 on the GPU: every 128 rows of dX and every 128 words of dW
    and db by the norm of what they are off, so that no single tile hides in the others.  fp32: root-mean-square growth as in
    `check`; 16 bits: the output's half step."""
    N, words = T * R, (V + 255) // 256 * 256
    most = (400 << 20) // ((2 if dtype == 'bf16' else 4) * N) // 256 * 256
    assert most < words <= 2 * most and words // 256 % 2 == 1
    a = inputs(T, R, R, E, V, 0, dtype, E)
    a['eos'] = torch.where(a['eos'] == PAD, 3, a['eos'])
    K, tau = 3, 2.0
    g = torch.Generator().manual_seed(7)
    a['ids'] = (torch.randint(0, V, (R, T, 1), generator=g) + torch.tensor([0, 5000, 15001])) % V
    a['top'], a['gs'] = torch.randn(R, T, K, generator=g), torch.rand(R, generator=g) + 0.5
    got = run(dev, a, tau)
    x, w, b = (a[k].to(dev).double() for k in ('final', 'W', 'b'))
    x = x.reshape(N, E)
    S = x @ w.t().contiguous() + b
    tgt, ids = a['eos'].to(dev).t().reshape(N, 1), a['ids'].to(dev).transpose(0, 1).reshape(N, K)
    sent = torch.arange(R, device=dev).repeat(T)
    gh, gs = (a[k].to(dev).double()[sent][:, None] for k in ('gh', 'gs'))
    lse, lse2 = torch.logsumexp(S, 1, keepdim=True), torch.logsumexp(S / tau, 1, keepdim=True)
    p = torch.softmax(a['top'].to(dev).double().transpose(0, 1).reshape(N, K) / tau, 1)
    add = lambda v: torch.zeros(R, dtype=torch.float64, device=dev).index_add(0, sent, v)
    want = dict(hard=add((lse - S.gather(1, tgt))[:, 0]),
                soft=add(tau ** 2 * (p * (torch.log(p) - S.gather(1, ids) / tau + lse2)).sum(1)))
    P = torch.exp(S - lse).mul_(gh)
    P += torch.exp(S / tau - lse2).mul_(gs * tau)
    del S
    P.scatter_add_(1, tgt, -gh)
    P.scatter_add_(1, ids, -p * gs * tau)
    want['dfinal'], want['dW'], want['db'] = P @ w, P.t().contiguous() @ x, P.sum(0)
    rel = 2 * (math.sqrt(E) + math.sqrt(max(V, N)) + 64) * U
    half = torch.finfo(DT[dtype]).eps / 2
    for k, v in want.items():
        u = got[k].detach().double().reshape(v.shape)
        n = 1 if k in ('hard', 'soft') else 128
        bound = rel if dtype == 'f32' or n == 1 else half
        for i in range(0, v.shape[0], n):
            off, size = float((u[i:i + n] - v[i:i + n]).norm()), float(v[i:i + n].norm())
            assert off <= bound * size, (k, i, off / size, bound)


@pytest.mark.parametrize('dtype', ['f32', 'f16'])
@pytest.mark.parametrize('tau', [1.0, 2.5])
@pytest.mark.parametrize('E', [40, 100, 200, 224])
def test_both_planes_of_every_entry(dev, E, tau, dtype):
    """States that are the unit vectors: dW then is d loss / d S itself, transposed, and every one of its 1500 E entries shows both
    of its fp16 planes alone, with nothing to average it out."""
    a = inputs(1, E, E, E, 1500, 3, dtype, 26)
    a['final'] = torch.eye(E)[None].to(DT[dtype])
    a['eos'] = torch.where(a['eos'] == PAD, 3, a['eos'])
    compare(dev, a, tau)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('K,V', [(1, 3), (2, 2), (16, 17), (17, 40), (64, 70), (65, 70), (100, 130), (128, 1100), (129, 1100), (513, 600), (1024, 1100)])
def test_many_entries_with_repeats(dev, K, V, dtype):
    """Entries drawn with replacement (and some outside the vocabulary), around the sizes at which the table of ids grows; one
    position lists one id K times, one lists no id twice, one the target last."""
    T, B, E = 3, 4, 40
    a = inputs(T, B, B, E, V, K, dtype, 24)
    g = torch.Generator().manual_seed(25)
    distinct = a['ids'].clone()
    a['ids'] = torch.randint(-2, V + 2, (B, T, K), generator=g)
    a['ids'][0, 0], a['ids'][0, 1] = 5, distinct[0, 1]
    a['eos'][0] = torch.tensor([7, 9, 11])
    a['ids'][0, 2, K - 1] = 11
    a['top'][1, 0, ::3] = float('-inf')
    compare(dev, a, 2.0)
    compare(dev, a, 1.0)
