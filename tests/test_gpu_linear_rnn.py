"""Gated linear recurrence (ops.linear_rnn, ops.linear_rnn_step) against a step-by-step float64 evaluation.

Tolerances are running bounds, from unit roundoff u = 2^-24 and carried along the recurrence beside the values:
 * a gate is exp2 (1 ulp) of a product, an addition, a reciprocal (1 ulp) and a product: 6 u relative at most, for
   tanh's series 6 u too, for its exp form 4 u absolute (its value is above 0.29: 14 u relative);
 * a step h = z h' + (1 - z) n adds at most 8 u |z h'| + 22 u |(1 - z) n|; composing maps of 8 steps and of the blocks of
   steps before them rounds each of those terms at most 8 more times -> E = z E' + 30 u (|z h'| + |(1 - z) n|);
 * the carry of the gradient obeys the same kind of recurrence; a product of k such factors adds their relative bounds;
 * values stored in 16 bits add half a step of their type, torch.finfo(t).eps / 2, of the value (and its smallest
   subnormal)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


@pytest.fixture(scope='module')
def dev():
    assert torch.cuda.is_available(), 'GPU tests need an MI355X'
    from cvae_amd import _lib
    _lib.init(0)
    return torch.device('cuda:0')


def oracle(u, gates, h0, length, reverse, dy, dlast):
    """float64 values and their bounds, step by step, on the CPU: {name: (value, bound)}."""
    u, dy, dlast, h0 = (t.detach().double().cpu() for t in (u, dy, dlast, h0))
    T, B, GH = u.shape
    H = GH // gates
    length = torch.full((B,), T) if length is None else length.cpu().clamp(0, T)
    z, n = torch.sigmoid(u[..., :H]), torch.tanh(u[..., H:2 * H])
    w = torch.sigmoid(-u[..., :H])
    o = torch.sigmoid(u[..., 2 * H:]) if gates == 3 else torch.ones_like(z)
    order = list(range(T))[::-1] if reverse else list(range(T))
    y, ey, du, edu = (torch.zeros(s, dtype=torch.float64) for s in ((T, B, H), (T, B, H), (T, B, GH), (T, B, GH)))
    h, eh, before = h0.clone(), torch.zeros_like(h0), {}
    for t in order:
        m = (length > t)[:, None]
        before[t] = (h, eh)
        zt, xt = z[t] * h, w[t] * n[t]
        h, eh = torch.where(m, zt + xt, h), torch.where(m, z[t] * eh + 30 * U * (zt.abs() + xt.abs()), eh)
        y[t] = torch.where(m, o[t] * h, 0.0)
        ey[t] = torch.where(m, o[t] * eh + 8 * U * (o[t] * h).abs(), 0.0)
    last, elast = h, eh
    c, ec = dlast.clone(), torch.zeros_like(dlast)
    for t in reversed(order):
        m = (length > t)[:, None]
        hp, ehp = before[t]
        dy_t = torch.where(m, dy[t], 0.0)
        ht = z[t] * hp + w[t] * n[t]
        eht = z[t] * ehp + 30 * U * ((z[t] * hp).abs() + (w[t] * n[t]).abs())
        d = c + dy_t * o[t]
        ed = ec + 8 * U * (c.abs() + (dy_t * o[t]).abs())
        diff, ediff = hp - n[t], ehp + 14 * U * (hp.abs() + n[t].abs())
        s = 1 - n[t] ** 2
        parts = [(d * diff * z[t] * w[t], z[t] * w[t] * (ed * diff.abs() + d.abs() * ediff + 20 * U * (d * diff).abs())),
                 (d * w[t] * s, w[t] * (ed * s + d.abs() * (30 * U * n[t] ** 2 + 14 * U * s)))]
        if gates == 3:
            q = 1 - o[t]
            parts.append((dy_t * ht * o[t] * q, (dy_t * o[t]).abs() * (eht * q + ht.abs() * (8 * U + 12 * U * q))))
        du[t] = torch.where(m, torch.cat([p[0] for p in parts], 1), 0.0)
        edu[t] = torch.where(m, torch.cat([p[1] for p in parts], 1), 0.0)
        c, ec = torch.where(m, z[t] * d, c), torch.where(m, z[t] * ed + 20 * U * (z[t] * d).abs(), ec)
    return dict(y=(y, ey), last=(last, elast), du=(du, edu), dh0=(c, ec))


def check(got, want, name):
    value, bound = want
    a = got.detach().double().cpu()
    fi = torch.finfo(got.dtype)
    assert a.shape == value.shape, name
    tol = bound * 1.01 + fi.eps / 2 * (value.abs() + bound) + (fi.tiny * fi.eps if got.dtype != torch.float32 else 1e-37)
    over = (a - value).abs() > tol
    assert not bool(over.any()), '%s: %d of %d outside, worst %.3g over %.3g' % (
        name, int(over.sum()), over.numel(), float((a - value).abs()[over].max()), float(tol[over].max()))
    assert bool(torch.isfinite(a).all()), name


def inputs(dev, T, B, H, gates, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn(T, B, gates * H, generator=g) * scale
    u[:, :, :H] += 1.5
    return (u.to(DT[dtype]).to(dev), torch.randn(B, H, generator=g).to(dev),
            torch.randn(T, B, H, generator=g).to(DT[dtype]).to(dev), torch.randn(B, H, generator=g).to(dev))


def run(u, gates, h0, length, reverse, dy, dlast):
    from cvae_amd import ops
    u, h0 = u.detach().requires_grad_(), h0.detach().requires_grad_()
    y, last = ops.linear_rnn(u, gates, h0=h0, length=length, reverse=reverse)
    du, dh0 = torch.autograd.grad([y, last], [u, h0], [dy, dlast])
    return dict(y=y, last=last, du=du, dh0=dh0)


# T around a wave's 8 steps and a round's 64, odd and even H (one or two channels a lane), more channels than a block,
# rows of few channels and many steps (segments: T >= 256)
SIZES = [(1, 1, 1), (1, 5, 130), (2, 3, 7), (7, 2, 33), (8, 1, 64), (9, 4, 66), (63, 2, 5), (64, 3, 20), (65, 2, 129),
         (130, 1, 6), (256, 1, 9), (300, 2, 70), (1000, 1, 130)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('gates', [2, 3])
@pytest.mark.parametrize('size', SIZES)
def test_whole_rows(dev, size, gates, dtype):
    T, B, H = size
    u, h0, dy, dlast = inputs(dev, T, B, H, gates, dtype, T + B + H)
    got = run(u, gates, h0, None, False, dy, dlast)
    want = oracle(u, gates, h0, None, False, dy, dlast)
    for k in got:
        check(got[k], want[k], k)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('T,H,gates', [(5, 8, 3), (70, 33, 2), (64, 64, 3), (400, 34, 3)])
def test_ragged_rows_with_garbage_past_their_end(dev, T, H, gates, reverse, dtype):
    """Lengths of 0, 1, T and past T; whatever stands behind a row's end (NaN, infinities) reaches nothing."""
    length = torch.tensor([0, 1, T, T // 2, T + 7, -3, T - 1])
    B = len(length)
    u, h0, dy, dlast = inputs(dev, T, B, H, gates, dtype, T + H, scale=2.0)
    want = oracle(u, gates, h0, length, reverse, dy, dlast)
    dead = (torch.arange(T)[:, None] >= length.clamp(0, T)[None]).to(dev)
    u, dy = u.clone(), dy.clone()
    u[dead] = float('nan')
    dy[dead] = float('inf')
    got = run(u, gates, h0, length.to(dev), reverse, dy, dlast)
    for k in got:
        check(got[k], want[k], k)
    assert not bool(got['y'][dead].any()) and not bool(got['du'][dead].any())


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_saturated_gates_and_long_memory(dev, dtype):
    """Gates far into their tails: a state that is kept for 500 steps, one that is replaced at every step, tiny inputs."""
    T, B, H, gates = 500, 1, 4, 3
    u, h0, dy, dlast = inputs(dev, T, B, H, gates, dtype, 3)
    u[:, :, 0], u[:, :, 1], u[:, :, 2] = 30.0, -30.0, 9.0
    u[:, :, H + 3] = 1e-4
    u[:, :, 2 * H] = 80.0
    u[:, :, 2 * H + 1] = -40.0
    got, want = run(u, gates, h0, None, False, dy, dlast), oracle(u, gates, h0, None, False, dy, dlast)
    for k in got:
        check(got[k], want[k], k)


def test_defaults_strides_and_alignment(dev):
    from cvae_amd import ops
    T, B, H = 20, 3, 10
    u, h0, dy, dlast = inputs(dev, T, B, H, 2, 'bf16', 5)
    zero = torch.zeros_like(h0)
    want = oracle(u, 2, zero, None, False, dy, dlast)
    y, last = ops.linear_rnn(u, 2)
    check(y, want['y'], 'y')
    check(last, want['last'], 'last')
    y2, _ = ops.linear_rnn(u.transpose(0, 1).contiguous().transpose(0, 1), 2)       # a batch-major tensor's view
    assert torch.equal(y, y2)
    store = torch.empty(u.numel() + 1, dtype=u.dtype, device=dev)                   # rows on odd 2-byte addresses
    odd = store[1:].view(T, B, 2 * H)
    odd.copy_(u)
    assert odd.data_ptr() % 4 == 2
    got = run(odd, 2, zero, None, False, dy, dlast)
    for k in got:
        check(got[k], want[k], k)


def test_step_equals_a_sequence_and_updates_in_place(dev):
    from cvae_amd import ops
    for dtype in DT:
        for B, H, gates in ((1, 1, 2), (4, 512, 3), (3, 33, 3), (257, 66, 2)):
            u, h0, dy, dlast = inputs(dev, 3, B, H, gates, dtype, B)
            want = oracle(u, gates, h0, None, False, dy, dlast)
            h = h0.clone()
            for t in range(3):
                y, out = ops.linear_rnn_step(u[t], gates, h, out=h)
                assert out is h
                check(y, (want['y'][0][t], want['y'][1][t]), 'y')
            check(h, want['last'], 'state')
            keep = h0.clone()
            y, new = ops.linear_rnn_step(u[0], gates, h0)
            check(y, (want['y'][0][0], want['y'][1][0]), 'y')
            assert torch.equal(h0, keep) and new.data_ptr() != h0.data_ptr()


def test_empty_shapes(dev):
    from cvae_amd import ops
    h0 = torch.randn(2, 4, device=dev)
    y, last = ops.linear_rnn(torch.empty(0, 2, 8, device=dev), 2, h0=h0)
    assert y.shape == (0, 2, 4) and torch.equal(last, h0)
    y, last = ops.linear_rnn(torch.empty(5, 0, 8, device=dev), 2)
    assert y.shape == (5, 0, 4) and last.shape == (0, 4)


def test_gradient_against_differences(dev):
    """Along one direction: (L(x + e v) - L(x - e v)) / 2e with L summed in float64.  Each L carries the forward bounds
    of the oracle, so the quotient is off by at most (their weighted sum) / e, plus the e^2 term, measured by halving e."""
    from cvae_amd import ops
    T, B, H, gates = 40, 2, 12, 3
    u, h0, dy, dlast = inputs(dev, T, B, H, gates, 'f32', 11)
    length = torch.tensor([40, 23], device=dev)
    got = run(u, gates, h0, length, False, dy, dlast)
    g = torch.Generator().manual_seed(1)
    vu, vh = torch.randn(u.shape, generator=g).to(dev), torch.randn(h0.shape, generator=g).to(dev)
    slope = float((got['du'].double() * vu).sum() + (got['dh0'].double() * vh).sum())

    def loss(e):
        y, last = ops.linear_rnn(u + e * vu, gates, h0=h0 + e * vh, length=length)
        return float((y.double() * dy).sum() + (last.double() * dlast).sum())
    bounds = oracle(u, gates, h0, length, False, dy, dlast)
    noise = float((bounds['y'][1] * dy.double().abs().cpu()).sum() + (bounds['last'][1] * dlast.double().abs().cpu()).sum())
    quot = {e: (loss(e) - loss(-e)) / (2 * e) for e in (2e-2, 1e-2)}
    curved = abs(quot[2e-2] - quot[1e-2])             # about 3/4 of the coarser quotient's e^2 term, 3x the finer one's
    assert abs(quot[1e-2] - slope) <= curved + 2 * noise / 1e-2 + 1e-4 * abs(slope)


def test_other_stream_and_repeatable(dev):
    u, h0, dy, dlast = inputs(dev, 300, 2, 70, 3, 'bf16', 9)
    first = run(u, 3, h0, None, False, dy, dlast)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run(u, 3, h0, None, False, dy, dlast)
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert torch.equal(first[k], again[k]), k


def test_captured_and_replayed(dev):
    """Forward and backward of a segmented sequence, and a step, in one graph; every replay on new inputs."""
    from cvae_amd import ops
    u, h0, dy, dlast = inputs(dev, 300, 2, 34, 3, 'f32', 2)
    length = torch.tensor([300, 111], device=dev)

    def work():
        out = run(u, 3, h0, length, True, dy, dlast)
        out['sy'], out['sh'] = ops.linear_rnn_step(u[0], 3, h0)
        return {k: v.detach() for k, v in out.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in (21, 22, 23):
        for dst, src in zip((u, h0, dy, dlast), inputs(dev, 300, 2, 34, 3, 'f32', seed)):
            dst.copy_(src)
        length.copy_(torch.tensor([seed, 300]))
        graph.replay()
        torch.cuda.synchronize()
        for k, v in work().items():
            assert torch.equal(out[k], v), (seed, k)


def test_offsets_past_32_bits(dev):
    """2.2e9 pre-activations: a row's results do not depend on how many rows there are (same kernels, same order of work)."""
    T, B, H = 16800, 64, 1024
    assert T * B * 2 * H > 2 ** 31
    g = torch.Generator(device=dev).manual_seed(0)
    u = torch.empty(T, B, 2 * H, dtype=torch.bfloat16, device=dev)
    dy = torch.empty(T, B, H, dtype=torch.bfloat16, device=dev)
    for t in range(0, T, 2100):
        u[t:t + 2100] = torch.randn(2100, B, 2 * H, generator=g, device=dev).bfloat16()
        dy[t:t + 2100] = torch.randn(2100, B, H, generator=g, device=dev).bfloat16()
    h0, dlast = torch.randn(B, H, generator=g, device=dev), torch.randn(B, H, generator=g, device=dev)
    whole = run(u, 2, h0, None, False, dy, dlast)
    part = run(u[:, 32:].contiguous(), 2, h0[32:], None, False, dy[:, 32:].contiguous(), dlast[32:])
    assert torch.equal(whole['y'][:, 32:], part['y']) and torch.equal(whole['du'][:, 32:], part['du'])
    assert torch.equal(whole['last'][32:], part['last']) and torch.equal(whole['dh0'][32:], part['dh0'])


def test_gradients_of_no_steps(dev):
    """A sequence of length zero hands its initial state on, and the state's gradient back."""
    from cvae_amd import ops
    h0 = torch.randn(2, 4, device=dev, requires_grad=True)
    u = torch.empty(0, 2, 8, device=dev, requires_grad=True)
    y, last = ops.linear_rnn(u, 2, h0=h0)
    g = torch.randn(2, 4, device=dev)
    du, dh0 = torch.autograd.grad((y, last), (u, h0), (torch.empty(0, 2, 4, device=dev), g))
    assert du.shape == u.shape and torch.equal(dh0, g)


def test_step_refuses_an_overlapping_out(dev):
    from cvae_amd import ops
    B, H = 3, 8
    room = torch.randn(2 * B * 3 * H, device=dev)
    u, h = room[:B * 3 * H].view(B, 3 * H), room[B * 3 * H:B * 4 * H].view(B, H)
    keep = room.clone()
    for at in (B * 3 * H + 1, B * 3 * H + B * H - 1, B * 3 * H - 1, 0):
        with pytest.raises(ValueError, match='overlap'):
            ops.linear_rnn_step(u, 3, h, out=room[at:at + B * H].view(B, H))
    assert torch.equal(room, keep)
    want = ops.linear_rnn_step(u, 3, h)[1]
    out = room[B * 4 * H:B * 5 * H].view(B, H)                    # right behind the state
    ops.linear_rnn_step(u, 3, h, out=out)
    assert torch.equal(out, want) and torch.equal(room[:B * 4 * H], keep[:B * 4 * H])


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('gates', [2, 3])
def test_the_small_side_of_saturated_gates(dev, gates, dtype):
    """Gates of 5 to 80 either way, no sums to hide in: with h0 = 0 the state is (1 - z) n, the gradient of a gate near 1 is made of
    1 - z, the gradient of h0 of a z near 0.  Each is held to the same few units of its own value; with 16-bit storage to |x| units
    more for a gate at x, whose exponent is rounded once (to x 2^-24) before it is raised."""
    B, H = 8, 256
    g = torch.Generator().manual_seed(31)
    u, h0, dy, dlast = inputs(dev, 1, B, H, gates, 'f32', 31)
    gate = (5 + 75 * torch.rand(B, H, generator=g)) * torch.where(torch.rand(B, H, generator=g) < 0.5, 1.0, -1.0)
    u[0, :, :H] = gate.to(dev)
    if gates == 3:
        u[0, :, 2 * H:] = gate.flip(1).to(dev)
    u = u.to(DT[dtype])
    for h in (torch.zeros_like(h0), h0):
        got, want = run(u, gates, h, None, False, dy.to(DT[dtype]), dlast), oracle(u, gates, h, None, False, dy.to(DT[dtype]), dlast)
        for k in got:
            value, bound = want[k]
            if dtype != 'f32':
                x = u[0, :, :H].double().abs().cpu() + (u[0, :, 2 * H:].double().abs().cpu() if gates == 3 else 0)
                bound = bound + U * value.abs() * (x if k != 'du' else x.repeat(1, gates))
            check(got[k], (value, bound), k)


def test_infinite_gates(dev):
    """A gate of +inf keeps the state, one of -inf replaces it, exactly; a NaN reaches its own channel only."""
    from cvae_amd import ops
    H = 6
    u = torch.zeros(2, 1, 3 * H, device=dev)
    u[:, 0, H:2 * H] = 0.5
    u[:, 0, 0], u[:, 0, 1], u[:, 0, 2] = float('inf'), float('-inf'), float('nan')
    u[:, 0, H + 3], u[:, 0, H + 4] = float('inf'), float('-inf')
    u[:, 0, 2 * H + 5] = float('-inf')
    h0 = torch.full((1, H), 0.25, device=dev)
    for step in (False, True):
        h = h0
        if step:
            for t in range(2):
                y, h = ops.linear_rnn_step(u[t], 3, h)
        else:
            y, h = ops.linear_rnn(u, 3, h0=h0)
            y = y[-1]
        assert h[0, 0] == 0.25 and abs(float(h[0, 1]) - 0.46211715726) < 1e-6 and torch.isnan(h[0, 2])
        assert float(h[0, 3]) == 0.25 * 0.25 + 0.5 * 1.5 and float(h[0, 4]) == 0.25 * 0.25 - 0.5 * 1.5 and float(y[0, 5]) == 0
        assert torch.isnan(y[0]).tolist() == [False, False, True, False, False, False]


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('T,B,H,gates,ragged', [(9, 3, 20, 3, True), (300, 2, 34, 3, True), (130, 5, 33, 2, False), (1, 4, 8, 2, False)])
def test_only_the_gradients_that_are_wanted(dev, T, B, H, gates, ragged, dtype):
    """Frozen pre-activations, or a frozen initial state: the other gradient does not change, and nothing is kept for the one that
    nobody wants."""
    from cvae_amd import ops
    u, h0, dy, dlast = inputs(dev, T, B, H, gates, dtype, 41)
    length = torch.arange(B, device=dev) * T // B if ragged else None
    full = run(u, gates, h0, length, False, dy, dlast)
    for wanted in ('u', 'h0'):
        leaves = dict(u=u.detach().requires_grad_(wanted == 'u'), h0=h0.detach().requires_grad_(wanted == 'h0'))
        y, last = ops.linear_rnn(leaves['u'], gates, h0=leaves['h0'], length=length)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got, = torch.autograd.grad([y, last], [leaves[wanted]], [dy, dlast])
        assert torch.equal(got, full['d' + wanted]), wanted
        if wanted == 'h0':
            spare = torch.cuda.max_memory_allocated() - before          # (its own gradient and the maps of segments, in 512-byte blocks)
            assert spare < max(u.numel() * u.element_size(), 64 << 10), spare


def test_a_graph_notices_that_its_saved_state_was_stepped(dev):
    """out = h is written in place: autograd refuses to use the old state's saved value, as behind torch's own in-place calls."""
    from cvae_amd import ops
    w = torch.ones(2, 8, device=dev, requires_grad=True)
    u, h = torch.randn(2, 24, device=dev), torch.randn(2, 8, device=dev)
    z = (w * h).sum()
    ops.linear_rnn_step(u, 3, h)                             # a new state: the old one stays
    z.backward(retain_graph=True)
    ops.linear_rnn_step(u, 3, h, out=h)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        z.backward()
    with torch.inference_mode():
        g = torch.randn(2, 8, device=dev)
        assert ops.linear_rnn_step(u, 3, g, out=g)[1] is g
