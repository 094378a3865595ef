"""Calls of the 16-bit cross-entropy and of the distillation loss that have to be refused before anything is launched."""
import pytest
import torch

from cvae_amd import _lib, ops

T, B, E, V, K = 4, 2, 8, 10, 3


def good():
    return dict(final=torch.zeros(T, B, E), W=torch.zeros(V, E), b=torch.zeros(V), eos=torch.ones(B, T, dtype=torch.int64), pad=0,
                teacher_ids=torch.zeros(B, T, K, dtype=torch.int64), teacher_logits=torch.zeros(B, T, K), tau=2.0)


@pytest.mark.parametrize('what,change', [
    ('must be \\(T,R,E\\)', dict(final=torch.zeros(T, B, E + 1))),
    ('must be \\(T,R,E\\)', dict(final=torch.zeros(T, E))),
    ('must be \\(T,R,E\\)', dict(b=torch.zeros(V + 1))),
    ('must share', dict(W=torch.zeros(V, E, dtype=torch.bfloat16))),
    ('must share', dict(final=torch.zeros(T, B, E, dtype=torch.float64), W=torch.zeros(V, E, dtype=torch.float64),
                        b=torch.zeros(V, dtype=torch.float64))),
    ('W is empty', dict(W=torch.zeros(0, E), b=torch.zeros(0))),
    ('eos must be', dict(eos=torch.ones(B, T + 1, dtype=torch.int64))),
    ('eos must be', dict(eos=torch.ones(3, T, dtype=torch.int64))),
    ('eos must be', dict(eos=torch.ones(B, T, dtype=torch.int32))),
    ('teacher_ids', dict(teacher_ids=torch.zeros(B, T, K, dtype=torch.int32))),
    ('teacher_ids', dict(teacher_ids=torch.zeros(T, B, K, dtype=torch.int64))),
    ('teacher_ids', dict(teacher_ids=torch.zeros(B, T, V + 1, dtype=torch.int64))),
    ('teacher_ids', dict(teacher_ids=torch.zeros(B, T, 0, dtype=torch.int64))),
    ('teacher_ids', dict(W=torch.zeros(2000, E), b=torch.zeros(2000), teacher_ids=torch.zeros(B, T, 1025, dtype=torch.int64))),
    ('teacher_logits', dict(teacher_logits=torch.zeros(B, T, K + 1))),
    ('teacher_logits', dict(teacher_logits=torch.zeros(B, T, K, dtype=torch.int64))),
    ('tau', dict(tau=0.0)), ('tau', dict(tau=-1.0)), ('tau', dict(tau=float('nan'))), ('tau', dict(tau=float('inf'))),
    ('current GPU', dict()),
])
def test_proj_distill_refuses(what, change, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match=what):
        ops.proj_distill(**dict(good(), **change))


@pytest.mark.parametrize('what,change', [
    ('must share', dict(W=torch.zeros(V, E))),
    ('eos must be', dict(eos=torch.ones(3, T, dtype=torch.int64))),
    ('current GPU', dict()),
])
def test_proj_ce_16_bit_refuses(what, change, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    a = good()
    a = {k: a[k].to(torch.bfloat16) if k in ('final', 'W', 'b') else a[k] for k in ('final', 'W', 'b', 'eos', 'pad')}
    for f in (ops.proj_ce, ops.proj_ce_sorted):
        with pytest.raises(ValueError, match=what):
            f(**dict(a, **change))
    with pytest.raises(ValueError, match='float32'):
        ops.proj_ce_pair([a['final']], [a['W']], [a['b']], a['eos'], 0)
    assert not ops.proj_ce_pair_ok([a['final']], [a['W']])


def test_c_entries_refuse_bad_arguments():
    one = 16                                   # never dereferenced: the call is refused first
    ok = dict(dtype=0, B=2, T=4, R=2, E=8, V=10, K=3, tau=2.0, ws=one)

    def forward(**kw):
        a = dict(ok, **kw)
        _lib.call('cvae_distill_forward', a['dtype'], one, one, one, one, 0, 0, a['B'], a['T'], a['R'], a['E'], a['V'], a['K'],
                  one, one, a['tau'], one, one, a['ws'], None)

    def backward(**kw):
        a = dict(ok, **kw)
        _lib.call('cvae_distill_backward', a['dtype'], one, one, one, one, 0, 0, a['B'], a['T'], a['R'], a['E'], a['V'], a['K'],
                  one, one, a['tau'], one, one, one, one, one, one, a['ws'], None)
    for f in (forward, backward):
        for bad in (dict(dtype=3), dict(B=0), dict(R=3), dict(T=-1), dict(T=1 << 20, R=1 << 12), dict(E=0), dict(V=0),
                    dict(V=1 << 31), dict(K=-1), dict(K=11), dict(K=1025, V=2000), dict(tau=0.0), dict(tau=float('nan')), dict(ws=None), dict(ws=24)):
            with pytest.raises(_lib.CvaeHipError, match='distill_'):
                f(**bad)
    with pytest.raises(_lib.CvaeHipError, match='go together'):
        _lib.call('cvae_distill_backward', 0, one, one, one, one, 0, 0, 2, 4, 2, 8, 10, 3, one, one, 2.0, one, one, one, one,
                  None, one, one, None)
    with pytest.raises(_lib.CvaeHipError, match='rows'):
        backward(T=1 << 14, R=1 << 9)
    for name in ('cvae_distill_workspace', 'cvae_distill_backward_workspace'):      # sizes of nothing, or refused ones: 0
        assert _lib.query(name, 1, 5, 8, 10, 3) > 0
        for sizes in ((0, 8, 10, 3), (-1, 8, 10, 3), (5, 0, 10, 3), (5, 8, 0, 0), (5, 8, 10, 11), (5, 8, 10, -1),
                      (1 << 40, 8, 10, 3), (5, 1 << 40, 10, 3), (5, 8, 1 << 40, 3)):
            assert _lib.query(name, 1, *sizes) == 0, sizes


def test_fp32_cross_entropy_refuses_16_bit_weights(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    a = good()
    for k in ('W', 'b'):
        bad = {n: a[n].float() if n in ('final', 'W', 'b') else a[n] for n in ('final', 'W', 'b', 'eos', 'pad')}
        bad[k] = bad[k].to(torch.bfloat16)
        for f in (ops.proj_ce, ops.proj_ce_sorted):
            with pytest.raises(ValueError, match='must share'):
                f(**bad)


def test_sizes_beyond_a_launch_are_refused():
    """A launch has fewer than 2^32 threads; the workspace of a refused size is 0."""
    for N, E, V in (((1 << 23) + 1, 8, 100), (8, 8, (1 << 26) + 1), (8, 65537, 100)):
        assert _lib.query('cvae_distill_workspace', 1, N, E, V, 0) == 0
    assert _lib.query('cvae_distill_workspace', 1, 1 << 23, 8, 100, 0) > 0
    with pytest.raises(_lib.CvaeHipError, match='bad shape'):
        _lib.call('cvae_distill_forward', 1, 16, 16, 16, 16, 0, 0, 1, 1, (1 << 23) + 1, 8, 100, 0, None, None, 1.0, 16, None, 16, None)
    with pytest.raises(_lib.CvaeHipError, match='too many rows'):
        _lib.call('cvae_distill_backward', 1, 16, 16, 16, 16, 0, 0, 1, 1, 1 << 22, 8192, 100, 0, None, None, 1.0, 16, None, 16, 16,
                  16, 16, 16, None)


@pytest.mark.parametrize('what,change', [
    ('must be \\(T,R,E\\)', dict(final=torch.zeros(T, B, E + 1))),
    ('must be \\(T,R,E\\)', dict(W=torch.zeros(V, E - 1))),
    ('must be \\(T,R,E\\)', dict(b=torch.zeros(V - 1))),
    ('eos must be', dict(eos=torch.ones(B, T - 1, dtype=torch.int64))),
    ('eos must be', dict(eos=torch.ones(3, T, dtype=torch.int64))),
    ('eos must be', dict(eos=torch.ones(B, T, dtype=torch.int32))),
    ('current GPU', dict()),
])
def test_fp32_cross_entropy_refuses_what_its_kernels_would_read_past(what, change, monkeypatch):
    """Host tensors and sizes that do not belong together, refused in fp32 as in 16 bits: the kernels would read past the
    operands' ends."""
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    a = dict(good(), **change)
    a = {k: a[k] for k in ('final', 'W', 'b', 'eos', 'pad')}
    for f in (ops.proj_ce, ops.proj_ce_sorted):
        with pytest.raises(ValueError, match=what):
            f(**a)
    with pytest.raises(ValueError, match=what):
        ops.proj_ce_pair([a['final']] * 2, [a['W']] * 2, [a['b']] * 2, a['eos'], 0)


@pytest.mark.parametrize('change', [dict(final=torch.zeros(T, 2 * B, E)), dict(W=torch.zeros(V + 1, E), b=torch.zeros(V + 1))])
def test_paired_cross_entropy_refuses_two_shapes(change, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: -1)      # (host tensors pass: the shapes are looked at)
    a, o = good(), dict(good(), **change)
    with pytest.raises(ValueError, match='one shape'):
        ops.proj_ce_pair([a['final'], o['final']], [a['W'], o['W']], [a['b'], o['b']], a['eos'], 0)


@pytest.mark.parametrize('t,r,e', [((1 << 32) + 1, 1, E), (0, (1 << 32) + 2, E), (1 << 20, 1 << 12, E), (1, 1, (1 << 32) + 8)])
def test_sizes_past_32_bits_are_refused(t, r, e, monkeypatch):
    """The C entries take 32-bit sizes: 2^32 + 8 columns must not run as 8."""
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    for dtype in (torch.float32, torch.bfloat16):
        z = torch.zeros(1, dtype=dtype)
        for f in (ops.proj_ce, ops.proj_ce_sorted):
            with pytest.raises(ValueError, match='too large'):
                f(z.expand(t, r, e), z.expand(V, e), z.expand(V), torch.ones(1, 1, dtype=torch.int64).expand(1, t), 0)


@pytest.mark.parametrize('tau', [1e-40, 1e-20, 9e-7])
def test_a_temperature_that_leaves_no_bits_is_refused(tau, monkeypatch):
    """S / tau times 2^-24 is then more than the logits' differences, and 1 / tau ends in infinity."""
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match='tau'):
        ops.proj_distill(**dict(good(), tau=tau))
    for name, n in (('cvae_distill_forward', 4), ('cvae_distill_backward', 8)):
        with pytest.raises(_lib.CvaeHipError, match='tau'):
            _lib.call(name, 0, 16, 16, 16, 16, 0, 0, B, T, B, E, V, K, 16, 16, tau, *([None] * n))
    with pytest.raises(ValueError, match='current GPU'):              # the smallest that is taken gets as far as the devices
        ops.proj_distill(**dict(good(), tau=1e-6))


@pytest.mark.parametrize('dtype', [0, 1, 2])
def test_workspaces_follow_the_sizes(dtype):
    """P of a range, the partial tiles of dX, an image of the rows: what is documented, and little for little."""
    def parts(N, E, V):
        planes, np_ = (1 if dtype == 1 else 2), (2 if dtype == 0 else 1)
        rows, words = (N + 255) // 256 * 256, (V + 255) // 256 * 256
        most = max(1024, (400 << 20) // (2 * planes * rows) // 256 * 256)
        words = min(words, most)
        return 2 * planes * rows * words, 131072 * max(1024, (rows // 128) * ((E + 127) // 128)), 2 * np_ * rows * (E + 64)
    for N, E, V in ((1, 8, 10), (35, 75, 1003), (7680, 200, 50000), (1 << 20, 200, 20000), (1 << 22, 75, 250)):
        got = 4 * _lib.query('cvae_distill_backward_workspace', dtype, N, E, V, 3)
        assert got <= sum(parts(N, E, V)) + 16 * N + (1 << 16), (N, E, V, got)
    for name in ('cvae_distill_workspace', 'cvae_distill_backward_workspace'):
        assert 4 * _lib.query(name, dtype, 1, 8, 10, 3) <= 2 << 20
