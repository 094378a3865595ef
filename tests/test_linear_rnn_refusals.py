"""Calls of the gated linear recurrence that have to be refused before anything is launched (no GPU needed)."""
import pytest
import torch

from cvae_amd import _lib, ops


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize('what,args,kw', [
    ('gates', (z(3, 2, 16), 4), {}),
    ('dimensions', (z(3, 16), 2), {}),
    ('float32, bfloat16 or float16', (z(3, 2, 16, dtype=torch.float64), 2), {}),
    ('no multiple of gates', (z(3, 2, 16), 3), {}),
    ('the state', (z(3, 2, 16), 2), dict(h0=z(2, 16))),
    ('the state', (z(3, 2, 16), 2), dict(h0=z(2, 8, dtype=torch.bfloat16))),
    ('length', (z(3, 2, 16), 2), dict(length=torch.zeros(3, dtype=torch.int64))),
    ('length', (z(3, 2, 16), 2), dict(length=torch.zeros(2, dtype=torch.int32))),
    ('current GPU', (z(3, 2, 16), 2), {}),                  # a CPU tensor
])
def test_linear_rnn_refuses(what, args, kw, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match=what):
        ops.linear_rnn(*args, **kw)


@pytest.mark.parametrize('what,args,kw', [
    ('dimensions', (z(1, 2, 16), 2, z(2, 8)), {}),
    ('missing', (z(2, 16), 2, None), {}),
    ('the state', (z(2, 16), 2, z(2, 16)), {}),
    ('out must be', (z(2, 16), 2, z(2, 8)), dict(out=z(2, 9))),
    ('out must be', (z(2, 16), 2, z(2, 8)), dict(out=z(2, 16)[:, :8])),
    ('current GPU', (z(2, 16), 2, z(2, 8)), {}),
])
def test_linear_rnn_step_refuses(what, args, kw, monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match=what):
        ops.linear_rnn_step(*args, **kw)


def test_c_entries_refuse_bad_arguments():
    one = 16                                   # never dereferenced: the call is refused first
    ok = dict(dtype=0, gates=3, T=4, B=2, H=8)
    for bad in (dict(dtype=3), dict(dtype=-1), dict(gates=1), dict(T=-1), dict(B=-1), dict(H=-2), dict(B=1 << 20, H=1 << 12)):
        a = dict(ok, **bad)
        with pytest.raises(_lib.CvaeHipError, match='linrnn_forward'):
            _lib.call('cvae_linrnn_forward', a['dtype'], a['gates'], 0, a['T'], a['B'], a['H'], one, None, None, one, one,
                      None, None, None)
        with pytest.raises(_lib.CvaeHipError, match='linrnn_backward'):
            _lib.call('cvae_linrnn_backward', a['dtype'], a['gates'], 0, a['T'], a['B'], a['H'], one, None, one, one, None,
                      one, None, None, None)
    with pytest.raises(_lib.CvaeHipError, match='null operand'):
        _lib.call('cvae_linrnn_forward', 0, 3, 0, 4, 2, 8, None, None, None, one, one, None, None, None)
    with pytest.raises(_lib.CvaeHipError, match='null operand'):
        _lib.call('cvae_linrnn_backward', 0, 3, 0, 4, 2, 8, one, None, None, one, None, one, None, None, None)
    with pytest.raises(_lib.CvaeHipError, match='null workspace'):       # a long row of few channels is cut into segments
        assert _lib.query('cvae_linrnn_workspace', 0, 1000, 1, 8) > 0
        _lib.call('cvae_linrnn_forward', 0, 3, 0, 1000, 1, 8, one, None, None, one, one, None, None, None)
    for name in ('cvae_linrnn_forward', 'cvae_linrnn_backward'):         # nothing to do
        n = len(_lib.SIGNATURES[name]) - 6
        _lib.call(name, 0, 3, 0, 4, 0, 8, *([None] * n))
    for sizes in ((0, 2, 8), (4, 0, 8), (4, 2, 0), (0, 0, 0), (1, 1, 1)):
        assert _lib.query('cvae_linrnn_workspace', 0, *sizes) == 0


def test_in_place_state_of_a_segmented_sequence_is_refused():
    """Segments run at once and each starts from h0, so the last one must not overwrite it."""
    assert _lib.query('cvae_linrnn_workspace', 0, 1000, 1, 8) > 0
    with pytest.raises(_lib.CvaeHipError, match='h_last may be h0'):
        _lib.call('cvae_linrnn_forward', 0, 3, 0, 1000, 1, 8, 16, 16, None, 16, 16, None, 16, None)


def test_more_channels_than_a_launch_are_refused():
    with pytest.raises(_lib.CvaeHipError, match='bad shape'):
        _lib.call('cvae_linrnn_forward', 0, 3, 0, 64, (1 << 14) + 1, 1 << 14, 16, None, None, 16, 16, None, None, None)


@pytest.mark.parametrize('shape', [((1 << 32) + 3, 1, 2), (1 << 30, 1, 2), (4, (1 << 32) + 1, 2), (4, 1, (1 << 33) + 2)])
def test_sizes_past_32_bits_are_refused(shape, monkeypatch):
    """The C entries take 32-bit sizes: 2^32 + 3 steps must not run as 3."""
    monkeypatch.setattr(torch.cuda, 'current_device', lambda: 0)
    with pytest.raises(ValueError, match='too large'):
        ops.linear_rnn(z(1).expand(shape), 2)
    if shape[0] == 4:
        with pytest.raises(ValueError, match='too large'):
            ops.linear_rnn_step(z(1).expand(shape[1:]), 2, z(1).expand(shape[1], shape[2] // 2))


def test_no_operator_hands_pageable_host_memory_to_a_kernel():
    """A kernel that is given it reads an address that the GPU has not mapped.  Every pointer passes through one place."""
    x, w, b = z(3, 8), z(4, 8), z(4)
    for bad in (lambda: _lib.ptr(x), lambda: _lib.ptr_array([x, w]), lambda: ops.linear(x, w, b), lambda: ops.sort_resort(torch.ones(3, dtype=torch.int64)),
                lambda: ops.gemm(x, w, transB=True)):
        with pytest.raises(ValueError, match='GPU memory'):
            bad()
    assert _lib.ptr(None) is None
