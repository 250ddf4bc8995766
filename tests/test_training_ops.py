"""Refusals of the training and sequence operators that need no device: the C entry points
check their arguments before any launch, and the Python layer before it touches a device."""

import ctypes

import pytest
import torch

from mlx_lattice_b200 import _ext, _native, nn, ops
from mlx_lattice_b200.core import SparseTensor

F32, F16 = 0, 1


def _refused(code, text):
    assert code == _native.LAT_INVALID_ARGUMENT
    assert text in _native.last_error()


def test_row_norm_entry_points_refuse_bad_arguments():
    lib = _native.load()
    buf = ctypes.c_void_p(4096)
    _refused(lib.lat_row_norm_forward(2, 0, buf, 4, 8, 8, None, None, 1e-5, buf, buf, buf, None), 'float32 and float16')
    _refused(lib.lat_row_norm_forward(F32, 0, buf, 4, 8, 8, None, None, 0.0, buf, buf, buf, None), 'eps must be positive')
    _refused(lib.lat_row_norm_forward(F32, 0, buf, 4, 0, 8, None, None, 1e-5, buf, buf, buf, None), 'shape (N, C)')
    _refused(lib.lat_row_norm_forward(F32, 0, buf, -1, 8, 8, None, None, 1e-5, buf, buf, buf, None), 'shape (N, C)')
    _refused(lib.lat_row_norm_forward(F32, 1, buf, 4, 8, 8, None, buf, 1e-5, buf, None, buf, None), 'no bias')
    _refused(lib.lat_row_norm_forward(F32, 0, buf, 4, 8, 8, None, None, 1e-5, buf, None, buf, None), 'statistics')
    _refused(lib.lat_row_norm_backward(F32, 0, buf, 8, buf, 4, 8, 8, None, None, buf, buf, None, None, None, 0, None),
             'statistics of the forward pass')
    _refused(lib.lat_row_norm_backward(F32, 1, buf, 8, buf, 4, 8, 8, None, None, buf, buf, None, buf, None, 0, None),
             'no bias')
    need = lib.lat_row_norm_backward_workspace_bytes(4, 8)
    assert lib.lat_row_norm_backward(F32, 0, buf, 8, buf, 4, 8, 8, None, buf, buf, buf, buf, None, buf, need - 1,
                                     None) == _native.LAT_WORKSPACE_TOO_SMALL
    # nothing to do is no error, and touches no pointer
    assert lib.lat_row_norm_forward(F32, 0, None, 0, 8, 8, None, None, 1e-5, None, None, None, None) == _native.LAT_OK


def test_dropout_entry_point_refuses_bad_arguments():
    lib = _native.load()
    buf = ctypes.c_void_p(4096)
    for p in (1.0, -0.1, float('nan')):
        _refused(lib.lat_dropout(F32, buf, None, 8, p, 1, None, 0, buf, None), '0 <= p < 1')
    _refused(lib.lat_dropout(3, buf, None, 8, 0.5, 1, None, 0, buf, None), 'float32 and float16')
    _refused(lib.lat_dropout(F16, buf, None, -8, 0.5, 1, None, 0, buf, None), 'shape (N, C)')
    _refused(lib.lat_dropout(F16, buf, None, 8, 0.5, 1, ctypes.c_void_p(4097), 0, buf, None), 'device seed')
    assert lib.lat_dropout(F16, None, None, 0, 0.5, 1, None, 0, None, None) == _native.LAT_OK


def test_recurrence_entry_points_refuse_bad_arguments():
    lib = _native.load()
    buf = ctypes.c_void_p(4096)

    def forward(dtype=F32, rows=4, channels=8, offsets=buf, sequences=1, x=buf, stride=8, ws=None, ws_bytes=0):
        return lib.lat_recurrence_forward(dtype, x, stride, buf, 8, rows, channels, offsets, sequences, None, 0, buf,
                                          None, None, ws, ws_bytes, None, None)

    _refused(forward(dtype=5), 'float32 and float16')
    _refused(forward(rows=-1), 'shape (N, C)')
    _refused(forward(rows=2 ** 31 - 1), 'shape (N, C)')
    _refused(forward(channels=0), 'shape (N, C)')
    _refused(forward(stride=-1), 'shape (N, C)')
    _refused(forward(sequences=-1), 'offsets')
    _refused(forward(offsets=None), 'offsets')
    _refused(forward(offsets=None, sequences=0), 'offsets')
    _refused(forward(x=None), 'shape (N, C)')
    need = lib.lat_recurrence_workspace_bytes(F32, 300, 8)
    assert forward(rows=300, ws=buf, ws_bytes=need - 1) == _native.LAT_WORKSPACE_TOO_SMALL
    assert forward(rows=300) == _native.LAT_WORKSPACE_TOO_SMALL
    assert forward(rows=0, x=None, offsets=None, sequences=0) == _native.LAT_OK
    _refused(lib.lat_recurrence_backward(F32, buf, 8, None, buf, 8, buf, 8, 4, 8, buf, 1, None, 0, None, buf, buf, None,
                                         None, 0, None, None), 'tile states')
    _refused(lib.lat_recurrence_step(F32, buf, 8, buf, 8, None, 4, 8, buf, buf, None), 'state must have shape')
    _refused(lib.lat_recurrence_step(F32, buf, 8, buf, 8, buf, 4, 0, buf, buf, None), 'shape (N, C)')
    assert [lib.lat_recurrence_carry_rows(n) for n in (-1, 0, 1, 8, 9)] == [0, 0, 1, 1, 2]


def test_rows_too_wide_for_a_launch_are_refused_before_it():
    lib = _native.load()
    buf = ctypes.c_void_p(4096)
    wide = 65535 * 256 + 1
    _refused(lib.lat_row_norm_forward(F32, 0, buf, 4, wide, wide, None, None, 1e-5, buf, buf, buf, None), 'channels')
    _refused(lib.lat_row_norm_backward(F16, 1, buf, wide, buf, 4, wide, wide, None, None, buf, buf, None, None, None, 0,
                                       None), 'channels')
    wide = 65535 * 32 + 1
    _refused(lib.lat_recurrence_forward(F32, buf, wide, buf, wide, 4, wide, buf, 1, None, 0, buf, None, None, buf,
                                        1 << 62, None, None), 'channels')
    _refused(lib.lat_recurrence_backward(F32, buf, wide, None, buf, wide, buf, wide, 4, wide, buf, 1, None, 0, buf, buf,
                                         buf, None, buf, 1 << 62, None, None), 'channels')


def test_host_tensors_are_refused():
    x = torch.zeros((4, 8))
    for call in (lambda: _ext.row_norm_forward(x, None, None, 1e-5, False),
                 lambda: _ext.dropout(x, 0.5, 1),
                 lambda: _ext.recurrence_forward(x, x, torch.zeros(2, dtype=torch.int32)),
                 lambda: _ext.recurrence_step(x, x, x)):
        with pytest.raises(RuntimeError, match='CUDA device'):
            call()


def test_exceptions_pass_through_the_bindings():
    """An exception thrown inside the extension itself reaches Python."""
    with pytest.raises(TypeError, match='integer'):
        _ext.dropout(torch.zeros((4, 8)), 0.5, 'seed')


def test_module_arguments():
    with pytest.raises(ValueError, match='0 <= p < 1'):
        nn.Dropout(1.0)
    assert nn.GatedRecurrence(reverse=True).reverse
    assert {'gated_recurrence', 'gated_recurrence_step', 'sequence_offsets'} <= set(ops.__all__)


def test_recurrence_sizes_near_the_end_of_an_int_are_refused():
    """Row numbers of the last group (1024 rows), and places that a search tries behind the last
    sequence, have to stay within 32 bits; calls beyond end before anything runs."""
    lib = _native.load()
    buf = ctypes.c_void_p(4096)
    top = 2 ** 31 - 1

    def forward(rows, sequences):
        return lib.lat_recurrence_forward(F16, buf, 1, buf, 1, rows, 1, buf, sequences, None, 0, buf, None, None, None,
                                          0, None, None)

    def backward(rows, sequences):
        return lib.lat_recurrence_backward(F16, buf, 1, None, buf, 1, buf, 1, rows, 1, buf, sequences, None, 0, buf, buf,
                                           buf, None, None, 0, None, None)

    for call in (forward, backward):
        for rows in (top - 32, top - 63, top - 1023):
            _refused(call(rows, 1), 'shape (N, C)')
        for sequences in (top, top - 1, top - 16):
            _refused(call(64, sequences), 'sequences')
        # the largest ones only lack a workspace
        assert call(top - 1024, top - 64) == _native.LAT_WORKSPACE_TOO_SMALL


def test_norms_without_a_gradient_need_no_bindings(monkeypatch):
    """Inference runs on the C library alone; only a call that records a gradient asks for the
    extension that is built against torch."""
    def missing():
        raise RuntimeError('_bindings.so is not built')

    calls = []
    monkeypatch.setattr(_ext, 'bindings', missing)
    monkeypatch.setattr(_ext, 'row_norm', lambda feats, weight, bias, eps, rms: calls.append(rms) or feats)
    coords = torch.zeros((3, 4), dtype=torch.int32)
    coords[:, 1] = torch.arange(3)
    x, weight = SparseTensor(coords, torch.ones((3, 8))), torch.ones(8, requires_grad=True)
    ops.layer_norm(x)
    ops.rms_norm(x, weight=weight.detach())
    with torch.no_grad():
        ops.layer_norm(x, weight=weight, bias=weight)
    assert calls == [False, True, False]
    for call in (ops.layer_norm, ops.rms_norm):
        with pytest.raises(RuntimeError, match='not built'):
            call(x, weight=weight)


def test_bindings_count_as_stale_after_a_change_of_torch_or_python(monkeypatch, tmp_path):
    from mlx_lattice_b200 import build

    for name in ('LIBRARY_PATH', 'BINDINGS_PATH'):
        path = tmp_path / name
        path.write_bytes(b'')
        monkeypatch.setattr(build, name, str(path))
    monkeypatch.setattr(build, 'BINDINGS_RECORD', str(tmp_path / 'record'))
    assert build.is_stale()            # nobody knows what they were built against
    build.record_bindings()
    assert not build.is_stale()
    with monkeypatch.context() as change:
        change.setattr(torch, '__version__', '0.0.1')
        assert build.is_stale()
    with monkeypatch.context() as change:
        change.setattr('sys.version', '3.0')
        assert build.is_stale()
    assert not build.is_stale()
