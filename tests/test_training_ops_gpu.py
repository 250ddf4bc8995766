"""Row normalisation with its gradients, counter-based dropout and the gated recurrence on the
GPU, against plain implementations in float64. Tolerances count one rounding to the feature
type (half a step, eps / 2 of the value) and the float32 roundings inside, each 2^-24 of the
magnitudes that enter: sums run over at most 64 dependent additions at these sizes."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FLOOR = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}   # half of the smallest step
DTYPES = [torch.float16, torch.float32]


def _np(t):
    return t.detach().cpu().double().numpy()


def _close(got, want, slop, dtype, name=''):
    got = _np(got)
    allowed = HALF_STEP[dtype] * (np.abs(want) + slop) + slop + FLOOR[dtype]
    bad = ~(np.abs(got - want) <= allowed)
    assert got.shape == want.shape
    assert not bad.any(), (name, np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5],
                           np.broadcast_to(allowed, want.shape)[bad][:5])


def _sparse(feats, counts=None):
    from mlx_lattice_b200.core import SparseTensor

    coords = torch.zeros((feats.shape[0], 4), dtype=torch.int32, device=feats.device)
    coords[:, 1] = torch.arange(feats.shape[0], dtype=torch.int32, device=feats.device)
    return SparseTensor(coords, feats, batch_counts=counts)


def _randn(rng, *shape, dtype=torch.float32, device='cuda', scale=1.0, shift=0.0):
    return torch.from_numpy(rng.normal(size=shape) * scale + shift).to(dtype).to(device)


# --------------------------------------------------------------------------- #
# row normalisation
# --------------------------------------------------------------------------- #


def _norm_reference(x, w, b, dy, eps, rms):
    """Values and gradients in float64, with the bound of the float32 error of each."""
    m = 0.0 if rms else x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + eps)
    xh = (x - m) * r
    wf = np.ones(x.shape[1]) if w is None else w
    y = xh * wf + (0.0 if b is None else b)
    g = dy * wf
    c1 = 0.0 if rms else g.mean(1, keepdims=True)
    c2 = (g * xh).mean(1, keepdims=True)
    dx = r * (g - c1 - xh * c2)
    # error of xh: of the mean, of the difference and of r
    top = np.abs(x).max(1, keepdims=True) * r
    exh = 64 * U32 * (top + np.abs(xh))
    ga = np.abs(g).max(1, keepdims=True)
    xa = np.abs(xh).max(1, keepdims=True)
    edx = r * (64 * U32 * ga * (2 + 2 * xa * xa) + 2 * ga * xa * (64 * U32 * (top + xa)))
    return {
        'y': (y, exh * np.abs(wf) + 2 * U32 * np.abs(y)),
        'dx': (dx, edx),
        'dw': ((dy * xh).sum(0), (np.abs(dy) * (64 * U32 * np.abs(xh) + exh)).sum(0)),
        'db': (dy.sum(0), 64 * U32 * np.abs(dy).sum(0)),
    }


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rms', [False, True])
@pytest.mark.parametrize('rows,channels', [
    (1, 64), (8, 256), (700, 1), (700, 2), (33, 7), (701, 20), (3001, 64), (257, 96), (130, 192), (300, 100),
    (65, 1000), (64, 1024), (37, 1025), (70, 2051), (5, 520),
])
def test_row_norm_values_and_gradients(cuda, dtype, rms, rows, channels):
    from mlx_lattice_b200 import _ext, ops

    rng = np.random.default_rng(rows * 7 + channels)
    feats = _randn(rng, rows, channels, dtype=dtype, scale=2.0, shift=1.0).requires_grad_(True)
    weight = _randn(rng, channels, dtype=dtype, shift=1.0).requires_grad_(True)
    bias = None if rms else _randn(rng, channels, dtype=dtype).requires_grad_(True)
    dy = _randn(rng, rows, channels, dtype=dtype)
    x = _sparse(feats)
    y = (ops.rms_norm(x, weight=weight, eps=1e-3) if rms
         else ops.layer_norm(x, weight=weight, bias=bias, eps=1e-3)).feats
    leaves = (feats, weight) if rms else (feats, weight, bias)
    grads = torch.autograd.grad(y, leaves, dy)
    want = _norm_reference(_np(feats), _np(weight), None if rms else _np(bias), _np(dy), 1e-3, rms)
    for got, name in zip((y, *grads), ('y', 'dx', 'dw', 'db')):
        assert got.dtype == dtype
        _close(got, *want[name], dtype, name)
    # the inference form of the same call: a sum in another order
    with torch.no_grad():
        plain = (ops.rms_norm(x, weight=weight, eps=1e-3) if rms
                 else ops.layer_norm(x, weight=weight, bias=bias, eps=1e-3)).feats
    _close(plain, *want['y'], dtype, 'inference')
    again = torch.autograd.grad((ops.rms_norm(x, weight=weight, eps=1e-3) if rms
                                 else ops.layer_norm(x, weight=weight, bias=bias, eps=1e-3)).feats, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    _ext.check_status()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rms', [False, True])
@pytest.mark.parametrize('rows,channels', [
    (9001, 3), (7003, 5), (6001, 21), (5003, 60), (5001, 62), (5000, 63), (2100, 130), (2003, 191), (901, 300),
    (700, 513), (401, 766), (301, 999), (1, 999), (2, 1023), (9, 1022),
])
def test_row_norm_of_rows_that_are_no_vectors(cuda, dtype, rms, rows, channels):
    """Rows of every width modulo 16 bytes, several batches a warp and a ragged last one; what
    lies behind the arrays stays as it was."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(rows + channels)
    x = _randn(rng, rows, channels, dtype=dtype, scale=2.0, shift=1.0)
    dy = _randn(rng, rows, channels, dtype=dtype)
    weight = _randn(rng, channels, dtype=dtype, shift=1.0)
    bias = None if rms else _randn(rng, channels, dtype=dtype)
    want = _norm_reference(_np(x), _np(weight), None if rms else _np(bias), _np(dy), 1e-3, rms)
    y, mean, rstd = _ext.row_norm_forward(x, weight, bias, 1e-3, rms)
    dx, dw, db = _ext.row_norm_backward(dy, x, weight, mean, rstd, rms, True, not rms)
    for got, name in ((y, 'y'), (dx, 'dx'), (dw, 'dw'), (db, 'db')):
        if got is not None:
            _close(got, *want[name], dtype, name)
    again, *stats = _ext.row_norm_forward(x, weight, bias, 1e-3, rms)
    assert torch.equal(y, again)
    assert all(torch.equal(a, b) for a, b in zip(
        (dx, dw), _ext.row_norm_backward(dy, x, weight, mean, rstd, rms, True, not rms)))
    # the same rows in a wider array, element by element
    wide = torch.zeros((rows, channels + 1), dtype=dtype, device=cuda)
    wide[:, :channels] = x
    y, mean, rstd = _ext.row_norm_forward(wide[:, :channels], weight, bias, 1e-3, rms)
    _close(y, *want['y'], dtype, 'y')
    dx, dw, db = _ext.row_norm_backward(dy, wide[:, :channels], weight, mean, rstd, rms, True, not rms)
    for got, name in ((dx, 'dx'), (dw, 'dw'), (db, 'db')):
        if got is not None:
            _close(got, *want[name], dtype, name)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('channels', [64, 60, 63])
def test_row_norm_of_arrays_off_a_boundary(cuda, dtype, channels):
    """Rows, or only weight and bias, that start at an odd element of their buffers."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(channels)
    rows = 700
    x, dy = _randn(rng, rows, channels, dtype=dtype), _randn(rng, rows, channels, dtype=dtype)
    weight, bias = _randn(rng, channels, dtype=dtype, shift=1.0), _randn(rng, channels, dtype=dtype)
    want = _norm_reference(_np(x), _np(weight), _np(bias), _np(dy), 1e-3, False)

    def off(t):
        buffer = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        buffer[1:] = t.flatten()
        return buffer[1:].view(t.shape)

    for args in ((x, off(weight), off(bias), dy), (off(x), weight, bias, dy), (x, weight, bias, off(dy)),
                 (off(x), off(weight), bias, off(dy))):
        y, mean, rstd = _ext.row_norm_forward(*args[:3], 1e-3, False)
        grads = _ext.row_norm_backward(args[3], args[0], args[1], mean, rstd, False, True, True)
        for got, name in zip((y, *grads), ('y', 'dx', 'dw', 'db')):
            _close(got, *want[name], dtype, name)


@pytest.mark.parametrize('rms', [0, 1])
@pytest.mark.parametrize('channels', [5, 63, 62, 999])
def test_row_norm_writes_its_rows_only(cuda, rms, channels):
    """Outputs in the middle of a buffer: the bytes around them stay."""
    from mlx_lattice_b200 import _native

    lib = _native.load()
    rows, pad = 37, 64
    x = torch.randn(rows, channels, device=cuda).half()
    ptr = lambda t: None if t is None else t.data_ptr()
    buffers = [torch.full((rows * channels + 2 * pad,), 7.0, device=cuda, dtype=torch.float16) for _ in range(2)]
    stats = [torch.full((rows + 2 * pad,), 7.0, device=cuda) for _ in range(2)]
    y, dx = (b[pad:pad + rows * channels] for b in buffers)
    mean, rstd = (s[pad:pad + rows] for s in stats)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.lat_row_norm_forward(1, rms, ptr(x), rows, channels, channels, None, None, 1e-5, ptr(y),
                                    None if rms else ptr(mean), ptr(rstd), stream) == _native.LAT_OK
    assert lib.lat_row_norm_backward(1, rms, ptr(x), channels, ptr(x), rows, channels, channels, None,
                                     None if rms else ptr(mean), ptr(rstd), ptr(dx), None, None, None, 0,
                                     stream) == _native.LAT_OK
    for buffer in (*buffers, *stats):
        assert (buffer[:pad] == 7).all() and (buffer[-pad:] == 7).all()
    assert (y.view(rows, channels).float() - x.float()).abs().max() > 0 and not (dx == 7).all()


@pytest.mark.parametrize('dtype', DTYPES)
def test_row_norm_strided_and_unaligned_rows(cuda, dtype):
    """Columns of a wider array, rows that start off a 16-byte boundary, a broadcast gradient,
    no weight, and only some of the gradients asked for."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(3)
    for channels, lo in ((64, 8), (64, 1), (24, 3)):
        wide = _randn(rng, 300, 100, dtype=dtype)
        feats = wide[:, lo:lo + channels].detach().requires_grad_(True)
        assert feats.stride(0) == 100
        want = _norm_reference(_np(feats), None, None, np.ones((300, channels)), 1e-5, False)
        y = ops.layer_norm(_sparse(feats)).feats
        dx, = torch.autograd.grad(y.sum(), (feats,))
        _close(y, *want['y'], dtype, 'y')
        _close(dx, *want['dx'], dtype, 'dx')
        weight = _randn(rng, channels, dtype=dtype).requires_grad_(True)
        want = _norm_reference(_np(feats), _np(weight), None, np.ones((300, channels)), 1e-5, True)
        y = ops.rms_norm(_sparse(feats.detach()), weight=weight).feats
        dw, = torch.autograd.grad(y.sum(), (weight,))
        _close(dw, *want['dw'], dtype, 'dw')


def test_row_norm_of_many_rows_and_of_none(cuda):
    """Several passes of the grid; the sums of 200,000 rows (about 150 dependent additions, more
    than the 64 of the bound, but of values whose errors are independent). No rows: zero sums."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(5)
    feats = _randn(rng, 200_003, 32).requires_grad_(True)
    weight, bias = _randn(rng, 32).requires_grad_(True), _randn(rng, 32).requires_grad_(True)
    dy = _randn(rng, 200_003, 32)
    y = ops.layer_norm(_sparse(feats), weight=weight, bias=bias).feats
    grads = torch.autograd.grad(y, (feats, weight, bias), dy)
    want = _norm_reference(_np(feats), _np(weight), _np(bias), _np(dy), 1e-5, False)
    for got, name in zip((y, *grads), ('y', 'dx', 'dw', 'db')):
        _close(got, *want[name], torch.float32, name)
    none = torch.empty((0, 32), device=cuda, requires_grad=True)
    y = ops.layer_norm(_sparse(none), weight=weight, bias=bias).feats
    dx, dw, db = torch.autograd.grad(y, (none, weight, bias), torch.empty((0, 32), device=cuda))
    assert dx.shape == (0, 32) and not dw.any() and not db.any()


def test_row_norm_gradient_against_differences(cuda):
    """The directional derivative of the float64 formula by central differences."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(6)
    x, w, b, dy = (rng.normal(size=s) for s in ((40, 24), (24,), (24,), (40, 24)))
    x, w, b, dy = (v.astype(np.float32).astype(np.float64) for v in (x, w, b, dy))
    leaves = [torch.from_numpy(v).float().to(cuda).requires_grad_(True) for v in (x, w, b)]
    y = ops.layer_norm(_sparse(leaves[0]), weight=leaves[1], bias=leaves[2]).feats
    grads = torch.autograd.grad(y, leaves, torch.from_numpy(dy).float().to(cuda))
    for i, step in enumerate(rng.normal(size=v.shape) for v in (x, w, b)):
        def value(t):
            args = [x, w, b]
            args[i] = args[i] + t * step
            return (_norm_reference(args[0], args[1], args[2], dy, 1e-5, False)['y'][0] * dy).sum()

        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        # differences: 1e-10 of the third derivative, 1e-16 / 1e-5 of the value; float32 gradient
        assert abs(slope - (_np(grads[i]) * step).sum()) <= 1e-5 * (1 + (np.abs(_np(grads[i]) * step)).sum())


def test_row_norm_refusals(cuda):
    from mlx_lattice_b200 import _ext, ops

    feats = torch.ones((4, 8), device=cuda, requires_grad=True)
    x = _sparse(feats)
    for weight in (torch.ones(7, device=cuda), torch.ones(8, device=cuda, dtype=torch.float16), torch.ones(8)):
        with pytest.raises(ValueError, match='weight'):
            ops.layer_norm(x, weight=weight)
    with pytest.raises(ValueError, match='eps'):
        ops.layer_norm(x, eps=0.0)
    with pytest.raises(ValueError, match='float32 and float16'):
        ops.rms_norm(_sparse(feats.detach().double().requires_grad_(True)))
    out, mean, rstd = _ext.row_norm_forward(feats.detach(), None, None, 1e-5, False)
    with pytest.raises(ValueError, match='grad must match'):
        _ext.row_norm_backward(out[:3], feats.detach(), None, mean, rstd, False, False, False)
    with pytest.raises(ValueError, match='rstd'):
        _ext.row_norm_backward(out, feats.detach(), None, mean, rstd[:3], False, False, False)


# --------------------------------------------------------------------------- #
# dropout
# --------------------------------------------------------------------------- #


def _philox(index, offset, seed):
    """Philox4x32-10 over uint64 numpy words: (len(index), 4) uint32."""
    low = np.uint64(0xFFFFFFFF)
    c = [index & low, index >> np.uint64(32), np.full_like(index, offset & 0xFFFFFFFF),
         np.full_like(index, (offset >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=1).astype(np.uint32)


def _keep(shape, p, seed, offset):
    total = int(np.prod(shape))
    words = _philox(np.arange((total + 3) // 4, dtype=np.uint64), offset, seed).reshape(-1)[:total]
    return (words >= np.uint32(min(round(p * 2 ** 32), 2 ** 32 - 1))).reshape(shape)


def test_philox_known_answers():
    """Published vectors of the generator that the masks are compared with."""
    zero = _philox(np.zeros(1, np.uint64), 0, 0)[0]
    assert [hex(v) for v in zero] == ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']
    ones = _philox(np.full(1, 2 ** 64 - 1, np.uint64), 2 ** 64 - 1, 2 ** 64 - 1)[0]
    assert [hex(v) for v in ones] == ['0x408f276d', '0x41c83b0e', '0xa20bc7c6', '0x6d5451fd']


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,channels,p,seed,offset,residual', [
    (1, 1, 0.5, 1, 0, False), (2003, 20, 0.5, 2 ** 63 + 5, 3, True), (4097, 64, 0.1, 17, 2 ** 40 + 1, True),
    (777, 33, 0.9, 0, 0, False), (5, 7, 0.25, -1, 1, True), (3000, 96, 0.0, 9, 0, True), (64, 8, 1 - 1e-12, 4, 0, False),
])
def test_dropout_values_and_gradients(cuda, dtype, rows, channels, p, seed, offset, residual):
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(rows + channels)
    feats = _randn(rng, rows, channels, dtype=dtype).requires_grad_(True)
    add = _randn(rng, rows, channels, dtype=dtype).requires_grad_(True) if residual else None
    dy = _randn(rng, rows, channels, dtype=dtype)
    y = ops.dropout(_sparse(feats), p=p, training=True, seed=seed, offset=offset, residual=add).feats
    keep = _keep((rows, channels), p, seed % 2 ** 64, offset)
    scaled = np.where(keep, _np(feats) / (1 - p), 0.0)
    with np.errstate(over='ignore'):
        want = scaled + (_np(add) if residual else 0.0)
    # two float32 roundings (scale, product) and the one of the sum
    _close(y, want, 3 * U32 * (np.abs(scaled) + np.abs(want)), dtype, 'y')
    assert not _np(y)[~keep].any() or residual
    leaves = (feats, add) if residual else (feats,)
    grads = torch.autograd.grad(y, leaves, dy)
    want = np.where(keep, _np(dy) / (1 - p), 0.0)
    _close(grads[0], want, 3 * U32 * np.abs(want), dtype, 'dx')
    if residual:
        assert torch.equal(grads[1], dy)


def test_dropout_keeps_the_stated_share_and_streams_differ(cuda):
    from mlx_lattice_b200 import _ext

    ones = torch.ones((100_000, 16), device=cuda)
    for p in (0.1, 0.5, 0.8):
        share = float((_ext.dropout(ones, p, 11) != 0).double().mean())
        assert abs(share - (1 - p)) <= 6 * np.sqrt(p * (1 - p) / ones.numel())
    masks = [_ext.dropout(ones, 0.5, seed, offset) != 0 for seed, offset in ((1, 0), (2, 0), (1, 1), (1, 2 ** 32))]
    for i in range(len(masks)):
        for j in range(i):
            assert abs(float((masks[i] == masks[j]).double().mean()) - 0.5) <= 6 * 0.5 / np.sqrt(ones.numel())


@pytest.mark.parametrize('dtype', DTYPES)
def test_dropout_selects_and_reads_any_layout(cuda, dtype):
    """A dropped NaN or infinity is zero, also in the gradient; unaligned and strided inputs draw
    the mask of the dense, aligned ones."""
    from mlx_lattice_b200 import _ext, ops

    keep = _keep((60, 12), 0.4, 5, 0)
    values = np.where(keep, 1.0, np.where(np.arange(12) % 2, np.nan, np.inf))
    feats = torch.from_numpy(values).to(dtype).to(cuda).requires_grad_(True)
    y = ops.dropout(_sparse(feats), p=0.4, training=True, seed=5).feats
    assert np.array_equal(_np(y) != 0, keep) and np.isfinite(_np(y)).all()
    dx, = torch.autograd.grad(y, (feats,), feats.detach())
    assert np.array_equal(_np(dx) != 0, keep) and np.isfinite(_np(dx)).all()

    rng = np.random.default_rng(8)
    flat = _randn(rng, 40 * 30 + 3, dtype=dtype)
    for shift in (1, 2, 3):
        view = flat[shift:shift + 1200].view(40, 30)
        assert torch.equal(_ext.dropout(view, 0.3, 7, 1, view), _ext.dropout(view.clone(), 0.3, 7, 1, view.clone()))
    wide = _randn(rng, 50, 64, dtype=dtype)
    assert torch.equal(_ext.dropout(wide[:, 5:37], 0.3, 7), _ext.dropout(wide[:, 5:37].contiguous(), 0.3, 7))
    assert torch.equal(_ext.dropout(wide.t(), 0.3, 7), _ext.dropout(wide.t().contiguous(), 0.3, 7))
    assert _ext.dropout(wide[:0], 0.3, 7).shape == (0, 64)


def test_dropout_seed_on_the_device(cuda):
    """A captured call reads the seed when it is replayed; the gradient notices a changed seed."""
    from mlx_lattice_b200 import _ext, ops

    feats = torch.ones((512, 24), device=cuda)
    seed = torch.tensor([41], dtype=torch.int64, device=cuda)
    assert torch.equal(_ext.dropout(feats, 0.5, seed, 2), _ext.dropout(feats, 0.5, 41, 2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _ext.dropout(feats, 0.5, seed, 2)
    for value in (5, -3, 2 ** 62):
        seed.fill_(value)
        graph.replay()
        assert torch.equal(out, _ext.dropout(feats, 0.5, value, 2))
    leaf = feats.clone().requires_grad_(True)
    y = ops.dropout(_sparse(leaf), p=0.5, training=True, seed=seed).feats
    seed.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y.sum(), (leaf,))


def test_dropout_refusals_and_evaluation(cuda):
    from mlx_lattice_b200 import _ext, nn, ops

    feats = torch.ones((16, 8), device=cuda)
    x = _sparse(feats)
    with pytest.raises(ValueError, match='needs a seed'):
        ops.dropout(x, p=0.5, training=True)
    for seed in (torch.zeros(2, dtype=torch.int64, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda),
                 torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match='seed must be'):
            ops.dropout(x, p=0.5, training=True, seed=seed)
    for residual in (feats[:8], feats.half(), feats.cpu()):
        with pytest.raises((ValueError, RuntimeError), match='residual'):
            ops.dropout(x, p=0.5, training=True, seed=1, residual=residual)
    with pytest.raises(ValueError, match='coordinates'):
        ops.dropout(x, p=0.5, training=True, seed=1, residual=_sparse(feats))
    with pytest.raises(ValueError, match='float32 and float16'):
        _ext.dropout(feats.double(), 0.5, 1)
    assert nn.Dropout(0.5)(x).feats is feats
    assert torch.equal(nn.Dropout(0.5)(x, residual=x).feats, feats * 2)
    assert torch.equal(nn.Dropout(0.5)(x, seed=3, offset=1).feats, _ext.dropout(feats, 0.5, 3, 1))


# --------------------------------------------------------------------------- #
# gated recurrence
# --------------------------------------------------------------------------- #


def _recurrence_reference(x, z, offsets, initial, reverse, dy=None, dfinal=None):
    """One row after the other in float64, and running bounds of the float32 error: a gate is
    off by a few 2^-24, an affine map by a few 2^-24 of the magnitudes in it, and what a row is
    off by reaches later rows times their gates."""
    n, c = x.shape
    s = len(offsets) - 1
    a, rest = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    out = {k: np.zeros((n, c)) for k in ('h', 'eh', 'dx', 'edx', 'dz', 'edz')}
    final, efinal = np.zeros((s, c)), np.zeros((s, c))
    dini, edini = np.zeros((s, c)), np.zeros((s, c))
    unit = 16 * U32
    # a and 1 - a below the smallest normal float32, 2^-126, may come out as zero (beyond
    # |z| = 87.3 the division 1 / (1 + exp(-z)) has a divisor above 2^126, for which the fast
    # division is defined to give 0): off by at most 2^-126, and the gradients by as much times
    # what multiplies it
    step = 2.0 ** -126
    # and whatever falls below 2^-126 is rounded to steps of 2^-149, in every operation of a row
    grid = 8 * 2.0 ** -149
    for j in range(s):
        rows = list(range(offsets[j], offsets[j + 1]))
        if reverse:
            rows.reverse()
        h = np.zeros(c) if initial is None else initial[j].copy()
        habs, e = np.abs(h), np.zeros(c)
        before = []
        for t in rows:
            before.append((h, habs, e))
            e = a[t] * e + unit * (habs + np.abs(x[t])) + grid
            h = a[t] * h + rest[t] * x[t]
            habs = a[t] * habs + rest[t] * np.abs(x[t])
            out['h'][t], out['eh'][t] = h, e
        final[j], efinal[j] = h, e
        if dy is None:
            continue
        flow = np.zeros(c) if dfinal is None else dfinal[j].copy()
        fabs, ef = np.abs(flow), np.zeros(c)
        for t, (hp, hpa, ehp) in zip(reversed(rows), reversed(before)):
            dh, dha = dy[t] + flow, np.abs(dy[t]) + fabs
            edh = ef + unit * dha
            out['dx'][t], out['edx'][t] = rest[t] * dh, rest[t] * (edh + unit * dha * (1 + np.abs(z[t]))) + step * dha + grid
            out['dz'][t] = a[t] * rest[t] * dh * (hp - x[t])
            out['edz'][t] = a[t] * rest[t] * (edh * np.abs(hp - x[t]) + dha * ehp
                                              + unit * dha * (hpa + np.abs(x[t])) * (1 + np.abs(z[t])))
            out['edz'][t] += (step * dha + grid) * (1 + hpa + np.abs(x[t]))
            flow, fabs, ef = a[t] * dh, a[t] * dha, a[t] * edh + unit * a[t] * dha + grid
        dini[j], edini[j] = flow, ef
    return {'h': (out['h'], out['eh']), 'final': (final, efinal), 'dx': (out['dx'], out['edx']),
            'dgate': (out['dz'], out['edz']), 'dinitial': (dini, edini)}


def _check_recurrence(cuda, dtype, rows, channels, offsets, reverse, initial, seed=0, grads=True):
    from mlx_lattice_b200 import _ext, ops

    rng = np.random.default_rng(seed + rows + channels)
    feats = _randn(rng, rows, channels, dtype=dtype, shift=0.5).requires_grad_(True)
    gate = _randn(rng, rows, channels, dtype=dtype, scale=2.0, shift=2.0).requires_grad_(True)
    dy = _randn(rng, rows, channels, dtype=dtype)
    s = len(offsets) - 1
    start = _randn(rng, s, channels).requires_grad_(True) if initial else None
    dfinal = _randn(rng, s, channels)
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda)
    x = _sparse(feats)
    y, final = ops.gated_recurrence(x, gate, initial_state=start, offsets=off, reverse=reverse, return_state=True)
    _ext.check_status(cuda)
    want = _recurrence_reference(_np(feats), _np(gate), offsets, None if start is None else _np(start), reverse,
                                 _np(dy), _np(dfinal))
    assert y.same_coords(x) and y.feats.dtype == dtype
    _close(y.feats, *want['h'], dtype, 'h')
    _close(final, *want['final'], torch.float32, 'final')
    leaves = (feats, gate, start) if initial else (feats, gate)
    got = torch.autograd.grad((y.feats, final), leaves, (dy, dfinal), retain_graph=True)
    _ext.check_status(cuda)
    _close(got[0], *want['dx'], dtype, 'dx')
    _close(got[1], *want['dgate'], dtype, 'dgate')
    if initial:
        _close(got[2], *want['dinitial'], torch.float32, 'dinitial')
    # the same bits again, and from the serving form
    again = torch.autograd.grad((y.feats, final), leaves, (dy, dfinal))
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    with torch.no_grad():
        y2, final2 = ops.gated_recurrence(x, gate, initial_state=start, offsets=off, reverse=reverse, return_state=True)
    assert torch.equal(y.feats, y2.feats) and torch.equal(final, final2)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('channels', [1, 3, 8, 16, 20, 24, 64, 96, 200])
def test_recurrence_ragged_sequences(cuda, dtype, reverse, channels):
    """Ends at, before and behind a tile's border, sequences without rows at both ends and in
    the middle, single rows, and rows behind the last sequence."""
    offsets = [0, 0, 1, 127, 128, 128, 129, 256, 300, 300, 300, 640, 641, 700, 700]
    _check_recurrence(cuda, dtype, 731, channels, offsets, reverse, initial=True)


@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('channels', [5, 7, 9, 63, 129, 513])
def test_recurrence_of_odd_widths(cuda, channels, reverse):
    """float16 rows whose starts fall on both halves of a four-byte word."""
    _check_recurrence(cuda, torch.float16, 300, channels, [0, 9, 150, 150, 270], reverse, True, seed=channels)


@pytest.mark.parametrize('reverse', [0, 1])
@pytest.mark.parametrize('channels,start', [(7, 0), (7, 1), (64, 1), (13, 3)])
def test_recurrence_writes_its_rows_only(cuda, channels, start, reverse):
    """Inputs and outputs at any element of a buffer: values as from the start of one, and the
    elements around the outputs stay."""
    from mlx_lattice_b200 import _ext, _native

    lib = _native.load()
    rows, pad = 75, 64
    rng = np.random.default_rng(channels)
    off = torch.tensor([0, 20, 75], dtype=torch.int32, device=cuda)

    def placed(t=None):
        buffer = torch.full((rows * channels + 2 * pad,), 7.0, device=cuda, dtype=torch.float16)
        view = buffer[pad + start:pad + start + rows * channels].view(rows, channels)
        if t is not None:
            view.copy_(t)
        return buffer, view

    x, z, dy = (_randn(rng, rows, channels, dtype=torch.float16) for _ in range(3))
    h, _, carries = _ext.recurrence_forward(x, z, off, None, bool(reverse), want_carries=True)
    dx, dz, _ = _ext.recurrence_backward(dy, None, x, z, off, None, bool(reverse), carries)
    kept = [placed(t) for t in (x, z, dy)]
    xp, zp, dyp = (view.data_ptr() for _, view in kept)
    outs = [placed() for _ in range(3)]
    need = lib.lat_recurrence_workspace_bytes(1, rows, channels)
    workspace = torch.empty(need, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.lat_recurrence_forward(
        1, xp, channels, zp, channels, rows, channels, off.data_ptr(), 2, None, reverse, outs[0][1].data_ptr(), None,
        carries.data_ptr(), workspace.data_ptr(), need, None, stream) == _native.LAT_OK
    assert lib.lat_recurrence_backward(
        1, dyp, channels, None, xp, channels, zp, channels, rows, channels, off.data_ptr(), 2, None, reverse,
        carries.data_ptr(), outs[1][1].data_ptr(), outs[2][1].data_ptr(), None, workspace.data_ptr(), need, None,
        stream) == _native.LAT_OK
    for (buffer, view), want in zip(outs, (h, dx, dz)):
        assert torch.equal(view, want)
        assert (buffer[:pad + start] == 7).all() and (buffer[pad + start + rows * channels:] == 7).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,offsets', [
    (1, [0, 1]), (1, [0, 0]), (7, [0, 7]), (127, [0, 127]), (128, [0, 128]), (129, [0, 129]), (2049, [0, 2049]),
    (300, [5, 20, 290]), (300, [300]), (2600, [0, 1300, 2600]),
])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_lengths(cuda, dtype, rows, offsets, reverse):
    _check_recurrence(cuda, dtype, rows, 40, offsets, reverse, initial=rows % 2 == 1)


@pytest.mark.parametrize('dtype,channels', [(torch.float16, 8), (torch.float32, 5)])
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_over_many_groups_of_tiles(cuda, dtype, channels, reverse):
    """70,000 rows: over a thousand tiles in many groups, crossed by one sequence; and the same
    rows cut into three."""
    _check_recurrence(cuda, dtype, 70_000, channels, [0, 70_000], reverse, initial=True)
    _check_recurrence(cuda, dtype, 70_000, channels, [0, 33_000, 69_000, 69_990], reverse, initial=False)


def test_recurrence_with_slow_and_fast_gates(cuda):
    """Gates near one (a memory of thousands of rows) and near zero, and saturated ones."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(2)
    z = np.concatenate([rng.normal(size=(9000, 4)) + 9, rng.normal(size=(9000, 4)) - 9,
                        np.where(rng.random((9000, 2)) < 0.5, 100.0, -100.0)], axis=1).astype(np.float32)
    x = (rng.normal(size=z.shape) + 1).astype(np.float32)
    offsets = torch.tensor([0, 9000], dtype=torch.int32, device=cuda)
    feats, gate = torch.from_numpy(x).to(cuda), torch.from_numpy(z).to(cuda)
    h, _, carries = _ext.recurrence_forward(feats, gate, offsets, want_carries=True)
    dy = _randn(rng, *z.shape)
    dx, dz, _ = _ext.recurrence_backward(dy, None, feats, gate, offsets, None, False, carries)
    want = _recurrence_reference(x.astype(np.float64), z.astype(np.float64), [0, 9000], None, False, _np(dy))
    for got, name in ((h, 'h'), (dx, 'dx'), (dz, 'dgate')):
        _close(got, *want[name], torch.float32, name)


def test_recurrence_keeps_sequences_apart(cuda):
    """NaN and infinities of one sequence, and of rows outside all of them, reach no other."""
    from mlx_lattice_b200 import _ext, ops

    rng = np.random.default_rng(4)
    rows, channels = 900, 24
    offsets = torch.tensor([10, 300, 500, 800], dtype=torch.int32, device=cuda)
    base, gates, dy = (_randn(rng, rows, channels) for _ in range(3))
    dirty, dirty_gates, dirty_dy = base.clone(), gates.clone(), dy.clone()
    for t, value in ((dirty, float('nan')), (dirty_gates, float('nan')), (dirty_dy, float('inf'))):
        t[:10] = value
        t[800:] = value
    dirty[350], dirty_gates[420], dirty_dy[400] = float('inf'), float('nan'), float('nan')
    for reverse in (False, True):
        results = []
        for x, z, g in ((base, gates, dy), (dirty, dirty_gates, dirty_dy)):
            x, z = x.clone().requires_grad_(True), z.clone().requires_grad_(True)
            y, final = ops.gated_recurrence(_sparse(x), z, offsets=offsets, reverse=reverse, return_state=True)
            results.append((y.feats, *torch.autograd.grad(y.feats, (x, z), g)))
        for clean, seen in zip(*results):
            for part in (slice(10, 300), slice(500, 800)):
                assert torch.equal(clean[part], seen[part])
            assert not seen[:10].any() and not seen[800:].any()
            assert not torch.isfinite(seen[300:500]).all()
    _ext.check_status(cuda)


@pytest.mark.parametrize('dtype', DTYPES)
def test_recurrence_strided_inputs(cuda, dtype):
    """Gate and values as the two halves of one projection, unaligned columns, a transposed
    gradient, and a broadcast one."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(9)
    offsets = torch.tensor([0, 100, 391], dtype=torch.int32, device=cuda)
    for lo, channels in ((0, 32), (3, 32), (0, 21)):
        both = _randn(rng, 391, 80, dtype=dtype)
        x = both[:, lo:lo + channels].detach().requires_grad_(True)
        z = both[:, 40:40 + channels].detach().requires_grad_(True)
        dense = [t.detach().clone().contiguous().requires_grad_(True) for t in (x, z)]
        dy = _randn(rng, channels, 391, dtype=dtype).t()
        got = ops.gated_recurrence(_sparse(x), z, offsets=offsets).feats
        want = ops.gated_recurrence(_sparse(dense[0]), dense[1], offsets=offsets).feats
        assert torch.equal(got, want)
        for p, q in zip(torch.autograd.grad(got, (x, z), dy), torch.autograd.grad(want, dense, dy.contiguous())):
            assert torch.equal(p, q)
        got = ops.gated_recurrence(_sparse(x), z, offsets=offsets).feats
        want = ops.gated_recurrence(_sparse(dense[0]), dense[1], offsets=offsets).feats
        for p, q in zip(torch.autograd.grad(got.sum(), (x, z)), torch.autograd.grad(want.sum(), dense)):
            assert torch.equal(p, q)


def test_recurrence_gradient_against_differences(cuda):
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(12)
    offsets = [0, 37, 37, 170]
    arrays = [rng.normal(size=s).astype(np.float32).astype(np.float64) for s in ((170, 6), (170, 6), (3, 6))]
    dy, dfinal = (rng.normal(size=s).astype(np.float32).astype(np.float64) for s in ((170, 6), (3, 6)))
    leaves = [torch.from_numpy(v).float().to(cuda).requires_grad_(True) for v in arrays]
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda)
    y, final = ops.gated_recurrence(_sparse(leaves[0]), leaves[1], initial_state=leaves[2], offsets=off,
                                    return_state=True)
    grads = torch.autograd.grad((y.feats, final), leaves,
                                (torch.from_numpy(dy).float().to(cuda), torch.from_numpy(dfinal).float().to(cuda)))
    for i in range(3):
        step = rng.normal(size=arrays[i].shape)

        def value(t):
            args = list(arrays)
            args[i] = args[i] + t * step
            out = _recurrence_reference(args[0], args[1], offsets, args[2], False)
            return (out['h'][0] * dy).sum() + (out['final'][0] * dfinal).sum()

        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        assert abs(slope - (_np(grads[i]) * step).sum()) <= 1e-5 * (1 + np.abs(_np(grads[i]) * step).sum())


def test_recurrence_only_the_final_state_or_only_some_gradients(cuda):
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(13)
    x, z = _randn(rng, 260, 16), _randn(rng, 260, 16).requires_grad_(True)
    counts = (100, 0, 160)
    y, final = ops.gated_recurrence(_sparse(x, counts), z, return_state=True)
    dfinal = _randn(rng, 3, 16)
    dz, = torch.autograd.grad(final, (z,), dfinal)
    want = _recurrence_reference(_np(x), _np(z), [0, 100, 100, 260], None, False, np.zeros((260, 16)), _np(dfinal))
    _close(dz, *want['dgate'], torch.float32, 'dgate')
    state = _randn(rng, 3, 16).requires_grad_(True)
    y = ops.gated_recurrence(_sparse(x, counts), z.detach(), initial_state=state).feats
    ds, = torch.autograd.grad(y, (state,), torch.ones_like(y))
    want = _recurrence_reference(_np(x), _np(z), [0, 100, 100, 260], _np(state), False, np.ones((260, 16)))
    _close(ds, *want['dinitial'], torch.float32, 'dinitial')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,channels', [(1, 1), (8, 256), (33, 20), (1000, 7)])
def test_recurrence_step_continues_a_sequence(cuda, dtype, rows, channels):
    """A step equals the recurrence over sequences of one row, and steps in a row equal the
    recurrence over a sequence."""
    from mlx_lattice_b200 import _ext, ops

    rng = np.random.default_rng(rows)
    wide = _randn(rng, rows, 2 * channels, dtype=dtype)
    x, z = wide[:, :channels], wide[:, channels:]
    state = _randn(rng, rows, channels)
    y, after = ops.gated_recurrence_step(_sparse(x), z, state)
    offsets = torch.arange(rows + 1, dtype=torch.int32, device=cuda)
    want, final = ops.gated_recurrence(_sparse(x), z, initial_state=state, offsets=offsets, return_state=True)
    assert torch.equal(y.feats, want.feats) and torch.equal(after, final)
    ref = _recurrence_reference(_np(x), _np(z), list(range(rows + 1)), _np(state), False)
    _close(y.feats, *ref['h'], dtype, 'h')
    _close(after, *ref['final'], torch.float32, 'state')
    kept = state.clone()
    out, same = _ext.recurrence_step(x, z, kept, kept)
    assert same is kept and torch.equal(kept, after) and torch.equal(out, y.feats)
    assert _ext.recurrence_step(x[:0], z[:0], state[:0])[0].shape == (0, channels)


def test_recurrence_step_into_a_given_state(cuda):
    """The next state may take the place of the state, or lie apart from all inputs; a graph that
    keeps the overwritten state for its gradient notices."""
    from mlx_lattice_b200 import ops

    feats = torch.ones((16, 8), device=cuda)
    x, pool = _sparse(feats), torch.zeros((64, 8), device=cuda)
    _, apart = ops.gated_recurrence_step(x, feats, pool[:16], out_state=pool[16:32])
    _, placed = ops.gated_recurrence_step(x, feats, pool[:16], out_state=pool[:16])
    assert torch.equal(apart, placed) and not pool[32:].any()
    with pytest.raises(ValueError, match='apart from it'):
        ops.gated_recurrence_step(x, feats, pool[:16], out_state=pool[8:24])
    for x_rows, gate in ((pool[32:48], feats), (feats, pool[40:56])):
        with pytest.raises(ValueError, match='apart from the features'):
            ops.gated_recurrence_step(_sparse(x_rows), gate, pool[:16], out_state=pool[32:48])
    state = torch.zeros((1, 8), device=cuda)
    leaf = feats.clone().requires_grad_(True)
    y = ops.gated_recurrence(_sparse(leaf), feats, initial_state=state,
                             offsets=torch.tensor([0, 16], dtype=torch.int32, device=cuda)).feats
    ops.gated_recurrence_step(_sparse(feats[:1]), feats[:1], state, out_state=state)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_many_sequences_without_rows_hand_their_state_on(cuda):
    """More empty sequences than a warp has threads, at both ends and between rows."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(60)
    for channels in (3, 40):
        cuts = [4] * 90 + [30] * 70 + [31, 75] + [75] * 41
        x, z, dy = (_randn(rng, 80, channels) for _ in range(3))
        off = torch.tensor(cuts, dtype=torch.int32, device=cuda)
        initial = _randn(rng, len(cuts) - 1, channels)
        for reverse in (False, True):
            h, final, carries = _ext.recurrence_forward(x, z, off, initial, reverse, want_state=True, want_carries=True)
            dfinal = _randn(rng, len(cuts) - 1, channels)
            _, _, dinitial = _ext.recurrence_backward(dy, dfinal, x, z, off, initial, reverse, carries, want_initial=True)
            empty = (off[1:] == off[:-1]).nonzero().flatten()
            assert len(empty) == len(cuts) - 1 - 3
            assert torch.equal(final[empty], initial[empty]) and torch.equal(dinitial[empty], dfinal[empty])
            ref = _recurrence_reference(_np(x), _np(z), cuts, _np(initial), reverse, _np(dy), _np(dfinal))
            _close(h, *ref['h'], torch.float32, 'h')
            _close(final, *ref['final'], torch.float32, 'final')
            _close(dinitial, *ref['dinitial'], torch.float32, 'dinitial')
    _ext.check_status(cuda)


def test_prefill_then_steps(cuda):
    """A cloud's rows in one call, or a part of them and then row by row from the state."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(21)
    x, z = _randn(rng, 140, 32, dtype=torch.float16), _randn(rng, 140, 32, dtype=torch.float16)
    offsets = torch.tensor([0, 140], dtype=torch.int32, device=cuda)
    whole, final = ops.gated_recurrence(_sparse(x), z, offsets=offsets, return_state=True)
    offsets = torch.tensor([0, 130], dtype=torch.int32, device=cuda)
    _, state = ops.gated_recurrence(_sparse(x[:130]), z[:130], offsets=offsets, return_state=True)
    for t in range(130, 140):
        h, state = ops.gated_recurrence_step(_sparse(x[t:t + 1]), z[t:t + 1], state)
    ref = _recurrence_reference(_np(x), _np(z), [0, 140], None, False)
    _close(h.feats, ref['h'][0][139:], ref['h'][1][139:], torch.float16)
    _close(state, *ref['final'], torch.float32)
    _close(final, *ref['final'], torch.float32)
    _close(whole.feats, *ref['h'], torch.float16)


def test_recurrence_refusals(cuda):
    from mlx_lattice_b200 import _ext, ops

    feats = torch.ones((16, 8), device=cuda)
    x = _sparse(feats)
    good = torch.tensor([0, 16], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match='batch_counts'):
        ops.gated_recurrence(x, feats)
    for gate in (feats[:8], feats.half(), feats[:, :4]):
        with pytest.raises(ValueError, match='gate must match'):
            ops.gated_recurrence(x, gate, offsets=good)
    with pytest.raises(ValueError, match='coordinates'):
        ops.gated_recurrence(x, _sparse(feats), offsets=good)
    with pytest.raises(ValueError, match='int32'):
        ops.gated_recurrence(x, feats, offsets=good.long())
    for offsets in (good[:0], good.view(1, 2)):
        with pytest.raises(ValueError, match='offsets'):
            ops.gated_recurrence(x, feats, offsets=offsets)
    for state in (torch.zeros((2, 8), device=cuda), torch.zeros((1, 8), device=cuda, dtype=torch.float16),
                  torch.zeros((1, 4), device=cuda)):
        with pytest.raises(ValueError, match='initial_state'):
            ops.gated_recurrence(x, feats, offsets=good, initial_state=state)
    with pytest.raises(ValueError, match='float32 and float16'):
        ops.gated_recurrence(_sparse(feats.double()), feats.double(), offsets=good)
    with pytest.raises(ValueError, match='state must have shape'):
        ops.gated_recurrence_step(x, feats, torch.zeros((15, 8), device=cuda))
    with pytest.raises(ValueError, match='state must have shape'):
        ops.gated_recurrence_step(x, feats, None)
    with pytest.raises(ValueError, match='contiguous'):
        ops.gated_recurrence_step(x, feats, torch.zeros((16, 8), device=cuda),
                                  out_state=torch.zeros((8, 16), device=cuda).t())
    with pytest.raises(ValueError, match='carries'):
        _ext.recurrence_backward(feats, None, feats, feats, good, None, False, torch.zeros((1, 8), device=cuda))
    _ext.check_status(cuda)


def test_recurrence_reports_falling_offsets(cuda):
    """Offsets that fall or leave the rows are clamped and reported; nothing outside the arrays
    is touched (the rows and sequences a tile writes are bounded by its own tables)."""
    from mlx_lattice_b200 import _ext

    feats = torch.ones((600, 8), device=cuda)
    for bad in ([0, 400, 100, 600], [0, 500, 200, 200]):
        off = torch.tensor(bad, dtype=torch.int32, device=cuda)
        _ext.recurrence_forward(feats, feats, off, want_state=True)
        with pytest.raises(RuntimeError, match='outside its range'):
            _ext.check_status(cuda)
    off = torch.tensor([-50, 900], dtype=torch.int32, device=cuda)
    h, final, _ = _ext.recurrence_forward(feats, feats, off, want_state=True)
    want, state, _ = _ext.recurrence_forward(feats, feats, torch.tensor([0, 600], dtype=torch.int32, device=cuda),
                                             want_state=True)
    assert torch.equal(h, want) and torch.equal(final, state)
    _ext.check_status(cuda)


# --------------------------------------------------------------------------- #
# together
# --------------------------------------------------------------------------- #


def _block(x, gate, weight, bias, offsets, seed):
    from mlx_lattice_b200 import ops

    mixed = ops.gated_recurrence(ops.layer_norm(x, weight=weight, bias=bias), gate, offsets=offsets)
    return ops.dropout(mixed, p=0.2, training=True, seed=seed, residual=x)


def test_block_of_the_operators(cuda):
    """x + dropout(recurrence(layer_norm(x), gate)) with its gradients, against the same in
    float64 by torch on the CPU; intermediate results are float32, so every stage is exact to a
    few hundred 2^-24 of the magnitudes (memory of at most about 60 rows)."""
    rng = np.random.default_rng(40)
    rows, channels, cuts = 500, 48, [0, 180, 180, 500]
    arrays = [rng.normal(size=s).astype(np.float32) for s in ((rows, channels), (rows, channels), (channels,), (channels,))]
    dy = rng.normal(size=(rows, channels)).astype(np.float32)
    leaves = [torch.from_numpy(v).to(cuda).requires_grad_(True) for v in arrays]
    off = torch.tensor(cuts, dtype=torch.int32, device=cuda)
    y = _block(_sparse(leaves[0]), leaves[1], leaves[2], leaves[3], off, 77).feats
    grads = torch.autograd.grad(y, leaves, torch.from_numpy(dy).to(cuda))

    ref = [torch.from_numpy(v).double().requires_grad_(True) for v in arrays]
    n = torch.nn.functional.layer_norm(ref[0], (channels,), ref[2], ref[3], 1e-5)
    a = torch.sigmoid(ref[1])
    h, outs = None, []
    for t in range(rows):
        h = (1 - a[t]) * n[t] if t in cuts else a[t] * h + (1 - a[t]) * n[t]
        outs.append(h)
    keep = torch.from_numpy(_keep((rows, channels), 0.2, 77, 0))
    want = ref[0] + torch.where(keep, torch.stack(outs) / 0.8, torch.zeros(()).double())
    wants = torch.autograd.grad(want, ref, torch.from_numpy(dy).double())
    for got, exact in zip((y, *grads), (want, *wants)):
        exact = exact.detach().numpy()
        assert np.abs(_np(got) - exact).max() <= 2000 * U32 * np.abs(exact).max()


def test_training_step_in_a_graph_and_on_another_stream(cuda):
    """A captured forward and backward pass, replayed on new data while another graph of the
    same operators lives and while eager calls run, gives the bits of the eager calls; so does
    a side stream."""
    rng = np.random.default_rng(50)
    rows, channels = 5000, 64
    off = torch.tensor([0, 1200, 5000], dtype=torch.int32, device=cuda)
    seed = torch.tensor([3], dtype=torch.int64, device=cuda)

    def make():
        return [_randn(rng, rows, channels, dtype=torch.float16), _randn(rng, rows, channels, dtype=torch.float16),
                _randn(rng, channels, dtype=torch.float16), _randn(rng, channels, dtype=torch.float16)]

    dy = _randn(rng, rows, channels, dtype=torch.float16)

    def step(leaves):
        y = _block(_sparse(leaves[0]), *leaves[1:], off, seed).feats
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    inputs = [make(), make()]
    eager = [step([t.clone().requires_grad_(True) for t in group]) for group in inputs]
    torch.cuda.synchronize()
    graphs = []
    for group in inputs:
        buffers = [torch.zeros_like(t).requires_grad_(True) for t in group]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(buffers)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = step(buffers)
        graphs.append((graph, buffers, outputs))
    for order in ((0, 1), (1, 0)):
        for k in order:
            with torch.no_grad():
                for buffer, t in zip(graphs[k][1], inputs[order[k]]):
                    buffer.copy_(t)
            graphs[k][0].replay()
        for k in order:
            for got, want in zip(graphs[k][2], eager[order[k]]):
                assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        results = step([t.clone().requires_grad_(True) for t in inputs[0]])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for got, want in zip(results, eager[0]):
        assert torch.equal(got, want)
    from mlx_lattice_b200 import _ext

    _ext.check_status(cuda)
