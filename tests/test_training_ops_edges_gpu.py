"""Places where the training and sequence operators are easily wrong: second derivatives, gates
near their ends, infinities, long memories, long runs of empty sequences."""

import numpy as np
import pytest
import torch
from test_training_ops_gpu import DTYPES, FLOOR, HALF_STEP, U32, _np, _randn, _sparse

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------------- #
# second derivatives
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize('op', ['layer_norm', 'rms_norm', 'dropout', 'dropout with residual', 'gated_recurrence'])
def test_a_second_derivative_raises(cuda, op):
    """A loss with a penalty on the gradient raises, whatever else the loss holds; the first
    derivatives taken with a graph are those taken without one."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(3)
    feats, gate = (_randn(rng, 40, 16).requires_grad_(True) for _ in range(2))
    weight = _randn(rng, 16, shift=1.0).requires_grad_(True)
    offsets = torch.tensor([0, 17, 40], dtype=torch.int32, device=cuda)
    x = _sparse(feats)
    call, leaves = {
        'layer_norm': (lambda: ops.layer_norm(x, weight=weight), (feats, weight)),
        'rms_norm': (lambda: ops.rms_norm(x, weight=weight), (feats, weight)),
        'dropout': (lambda: ops.dropout(x, p=0.3, seed=1), (feats,)),
        'dropout with residual': (lambda: ops.dropout(x, p=0.3, seed=1, residual=gate), (feats, gate)),
        'gated_recurrence': (lambda: ops.gated_recurrence(x, gate, offsets=offsets), (feats, gate)),
    }[op]
    plain = torch.autograd.grad(call().feats.pow(2).sum(), leaves)
    for place in range(len(leaves)):
        loss = call().feats.pow(2).sum()
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, plain))
        assert grads[place].requires_grad
        with pytest.raises(RuntimeError, match='no second derivative'):
            (loss + grads[place].pow(2).sum()).backward()


# --------------------------------------------------------------------------- #
# gates near their ends
# --------------------------------------------------------------------------- #


def _reference(x, z, offsets, initial, reverse, dy, dfinal):
    """The recurrence and its gradient row by row in float64, each with a bound of the float32 error.

    The weights a and 1 - a come from s = exp(-z), which is off by the rounding of its exponent,
    1.25 |z| 2^-24, and the instruction's 2^-22; the sum, the reciprocal and a product add four more
    2^-24. So the smaller one, m, is off by (8 + 1.5 |z|) 2^-24 of itself, the larger one by three. A
    row adds two roundings: 6 2^-24 of |a h| + |(1 - a) x|. The maps of 8 rows hold the product of the
    weights of h, or one less that, whichever is smaller: eight weights more (24 2^-24), and a
    composition of two maps rounds three times. There are fewer compositions than rows where the
    state changes slowly, and at most eight deep where it forgets at once (32 2^-24 of the state at the
    end). Weights below 2^-126 may be zero; results below it lie on a grid of 2^-149."""
    n, c = x.shape
    s = len(offsets) - 1
    with np.errstate(over='ignore'):
        a, k = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    m, g = np.minimum(a, k), (35 + 1.5 * np.abs(z)) * U32
    tiny, grid = 2.0 ** -126, 8 * 2.0 ** -149
    out = {name: np.zeros((n, c)) for name in ('h', 'eh', 'dx', 'edx', 'dgate', 'edgate')}
    ends = {name: np.zeros((s, c)) for name in ('final', 'efinal', 'dinitial', 'edinitial')}
    for j in range(s):
        rows = list(range(offsets[j], offsets[j + 1]))
        if reverse:
            rows.reverse()
        h = initial[j].copy()
        size, e = np.abs(h), np.zeros(c)
        before = []
        for t in rows:
            before.append((h, size, e))
            e = a[t] * e + (m[t] * g[t] + tiny) * (size + np.abs(x[t])) + grid
            h, size = a[t] * h + k[t] * x[t], a[t] * size + k[t] * np.abs(x[t])
            e = e + 6 * U32 * size
            out['h'][t], out['eh'][t] = h, e + 32 * U32 * size
        ends['final'][j], ends['efinal'][j] = h, e + 32 * U32 * size
        flow = dfinal[j].copy()
        size, e = np.abs(flow), np.zeros(c)
        for t, (hp, hp_size, ehp) in zip(reversed(rows), reversed(before)):
            dh, size = dy[t] + flow, np.abs(dy[t]) + size
            e = e + 33 * U32 * size if t == rows[-1] else e + U32 * size
            edh = e + 32 * U32 * size
            out['dx'][t] = k[t] * dh
            out['edx'][t] = k[t] * (edh + g[t] * size) + tiny * size + grid
            gap = hp_size + np.abs(x[t])
            out['dgate'][t] = a[t] * k[t] * dh * (hp - x[t])
            out['edgate'][t] = a[t] * k[t] * (edh * gap + size * (ehp + 32 * U32 * hp_size) + size * gap * 2 * g[t])
            out['edgate'][t] += (tiny * size + grid) * (1 + gap)
            e = a[t] * e + (m[t] * g[t] + tiny) * size + 6 * U32 * a[t] * size + grid
            flow, size = a[t] * dh, a[t] * size
        ends['dinitial'][j], ends['edinitial'][j] = flow, e + 32 * U32 * size
    out.update(ends)
    return {name: (out[name], out['e' + name]) for name in ('h', 'final', 'dx', 'dgate', 'dinitial')}


def _within(got, want, error, dtype, name):
    got = _np(got)
    allowed = error + HALF_STEP[dtype] * (np.abs(want) + error) + FLOOR[dtype]
    bad = ~(np.abs(got - want) <= allowed)
    assert not bad.any(), (name, np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3], allowed[bad][:3])


def _gate_case(case, rng, rows, channels, dtype, sequences):
    """(x, gate, initial state) as float64 arrays of exact float16 / float32 values."""
    normal = lambda *shape: rng.normal(size=shape)
    large = 6e4 if dtype == torch.float16 else 1e8
    if case == 'nothing kept at first':        # 1 - a down to 1e-13, from a zero state
        x, z, state = normal(rows, channels) + 1, rng.uniform(12, 30, (rows, channels)), np.zeros((sequences, channels))
    elif case == 'closed to large values':     # the state stays what it is
        x, z = large * np.sign(normal(rows, channels)), rng.uniform(27, 33, (rows, channels))
        state = 0.1 * normal(sequences, channels)
    elif case == 'open to small values':       # the large state is gone
        x, z = normal(rows, channels), rng.uniform(-33, -27, (rows, channels))
        state = 1e8 * normal(sequences, channels)
    else:                                      # anything, of any size
        x = np.clip(normal(rows, channels) * 10.0 ** rng.uniform(-4, 4, (rows, channels)), -large, large)
        z, state = rng.uniform(-40, 40, (rows, channels)), normal(sequences, channels) * 1e3
    as_held = lambda v, to: torch.from_numpy(v).to(to).double().numpy()
    return as_held(x, dtype), as_held(z, dtype), as_held(state, torch.float32)


CASES = ['nothing kept at first', 'closed to large values', 'open to small values', 'anything']


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('case', CASES)
@pytest.mark.parametrize('reverse', [False, True])
@pytest.mark.parametrize('channels', [5, 16])
def test_recurrence_at_the_ends_of_its_gates(cuda, dtype, case, reverse, channels):
    """Each row is as exact as its smaller weight allows, over several tiles and groups."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(len(case) + channels)
    cuts = [0, 40, 40, 2500]
    x, z, state = _gate_case(case, rng, 2510, channels, dtype, 3)
    dy, dfinal = _randn(rng, 2510, channels, dtype=dtype), _randn(rng, 3, channels)
    leaves = [torch.from_numpy(v).to(to).to(cuda).requires_grad_(True)
              for v, to in ((x, dtype), (z, dtype), (state, torch.float32))]
    y, final = ops.gated_recurrence(_sparse(leaves[0]), leaves[1], initial_state=leaves[2], reverse=reverse,
                                    offsets=torch.tensor(cuts, dtype=torch.int32, device=cuda), return_state=True)
    grads = torch.autograd.grad((y.feats, final), leaves, (dy, dfinal))
    want = _reference(x, z, cuts, state, reverse, _np(dy), _np(dfinal))
    _within(y.feats, *want['h'], dtype, 'h')
    _within(final, *want['final'], torch.float32, 'final')
    for got, name, to in zip(grads, ('dx', 'dgate', 'dinitial'), (dtype, dtype, torch.float32)):
        limit = torch.finfo(to).max
        inside = np.abs(want[name][0]) < 0.9 * limit     # what float16 can hold
        _within(torch.where(torch.from_numpy(inside).to(cuda), got, torch.zeros_like(got)),
                np.where(inside, want[name][0], 0.0), np.where(inside, want[name][1], 0.0), to, name)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('case', CASES)
def test_recurrence_step_at_the_ends_of_its_gates(cuda, dtype, case):
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(len(case))
    x, z, state = _gate_case(case, rng, 300, 12, dtype, 300)
    on = lambda v, to: torch.from_numpy(v).to(to).to(cuda)
    h, after = ops.gated_recurrence_step(_sparse(on(x, dtype)), on(z, dtype), on(state, torch.float32))
    zeros = np.zeros((300, 12))
    want = _reference(x, z, list(range(301)), state, False, zeros, zeros)
    _within(after, *want['final'], torch.float32, 'state')
    _within(h.feats, *want['h'], dtype, 'h')


@pytest.mark.parametrize('value', [10.0, 12.0])
def test_recurrence_with_a_long_memory(cuda, value):
    """Constant inputs over 96,000 rows: h = 1 - a^t and, backwards, the same sums. The memory, 22,000
    rows at a gate of 10 and 160,000 at 12, must not gather the rounding of a, which is up to 7e-4
    and 5e-3 of 1 - a there. Bound, in 2^-24 of h: 1 - a itself is off by 8 + 1.5 |z| < 30. What a piece
    of 8 rows adds is off by 6 a row, 48, its share of change by 24 more; 4 + 16 compositions make a group
    of pieces, 8 + 8 a window of groups, and three or fewer windows the rest, at three roundings each of
    what they hold, 120. These are errors relative to what each part adds, so the number of parts does
    not matter. From a tile's start the walk adds 6 a row, over 64 rows at most, 384. Below 1000 in all."""
    from mlx_lattice_b200 import _ext

    rows = 96_000
    ones = torch.ones((rows, 8), device=cuda)
    gate = torch.full_like(ones, value)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=cuda)
    rest = 1 / (1 + np.exp(value))
    h, final, carries = _ext.recurrence_forward(ones, gate, offsets, want_state=True, want_carries=True)
    want = -np.expm1(np.arange(1, rows + 1) * np.log1p(-rest))
    off = np.abs(_np(h) / want[:, None] - 1).max()
    assert off <= 1000 * U32, off / U32
    # dh counts the rows behind, each by its product of gates: (1 - a^(n - t)) / (1 - a)
    dx, _, _ = _ext.recurrence_backward(ones, None, ones, gate, offsets, None, False, carries)
    off = np.abs(_np(dx) / want[::-1, None] - 1).max()
    assert off <= 1000 * U32, off / U32


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('reverse', [False, True])
def test_recurrence_carries_infinities(cuda, dtype, reverse):
    """An infinite value, state or gradient gives what the formula gives, not a NaN of its own
    making; one of each sign gives NaN."""
    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(11)
    rows, channels, cuts = 300, 12, [0, 130, 260, 300]
    x, z = _randn(rng, rows, channels, dtype=dtype), _randn(rng, rows, channels, dtype=dtype, scale=4.0)
    dy, state = _randn(rng, rows, channels, dtype=dtype), _randn(rng, 3, channels)
    inf = float('inf')
    x[50, 0:4], x[60, 2:4] = inf, torch.tensor([inf, -inf], dtype=dtype, device=cuda)
    x[129 if not reverse else 0, 5] = -inf      # the last row of a sequence
    state[1, 4:6] = torch.tensor([inf, -inf], device=cuda)
    dy[220, 8:10] = torch.tensor([inf, -inf], dtype=dtype, device=cuda)
    off = torch.tensor(cuts, dtype=torch.int32, device=cuda)
    leaves = [t.requires_grad_(True) for t in (x, z, state)]
    y, final = ops.gated_recurrence(_sparse(x), z, initial_state=state, offsets=off, reverse=reverse, return_state=True)
    dx, dz, dstate = torch.autograd.grad(y.feats, leaves, dy)

    ref = [t.detach().double().cpu() for t in (x, z, state, dy)]
    a, k = torch.sigmoid(ref[1]), torch.sigmoid(-ref[1])
    h, flow = torch.zeros_like(ref[0]), torch.zeros_like(ref[0])
    last, first = torch.zeros_like(ref[2]), torch.zeros_like(ref[2])
    wdx, wdz = torch.zeros_like(ref[0]), torch.zeros_like(ref[0])
    for j in range(3):
        order = list(range(cuts[j], cuts[j + 1]))
        order = order[::-1] if reverse else order
        now, seen = ref[2][j], []
        for t in order:
            seen.append(now)
            now = a[t] * now + k[t] * ref[0][t]
            h[t] = now
        last[j] = now
        back = torch.zeros(channels, dtype=torch.float64)
        for t, prior in zip(order[::-1], seen[::-1]):
            dh = ref[3][t] + back
            wdx[t], wdz[t] = k[t] * dh, a[t] * k[t] * dh * (prior - ref[0][t])
            back = a[t] * dh
        first[j] = back
    for got, want, name in ((y.feats, h, 'h'), (final, last, 'final'), (dx, wdx, 'dx'), (dz, wdz, 'dgate'),
                            (dstate, first, 'dinitial')):
        got = got.detach().double().cpu()
        assert torch.equal(got.isnan(), want.isnan()), (name, (got.isnan() != want.isnan()).nonzero()[:5].tolist())
        assert torch.equal(got.isposinf(), want.isposinf()) and torch.equal(got.isneginf(), want.isneginf()), name
    one = torch.full((2, 4), inf, device=cuda, dtype=dtype)
    gate = torch.tensor([[-3.0, 3.0, -3.0, 3.0]] * 2, device=cuda).to(dtype)
    start = torch.tensor([[0.0] * 4, [1.0, inf, -inf, -inf]], device=cuda)
    h, _ = ops.gated_recurrence_step(_sparse(one), gate, start)
    assert (h.feats[0] == inf).all() and (h.feats[1, :2] == inf).all() and h.feats[1, 2:].isnan().all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('far', [100.0, float('inf')])
def test_recurrence_behind_shut_gates(cuda, dtype, far):
    """Masks of the type's lowest value: a shut gate keeps the state whatever lies in the row, and one
    that is wide open forgets the state whatever it was, in rows and steps."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(19)
    lowest = torch.finfo(dtype).min
    rows, offsets = 200, torch.tensor([0, 200], dtype=torch.int32, device=cuda)
    x = _randn(rng, rows, 6, dtype=dtype)
    state = _randn(rng, 1, 6)
    masked, gate = x.clone(), torch.full_like(x, -far)
    for t in range(0, rows, 3):
        gate[t], masked[t] = far, lowest
    state_far = torch.full_like(state, torch.finfo(torch.float32).min)
    for initial, first in ((state, far), (state_far, -far)):
        gate[0] = first
        values = masked if first == far else torch.cat([x[:1], masked[1:]])
        want, now = torch.empty_like(x), initial[0]
        for t in range(rows):
            now = now if gate[t, 0] > 0 else values[t].float()
            want[t] = now.to(dtype)
        h, final, _ = _ext.recurrence_forward(values, gate, offsets, initial, want_state=True)
        assert torch.equal(h, want) and torch.equal(final[0], now)
        one, after = _ext.recurrence_step(values[:1], gate[:1], initial)
        assert torch.equal(one, want[:1]) and torch.equal(after, (initial if first == far else values[:1].float()))


def test_recurrence_of_values_near_the_largest(cuda):
    """h - x may leave the range of float32 where neither the weights nor the result do."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(14)
    x = np.where(rng.random((200, 8)) < 0.5, 3e38, -3e38).astype(np.float32).astype(np.float64)
    z = rng.uniform(-4, 4, (200, 8)).astype(np.float32).astype(np.float64)
    state = np.full((1, 8), -3e38, np.float32).astype(np.float64)
    on = lambda v: torch.from_numpy(v).float().to(cuda)
    h, final, _ = _ext.recurrence_forward(on(x), on(z), torch.tensor([0, 200], dtype=torch.int32, device=cuda),
                                          on(state), want_state=True)
    zeros = np.zeros((200, 8))
    want = _reference(x, z, [0, 200], state, False, zeros, zeros[:1])
    _within(h, *want['h'], torch.float32, 'h')
    _within(final, *want['final'], torch.float32, 'final')


# --------------------------------------------------------------------------- #
# long runs of empty sequences
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize('reverse', [False, True])
def test_a_million_empty_sequences_between_two(cuda, reverse):
    """A pool of streams that is mostly unused: values as without the empty ones, and the time of a
    few searches, not of a walk over a million entries (tens of milliseconds in each kernel)."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(31)
    rows, empty = 6000, 1_000_000
    x, z, dy = (_randn(rng, rows, 8) for _ in range(3))
    few = torch.tensor([0, 2990, 3001, rows], dtype=torch.int32, device=cuda)
    many = torch.cat([few[:1], torch.full((empty,), 2990, dtype=torch.int32, device=cuda),
                      torch.full((empty,), 3001, dtype=torch.int32, device=cuda), few[3:]])
    h, _, carries = _ext.recurrence_forward(x, z, few, None, reverse, want_carries=True)
    dx, dz, _ = _ext.recurrence_backward(dy, None, x, z, few, None, reverse, carries)

    def run():
        got, _, kept = _ext.recurrence_forward(x, z, many, None, reverse, want_carries=True)
        return (got, *_ext.recurrence_backward(dy, None, x, z, many, None, reverse, kept)[:2])

    assert all(torch.equal(a, b) for a, b in zip(run(), (h, dx, dz)))
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    run()
    end.record()
    end.synchronize()
    assert begin.elapsed_time(end) < 20.0, begin.elapsed_time(end)
    _ext.check_status(cuda)


@pytest.mark.parametrize('rows', [64, 6000])
def test_a_million_empty_sequences_hand_on_their_states(cuda, rows):
    """Few rows, many states: all blocks that there are copy them (one block alone takes 60 ms)."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(37)
    many = 1_000_000
    x, dy = _randn(rng, rows, 16), _randn(rng, rows, 16)
    offsets = torch.full((many + 1,), rows // 2, dtype=torch.int32, device=cuda)
    offsets[0], offsets[-1] = 0, rows
    state = torch.randn((many, 16), device=cuda)
    flow = torch.randn((many, 16), device=cuda)

    def run():
        h, final, carries = _ext.recurrence_forward(x, x, offsets, state, want_state=True, want_carries=True)
        return final, _ext.recurrence_backward(dy, flow, x, x, offsets, state, False, carries, want_initial=True)[2]

    final, dstate = run()
    assert torch.equal(final[1:-1], state[1:-1]) and torch.equal(dstate[1:-1], flow[1:-1])
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    run()
    end.record()
    end.synchronize()
    assert begin.elapsed_time(end) < 20.0, begin.elapsed_time(end)
    _ext.check_status(cuda)


@pytest.mark.parametrize('reverse', [False, True])
def test_falling_offsets_stay_within_the_arrays(cuda, reverse):
    """Offsets that fall, with runs of empty sequences longer than those stepped over one by one:
    both passes report them, and write nothing around their outputs."""
    from mlx_lattice_b200 import _ext, _native

    lib, pad, rows = _native.load(), 64, 200
    rng = np.random.default_rng(33)
    x = _randn(rng, rows, 4)
    for trial in range(8):
        cuts = rng.integers(-20, rows + 20, size=40)
        cuts[5:20] = cuts[4]
        off = torch.from_numpy(cuts.astype(np.int32)).to(cuda)
        buffers = [torch.full((n * 4 + 2 * pad,), 7.0, device=cuda) for n in (rows, 39, rows, rows, 39)]
        h, final, dx, dz, dinitial = (b[pad:].data_ptr() for b in buffers)
        state = _randn(rng, 39, 4)
        carries = torch.zeros((lib.lat_recurrence_carry_rows(rows), 4), device=cuda)
        need = lib.lat_recurrence_workspace_bytes(0, rows, 4)
        workspace = torch.empty(need, dtype=torch.uint8, device=cuda)
        status, stream = torch.zeros(1, dtype=torch.int32, device=cuda), torch.cuda.current_stream().cuda_stream
        assert lib.lat_recurrence_forward(
            0, x.data_ptr(), 4, x.data_ptr(), 4, rows, 4, off.data_ptr(), 39, state.data_ptr(), int(reverse), h, final,
            carries.data_ptr(), workspace.data_ptr(), need, status.data_ptr(), stream) == _native.LAT_OK
        assert lib.lat_recurrence_backward(
            0, x.data_ptr(), 4, state.data_ptr(), x.data_ptr(), 4, x.data_ptr(), 4, rows, 4, off.data_ptr(), 39,
            state.data_ptr(), int(reverse), carries.data_ptr(), dx, dz, dinitial, workspace.data_ptr(), need,
            status.data_ptr(), stream) == _native.LAT_OK
        assert int(status) != 0
        for buffer in buffers:
            assert (buffer[:pad] == 7).all() and (buffer[-pad:] == 7).all()
    _ext.check_status(cuda)


# --------------------------------------------------------------------------- #
# the step and gradients
# --------------------------------------------------------------------------- #


def test_recurrence_step_does_not_lose_a_gradient_silently(cuda):
    """The step has values only: results that depend on something with a gradient say so when one
    is asked of them. Streams may go on from such a state, in place too."""
    from mlx_lattice_b200 import _ext, ops

    rng = np.random.default_rng(17)
    feats, gate, state = (_randn(rng, 6, 8) for _ in range(3))
    want, after = ops.gated_recurrence_step(_sparse(feats), gate, state)
    assert not want.feats.requires_grad and not after.requires_grad
    for place in range(3):
        args = [feats, gate, state]
        args[place] = args[place].clone().requires_grad_(True)
        h, new = ops.gated_recurrence_step(_sparse(args[0]), args[1], args[2])
        assert torch.equal(h.feats, want.feats) and torch.equal(new, after)
        for result in (h.feats, new):
            with pytest.raises(RuntimeError, match='gated_recurrence'):
                result.sum().backward()
        with torch.no_grad():
            h, new = ops.gated_recurrence_step(_sparse(args[0]), args[1], args[2])
        assert not h.feats.requires_grad and not new.requires_grad
    leaf, held = feats.clone().requires_grad_(True), state.clone()
    h, new = ops.gated_recurrence_step(_sparse(leaf), gate, held, out_state=held)
    assert torch.equal(held, after) and new.data_ptr() == held.data_ptr()
    h, new = ops.gated_recurrence_step(_sparse(leaf), gate, new, out_state=new)
    with pytest.raises(RuntimeError, match='gated_recurrence'):
        h.feats.sum().backward()
    with pytest.raises(ValueError, match='out_state'):
        ops.gated_recurrence_step(_sparse(feats), gate, state, out_state=state.clone().requires_grad_(True))
    with torch.no_grad():
        owner = state.clone().requires_grad_(True)
        _ext.recurrence_step(feats, gate, state, owner)
        assert torch.equal(owner, after)


def test_operators_without_a_gradient_say_that_they_detach(cuda):
    """A projection of this package between two recorded operators cuts the gradient: with a warning,
    where a gradient is asked for."""
    import warnings

    from mlx_lattice_b200 import _ext, ops

    feats = torch.ones((8, 16), device=cuda, requires_grad=True)
    places = torch.zeros((8, 8), dtype=torch.int32, device=cuda)
    weight = torch.ones((16, 16), device=cuda)
    x = ops.layer_norm(_sparse(feats))
    for call in (lambda y: ops.linear(y, weight), ops.silu, ops.relu,
                 lambda y: ops.batch_norm(y, mean=weight[0], var=weight[0]), lambda y: ops.sparse_add(y, y),
                 lambda y: _ext.interpolate_point_features(y.feats, places, torch.ones((8, 8), device=cuda))):
        with pytest.warns(UserWarning, match='no gradient'):
            call(x)
        with warnings.catch_warnings():
            warnings.simplefilter('error')
            with torch.no_grad():
                call(x)
            call(x.replace(feats=x.feats.detach()))
    with warnings.catch_warnings():   # the recorded ones say nothing
        warnings.simplefilter('error')
        ops.rms_norm(x)
        ops.dropout(x, p=0.5, seed=1)
        ops.gated_recurrence(x, x, offsets=torch.tensor([0, 8], dtype=torch.int32, device=cuda))


# --------------------------------------------------------------------------- #
# norms over frozen features, and their quotient
# --------------------------------------------------------------------------- #


@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_parameters_alone_over_frozen_features(cuda, dtype):
    """The first norm over a frozen backbone: features without a gradient, many rows; the bound and
    its reasons are those of the sums over 200,000 rows beside the other norm tests."""
    from test_training_ops_gpu import _close, _norm_reference

    from mlx_lattice_b200 import ops

    rng = np.random.default_rng(51)
    feats, dy = _randn(rng, 200_003, 24, dtype=dtype), _randn(rng, 200_003, 24, dtype=dtype)
    weight = _randn(rng, 24, dtype=dtype, shift=1.0).requires_grad_(True)
    bias = _randn(rng, 24, dtype=dtype).requires_grad_(True)
    y = ops.layer_norm(_sparse(feats), weight=weight, bias=bias).feats
    dw, db = torch.autograd.grad(y, (weight, bias), dy)
    want = _norm_reference(_np(feats), _np(weight), _np(bias), _np(dy), 1e-5, False)
    for got, name in ((y, 'y'), (dw, 'dw'), (db, 'db')):
        _close(got, *want[name], dtype, name)
    assert feats.grad is None


@pytest.mark.parametrize('channels', [3, 7, 24, 63, 64, 100, 191, 1000, 1023])
def test_row_means_are_within_one_unit_of_the_quotient(cuda, channels):
    """Integers whose sums are exact in any order (below 2^24): what is off is the division alone, by at
    most one unit in the last place, 2^-23 of the mean at most."""
    from mlx_lattice_b200 import _ext

    rng = np.random.default_rng(channels)
    x = rng.integers(-8000, 8000, size=(3000, channels)).astype(np.float32)
    _, mean, _ = _ext.row_norm_forward(torch.from_numpy(x).to(cuda), None, None, 1e-5, False)
    want = x.astype(np.float64).sum(1) / channels
    assert (np.abs(_np(mean) - want) <= 2.0 ** -23 * np.abs(want)).all()
