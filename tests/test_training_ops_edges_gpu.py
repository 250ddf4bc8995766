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
