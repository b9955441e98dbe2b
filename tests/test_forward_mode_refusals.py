"""CPU: tensors that carry a forward-mode derivative are refused by the operators that have none, before a kernel
runs (a dual tensor requires no gradient, so nothing else would notice that its tangent is lost)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from lvmhelpers import _native

NODES = {
    "linear_act": ([torch.ones(2, 3), torch.ones(4, 3), torch.ones(4), torch.ones(2, 4)], lambda f, t: f(*t, 0)),
    "token_logprobs": ([torch.ones(1, 2, 3)], lambda f, t: f(t[0], torch.zeros(1, 2, dtype=torch.int64), None)),
    "clipped_policy_loss": ([torch.ones(1, 2, 3), torch.ones(1, 2), torch.ones(1, 2), torch.ones(1, 2)],
                            lambda f, t: f(t[0], torch.zeros(1, 2, dtype=torch.int64), *t[1:], None, 0.2, 0.2, 0.0, 0.0, True)),
}


@pytest.mark.parametrize("name,i", [(n, i) for n, (t, _) in NODES.items() for i in range(len(t))])
@pytest.mark.parametrize("record", [False, True])
def test_tangents_are_refused(name, i, record):
    tensors, call = NODES[name]
    with fwad.dual_level(), torch.set_grad_enabled(record):
        given = [t.clone().requires_grad_(record and j == 0 and i != 0) for j, t in enumerate(tensors)]
        given[i] = fwad.make_dual(given[i], torch.ones_like(given[i]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(getattr(_native.autograd(), name), given)
