"""Forward-mode derivatives of the row operators: there are none, and a tensor that carries a tangent is told so."""
import pytest
import torch
from torch.autograd import forward_ad

import ogl_amd  # noqa: F401
from ogl_amd import ops


def calls(device):
    x, w, b = torch.randn(4, 12, device=device), torch.ones(12, device=device), torch.zeros(12, device=device)
    weight = ops.quant_rows(6, 12, device=device)
    bias = torch.zeros(6, device=device)
    norm = lambda x, w, b: ops.group_norm(x, 3, w, b, activation="silu")  # noqa: E731
    return [(norm, (x, w, b), i) for i in range(3)] + [(lambda x, b: ops.linear_int8(x, weight, b), (x, bias), i) for i in range(2)]


def refused(device):
    for fn, args, i in calls(device):
        for grad in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = list(args)
                dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    fn(*dual)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(lambda t: fn(*[t if j == i else a for j, a in enumerate(args)]), (args[i],), (torch.ones_like(args[i]),))


def test_tangents_are_refused():
    refused("cpu")


@pytest.mark.gpu
def test_tangents_are_refused_on_the_gpu():
    refused("cuda")
    for fn, args, i in calls("cuda"):                                       # (inside a dual level, tensors without one are served)
        want = fn(*args)
        with forward_ad.dual_level():
            assert torch.equal(fn(*args), want)


@pytest.mark.gpu
def test_as_the_other_operators_do():
    x, w = torch.randn(4, 12, device="cuda"), torch.randn(6, 12, device="cuda")
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.linear(forward_ad.make_dual(x, torch.ones_like(x)), w)
