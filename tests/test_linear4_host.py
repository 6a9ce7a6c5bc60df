"""CPU checks of the 4-bit products: gradients in either mode are refused; the entries' arguments."""

import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from qllm2_amd.linear4 import Weight4, complex_linear4, linear4
from tests.conftest import ROOT


def _calls():
    """(a call of one tensor, that tensor's shape): rows, bias and tail of both products."""
    w, c = Weight4.quantize(torch.randn(8, 32)), Weight4.quantize(torch.randn(8, 32), torch.randn(8, 32))
    x, z = torch.randn(2, 32), torch.randn(2, 32, 2)
    return [(lambda t: linear4(t, w), (2, 32)), (lambda t: linear4(x, w, t), (8,)), (lambda t: complex_linear4(t, c), (2, 32, 2)),
            (lambda t: complex_linear4(z, c, t), (8, 2)), (lambda t: complex_linear4(z, c, planes=True, tail=t), (3, 64))]


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("call,shape", _calls())
def test_forward_mode_gradients_are_refused(call, shape, no_grad):
    """No answer without its tangent; torch.no_grad() leaves forward mode on."""
    with torch.set_grad_enabled(not no_grad):
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="no gradient"):
                call(forward_ad.make_dual(torch.randn(shape), torch.randn(shape)))
            with pytest.raises(ValueError, match="GPU"):   # a tensor without a tangent is as ever
                call(torch.randn(shape))
        with pytest.raises(ValueError, match="no gradient"):
            torch.func.jvp(call, (torch.randn(shape),), (torch.randn(shape),))


@pytest.mark.parametrize("call,shape", _calls())
def test_reverse_mode_gradients_are_refused(call, shape):
    with pytest.raises(ValueError, match="no gradient"):
        call(torch.randn(shape, requires_grad=True))
    with pytest.raises(ValueError, match="no gradient"):
        torch.func.grad(lambda t: call(t).sum())(torch.randn(shape))
    with pytest.raises(ValueError, match="no gradient"):
        torch.func.vmap(torch.func.grad(lambda t: call(t).sum()))(torch.randn(3, *shape))


def test_entries_take_null_arguments():
    """No bytes and an error (in a process of its own: reading them ended it)."""
    code = ("from qllm2_amd import _lib; L = _lib.lib(); "
            "assert L.qpam_linear4_workspace_size(None) == 0 and L.qpam_linear4(None, None) == _lib.QPAM_ERR_ARG; "
            "assert L.qpam_copy_slots(None, None) == _lib.QPAM_ERR_ARG")
    assert subprocess.run([sys.executable, "-c", code], cwd=ROOT, timeout=300).returncode == 0
