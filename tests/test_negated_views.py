"""Views whose values are those in memory negated (z.conj().imag of a complex tensor): operators
read memory, so they are given a copy, in direct calls as in dispatched ones."""

import pytest
import torch
from torch import Tensor

from qllm2_amd import _ops


def _negated(a: Tensor, b: Tensor) -> Tensor:
    """What a kernel that reads memory would meet."""
    return torch.tensor([a.is_neg(), b.is_neg()])


def test_operators_meet_no_negated_views():
    z = torch.randn(3, 4, dtype=torch.complex64)
    neg, plain = z.conj().imag, z.imag
    assert neg.is_neg() and not plain.is_neg()
    for name, direct in (("qpam::t_neg_direct", True), ("qpam::t_neg", False)):
        f = _ops.op(name, direct=direct)(_negated)
        for args in ((neg, plain), (plain, neg), (torch.nn.Parameter(plain), neg), (plain, plain)):
            with torch.no_grad():
                assert not f(*args).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_lookups_and_scores_of_negated_views(gpu_lib, dtype):
    from qllm2_amd.embedding import complex_embedding
    from qllm2_amd.linear4 import Weight4, linear4
    from qllm2_amd.token_logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch._neg_view(torch.randn(5, 64, device="cuda", generator=g).to(dtype))
    w = Weight4.quantize(torch.randn(20, 64, device="cuda", generator=g))
    ids = torch.tensor([0, 3, 4], device="cuda")
    with torch.no_grad():
        assert x.is_neg() and torch.equal(linear4(x, w), linear4(x.resolve_neg(), w))
        assert torch.equal(token_logprobs(x[:3], ids).logprobs, token_logprobs(x[:3].resolve_neg(), ids).logprobs)
        z = torch.view_as_complex(torch.randn(5, 8, 2, device="cuda", generator=g))
        table = z.conj().imag
        assert table.is_neg() and torch.equal(complex_embedding(ids, z.real, table)[..., 1], table[ids])
