"""Scores of a decoder with a 4-bit table.

A score is the log probability of a softmax over logits that are fp32 sums of exact products
of the head's rows and the codes' values; a log probability is off by at most twice the
largest error of a logit, below 2e-5 here (logits up to some tens, sums of 256 terms: 2^-24
times the sum of magnitudes, at most 16 times the logit's, and the softmax's own sums)."""

import pytest
import torch

from tests.test_gpu_model_decode import VOCAB
from tests.test_gpu_serving import _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 128])
@torch.no_grad()
def test_scores_are_those_of_the_codes_values(gpu_lib, dtype, group, bits):
    from qllm2_amd.model_decode import ModelDecoder
    dec = ModelDecoder(_model("e3_swish"), n_slots=2, dtype=dtype, weight_bits=bits, table_bits=4, weight_group=group)
    ids = _tokens(110, 40)
    h, _ = dec._prompt_rows(ids)
    logits = dec._lm_rows(h[:-1]).double() @ dec._table4.dequantize().double().T.contiguous()
    for temperature in (1.0, 0.7):
        lp = torch.log_softmax(logits / temperature, -1)
        got = dec.score(ids, temperature=temperature)
        assert (got.logprobs - lp.gather(1, ids[1:, None])[:, 0]).abs().max() < 2e-5
        assert (got.entropy + (lp.exp() * lp).sum(-1)).abs().max() < 1e-4
        assert got.logprobs.dtype == got.entropy.dtype == torch.float32 and got.logprobs.shape == (39,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_long_scores_in_pieces(gpu_lib, monkeypatch, dtype):
    """As many pieces of rows as it takes, the last one odd; ids outside the vocabulary."""
    from qllm2_amd import model_decode
    dec = model_decode.ModelDecoder(_model("one_state_relu"), n_slots=2, dtype=dtype, table_bits=4)
    ids = _tokens(111, 150)
    whole = dec.score(ids)
    monkeypatch.setattr(model_decode, "SCORE_LOGITS", 64 * VOCAB)
    pieces = dec.score(ids)
    assert torch.allclose(pieces.logprobs, whole.logprobs, rtol=0, atol=2e-5)
    assert torch.allclose(pieces.entropy, whole.entropy, rtol=0, atol=1e-4)
    bad = ids[:70].clone()   # (64 rows, and the rest)
    bad[66] = VOCAB
    got = dec.score(bad).logprobs
    assert torch.isnan(got[65:]).all() and not torch.isnan(got[:60]).any()
    assert dec.score(ids[:2]).logprobs.shape == (1,)


def test_a_four_bit_table_is_not_kept_whole_beside_its_codes(gpu_lib):
    """The fp32 table of the lookups and the codes; no dense copy of the codes' values."""
    from qllm2_amd.model_decode import ModelDecoder
    dec = ModelDecoder(_model("e3_swish"), n_slots=2, dtype=torch.bfloat16, table_bits=4)
    size = dec.vocab * 2 * dec.dim
    held = [v for v in vars(dec).values() if torch.is_tensor(v) and v.numel() == size]
    assert not held
