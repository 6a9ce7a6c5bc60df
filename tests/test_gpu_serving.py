"""ModelDecoder with 4-bit weights, and sequences forked, reordered and moved in its pool.

An fp32 decoder with weight_bits=4 is compared with one whose model holds the values that
the codes stand for: the same products but for the order of their sums, so the bound is that
of the full-precision decoder (test_gpu_model_decode.py: 1e-4 of a row's largest logit).  A
bf16 one is compared with itself on plain products in 64 bits rounded once: bf16 matrices
cannot hold the codes' values (a product of 3 and 8 bits), and two bf16 decoders that round
differently drift apart with the model (0.11 of a row's largest logit between bf16 and fp32
GEMMs here), while these two round alike but where a sum is within its fp32 error of a
border.  Its bound is that of the bf16 decoder, 3e-2."""

import copy

import pytest
import torch

from oracle import v11_model as VM
from tests.test_gpu_model_decode import CFGS, VOCAB, _row_rel

pytestmark = pytest.mark.gpu


def _model(name):
    cfg, act = CFGS[name]
    p = VM.make_model_params(cfg, 2, VOCAB, 910, activation=act)
    return VM.V11LM(cfg, 2, {k: v.float() for k, v in p.items()}, activation=act, dtype=torch.float32).cuda().eval()


def _dequantized(model, group):
    """The model with every ComplexLinear's weights at the values of their codes."""
    from qllm2_amd.linear4 import Weight4
    model = copy.deepcopy(model)
    with torch.no_grad():
        for m in model.modules():
            if hasattr(m, "weight_real"):
                w = Weight4.quantize(m.weight_real, m.weight_imag, group).dequantize()
                m.weight_real.copy_(w[..., 0]), m.weight_imag.copy_(w[..., 1])
    return model


def _plain_products(monkeypatch):
    """4-bit products of the decoders in plain float64, rounded once."""
    from qllm2_amd import engine, model_decode
    from tests.test_gpu_linear4 import _matrix

    def complex_product(x, w, bias=None, planes=False, tail=None):
        y = x.double().flatten(1) @ _matrix(w).T.contiguous()
        if bias is not None:
            y = y + bias.double().flatten()
        if not planes:
            return y.to(x.dtype).view(x.shape[0], -1, 2)
        parts = [y[:, 0::2], y[:, 1::2]] + ([] if tail is None else [x.double().flatten(1) @ tail.double().T.contiguous()])
        return torch.cat(parts, 1).to(x.dtype)

    monkeypatch.setattr(engine, "complex_linear4", complex_product)
    monkeypatch.setattr(model_decode, "linear4", lambda x, w: (x.double() @ _matrix(w).T.contiguous()).to(x.dtype))


def _tokens(seed, *shape):
    return torch.randint(0, VOCAB, shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("dtype,group", [(torch.float32, 32), (torch.float32, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("name", list(CFGS))
def test_four_bit_decoder_is_that_of_the_codes_values(gpu_lib, monkeypatch, name, dtype, group, graphs):
    from qllm2_amd.model_decode import ModelDecoder
    model = _model(name)
    kw = dict(n_slots=4, max_len=16, dtype=dtype, graphs=graphs, graph_bucket=2)
    dec = ModelDecoder(model, weight_bits=4, weight_group=group, **kw)
    prompts, steps, scored = [_tokens(n, n) for n in (5, 12, 3)], [_tokens(50 + i, 3 if i < 3 else 2) for i in range(5)], _tokens(60, 20)

    def all_of(d):
        """Logits of the prompts and of the steps, log probabilities of a scored sequence."""
        slots, out = [], []
        for prompt in prompts:
            slot, logits = d.admit(prompt)
            slots.append(slot), out.append(logits[None])
        live = torch.tensor(slots, device="cuda", dtype=torch.int32)
        out += [d.step(ids, live[:ids.numel()]).clone() for ids in steps]
        return out, d.score(scored).logprobs

    got = all_of(dec)
    if dtype == torch.float32:
        tol, ref = 1e-4, ModelDecoder(_dequantized(model, group), **kw)
    else:
        _plain_products(monkeypatch)
        tol, ref = 3e-2, ModelDecoder(model, weight_bits=4, weight_group=group, **{**kw, "graphs": False})
    want = all_of(ref)
    for a, b in zip(got[0], want[0]):
        assert _row_rel(a, b) < tol
    assert (got[1] - want[1]).abs().max() < 20 * tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_four_bit_table(gpu_lib, dtype):
    """The logits of the decoder's own rows against the codes' values, and a score that goes with them."""
    from qllm2_amd.model_decode import ModelDecoder
    model = _model("e3_swish")
    dec = ModelDecoder(model, n_slots=2, dtype=dtype, table_bits=4, weight_group=64)
    plain = ModelDecoder(model, n_slots=2, dtype=dtype)
    ids = _tokens(70, 12)
    h, _ = dec._prompt_rows(ids)
    lm = dec._lm_rows(h)
    want = lm.double() @ dec._table4.dequantize().double().T.contiguous()
    assert _row_rel(dec._head(h), want) < (1e-5 if dtype == torch.float32 else 2.0 ** -8)
    lp = torch.log_softmax(want[:-1], -1).gather(1, ids[1:, None])[:, 0]
    assert (dec.score(ids).logprobs - lp).abs().max() < (1e-3 if dtype == torch.float32 else 0.2)
    assert torch.equal(dec._embedded(ids), plain._embedded(ids))   # the lookup keeps the table's values
    slot, logits = dec.admit(ids)
    assert logits.shape == (VOCAB,) and dec.step(ids[:1], torch.tensor([slot], device="cuda", dtype=torch.int32)).dtype == torch.float32


def test_projection_biases(gpu_lib):
    """q, k, v, o and head biases go with 4-bit weights."""
    from qllm2_amd.model_decode import ModelDecoder
    model = _model("one_state_relu")
    g = torch.Generator(device="cuda").manual_seed(80)
    for m in model.modules():
        if hasattr(m, "weight_real") and hasattr(m, "bias_real"):
            for name in ("bias_real", "bias_imag"):
                setattr(m, name, torch.nn.Parameter(torch.randn(m.weight_real.shape[0], device="cuda", generator=g) * 0.1))
    dec = ModelDecoder(model, n_slots=2, weight_bits=4)
    ref = ModelDecoder(_dequantized(model, 32), n_slots=2)
    prompt = _tokens(81, 9)
    (a, la), (b, lb) = dec.admit(prompt), ref.admit(prompt)
    assert _row_rel(la[None], lb[None]) < 1e-4
    live, ids = torch.tensor([a], device="cuda", dtype=torch.int32), _tokens(82, 1)
    assert _row_rel(dec.step(ids, live), ref.step(ids, live)) < 1e-4


def test_new_weights(gpu_lib):
    from qllm2_amd.model_decode import ModelDecoder
    model = _model("e3_swish")
    dec = ModelDecoder(model, n_slots=4, weight_bits=4, table_bits=4, graphs=True, graph_bucket=2)
    slot, _ = dec.admit(_tokens(90, 4))
    live = torch.tensor([slot], device="cuda", dtype=torch.int32)
    for i in range(3):
        dec.step(_tokens(91 + i, 1), live)
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(1.25)
    dec.refresh_weights()
    other = ModelDecoder(model, n_slots=4, weight_bits=4, table_bits=4)
    ids = _tokens(95, 6)
    assert torch.equal(dec.prefill(ids)[0], other.prefill(ids)[0])


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("bits", [None, 4])
def test_forked_reordered_and_moved_sequences_decode_as_their_own(gpu_lib, bits, graphs):
    """Samples of one prompt, a beam step with host and with device lists, a compacted pool: each sequence's
    logits are those of the same tokens decoded alone (the rows of a step do not mix: bit for bit where the
    batch is the same, else to the products' bounds)."""
    from qllm2_amd.model_decode import ModelDecoder
    model = _model("e3_swish")
    dec = ModelDecoder(model, n_slots=8, max_len=8, weight_bits=bits, graphs=graphs, graph_bucket=4)
    prompt = _tokens(100, 6)
    other, _ = dec.admit(_tokens(101, 9))
    first, _ = dec.admit(prompt)
    slots = [first, *dec.fork(first, 3)]
    said = {s: [] for s in slots}

    def step(seed):
        ids = _tokens(seed, len(slots))
        live = torch.tensor(slots, device="cuda", dtype=torch.int32)
        out = dec.step(ids, live, host_slots=slots).clone()
        for s, t in zip(slots, ids.tolist()):
            said[s] = [*said[s], t]
        return out

    step(102)
    step(103)
    parents = [slots[2], slots[0], slots[0], slots[3]]
    dec.reorder(slots, parents)
    said = dict(zip(slots, [said[p] for p in parents]))
    step(104)
    parents = [slots[1], slots[1], slots[3], slots[2]]
    dec.reorder(*(torch.tensor(v, device="cuda", dtype=torch.int32) for v in (slots, parents)))
    said = dict(zip(slots, [said[p] for p in parents]))
    step(105)
    dec.release(other)
    moved = dec.compact()
    slots = [moved.get(s, s) for s in slots]
    said = dict(zip(slots, said.values()))
    got = step(106)
    alone = ModelDecoder(model, n_slots=2, max_len=8, weight_bits=bits)
    for row, s in zip(got, slots):
        slot, _ = alone.admit(prompt)
        live = torch.tensor([slot], device="cuda", dtype=torch.int32)
        for t in said[s]:
            want = alone.step(torch.tensor([t], device="cuda"), live)
        assert _row_rel(row[None], want) < 1e-4
        assert int(dec.pool.pos[s]) == int(alone.pool.pos[slot]) == 6 + len(said[s])
        alone.release(slot)
