"""Captured steps of beams whose parents are chosen on the device."""

import pytest
import torch

from tests.test_gpu_model_decode import _row_rel
from tests.test_gpu_serving import _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [None, 4])
def test_beams_reordered_on_the_device_keep_the_table_and_the_graphs(gpu_lib, bits):
    """Searches of short sequences one after another beside one that stays: more steps than the rotary table has rows,
    the table and the captured graphs the same throughout, the logits those of the sequences alone."""
    from qllm2_amd.model_decode import ModelDecoder
    model = _model("e3_swish")
    dec = ModelDecoder(model, n_slots=6, max_len=16, weight_bits=bits, graphs=True, graph_bucket=4)
    stays, _ = dec.admit(_tokens(120, 2))
    rope = graphs = None
    for search in range(8):
        first, _ = dec.admit(_tokens(121 + search, 4))
        beams = [first, *dec.fork(first, 2)]
        live = torch.tensor(beams, device="cuda", dtype=torch.int32)
        said = [[], [], []]
        for i in range(6):
            ids = _tokens(130 + 10 * search + i, 3)
            got = dec.step(ids, live, host_slots=beams).clone()
            said = [[*s, t] for s, t in zip(said, ids.tolist())]
            if i < 5:
                parents = [i % 3, 0, (i + 1) % 3]
                dec.reorder(live, live[torch.tensor(parents, device="cuda")])
                said = [said[p] for p in parents]
        if rope is None:
            rope, graphs = dec.pool.rope, dict(dec._graphs)
        assert dec.pool.rope is rope and dec._graphs == graphs and graphs
        assert dec.pool.pos[beams].tolist() == [10] * 3 and int(dec.pool.pos[stays]) == 2
        if search in (0, 7):
            alone = ModelDecoder(model, n_slots=1, max_len=16, weight_bits=bits)
            for row, tokens in zip(got, said):
                slot, _ = alone.admit(_tokens(121 + search, 4))
                for t in tokens:
                    want = alone.step(torch.tensor([t], device="cuda"), torch.tensor([slot], device="cuda", dtype=torch.int32))
                assert _row_rel(row[None], want) < 1e-4
                alone.release(slot)
        for s in beams:
            dec.release(s)
