"""The tied table's two ends together, as a model uses them: token ids -> embedding
lookup -> ComplexNorm -> a projection -> token log probabilities against the same
tables, with the gradients of both uses summed; the model decoder's scores and
alternatives against the float64 oracle model; and what holds for every operator:
no output shares memory with an input, a second derivative raises, calls through the
dispatcher and around it agree, torch.compile traces it."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from oracle import complex_ops as C
from oracle import v11_model as VM

pytestmark = pytest.mark.gpu


def _objective(ids, targets, re, im, scale, proj, ops):
    """Mean log probability of the targets plus 0.1 of the mean entropy."""
    z = ops["norm"](ops["embed"](ids, re, im), scale)
    h = z.reshape(z.shape[0], -1) @ proj
    lp, ent = ops["scores"](h, torch.cat([re, im], 1), targets)
    return lp.sum() / (targets >= 0).sum() + 0.1 * ent.mean()


def _torch_scores(h, w, t):
    logp = torch.log_softmax(h @ w.T, -1)
    return (torch.where(t >= 0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0), -(logp.exp() * logp).sum(-1))


@pytest.mark.parametrize("dtype,n", [(torch.float32, 333), (torch.bfloat16, 700), (torch.float32, 20)])
def test_training_step_through_both_ends(gpu_lib, dtype, n):
    """Gradients of a tied model's tables, norm scale and projection against float64
    autograd.  fp32: sums of a few hundred terms of either sign, 1e-4 of the largest
    entry; bf16: lookup, norm, projection, dx and each gradient round once (2^-8 each),
    and the two uses of the tables add: 6 * 2^-8 norm-wise."""
    from qllm2_amd import triton_kernels as tk
    from qllm2_amd.embedding import complex_embedding
    from qllm2_amd.token_logprobs import linear_token_logprobs
    V, dim = 515, 48
    g = torch.Generator().manual_seed(n)
    ids = (V ** torch.rand(n, generator=g) - 1).long()
    targets = torch.randint(0, V, (n,), generator=g)
    targets[::6] = -100
    leaves = [(torch.randn(s, generator=g) * std + mean).to(dt) for s, std, mean, dt in (
        ((V, dim), 0.3, 0, dtype), ((V, dim), 0.3, 0, dtype), ((dim,), 0.1, 1, torch.float32),
        ((2 * dim, 2 * dim), (2 * dim) ** -0.5, 0, dtype))]
    own = [t.cuda().requires_grad_() for t in leaves]
    ref = [t.double().requires_grad_() for t in leaves]
    got = _objective(ids.cuda(), targets.cuda(), *own, dict(
        norm=tk.fused_complex_norm, embed=lambda i, a, b: complex_embedding(i, a, b, scale=7.0),
        scores=lambda h, w, t: linear_token_logprobs(h, w, t)[:2]))
    want = _objective(ids, targets, *ref, dict(
        norm=lambda z, s: C.complex_norm(z, s, 1e-6), embed=lambda i, a, b: 7.0 * torch.stack([a[i], b[i]], -1),
        scores=_torch_scores))
    tol = 1e-4 if dtype == torch.float32 else 6 * 2.0 ** -8
    assert abs(got.item() - want.item()) <= tol * abs(want.item())
    for a, b in zip(torch.autograd.grad(got, own), torch.autograd.grad(want, ref)):
        a = a.cpu().double()
        if dtype == torch.float32:
            assert ((a - b).abs().max() / b.abs().max()).item() < tol
        else:
            assert ((a - b).norm() / b.norm()).item() < tol


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 3e-2)])
def test_model_decoder_scores_and_alternatives(gpu_lib, dtype, tol):
    """score() of a sequence, and logprobs() of prefill and steps fed the same tokens,
    against the oracle model's log-softmax.  The logits agree to tol of a row's largest
    (what the decoder's own test holds), log probabilities to twice that."""
    from qllm2_amd.model_decode import ModelDecoder
    cfg = dict(dim=128, n_heads=2, head_dim=64, n_states=1, chunk_size=64)
    p = VM.make_model_params(cfg, 2, 300, 77)
    ref = VM.V11LM(cfg, 2, p).eval()
    gpu = VM.V11LM(cfg, 2, {k: v.float() for k, v in p.items()}, dtype=torch.float32).cuda().eval()
    dec = ModelDecoder(gpu, n_slots=2, max_len=64, dtype=dtype, graphs=True, graph_bucket=2)
    ids = torch.randint(0, 300, (23,), generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        logits = ref(ids.view(1, -1))[0][0]
    logp = torch.log_softmax(logits, -1)
    bound = 2 * tol * logits.abs().max().item()
    r = dec.score(ids.cuda())
    assert r.logprobs.shape == r.entropy.shape == (22,)
    assert (r.logprobs.cpu() - logp[:-1].gather(1, ids[1:, None])[:, 0]).abs().max() < bound
    ent = -(logp.exp() * logp).sum(-1)
    # d H = -sum p (ln p + H) d x: at most max |ln p + H| times the logits' error
    slack = bound * (1 + (logp + ent[:, None]).abs().max().item())
    assert (r.entropy.cpu() - ent[:-1]).abs().max() < slack
    with pytest.raises(ValueError, match="two tokens"):
        dec.score(ids[:1])

    slot, row = dec.admit(ids[:10].cuda())
    rows = [row]
    for t in range(10, 22):
        rows.append(dec.step(ids[t:t + 1].cuda(), torch.tensor([slot], dtype=torch.int32, device="cuda"), [slot])[0].clone())
    rows = torch.stack(rows)                      # after tokens 9 .. 21
    s = dec.logprobs(rows, ids[10:23].cuda(), top_k=4)
    assert (s.logprobs.cpu() - logp[9:22].gather(1, ids[10:23, None])[:, 0]).abs().max() < bound
    assert torch.equal(s.top_ids, torch.sort(rows, dim=-1, descending=True, stable=True).indices[:, :4])
    assert (s.top_logprobs.cpu() - logp[9:22].gather(1, s.top_ids.cpu())).abs().max() < bound
    assert (s.logprobs - r.logprobs[9:]).abs().max() < bound


class _Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen, self.bad = set(), []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if func.namespace == "qpam":
            name = func._schema.name.split("::")[1]
            self.seen.add(name)
            ins = {a.untyped_storage().data_ptr() for a in args if isinstance(a, torch.Tensor) and a.numel()}
            outs = out if isinstance(out, (list, tuple)) else [out]
            if any(o.numel() and o.untyped_storage().data_ptr() in ins for o in outs):
                self.bad.append(name)
        return out


def _calls(dtype):
    from qllm2_amd.embedding import complex_embedding
    from qllm2_amd.token_logprobs import linear_token_logprobs, token_logprobs
    rn = lambda *s: torch.randn(*s, device="cuda").to(dtype).requires_grad_()  # noqa: E731
    ids = torch.randint(0, 64, (40,), device="cuda")
    re, im, x, h, w = rn(64, 32), rn(64, 32), rn(40, 64), rn(40, 32), rn(64, 32)
    yield complex_embedding(ids, re, im), [re, im]
    r = token_logprobs(x, ids, top_k=3)
    yield [r.logprobs, r.entropy, r.top_logprobs], [x]
    r = linear_token_logprobs(h, w, ids)
    yield [r.logprobs, r.entropy], [h, w]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_outputs_are_their_own_and_second_derivatives_raise(gpu_lib, dtype):
    with _Watch() as watch:
        watched = []
        for outs, leaves in _calls(dtype):
            outs = outs if isinstance(outs, list) else [outs]
            watched.append([o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])))
    assert not watch.bad, watch.bad
    assert {"embed_fwd", "embed_bwd", "logprobs_fwd", "logprobs_bwd", "linear_logprobs_fwd",
            "linear_logprobs_bwd"} <= watch.seen
    for outs, leaves in _calls(dtype):
        outs = outs if isinstance(outs, list) else [outs]
        seeds = [torch.ones_like(o).requires_grad_() for o in outs]
        first = torch.autograd.grad(outs, leaves, seeds, create_graph=True)
        with pytest.raises(RuntimeError, match="no backward"):
            torch.autograd.grad([f.float().sum() for f in first], seeds, allow_unused=True)


def test_direct_and_dispatched_calls_agree(gpu_lib):
    """The same bits through the dispatcher (under a mode) and around it."""
    for dtype in (torch.float32, torch.bfloat16):
        torch.manual_seed(3)
        plain = [torch.autograd.grad(o, v, [torch.ones_like(t) for t in (o if isinstance(o, list) else [o])])
                 for o, v in _calls(dtype)]
        torch.manual_seed(3)
        with _Watch():
            through = [torch.autograd.grad(o, v, [torch.ones_like(t) for t in (o if isinstance(o, list) else [o])])
                       for o, v in _calls(dtype)]
        for a, b in zip(plain, through):
            for s, t in zip(a, b):
                assert torch.equal(s, t)


def test_compiled_program_traces_the_operators(gpu_lib):
    """torch.compile keeps each operator one node (eager backend: no generated code)."""
    from qllm2_amd.embedding import complex_embedding
    from qllm2_amd.token_logprobs import linear_token_logprobs, token_logprobs
    ids = torch.randint(0, 64, (40,), device="cuda")
    re, im, w = (torch.randn(64, 32, device="cuda") for _ in range(3))

    def f(ids, re, im, w):
        h = complex_embedding(ids, re, im).flatten(1)[:, :32]
        a = linear_token_logprobs(h, w, ids)
        b = token_logprobs(h @ w.T, ids, top_k=2)
        return a.logprobs, a.entropy, b.logprobs, b.top_ids

    for got, want in zip(torch.compile(f, backend="eager", fullgraph=True)(ids, re, im, w), f(ids, re, im, w)):
        assert torch.equal(got, want)


def _decoder(dtype, graphs):
    from qllm2_amd.model_decode import ModelDecoder
    cfg = dict(dim=128, n_heads=2, head_dim=64, n_states=1, chunk_size=64)
    p = VM.make_model_params(cfg, 2, 300, 78)
    gpu = VM.V11LM(cfg, 2, {k: v.float() for k, v in p.items()}, dtype=torch.float32).cuda().eval()
    return ModelDecoder(gpu, n_slots=4, max_len=64, dtype=dtype, graphs=graphs, graph_bucket=2)


@pytest.mark.parametrize("graphs", [False, True])
def test_model_decoder_ids_outside_the_vocabulary(gpu_lib, graphs):
    """Host ids are refused; ids on the device, which the host does not read, give NaN logits, states and
    scores from there on, in their own sequence alone (within a prompt the prefill's products of a chunk
    may spread them to the tokens before)."""
    dec = _decoder(torch.float32, graphs)
    ok = torch.randint(0, 300, (9,), generator=torch.Generator().manual_seed(6))
    for wrong in (300, -1, -100, 2 ** 40):
        bad = ok.clone()
        bad[4] = wrong
        for call in (dec.prefill, dec.admit, dec.score):
            with pytest.raises(ValueError, match="vocabulary"):
                call(bad)
        assert dec.prefill(bad.cuda())[0].isnan().all()
        s = dec.score(bad.cuda())
        assert s.logprobs[3:].isnan().all() and s.entropy[4:].isnan().all()
        bad = ok.clone()
        bad[-1] = wrong
        assert dec.score(bad.cuda()).logprobs[-1].isnan()
    assert torch.equal(dec.score(ok).logprobs, dec.score(ok.cuda()).logprobs)
    first, _ = dec.admit(ok)
    second, _ = dec.admit(ok.cuda())
    slots, host = torch.tensor([first, second], dtype=torch.int32, device="cuda"), [first, second]
    with pytest.raises(ValueError, match="vocabulary"):
        dec.step(torch.tensor([5, 300]), slots, host)
    a = dec.step(torch.tensor([5, 5], device="cuda"), slots, host).clone()
    assert torch.equal(a[0], a[1])
    b = dec.step(torch.tensor([7, 300], device="cuda"), slots, host).clone()
    assert not b[0].isnan().any() and b[1].isnan().all()
    c = dec.step(torch.tensor([8, 8]), slots, host).clone()    # host ids, as device ids
    assert not c[0].isnan().any() and c[1].isnan().all()


def test_model_decoder_keeps_one_fp32_table(gpu_lib):
    """The lookups read the LM head's own table where that is fp32."""
    dec = _decoder(torch.float32, False)
    assert {t.untyped_storage().data_ptr() for t in dec._embed} == {dec._embed_w.untyped_storage().data_ptr()}
