"""Log probabilities and entropies from hidden rows and the tied table, and their
gradients (qpam_linear_logprobs_fwd / qpam_linear_logprobs_bwd), against plain torch
in float64 on the operands' own values.

Tolerances, u = 2^-24 and a_v = sum |h_k w_vk| / T: a logit is a sum of D products
in fp32 (exact products of bf16 parts; fp32 ones round), off by at most E_v =
(D + 4) u a_v however it is grouped, and E = max E_v over the row.  With d = (max - x)
/ T, A = sum p d, B = sum p d^2 and L = V / 16 + 60 steps of joining sums:
  ln s, log prob: 2 E + u (L + 4 A + 3 d_t + 3 |ln s| + |log prob|)
  entropy:        ln s's + u (2 L A + 4 B + 4 A) + 2 E (1 + A + sqrt(B))
      (d entropy = -sum p (ln p + H) dx, and sum p |ln p + H| <= A + sqrt(B))
  dx_v: p_v / T (relative error of p (2 E + u (4 d + L + 4 A)) |bracket| + that of the
      bracket) + 4 u |dx_v|, + r |dx_v| for its rounding to bf16 (r = 2^-8, else 0)
  dh = dx w: sum_v tol(dx_v) |w_v| + V u sum_v |dx_v w_v| + eps / 2 |dh|; dw alike.
These are worst cases; the products' sums are checked norm-wise as well."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _reference(h, w, ids, T, gs, rounded):
    """float64 (outputs, tolerances); h, w on the CPU in the dtype the products read."""
    h, w = h.double(), w.double()
    n, D = h.shape
    V = w.shape[0]
    x, E = h @ w.T, ((D + 4) * U / T * (h.abs() @ w.abs().T).max(-1).values)
    m = x.max(-1, keepdim=True).values
    d = (m - x) / T
    s = torch.exp(-d).sum(-1)
    ln_s = s.log()
    p = torch.exp(-d) / s[:, None]
    A, B = (p * d).sum(-1), (p * d * d).sum(-1)
    H = ln_s + A
    logp = -d - ln_s[:, None]
    valid = (ids != -100) & (ids >= 0) & (ids < V)
    safe = torch.where(valid, ids, 0)
    lp = torch.where(valid, logp.gather(1, safe[:, None])[:, 0], 0.0)
    L = V / 16 + 60
    t_s = 2 * E + U * (L + 4 * A + 3 * ln_s.abs())
    t_lp = t_s + U * (3 * d.gather(1, safe[:, None])[:, 0] + lp.abs())
    t_H = t_s + U * (2 * L * A + 4 * B + 4 * A + H.abs()) + 2 * E * (1 + A + B.sqrt())
    out = dict(lp=lp, H=H, t_lp=t_lp, t_H=t_H)
    if gs is None:
        return out
    g_lp, g_ent = torch.where(valid, gs[0], 0.0), gs[1]
    br = g_lp[:, None] + g_ent[:, None] * (logp + H[:, None])
    extra = torch.zeros_like(x).scatter_add_(1, safe[:, None], g_lp[:, None])
    dx = (extra - p * br) / T
    rel = (2 * E + U * (L + 4 * A))[:, None] + 4 * U * d
    err_b = g_ent.abs()[:, None] * (t_H + t_s + 2 * E + 8 * U * (ln_s.abs() + H.abs()))[:, None] + 8 * U * (
        g_lp.abs()[:, None] + g_ent.abs()[:, None] * d)
    tol = p / T * (rel * br.abs() + err_b) + (4 * U + rounded) * (dx.abs() + extra.abs() / T * (4 * U)) + 2.0 ** -126
    out.update(dh=dx @ w, t_dh=tol @ w.abs() + V * U * (dx.abs() @ w.abs()),
               dw=dx.T @ h, t_dw=tol.T @ h.abs() + n * U * (dx.abs().T @ h.abs()))
    return out


def _close(got, want, tol, eps=0.0):
    err = (got.detach().cpu().double() - want).abs()
    bound = tol + eps / 2 * want.abs()
    assert (err <= bound).all(), ((err - bound).max().item(), err.max().item())


def _data(n, V, D, dtype, wdtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, D, generator=g).to(dtype)
    w = (torch.randn(V, D, generator=g) * std / D ** 0.5).to(wdtype)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[::5] = -100
    ids[3::7] = V + 1
    return h, w, ids, [torch.randn(n, generator=g) / n, torch.randn(n, generator=g) / n]


F32, BF16 = torch.float32, torch.bfloat16
SIZES = [(1, 1, 32), (1, 50261, 64), (2, 300, 96), (16, 1000, 160), (17, 257, 64), (33, 129, 32), (64, 4099, 128),
         (65, 255, 224), (129, 256, 64), (257, 1023, 96), (300, 513, 40), (5, 70, 7), (700, 2000, 64)]


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("n,V,D", SIZES)
def test_values_and_gradients(gpu_lib, n, V, D, dtype, wdtype):
    from qllm2_amd.token_logprobs import linear_token_logprobs
    print(f"case n={n} V={V} D={D} {dtype} {wdtype}", flush=True)
    h, w, ids, gs = _data(n, V, D, dtype, wdtype, n + V + D)
    T = 0.7 if n % 2 else 1.0
    bf = BF16 in (dtype, wdtype)
    hr, wr = (h.to(BF16), w.to(BF16)) if bf else (h, w)
    R = _reference(hr, wr, ids, T, [g.double() for g in gs], 2.0 ** -8 if bf else 0.0)
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda(), temperature=T)
    _close(r.logprobs, R["lp"], R["t_lp"])
    _close(r.entropy, R["H"], R["t_H"])
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hc, wc], [g.cuda() for g in gs])
    assert dh.dtype == dtype and dw.dtype == wdtype
    # a bf16 product leaves as bf16 where the operand's own type is wider, too; a master table's does not
    _close(dh, R["dh"], R["t_dh"], torch.finfo(BF16 if bf else F32).eps)
    _close(dw, R["dw"], R["t_dw"], torch.finfo(wdtype).eps)
    for got, k in ((dh, "dh"), (dw, "dw")):
        if R[k].norm() > 0:
            rel = ((got.cpu().double() - R[k]).norm() / R[k].norm()).item()
            assert rel < (2.0 ** -7 if bf else 1e-4), (k, rel)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rounds_of_the_backward_and_no_gradient(gpu_lib, dtype):
    """A chunk smaller than the rows (several passes add into dW), one output's gradient
    alone, rows of zeros' gradient, and the forward alone."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(1100, 700, 96, dtype, dtype, 3)
    eps, r8 = torch.finfo(dtype).eps, 2.0 ** -8 if dtype == BF16 else 0.0
    zero = torch.zeros(1100, dtype=torch.float64)
    for which in (0, 1):
        g64 = [zero, zero]
        g64[which] = gs[which].double()
        R = _reference(h, w, ids, 1.0, g64, r8)
        hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
        r = linear_token_logprobs(hc, wc, ids.cuda(), chunk=64)
        dh, dw = torch.autograd.grad([r[which]], [hc, wc], [gs[which].cuda()])
        _close(dh, R["dh"], R["t_dh"], eps)
        _close(dw, R["dw"], R["t_dw"], eps)
        if which == 0:
            assert (dh[::5] == 0).all()     # rows without a token
    plain = linear_token_logprobs(h.cuda(), w.cuda(), ids.cuda())
    assert not plain.logprobs.requires_grad and torch.equal(plain.logprobs, r.logprobs)
    z = linear_token_logprobs(hc[:0], wc, ids[:0].cuda())
    dh, dw = torch.autograd.grad([z.logprobs, z.entropy], [hc, wc], [torch.zeros(0, device="cuda")] * 2)
    assert z.logprobs.shape == (0,) and (dw == 0).all() and (dh == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts_and_shapes(gpu_lib, dtype):
    """[B, T, D] rows, strided rows and tables, int32 ids."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, _ = _data(60, 500, 64, dtype, dtype, 4)
    R = _reference(h, w, ids, 1.0, None, 0.0)
    wide_h, wide_w = torch.full((60, 80), float("nan"), dtype=dtype).cuda(), torch.full((500, 75), float("nan"), dtype=dtype).cuda()
    wide_h[:, 8:72], wide_w[:, 3:67] = h.cuda(), w.cuda()
    for hc, wc in ((wide_h[:, 8:72], wide_w[:, 3:67]), (h.T.contiguous().cuda().T, w.cuda())):
        r = linear_token_logprobs(hc.unflatten(0, (6, 10)), wc, ids.view(6, 10).to(torch.int32).cuda())
        assert r.logprobs.shape == (6, 10)
        _close(r.logprobs.view(-1), R["lp"], R["t_lp"])
        _close(r.entropy.view(-1), R["H"], R["t_H"])
    one = linear_token_logprobs(h[7].cuda(), w.cuda(), ids[7].cuda())
    assert one.logprobs.shape == ()


def test_same_values_as_from_logits(gpu_lib):
    """Both entry points give the same numbers where the logits are exact."""
    from qllm2_amd.token_logprobs import linear_token_logprobs, token_logprobs
    g = torch.Generator().manual_seed(5)
    h, w = torch.randint(-2, 3, (90, 64), generator=g).float(), torch.randint(-1, 2, (1001, 64), generator=g).float()
    ids = torch.randint(0, 1001, (90,), generator=g).cuda()
    want = token_logprobs((h @ w.T).cuda(), ids, temperature=2.0)
    for dtype in (F32, BF16):
        got = linear_token_logprobs(h.to(dtype).cuda(), w.to(dtype).cuda(), ids, temperature=2.0)
        R = _reference(h, w, ids.cpu(), 2.0, None, 0.0)
        for a, b, t in ((got.logprobs, want.logprobs, R["t_lp"]), (got.entropy, want.entropy, R["t_H"])):
            _close(a, b.cpu().double(), 2 * t)


def test_extreme_rows_stay_their_own(gpu_lib):
    """Rows far apart in scale: a zero row is uniform, a huge one has one token, a NaN
    row stays NaN alone."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    for dtype in (F32, BF16):
        h, w, ids, gs = _data(300, 600, 64, dtype, dtype, 6)
        ids = ids.clamp(0, 599)
        h[0], h[1], h[299] = 0, h[1] * 1000, float("nan")
        hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
        r = linear_token_logprobs(hc, wc, ids.cuda())
        R = _reference(h[:299], w, ids[:299], 1.0, None, 0.0)
        _close(r.logprobs[:299], R["lp"], R["t_lp"])
        _close(r.entropy[:299], R["H"], R["t_H"])
        assert r.logprobs[299].isnan() and r.entropy[299].isnan()
        g = [t.cuda() for t in gs]
        dh, = torch.autograd.grad([r.logprobs, r.entropy], [hc], g)
        assert dh[299].isnan().all() and not dh[:299].isnan().any()


def test_captured_training_step_replays(gpu_lib):
    from qllm2_amd.token_logprobs import linear_token_logprobs
    for dtype in (F32, BF16):
        h, w, ids, gs = _data(200, 900, 64, dtype, dtype, 7)
        hc, wc, ic, gc = h.cuda().requires_grad_(), w.cuda().requires_grad_(), ids.cuda(), [g.cuda() for g in gs]

        def step():
            r = linear_token_logprobs(hc, wc, ic, temperature=0.9)
            return [r.logprobs.detach(), r.entropy.detach(), *torch.autograd.grad([r.logprobs, r.entropy], [hc, wc], gc)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for seed in range(4):
            nh, nw, nids, ngs = _data(200, 900, 64, dtype, dtype, 80 + seed)
            with torch.no_grad():
                hc.copy_(nh), wc.copy_(nw), ic.copy_(nids)
                for a, b in zip(gc, ngs):
                    a.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step()):
                assert torch.equal(a, b)


def test_full_vocabulary_batch(gpu_lib):
    """16384 rows against 50261 x 512 in bf16 (a G of 823 million entries), float64 on the
    GPU beside it; norms: a value is off by 2^-20 or so, dh and dw by the roundings of dx
    and of themselves (2^-8 each)."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    g = torch.Generator("cuda").manual_seed(2)
    n, V, D = 16384, 50261, 512
    h = torch.randn(n, D, device="cuda", generator=g).bfloat16().requires_grad_()
    w = (torch.randn(V, D, device="cuda", generator=g) * 2.5 / D ** 0.5).bfloat16().requires_grad_()
    ids = torch.randint(0, V, (n,), device="cuda", generator=g)
    ids[::9] = -100
    gs = [torch.randn(n, device="cuda", generator=g) / n, torch.randn(n, device="cuda", generator=g) / n]
    r = linear_token_logprobs(h, w, ids)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [h, w], gs)
    hd, wd = h.detach().double(), w.detach().double()
    logp = torch.log_softmax(hd @ wd.T, -1)
    p = logp.exp()
    ent = -(p * logp).sum(-1)
    valid = ids >= 0
    lp = torch.where(valid, logp.gather(1, ids.clamp(min=0)[:, None])[:, 0], 0.0)
    g_lp = torch.where(valid, gs[0].double(), 0.0)
    dx = -p * (g_lp[:, None] + gs[1].double()[:, None] * (logp + ent[:, None]))
    dx.scatter_add_(1, ids.clamp(min=0)[:, None], g_lp[:, None])
    for got, want, tol in ((r.logprobs, lp, 2.0 ** -20), (r.entropy, ent, 2.0 ** -20), (dh, dx @ wd, 2.0 ** -7),
                           (dw, dx.T @ hd, 2.0 ** -7)):
        assert ((got.double() - want).norm() / want.norm()).item() < tol


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_operand_frozen(gpu_lib, dtype):
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(150, 300, 64, dtype, dtype, 8)
    both = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    r = linear_token_logprobs(*both, ids.cuda())
    want = torch.autograd.grad([r.logprobs, r.entropy], both, [g.cuda() for g in gs])
    for i in (0, 1):
        ops = [h.cuda(), w.cuda()]
        ops[i].requires_grad_()
        r = linear_token_logprobs(*ops, ids.cuda())
        got, = torch.autograd.grad([r.logprobs, r.entropy], [ops[i]], [g.cuda() for g in gs])
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("n,V,D,chunk", [(900, 500, 96, 70), (300, 700, 64, 4096), (5, 40, 32, 1)])
def test_one_operand_frozen_over_several_passes(gpu_lib, n, V, D, chunk, dtype, wdtype):
    """The product of an operand without a gradient is left out; the other's stays the same bits."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(n, V, D, dtype, wdtype, 9)
    both = [h.cuda().requires_grad_(), w.cuda().requires_grad_()]
    r = linear_token_logprobs(*both, ids.cuda(), temperature=0.8, chunk=chunk)
    want = torch.autograd.grad([r.logprobs, r.entropy], both, [g.cuda() for g in gs])
    for i in (0, 1):
        ops = [h.cuda(), w.cuda()]
        ops[i].requires_grad_()
        r = linear_token_logprobs(*ops, ids.cuda(), temperature=0.8, chunk=chunk)
        got, = torch.autograd.grad([r.logprobs, r.entropy], [ops[i]], [g.cuda() for g in gs])
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("n,V,D", [(2047, 50261, 32), (4096, 50261, 96), (4100, 50261, 64), (300, 5000, 96), (300, 10000, 32)])
def test_tiles_that_do_not_fill_their_last_round(gpu_lib, n, V, D):
    """bf16 rows against vocabularies whose tiles leave a part of a round over, beside float64 on the GPU."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, _ = (x if isinstance(x, list) else x.cuda() for x in _data(n, V, D, BF16, BF16, 11))
    r = linear_token_logprobs(h, w, ids, temperature=0.9)
    want = _reference(h, w, ids, 0.9, None, 0.0)
    _close(r.logprobs, want["lp"].cpu(), want["t_lp"].cpu())
    _close(r.entropy, want["H"].cpu(), want["t_H"].cpu())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D,chunk", [(1300, 300, 64, 300), (520, 150, 160, 4096), (66, 1500, 256, 4096), (200, 900, 64, 33)])
def test_gradients_of_small_tables_and_several_passes(gpu_lib, n, V, D, chunk, dtype):
    """Products with few tiles and long sums: shared K ranges, their partial sums added over the passes."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(n, V, D, dtype, dtype, n)
    R = _reference(h, w, ids, 1.3, [g.double() for g in gs], 2.0 ** -8 if dtype == BF16 else 0.0)
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda(), temperature=1.3, chunk=chunk)
    _close(r.logprobs, R["lp"], R["t_lp"])
    _close(r.entropy, R["H"], R["t_H"])
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hc, wc], [g.cuda() for g in gs])
    _close(dh, R["dh"], R["t_dh"], torch.finfo(dtype).eps)
    _close(dw, R["dw"], R["t_dw"], torch.finfo(dtype).eps)


@pytest.mark.parametrize("n,V,D", [(2047, 50261, 32), (4096, 50261, 64), (300, 10000, 96), (129, 700, 64)])
def test_gradients_of_tiles_that_do_not_fill_their_last_round(gpu_lib, n, V, D):
    """The gradient's tiles of the same kind, bf16, every row and column: dx rounded to bf16 (2^-8 each)
    between the products, dh and dw rounded once more."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = (x if isinstance(x, list) else x.cuda() for x in _data(n, V, D, BF16, BF16, 12))
    gs = [g.cuda() for g in gs]
    h.requires_grad_(), w.requires_grad_()
    r = linear_token_logprobs(h, w, ids)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [h, w], gs)
    R = _reference(h.detach(), w.detach(), ids, 1.0, [g.double() for g in gs], 2.0 ** -8)
    for got, k in ((dh, "dh"), (dw, "dw")):
        _close(got, R[k].cpu(), R["t_" + k].cpu(), torch.finfo(BF16).eps)


@pytest.mark.parametrize("n,V,D,chunk", [(300, 700, 64, 4096), (900, 500, 96, 70), (2, 300, 32, 1)])
def test_hand_written_products(gpu_lib, monkeypatch, n, V, D, chunk):
    """QPAM_CE_GEMM=hip changes the passes and their workspace; a frozen operand's product is left out."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    monkeypatch.setenv("QPAM_CE_GEMM", "hip")
    h, w, ids, gs = _data(n, V, D, BF16, BF16, 13)
    R = _reference(h, w, ids, 1.0, [g.double() for g in gs], 2.0 ** -8)
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    for ops in ([hc, wc], [hc, wc.detach()], [hc.detach(), wc]):
        r = linear_token_logprobs(*ops, ids.cuda(), chunk=chunk)
        live = [o for o in ops if o.requires_grad]
        got = torch.autograd.grad([r.logprobs, r.entropy], live, [g.cuda() for g in gs])
        for o, g in zip(live, got):
            k = "dh" if o is hc else "dw"
            _close(g, R[k], R["t_" + k], torch.finfo(BF16).eps)
