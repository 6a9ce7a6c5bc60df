"""Token scores where rounding decides (qpam_linear_logprobs_fwd / _bwd): rows that are certain or
all but certain of their token, low temperatures; the kernel of few rows at its own widths; the
layouts that rows and tables arrive in.  Tolerances beside each test, u = 2^-24."""

import pytest
import torch

from test_gpu_linear_logprobs import BF16, F32, U, _close, _data, _reference

pytestmark = pytest.mark.gpu


def _toward(w, first, second, a, b):
    """Rows h with h . w[first] = a and h . w[second] = b, of least norm."""
    f, s = w[first].double(), w[second].double()
    ff, fs, ss = (f * f).sum(-1), (f * s).sum(-1), (s * s).sum(-1)
    det = ff * ss - fs * fs
    return ((a * ss - b * fs) / det)[:, None] * f + ((b * ff - a * fs) / det)[:, None] * s


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(1, 700, 1536), (16, 1000, 512), (40, 33000, 512), (64, 300, 640), (65, 1000, 512),
                                   (300, 1023, 512), (600, 9000, 256)])
def test_certain_rows(gpu_lib, n, V, D, dtype):
    """The token leads by 60 or more: 1 - p, the entropy and the row of dx are 0 to within V e^-60
    (10^-22).  The token's logit is the row's maximum, so its own term is 2^0 and the sum is 1:
    what is left is a rounding or two of numbers near 1, 4 u, and of one below 0 nothing."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    g = torch.Generator().manual_seed(n + V)
    w = (torch.randn(V, D, generator=g) * 2.5 / D ** 0.5).to(dtype)
    ids = torch.randint(0, V, (n,), generator=g)
    h = (300 * w[ids].double() / (w[ids].double() ** 2).sum(-1, keepdim=True)).to(dtype)
    x = h.double() @ w.double().T
    lead = x.gather(1, ids[:, None])[:, 0] - x.scatter(1, ids[:, None], float("-inf")).max(-1).values
    assert lead.min() >= 60
    gs = [torch.randn(n, generator=g), torch.randn(n, generator=g)]
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda())
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hc, wc], [t.cuda() for t in gs])
    assert (r.logprobs <= 0).all() and (r.logprobs >= -4 * U).all(), r.logprobs.abs().max()
    assert (r.entropy >= 0).all() and (r.entropy <= 4 * U).all(), r.entropy.abs().max()
    dx = (8 * U * (gs[0].abs() + gs[1].abs())).double()
    _close(dh, torch.zeros(n, D).double(), dx[:, None] * w[ids].double().abs() + 1e-20)
    _close(dw, torch.zeros(V, D).double(),
           torch.zeros(V, D).double().index_add_(0, ids, dx[:, None] * h.double().abs()) + 1e-18)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(1, 300, 512), (24, 700, 768), (64, 40000, 512), (65, 1000, 512), (300, 1023, 512)])
def test_nearly_certain_rows(gpu_lib, n, V, D, dtype):
    """One other token eight below the row's own: 1 - p = e^-8 (3e-4).  A logit is off by the roundings
    of its fp32 sum, at most E = (D + 4) u sum |h w| and in earnest about sqrt(D) of the D, so d ln p
    = (1 - p) times that of the lead: relative to dx 2 E sqrt(D) / D at three times its deviation (6 E /
    sqrt(D)), 4 u / (1 - p) for 1 - e^lp, and dx's rounding to bf16 (2^-8), as of the outputs."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    g = torch.Generator().manual_seed(n + V)
    w = (torch.randn(V, D, generator=g) * 2.5 / D ** 0.5).to(dtype)
    ids = torch.randperm(V, generator=g)[:n]
    other = (ids + 1 + torch.randint(0, V - 1, (n,), generator=g)) % V
    h = _toward(w, ids, other, 100.0, 92.0).to(dtype)
    hd, wd = h.double(), w.double()
    logp = torch.log_softmax(hd @ wd.T, -1)
    p, g_lp = logp.exp(), torch.rand(n, generator=g) + 0.5
    lp = logp.gather(1, ids[:, None])
    assert ((lp > -0.01) & (lp < -1e-5)).all()
    dx = -p * g_lp.double()[:, None]
    dx.scatter_(1, ids[:, None], -torch.expm1(lp) * g_lp.double()[:, None])
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda())
    dh, = torch.autograd.grad(r.logprobs, hc, g_lp.cuda())
    assert (r.logprobs < 0).all() and (r.entropy > 0).all()
    E = (D + 4) * U * (hd.abs() * wd[ids].abs()).sum(-1)
    rel = 6 * E / D ** 0.5 + 4 * U / 1e-5 + (2.0 ** -7 if dtype == BF16 else 0.0)
    want = dx @ wd
    err = (dh.cpu().double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert (err <= rel).all(), (err / rel).max()


def _whole(n, V, D, dtype, T):
    """Operands whose logits are whole numbers, exact in every sum, with what they give at a low temperature T:
    each row's k largest entries have p = 1 / k, the others 0 (e^-1000 and less).  The sum counts k exactly
    up to L = V / 16 + 60 roundings, so ln k is off by 2 u (L + ln k + 1)."""
    g = torch.Generator().manual_seed(n)
    h, w = torch.randint(-2, 3, (n, D), generator=g).to(dtype), torch.randint(-1, 2, (V, D), generator=g).to(dtype)
    ids = torch.randint(0, V, (n,), generator=g)
    x = h.double() @ w.double().T
    ids[::3] = x.argmax(-1)[::3]
    ids[4::5] = -100
    d = x.max(-1, keepdim=True).values - x
    p = (d == 0).double()
    ln_k = p.sum(-1).log()
    t_ln = 2 * U * (V / 16 + 60 + ln_k + 1)
    lp = torch.where(ids >= 0, -d.gather(1, ids.clamp(min=0)[:, None])[:, 0] / T - ln_k, 0.0)
    return h, w, ids, p / p.sum(-1, keepdim=True), lp, ln_k, t_ln


@pytest.mark.parametrize("T", [1e-3, 1e-9, 1e-12, 1e-25])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 300, 2000])
def test_low_temperatures(gpu_lib, n, dtype, T):
    """A log probability -d / T is the product of three rounded factors: 8 u of it with the last sum."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, _, lp, ln_k, t_ln = _whole(n, 4200, 64, dtype, T)
    r = linear_token_logprobs(h.cuda(), w.cuda(), ids.cuda(), temperature=T)
    _close(r.logprobs, lp, 8 * U * lp.abs() + t_ln)
    _close(r.entropy, ln_k, 2 * t_ln)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [20, 300])
def test_low_temperature_of_rounded_logits(gpu_lib, n, dtype):
    """At T = 1e-9 a logit's last bits are hundreds of units of u, so which entry leads is a matter of the
    sums' order; each row's values stay a distribution's: lp <= 0, entropy of [0, ln V]."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, _ = _data(n, 700, 96, dtype, dtype, 21)
    r = linear_token_logprobs(h.cuda(), w.cuda(), ids.cuda(), temperature=1e-9)
    assert (r.logprobs <= 0).all() and r.logprobs.isfinite().all()
    assert (r.entropy >= 0).all() and (r.entropy <= 6.5511).all()    # ln 700


@pytest.mark.parametrize("T", [1e-3, 1e-9, 1e-12, 1e-25])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V", [(5, 600), (300, 600), (1200, 4200)])
def test_gradients_at_low_temperatures(gpu_lib, n, V, dtype, T):
    """dx = ([v = token] - p) g_lp / T: the entropy's term is p (ln p + entropy) = 0 at the largest entries, off by
    the errors of both logarithms, and 0 at the others however large their u."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, p, _, _, t_ln = _whole(n, V, 64, dtype, T)
    g = torch.Generator().manual_seed(1)
    gs = [torch.randn(n, generator=g) / n, torch.randn(n, generator=g) / n]
    g_lp, g_ent = torch.where(ids >= 0, gs[0].double(), 0.0), gs[1].double()
    one = torch.zeros_like(p).scatter_add_(1, ids.clamp(min=0)[:, None], g_lp[:, None])
    dx = (one - p * g_lp[:, None]) / T
    tol = p / T * (g_lp.abs() * (2 * t_ln + 8 * U) + g_ent.abs() * (4 * t_ln + 8 * U))[:, None] + 16 * U * one.abs() / T
    tol += (2.0 ** -8 if dtype == BF16 else 4 * U) * (dx.abs() + tol)
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda(), temperature=T)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hc, wc], [t.cuda() for t in gs])
    hd, wd = h.double(), w.double()
    _close(dh, dx @ wd, tol @ wd.abs() + V * U * (dx.abs() @ wd.abs()), torch.finfo(dtype).eps)
    _close(dw, dx.T @ hd, tol.T @ hd.abs() + n * U * (dx.abs().T @ hd.abs()), torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [20, 300])
def test_gradients_at_a_low_temperature_of_rounded_logits(gpu_lib, n, dtype):
    """Where the forward's product and the backward's own differ in a logit's last bits (few fp32 rows), p =
    2^u / s is of [0, 1] all the same: |dx| sums to at most 2 |g_lp| + 2 |g_ent| (1 + ln V) over a row, times
    1 / T, and 4 for more than one entry at u = 0."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(n, 700, 96, dtype, dtype, 21)
    hc, T = h.cuda().requires_grad_(), 1e-9
    r = linear_token_logprobs(hc, w.cuda(), ids.cuda(), temperature=T)
    dh, = torch.autograd.grad([r.logprobs, r.entropy], [hc], [t.cuda() for t in gs])
    bound = 8 * (gs[0].abs() + gs[1].abs() * 7.56) / T * w.float().abs().max()
    assert (dh.float().abs().cpu() <= bound[:, None]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,V,D", [(16, 1000, 1536), (9, 33000, 640), (20, 1000, 896), (30, 33000, 672), (33, 1000, 640),
                                   (64, 33000, 1568), (1, 33000, 896), (64, 300, 1184)])
def test_few_rows_of_real_widths(gpu_lib, n, V, D, dtype):
    """Up to 64 rows over 5 to 25 stages of 256 bytes a row: every body of the unrolled loop and its return
    to the first, with 16, 32 and 64 rows in blocks of 4 and of 16 waves.  Tolerances as for all sizes."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, _ = _data(n, V, D, dtype, dtype, n + D)
    r = linear_token_logprobs(h.cuda(), w.cuda(), ids.cuda(), temperature=0.8)
    R = _reference(h, w, ids, 0.8, None, 0.0)
    _close(r.logprobs, R["lp"], R["t_lp"])
    _close(r.entropy, R["H"], R["t_H"])


def _off_16(t):
    """t in contiguous storage that starts one element off 16 bytes, as a slice of a flat parameter buffer does."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:].copy_(t.reshape(-1))
    return flat[1:].view(t.shape)


def _far_apart(t):
    """t's rows 2^22 elements apart, as one position's rows of a long batch are."""
    return torch.zeros(t.shape[0], 2 ** 22 // t.shape[1], t.shape[1], dtype=t.dtype, device=t.device).index_copy_(
        1, torch.tensor([3], device=t.device), t[:, None])[:, 3]


LAYOUTS = {
    "one row for all": (lambda h: h[:1].expand(h.shape[0], -1), lambda w: w[:1].expand(w.shape[0], -1)),
    "a column as one row": (lambda h: h[:1].T.contiguous().T, lambda w: w),
    "storage off 16 bytes": (_off_16, _off_16),
    "rows 2^22 apart": (_far_apart, _far_apart),
}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", list(LAYOUTS))
def test_layouts_of_rows_and_table(gpu_lib, name, dtype):
    """Every layout gives the bits of the same values laid out row after row, with both gradients."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(7, 20, 64, dtype, dtype, 31)
    f, k = LAYOUTS[name]
    for a, b in ((f(h.cuda()), w.cuda()), (h.cuda(), k(w.cuda()))):
        res = []
        for x, y in ((a, b), (a.clone(memory_format=torch.contiguous_format), b.clone(memory_format=torch.contiguous_format))):
            x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
            n = x.shape[0]
            r = linear_token_logprobs(x, y, ids[:n].cuda())
            res.append([r.logprobs, r.entropy, *torch.autograd.grad([r.logprobs, r.entropy], [x, y], [t[:n].cuda() for t in gs])])
        for s, t in zip(*res):
            assert torch.equal(s, t)


@pytest.mark.parametrize("name", ["one row for all", "a column as one row", "storage off 16 bytes"])
def test_layouts_of_the_loss(gpu_lib, name):
    """fused_linear_cross_entropy takes its operands the same way."""
    from qllm2_amd.fused_ce import fused_linear_cross_entropy, linear_ce_per_token
    for dtype in (F32, BF16):
        h, w, ids, _ = _data(7, 20, 64, dtype, dtype, 32)
        ids = ids.clamp(max=19)
        f, k = LAYOUTS[name]
        for a, b in ((f(h.cuda()), w.cuda()), (h.cuda(), k(w.cuda()))):
            res = []
            for x, y in ((a, b), (a.clone(memory_format=torch.contiguous_format), b.clone(memory_format=torch.contiguous_format))):
                x, y = x.detach().requires_grad_(), y.detach().requires_grad_()
                t = ids[:x.shape[0]].cuda()
                loss = fused_linear_cross_entropy(x, y, t)
                res.append([loss, linear_ce_per_token(x, y, t), *torch.autograd.grad(loss, [x, y])])
            for s, t in zip(*res):
                assert torch.equal(s, t)


@pytest.mark.parametrize("wdtype", [BF16, F32])
@pytest.mark.parametrize("n,V,D,chunk,same", [(300, 700, 64, 4096, False), (1, 300, 96, 4096, False), (40, 5000, 96, 4096, False),
                                              (1100, 700, 96, 64, False), (2500, 9000, 64, 4096, False), (700, 600, 32, 4096, True),
                                              (20000, 1000, 32, 8192, False)])
def test_token_terms_are_not_rounded_between_the_products(gpu_lib, n, V, D, chunk, same, wdtype):
    """bf16 rows: dx is rounded to bf16 (2^-8 of each entry) in front of the products but for the entries at the
    rows' tokens, which join them in fp32.  All else as for fp32; an fp32 table's dw shows it undimmed."""
    from qllm2_amd.token_logprobs import linear_token_logprobs
    h, w, ids, gs = _data(n, V, D, BF16, wdtype, n + V)
    if same:
        ids = torch.where(ids == V + 1, ids, V // 2)
    wr = w.to(BF16)
    R = _reference(h, wr, ids, 0.9, [g.double() for g in gs], 0.0)
    hd, wd = h.double(), wr.double()
    logp = torch.log_softmax(hd @ wd.T / 0.9, -1)
    p = logp.exp()
    valid = (ids >= 0) & (ids < V)
    dx = p * (torch.where(valid, gs[0].double(), 0.0)[:, None] + gs[1].double()[:, None] * (logp - (p * logp).sum(-1, keepdim=True))) / 0.9
    dx[valid, ids[valid]] = 0
    hc, wc = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    r = linear_token_logprobs(hc, wc, ids.cuda(), temperature=0.9, chunk=chunk)
    for needs in ((hc, wc), (hc,), (wc,)):
        for o, got in zip(needs, torch.autograd.grad([r.logprobs, r.entropy], needs, [g.cuda() for g in gs], retain_graph=True)):
            if o is hc:
                _close(got, R["dh"], R["t_dh"] + 2.0 ** -8 * (dx.abs() @ wd.abs()), torch.finfo(BF16).eps)
            else:
                _close(got, R["dw"], R["t_dw"] + 2.0 ** -8 * (dx.abs().T @ hd.abs()), torch.finfo(wdtype).eps)
