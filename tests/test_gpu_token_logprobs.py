"""Log probabilities, entropy and top alternatives of rows of logits, and their
gradient (qpam_logprobs_fwd / qpam_logprobs_bwd), against plain torch in float64.

Tolerances, with u = 2^-24, d_v = (max - x_v) / T, p the probabilities, A = sum p d,
B = sum p d^2.  An exponent is off by 4 u d (the subtraction, 1 / T, log2 e and the
product), an exponential by 4 u d + 2 u; a thread adds up to V / 256 terms and may
rescale as often as it has batches, the block joins the threads in some 20 steps:
  ln s:     u (V / 128 + 40 + 4 A) + 3 u |ln s|
  log prob: that of ln s + 3 u |x_t - max| / T + u |log prob|
  entropy:  that of ln s + u (2 (V / 128 + 40) A + 4 B + 4 A + |H|)
  gradient: per entry p / T times (relative error of p times |bracket| + the error of
            the bracket) + 4 u |g| + eps / 2 |g| for the result's type."""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


def _reference(x, ids, T, ignore=-100):
    """float64 outputs and tolerances of rows x (any float dtype, on the CPU)."""
    x = x.double()
    n, V = x.shape
    m = x.max(-1, keepdim=True).values
    empty = m[:, 0] == -INF
    d = torch.where(x == -INF, INF, (torch.where(empty[:, None], 0.0, m) - x) / T)
    e = torch.exp(-d)
    s = e.sum(-1)
    ln_s = s.log()
    p = torch.where(empty[:, None], 0.0, e / s[:, None])
    dz = torch.where(p > 0, d, 0.0)
    A, B = (p * dz).sum(-1), (p * dz * dz).sum(-1)
    H = torch.where(empty, 0.0, ln_s + A)
    logp = torch.where(empty[:, None], -INF, -d - ln_s[:, None])
    valid = (ids != ignore) & (ids >= 0) & (ids < V)
    safe = torch.where(valid, ids, 0)
    lp = torch.where(valid, logp.gather(1, safe[:, None])[:, 0], 0.0)
    steps = V / 128 + 40
    t_ln = U * (steps + 4 * A) + 3 * U * ln_s.abs()
    t_lp = torch.where(torch.isinf(logp), 0.0, t_ln[:, None] + 3 * U * torch.where(torch.isinf(d), 0.0, d) + U * logp.abs())
    t_H = t_ln + U * (2 * steps * A + 4 * B + 4 * A + H.abs())
    return dict(x=x, d=d, p=p, logp=logp, lp=lp, H=H, ln_s=ln_s, empty=empty, valid=valid, safe=safe, t_ln=t_ln, t_lp=t_lp,
                t_H=t_H, A=A, steps=steps)


def _close(got, want, tol):
    got = got.detach().cpu().double()
    # finfo.min / 0.7 = -4.9e38 lies past fp32's largest value, so its fp32 value is -inf
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want * INF, want)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bad.any(), (got[bad][:4], want[bad][:4], (got - want).abs()[bad].max())


def _order(x):
    """Ids by value, equal values by the lower id, NaN first."""
    return torch.sort(x.double() + 0.0, dim=-1, descending=True, stable=True).indices


def _check(x, ids, k, T, r):
    R = _reference(x, ids, T)
    tol_t = R["t_lp"].gather(1, R["safe"][:, None])[:, 0]
    _close(r.logprobs, R["lp"], tol_t)
    _close(r.entropy, R["H"], R["t_H"])
    if k:
        order = _order(x)[:, :k]
        assert torch.equal(r.top_ids.cpu(), order)
        _close(r.top_logprobs, R["logp"].gather(1, order), R["t_lp"].gather(1, order))
    return R


def _rows(kind, n, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, V, generator=g) * 2.5
    i = torch.arange(V)
    if kind == "peaked":
        x[torch.arange(n), torch.randint(0, V, (n,), generator=g)] += 30
    elif kind == "constant":
        x[:] = 0.75
    elif kind == "ascending":
        x = (i * 0.01).expand(n, V).clone()
    elif kind == "descending":
        x = (-i * 0.01).expand(n, V).clone()
    elif kind == "ties":
        x = x.round()
    elif kind == "zeros":           # +0 and -0 are equal
        x = torch.where(torch.rand(n, V, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "half":
        x[:, torch.rand(V, generator=g) < 0.5] = -INF
    elif kind == "few":             # row r keeps r tokens, row 0 none
        for r in range(n):
            keep = torch.randperm(V, generator=g)[:min(r, V)]
            y = torch.full((V,), -INF)
            y[keep] = x[r, keep]
            x[r] = y
    elif kind == "block":           # a handful of adjacent tokens
        x[:, 5:] = -INF
        x[:, :max(0, min(3, V - 1))] = -INF
    elif kind == "lowest":
        x[:, torch.rand(V, generator=g) < 0.7] = torch.finfo(dtype).min
    elif kind == "all_lowest":
        x[:] = torch.finfo(dtype).min
    elif kind == "groups":          # all the large entries in a few of the 64 lanes' groups
        e = 16 // dtype.itemsize
        x = torch.where(((i // e) % 64 < 4), 20 + x, x - 20)
    elif kind == "wide":
        x = x * 1e4
    else:
        assert kind == "normal"
    return x.to(dtype), torch.randint(0, V, (n,), generator=g)


KINDS = ["normal", "peaked", "constant", "ascending", "descending", "ties", "zeros", "half", "few", "block", "lowest",
         "all_lowest", "groups", "wide"]
SIZES = [(1, 1, 1), (3, 2, 2), (5, 3, 1), (4, 7, 7), (30, 64, 64), (3, 65, 20), (70, 255, 0), (9, 1000, 32), (6, 4097, 5),
         (3, 16384, 64), (2, 50261, 20), (600, 16385, 3), (1, 160001, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", KINDS)
def test_values_and_alternatives(gpu_lib, kind, dtype):
    from qllm2_amd.token_logprobs import token_logprobs
    for n, V, k in SIZES:
        print(f"case {kind} n={n} V={V} k={k} {dtype}", flush=True)
        x, ids = _rows(kind, n, V, dtype, n + V)
        T = 1.0 if V % 2 else 0.7
        ids[::5] = -100
        ids[3::7] = V + 3
        r = token_logprobs(x.cuda(), ids.cuda(), temperature=T, top_k=k)
        assert (r.top_ids is None) == (k == 0) and r.logprobs.dtype == torch.float32
        _check(x, ids, k, T, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,n", [(3, 4), (100, 5), (16400, 3), (16400, 600)])
def test_rows_of_any_alignment(gpu_lib, V, n, dtype):
    """Rows that start anywhere, with strides that shift the start from row to row;
    what lies beside the rows is NaN and must not be read into them."""
    from qllm2_amd.token_logprobs import token_logprobs
    x, ids = _rows("normal", n, V, dtype, 3)
    for off in range(9):
        for extra in (off, 8, 3):
            buf = torch.full((n, V + extra + 9), float("nan"), dtype=dtype)
            buf[:, off:off + V] = x
            r = token_logprobs(buf.cuda()[:, off:off + V], ids.cuda(), top_k=3)
            _check(x, ids, 3, 1.0, r)
        if n == 600:
            break


def test_shapes_int32_and_other_layouts(gpu_lib):
    from qllm2_amd.token_logprobs import token_logprobs
    x, ids = _rows("normal", 12, 90, torch.float32, 4)
    want = token_logprobs(x.cuda(), ids.cuda(), top_k=4)
    r = token_logprobs(x.view(3, 4, 90).cuda(), ids.view(3, 4).to(torch.int32).cuda(), top_k=4)
    assert r.logprobs.shape == (3, 4) and r.top_ids.shape == (3, 4, 4)
    for a, b in zip(r, want):
        assert torch.equal(a.reshape(b.shape), b)
    one = token_logprobs(x[0].cuda(), ids[0].cuda(), top_k=4)
    assert one.entropy.shape == () and torch.equal(one.top_ids, want.top_ids[0])
    t = token_logprobs(x.T.contiguous().cuda().T, ids.cuda(), top_k=4)
    e = token_logprobs(x[:1].cuda().expand(12, 90), ids[:1].cuda().expand(12), top_k=4)
    for a, b in zip(t, want):
        assert torch.equal(a, b)
    assert torch.equal(e.entropy, want.entropy[:1].expand(12))
    z = token_logprobs(x[:0].cuda(), ids[:0].cuda(), top_k=4)
    assert z.logprobs.shape == (0,) and z.top_ids.shape == (0, 4)


def test_nan_and_infinity(gpu_lib):
    """A row with NaN or +inf gives NaN, its ids by the order (NaN first); the rows
    beside it are as they were."""
    from qllm2_amd.token_logprobs import token_logprobs
    for dtype in (torch.float32, torch.bfloat16):
        for V in (40, 20000):
            x, ids = _rows("normal", 6, V, dtype, 5)
            x[1, 7], x[1, 30], x[2, 9], x[3] = float("nan"), float("nan"), INF, float("nan")
            x[4, :20] = -INF
            r = token_logprobs(x.cuda(), ids.cuda(), top_k=5)
            assert torch.equal(r.top_ids.cpu(), _order(x)[:, :5])
            keep = [0, 4, 5]
            for row in (1, 2, 3):
                assert r.logprobs[row].isnan() and r.entropy[row].isnan() and r.top_logprobs[row, 0].isnan()
            _check(x[keep], ids[keep], 5, 1.0, type(r)(*(t[keep] for t in r)))


def _grad_check(x, ids, k, T, g, got, top_ids):
    """g: (g_logprobs, g_entropy, g_top or None), float64 on the CPU."""
    R = _reference(x, ids, T)
    g_lp, g_ent, g_top = g
    g_lp = torch.where(R["valid"], g_lp, 0.0)
    all_g, mass = g_lp.clone(), g_lp.abs()
    extra = torch.zeros_like(R["x"]).scatter_add_(1, R["safe"][:, None], g_lp[:, None])
    size = extra.abs()
    if g_top is not None:
        all_g = all_g + g_top.sum(-1)
        mass = mass + g_top.abs().sum(-1)
        extra = extra.scatter_add_(1, top_ids, g_top)
        size = size.scatter_add_(1, top_ids, g_top.abs())
    p = R["p"]
    lnp = torch.where(p > 0, R["logp"], 0.0)
    bracket = all_g[:, None] + g_ent[:, None] * torch.where(p > 0, lnp + R["H"][:, None], 0.0)
    want = (extra - p * bracket) / T
    want[R["empty"]] = 0
    size[R["empty"]] = 0
    d = torch.where(p > 0, R["d"], 0.0)
    rel_p = U * (4 * d + 10 + R["steps"] + 4 * R["A"][:, None])
    err_b = g_ent.abs()[:, None] * (R["t_H"] + R["t_ln"])[:, None] + 8 * U * (
        mass[:, None] + g_ent.abs()[:, None] * (d + (R["ln_s"].abs() + R["H"].abs())[:, None]))
    err_b[R["empty"]] = 0
    tol = p / T * (rel_p * bracket.abs() + err_b) + 4 * U * (want.abs() + size / T) + torch.finfo(x.dtype).eps / 2 * want.abs()
    # an exponential below 2^-126 is flushed to zero
    _close(got, want, tol * 1.001 + 2.0 ** -126 / T * (1 + 200 * g_ent.abs()[:, None] + mass[:, None]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["normal", "peaked", "constant", "half", "few", "block", "lowest", "all_lowest"])
def test_gradient_against_the_formula(gpu_lib, kind, dtype):
    from qllm2_amd.token_logprobs import token_logprobs
    for n, V, k in [(1, 1, 1), (4, 7, 3), (5, 64, 0), (9, 1001, 6), (70, 255, 64), (3, 16384, 5), (2, 50261, 0)]:
        print(f"case {kind} n={n} V={V} k={k} {dtype}", flush=True)
        x, ids = _rows(kind, n, V, dtype, n + V)
        ids[::4] = -100
        T = 0.7 if n % 2 else 1.0
        g = torch.Generator().manual_seed(n)
        gs = [torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn(n, k, generator=g) if k else None]
        xc = x.cuda().requires_grad_()
        r = token_logprobs(xc, ids.cuda(), temperature=T, top_k=k)
        if k > 1:     # the token among its own alternatives
            ids[-1] = r.top_ids[-1, 1].item()
            r = token_logprobs(xc, ids.cuda(), temperature=T, top_k=k)
        outs = [o for o in r[:3] if o is not None]
        got, = torch.autograd.grad(outs, [xc], [t.cuda() for t in gs if t is not None])
        assert got.dtype == dtype
        # a row with no finite entry has infinities among its outputs and no gradient
        _grad_check(x, ids, k, T, [None if t is None else t.double() for t in gs], got, None if not k else r.top_ids.cpu())


def test_gradient_of_each_output_alone(gpu_lib):
    """One output at a time, gradients that are broadcast, rows in other layouts."""
    from qllm2_amd.token_logprobs import token_logprobs
    x, ids = _rows("normal", 8, 130, torch.float32, 6)
    ids[2] = -100
    zero = torch.zeros(8, dtype=torch.float64)
    buf = torch.zeros(8, 137, device="cuda")
    for layout in ("plain", "offset", "transposed"):
        for which in range(3):
            base = {"plain": x.cuda(), "offset": buf, "transposed": x.T.contiguous().cuda()}[layout].clone().requires_grad_()
            xc = {"plain": lambda b: b, "offset": lambda b: b[:, 3:133], "transposed": lambda b: b.T}[layout](base)
            if layout == "offset":
                with torch.no_grad():
                    xc.copy_(x)
            r = token_logprobs(xc, ids.cuda(), top_k=4)
            got, = torch.autograd.grad(r[which].sum(), [base])
            g = [zero, zero, torch.zeros(8, 4, dtype=torch.float64)]
            g[which] = torch.ones_like(g[which])
            got = {"plain": lambda b: b, "offset": lambda b: b[:, 3:133], "transposed": lambda b: b.T}[layout](got)
            _grad_check(x, ids, 4, 1.0, g, got, r.top_ids.cpu())


def test_gradient_against_differences(gpu_lib):
    """Central differences of the float64 definition agree with the kernel's gradient:
    step h, third derivatives of order one, so the difference is off by about h^2."""
    from qllm2_amd.token_logprobs import token_logprobs
    x, ids = _rows("normal", 3, 11, torch.float32, 7)
    xc = x.cuda().requires_grad_()
    r = token_logprobs(xc, ids.cuda(), temperature=0.8)
    gl, ge = torch.tensor([1.0, -2.0, 0.5]), torch.tensor([0.3, 0.7, -1.0])
    got, = torch.autograd.grad([r.logprobs, r.entropy], [xc], [gl.cuda(), ge.cuda()])

    def f(y):
        R = _reference(y, ids, 0.8)
        return (R["lp"] * gl.double() + R["H"] * ge.double()).sum()

    h = 1e-4
    for i in range(3):
        for j in range(11):
            e = torch.zeros(3, 11, dtype=torch.float64)
            e[i, j] = h
            num = (f(x.double() + e) - f(x.double() - e)) / (2 * h)
            assert abs(num.item() - got[i, j].item()) < 1e-5


def test_captured_pass_replays(gpu_lib):
    """Values, alternatives and gradient captured into one graph and replayed on new
    logits with eager work between."""
    from qllm2_amd.token_logprobs import token_logprobs
    x, ids = _rows("normal", 40, 3001, torch.float32, 8)
    xc, ic = x.cuda().requires_grad_(), ids.cuda()

    def step():
        r = token_logprobs(xc, ic, temperature=0.9, top_k=5)
        d, = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], [xc],
                                 [torch.ones_like(r.logprobs), torch.ones_like(r.entropy), torch.ones_like(r.top_logprobs)])
        return [t.detach() for t in r] + [d]

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
        nx, nids = _rows(["ties", "half", "normal", "few"][seed], 40, 3001, torch.float32, 70 + seed)
        with torch.no_grad():
            xc.copy_(nx)
        ic.copy_(nids)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a,
                               b.nan_to_num(7.0) if b.is_floating_point() else b)


def test_offsets_past_31_bits(gpu_lib):
    """43000 bf16 rows of 50300: the last rows' elements lie past 2^31, forward and in
    the gradient."""
    from qllm2_amd.token_logprobs import token_logprobs
    n, V = 43000, 50300
    buf = torch.zeros(n, V, device="cuda", dtype=torch.bfloat16)
    assert buf.numel() > 2 ** 31
    x, ids = _rows("normal", 4, V, torch.bfloat16, 9)
    buf[-4:] = x.cuda()
    all_ids = torch.full((n,), 7, device="cuda")
    all_ids[-4:] = ids.cuda()
    buf.requires_grad_()
    r = token_logprobs(buf, all_ids, top_k=3)
    _check(x, ids, 3, 1.0, type(r)(*(t[-4:] for t in r)))
    _check(torch.zeros(1, V), torch.tensor([7]), 3, 1.0, type(r)(*(t[:1] for t in r)))
    g = torch.zeros(n, device="cuda")
    g[-4:] = torch.tensor([1.0, -2.0, 0.5, 3.0], device="cuda")
    got, = torch.autograd.grad([r.logprobs, r.entropy], [buf], [g, 0.1 * g])
    g4 = g[-4:].cpu()
    _grad_check(x, ids, 0, 1.0, [g4.double(), (0.1 * g4).double(), None], got[-4:], None)
    assert (got[:-4] == 0).all()


def test_more_rows_than_one_launch_holds(gpu_lib):
    """2^23 blocks of 256 threads are a launch; rows behind it go in a second one."""
    from qllm2_amd.token_logprobs import token_logprobs
    n, V = 2 ** 23 + 5, 8
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(n, V, device="cuda", dtype=torch.bfloat16, generator=g).requires_grad_()
    ids = torch.randint(0, V, (n,), device="cuda", generator=g)
    r = token_logprobs(x, ids, top_k=1)
    (r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum()).backward()
    rows = torch.cat([torch.arange(3), torch.arange(2 ** 23 - 4, n)]).cuda()
    y = x.detach()[rows].requires_grad_()
    q = token_logprobs(y, ids[rows], top_k=1)
    (q.logprobs.sum() + q.entropy.sum() + q.top_logprobs.sum()).backward()
    for a, b in zip(r, q):
        assert torch.equal(a[rows], b)
    assert torch.equal(x.grad[rows], y.grad)
    assert (r.logprobs.detach() < 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,k", [(3, 200001, 64), (300, 200001, 64), (260, 131072, 7), (5, 65536 + 13, 33), (700, 3, 2)])
def test_alternatives_of_long_rows(gpu_lib, n, V, k, dtype):
    """Vocabularies of many batches a thread: the order of a stable sort, and its log softmax."""
    from qllm2_amd.token_logprobs import token_logprobs
    g = torch.Generator(device="cuda").manual_seed(V + n)
    x = (torch.randn(n, V, device="cuda", generator=g) * 3).to(dtype)
    x[1::3, V // 2:] = float("-inf")
    x[2::3] = x[2::3].sort(-1).values  # the largest entries side by side at the end
    ids = torch.randint(0, V, (n,), device="cuda", generator=g)
    r = token_logprobs(x, ids, top_k=k)
    _, order = torch.sort(x, dim=-1, descending=True, stable=True)
    assert torch.equal(r.top_ids, order[:, :k])
    # a log probability of at most 40 (or -inf): V additions in 1024 or 256 chains and their joining, the
    # maximum's rescalings and two roundings of the result, below (V / 256 + 100) 2^-24 of s in all
    want = torch.log_softmax(x.double(), -1).gather(1, order[:, :k])
    assert torch.equal(r.top_logprobs.isinf(), want.isinf())
    live = ~want.isinf()
    err = (r.top_logprobs.double() - want)[live].abs().max().item()
    assert err <= (V / 256 + 100) * 2.0 ** -24 + 40 * 2.0 ** -22
