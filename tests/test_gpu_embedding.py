"""The complex embedding lookup and its gradient (qpam_embed_fwd / qpam_embed_bwd)
against plain torch in float64.

Lookup: one fp32 product and one rounding, so it equals torch's bit for bit.
Gradient: fp32 sums of c terms, in any grouping, are off by at most
(c - 1) 2^-24 sum |x| (to first order; c 2^-24 covers the second), the product with
the scale and the final rounding add eps / 2 each:
    |error| <= scale c 2^-24 sum |x| + (2^-24 + eps / 2) |y|,
checked element by element."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ids(kind, n, V, g):
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g)
    if kind == "text":      # few tokens make up most of it
        return (V ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    if kind == "one":       # one run through every chunk
        return torch.full((n,), V // 2)
    if kind == "two":       # half padding, half another token
        return torch.where(torch.rand(n, generator=g) < 0.5, 0, V - 1)
    if kind == "outside":   # ids outside the table between others
        return torch.randint(-V, 2 * V, (n,), generator=g)
    raise ValueError(kind)


def _data(kind, n, V, dim, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    re, im = (torch.randn(V, dim, generator=g).to(dtype) for _ in range(2))
    return _ids(kind, n, V, g), re, im, torch.randn(n, dim, 2, generator=g).to(dtype)


def _want(ids, re, im, scale):
    ok = (ids >= 0) & (ids < re.shape[0])
    z = torch.stack([re[ids.clamp(0, re.shape[0] - 1)], im[ids.clamp(0, re.shape[0] - 1)]], -1)
    return torch.where(ok[..., None, None], (z.float() * scale).to(re.dtype), 0)


def _check_grad(got, ids, dz, V, scale, pad=None, part=0):
    """got: the gradient of table `part` on the CPU."""
    ok = (ids >= 0) & (ids < V)
    if pad is not None:
        ok &= ids != pad
    x = dz[..., part].reshape(-1, dz.shape[-2])[ok.reshape(-1)].double()
    at = ids.reshape(-1)[ok.reshape(-1)]
    shape = (V, dz.shape[-2])
    s = torch.zeros(shape, dtype=torch.float64).index_add_(0, at, x)
    mass = torch.zeros(shape, dtype=torch.float64).index_add_(0, at, x.abs())
    c = torch.zeros(V, dtype=torch.float64).index_add_(0, at, torch.ones(len(at), dtype=torch.float64))
    want, u = s * scale, 2.0 ** -24
    bound = abs(scale) * c[:, None] * u * mass + (u + torch.finfo(dz.dtype).eps / 2) * want.abs()
    err = (got.double() - want).abs()
    assert (err <= bound * 1.001).all(), (err - bound).max().item()
    assert (got[c == 0] == 0).all()


CASES = [
    # kind, n, V, dim
    ("uniform", 1, 1, 1), ("uniform", 1, 50261, 8), ("uniform", 2, 3, 2), ("one", 16, 5, 4), ("one", 17, 5, 6),
    ("uniform", 63, 64, 5), ("uniform", 64, 65, 3), ("text", 257, 255, 33), ("two", 1000, 256, 64),
    ("outside", 999, 300, 65), ("one", 5000, 1000, 130), ("text", 16384, 50261, 36), ("uniform", 16383, 65536, 16),
    ("text", 16385, 65535, 7), ("two", 40001, 70000, 12), ("one", 20000, 3, 68), ("outside", 33000, 1000, 4),
    ("uniform", 4097, 17000000, 1),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,n,V,dim", CASES)
def test_lookup_and_gradient(gpu_lib, kind, n, V, dim, dtype):
    from qllm2_amd.embedding import complex_embedding
    print(f"case {kind} n={n} V={V} dim={dim} {dtype}", flush=True)
    ids, re, im, dz = _data(kind, n, V, dim, dtype, n + V + dim)
    scale = 1.0 if n % 2 else dim ** 0.5
    rc, ic = re.cuda().requires_grad_(), im.cuda().requires_grad_()
    z = complex_embedding(ids.cuda(), rc, ic, scale=scale)
    assert z.dtype == dtype and torch.equal(z.detach().cpu(), _want(ids, re, im, scale))
    grads = torch.autograd.grad(z, [rc, ic], dz.cuda())
    again = torch.autograd.grad(complex_embedding(ids.cuda(), rc, ic, scale=scale), [rc, ic], dz.cuda())
    for part, (got, same) in enumerate(zip(grads, again)):
        assert got.dtype == dtype and torch.equal(got, same)      # the same bits on every call
        _check_grad(got.cpu(), ids, dz, V, scale, part=part)


@pytest.mark.parametrize("pad", [0, 7, -1])
def test_padding_token_shapes_and_int32(gpu_lib, pad):
    """[B, T] int32 ids; the padding token is looked up and gets no gradient."""
    from qllm2_amd.embedding import complex_embedding
    ids, re, im, dz = _data("text", 600, 9, 24, torch.float32, 5)
    ids = ids.view(3, 200).to(torch.int32)
    rc, ic = re.cuda().requires_grad_(), im.cuda().requires_grad_()
    z = complex_embedding(ids.cuda(), rc, ic, scale=0.5, padding_idx=pad)
    assert z.shape == (3, 200, 24, 2) and torch.equal(z.detach().cpu(), _want(ids.long(), re, im, 0.5))
    grads = torch.autograd.grad(z, [rc, ic], dz.view(3, 200, 24, 2).cuda())
    for part, got in enumerate(grads):
        _check_grad(got.cpu(), ids.long(), dz.view(3, 200, 24, 2), 9, 0.5, pad=pad % 9, part=part)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_tables_ids_and_gradients(gpu_lib, dtype):
    """Tables as the halves of one [V, 2 dim] matrix or as transposed storage, every
    other id of a longer list, dz from a broadcast sum and from a strided view."""
    from qllm2_amd.embedding import complex_embedding
    ids, re, im, dz = _data("text", 500, 77, 20, dtype, 6)
    wide = torch.cat([re, im], 1).cuda()
    every = torch.stack([ids, ids + 1], 1).cuda()[:, 0]
    for rc, ic in ((wide[:, :20], wide[:, 20:]), (re.T.contiguous().cuda().T, im.cuda()),
                   (wide[:, 1:20], wide[:, 3:22])):
        want = _want(ids, rc.cpu(), ic.cpu(), 1.5)
        rc, ic = rc.detach().requires_grad_(), ic.detach().requires_grad_()
        z = complex_embedding(every, rc, ic, scale=1.5)
        assert torch.equal(z.detach().cpu(), want)
        d = z.shape[1]
        strided = torch.zeros(500, d, 5, device="cuda", dtype=dtype)
        strided[:, :, 1:3] = dz[:, :d].cuda()
        ones = torch.ones(1, 1, 1, device="cuda", dtype=dtype).expand(500, d, 2)
        for g in (strided[:, :, 1:3], ones):
            for part, got in enumerate(torch.autograd.grad(z, [rc, ic], g, retain_graph=True)):
                _check_grad(got.cpu(), ids, g.cpu(), 77, 1.5, part=part)


def test_one_table_and_no_gradient(gpu_lib):
    """Only one table asks for a gradient; neither does; an empty list of ids."""
    from qllm2_amd.embedding import complex_embedding
    ids, re, im, dz = _data("text", 100, 30, 8, torch.float32, 7)
    rc = re.cuda().requires_grad_()
    got, = torch.autograd.grad(complex_embedding(ids.cuda(), rc, im.cuda()), [rc], dz.cuda())
    _check_grad(got.cpu(), ids, dz, 30, 1.0)
    assert not complex_embedding(ids.cuda(), re.cuda(), im.cuda()).requires_grad
    z = complex_embedding(ids[:0].cuda(), rc, im.cuda())
    assert z.shape == (0, 8, 2)
    got, = torch.autograd.grad(z, [rc], torch.zeros_like(z))
    assert got.shape == rc.shape and (got == 0).all()


def test_gradient_against_differences(gpu_lib):
    """The lookup is linear in the tables: <dz, f(W + D) - f(W)> = <grad, D>.  Small
    whole numbers, so that every product and sum is exact in fp32."""
    from qllm2_amd.embedding import complex_embedding
    g = torch.Generator().manual_seed(8)
    ids = _ids("text", 700, 50, g)
    w, d = (torch.randint(-4, 5, (2, 50, 12), generator=g).float().cuda() for _ in range(2))
    dz = torch.randint(-4, 5, (700, 12, 2), generator=g).float().cuda()
    re, im = w[0].clone().requires_grad_(), w[1].clone().requires_grad_()
    z = complex_embedding(ids.cuda(), re, im, scale=2.0)
    grads = torch.autograd.grad(z, [re, im], dz)
    moved = complex_embedding(ids.cuda(), w[0] + d[0], w[1] + d[1], scale=2.0)
    assert ((moved - z) * dz).double().sum().item() == sum((a * b).double().sum().item() for a, b in zip(grads, d))


def test_infinities_and_nan_stay_in_their_rows(gpu_lib):
    from qllm2_amd.embedding import complex_embedding
    for dtype in (torch.float32, torch.bfloat16):
        ids, re, im, dz = _data("uniform", 200, 20, 16, dtype, 9)
        re[3, 4], im[5, 6] = float("nan"), float("inf")
        dz[0, 1, 0], dz[1, 2, 1] = float("nan"), float("-inf")
        ids[0], ids[1] = 11, 12
        rc, ic = re.cuda().requires_grad_(), im.cuda().requires_grad_()
        z = complex_embedding(ids.cuda(), rc, ic)
        assert torch.equal(z.detach().cpu().nan_to_num(7.0), _want(ids, re, im, 1.0).nan_to_num(7.0))
        d_re, d_im = torch.autograd.grad(z, [rc, ic], dz.cuda())
        assert d_re.isnan().nonzero().tolist() == [[11, 1]] and not d_re.isinf().any()
        assert d_im.isinf().nonzero().tolist() == [[12, 2]] and d_im[12, 2] < 0 and not d_im.isnan().any()


def test_captured_training_step_replays(gpu_lib):
    """Lookup and gradient captured into one graph, replayed on new ids and
    gradients with eager work between."""
    from qllm2_amd.embedding import complex_embedding
    for n in (300, 17000):
        ids, re, im, dz = _data("text", n, 1000, 32, torch.float32, n)
        sid, sdz = ids.cuda(), dz.cuda()
        rc, ic = re.cuda().requires_grad_(), im.cuda().requires_grad_()

        def step():
            z = complex_embedding(sid, rc, ic, scale=3.0)
            return (z.detach(), *torch.autograd.grad(z, [rc, ic], sdz))

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
            nid, _, _, ndz = _data("two" if seed % 2 else "text", n, 1000, 32, torch.float32, 50 + seed)
            sid.copy_(nid)
            sdz.copy_(ndz)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step()):
                assert torch.equal(a, b)


def test_two_streams_at_once(gpu_lib):
    """Calls on two streams share nothing."""
    from qllm2_amd.embedding import complex_embedding
    data = [_data("text", 5000, 500, 64, torch.float32, 60 + i) for i in range(2)]
    dev = [[t.cuda() for t in d] for d in data]
    torch.cuda.synchronize()
    outs = [None, None]
    for i, s in enumerate((torch.cuda.Stream(), torch.cuda.Stream())):
        with torch.cuda.stream(s):
            ids, re, im, dz = dev[i]
            re.requires_grad_(), im.requires_grad_()
            outs[i] = torch.autograd.grad(complex_embedding(ids, re, im), [re, im], dz)
    torch.cuda.synchronize()
    for (ids, _, _, dz), got in zip(data, outs):
        for part in (0, 1):
            _check_grad(got[part].cpu(), ids, dz, 500, 1.0, part=part)


def test_offsets_past_31_bits(gpu_lib):
    """1.1 million ids of 1024 columns: the rows' elements pass 2^31.  Gradients of small
    whole numbers, so that every sum is exact: token v gets the sum over its positions i
    of (i % 7) - 3 in every column."""
    from qllm2_amd.embedding import complex_embedding
    n, V, dim = 1100000, 1000, 1024
    ids = torch.randint(0, V, (n,), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    re, im = (torch.randn(V, dim, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    with torch.no_grad():
        z = complex_embedding(ids, re, im)
    assert z.numel() > 2 ** 31
    for rows in (slice(0, 3), slice(n // 2, n // 2 + 3), slice(n - 3, n)):
        assert torch.equal(z[rows], torch.stack([re[ids[rows]], im[ids[rows]]], -1))
    del z
    step = (torch.arange(n, device="cuda") % 7 - 3).bfloat16()
    from qllm2_amd.embedding import embed_bwd_op
    d_re, d_im = embed_bwd_op(ids, step[:, None, None].expand(n, dim, 2).contiguous(), V, 1.0, -1)
    want = torch.zeros(V, device="cuda", dtype=torch.float64).index_add_(0, ids, step.double()).bfloat16()
    for d in (d_re, d_im):
        assert torch.equal(d, want[:, None].expand(V, dim))


def test_more_rows_than_one_launch_holds(gpu_lib):
    """2^25 rows of 64 lanes are a launch; rows behind it go in a second one."""
    from qllm2_amd.embedding import complex_embedding
    n, V, dim = 2 ** 25 + 5, 50, 33
    g = torch.Generator(device="cuda").manual_seed(5)
    re, im = (torch.randn(V, dim, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(2))
    ids = torch.randint(0, V, (n,), device="cuda", dtype=torch.int32, generator=g)
    z = complex_embedding(ids, re, im)
    for rows in (slice(0, 3), slice(2 ** 25 - 4, n)):
        t = ids[rows].long()
        assert torch.equal(z[rows], torch.stack([re[t], im[t]], -1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("outside", [0.0, -2.5, float("inf"), float("nan")])
@pytest.mark.parametrize("dim", [32, 7])
def test_rows_of_ids_outside_the_table(gpu_lib, dim, outside, dtype):
    """`outside` as it is, in whole rows; the table's rows and both gradients as without it."""
    from qllm2_amd.embedding import complex_embedding
    g = torch.Generator().manual_seed(dim)
    re, im = (torch.randn(20, dim, generator=g).to(dtype).cuda().requires_grad_() for _ in range(2))
    ids = torch.tensor([3, 20, -1, 0, 19, 2 ** 40, -2 ** 40, 3], device="cuda")
    bad = (ids < 0) | (ids >= 20)
    z = complex_embedding(ids, re, im, scale=1.5, outside=outside)
    want = torch.full((4, dim, 2), outside, dtype=dtype, device="cuda")
    assert torch.allclose(z[bad], want, rtol=0, atol=0, equal_nan=True)
    plain = complex_embedding(ids, re, im, scale=1.5)
    assert torch.equal(z[~bad], plain[~bad])
    dz = torch.randn(8, dim, 2, generator=g).to(dtype).cuda()
    for a, b in zip(torch.autograd.grad(z, [re, im], dz), torch.autograd.grad(plain, [re, im], dz)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 7, 64, 100])
def test_tables_of_any_column_stride(gpu_lib, dim, dtype):
    """Views of one interleaved table (16-byte aligned and not), columns two and five apart, a transposed and an
    expanded table: the bits of contiguous ones, with both gradients."""
    from qllm2_amd.embedding import complex_embedding
    g = torch.Generator().manual_seed(dim)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    ids, dz = torch.randint(-1, 31, (2, 40), generator=g).cuda(), rn(2, 40, dim, 2)
    flat = rn(30 * dim * 2 + 1)[1:].view(30, dim, 2)
    tables = [rn(30, dim, 2).unbind(-1), rn(30, dim, 2).unbind(-1)[::-1], flat.unbind(-1), rn(30, dim + 3, 2)[:, 2:2 + dim].unbind(-1),
              (rn(30, dim * 5)[:, ::5], rn(30, dim * 2)[:, 1::2]), (rn(dim, 30).T, rn(30, dim)), (rn(1, dim).expand(30, dim), rn(30, dim)),
              (rn(30, 1).expand(30, dim), rn(30, 2 * dim).view(30, dim, 2)[..., 0])]
    for re, im in tables:
        res = []
        for a, b in ((re, im), (re.clone(memory_format=torch.contiguous_format), im.clone(memory_format=torch.contiguous_format))):
            a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
            z = complex_embedding(ids, a, b, scale=1.5, padding_idx=3)
            res.append([z, *torch.autograd.grad(z, [a, b], dz)])
        for s, t in zip(*res):
            assert torch.equal(s, t)


def test_interleaved_tables_are_not_copied(gpu_lib):
    from qllm2_amd.embedding import complex_embedding
    for dtype in (torch.float32, torch.bfloat16):
        table = torch.randn(20000, 64, 2, device="cuda").to(dtype)
        ids = torch.arange(50, device="cuda")
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        z = complex_embedding(ids, *table.unbind(-1))
        assert torch.equal(z, table[:50])
        assert torch.cuda.max_memory_allocated() - before < table.numel() * table.element_size() // 4
