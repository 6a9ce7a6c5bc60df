"""Products with 4-bit weights (qllm2_amd/linear4.py, qpam_linear4) against float64.

Bound of a finished fp32 sum: the products are exact (a bf16 times a value of at most 3
bits; an fp32 value is the exact sum of three bf16 parts), each addition of a group's sum
(group terms, three times as many in fp32), of the groups and of the waves (at most 16) is
off by at most 2^-23 of the sum of magnitudes, the scale's product and a bias by 2^-24 each.
A bf16 result adds its rounding, half a step: 2^-8 of its value."""

import pytest
import torch

from qllm2_amd.linear4 import MAGNITUDES, Weight4, complex_linear4, dequantize4, linear4, quantize4

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _codes(n, columns, group, seed, device="cuda"):
    """Every code at random (-0 among them) and scales over three decades, of the sign of either."""
    g = torch.Generator(device=device).manual_seed(seed)
    codes = torch.randint(0, 256, (n, -(-columns // 2)), device=device, generator=g, dtype=torch.uint8)
    scales = torch.randn(n, -(-columns // group), device=device, generator=g) * 10 ** (
        3 * torch.rand(n, -(-columns // group), device=device, generator=g) - 2)
    return codes, scales.to(BF16)


def _rows(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _matrix(w):
    """float64 [out, K] of a real weight; of a complex one the real matrix [2 out, 2 in] on interleaved rows and outputs."""
    v = w.dequantize().double()
    if not w.complex:
        return v
    re, im = v[..., 0], v[..., 1]
    return torch.stack([torch.stack([re, -im], -1), torch.stack([im, re], -1)], 1).reshape(2 * w.out_features, -1)


def _check(y, x, w, bias=None, tail=None, planes=False):
    """y against float64 within the bound above."""
    m, x2 = _matrix(w), x.double().reshape(-1, w.in_features * (2 if w.complex else 1))
    want, size = x2 @ m.T.contiguous(), x2.abs() @ m.abs().T.contiguous()
    parts = 3 if x.dtype == F32 else 1
    steps = parts * w.group + -(-x2.shape[1] // w.group) + 17
    tol = (steps * 2.0 ** -23 + 2.0 ** -23) * size + 1e-36
    if bias is not None:
        want = want + bias.double().reshape(-1)
        tol = tol + 2.0 ** -24 * (want.abs() + tol)
    if planes:
        want, tol = (torch.cat([t[:, 0::2], t[:, 1::2]], 1) for t in (want, tol))
    if tail is not None:   # fp32 multiply-adds over 64 lanes and their joining
        t = tail.double().T.contiguous()
        n = -(-x2.shape[1] // 64) + 7
        want, tol = torch.cat([want, x2 @ t], 1), torch.cat([tol, n * 2.0 ** -24 * (x2.abs() @ t.abs()) + 1e-36], 1)
    if y.dtype == BF16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    off = (y.double().reshape(want.shape) - want).abs()
    bad = off > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((off / tol).max()):.2f} of the bound"


REAL = [  # n, K, N, group
    (1, 1, 1, 32), (1, 128, 16, 32), (1, 1536, 300, 32), (2, 33, 17, 64), (3, 127, 15, 128), (16, 129, 33, 32), (17, 500, 100, 64),
    (33, 1000, 65, 128), (64, 255, 48, 32), (65, 384, 130, 64), (130, 2049, 40, 32), (300, 96, 515, 128), (1000, 160, 200, 32),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,K,N,group", REAL)
def test_real_products(gpu_lib, n, K, N, group, dtype):
    w = Weight4(*_codes(N, K, group, 1), K, group)
    x = _rows((n, K), dtype, 2)
    _check(linear4(x, w), x, w)
    b = _rows((N,), F32, 3)
    _check(linear4(x, w, b), x, w, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,K,N,group", REAL)
def test_complex_products(gpu_lib, n, K, N, group, dtype):
    w = Weight4(*_codes(N, 2 * K, group, 4), K, group, complex=True)
    x = _rows((n, K, 2), dtype, 5)
    y = complex_linear4(x, w)
    assert y.shape == (n, N, 2) and y.dtype == dtype
    _check(y, x, w)
    b, tail = _rows((N, 2), F32, 6), _rows((5, 2 * K), dtype, 7)
    _check(complex_linear4(x, w, b), x, w, b)
    _check(complex_linear4(x, w, planes=True), x, w, planes=True)
    y = complex_linear4(x, w, b, planes=True, tail=tail)
    assert y.shape == (n, 2 * N + 5)
    # the bias belongs to the complex outputs
    _check(y[:, :2 * N], x, w, b, planes=True)
    _check(complex_linear4(x, w, planes=True, tail=tail), x, w, tail=tail, planes=True)


SHAPES = [  # sizes on either side of where the blocks' shape changes, few inputs; long rows of few outputs
    (16, 64, 4100), (16, 72, 8300), (3, 100, 16500), (20, 130, 1500), (40, 96, 2000), (100, 96, 1700), (200, 130, 2000),
    (300, 64, 3300), (600, 96, 4000), (1000, 72, 4000), (10, 3100, 40), (16, 6200, 1000), (60, 3100, 17),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,K,N", SHAPES)
@pytest.mark.parametrize("group", [32, 128])
def test_every_shape_of_blocks(gpu_lib, n, K, N, group, dtype):
    w = Weight4(*_codes(N, K, group, 50), K, group)
    x, b = _rows((n, K), dtype, 51), _rows((N,), F32, 52)
    _check(linear4(x, w, b), x, w, b)
    K = K // 2
    w = Weight4(*_codes(N, 2 * K, group, 53), K, group, complex=True)
    x, tail = _rows((n, K, 2), dtype, 54), _rows((3, 2 * K), dtype, 55)
    _check(complex_linear4(x, w), x, w)
    _check(complex_linear4(x, w, planes=True, tail=tail), x, w, tail=tail, planes=True)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_weight_in_its_place(gpu_lib, group):
    """Unit rows give the weights back bit for bit: the layout, the codes, their scales."""
    K, N = 261, 77
    w = Weight4(*_codes(N, K, group, 8), K, group)
    assert torch.equal(linear4(torch.eye(K, device="cuda"), w).T, w.dequantize() + 0.0)
    c = Weight4(*_codes(N, 2 * K, group, 9), K, group, complex=True)
    v = c.dequantize()
    e = torch.eye(K, device="cuda")
    for x, want in ((torch.stack([e, 0 * e], -1), v), (torch.stack([0 * e, e], -1), torch.stack([-v[..., 1], v[..., 0]], -1))):
        assert torch.equal(complex_linear4(x, c).transpose(0, 1) + 0.0, want + 0.0)


def _layouts(x):
    """x in other strides: rows of a wider matrix off 16 bytes, transposed, a row expanded, every second row."""
    n, k = x.shape
    wide = torch.empty(n, k + 3, device=x.device, dtype=x.dtype)
    wide[:, 1:k + 1] = x
    twice = x.repeat_interleave(2, 0)
    return {"wide": wide[:, 1:k + 1], "transposed": x.T.contiguous().T, "expanded": x[:1].expand(n, k), "every second": twice[::2]}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 7, 70])
def test_layouts_of_the_rows(gpu_lib, n, dtype):
    K, N = 144, 50
    w = Weight4(*_codes(N, K, 32, 10), K, 32)
    c = Weight4(*_codes(N, K, 32, 11), K // 2, 32, complex=True)
    for name, v in _layouts(_rows((n, K), dtype, 12)).items():
        assert torch.equal(linear4(v, w), linear4(v.contiguous(), w)), name
        z = v.unflatten(1, (K // 2, 2))
        assert torch.equal(complex_linear4(z, c), complex_linear4(z.contiguous(), c)), name
    planes = _rows((2, n, K // 2), dtype, 13).permute(1, 2, 0)
    assert torch.equal(complex_linear4(planes, c), complex_linear4(planes.contiguous(), c))
    x = _rows((3, n, K), dtype, 14)
    assert torch.equal(linear4(x, w), linear4(x.view(-1, K), w).view(3, n, N))
    assert torch.equal(linear4(x[1, 0], w), linear4(x[1, :1], w)[0])
    t = _rows((9, K + 1), dtype, 15)[:, 1:]
    z = _rows((n, K // 2, 2), dtype, 16)
    assert torch.equal(complex_linear4(z, c, planes=True, tail=t), complex_linear4(z, c, planes=True, tail=t.contiguous()))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_rows(gpu_lib, dtype):
    w = Weight4(*_codes(20, 64, 32, 17), 32, 32, complex=True)
    assert complex_linear4(torch.empty(0, 32, 2, device="cuda", dtype=dtype), w).shape == (0, 20, 2)
    assert complex_linear4(torch.empty(4, 0, 32, 2, device="cuda", dtype=dtype), w, planes=True).shape == (4, 0, 40)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 40, 200])
def test_infinities_and_nan_stay_in_their_rows(gpu_lib, n, dtype):
    """As IEEE products and sums have them, and the other rows as if they were not there."""
    K, N = 200, 60
    w = Weight4(*_codes(N, K, 32, 18), K, 32)
    x = _rows((n, K), dtype, 19)
    clean = linear4(x, w)
    bad = x.clone()
    bad[0, 5], bad[1, 150], bad[2, 199] = float("inf"), float("nan"), float("-inf")
    y = linear4(bad, w)
    assert torch.equal(y[3:], clean[3:])
    want = bad[:3].double() @ w.dequantize().double().T.contiguous()
    assert torch.equal(torch.isnan(y[:3]), torch.isnan(want))
    assert torch.equal(torch.isinf(y[:3]), torch.isinf(want)) and torch.equal(y[:3].sign().nan_to_num(0), want.sign().nan_to_num(0).to(dtype))


def test_nan_payloads_in_low_bits(gpu_lib):
    """A NaN whose payload is behind the first 16 bits is no infinity."""
    w = Weight4(*_codes(16, 32, 32, 20), 32, 32)
    x = torch.zeros(1, 32, device="cuda")
    x[0, 3] = torch.tensor(0x7F800001, dtype=torch.int32).view(F32).cuda()
    assert torch.isnan(linear4(x, w)).all()


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_small_and_large_values(gpu_lib, scale):
    w = Weight4(*_codes(40, 96, 32, 21), 96, 32)
    x = _rows((5, 96), F32, 22) * scale
    _check(linear4(x, w), x, w)
    mixed = x * 10.0 ** torch.arange(-3, 3, device="cuda").repeat(16)
    _check(linear4(mixed, w), mixed, w)


def test_more_rows_than_a_grid_takes(gpu_lib):
    """Rows in pieces of 2^19, the tail's with them."""
    n = (1 << 19) + 100
    w = Weight4(*_codes(5, 32, 32, 70), 16, 32, complex=True)
    x, tail = _rows((n, 16, 2), BF16, 71), _rows((3, 32), BF16, 72)
    y = complex_linear4(x, w, planes=True, tail=tail)
    for at in (slice(0, 64), slice((1 << 19) - 32, (1 << 19) + 32), slice(n - 64, n)):
        _check(y[at], x[at], w, tail=tail, planes=True)
    w = Weight4(*_codes(40, 90, 64, 73), 90, 64)
    x = _rows((n, 90), F32, 74)
    y = linear4(x, w)
    for at in (slice(0, 64), slice((1 << 19) - 32, (1 << 19) + 32), slice(n - 64, n)):
        _check(y[at], x[at], w)


def test_offsets_past_32_bits(gpu_lib):
    """Outputs, then rows, of more than 2^31 elements."""
    K, N, n = 32, 50000, 45000
    w = Weight4(*_codes(N, K, 32, 23), K, 32)
    x = _rows((n, K), BF16, 24)
    y = linear4(x, w)
    _check(y[-3:], x[-3:], w)
    _check(y[22000:22003], x[22000:22003], w)
    del y
    w = Weight4(*_codes(8, 64, 32, 25), 64, 32)
    x = torch.empty(40000, 60000, device="cuda", dtype=BF16)[:, :64]
    x.copy_(_rows((40000, 64), BF16, 26))
    _check(linear4(x, w), x, w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 40])
def test_rows_far_apart(gpu_lib, n, dtype):
    """A row stride above 2^24 elements; from there on rows are laid out for the kernels."""
    K = 200
    x = torch.empty(n, (1 << 24) + 8, device="cuda", dtype=dtype)[:, 3:3 + K]
    x.copy_(_rows((n, K), dtype, 60))
    for N in (50, 5000, 9000):
        w = Weight4(*_codes(N, K, 64, 61), K, 64)
        _check(linear4(x, w), x, w)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_far_apart_in_every_shape(gpu_lib, dtype, group):
    """The laid rows' shapes of blocks between the ones above, real and complex."""
    K, n = 150, 40
    x = torch.empty(n, (1 << 24) + 8, device="cuda", dtype=dtype)[:, 3:3 + K]
    x.copy_(_rows((n, K), dtype, 62))
    for N in (1700, 3200, 16000):
        w = Weight4(*_codes(N, K, group, 63), K, group)
        _check(linear4(x, w), x, w)
        w = Weight4(*_codes(N, K, group, 64), K // 2, group, complex=True)
        _check(complex_linear4(x.unflatten(1, (K // 2, 2)), w), x, w)


def test_streams_and_graphs(gpu_lib):
    K, N = 256, 130
    w = Weight4(*_codes(N, 2 * K, 32, 27), K, 32, complex=True)
    tail = _rows((3, 2 * K), BF16, 28)
    x = _rows((6, K, 2), BF16, 29)
    want = complex_linear4(x, w, planes=True, tail=tail)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = complex_linear4(x, w, planes=True, tail=tail)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = complex_linear4(x, w, planes=True, tail=tail)
    for seed in range(30, 34):
        x.copy_(_rows((6, K, 2), BF16, seed))
        graph.replay()
        want = complex_linear4(x, w, planes=True, tail=tail)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_same_bits_on_every_call(gpu_lib):
    for n in (1, 20, 200):
        w = Weight4(*_codes(100, 600, 64, 35), 300, 64, complex=True)
        x = _rows((n, 300, 2), F32, 36)
        first = complex_linear4(x, w)
        assert all(torch.equal(complex_linear4(x, w), first) for _ in range(3))


def test_compiled_and_faked(gpu_lib):
    from torch._subclasses.fake_tensor import FakeTensorMode
    w = Weight4(*_codes(24, 128, 32, 37), 64, 32, complex=True)
    x, tail = _rows((4, 64, 2), BF16, 38), _rows((2, 128), BF16, 39)
    for kw in (dict(), dict(planes=True), dict(planes=True, tail=tail)):
        real = complex_linear4(x, w, **kw)
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            fake = complex_linear4(mode.from_tensor(x), w, **kw)
        assert fake.shape == real.shape and fake.dtype == real.dtype and fake.stride() == real.stride()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(5, 1), (16, 128), (33, 201)])
def test_quantized_on_the_device_as_on_the_host(gpu_lib, shape, group):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(40))
    codes, scales = quantize4(w, group=group)
    on = Weight4(codes.cuda(), scales.cuda(), shape[1], group)
    assert torch.equal(on.dequantize().cpu(), dequantize4(codes, scales, shape[1], group))
    assert set(dequantize4(codes, torch.ones_like(scales), shape[1], group).abs().unique().tolist()) <= set(MAGNITUDES)


def test_gradients_are_refused(gpu_lib):
    w = Weight4(*_codes(16, 32, 32, 41), 32, 32)
    x = _rows((2, 32), F32, 42).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        linear4(x, w)
    with torch.no_grad():
        assert not linear4(x, w).requires_grad
