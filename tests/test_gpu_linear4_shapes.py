"""Products with 4-bit weights in every shape of blocks that the library chooses by the
sizes: the exactness of fp32 rows' three parts bit for bit, values up to the largest ones,
infinities and NaN, the rows' layouts, repeated and captured calls."""

import pytest
import torch

from qllm2_amd.linear4 import Weight4, complex_linear4, linear4
from tests.test_gpu_linear4 import BF16, F32, _check, _codes, _layouts, _matrix, _rows

pytestmark = pytest.mark.gpu

# rows, outputs: step kernels of one (one and several blocks of rows), two and four tiles, tiles split along the
# inputs, tiles of 32 rows, then the large ones, the last with blocks of half the outputs behind the whole rounds
CASES = [(5, 200), (40, 300), (16, 4100), (16, 16500), (40, 1500), (100, 1500), (200, 2000), (520, 1100), (700, 1900), (700, 6100)]
INPUTS = [192, 200]   # real ones: whole blocks of 64 (bf16 tiles read such rows as they stand), and not


def _product(x, w, bias=None):
    return complex_linear4(x.unflatten(1, (-1, 2)), w, bias).flatten(1) if w.complex else linear4(x, w, bias)


def _weight(N, K, group, seed, cplx):
    return Weight4(*_codes(N, K, group, seed), K // 2 if cplx else K, group, complex=cplx)


def _powers(N, K, group, cplx, lo, hi, seed=1, codes=(1, 2, 4, 6)):
    """Weights whose values are powers of two: codes of 0.5, 1, 2 or 4, scales 2^lo to 2^hi, either sign."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.tensor(codes, device="cuda")[torch.randint(0, len(codes), (N, K), device="cuda", generator=g)]
    idx = idx + 8 * torch.randint(0, 2, (N, K), device="cuda", generator=g)
    scales = torch.exp2(torch.randint(lo, hi + 1, (N, -(-K // group)), device="cuda", generator=g).float()).to(BF16)
    return Weight4((idx[:, 0::2] | idx[:, 1::2] << 4).to(torch.uint8), scales, K // 2 if cplx else K, group, complex=cplx)


def _bits(n, lo, hi, seed):
    """fp32 values of 24 significant bits at random, the last one set, of magnitudes 2^lo to 2^hi."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    mantissa = torch.randint(0, 1 << 23, (n,), device="cuda", generator=g, dtype=torch.int32) | 1
    exponent = torch.randint(lo + 127, hi + 127, (n,), device="cuda", generator=g, dtype=torch.int32)
    sign = torch.randint(0, 2, (n,), device="cuda", generator=g, dtype=torch.int32)
    return (mantissa | exponent << 23 | sign << 31).view(F32)


def _one_a_row(values, K, dtype):
    """Rows of zeros with one value each, in every column in turn."""
    n = values.numel()
    x = torch.zeros(n, K, device="cuda", dtype=dtype)
    at = (torch.arange(n, device="cuda") * 37 + 3) % K
    x[torch.arange(n, device="cuda"), at] = values.to(dtype)
    return x, at


def _one_product(x, at, w):
    """What rows of _one_a_row give: one exact product in each place."""
    m = _matrix(w)
    want = x.double().gather(1, at[:, None]) * m.T.contiguous()[at]
    assert torch.equal(want.to(x.dtype).double(), want)   # (a power of two takes no bits)
    return want.to(x.dtype)


def test_two_parts_do_not_hold_a_value():
    """The values below tell three bf16 parts from two."""
    x = _bits(4000, -10, 10, 2)
    hi = x.to(BF16).float()
    mid = (x - hi).to(BF16).float()
    assert (hi + mid != x).float().mean() > 0.9 and torch.equal(hi + mid + (x - hi - mid).to(BF16).float(), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("K", INPUTS)
@pytest.mark.parametrize("n,N", CASES)
def test_every_bit_of_a_row(gpu_lib, n, N, K, cplx, dtype):
    """24 significant bits times a power of two come out as they went in."""
    for group in (32, 128):
        w = _powers(N, K, group, cplx, -8, 8)
        x, at = _one_a_row(_bits(n, -20, 20, 3), K, dtype)
        assert torch.equal(_product(x, w), _one_product(x, at, w))


@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("n,N", [c for c in CASES if c[0] <= 200])
def test_every_bit_of_rows_far_apart(gpu_lib, n, N, cplx):
    """Rows that are laid out in front of the kernels."""
    K = 200
    w = _powers(N, K, 64, cplx, -8, 8)
    values, at = _one_a_row(_bits(n, -20, 20, 4), K, F32)
    x = torch.empty(n, (1 << 24) + 8, device="cuda")[:, 3:3 + K]
    x.copy_(values)
    assert torch.equal(_product(x, w), _one_product(values, at, w))


@pytest.mark.parametrize("lo,hi", [(119, 127), (127, 128)])
@pytest.mark.parametrize("n,N", [(5, 200), (16, 4100), (16, 16500), (520, 1100), (700, 1900)])
def test_the_largest_values(gpu_lib, n, N, lo, hi):
    """Finite ones up to the largest, alone in their group and so with no sum to pass the range: those from near 2^128
    on are cut into their parts in another way."""
    values = _bits(n, lo, hi, 5)
    if hi == 128:
        values[0], values[1] = torch.finfo(F32).max, -torch.finfo(F32).max
        values[2], values[3] = 3.3895314e38, 3.35e38   # the largest bf16 value, one between the borders
        assert torch.isfinite(values).all() and (values.abs() > 3.3e38).any()
    for cplx in (False, True):
        for K in INPUTS:
            w = _powers(N, K, 32, cplx, -20, -4, codes=(1, 2))
            x, at = _one_a_row(values, K, F32)
            assert torch.equal(_product(x, w), _one_product(x, at, w))


@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("n,N", [(5, 200), (16, 4100), (16, 16500), (520, 1100), (700, 1900)])
def test_the_smallest_values(gpu_lib, n, N, cplx):
    """Exact from 2^-110 on, where the third part's last bit is bf16's smallest step of 2^-133; below it the nearest
    multiple of that, subnormal parts among them."""
    K = 200
    w = _powers(N, K, 32, cplx, 40, 60)
    x, at = _one_a_row(_bits(n, -110, -100, 21), K, F32)
    assert torch.equal(_product(x, w), _one_product(x, at, w))
    x, at = _one_a_row(_bits(n, -126, -110, 22), K, F32)
    near = (torch.round(x.double() * 2.0 ** 133) * 2.0 ** -133).to(F32)   # (24 bits at most: exact)
    assert torch.equal(_product(x, w), _one_product(near, at, w)) and (near != x).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,N", [(5, 40), (40, 1500), (520, 1100)])
def test_whole_groups_of_the_largest_magnitude(gpu_lib, n, N, group, cplx, dtype):
    """Rows just below 2^119 and weights of 6, all of one sign, under small scales: a group's sum is finite."""
    K = 256
    codes = torch.full((N, K // 2), 0xF7 if cplx else 0x77, device="cuda", dtype=torch.uint8)   # 6 and -6, or 6
    scales = torch.full((N, K // group), 2.0 ** -60, device="cuda", dtype=BF16)
    w = Weight4(codes, scales, K // 2 if cplx else K, group, complex=cplx)
    largest = torch.tensor((2 - 2.0 ** -(23 if dtype == F32 else 7)) * 2.0 ** 118, device="cuda", dtype=dtype)
    x = largest.expand(n, K).contiguous()
    y = _product(x, w)
    assert torch.isfinite(y).all()
    z = x.unflatten(1, (-1, 2)) if cplx else x
    _check(y.unflatten(1, (-1, 2)) if cplx else y, z, w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("K", INPUTS)
@pytest.mark.parametrize("n,N", CASES)
def test_infinities_and_nan_stay_in_their_rows(gpu_lib, n, N, K, cplx, dtype):
    w = _weight(N, K, 64, 6, cplx)
    x = _rows((n, K), dtype, 7)
    clean = _product(x, w)
    z = x.unflatten(1, (-1, 2)) if cplx else x
    _check(clean.unflatten(1, (-1, 2)) if cplx else clean, z, w)
    bad = x.clone()
    at = [0, n // 2, n - 1]
    bad[at[0], 5], bad[at[1], 150], bad[at[2], K - 1] = float("inf"), float("nan"), float("-inf")
    y = _product(bad, w)
    rest = [i for i in range(n) if i not in at]
    assert torch.equal(y[rest], clean[rest])
    want = bad[at].double() @ _matrix(w).T.contiguous()
    assert torch.equal(torch.isnan(y[at]), torch.isnan(want)) and torch.equal(torch.isinf(y[at]), torch.isinf(want))
    assert torch.equal(y[at].sign().nan_to_num(0), want.sign().nan_to_num(0).to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,N", CASES)
def test_layouts_of_the_rows(gpu_lib, n, N, dtype):
    for cplx in (False, True):
        for K in INPUTS:
            w = _weight(N, K, 32, 8, cplx)
            for name, v in _layouts(_rows((n, K), dtype, 9)).items():
                assert torch.equal(_product(v, w), _product(v.contiguous(), w)), (name, cplx, K)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cplx", [False, True])
@pytest.mark.parametrize("n,N", CASES)
def test_repeated_and_captured(gpu_lib, n, N, cplx, dtype):
    """The same bits on every call and at every replay, laid rows and others."""
    for K in INPUTS:
        w, b = _weight(N, K, 128, 10, cplx), _rows((N, 2) if cplx else (N,), F32, 11)
        x = _rows((n, K), dtype, 12)
        first = _product(x, w, b)
        assert all(torch.equal(_product(x, w, b), first) for _ in range(3))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _product(x, w, b)
        for seed in range(13, 17):
            x.copy_(_rows((n, K), dtype, seed))
            graph.replay()
            want = _product(x, w, b)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        del graph


@pytest.mark.parametrize("n,N", [(700, 6100), (2000, 4608)])
@pytest.mark.parametrize("K", [192, 360])
def test_blocks_of_half_the_outputs(gpu_lib, n, N, K):
    """bf16 prompts of complex weights with blocks behind the last whole round, every row and output."""
    for group in (32, 64):
        w = _weight(N, K, group, 18, True)
        x, tail = _rows((n, K // 2, 2), BF16, 19), _rows((5, K), BF16, 20)
        _check(complex_linear4(x, w), x, w)
        _check(complex_linear4(x, w, planes=True, tail=tail), x, w, tail=tail, planes=True)
