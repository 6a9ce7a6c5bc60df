"""CPU checks of the 4-bit products and the pool copies: codes, layout, refusals, structures."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qllm2_amd import _lib
from qllm2_amd.linear4 import MAGNITUDES, Weight4, complex_linear4, dequantize4, linear4, quantize4
from tests.test_abi import _header_struct_fields


@pytest.mark.parametrize("cname,pyname", [("qpam_linear4_args", "Linear4Args"), ("qpam_slots_args", "SlotsArgs")])
def test_structs_match_the_header(cname, pyname):
    assert [f[0] for f in getattr(_lib, pyname)._fields_] == _header_struct_fields(cname)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (4, 64), (5, 65), (2, 300)])
def test_codes_are_the_nearest(shape, group):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1)) * torch.logspace(-3, 2, shape[0])[:, None]
    codes, scales = quantize4(w, group=group)
    assert codes.shape == (shape[0], -(-shape[1] // 2)) and scales.shape == (shape[0], -(-shape[1] // group))
    got = dequantize4(codes, scales, shape[1], group)
    s = scales.float().repeat_interleave(group, 1)[:, :shape[1]]
    values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES))
    best = (values * s[..., None] - w[..., None]).abs().amin(-1)
    # a weight on the border of two codes may fall on either by the quotient's rounding
    assert ((got - w).abs() <= best + 2.0 ** -22 * w.abs()).all()
    # the largest of a group is 6 scales, off by the scale's rounding
    top = torch.stack([c.abs().amax(1) for c in w.split(group, 1)], 1)
    assert ((scales.float() * 6 - top).abs() <= 2.0 ** -8 * top).all()


def test_codes_of_zeros_of_the_smallest_and_of_the_largest_values():
    w = torch.zeros(4, 64)
    w[1], w[2] = 1e-42, torch.finfo(torch.float32).max
    w[3, 5] = 1.0
    codes, scales = quantize4(w)
    got = dequantize4(codes, scales, 64)
    assert not got[0].any() and torch.isfinite(got[:2]).all() and torch.equal(got[3] != 0, w[3] != 0)
    assert ((got[2].double() / w[2].double() - 1).abs() <= 2.0 ** -8).all()
    with pytest.raises(ValueError, match="not finite"):
        quantize4(torch.tensor([[1.0, float("nan")]]))


def test_values_of_the_format_come_back():
    """Codes whose scale is a power of two and whose largest is 6: quantising their values gives them again."""
    g = torch.Generator().manual_seed(2)
    idx = torch.randint(0, 16, (7, 96), generator=g)
    idx[:, ::32] = 7
    idx[idx == 8] = 0   # minus zero is a code no weight gets
    codes = (idx[:, 0::2] | idx[:, 1::2] << 4).to(torch.uint8)
    scales = torch.exp2(torch.randint(-20, 20, (7, 3), generator=g).float()).to(torch.bfloat16)
    again, s = quantize4(dequantize4(codes, scales, 96))
    assert torch.equal(again, codes) and torch.equal(s, scales)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (40, 65), (5, 300)])
def test_layout_and_back(n, k, group):
    for z in (1, 2):
        g = torch.Generator().manual_seed(3)
        codes = torch.randint(0, 256, (n, -(-k * z // 2)), generator=g, dtype=torch.uint8)
        scales = torch.randn(n, -(-k * z // group), generator=g).to(torch.bfloat16)
        w = Weight4(codes, scales, k, group, complex=z == 2)
        tiles, blocks = -(-n // 16), -(-k * z // 64)
        assert w.codes.numel() == tiles * blocks * 512
        assert w.scales.numel() == tiles * 16 * (-(-k * z // 128) if group == 128 else blocks * 64 // group)
        assert torch.equal(w.dequantize().reshape(n, -1), dequantize4(codes, scales, k * z, group))
        # the places that the header names: output r, input 32 s + 8 q + 2 b of a block
        r, c = n - 1, k * z - 1
        at = ((r // 16) * blocks + c // 64) * 512 + 8 * (16 * (c % 32 // 8) + r % 16) + 4 * (c % 64 // 32) + c % 8 // 2
        assert int(w.codes[at] >> 4 * (c % 2)) & 15 == int(codes[r, c // 2] >> 4 * (c % 2)) & 15
        per, each = (-(-k * z // 128), 1) if group == 128 else (blocks, 64 // group)
        at = (((r // 16) * per + c // (group * each)) * 16 + r % 16) * each + c // group % each
        assert w.scales[at] == scales[r, c // group]
        if c % 2 == 0:
            at = ((r // 16) * blocks + c // 64) * 512 + 8 * (16 * (c % 32 // 8) + r % 16) + 4 * (c % 64 // 32) + c % 8 // 2
            assert int(w.codes[at]) >> 4 == 0


def test_complex_weights():
    g = torch.Generator().manual_seed(4)
    re, im = torch.randn(6, 50, generator=g), torch.randn(6, 50, generator=g)
    w = Weight4.quantize(re, im)
    codes, scales = quantize4(re, im)
    assert w.complex and w.in_features == 50 and codes.shape == (6, 50) and scales.shape == (6, 4)
    pair = torch.stack([re, im], -1)
    step = torch.cat([c.abs().amax(1, keepdim=True).expand_as(c) for c in pair.flatten(1).split(32, 1)], 1).view_as(pair) / 6
    assert ((w.dequantize() - pair).abs() <= 1.02 * step).all()


def test_weight_refusals():
    ok = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    Weight4(*ok, 32)
    for bad, what in [((ok[0].int(), ok[1], 32), "uint8"), ((ok[0], ok[1], 34), "uint8"), ((ok[0], ok[1].float(), 32), "bfloat16"),
                      ((ok[0], ok[1][:3], 32), "bfloat16"), ((ok[0], ok[1], 32, 48), "group"), ((ok[0][:0], ok[1][:0], 32), "uint8"),
                      ((ok[0], ok[1], 0), "uint8")]:
        with pytest.raises(ValueError, match=what):
            Weight4(*bad)
    with pytest.raises(ValueError, match="weight"):
        quantize4(torch.zeros(3))
    with pytest.raises(ValueError, match="weight"):
        quantize4(torch.zeros(3, 4, dtype=torch.int32))
    with pytest.raises(ValueError, match="imaginary"):
        quantize4(torch.zeros(3, 4), torch.zeros(3, 5))
    with pytest.raises(ValueError, match="group"):
        quantize4(torch.zeros(3, 4), group=16)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_scales_that_are_not_finite_are_refused(value):
    codes, scales = quantize4(torch.randn(4, 64))
    scales[2, 1] = value
    with pytest.raises(ValueError, match="finite"):
        Weight4(codes, scales, 64)


def test_product_refusals():
    w, c = Weight4.quantize(torch.randn(8, 32)), Weight4.quantize(torch.randn(8, 32), torch.randn(8, 32))
    with pytest.raises(ValueError, match="GPU"):
        linear4(torch.zeros(2, 32), w)
    with pytest.raises(ValueError, match="complex weight"):
        linear4(torch.zeros(2, 32), c)
    with pytest.raises(ValueError, match="real weight"):
        complex_linear4(torch.zeros(2, 32, 2), w)
    with pytest.raises(ValueError, match="no gradient"):
        linear4(torch.zeros(2, 32, requires_grad=True), w)
    with pytest.raises(ValueError, match="no gradient"):
        linear4(torch.zeros(2, 32), w, torch.zeros(8, requires_grad=True))
    from qllm2_amd.linear4 import _check_rows
    with FakeTensorMode():
        e = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        b16 = dict(dtype=torch.bfloat16)
        codes, scales = e(1024, dtype=torch.uint8), e(64, **b16)
        for args, what in [
            ((e(2, 32, dtype=torch.float16), codes, scales, 8, 32, False, None, False, None), "float32 or bfloat16"),
            ((e(2, 31), codes, scales, 8, 32, False, None, False, None), "rows of"),
            ((e(2, 32), codes, scales, 8, 32, True, None, False, None), "rows of"),
            ((e(2), codes, scales, 8, 1, True, None, False, None), "rows of"),
            ((e(2, 32), codes, scales, 8, 32, False, e(7), False, None), "bias"),
            ((e(2, 32, 2), codes, scales, 8, 32, True, e(8), False, None), "bias"),
            ((e(2, 32, 2), codes, scales, 8, 32, True, None, False, e(3, 64)), "tail"),
            ((e(2, 32, 2), codes, scales, 8, 32, True, None, True, e(3, 63)), "tail"),
            ((e(2, 32, 2), codes, scales, 8, 32, True, None, True, e(3, 64, **b16)), "tail"),
            ((e(2, 32, 2), codes, scales, 8, 32, True, None, True, e(0, 64)), "tail"),
        ]:
            with pytest.raises(ValueError, match=what):
                _check_rows(*args)


def test_product_entry_errors_without_gpu():
    lib = _lib.lib()

    def err(**kw):
        a = _lib.Linear4Args()
        a.rows, a.n, a.k, a.group, a.dtype, a.ldx, a.ldy = 4, 10, 64, 32, _lib.QPAM_F32, 64, 10
        a.x = a.codes = a.scales = a.y = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        assert lib.qpam_linear4(ctypes.byref(a), None) == _lib.QPAM_ERR_ARG
        return lib.qpam_last_error().decode()

    assert "dtype" in err(dtype=7)
    assert "rows" in err(rows=-1)
    assert "sizes" in err(n=0) and "sizes" in err(k=(1 << 24) + 1) and "sizes" in err(k=0)
    assert "group" in err(group=16)
    assert "null" in err(x=None) and "null" in err(codes=None) and "null" in err(scales=None) and "null" in err(y=None)
    assert "aligned" in err(codes=4104) and "aligned" in err(scales=4098) and "aligned" in err(x=4098) and "aligned" in err(bias=4097)
    assert "strides" in err(ldx=63) and "strides" in err(ldy=9)
    assert "planes" in err(planes=1) and "planes" in err(tail_n=2, tail=4096)
    assert "tail" in err(tail_n=5000, is_complex=1, planes=1)
    z = dict(is_complex=1, k=32, ldx=64, ldy=25)
    assert "tail" in err(tail_n=2, tail=4096, ld_tail=64, **z)
    assert "null" in err(planes=1, tail_n=2, ld_tail=64, **z)
    assert "strides" in err(planes=1, tail_n=2, tail=4096, ld_tail=63, **z)
    a = _lib.Linear4Args()
    a.n, a.k, a.group = 10, 64, 32
    assert lib.qpam_linear4(ctypes.byref(a), None) == 0   # no rows: nothing to do


def test_copy_refusals():
    from qllm2_amd.decode import copy_slots
    with pytest.raises(ValueError, match="GPU"):
        copy_slots(torch.zeros(4, 8), [0], [1])
    with FakeTensorMode():
        e = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        ok, ids = e(4, 8), e(2, dtype=torch.int32)
        for args, kw, what in [
            ((e(4, 8, dtype=torch.bfloat16), [0], [1]), {}, "state"),
            ((e(4), [0], [1]), {}, "state"),
            ((e(8, 4).t(), [0], [1]), {}, "state"),
            ((e(1, 8).expand(4, 8), [0], [1]), {}, "state"),
            ((ok, [0], [1]), dict(pos=e(4)), "pos"),
            ((ok, [0], [1]), dict(pos=e(5, dtype=torch.int32)), "pos"),
            ((ok, [0], [1]), dict(pos=e(8, dtype=torch.int32)[::2]), "pos"),
            ((ok, [0], ids), {}, "both host lists or both"),
            ((ok, ids, [0, 1]), {}, "both host lists or both"),
            ((ok, ids, e(3, dtype=torch.int32)), {}, "lengths"),
            ((ok, ids, e(2)), {}, "int32 or int64"),
            ((ok, ids, e(1, 2, dtype=torch.int32)), {}, "int32 or int64"),
            ((ok, [0, 1], [1]), {}, "lengths"),
            ((ok, [4], [1]), {}, "outside"),
            ((ok, [-2], [1]), {}, "outside"),
            ((ok, [0], [4]), {}, "outside"),
            ((ok, [0], [-1]), {}, "outside"),
            ((ok, [0, 2], [1, 1]), {}, "twice"),
            ((ok, e(5000, dtype=torch.int32), e(5000, dtype=torch.int32)), {}, "at most 4096"),
            ((e(9000, 8), list(range(1, 5001)), list(range(5000))), {}, "at most 4096"),
        ]:
            with pytest.raises(ValueError, match=what):
                copy_slots(*args, **kw)


def test_copy_entry_errors_without_gpu():
    lib = _lib.lib()
    ids = (ctypes.c_int32 * 600)(*range(600))

    def err(**kw):
        a = _lib.SlotsArgs()
        a.state, a.slot_bytes, a.page_bytes, a.n_slots, a.count = 4096, 64, 64, 8, 2
        a.src = a.dst = ctypes.addressof(ids)
        a.host_lists = 1
        for k, v in kw.items():
            setattr(a, k, v)
        assert lib.qpam_copy_slots(ctypes.byref(a), None) == _lib.QPAM_ERR_ARG
        return lib.qpam_last_error().decode()

    assert "slots" in err(n_slots=0) and "moves" in err(count=-1)
    assert "multiples" in err(page_bytes=0) and "multiples" in err(page_bytes=6) and "multiples" in err(slot_bytes=66)
    assert "overlap" in err(slot_bytes=60)
    assert "at most" in err(count=449) and "at most" in err(count=5000, host_lists=0)
    assert "null" in err(state=None) and "null" in err(src=None) and "null" in err(dst=None)
    assert "aligned" in err(state=4098) and "aligned" in err(pos=4098)
    a = _lib.SlotsArgs()
    a.n_slots, a.page_bytes, a.slot_bytes = 8, 64, 64
    assert lib.qpam_copy_slots(ctypes.byref(a), None) == 0   # no moves


def test_decoder_options_are_checked():
    from qllm2_amd.engine import check_weight_bits
    for bits, group, what in [(8, 32, "4-bit"), (4, 16, "weight_group"), (None, 100, "weight_group")]:
        with pytest.raises(ValueError, match=what):
            check_weight_bits("ModelDecoder", bits, group)
