"""Products with weights of 4 bits and group scales (qpam_linear4), real ones and those
of a ComplexLinear: a decode step's projections and logits from a quarter of the bytes
of bf16 weights (an eighth of a ComplexLinear's as one real matrix, which holds every
weight twice).

ComplexLinear.forward (v11/complex_ops.py:165-172) runs two or four nn.Linear products;
here a complex weight is two neighbouring codes, read once.  A code is a 4-bit float
(sign, 2 bits of exponent, 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6), `group`
neighbouring codes of an output's row share a bf16 scale.  The products are exact and
summed in fp32; nothing but the result is rounded to the rows' dtype.  (A group's sum is
formed before its scale, of up to 64 inputs at once: rows of magnitudes below 2^119.  fp32
rows are cut into three bf16 parts: a value below 2^-110 counts as its nearest multiple of
2^-133, bf16's smallest step.)
"""

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib, _ops

__all__ = ["Weight4", "complex_linear4", "dequantize4", "linear4", "quantize4"]

GROUPS = (32, 64, 128)
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_ROWS, _COLS = 16, 64    # outputs and inputs of a block of the kernel's layout
_CODE = {torch.float32: _lib.QPAM_F32, torch.bfloat16: _lib.QPAM_BF16}


def _check_group(group):
    if group not in GROUPS:
        raise ValueError(f"qpam linear4: group {group} (one of {GROUPS})")


def _interleaved(weight, weight_imag):
    """[N, K] of a real weight, [N, 2K] of a complex one with its parts side by side."""
    if weight.dim() != 2 or not weight.numel() or not weight.is_floating_point():
        raise ValueError(f"qpam linear4: a weight [out, in] of real numbers expected, got {weight.dtype} {tuple(weight.shape)}")
    if weight_imag is None:
        return weight.detach().float()
    if weight_imag.shape != weight.shape or weight_imag.device != weight.device:
        raise ValueError(f"qpam linear4: imaginary parts {tuple(weight_imag.shape)} of weights {tuple(weight.shape)}")
    return torch.stack([weight.detach().float(), weight_imag.detach().float()], -1).flatten(1)


def quantize4(weight: Tensor, weight_imag: Optional[Tensor] = None, group: int = 32):
    """(codes, scales) of weights [N, K] (with weight_imag: complex weights, K doubled, re
    and im side by side): codes uint8 [N, ceil(K / 2)], the even column in the low half of a
    byte, scales bf16 [N, ceil(K / group)].

    A group's scale is its largest magnitude over 6, rounded to bf16, each weight the code
    nearest to it over the scale.  Weights that are not finite: ValueError."""
    _check_group(group)
    w = _interleaved(weight, weight_imag)
    if not bool(torch.isfinite(w).all()):
        raise ValueError("qpam linear4: weights that are not finite")
    n, k = w.shape
    groups = -(-k // group)
    w = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
    # (no higher than the bf16 below the largest fp32 value over 6, whose codes stay finite)
    scales = (w.abs().amax(-1) / 6).to(torch.bfloat16).clamp_max(170 * 2.0 ** 118)
    # (a scale that rounded to zero belongs to weights below 1e-39: codes of 0)
    inv = torch.where(scales == 0, 0.0, 1.0 / scales.float()).clamp_max(torch.finfo(torch.float32).max)
    r = (w * inv[..., None]).view(n, -1)
    borders = torch.tensor([(a + b) / 2 for a, b in zip(MAGNITUDES, MAGNITUDES[1:])], device=w.device)
    codes = torch.bucketize(r.abs(), borders).to(torch.uint8)
    codes = torch.where((r < 0) & (codes > 0), codes + 8, codes)[:, :k + k % 2]
    if k % 2:
        codes[:, k] = 0
    return (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous(), scales


def _check_codes(codes, scales, columns, group):
    _check_group(group)
    if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.shape[0] or columns < 1 \
            or codes.shape[1] != -(-columns // 2):
        raise ValueError(f"qpam linear4: codes must be uint8 [N, {-(-columns // 2)}] for {columns} columns, got {codes.dtype} "
                         f"{tuple(codes.shape)}")
    if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (codes.shape[0], -(-columns // group)):
        raise ValueError(f"qpam linear4: scales must be bfloat16 [{codes.shape[0]}, {-(-columns // group)}], got {scales.dtype} "
                         f"{tuple(scales.shape)}")
    if scales.device != codes.device:
        raise ValueError("qpam linear4: codes and scales must be on one device")


def dequantize4(codes: Tensor, scales: Tensor, columns: int, group: int = 32) -> Tensor:
    """The fp32 weights [N, columns] that quantize4's codes and scales stand for (exact)."""
    _check_codes(codes, scales, columns, group)
    values = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    idx = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :columns]
    return values[idx.int()] * scales.float().repeat_interleave(group, 1)[:, :columns]


def _scales_of(columns, group):
    """Steps along a row that have scales of their own in the layout, and how many each."""
    return -(-columns // max(group, _COLS)), max(1, _COLS // group)


class Weight4:
    """A weight [out_features, in_features] of 4-bit codes and group scales (quantize4's),
    laid out once for the kernel on the codes' device.  With `complex` the columns are
    2 * in_features, re and im side by side.  The codes and scales are copied; scales
    that are not finite: ValueError (a group of zeros times infinity would be zeros)."""

    def __init__(self, codes: Tensor, scales: Tensor, in_features: int, group: int = 32, complex: bool = False):
        columns = 2 * in_features if complex else in_features
        _check_codes(codes, scales, columns, group)
        if not bool(torch.isfinite(scales).all()):
            raise ValueError("qpam linear4: scales that are not finite")
        n = codes.shape[0]
        if n > 1 << 22 or in_features > 1 << 24:
            raise ValueError(f"qpam linear4: weight [{n}, {in_features}] too large (2^22, 2^24)")
        self.out_features, self.in_features, self.group, self.complex = n, int(in_features), int(group), bool(complex)
        tiles, blocks = -(-n // _ROWS), -(-columns // _COLS)
        pad = torch.nn.functional.pad
        if columns % 2:  # the half of a byte behind the last column
            codes = torch.cat([codes[:, :-1], codes[:, -1:] & 15], 1)
        c = pad(codes, (0, blocks * _COLS // 2 - codes.shape[1], 0, tiles * _ROWS - n))
        # [tile, output, block, step, quarter, byte] -> [tile, block, quarter, output, step, byte]
        self.codes = c.view(tiles, _ROWS, blocks, 2, 4, 4).permute(0, 2, 4, 1, 3, 5).contiguous().view(-1)
        per, g = _scales_of(columns, group)
        s = pad(scales, (0, per * g - scales.shape[1], 0, tiles * _ROWS - n))
        self.scales = s.view(tiles, _ROWS, per, g).permute(0, 2, 1, 3).contiguous().view(-1)

    @classmethod
    def quantize(cls, weight: Tensor, weight_imag: Optional[Tensor] = None, group: int = 32) -> "Weight4":
        """The nearest Weight4 of a weight [out, in] (with weight_imag: a complex one)."""
        codes, scales = quantize4(weight, weight_imag, group)
        return cls(codes, scales, weight.shape[1], group, complex=weight_imag is not None)

    def dequantize(self) -> Tensor:
        """The fp32 values: [out, in], complex [out, in, 2]."""
        n, columns = self.out_features, self.in_features * (2 if self.complex else 1)
        tiles, blocks = -(-n // _ROWS), -(-columns // _COLS)
        per, g = _scales_of(columns, self.group)
        c = self.codes.view(tiles, blocks, 4, _ROWS, 2, 4).permute(0, 3, 1, 4, 2, 5).reshape(tiles * _ROWS, -1)
        s = self.scales.view(tiles, per, _ROWS, g).permute(0, 2, 1, 3).reshape(tiles * _ROWS, -1)
        w = dequantize4(c[:n, :-(-columns // 2)], s[:n, :-(-columns // self.group)], columns, self.group)
        return w.view(n, self.in_features, 2) if self.complex else w


def _check_rows(x, codes, scales, n, k, is_complex, bias, planes, tail):
    if not (x.is_cuda and codes.is_cuda):
        raise ValueError("qpam linear4: tensors must be on the GPU (no CPU path in this library)")
    dev = x.device
    if codes.device != dev or scales.device != dev or (bias is not None and bias.device != dev) \
            or (tail is not None and tail.device != dev):
        raise ValueError("qpam linear4: rows, weight, bias and tail must be on one device")
    if x.dtype not in _CODE:
        raise ValueError(f"qpam linear4: rows must be float32 or bfloat16, got {x.dtype}")
    shape = x.shape
    if not (len(shape) > 1 and shape[-1] == 2 and shape[-2] == k if is_complex else len(shape) and shape[-1] == k):
        raise ValueError(f"qpam linear4: rows of {[k, 2] if is_complex else [k]} expected, got {tuple(shape)}")
    if bias is not None and tuple(bias.shape) != ((n, 2) if is_complex else (n,)):
        raise ValueError(f"qpam linear4: bias must be {[n, 2] if is_complex else [n]}, got {tuple(bias.shape)}")
    if tail is not None and (not planes or tail.dim() != 2 or tail.shape[1] != 2 * k or tail.dtype != x.dtype
                             or not 1 <= tail.shape[0] <= 4096):
        raise ValueError(f"qpam linear4: a tail stands behind planes and is [1 to 4096, {2 * k}] in the rows' dtype, got {tail.dtype} "
                         f"{tuple(tail.shape)}")


def _rows(x, columns, is_complex):
    """x as rows of unit column stride that do not overlap, and their stride; a copy where its strides do not give that."""
    if x.is_contiguous():
        return x, columns
    if is_complex:
        x = x.flatten(-2) if x.stride(-1) == 1 and x.stride(-2) == 2 else x.contiguous().flatten(-2)
    x = x.reshape(-1, columns)
    if (columns > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < columns):
        x = x.contiguous()
    return x, x.stride(0) if x.shape[0] > 1 else columns


def _product(x: Tensor, codes: Tensor, scales: Tensor, n: int, k: int, group: int, is_complex: bool, bias: Optional[Tensor],
             planes: bool, tail: Optional[Tensor]) -> Tensor:
    """[*, n] (complex [*, n, 2]; with planes [*, 2 n + tail rows]) in x's dtype."""
    _check_rows(x, codes, scales, n, k, is_complex, bias, planes, tail)
    z = 2 if is_complex else 1
    extra = 0 if tail is None else tail.shape[0]
    wide = z * n + extra
    out = x.new_empty((*x.shape[:-z], n, 2) if is_complex and not planes else (*x.shape[:-z], wide))
    count = out.numel() // wide
    if not count:
        return out
    rows, ldx = _rows(x, z * k, is_complex)
    if bias is not None and not (bias.dtype == torch.float32 and bias.is_contiguous()):
        bias = bias.detach().float().contiguous()
    if tail is not None and (tail.stride(1) != 1 or tail.stride(0) < 2 * k):
        tail = tail.contiguous()
    a = _lib.Linear4Args(count, n, k, group, is_complex, _CODE[x.dtype], planes, rows.data_ptr(), ldx, codes.data_ptr(),
                         scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), wide, extra,
                         None if tail is None else tail.data_ptr(), 0 if tail is None else tail.stride(0))
    L, dev = _lib.lib(), x.device
    nbytes = L.qpam_linear4_workspace_size(a)
    if nbytes:
        ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    status = _lib.launch(L.qpam_linear4, a, dev)
    if status:
        _lib.check(status, "qpam_linear4")
    return out


linear4_op = _ops.op("qpam::linear4", direct=True)(_product)


@linear4_op.register_fake
def _(x, codes, scales, n, k, group, is_complex, bias, planes, tail):
    z = 2 if is_complex else 1
    extra = 0 if tail is None else tail.shape[0]
    return x.new_empty(*x.shape[:-z], *((n, 2) if is_complex and not planes else (z * n + extra,)))


def _refuse_gradients(x, bias, tail):
    if (x.requires_grad or (bias is not None and bias.requires_grad) or (tail is not None and tail.requires_grad)) \
            and torch.is_grad_enabled():
        raise ValueError("qpam linear4: products with 4-bit weights have no gradient (call under torch.no_grad())")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None
                                              for t in (x, bias, tail)):
        raise ValueError("qpam linear4: products with 4-bit weights have no gradient, in forward mode neither")


def linear4(x: Tensor, weight: Weight4, bias: Optional[Tensor] = None) -> Tensor:
    """x [..., in] times a real Weight4: [..., out] in x's dtype (float32 or bfloat16, any
    strides; fp32 sums, one rounding).  bias [out].  No gradient, in either mode (ValueError)."""
    if weight.complex:
        raise ValueError("qpam linear4: a complex weight (complex_linear4)")
    _refuse_gradients(x, bias, None)
    return linear4_op(x, weight.codes, weight.scales, weight.out_features, weight.in_features, weight.group, False, bias, False,
                      None)


def complex_linear4(x: Tensor, weight: Weight4, bias: Optional[Tensor] = None, planes: bool = False,
                    tail: Optional[Tensor] = None) -> Tensor:
    """x [..., in, 2] times a complex Weight4, as ComplexLinear.forward
    (v11/complex_ops.py:165-172): [..., out, 2] in x's dtype.  bias [out, 2].

    planes: [..., 2 out + T] instead, the real parts, the imaginary parts and the T real
    outputs x . tail[t] of a tail [T, 2 in] (re and im side by side, x's dtype): outputs
    whose weights stay whole, as a PAM layer's decay logits beside its q, k, v.  No gradient."""
    if not weight.complex:
        raise ValueError("qpam linear4: a real weight (linear4)")
    _refuse_gradients(x, bias, tail)
    return linear4_op(x, weight.codes, weight.scales, weight.out_features, weight.in_features, weight.group, True, bias, planes,
                      tail)
