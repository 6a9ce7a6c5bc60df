"""The complex embedding lookup with scaling, and its gradient by sorted tokens
(qpam_embed_fwd / qpam_embed_bwd).

ComplexEmbed.forward (v11/complex_ops.py:223-235) stacks two nn.Embedding rows;
here one launch reads both tables' rows and writes the scaled, interleaved
[..., dim, 2] result.  The gradient of both tables comes from the token positions
in sorted order: fp32 sums in ascending position, rounded once, the same bits on
every call.
"""

import ctypes
from typing import List, Optional

import torch
from torch import Tensor

from . import _lib, _ops

__all__ = ["complex_embedding"]

_CODE = {torch.float32: _lib.QPAM_F32, torch.bfloat16: _lib.QPAM_BF16}


def _check(ids, weight_real, weight_imag):
    if not (weight_real.is_cuda and weight_imag.is_cuda and ids.is_cuda):
        raise ValueError("qpam complex_embedding: tensors must be on the GPU (no CPU path in this library)")
    if not (ids.device == weight_real.device == weight_imag.device):
        raise ValueError("qpam complex_embedding: ids and tables must be on one device")
    if weight_real.dim() != 2 or weight_real.shape != weight_imag.shape or not weight_real.numel():
        raise ValueError(f"qpam complex_embedding: two tables [V, dim] expected, got {tuple(weight_real.shape)} and "
                         f"{tuple(weight_imag.shape)}")
    if weight_real.shape[0] >= 2 ** 30 or weight_real.shape[1] > 2 ** 20:  # 32-bit sizes below
        raise ValueError(f"qpam complex_embedding: table {tuple(weight_real.shape)} too large (below 2^30 rows of at most 2^20)")
    if weight_real.dtype not in _CODE or weight_real.dtype != weight_imag.dtype:
        raise ValueError("qpam complex_embedding: both tables must be float32 or both bfloat16, got "
                         f"{weight_real.dtype} and {weight_imag.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"qpam complex_embedding: ids must be int64 or int32, got {ids.dtype}")


def _args(ids, V, dim, dtype, padding_idx, scale, *more):
    """EmbedArgs, `more` being the fields from `outside` on."""
    return _lib.EmbedArgs(ids.numel(), V, dim, _CODE[dtype], ids.dtype == torch.int64, ids.data_ptr(), padding_idx, scale,
                          *more)


def _table(w):
    """w [V, dim] with its strides as the kernel reads them: columns apart, rows apart by their length; a copy
    where it is not (a transposed or expanded table)."""
    dim = w.shape[1]
    cs = w.stride(1) if dim > 1 else 1
    if cs < 1 or w.stride(0) <= (dim - 1) * cs:
        w, cs = w.contiguous(), 1
    return w, max(w.stride(0), dim), cs


def _lookup(ids: Tensor, weight_real: Tensor, weight_imag: Tensor, scale: float, padding_idx: int,
            outside: float = 0.0) -> Tensor:
    """[*ids.shape, dim, 2] in the tables' dtype."""
    _check(ids, weight_real, weight_imag)
    V, dim = weight_real.shape
    ids, (re, ld_re, cs_re), (im, ld_im, cs_im) = ids.contiguous(), _table(weight_real), _table(weight_imag)
    dev = re.device
    out = torch.empty(*ids.shape, dim, 2, device=dev, dtype=re.dtype)
    a = _args(ids, V, dim, re.dtype, padding_idx, scale, outside, re.data_ptr(), ld_re, cs_re, im.data_ptr(), ld_im, cs_im,
              out.data_ptr())
    with _lib.device(dev):
        _lib.check(_lib.lib().qpam_embed_fwd(ctypes.byref(a), _lib.stream_ptr(dev)), "qpam_embed_fwd")
    return out


embed_fwd_op = _ops.op("qpam::embed_fwd", direct=True)(_lookup)


@embed_fwd_op.register_fake
def _(ids, weight_real, weight_imag, scale, padding_idx, outside=0.0):
    return weight_real.new_empty(*ids.shape, weight_real.shape[1], 2)


def _gradient(ids: Tensor, dz: Tensor, num_embeddings: int, scale: float, padding_idx: int) -> List[Tensor]:
    """[d weight_real, d weight_imag], each [num_embeddings, dim] in dz's dtype."""
    dim = dz.shape[-2]
    ids, dz = ids.contiguous(), dz.contiguous()
    if dz.data_ptr() % 16:
        dz = dz.clone()
    grads = [torch.empty(num_embeddings, dim, device=dz.device, dtype=dz.dtype) for _ in range(2)]
    a = _args(ids, num_embeddings, dim, dz.dtype, padding_idx, scale, 0.0, None, 0, 0, None, 0, 0, None, dz.data_ptr(),
              grads[0].data_ptr(), grads[1].data_ptr())
    L = _lib.lib()
    nbytes = L.qpam_embed_bwd_workspace_size(ctypes.byref(a))
    ws = torch.empty(nbytes, device=dz.device, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    with _lib.device(dz.device):
        _lib.check(L.qpam_embed_bwd(ctypes.byref(a), _lib.stream_ptr(dz.device)), "qpam_embed_bwd")
    return grads


embed_bwd_op = _ops.op("qpam::embed_bwd", direct=True)(_gradient)


@embed_bwd_op.register_fake
def _(ids, dz, num_embeddings, scale, padding_idx):
    return [dz.new_empty(num_embeddings, dz.shape[-2]) for _ in range(2)]


def _setup(ctx, inputs, output):
    ids, weight_real, _, ctx.scale, ctx.padding_idx, _ = inputs
    ctx.save_for_backward(ids)
    ctx.num_embeddings, ctx.dtype = weight_real.shape[0], weight_real.dtype


def _backward(ctx, dz):
    if dz is None:
        return None, None, None, None, None, None
    ids, = ctx.saved_tensors
    d_re, d_im = embed_bwd_op(ids, dz.to(ctx.dtype), ctx.num_embeddings, ctx.scale, ctx.padding_idx)
    return None, d_re, d_im, None, None, None


embed_fwd_op.register_autograd(_backward, setup_context=_setup)


def complex_embedding(ids: Tensor, weight_real: Tensor, weight_imag: Tensor, scale: float = 1.0,
                      padding_idx: Optional[int] = None, outside: float = 0.0) -> Tensor:
    """scale * (weight_real[ids], weight_imag[ids]) as [*ids.shape, dim, 2] in the
    tables' dtype (float32 or bfloat16; products in fp32, rounded once).

    ids int64 or int32, any shape; tables [V, dim], rows and columns of any
    stride: those of one interleaved [V, dim, 2] are read where they stand.  An id
    outside [0, V) gives a row of `outside` (zeros; NaN where it must not pass for a
    token) and no gradient.  padding_idx (of [-V, V),
    as nn.Embedding's) is looked up like any id and gets no gradient.
    Differentiable in both tables (dense gradients, once: a second derivative
    raises), up to 2^27 ids, fewer by the 512-byte pieces of a table's row."""
    pad = -1
    if padding_idx is not None:
        V = weight_real.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"qpam complex_embedding: padding_idx {padding_idx} outside [-{V}, {V})")
        pad = padding_idx + V if padding_idx < 0 else padding_idx
    return embed_fwd_op(ids, weight_real, weight_imag, float(scale), pad, float(outside))
