"""Log probabilities of given tokens, with entropy and top alternatives.

token_logprobs reads rows of logits (qpam_logprobs_fwd / _bwd): what a serving
loop reports beside the tokens of ModelDecoder.step, and what policy gradients and
distillation differentiate.  The reference's V11LM.generate (v11/model.py:1207-1245)
forms these softmax rows to draw from them and returns none of it.

linear_token_logprobs gives the same values from the hidden rows and the tied table
(qpam_linear_logprobs_fwd / _bwd), with the operands of
fused_ce.fused_linear_cross_entropy and no logits in memory: scoring of whole
sequences, and policy-gradient steps with an entropy term.
"""

import ctypes
from typing import List, NamedTuple, Optional

import torch
import torch.nn.functional as F
from torch import Tensor

from . import _lib, _ops
from .fused_ce import _operands

__all__ = ["TokenLogprobs", "token_logprobs", "linear_token_logprobs"]

MAX_TOP_K = 64
MAX_VOCAB = 2 ** 30  # 32-bit sizes below
MAX_ROWS = 65535 * 128  # hidden rows: a launch's second axis
MAX_STRIDE = 2 ** 22 - 1  # elements between hidden rows and between table rows: 32-bit offsets in a tile
MAX_D = 2 ** 22 - 32     # ... and columns, padded to whole 32

_CODE = {torch.float32: _lib.QPAM_F32, torch.bfloat16: _lib.QPAM_BF16}


class TokenLogprobs(NamedTuple):
    """logprobs and entropy fp32 in the shape of ids; top_logprobs (fp32) and top_ids
    (int64) with a last axis of top_k, or None without top_k."""
    logprobs: Tensor
    entropy: Tensor
    top_logprobs: Optional[Tensor] = None
    top_ids: Optional[Tensor] = None


def _check_temperature(temperature, name):
    if not 1e-30 <= temperature <= 1e30:  # its reciprocal and what it scales stay in fp32's range
        raise ValueError(f"qpam {name}: temperature {temperature} outside 1e-30 .. 1e30")


def _check(logits, ids, temperature, top_k):
    if not (logits.is_cuda and ids.is_cuda and logits.device == ids.device):
        raise ValueError("qpam token_logprobs: logits and ids must be on one GPU (no CPU path in this library)")
    if logits.dtype not in _CODE:
        raise ValueError(f"qpam token_logprobs: logits must be float32 or bfloat16, got {logits.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"qpam token_logprobs: ids must be int64 or int32, got {ids.dtype}")
    if logits.dim() < 1 or logits.shape[:-1] != ids.shape or logits.shape[-1] < 1:
        raise ValueError(f"qpam token_logprobs: logits [..., V] and ids [...] expected, got {tuple(logits.shape)} and "
                         f"{tuple(ids.shape)}")
    if logits.shape[-1] > MAX_VOCAB:
        raise ValueError(f"qpam token_logprobs: rows of {logits.shape[-1]} logits (at most 2^30)")
    if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
        raise ValueError(f"qpam token_logprobs: top_k {top_k} outside 0 .. {min(MAX_TOP_K, logits.shape[-1])}")
    _check_temperature(temperature, "token_logprobs")


def _args(logits, ids, temperature, top_k, ignore_index, *more):
    """LogprobsArgs, `more` being the fields from `logprobs` on."""
    n, V = logits.shape
    return _lib.LogprobsArgs(n, V, _CODE[logits.dtype], top_k, temperature, logits.data_ptr(), max(logits.stride(0), V),
                             ids.data_ptr(), ignore_index, *more)


def _rows(logits):
    """[n, V] rows as the kernels read them: unit column stride, rows apart (one row: any stride)."""
    return logits if logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1] else logits.contiguous()


def _forward(logits: Tensor, ids: Tensor, temperature: float, top_k: int, ignore_index: int) -> List[Tensor]:
    """logits [n, V], ids [n] int64 -> [logprobs, entropy, stats [n, 2], top_logprobs [n, k], top_ids [n, k]]."""
    x, ids = _rows(logits), ids.contiguous()
    n, dev = x.shape[0], x.device
    lp, ent, stats = (torch.empty(s, device=dev, dtype=torch.float32) for s in ((n,), (n,), (n, 2)))
    top = torch.empty(n, top_k, device=dev, dtype=torch.float32)
    top_ids = torch.empty(n, top_k, device=dev, dtype=torch.int64)
    a = _args(x, ids, temperature, top_k, ignore_index, lp.data_ptr(), ent.data_ptr(), stats.data_ptr(), top.data_ptr(),
              top_ids.data_ptr())
    with _lib.device(dev):
        _lib.check(_lib.lib().qpam_logprobs_fwd(ctypes.byref(a), _lib.stream_ptr(dev)), "qpam_logprobs_fwd")
    return [lp, ent, stats, top, top_ids]


logprobs_fwd_op = _ops.op("qpam::logprobs_fwd", direct=True)(_forward)


@logprobs_fwd_op.register_fake
def _(logits, ids, temperature, top_k, ignore_index):
    n = logits.shape[0]
    f = lambda *s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    return [f(n), f(n), f(n, 2), f(n, top_k), logits.new_empty((n, top_k), dtype=torch.int64)]


def _gradient(logits: Tensor, ids: Tensor, entropy: Tensor, stats: Tensor, top_ids: Tensor, g_logprobs: Optional[Tensor],
              g_entropy: Optional[Tensor], g_top: Optional[Tensor], temperature: float, ignore_index: int) -> Tensor:
    """d logits [n, V] in the logits' dtype."""
    x, ids = _rows(logits), ids.contiguous()
    n, V = x.shape
    out = torch.empty(n, V, device=x.device, dtype=x.dtype)
    gs = [g if g is None else g.to(torch.float32).contiguous() for g in (g_logprobs, g_entropy, g_top)]
    a = _args(x, ids, temperature, top_ids.shape[1], ignore_index, None, entropy.data_ptr(), stats.data_ptr(), None,
              top_ids.data_ptr(), *(g if g is None else g.data_ptr() for g in gs), out.data_ptr(), V)
    with _lib.device(x.device):
        _lib.check(_lib.lib().qpam_logprobs_bwd(ctypes.byref(a), _lib.stream_ptr(x.device)), "qpam_logprobs_bwd")
    return out


logprobs_bwd_op = _ops.op("qpam::logprobs_bwd", direct=True)(_gradient)


@logprobs_bwd_op.register_fake
def _(logits, ids, entropy, stats, top_ids, g_logprobs, g_entropy, g_top, temperature, ignore_index):
    return logits.new_empty(logits.shape)


def _setup(ctx, inputs, output):
    logits, ids, ctx.temperature, ctx.top_k, ctx.ignore_index = inputs
    ctx.mark_non_differentiable(output[2], output[4])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(logits, ids, output[1], output[2], output[4])


def _backward(ctx, grads):
    g_lp, g_ent, _, g_top, _ = grads
    if g_lp is None and g_ent is None and g_top is None:
        return None, None, None, None, None
    if not ctx.top_k:
        g_top = None
    return logprobs_bwd_op(*ctx.saved_tensors, g_lp, g_ent, g_top, ctx.temperature, ctx.ignore_index), None, None, None, None


logprobs_fwd_op.register_autograd(_backward, setup_context=_setup)


def token_logprobs(logits: Tensor, ids: Tensor, temperature: float = 1.0, top_k: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Of p = softmax(logits / temperature) in each row: ln p of the given token, the
    entropy -sum p ln p, and the top_k (0 to 64) largest entries with their ids,
    equal logits by the lower id.

    logits [..., V] float32 or bfloat16 (rows of any stride), ids [...] int64 or
    int32.  A row whose id is ignore_index or outside [0, V) has log probability 0
    and its entropy and alternatives.  Logits of -inf are masked: probability 0; a
    row of nothing else has log probabilities -inf, entropy 0 and no gradient.  A
    row with NaN or +inf gives NaN.  Statistics are fp32.  Differentiable in
    logits through logprobs, entropy and top_logprobs (once: a second derivative
    raises); the gradient has the logits' dtype."""
    _check(logits, ids, temperature, top_k)
    shape = ids.shape
    flat = len(shape) == 1
    if not flat:
        logits, ids = logits.reshape(-1, logits.shape[-1]), ids.reshape(-1)
    lp, ent, _, top, top_ids = logprobs_fwd_op(logits, ids if ids.dtype == torch.int64 else ids.long(), float(temperature),
                                               top_k, ignore_index)
    if flat:
        return TokenLogprobs(lp, ent, top, top_ids) if top_k else TokenLogprobs(lp, ent)
    if not top_k:
        return TokenLogprobs(lp.view(shape), ent.view(shape))
    return TokenLogprobs(lp.view(shape), ent.view(shape), top.view(*shape, top_k), top_ids.view(*shape, top_k))


# ------------------------------------------------------------ from hidden rows

def _check_linear(hidden_rows, weight_matrix, ids, temperature, chunk):
    name = "linear_token_logprobs"
    if not (hidden_rows.is_cuda and hidden_rows.device == weight_matrix.device == ids.device):
        raise ValueError(f"qpam {name}: tensors must be on one GPU (no CPU path in this library)")
    if hidden_rows.dtype not in _CODE or weight_matrix.dtype not in _CODE:
        raise ValueError(f"qpam {name}: float32 or bfloat16 expected, got {hidden_rows.dtype} and {weight_matrix.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"qpam {name}: ids must be int64 or int32, got {ids.dtype}")
    if (hidden_rows.dim() < 1 or weight_matrix.dim() != 2 or hidden_rows.shape[-1] != weight_matrix.shape[1]
            or hidden_rows.shape[:-1] != ids.shape or not weight_matrix.numel()):
        raise ValueError(f"qpam {name}: hidden_rows [..., D], weight_matrix [V, D] and ids [...] expected, got "
                         f"{tuple(hidden_rows.shape)}, {tuple(weight_matrix.shape)} and {tuple(ids.shape)}")
    if weight_matrix.shape[0] > MAX_VOCAB or weight_matrix.shape[1] > MAX_D or ids.numel() > MAX_ROWS:
        raise ValueError(f"qpam {name}: at most 2^30 table rows, {MAX_ROWS} hidden rows, {MAX_D} columns, got "
                         f"{tuple(weight_matrix.shape)} and {ids.numel()}")
    if chunk < 1:
        raise ValueError(f"qpam {name}: chunk {chunk} must be at least 1")
    _check_temperature(temperature, name)


def _linear_args(h, w, dtype, ids, logprobs, entropy, stats, temperature, ignore_index):
    a = _lib.LinearLogprobsArgs()
    a.N, a.V, a.D, a.dtype, a.temperature = h.shape[0], w.shape[0], h.shape[1], dtype, temperature
    a.h, a.ldh, a.w, a.ldw = h.data_ptr(), h.stride(0), w.data_ptr(), w.stride(0)
    a.ids, a.ignore_index = ids.data_ptr(), ignore_index
    a.logprobs, a.entropy, a.stats = logprobs.data_ptr(), entropy.data_ptr(), stats.data_ptr()
    return a


def _workspace(a, nbytes, device):
    ws = torch.empty(nbytes, device=device, dtype=torch.uint8)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    return ws


def _linear_forward(hidden_rows: Tensor, weight_matrix: Tensor, weight_copy: Optional[Tensor], ids: Tensor,
                    temperature: float, chunk: int, ignore_index: int) -> List[Tensor]:
    """hidden_rows [n, D], ids [n] int64 -> [logprobs, entropy, stats [n, 2]]; weight_copy:
    an fp32 weight_matrix in the rows' bf16."""
    h, w, dtype = _operands(hidden_rows, weight_matrix if weight_copy is None else weight_copy, MAX_STRIDE)
    n, dev = h.shape[0], h.device
    lp, ent, stats = (torch.empty(s, device=dev, dtype=torch.float32) for s in ((n,), (n,), (n, 2)))
    if n:
        ids = ids.contiguous()
        a = _linear_args(h, w, dtype, ids, lp, ent, stats, temperature, ignore_index)
        L = _lib.lib()
        ws = _workspace(a, L.qpam_linear_logprobs_fwd_workspace_size(ctypes.byref(a)), dev)  # noqa: F841
        with _lib.device(dev):
            _lib.check(L.qpam_linear_logprobs_fwd(ctypes.byref(a), _lib.stream_ptr(dev)), "qpam_linear_logprobs_fwd")
    return [lp, ent, stats]


linear_logprobs_fwd_op = _ops.op("qpam::linear_logprobs_fwd", direct=True)(_linear_forward)


@linear_logprobs_fwd_op.register_fake
def _(hidden_rows, weight_matrix, weight_copy, ids, temperature, chunk, ignore_index):
    n = hidden_rows.shape[0]
    f = lambda *s: hidden_rows.new_empty(s, dtype=torch.float32)  # noqa: E731
    return [f(n), f(n), f(n, 2)]


def _linear_gradient(hidden_rows: Tensor, weight_matrix: Tensor, ids: Tensor, logprobs: Tensor, entropy: Tensor,
                     stats: Tensor, g_logprobs: Optional[Tensor], g_entropy: Optional[Tensor], temperature: float, chunk: int,
                     ignore_index: int, dw_fp32: bool, need_dh: bool = True, need_dw: bool = True) -> List[Tensor]:
    """[d hidden_rows, d weight_matrix] in the inputs' dtypes (d weight_matrix in fp32
    with dw_fp32); one that is not needed is an empty tensor."""
    h, w, dtype = _operands(hidden_rows, weight_matrix, MAX_STRIDE)
    n, dev = h.shape[0], h.device
    dw_fp32 = dw_fp32 or weight_matrix.dtype != w.dtype
    dh = torch.empty(h.shape if need_dh else 0, device=dev, dtype=h.dtype)
    dw = torch.empty(w.shape if need_dw else 0, device=dev, dtype=torch.float32 if dw_fp32 else w.dtype)
    if not n or not (need_dh or need_dw):
        return [dh.to(hidden_rows.dtype), dw.zero_()]
    ids = ids.contiguous()
    gs = [g if g is None else g.to(torch.float32).contiguous() for g in (g_logprobs, g_entropy)]
    a = _linear_args(h, w, dtype, ids, logprobs, entropy, stats, temperature, ignore_index)
    a.g_logprobs, a.g_entropy = (g if g is None else g.data_ptr() for g in gs)
    if need_dh:
        a.dh, a.lddh = dh.data_ptr(), dh.stride(0)
    if need_dw:
        a.dw, a.lddw = dw.data_ptr(), dw.stride(0)
    a.chunk, a.dw_out = min(chunk, n), 2 if dw_fp32 else 1
    L = _lib.lib()
    ws = _workspace(a, L.qpam_linear_logprobs_bwd_workspace_size(ctypes.byref(a)), dev)  # noqa: F841
    with _lib.device(dev):
        _lib.check(L.qpam_linear_logprobs_bwd(ctypes.byref(a), _lib.stream_ptr(dev)), "qpam_linear_logprobs_bwd")
    return [dh.to(hidden_rows.dtype), dw]


linear_logprobs_bwd_op = _ops.op("qpam::linear_logprobs_bwd", direct=True)(_linear_gradient)


@linear_logprobs_bwd_op.register_fake
def _(hidden_rows, weight_matrix, ids, logprobs, entropy, stats, g_logprobs, g_entropy, temperature, chunk, ignore_index,
      dw_fp32, need_dh=True, need_dw=True):
    return [hidden_rows.new_empty(hidden_rows.shape if need_dh else 0),
            weight_matrix.new_empty(weight_matrix.shape if need_dw else 0,
                                    dtype=torch.float32 if dw_fp32 else weight_matrix.dtype)]


def _linear_setup(ctx, inputs, output):
    hidden_rows, weight_matrix, weight_copy, ids, ctx.temperature, ctx.chunk, ctx.ignore_index = inputs
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)
    ctx.master = weight_copy is not None
    ctx.save_for_backward(hidden_rows, weight_copy if ctx.master else weight_matrix, ids, *output)


def _linear_backward(ctx, grads):
    g_lp, g_ent, _ = grads
    if g_lp is None and g_ent is None:
        return (None,) * 7
    need_dh, need_dw = ctx.needs_input_grad[:2]
    dh, dw = linear_logprobs_bwd_op(*ctx.saved_tensors, g_lp, g_ent, ctx.temperature, ctx.chunk, ctx.ignore_index,
                                    ctx.master, need_dh, need_dw)
    return dh if need_dh else None, dw if need_dw else None, None, None, None, None, None


linear_logprobs_fwd_op.register_autograd(_linear_backward, setup_context=_linear_setup)


def linear_token_logprobs(hidden_rows: Tensor, weight_matrix: Tensor, ids: Tensor, temperature: float = 1.0,
                          chunk: int = 4096, ignore_index: int = -100) -> TokenLogprobs:
    """token_logprobs(hidden_rows @ weight_matrix.T, ids, temperature) without the
    logits in memory: log probabilities and entropies of rows [..., D] against a table
    [V, D], float32 or bfloat16, ids [...] int64 or int32.

    Differentiable in hidden_rows and weight_matrix (once: a second derivative
    raises).  If either operand is bf16, both enter the products as bf16, with fp32
    sums; the logits' gradient is rounded to bf16 before the two products that give
    the operands' gradients, but for its entries at the given ids, most rows' largest,
    which join them in fp32.  The gradients have the operands' dtypes; that of an fp32
    weight_matrix with bf16 rows (a master table) leaves from the fp32 sums.  chunk
    bounds the backward's memory as in fused_ce.fused_linear_cross_entropy.  D off the
    multiples of 32 pads both operands by copies; operands whose rows share memory, start
    off 16 bytes or lie 2^22 elements apart are copied, too.  Log probabilities are at
    most 0.  Alternatives need the logits: token_logprobs gives them."""
    _check_linear(hidden_rows, weight_matrix, ids, temperature, chunk)
    D = hidden_rows.shape[-1]
    h, w = hidden_rows.reshape(-1, D), weight_matrix
    if D % 32:
        h, w = F.pad(h, (0, -D % 32)), F.pad(w, (0, -D % 32))
    copy = w.detach().to(torch.bfloat16) if w.dtype == torch.float32 and h.dtype == torch.bfloat16 else None
    lp, ent, _ = linear_logprobs_fwd_op(h, w, copy, ids.reshape(-1).long(), float(temperature), chunk, ignore_index)
    return TokenLogprobs(lp.view(ids.shape), ent.view(ids.shape))
