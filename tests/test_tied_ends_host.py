"""CPU checks of the tied table's two ends (embedding lookup, token log
probabilities): refusals, argument structures, fake kernels."""

import ctypes
from typing import List

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qllm2_amd import _lib, _ops
from test_abi import _header_struct_fields


@pytest.mark.parametrize("cname,pyname", [("qpam_embed_args", "EmbedArgs"), ("qpam_logprobs_args", "LogprobsArgs"),
                                          ("qpam_linear_logprobs_args", "LinearLogprobsArgs")])
def test_ctypes_structs_match_header(cname, pyname):
    assert [f[0] for f in getattr(_lib, pyname)._fields_] == _header_struct_fields(cname)


def test_embedding_refusals():
    from qllm2_amd.embedding import complex_embedding
    ids, w = torch.zeros(3, dtype=torch.long), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="GPU"):
        complex_embedding(ids, w, w)
    with pytest.raises(ValueError, match="padding_idx"):
        complex_embedding(ids, w, w, padding_idx=5)
    with pytest.raises(ValueError, match="padding_idx"):
        complex_embedding(ids, w, w, padding_idx=-6)
    with FakeTensorMode():
        c = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        from qllm2_amd.embedding import _check
        bad = [
            (c(3, dtype=torch.float32), c(5, 4), c(5, 4), "int64 or int32"),
            (c(3, dtype=torch.int16), c(5, 4), c(5, 4), "int64 or int32"),
            (c(3, dtype=torch.long), c(5, 4), c(5, 6), "two tables"),
            (c(3, dtype=torch.long), c(5, 4, 1), c(5, 4, 1), "two tables"),
            (c(3, dtype=torch.long), c(0, 4), c(0, 4), "two tables"),
            (c(3, dtype=torch.long), c(5, 4), c(5, 4, dtype=torch.bfloat16), "float32"),
            (c(3, dtype=torch.long), c(5, 4, dtype=torch.float16), c(5, 4, dtype=torch.float16), "float32"),
            # sizes that 32 bits would wrap to small ones
            (c(3, dtype=torch.long), c(2 ** 32 + 5, 4), c(2 ** 32 + 5, 4), "too large"),
            (c(3, dtype=torch.long), c(5, 2 ** 32 + 4), c(5, 2 ** 32 + 4), "too large"),
        ]
        for ids, re, im, what in bad:
            with pytest.raises(ValueError, match=what):
                _check(ids, re, im)


def test_embedding_entry_errors_without_gpu():
    """Bad sizes, types, alignment and workspaces come back before any launch."""
    lib = _lib.lib()

    def err(fn, **kw):
        a = _lib.EmbedArgs()
        a.n, a.V, a.dim, a.dtype, a.ids = 4, 10, 8, _lib.QPAM_F32, 64
        a.re = a.im = a.out = a.dz = a.d_re = a.d_im = a.workspace = 4096
        a.ld_re = a.ld_im = 8
        a.padding_idx, a.workspace_bytes = -1, 1 << 20
        for k, v in kw.items():
            setattr(a, k, v)
        assert getattr(lib, fn)(ctypes.byref(a), None) == _lib.QPAM_ERR_ARG
        return lib.qpam_last_error().decode()

    assert "dtype" in err("qpam_embed_fwd", dtype=7)
    assert "ids" in err("qpam_embed_fwd", n=(1 << 30) + 1)
    assert "ids" in err("qpam_embed_bwd", n=-1)
    assert "null ids" in err("qpam_embed_fwd", ids=None)
    assert "table" in err("qpam_embed_fwd", V=0)
    assert "strides" in err("qpam_embed_fwd", ld_im=7)
    assert "null" in err("qpam_embed_fwd", out=None)
    assert "null" in err("qpam_embed_bwd", dz=None)
    assert "aligned" in err("qpam_embed_bwd", d_im=4104)
    assert "too many ids" in err("qpam_embed_bwd", n=1 << 28, dim=65, workspace_bytes=1 << 50)
    assert "workspace" in err("qpam_embed_bwd", workspace_bytes=16)
    a = _lib.EmbedArgs()
    a.n, a.dim = 0, 8
    assert lib.qpam_embed_bwd_workspace_size(ctypes.byref(a)) == 0
    a.n = (1 << 30) + 1
    assert lib.qpam_embed_bwd_workspace_size(ctypes.byref(a)) == 0


def test_embedding_fake_kernels():
    from qllm2_amd.embedding import complex_embedding, embed_bwd_op
    with FakeTensorMode():
        ids = torch.empty(2, 5, device="cuda", dtype=torch.int32)
        re, im = (torch.empty(9, 6, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
        z = complex_embedding(ids, re, im, scale=2.0, padding_idx=0)
        assert z.shape == (2, 5, 6, 2) and z.dtype == torch.bfloat16 and z.device.type == "cuda"
        for g in embed_bwd_op(ids, torch.empty_like(z), 9, 2.0, 0):
            assert g.shape == (9, 6) and g.dtype == torch.bfloat16


def test_token_logprobs_refusals():
    from qllm2_amd.token_logprobs import _check, token_logprobs
    with pytest.raises(ValueError, match="GPU"):
        token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    with FakeTensorMode():
        c = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        x, ids = c(4, 9), c(4, dtype=torch.long)
        for args, what in [
            ((c(4, 9, dtype=torch.float16), ids, 1.0, 0), "float32 or bfloat16"),
            ((c(4, 9, dtype=torch.float64), ids, 1.0, 0), "float32 or bfloat16"),
            ((x, c(4), 1.0, 0), "int64 or int32"),
            ((x, c(5, dtype=torch.long), 1.0, 0), "ids"),
            ((x, c(4, 1, dtype=torch.long), 1.0, 0), "ids"),
            ((c(4, 0), ids, 1.0, 0), "ids"),
            ((x, ids, 1.0, 10), "top_k"), ((x, ids, 1.0, -1), "top_k"), ((c(4, 100), ids, 1.0, 65), "top_k"),
            ((c(4, 2 ** 32 + 9), ids, 1.0, 0), "at most 2\\^30"),
            ((x, ids, 0.0, 0), "temperature"), ((x, ids, -1.0, 0), "temperature"),
            ((x, ids, float("inf"), 0), "temperature"), ((x, ids, float("nan"), 0), "temperature"),
        ]:
            with pytest.raises(ValueError, match=what):
                _check(*args)


def test_token_logprobs_entry_errors_without_gpu():
    lib = _lib.lib()

    def err(fn, **kw):
        a = _lib.LogprobsArgs()
        a.n, a.V, a.dtype, a.top_k, a.temperature, a.ld, a.ldd = 4, 10, _lib.QPAM_F32, 0, 1.0, 10, 10
        a.logits = a.ids = a.logprobs = a.entropy = a.stats = a.d_logits = 4096
        for k, v in kw.items():
            setattr(a, k, v)
        assert getattr(lib, fn)(ctypes.byref(a), None) == _lib.QPAM_ERR_ARG
        return lib.qpam_last_error().decode()

    for fn in ("qpam_logprobs_fwd", "qpam_logprobs_bwd"):
        assert "dtype" in err(fn, dtype=3)
        assert "sizes" in err(fn, V=0) and "sizes" in err(fn, n=-1)
        for t in (0.0, -1.0, float("inf"), float("nan")):
            assert "temperature" in err(fn, temperature=t)
        assert "top_k" in err(fn, top_k=11) and "top_k" in err(fn, top_k=65, V=100)
        assert "stride" in err(fn, ld=9) and "null" in err(fn, ids=None)
        assert "aligned" in err(fn, logits=4098)
    assert "null output" in err("qpam_logprobs_fwd", top_k=3)
    assert "stats" in err("qpam_logprobs_bwd", stats=None) and "stride" in err("qpam_logprobs_bwd", ldd=5)
    assert "g_top" in err("qpam_logprobs_bwd", g_top=4096)
    assert "aligned" in err("qpam_logprobs_bwd", d_logits=4097)


def test_token_logprobs_fake_kernels():
    from qllm2_amd.token_logprobs import logprobs_bwd_op, token_logprobs
    with FakeTensorMode():
        x = torch.empty(3, 4, 50, device="cuda", dtype=torch.bfloat16)
        ids = torch.empty(3, 4, device="cuda", dtype=torch.int32)
        r = token_logprobs(x, ids, top_k=6)
        assert [tuple(t.shape) for t in r] == [(3, 4), (3, 4), (3, 4, 6), (3, 4, 6)]
        assert r.top_ids.dtype == torch.int64 and r.top_logprobs.dtype == torch.float32
        f = torch.empty(12, device="cuda")
        d = logprobs_bwd_op(x.view(12, 50), ids.view(12).long(), f, torch.empty(12, 2, device="cuda"),
                            r.top_ids.view(12, 6), f, None, None, 1.0, -100)
        assert d.shape == (12, 50) and d.dtype == torch.bfloat16


def test_linear_token_logprobs_refusals():
    from qllm2_amd.token_logprobs import _check_linear, linear_token_logprobs
    with pytest.raises(ValueError, match="GPU"):
        linear_token_logprobs(torch.zeros(2, 32), torch.zeros(5, 32), torch.zeros(2, dtype=torch.long))
    with FakeTensorMode():
        c = lambda *s, **k: torch.empty(*s, device="cuda", **k)  # noqa: E731
        h, w, ids = c(4, 32), c(9, 32), c(4, dtype=torch.long)
        for args, what in [
            ((h.half(), w, ids, 1.0, 1), "float32 or bfloat16"), ((h, w.double(), ids, 1.0, 1), "float32 or bfloat16"),
            ((h, w, c(4), 1.0, 1), "int64 or int32"), ((h, w, c(5, dtype=torch.long), 1.0, 1), "hidden_rows"),
            ((h, c(9, 31), ids, 1.0, 1), "hidden_rows"), ((h, c(0, 32), ids, 1.0, 1), "hidden_rows"),
            ((h, c(1, 9, 32), ids, 1.0, 1), "hidden_rows"), ((h, w, ids, 1.0, 0), "chunk"),
            ((h, w, ids, 0.0, 1), "temperature"), ((h, w, ids, float("nan"), 1), "temperature"),
            ((h, c(2 ** 32 + 9, 32), ids, 1.0, 1), "at most 2\\^30"),
            ((c(2 ** 32 + 4, 32), w, c(2 ** 32 + 4, dtype=torch.long), 1.0, 1), "hidden rows"),
        ]:
            with pytest.raises(ValueError, match=what):
                _check_linear(*args)


def test_linear_token_logprobs_entry_errors_without_gpu():
    lib = _lib.lib()

    def err(fn, **kw):
        a = _lib.LinearLogprobsArgs()
        a.N, a.V, a.D, a.dtype, a.temperature, a.chunk, a.dw_out = 4, 10, 64, _lib.QPAM_F32, 1.0, 4, 1
        a.ldh = a.ldw = a.lddh = a.lddw = 64
        a.h = a.w = a.ids = a.logprobs = a.entropy = a.stats = a.dh = a.dw = a.workspace = 4096
        a.workspace_bytes = 1 << 30
        for k, v in kw.items():
            setattr(a, k, v)
        assert getattr(lib, fn)(ctypes.byref(a), None) == _lib.QPAM_ERR_ARG
        return lib.qpam_last_error().decode()

    for fn in ("qpam_linear_logprobs_fwd", "qpam_linear_logprobs_bwd"):
        assert "sizes" in err(fn, N=0) and "sizes" in err(fn, V=0) and "dtype" in err(fn, dtype=5)
        assert "multiple" in err(fn, D=63) and "null" in err(fn, ids=None) and "aligned" in err(fn, h=4100)
        assert "temperature" in err(fn, temperature=0.0) and "temperature" in err(fn, temperature=float("nan"))
        assert "stats" in err(fn, stats=None) and "workspace" in err(fn, workspace_bytes=64)
        assert "logprobs" in err(fn, logprobs=None) and "2^30" in err(fn, V=(1 << 30) + 1)
    assert "dh" in err("qpam_linear_logprobs_bwd", dh=None, dw=None) and "dw_out" in err("qpam_linear_logprobs_bwd", dw_out=0)
    assert "chunk" in err("qpam_linear_logprobs_bwd", chunk=0)
    assert "leading" in err("qpam_linear_logprobs_bwd", lddw=60)


def test_linear_token_logprobs_fake_kernels():
    from qllm2_amd.token_logprobs import linear_logprobs_bwd_op, linear_token_logprobs
    with FakeTensorMode():
        h = torch.empty(3, 4, 40, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(70, 40, device="cuda")
        r = linear_token_logprobs(h, w, torch.empty(3, 4, device="cuda", dtype=torch.int32))
        assert r.logprobs.shape == r.entropy.shape == (3, 4) and r.top_ids is None
        f = torch.empty(12, device="cuda")
        for fp32 in (False, True):
            dh, dw = linear_logprobs_bwd_op(h.view(12, 40), w.bfloat16(), f.long(), f, f, torch.empty(12, 2, device="cuda"),
                                            f, None, 1.0, 8, -100, fp32)
            assert dh.shape == (12, 40) and dw.shape == (70, 40)
            dh1, dw0 = linear_logprobs_bwd_op(h.view(12, 40), w.bfloat16(), f.long(), f, f, torch.empty(12, 2, device="cuda"),
                                              f, None, 1.0, 8, -100, fp32, True, False)
            assert dh1.shape == (12, 40) and dw0.shape == (0,) and dw0.dtype == dw.dtype
            assert dh.dtype == torch.bfloat16 and dw.dtype == (torch.float32 if fp32 else torch.bfloat16)


def _toy(a: torch.Tensor, b: torch.Tensor, s: float) -> List[torch.Tensor]:
    return [a * s + b, a * a]


def _wired(name, direct):
    f = _ops.op(name, direct=direct)(_toy)
    f.register_fake(lambda a, b, s: [torch.empty_like(a), torch.empty_like(a)])

    def setup(ctx, inputs, output):
        ctx.save_for_backward(inputs[0])
        ctx.s = inputs[2]
        ctx.set_materialize_grads(False)

    def back(ctx, grads):
        a, = ctx.saved_tensors
        with torch.no_grad():
            da = (grads[0] * ctx.s if grads[0] is not None else 0) + (2 * a * grads[1] if grads[1] is not None else 0)
        return da, grads[0], None

    f.register_autograd(back, setup_context=setup)
    return f


def test_direct_operators_equal_the_dispatched_ones():
    """op(direct=True): same values and gradients outside the dispatcher; every listener
    of the dispatcher still sees the operator."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    direct, plain = _wired("qpam::t_direct", True), _wired("qpam::t_dispatched", False)
    g = torch.Generator().manual_seed(1)
    res = []
    for f in (direct, plain):
        g.manual_seed(1)
        a, b = (torch.randn(4, 3, generator=g, requires_grad=True) for _ in range(2))
        y = f(a, b, 1.5)
        assert [t.requires_grad for t in y] == [True, True] and type(y) is list
        gs = torch.autograd.grad(y, [a, b], [torch.ones(4, 3), torch.full((4, 3), 2.0)], retain_graph=True)
        first, = torch.autograd.grad(y[0].sum(), [a])
        with torch.no_grad():
            assert not f(a, b, 1.5)[0].requires_grad
        with torch.inference_mode():
            assert f(a, b, 1.5)[0].is_inference()
        res.append([*y, *gs, first])
    for x, z in zip(*res):
        assert torch.equal(x, z)

    class Watch(TorchDispatchMode):
        seen = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen += func.namespace == "qpam"
            return func(*args, **(kwargs or {}))

    a = torch.ones(2)
    with Watch() as w:
        direct(a, a, 2.0)
    assert w.seen == 1
    with FakeTensorMode():
        assert direct(torch.empty(3), torch.empty(3), 2.0)[0].shape == (3,)
    assert "t_direct" in str(make_fx(lambda x: direct(x, x, 2.0)[0])(a).graph)
    with pytest.raises(Exception):
        torch.func.vmap(lambda x: direct(x, x, 2.0)[0])(torch.ones(3, 2))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(Exception):
        d = torch.autograd.forward_ad.make_dual(a.clone().requires_grad_(), a)
        direct(d, a, 2.0)
    assert torch.equal(torch.compile(lambda x: direct(x, x, 2.0)[0], backend="eager", fullgraph=True)(a), a * 3)


def test_linear_token_logprobs_columns_that_pad_to_the_limit():
    """Columns are padded to whole 32, and the padded rows stay below 2^22 apart."""
    from qllm2_amd.token_logprobs import MAX_D, MAX_STRIDE, _check_linear
    assert MAX_D % 32 == 0 and MAX_D <= MAX_STRIDE < MAX_D + 32
    with FakeTensorMode():
        h, w = (torch.empty(n, MAX_D + 1, device="cuda") for n in (4, 9))
        ids = torch.empty(4, device="cuda", dtype=torch.long)
        with pytest.raises(ValueError, match="columns"):
            _check_linear(h, w, ids, 1.0, 1)
        _check_linear(h[:, :-1], w[:, :-1], ids, 1.0, 1)


def test_model_decoder_refuses_host_ids_outside_the_vocabulary():
    """Before anything moves to the device."""
    from qllm2_amd.model_decode import ModelDecoder
    dec = object.__new__(ModelDecoder)
    dec.vocab, dec._embed = 300, [torch.empty(0)]
    assert dec._device_ids(torch.tensor([0, 299])).tolist() == [0, 299]
    assert dec._device_ids(torch.empty(0, dtype=torch.long)).numel() == 0
    for wrong in ([5, 300], [-1], [0, 2 ** 40]):
        for call in (dec.prefill, dec.admit, dec.score, lambda ids: dec.step(ids, None)):
            with pytest.raises(ValueError, match="vocabulary"):
                call(torch.tensor(wrong))
