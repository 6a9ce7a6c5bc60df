"""CPU checks of the tied table's two ends (embedding lookup, token log
probabilities): refusals, argument structures, fake kernels."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from qllm2_amd import _lib
from test_abi import _header_struct_fields


@pytest.mark.parametrize("cname,pyname", [("qpam_embed_args", "EmbedArgs")])
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
