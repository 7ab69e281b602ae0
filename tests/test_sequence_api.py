"""What the packed-sequence operators refuse, without a GPU: the Python checks and the
library's own argument checks, which answer before any launch."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    import atmlgraphattentionnetworks_amd as gat
    x, ids = torch.randn(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        gat.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        gat.embedding(ids, x)
    with pytest.raises(TypeError):
        gat.layer_norm([1.0])
    with pytest.raises(ValueError):
        gat.Embedding(4, 8, padding_idx=4)
    with pytest.raises(ValueError):
        gat.LayerNorm(8)(torch.randn(3, 9))


def test_layer_norm_library_checks():
    from atmlgraphattentionnetworks_amd import _lib
    lib = _lib.load()

    def fwd(rows=4, cols=8, ld=8, dt=0, eps=1e-5, x=64, y=64):
        return lib.gat_layer_norm(x, ld, rows, cols, None, None, eps, y, ld, None, dt, None)
    assert fwd(rows=0) == _lib.GAT_OK
    for bad in (dict(rows=-1), dict(cols=0), dict(dt=3), dict(dt=-1), dict(eps=-1.0),
                dict(eps=float("nan")), dict(x=None), dict(y=None), dict(ld=7), dict(x=66)):
        assert fwd(**bad) == _lib.GAT_EINVAL, bad
    assert fwd(cols=16385, ld=16385) == _lib.GAT_EUNSUPPORTED
    assert fwd(cols=16382, ld=16382) == _lib.GAT_EUNSUPPORTED  # float32 rows off 16 bytes

    def bwd(rows=4, cols=8, ld=8, size=1 << 20, ws=64, dw=64, g=64, st=64):
        return lib.gat_layer_norm_backward(g, ld, 64, ld, rows, cols, None, st, 64, ld, dw, None, ws,
                                           size, 0, None)
    assert bwd(size=0) == _lib.GAT_EWORKSPACE
    for bad in (dict(g=None), dict(st=None), dict(ws=None), dict(rows=-1), dict(ld=7)):
        assert bwd(**bad) == _lib.GAT_EINVAL, bad
    out = ctypes.c_size_t()
    size = lib.gat_layer_norm_backward_workspace_size
    assert size(100, 64, 0, ctypes.byref(out)) == _lib.GAT_OK and out.value >= 2 * 64 * 4
    assert size(100, 20000, 0, ctypes.byref(out)) == _lib.GAT_EUNSUPPORTED
    assert size(100, 64, 0, None) == _lib.GAT_EINVAL


def test_embedding_library_checks():
    from atmlgraphattentionnetworks_amd import _lib
    lib = _lib.load()

    def fwd(tokens=4, vocab=8, cols=8, ld=8, dt=0, ids=64, w=64, out=64, ids64=1):
        return lib.gat_embedding(ids, ids64, tokens, w, ld, vocab, cols, 1.0, out, ld, dt, None)
    assert fwd(tokens=0) == _lib.GAT_OK
    for bad in (dict(tokens=-1), dict(tokens=(1 << 30) + 1), dict(vocab=0), dict(cols=0),
                dict(ld=7), dict(dt=5), dict(ids=None), dict(w=None), dict(out=None),
                dict(ids=68), dict(ids=66, ids64=0), dict(w=66)):
        assert fwd(**bad) == _lib.GAT_EINVAL, bad

    def grad(tokens=4, vocab=8, ld=8, size=1 << 24, ws=64, g=64, dw=64):
        return lib.gat_embedding_grad(64, 1, tokens, g, ld, vocab, 8, 1.0, -1, dw, ld, ws, size, 0,
                                      None)
    assert grad(size=16) == _lib.GAT_EWORKSPACE
    assert grad(ws=None) == _lib.GAT_EWORKSPACE
    for bad in (dict(ws=68), dict(g=None), dict(dw=None), dict(ld=7), dict(tokens=-1)):
        assert grad(**bad) == _lib.GAT_EINVAL, bad
    small = _lib.embedding_grad_workspace_size(100, 50, 8)
    assert 0 < small < _lib.embedding_grad_workspace_size(100000, 50, 8)
