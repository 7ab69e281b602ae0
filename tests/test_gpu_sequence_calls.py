"""Ways of calling layer_norm, embedding and packed_attention beside a plain eager call, on
the GPU: traced, compiled, inside a forward-mode level, in place at the C-ABI."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def cases():
    import atmlgraphattentionnetworks_amd as gat
    torch.manual_seed(0)
    x, w, b = torch.randn(50, 40, device=DEV), torch.rand(40, device=DEV), torch.rand(40, device=DEV)
    ids = torch.randint(0, 30, (70,), device=DEV)
    table = torch.randn(30, 24, device=DEV)
    q, k, v = (torch.randn(33, 2, 20, device=DEV).bfloat16() for _ in range(3))
    ptr = torch.tensor([0, 10, 33], device=DEV)
    return [("layer_norm", lambda a, c, d: gat.layer_norm(a, c, d), (x, w, b)),
            ("embedding", lambda t: gat.embedding(ids, t, 2.0, 3), (table,)),
            ("packed_attention", lambda a, c, d: gat.packed_attention(a, c, d, ptr, causal=True), (q, k, v))]


def fresh(args):
    return tuple(torch.randn_like(a) for a in args)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_traced_calls_compute_on_their_inputs(which):
    name, call, args = cases()[which]
    for grad in (False, True):
        with torch.set_grad_enabled(grad), warnings.catch_warnings():
            warnings.simplefilter("ignore")  # the argument checks become constants
            leaves = tuple(a.clone().requires_grad_(grad) for a in args)
            traced = torch.jit.trace(call, leaves)
        for _ in range(3):
            with torch.set_grad_enabled(grad):
                new = tuple(a.requires_grad_(grad) for a in fresh(args))
                got, want = traced(*new), call(*new)
            assert torch.equal(got, want), name
            if grad:
                g = torch.randn_like(want)
                for a, c in zip(torch.autograd.grad(got, new, g), torch.autograd.grad(want, new, g)):
                    assert torch.equal(a, c), name
    if which != 2:  # another number of rows (the attention's ptr belongs to its trace)
        more = tuple(torch.cat((a, a)) if a.dim() == 2 else a for a in args)
        assert torch.equal(traced(*more), call(*more)), name


@pytest.mark.parametrize("which", [0, 1, 2])
def test_compiled_calls(which):
    name, call, args = cases()[which]
    compiled = torch.compile(lambda *a: call(*a) * 2, backend="eager")
    for grad in (False, True):
        new = tuple(a.requires_grad_(grad) for a in fresh(args))
        assert torch.equal(compiled(*new), call(*new) * 2), name


@pytest.mark.parametrize("which", [0, 1, 2])
def test_tangents_are_refused_wherever_they_are(which):
    from torch.autograd import forward_ad
    name, call, args = cases()[which]
    want = call(*args)
    with forward_ad.dual_level():
        assert torch.equal(call(*args), want)
        for i in range(len(args)):
            duals = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a
                     for j, a in enumerate(args)]
            with pytest.raises(NotImplementedError, match=name):
                call(*duals)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_recording_by_make_fx_is_refused(which):
    from torch.fx.experimental.proxy_tensor import make_fx
    name, call, args = cases()[which]
    with pytest.raises(RuntimeError, match="cannot be recorded"):
        make_fx(call)(*args)


def test_traced_layer_without_gradients_is_refused():
    import atmlgraphattentionnetworks_amd as gat
    layer = gat.GraphAttentionLayer(8, 4, dropout=0.0).to(DEV)
    x, edges = torch.randn(5, 8, device=DEV), torch.tensor([[0, 1, 2], [1, 2, 3]], device=DEV)
    with torch.no_grad():
        layer(x, edges)
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(layer, (x, edges))
        layer(x, edges)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("cols", [64, 300, 1433, 4100])
def test_layer_norm_in_place(cols, t):
    """gat_layer_norm with y = x: the same bits as with an output of its own."""
    import atmlgraphattentionnetworks_amd as gat
    from atmlgraphattentionnetworks_amd import _lib
    torch.manual_seed(cols)
    x = torch.randn(6000, cols, device=DEV).to(t)
    w, b = torch.randn(2, cols, device=DEV).to(t)
    want = gat.layer_norm(x, w, b)
    code = {torch.float32: _lib.GAT_F32, torch.bfloat16: _lib.GAT_BF16, torch.float16: _lib.GAT_F16}[t]
    _lib.check(_lib.load().gat_layer_norm(x.data_ptr(), cols, 6000, cols, w.data_ptr(), b.data_ptr(), 1e-5,
                                          x.data_ptr(), cols, None, code,
                                          torch.cuda.current_stream().cuda_stream), "gat_layer_norm")
    torch.cuda.synchronize()
    assert torch.equal(x, want)


def test_outputs_can_be_changed_in_place():
    """As torch's own operators allow it: the output is no view, and not kept for the backward."""
    import atmlgraphattentionnetworks_amd as gat
    torch.manual_seed(2)
    w = torch.rand(24, device=DEV)
    table = torch.randn(30, 24, device=DEV, requires_grad=True)
    for shape in ((24,), (5, 24), (2, 5, 24), (2, 3, 5, 24)):
        x, g = torch.randn(*shape, device=DEV, requires_grad=True), torch.randn(*shape, device=DEV)
        y = gat.layer_norm(x, w)
        z = gat.layer_norm(x, w)
        z += 1.0
        z.mul_(2.0)
        assert torch.equal(z, (y + 1.0) * 2.0), shape
        a, b = torch.autograd.grad(z, x, g)[0], torch.autograd.grad(y, x, g * 2.0)[0]
        assert torch.equal(a, b), shape
        ids = torch.randint(0, 30, shape[:-1], device=DEV)
        y, z = gat.embedding(ids, table), gat.embedding(ids, table)
        z += 1.0
        z.mul_(2.0)
        assert torch.equal(z, (y + 1.0) * 2.0), shape
        a, b = torch.autograd.grad(z, table, g)[0], torch.autograd.grad(y, table, g * 2.0)[0]
        assert torch.equal(a, b), shape
