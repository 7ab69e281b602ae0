"""GlobalGATNet: embedding, layer norm and packed attention as a model uses them together,
with the edge-attention layers, against the same composition in float64 on the CPU."""
import pytest
import torch
import torch.nn.functional as F

from oracle import gat_layer_forward_differentiable

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def sub(params, prefix):
    return {k[len(prefix):]: v for k, v in params.items() if k.startswith(prefix)}


def norm(p, prefix, x):
    return F.layer_norm(x, (x.shape[1],), p[prefix + "weight"], p[prefix + "bias"])


def attend(q, k, v, qlens, klens):
    out, i, j = [], 0, 0
    for a, b in zip(qlens, klens):
        qs, ks, vs = (t.transpose(0, 1) for t in (q[i:i + a], k[j:j + b], v[j:j + b]))
        w = torch.softmax(qs @ ks.transpose(1, 2) * q.shape[2] ** -0.5, 2)
        out.append((w @ vs).transpose(0, 1))
        i, j = i + a, j + b
    return torch.cat(out)


def composition(p, data, lens):
    """float64 forward of GlobalGATNet from its state_dict."""
    h, d = 8, 8
    lin = lambda name, x: F.linear(x, p[name + ".weight"], p[name + ".bias"])  # noqa: E731
    x, ei = data.x.double(), data.edge_index
    deg = torch.bincount(ei[1], minlength=x.size(0)).clamp(max=63)
    x = F.elu(gat_layer_forward_differentiable(sub(p, "conv1."), x, ei, h, True)) + \
        0.1 * p["degree.weight"][deg]
    q, k, v = lin("qkv", norm(p, "norm1.", x)).view(-1, 3, h, d).unbind(1)
    x = x + lin("proj", attend(q, k, v, lens, lens).reshape(-1, h * d))
    x = x + F.elu(gat_layer_forward_differentiable(sub(p, "conv2."), norm(p, "norm2.", x), ei, h, True))
    k, v = lin("kv", norm(p, "norm3.", x)).view(-1, 2, h, d).unbind(1)
    n = len(lens)
    x = attend(p["query"].expand(n, h, d), k, v, [1] * n, lens)
    x = F.relu(lin("lin1", x.reshape(-1, h * d)))
    return F.log_softmax(lin("lin2", x), dim=1)


def batch(count, seed):
    from atmlgraphattentionnetworks_amd.datasets import collate, synthetic_cifar_graphs
    graphs = synthetic_cifar_graphs(count, seed=seed)
    return collate(graphs), [g.x.size(0) for g in graphs]


def test_output_and_gradients_match_the_composition():
    from atmlgraphattentionnetworks_amd.gatnet import GlobalGATNet
    torch.manual_seed(0)
    data, lens = batch(7, 3)
    model = GlobalGATNet(3)
    p = {k: v.detach().double().requires_grad_() for k, v in model.state_dict().items()}
    want = composition(p, data, lens)
    F.nll_loss(want, data.y).backward()
    model = model.to(DEV)
    out = model(data.to(DEV))
    F.nll_loss(out, data.y.to(DEV)).backward()
    # the edge layers meet their oracle to 1e-5 and its gradients to 1e-4 of their scale
    # (test_gpu_training); the operators between are float32 at 2^-24 a step
    assert float((out.detach().cpu().double() - want.detach()).abs().max()) < 5e-5
    for name, q in model.named_parameters():
        ref = p[name].grad
        scale = float(ref.abs().max()) + 1e-8
        assert float((q.grad.cpu().double() - ref).abs().max()) < 2e-4 * scale + 1e-7, name


def test_block_captured_and_replayed():
    """Embedding, layer norm, attention over graphs and its readout in one HIP graph, with
    their gradients: every replay gives the eager step's bits.  (The model's Linear layers
    stay outside: their bias gradients are torch sums, whose captured form goes wrong on
    replays after the first.)"""
    import atmlgraphattentionnetworks_amd as gat
    torch.manual_seed(1)
    lens = [85, 150, 1, 99]
    n = sum(lens)
    ptr = torch.tensor([0, 85, 235, 236, 335], dtype=torch.int32, device=DEV)
    each = torch.arange(5, dtype=torch.int32, device=DEV)
    ids = torch.randint(0, 64, (n,), device=DEV)
    table = torch.randn(64, 192, device=DEV, requires_grad=True)
    w, b = (torch.rand(192, device=DEV, requires_grad=True) for _ in range(2))
    query = torch.randn(4, 8, 8, device=DEV, requires_grad=True)
    g = torch.randn(4, 8, 8, device=DEV)

    def step():
        x = gat.layer_norm(gat.embedding(ids, table, 0.5), w, b)
        q, k, v = x.view(n, 3, 8, 8).unbind(1)
        y = gat.packed_attention(q, k, v, ptr)
        out = gat.packed_attention(query, k, y, each, ptr)
        return [out.detach(), *torch.autograd.grad(out, (table, w, b, query), g)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            table.normal_()
            ids.copy_(torch.randint(0, 64, (n,), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        for a, c in zip(kept, step()):
            assert torch.equal(a, c), k


def test_run_command_trains_it(capsys):
    from atmlgraphattentionnetworks_amd.run import main
    out = main(["graph", "--model", "global", "--train-graphs", "64", "--eval-graphs", "16",
                "--batch-size", "16", "--max-epochs", "2", "--runs", "1"])
    assert out["runs"] == 1 and 0.0 <= out["mean"] <= 1.0
