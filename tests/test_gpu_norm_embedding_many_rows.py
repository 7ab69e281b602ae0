"""layer_norm and embedding where a group of lanes walks several rows, and layer_norm of
constant rows; the float64 definitions and tolerances are those of test_gpu_norm_embedding."""
import pytest
import torch

from test_gpu_norm_embedding import DEV, TYPES, U, close, embed_case, half_step, norm_case, ops

pytestmark = pytest.mark.gpu


# a launch has at most 256 x (resident workgroups a CU) workgroups of 256 / lanes rows each,
# the backward at most 1024 workgroups: more rows than that for every number of lanes
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(140000, 31), (90000, 63), (70003, 120), (40001, 300), (20011, 515),
                                       (9001, 1433), (8200, 2049), (4700, 4099), (2500, 8191)])
def test_norm_groups_of_several_rows(rows, cols, t):
    torch.manual_seed(cols)
    x = (torch.randn(rows, cols, device=DEV) * 1.5 + 0.3).to(t)
    w, b = ((torch.randn(cols, device=DEV) * 0.2 + k).to(t) for k in (1.0, 0.0))
    norm_case(x, w, b, torch.randn(rows, cols, device=DEV).to(t), what=f"{rows} {cols} {t}")


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(90000, 61), (9100, 1029)])
def test_norm_several_rows_of_a_view(rows, cols, t):
    torch.manual_seed(rows)
    big = torch.randn(rows, cols + 10, device=DEV).to(t)
    w, b = torch.rand(2, cols, device=DEV).to(t)
    g = torch.randn(rows, cols + 3, device=DEV).to(t)[:, 3:]
    norm_case(big[:, 5:5 + cols], w, b, g, what=f"{rows} {cols} {t}")

@pytest.mark.parametrize("t", TYPES, ids=str)
def test_norm_of_constant_rows_is_the_bias(t):
    """The mean of equal values whose sum float32 holds is that value, so nothing is left for
    1 / sqrt(eps) to enlarge."""
    gat = ops()
    for cols in list(range(1, 140)) + [255, 257, 511, 1000, 1433, 2049, 5001]:
        x = torch.tensor([[2.5], [1000.0], [-768.0], [0.0]], device=DEV).expand(4, cols).to(t)
        w, b = torch.rand(2, cols, device=DEV).to(t)
        leaf = x.detach().requires_grad_()
        y = gat.layer_norm(leaf, w, b)
        assert torch.equal(y, b.expand(4, cols)), cols
        g = torch.randn(4, cols, device=DEV).to(t)
        dx, = torch.autograd.grad(y, leaf, g)
        h = (g.double() * w.double()).cpu()
        r = (1.0 / torch.tensor(1e-5, dtype=torch.float32).double() ** 0.5)
        want = r * (h - h.mean(1, keepdim=True))
        e = r * ((cols + 16) * U * h.abs().mean(1, keepdim=True) + 8 * U * h.abs()) + 8 * U * want.abs()
        close(dx, want, e + half_step(t) * (want.abs() + e) + torch.finfo(t).tiny, f"{cols} dx")


# tables with enough rows that a group takes four of them, for each number of lanes, with
# some ids over and most under a piece
@pytest.mark.parametrize("vocab,cols,t", [(300000, 20, torch.float32), (150001, 60, torch.float32),
                                          (70001, 128, torch.float32), (40000, 250, torch.float32),
                                          (20000, 600, torch.float32), (270000, 64, torch.bfloat16),
                                          (140000, 100, torch.float16), (66000, 256, torch.bfloat16),
                                          (33001, 512, torch.bfloat16), (17001, 1000, torch.float16)],
                         ids=str)
def test_embedding_gradient_of_large_tables(vocab, cols, t):
    torch.manual_seed(vocab)
    tokens = 20000
    ids = torch.randint(0, vocab, (tokens,), device=DEV)
    ids[:3000] = vocab // 3
    ids[3000:3040] = vocab - 1
    ids[3040:6000] = torch.randint(vocab // 2, vocab // 2 + 300, (2960,), device=DEV)
    ids = ids[torch.randperm(tokens, device=DEV)]
    embed_case(ids, torch.randn(vocab, cols, device=DEV).to(t), torch.randn(tokens, cols, device=DEV).to(t),
               1.7, padding=5, what=f"{vocab} {cols} {t}")
