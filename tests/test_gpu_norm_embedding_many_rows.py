"""layer_norm and embedding where a group of lanes walks several rows, and layer_norm of
constant rows; the float64 definitions and tolerances are those of test_gpu_norm_embedding."""
import pytest
import torch

from test_gpu_norm_embedding import (DEV, TYPES, U, close, embed_case, half_step, norm_case,
                                     norm_reference, ops)

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


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("cols", [7, 20, 64, 100, 300, 1030])
def test_norm_rows_of_huge_constants(cols, t):
    """Lanes outside a row have no part in it, whatever its mean: values whose product with
    1 / sqrt(eps) passes float32's range."""
    gat = ops()
    c = 2.0 ** 117  # cols times this is finite and their mean exact: deviations of 0
    x = torch.full((5, cols), c, device=DEV, dtype=t)
    x[1], x[3] = -c, torch.randn(cols, device=DEV).to(t)
    w, b = torch.rand(2, cols, device=DEV).to(t)
    g = torch.randn(5, cols, device=DEV).to(t)
    eps = 1e-12
    leaves = [p.detach().requires_grad_() for p in (x, w, b)]
    y = gat.layer_norm(*leaves, eps)
    got = [y, *torch.autograd.grad(y, leaves, g)]
    want = norm_reference(x.cpu(), w.cpu(), b.cpu(), eps, g.cpu())
    # of a constant row z = 0 exactly: dx = r (h - mean(h)), y = b
    h = (g.double() * w.double()).cpu()
    r = 1.0 / (torch.tensor(eps, dtype=torch.float32).double() ** 0.5)
    for i in (0, 1, 2, 4):
        assert torch.equal(y[i], leaves[2].detach())
        dx = r * (h[i] - h[i].mean())
        bound = r * ((cols + 16) * U * h[i].abs().mean() + 8 * U * h[i].abs()) + 8 * U * dx.abs()
        close(got[1][i], dx, bound + half_step(t) * (dx.abs() + bound), f"{cols} dx {i}")
    v, e = (p[3] for p in want[1])
    close(got[1][3], v, e + half_step(t) * (v.abs() + e), "dx of the ordinary row")
    db = g.double().sum(0).cpu()
    close(got[3], db, 45 * U * g.double().abs().sum(0).cpu() + half_step(t) * db.abs() * (1 + 45 * U), "db")
    x3, w1, b0 = x[3:4].cpu(), torch.ones(cols).to(t), torch.zeros(cols).to(t)
    (z, ez), _, _, _ = norm_reference(x3, w1, b0, eps, g[3:4].cpu())
    dw, e = (g[3].cpu().double() * z[0]), g[3].cpu().double().abs() * (ez[0] + 45 * U * z[0].abs())
    close(got[2], dw, e + half_step(t) * (dw.abs() + e), "dw: the ordinary row's share alone")


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
