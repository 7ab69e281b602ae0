"""packed_attention where its tiles end and where many waves share them: hidden and trailing
rows next to infinities and NaN, in the forward and in all gradients, and workgroups of four
waves, against the float64 definition and tolerances of test_gpu_packed_attention."""
import math

import pytest
import torch

from test_gpu_packed_attention import BOTH, U, attend, close, definition, offsets, tensors

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def run(q, k, v, g, ptr, kv_ptr=None, **kw):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    y = attend(*leaves, ptr, kv_ptr, **kw)
    return [y.detach(), *torch.autograd.grad(y, leaves, g)]


# rows of a key's tile: below, at and above 16, 32 and 64 rows of queries and heads
@pytest.mark.parametrize("t,d", [(torch.float32, 8), (torch.float32, 16), (torch.float32, 40),
                                 (torch.bfloat16, 16), (torch.bfloat16, 64), (torch.bfloat16, 128)], ids=str)
@pytest.mark.parametrize("h,hk", [(1, 1), (6, 2)])
@pytest.mark.parametrize("causal", [False, True])
def test_a_key_of_probability_zero(causal, h, hk, t, d):
    """A key with -inf in a dimension where all queries are positive: its probability is 0 and
    so are dk and dv, at every number of rows, as with a finite value far enough down."""
    for n in (2, 5, 11, 16, 22, 31, 32, 33, 43, 64, 65, 100, 700):
        q, k, v = tensors(n, n, h, hk, d, t, seed=n)
        g = torch.randn(n, h, d, device=DEV).to(t)
        q[..., 0] = q[..., 0].abs() + 0.5
        ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        for at in {1, n // 2, n - 1} - {0}:
            got = []
            for low in (-1e30, -math.inf):
                k[at, :, 0] = low
                got.append(run(q, k, v, g, ptr, causal=causal))
            k[at, :, 0] = 1.0
            for name, j in (("y", 0), ("dk", 2), ("dv", 3)):
                assert bool(got[1][j].isfinite().all()), (name, n, at)
                assert torch.equal(got[0][j], got[1][j]), (name, n, at)
            assert not got[1][2][at].any() and not got[1][3][at].any()
            # dq: 0 times -inf in that dimension alone
            assert torch.equal(got[0][1][..., 1:], got[1][1][..., 1:])


HIDDEN = [(torch.float32, 8, 2, 2, 300, 150), (torch.float32, 32, 4, 1, 300, 131),
          (torch.float32, 8, 2, 1, 1300, 700), (torch.bfloat16, 16, 3, 1, 200, 97),
          (torch.bfloat16, 64, 4, 2, 300, 150), (torch.bfloat16, 128, 2, 1, 300, 160),
          (torch.bfloat16, 64, 2, 2, 1300, 640), (torch.bfloat16, 128, 4, 1, 1300, 777)]


@pytest.mark.parametrize("t,d,h,hk,n,at", HIDDEN, ids=str)
def test_hidden_keys_have_no_part_in_dq(t, d, h, hk, n, at):
    q, k, v = tensors(n, n, h, hk, d, t, seed=n)
    g = torch.randn(n, h, d, device=DEV).to(t)
    ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    want = run(q, k, v, g, ptr, causal=True)
    for bad in (math.nan, math.inf, -math.inf):
        for which in (0, 1):
            kv = [k.clone(), v.clone()]
            kv[which][at:] = bad
            got = run(q, *kv, g, ptr, causal=True)
            assert torch.equal(got[0][:at], want[0][:at]), (bad, which)
            assert torch.equal(got[1][:at], want[1][:at]), (bad, which)
            # the last query sees them: nothing finite can come of it
            assert not bool(got[1][-1].isfinite().any()), (bad, which)


@pytest.mark.parametrize("t,d,h,hk,n,at", HIDDEN, ids=str)
def test_queries_that_do_not_see_a_key_have_no_part_in_its_gradients(t, d, h, hk, n, at):
    q, k, v = tensors(n, n, h, hk, d, t, seed=n)
    g = torch.randn(n, h, d, device=DEV).to(t)
    ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    want = run(q, k, v, g, ptr, causal=True)
    alone = definition(q[at:], k, v, g[at:], [0, n - at], [0, n], True, d ** -0.5)[3:]
    for bad in (math.nan, math.inf, -math.inf):
        for which in (0, 1):
            qg = [q.clone(), g.clone()]
            qg[which][:at] = bad
            got = run(qg[0], k, v, qg[1], ptr, causal=True)
            for j, (b, e) in zip((2, 3), alone):  # of the queries from `at` on
                close(got[j][at:], b[at:], e[at:], t, (bad, which, j))
                # g has no part in the forward; an infinite q may move the reference of the
                # softmax sums of its tile's other rows
                assert which == 0 or torch.equal(got[j][at:], want[j][at:]), (bad, j)
            # key 0 is seen by all of them
            assert not bool(got[2][0].isfinite().any()), (bad, which)
            if which == 0 or bad is not math.nan:
                assert not bool(got[3][0].isfinite().all()), (bad, which)


@pytest.mark.parametrize("t,d,h,hk", [(torch.float32, 8, 2, 1), (torch.bfloat16, 64, 4, 2),
                                      (torch.bfloat16, 128, 2, 2)], ids=str)
def test_one_bad_value_among_hidden_and_seen_rows(t, d, h, hk):
    """A single infinity or NaN in a tile that some rows see and others do not."""
    n = 150
    q, k, v = tensors(n, n, h, hk, d, t)
    g = torch.randn(n, h, d, device=DEV).to(t)
    ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    clean = run(q, k, v, g, ptr, causal=True)
    for at in (0, 31, 32, 70, n - 1):
        for bad in (math.nan, math.inf):
            vb = v.clone()
            vb[at, 0, 3] = bad
            y, dq, dk, dv = run(q, k, vb, g, ptr, causal=True)
            grp = h // hk
            assert torch.equal(y[:at], clean[0][:at]) and torch.equal(dq[:at], clean[1][:at])
            keep = [c for c in range(d) if c != 3]
            assert torch.equal(y[..., keep], clean[0][..., keep])  # the other dimensions of y
            assert not bool(y[at:, :grp, 3].isfinite().any())
            assert torch.equal(y[:, grp:], clean[0][:, grp:])      # and the other key heads
            gb = g.clone()
            gb[at, 0, 3] = bad
            y, dq, dk, dv = run(q, k, v, gb, ptr, causal=True)
            assert torch.equal(y, clean[0])
            rest = [i for i in range(n) if i != at]
            assert torch.equal(dq[rest], clean[1][rest])
            assert torch.equal(dk[at + 1:], clean[2][at + 1:]) and torch.equal(dv[at + 1:], clean[3][at + 1:])
            assert not bool(dv[:at + 1, 0, 3].isfinite().any())
            assert torch.equal(dv[..., keep], clean[3][..., keep])


def waves(cols, count, kv_heads, w):
    """The library's choice of waves a workgroup for an axis of `cols` rows in `count`
    sequences, w columns a wave."""
    def tiles(n):
        return max(count, -(-cols // (w * n))) * kv_heads
    return 1 if cols <= w * count else 2 if cols <= 2 * w * count or tiles(4) < 1024 else 4


LENS = [700, 1, 0, 1500, 64, 63, 333, 130, 900, 1200, 31, 1024, 515, 2, 96, 1800, 640, 777, 256, 257,
        1450, 33, 1111, 888, 1000, 640, 1279]


# float32 heads up to 16 take 16 columns a wave, all others 32
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t,d,grp", [(torch.float32, 7, 1), (torch.float32, 8, 2), (torch.float32, 16, 1),
                                     (torch.float32, 24, 1), (torch.float32, 64, 2), (torch.float32, 96, 1),
                                     (torch.float32, 128, 1), (torch.bfloat16, 8, 1), (torch.bfloat16, 32, 2),
                                     (torch.bfloat16, 64, 1), (torch.bfloat16, 80, 2), (torch.bfloat16, 96, 1),
                                     (torch.bfloat16, 128, 3)], ids=str)
def test_workgroups_of_four_waves(t, d, grp, causal):
    hk, n = 8, sum(LENS)
    w = 16 if t == torch.float32 and d <= 16 else 32
    assert waves(n * grp, len(LENS), hk, w) == 4 and waves(n, len(LENS), hk, w) == 4
    q, k, v = tensors(n, n, hk * grp, hk, d, t)
    g = torch.randn(n, hk * grp, d, device=DEV).to(t)
    ptr = torch.tensor(offsets(LENS), dtype=torch.int32, device=DEV)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    y, lse = attend(*leaves, ptr, causal=causal, return_lse=True)
    got = [y.detach(), lse, *torch.autograd.grad(y, leaves, g)]
    assert all(bool(x.isfinite().all()) for x in got)
    at = offsets(LENS)
    for s in (0, 1, 4, 5, 6, 11, 13, 19, 21):  # some sequences against the definition
        rows = slice(at[s], at[s + 1])
        keep = slice(0, 2 * grp), slice(0, 2)  # two key heads
        want = definition(q[rows, keep[0]], k[rows, keep[1]], v[rows, keep[1]], g[rows, keep[0]],
                          [0, LENS[s]], [0, LENS[s]], causal, d ** -0.5)
        for name, a, (b, e) in zip(("y", "lse", "dq", "dk", "dv"), got, want):
            a = a[rows, keep[1] if name in ("dk", "dv") else keep[0]]
            close(a, b, e, a.dtype, f"{d} {grp} {causal} {t} {name} {s}")
    # each sequence by itself (other waves a workgroup): bf16 sums cut at other places
    with torch.no_grad():
        for s in (3, 15, 20):
            rows = slice(at[s], at[s + 1])
            one = torch.tensor([0, LENS[s]], dtype=torch.int32, device=DEV)
            alone = attend(q[rows], k[rows], v[rows], one, causal=causal).double()
            mag = attend(q[rows], k[rows], v[rows].abs(), one, causal=causal).double()
            h = torch.finfo(t).eps / 2
            # both sides' rounded probabilities and results, and 2 x 1800 float32 roundings each
            tol = (4 * h + 2 * 3600 * 2.0 ** -24) * (1 + 4 * h) * mag
            assert bool(((alone - y[rows].double()).abs() <= tol).all()), s


@pytest.mark.parametrize("t", BOTH, ids=str)
def test_four_waves_with_infinities_that_the_mask_hides(t):
    hk, d, n = 8, 64 if t == torch.bfloat16 else 8, sum(LENS)
    q, k, v = tensors(n, n, hk, hk, d, t)
    g = torch.randn(n, hk, d, device=DEV).to(t)
    ptr = torch.tensor(offsets(LENS), dtype=torch.int32, device=DEV)
    want = run(q, k, v, g, ptr, causal=True)
    kb, vb = k.clone(), v.clone()
    at = torch.tensor(offsets(LENS))
    last = [int(e) - 1 for e, x in zip(at[1:], LENS) if x > 1]  # seen by the last query alone
    kb[last], vb[last] = math.nan, math.inf
    got = run(q, kb, vb, g, ptr, causal=True)
    rest = [i for i in range(n) if i not in set(last)]
    assert torch.equal(got[0][rest], want[0][rest]) and torch.equal(got[1][rest], want[1][rest])
    first = [int(a) for a, x in zip(at, LENS) if x > 1]  # see their own key alone
    qb, gb = q.clone(), g.clone()
    qb[first], gb[first] = math.inf, math.nan
    got = run(qb, k, v, gb, ptr, causal=True)
    rest = [i for i in range(n) if i not in set(first)]
    for j in (0, 1, 2, 3):
        assert torch.equal(got[j][rest], want[j][rest]), j


FAR = [(torch.float32, 8, 2, 2), (torch.float32, 16, 3, 1), (torch.float32, 32, 2, 1), (torch.float32, 128, 2, 2),
       (torch.bfloat16, 16, 2, 2), (torch.bfloat16, 64, 6, 2), (torch.bfloat16, 128, 2, 1)]


def far_inputs(nq, nk, h, hk, d, t, root):
    """Scores of `root`^2 + 0 .. 5, which float32 holds exactly, and the inputs of the same
    softmax without the offset."""
    q, k, v = tensors(nq, nk, h, hk, d, t)
    q.zero_()
    q[..., 1] = 1
    k[..., 1] = torch.randint(0, 6, k.shape[:2], device=DEV).to(t)
    k[..., 0] = 0
    qf, kf = q.clone(), k.clone()
    qf[..., 0], kf[..., 0] = abs(root), root
    return q, k, v, qf, kf


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t,d,h,hk", FAR, ids=str)
@pytest.mark.parametrize("lens,kl", [([200, 1, 33, 0, 64], None), ([1300], None), ([1, 1, 2], [3000, 70, 900])],
                         ids=str)
def test_scores_far_from_zero(lens, kl, t, d, h, hk, causal):
    """The softmax goes by differences of scores: a common offset of up to 2^22 does not change
    the output.  The gradients go by the float32 lse: with the error of its rounding up to
    where that leaves nothing, and NaN from there on."""
    kl = lens if kl is None else kl
    nq, nk = sum(lens), sum(kl)
    ptr, kv = (torch.tensor(offsets(x), dtype=torch.int32, device=DEV) for x in (lens, kl))
    g = torch.randn(nq, h, d, device=DEV).to(t)
    for root in (64.0, 1024.0, -1024.0, 2048.0):
        q, k, v, qf, kf = far_inputs(nq, nk, h, hk, d, t, root)
        (wy, ey), (wl, el), _, _, _ = definition(q, k, v, g, offsets(lens), offsets(kl), causal, 1.0)
        leaves = [x.requires_grad_() for x in (qf, kf, v)]
        y, lse = attend(*leaves, ptr, kv, causal=causal, scale=1.0, return_lse=True)
        off = root * abs(root)
        close(y, wy, ey, t, (root, "y"))
        close(lse, wl + off, el + 4 * U * abs(off), torch.float32, (root, "lse"))
        grads = torch.autograd.grad(y, leaves, g)
        if abs(off) <= 4096:  # the offset is part of the bounds: 4 U |lse|
            want = definition(qf, kf, v, g, offsets(lens), offsets(kl), causal, 1.0)[2:]
            for name, a, (b, e) in zip(("dq", "dk", "dv"), grads, want):
                close(a, b, e, t, (root, name))
        if off > 1 << 21:
            seen = (lse > -math.inf).cpu()
            assert bool(grads[0].cpu()[seen].isnan().all())


@pytest.mark.parametrize("t,d,h,hk", FAR, ids=str)
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 31, 2.0 ** 58])
def test_scores_of_any_size(size, t, d, h, hk):
    """Scores up to float32's range, each key's far above the one before: all of a query's
    weight is on its last key, exactly; and equal scores, however large, share it."""
    n = 150
    q, k, v = tensors(n, n, h, hk, d, t)
    g = torch.randn(n, h, d, device=DEV).to(t)
    ptr = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    q.zero_()
    q[..., 0] = size
    for sign in (1.0, -1.0):
        k[..., 0] = sign * size * (torch.arange(n, device=DEV)[:, None] + 1)
        y = attend(q, k, v, ptr, causal=True)
        each = v if sign > 0 else v[:1].expand(n, hk, d)
        assert torch.equal(y, each.repeat_interleave(h // hk, 1))
    k[..., 0] = torch.where(torch.arange(n, device=DEV)[:, None] % 2 == 0, size, -size)
    y = attend(q, k, v, ptr)
    even = v[::2].double().mean(0).cpu()
    hp = 0.0 if t == torch.float32 else torch.finfo(t).eps / 2
    e = (4 * n * U + 2 * hp) * v[::2].double().abs().mean(0).cpu()
    even, e = (x.repeat_interleave(h // hk, 0).expand(n, h, d) for x in (even, e))
    close(y, even, e, t, (size, "mean"))
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    for x in torch.autograd.grad(attend(*leaves, ptr), leaves, g):  # beyond the lse's digits
        assert bool(x.isnan().all())


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t,d,h,hk", FAR, ids=str)
@pytest.mark.parametrize("size", [1e7, 1e9, 1e30])
def test_far_rows_without_a_gradient(size, t, d, h, hk, causal):
    """Queries all of whose scores are far below 0, as a padded row's are whose keys were put
    out of reach, and whose output nothing uses: no gradient comes from them, as from any row
    with g = 0, and those of the other rows are what they are."""
    lens = [150, 33, 70]
    n = sum(lens)
    q, k, v = tensors(n, n, h, hk, d, t)
    g = torch.randn(n, h, d, device=DEV).to(t)
    k[..., 0] = 1
    q[..., 0] = 0
    far = [3, 17, 40, 41, 42, 149, 150, 199, n - 1]
    q[far] = 0
    q[far, :, 0] = -size
    g[far] = 0
    ptr = torch.tensor(offsets(lens), dtype=torch.int32, device=DEV)
    want = definition(q, k, v, g, offsets(lens), offsets(lens), causal, d ** -0.5)[2:]
    _, *got = run(q, k, v, g, ptr, causal=causal)
    for name, a, (b, e) in zip(("dq", "dk", "dv"), got, want):
        close(a, b, e, t, (size, name))
    assert not got[0][far].any()
    if size * d ** -0.5 * math.log2(math.e) < 1 << 22:
        return
    g[far[0], 0, d - 1] = 1  # one that is used: NaN, in its own sequence
    _, *got = run(q, k, v, g, ptr, causal=causal)
    assert bool(got[0][far[0], 0].isnan().all()) and bool(got[1][0, 0].isnan().all())
    assert bool(got[2][0, 0].isnan().all())
    for a, (b, e) in zip(got, want):
        close(a[150:], b[150:], e[150:], t, (size, "other sequences"))
