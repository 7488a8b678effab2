"""top_logits, topk_distill and the losses made of them against their formulas in 64 bits.

Tolerances.  top_logits: values and indices are exact; a log-sum-exp is off by the rounding of its terms'
exponents, 2^-23 of the row's range of |x| / T (a few float32 steps), and of the sum, 2^-20 in all.  The
loss sums k terms t (log t - s + lse), each off by that much of its magnitude: 2^-20 of the sum of
magnitudes, rows' and the mean's.  The gradient is g (tau p - t) / T, rounded once: u = finfo.eps / 2 of it,
and 2^-18 of g (tau p + t) / T for the exponentials (the exponent x / T - lse rounds to 2^-24 of up to 60)."""
import math

import pytest
import torch

from scmiac_amd import _hip
from scmiac_amd.modeling import NeighborDistillLoss, NTXentLoss2, TopKDistillLoss, linear_act, top_logits, topk_distill

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _wide(x, idx, top, T, lse=None, Ta=None):
    """(loss, dloss/dx, size of the loss's terms, size of the gradient's terms, counted rows) in 64 bits, row by row."""
    Ta = T if Ta is None else Ta
    x = x.double() / T
    n, v = x.shape
    loss, grad = torch.zeros(n, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    lsize, gsize, counted = torch.zeros_like(loss), torch.zeros_like(grad), torch.zeros(n, dtype=torch.bool)
    x, idx, top = x.cpu(), idx.cpu(), top.cpu()
    for i in range(n):
        real = idx[i] >= 0
        a, j = top[i][real].double() / Ta, idx[i][real].long()
        if j.numel() == 0 or bool((a == -math.inf).all()) or bool((x[i] == -math.inf).all()):
            continue
        counted[i] = True
        x[i] -= x[i].max()      # (of rows at the lowest value of a type, 64 bits would lose the logarithm of the sum, too)
        c = torch.logsumexp(a, 0) if lse is None else lse.cpu()[i].double()
        t = torch.exp(a - c)
        z = torch.logsumexp(x[i], 0)
        for w, aa, jj in zip(t.tolist(), a.tolist(), j.tolist()):
            if w > 0:
                loss[i] += w * (aa - float(c) - float(x[i, jj]) + float(z))
                lsize[i] += w * (abs(aa) + abs(float(c)) + abs(float(x[i, jj])) + abs(float(z)) + 1)
        p = torch.exp(x[i] - z) * t.sum()
        grad[i], gsize[i] = p / T, p / T
        grad[i].index_add_(0, j, -t / T)
        gsize[i].index_add_(0, j, t / T)
    return loss, grad, lsize, gsize, counted


def _check(x, idx, top, T=1.0, lse=None, Ta=None):
    dtype = x.dtype
    want, grad, lsize, gsize, counted = _wide(x, idx, top, T, lse, Ta)
    n = x.shape[0]
    g = 0.5 + torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal
    for reduction in ("none", "sum", "mean"):
        leaf = x.detach().requires_grad_()
        loss = topk_distill(leaf, idx, top, T, lse, Ta, reduction)
        up = g if reduction == "none" else torch.tensor(1.75, device="cuda")
        dx, = torch.autograd.grad(loss, [leaf], up)
        assert loss.dtype == torch.float32 and dx.dtype == dtype and dx.shape == x.shape
        with torch.no_grad():
            assert torch.equal(topk_distill(leaf, idx, top, T, lse, Ta, reduction), loss)
        count = max(1, int(counted.sum()))
        if reduction == "none":
            w, scale = want, g.cpu().double()
            bound = lsize * 2.0 ** -20
        else:
            d = count if reduction == "mean" else 1
            w, scale, bound = want.sum() / d, torch.full((n,), 1.75 / d, dtype=torch.float64), lsize.sum() / d * 2.0 ** -20
        lo = loss.cpu().double()
        assert bool(((lo - w).abs() <= bound + 1e-30).logical_or(lo == w).all()), (reduction, lo, w)
        wg = grad * scale[:, None]
        err = (dx.cpu().double() - wg).abs()
        assert bool((err <= u * wg.abs() + 2.0 ** -18 * gsize * scale[:, None] + tiny * (dtype != torch.float32) + 1e-37).all()), \
            (reduction, float(err.max()))
        assert not dx[~counted.cuda()].any()


def _rand(n, v, k, dtype, seed=0, spread=2.0, pads=True):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1009 + n * 31 + v + k)
    x = (torch.randn(n, v, device="cuda", generator=gen) * spread).to(dtype)
    idx = torch.randint(0, v, (n, k), device="cuda", generator=gen, dtype=torch.int32)      # repeats among them
    if pads:
        idx[torch.rand(n, k, device="cuda", generator=gen) < 0.2] = -1
        idx[n // 2] = -1
    return x, idx, torch.randn(n, k, device="cuda", generator=gen) * 2, gen


# ------------------------------------------------------------------ the loss

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (2, 2, 3), (5, 7, 2), (9, 64, 64), (6, 200, 8), (3, 1023, 30), (3, 1024, 30),
                                   (3, 1025, 30), (2, 4099, 100), (1, 20011, 17), (2, 8192, 1024), (1, 70000, 5), (4099, 1501, 7), (4096, 4096, 3)])
def test_loss_and_gradient(n, v, k, dtype):
    x, idx, top, gen = _rand(n, v, k, dtype)
    _check(x, idx, top, T=1.0)
    _check(x, idx, top, T=2.0, Ta=0.7)
    lse = torch.logsumexp(top / 0.5, 1) + torch.rand(n, device="cuda", generator=gen)
    _check(x, idx, top, T=0.5, lse=lse)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks(dtype):
    x, idx, top, _ = _rand(12, 300, 9, dtype, seed=4, pads=False)
    low = torch.finfo(dtype).min
    x[0, ::2] = -math.inf
    idx[0] = (idx[0] // 2) * 2 + 1                      # the teacher's classes are not masked
    idx[0].clamp_(max=299)
    x[1, ::2] = low                                     # the type's lowest value as a mask
    idx[1] = (idx[1] // 2) * 2 + 1
    idx[1].clamp_(max=299)
    x[2] = -math.inf                                    # nothing left: no loss, no gradient
    idx[3] = -1                                         # no teacher
    top[4] = -math.inf                                  # a teacher without weight
    top[5, 3:] = -math.inf                              # weights of zero
    idx[6, 1:] = -1
    idx[7] = 17                                         # one class nine times
    idx[8, ::2] = idx[8, 0].clone()
    x[9] = 3.0                                          # equal everywhere
    x[10, 1:] = -math.inf
    idx[10] = 0                                         # a single class left, listed nine times
    _check(x, idx, top)
    x[11] = low                                         # all at the type's lowest value: uniform
    _check(x, idx, top)
    # a weight on a masked class: an infinite loss, and a gradient that is still the formula's
    x[5, int(idx[5, 0])] = -math.inf
    leaf = x.detach().requires_grad_()
    loss = topk_distill(leaf, idx, top, reduction="none")
    dx, = torch.autograd.grad(loss.nan_to_num(posinf=0.0).sum(), [leaf])
    assert loss[5] == math.inf and torch.isfinite(loss[[0, 1, 2, 3, 4, 6, 7, 8, 9, 10]]).all()
    assert torch.isfinite(dx[torch.arange(12) != 5]).all()


def test_an_index_that_is_no_class_poisons_its_row_alone():
    x, idx, top, _ = _rand(6, 100, 4, torch.float32, seed=2, pads=False)
    idx[1, 2], idx[3, 0] = 100, -2
    top[4, 1] = math.nan
    wide = idx.long()
    wide[5, 0] = 2 ** 32 + 5                            # would be class 5 in 32 bits
    for table in (idx, wide):
        leaf = x.detach().requires_grad_()
        loss = topk_distill(leaf, table, top, reduction="none")
        dx, = torch.autograd.grad(loss, [leaf], torch.ones(6, device="cuda"))
        bad = [1, 3, 4] + ([5] if table is wide else [])
        assert torch.isnan(loss).nonzero().flatten().tolist() == bad
        assert torch.isnan(dx).all(1).nonzero().flatten().tolist() == bad
        assert torch.isfinite(dx[[0, 2]]).all()
    x[0, 50] = math.nan
    assert torch.isnan(topk_distill(x, idx, top, reduction="none")[0])
    assert torch.isnan(topk_distill(x, idx, top))


def test_a_good_student_has_a_small_and_exact_gradient():
    # the student's softmax equals the teacher's but for a thousandth: p and t cancel almost completely
    gen = torch.Generator(device="cuda").manual_seed(8)
    v, k = 500, 20
    x = torch.full((4, v), -9.0, device="cuda")
    idx = torch.stack([torch.randperm(v, device="cuda", generator=gen)[:k] for _ in range(4)]).int()
    top = torch.randn(4, k, device="cuda", generator=gen)
    x.scatter_(1, idx.long(), top + 1e-3 * torch.randn(4, k, device="cuda", generator=gen))
    _check(x, idx, top)


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_offsets_and_leading_dimensions(dtype):
    x, idx, top, _ = _rand(10, 1200, 6, dtype, seed=5)
    for store, cut in [(torch.empty(10, 1208, dtype=dtype, device="cuda"), slice(0, 1200)),
                       (torch.empty(10, 1201, dtype=dtype, device="cuda"), slice(1, 1201)),
                       (torch.empty(10, 4000, dtype=dtype, device="cuda"), slice(7, 1207)),
                       (torch.empty(1200, 10, dtype=dtype, device="cuda").t(), slice(0, 1200))]:
        store.fill_(7.0)
        store[:, cut] = x
        leaf = store.detach().requires_grad_()
        loss = topk_distill(leaf[:, cut], idx, top, reduction="none")
        grad, = torch.autograd.grad(loss, [leaf], torch.ones(10, device="cuda"))
        flat = x.detach().requires_grad_()
        want = topk_distill(flat, idx, top, reduction="none")
        wgrad, = torch.autograd.grad(want, [flat], torch.ones(10, device="cuda"))
        # another start of the rows groups the sum of exponentials differently: float32 roundings of it
        torch.testing.assert_close(loss, want, rtol=2e-6, atol=2e-6)
        torch.testing.assert_close(grad[:, cut].float(), wgrad.float(), rtol=2 * torch.finfo(dtype).eps + 1e-5, atol=1e-7)
        keep = torch.ones(store.shape[1], dtype=torch.bool, device="cuda")
        keep[cut] = False
        assert not grad[:, keep].any()
    x3, i3, t3 = x.view(2, 5, 1200), idx.view(2, 5, 6), top.view(2, 5, 6)
    loss = topk_distill(x3, i3, t3, reduction="none")
    assert loss.shape == (2, 5) and torch.equal(loss.view(-1), topk_distill(x, idx, top, reduction="none"))
    assert topk_distill(x[0], idx[0], top[0], reduction="none").shape == ()
    strided = torch.stack([idx, idx], 2)[:, :, 0]
    assert torch.equal(topk_distill(x, strided.long(), top.double()), topk_distill(x, idx, top))


def test_no_rows_and_no_rows_that_count():
    x = torch.empty(0, 9, device="cuda", requires_grad=True)
    idx, top = torch.empty(0, 3, dtype=torch.int32, device="cuda"), torch.empty(0, 3, device="cuda")
    assert topk_distill(x, idx, top, reduction="none").shape == (0,)
    for reduction in ("mean", "sum"):
        loss = topk_distill(x, idx, top, reduction=reduction)
        assert loss == 0
        assert torch.autograd.grad(loss, [x])[0].shape == (0, 9)
    x = torch.randn(4, 9, device="cuda", requires_grad=True)
    idx = torch.full((4, 3), -1, dtype=torch.int32, device="cuda")
    loss = topk_distill(x, idx, torch.zeros(4, 3, device="cuda"))
    assert loss == 0 and not torch.autograd.grad(loss, [x])[0].any()


def test_gradient_against_differences():
    x, idx, top, _ = _rand(3, 40, 6, torch.float32, seed=9)
    leaf = x.detach().requires_grad_()
    grad, = torch.autograd.grad(topk_distill(leaf, idx, top, 1.5, reduction="sum"), [leaf])
    h = 2.0 ** -5
    for i in range(3):
        for j in range(0, 40, 3):
            vals = []
            for sign in (1, -1):
                moved = x.clone()
                moved[i, j] += sign * h
                vals.append(float(topk_distill(moved, idx, top, 1.5, reduction="none")[i].double()))
            # h^2 / 6 of a third derivative below 1, and float32 losses of about 5 over 2 h
            assert abs((vals[0] - vals[1]) / (2 * h) - float(grad[i, j])) < 2e-4


# ------------------------------------------------------------------ the teacher's table

def _check_top(x, k, T=1.0):
    values, idx, lse = top_logits(x, k, T)
    w = x.float()
    order = torch.sort(w, dim=1, descending=True, stable=True).indices[:, :k]
    kept = order.shape[1]
    assert values.dtype == x.dtype and idx.dtype == torch.int32
    assert torch.equal(idx[:, :kept].long(), order)
    assert torch.equal(values[:, :kept], x.gather(1, order))
    assert (idx[:, kept:] == -1).all() and (values[:, kept:] == -math.inf).all()
    want = torch.logsumexp(x.double() / T, 1)
    bound = 2.0 ** -20 * (1 + (w.masked_fill(w == -math.inf, 0).abs().amax(1).double() / T))
    assert bool(((lse.double() - want).abs() <= bound).logical_or(lse.double() == want).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (3, 5, 8), (7, 64, 64), (300, 200, 8), (5, 1023, 64), (5, 1024, 1), (4, 1025, 64),
                                   (3, 2049, 30), (2, 10412, 30), (1, 200003, 64), (3, 65537, 7), (1100, 1500, 13), (2049, 3001, 20)])
def test_top_logits(n, v, k, dtype):
    x = _rand(n, v, 1, dtype, seed=11)[0]
    _check_top(x, k)
    _check_top(x, k, 0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [150, 5000, 40000])
def test_top_logits_ties_orders_and_masks(v, dtype):
    gen = torch.Generator(device="cuda").manual_seed(v)
    rows = [torch.zeros(v), torch.arange(v) / 8.0 % 4000, -(torch.arange(v) / 8.0 % 4000), torch.arange(v) % 3,
            torch.full((v,), -math.inf), torch.full((v,), torch.finfo(dtype).min),
            torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0),                 # one value, two signs
            torch.where(torch.arange(v) == v - 1, 5.0, -math.inf), torch.randint(0, 4, (v,)).float()]
    x = torch.stack([r.float() for r in rows]).to("cuda").to(dtype)
    x = torch.cat([x, (torch.randn(3, v, device="cuda", generator=gen) * 2).to(dtype)])
    x[-1, ::2] = -math.inf
    for k in (1, 33, 64):
        _check_top(x, k)
    x[0, v // 2] = math.inf
    values, idx, lse = top_logits(x, 3)
    assert idx[0, 0] == v // 2 and values[0, 0] == math.inf and lse[0] == math.inf
    x[1, 7] = math.nan                                                       # its own row alone, indices within it
    values, idx, lse = top_logits(x, 3)
    assert torch.isnan(lse[1]) and not torch.isnan(lse[[0, 2, 3]]).any()
    assert int(idx[1].min()) >= -1 and int(idx[1].max()) < v


@pytest.mark.parametrize("good", [1, 20, 63, 64, 500])
def test_top_logits_where_every_piece_of_a_long_row_is_alike(good):
    """The best of a row in the same few places of every 4096 classes, many of them equal."""
    v = 245 * 4096
    at = torch.arange(v, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(good)
    x = torch.full((3, v), -math.inf, device="cuda")
    x[0, at % 4096 < good] = 1.0
    x[1] = torch.where(at % 4096 < good, torch.randn(v, device="cuda", generator=gen), torch.tensor(-9.0, device="cuda"))
    x[2] = torch.where(4095 - at % 4096 < good, at / 4096, -at / 4096.0)
    for k in (1, 31, 64):
        for row in range(3):
            _check_top(x[row:row + 1], k)
        _check_top(x, k)


def test_top_logits_strides_and_shapes():
    x = torch.randn(6, 3001, device="cuda")
    want = top_logits(x[:, 1:2990].contiguous(), 20)
    got = top_logits(x[:, 1:2990], 20)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.testing.assert_close(got[2], want[2], rtol=2e-6, atol=0)
    turned = top_logits(x.t()[:2000], 5)
    assert torch.equal(turned[1], top_logits(x.t()[:2000].contiguous(), 5)[1])
    v3, i3, l3 = top_logits(x.view(2, 3, 3001), 4)
    assert v3.shape == (2, 3, 4) and i3.shape == (2, 3, 4) and l3.shape == (2, 3)
    assert top_logits(x[0], 4)[0].shape == (4,) and top_logits(x[:0], 4)[1].shape == (0, 4)
    assert not top_logits(x.requires_grad_(), 4)[0].requires_grad


# ------------------------------------------------------------------ together, as a training step uses them

def test_a_teachers_table_trains_a_student_to_it():
    torch.manual_seed(1)
    teacher = torch.randn(64, 500, device="cuda") * 3
    values, idx, lse = top_logits(teacher, 16, temperature=2.0)
    # a student that equals the teacher: the loss is what the listed classes contribute to the divergence, 0
    loss = topk_distill(teacher, idx, values, 2.0, teacher_lse=lse, reduction="none")
    assert float(loss.abs().max()) < 2e-5
    x, w = torch.randn(64, 40, device="cuda"), torch.randn(500, 40, device="cuda", requires_grad=True)
    b = torch.zeros(500, device="cuda", requires_grad=True)
    loss = TopKDistillLoss(2.0)(linear_act(x, w, b), idx, values, lse)
    dw, db = torch.autograd.grad(loss, [w, b])
    wd, bd = w.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    logp = torch.log_softmax((x.double() @ wd.t() + bd) / 2.0, 1)
    t = torch.exp(values.double() / 2.0 - lse[:, None].double())
    want = (t * (torch.log(t) - logp.gather(1, idx.long()))).sum(1).mean()
    ww, wb = torch.autograd.grad(want, [wd, bd])
    # float32 logits of about 20: the softmax carries 2^-24 x 20 x a few, relative to the largest gradient
    assert abs(loss.item() - want.item()) < 2e-5 * want.item()
    assert float((dw - ww).abs().max()) < 2e-5 * float(ww.abs().max())
    assert float((db - wb).abs().max()) < 2e-5 * float(wb.abs().max())


@pytest.mark.parametrize("metric", ["cosine", "euclidean"])
def test_neighbor_loss_from_a_search_table(metric):
    gen = torch.Generator(device="cuda").manual_seed(3)
    ref, q = torch.randn(900, 30, device="cuda", generator=gen), torch.randn(257, 30, device="cuda", generator=gen)
    table = _hip.knn_search(q, ref, 12)
    zq = torch.randn(257, 16, device="cuda", generator=gen, requires_grad=True)
    zr = torch.randn(900, 16, device="cuda", generator=gen, requires_grad=True)
    loss = NeighborDistillLoss(0.5, 4.0, metric)(zq, zr, table.idx, -table.dist2)
    grads = torch.autograd.grad(loss, [zq, zr])
    a, b = (t.detach().double().requires_grad_() for t in (zq, zr))
    if metric == "cosine":
        s = torch.nn.functional.normalize(a, dim=1) @ torch.nn.functional.normalize(b, dim=1).t()
    else:
        s = -0.5 * torch.cdist(a, b) ** 2
    t = torch.softmax(-table.dist2.double() / 4.0, 1)
    want = (t * (torch.log(t) - torch.log_softmax(s / 0.5, 1).gather(1, table.idx.long()))).sum(1).mean()
    wide = torch.autograd.grad(want, [a, b])
    assert abs(loss.item() - want.item()) < 1e-5 * want.item()
    for g, w in zip(grads, wide):
        assert float((g - w).abs().max()) < 5e-5 * float(w.abs().max())
    # beside the contrastive loss of the same embeddings, and with a table that pads
    few = _hip.knn_search(q, ref[:8].contiguous(), 12)
    assert bool((few.idx[:, 8:] == -1).all())
    both = NTXentLoss2(0.5)(zq, zr[:257]) + NeighborDistillLoss(0.5, 1.0, metric)(zq, zr, few.idx, -few.dist2)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(both, [zq, zr]))


def test_streams_and_capture():
    x, idx, top, _ = _rand(3, 50000, 40, torch.bfloat16, seed=6)
    want, table = topk_distill(x, idx, top, reduction="none"), top_logits(x, 40)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((topk_distill(x, idx, top, reduction="none"), *top_logits(x, 40)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want) and all(torch.equal(p, q) for p, q in zip(g[1:], table))
    leaf = x.detach().clone().requires_grad_()
    up = torch.tensor(2.0, device="cuda")

    def step():
        t = top_logits(leaf, 20)
        loss = topk_distill(leaf, idx, top)
        return (*t, loss.detach(), torch.autograd.grad(loss, [leaf], up)[0])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        with torch.no_grad():
            leaf.copy_(_rand(3, 50000, 40, torch.bfloat16, seed=20 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, step()))
        torch.cuda.synchronize()


def test_a_teacher_of_vanishing_weight_still_counts():
    x, idx, top, _ = _rand(4, 50, 3, torch.float32, seed=3, pads=False)
    lse = torch.tensor([500.0, 0.0, 0.0, 0.0], device="cuda")     # weights exp(-500): zero in float32
    idx[1] = -1
    rows = topk_distill(x, idx, top, teacher_lse=lse, reduction="none")
    assert rows[0] == 0 and rows[1] == 0
    # the mean is over the three rows that have a teacher
    torch.testing.assert_close(topk_distill(x, idx, top, teacher_lse=lse), rows.sum() / 3, rtol=1e-6, atol=0)


# ------------------------------------------------------------------ values far from the rest of their row

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(8, 200), (8, 3000), (2049, 3000), (8, 40000)])
def test_top_logits_of_finite_masks_and_of_large_logits(n, v, dtype):
    """Rows, starts, ends and whole pieces of rows at finite mask values, and logits as large the other way.

    The log-sum-exp is m / T + log s: 1 / T and the sum rounded, 2^-22 of |m| / T with room, and s off by at most
    2^-23 for every addition to a lane's part of it, and as much for terms whose exponents are a few hundred at most."""
    x = _rand(n, v, 1, dtype, seed=13)[0]
    masks = [-6e4, -3e4, -100.0] if dtype == torch.float16 else [-1e9, -5e9, -1e10, -1e12, -1e30, -1e36]
    for mask in masks:
        m = x.clone()
        m[0] = mask
        m[1, :3 * v // 4] = mask
        m[2, v // 4:] = mask
        m[3, :v // 2] = mask
        m[3, 0] = mask * 1.05
        m[4] = -mask
        m[5, v // 3] = -mask
        m[6, ::2] = mask
        m[7, v // 2:] = mask
        m[7, :v // 2] = mask * 1.05
        order = torch.sort(m.float(), dim=1, descending=True, stable=True).indices[:, :5]
        for T in (1e-5, 1e-3, 1.0) if dtype == torch.float16 else (0.1, 1.0, 30.0):
            values, idx, lse = top_logits(m, 5, T)
            assert torch.equal(idx.long(), order) and torch.equal(values, m.gather(1, order))
            wide = m.double() / T
            bound = 2.0 ** -22 * wide.amax(1).abs() + 2.0 ** -23 * (v / 64 + 300)
            assert bool(((lse.double() - torch.logsumexp(wide, 1)).abs() <= bound).all()), (mask, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(6, 1001), (6, 1023), (6, 3001), (2052, 3001), (6, 10411), (6, 40003)])
def test_top_logits_of_equal_values_in_rows_that_start_anywhere(n, v, dtype):
    gen = torch.Generator(device="cuda").manual_seed(v)
    at = torch.arange(v + 1, device="cuda")
    x = torch.randint(0, 3, (n, v + 1), device="cuda", generator=gen).float()
    x[0] = 1.0
    x[1] = torch.where(at % 97 == 5, 2.0, -math.inf)
    x[2] = -math.inf
    x[3] = (torch.randn(v + 1, device="cuda", generator=gen) * 2).round()
    x = x.to(dtype)
    for rows in (x[:, :v], x[:, 1:], x[:, 1:v], x[:, :v].contiguous()):
        for k in (1, 16, 33, 64):
            _check_top(rows, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [150, 5000, 40000])
def test_top_logits_of_a_nan_beside_an_infinity(v, dtype):
    x = _rand(8, v, 1, dtype, seed=3)[0]
    for row, (i, j) in enumerate([(0, 1), (1, 0), (0, v - 1), (v - 1, 0), (v // 2, v // 2 + 1), (v // 3, 2 * v // 3)]):
        x[row, i], x[row, j] = math.inf, math.nan
    x[6, [0, v // 2, v - 1]] = math.inf
    lse = top_logits(x, 3)[2]
    assert torch.isnan(lse[:6]).all() and lse[6] == math.inf and torch.isfinite(lse[7])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [150, 5000, 40000, 420000])
def test_a_nan_among_masked_classes_is_seen(v, dtype):
    x = torch.full((4, v), -math.inf, device="cuda", dtype=dtype)
    x[:, :20] = 1.0
    x[2, : v // 2 - 1] = 1.0
    x[2, v // 2 + v // 8:] = 1.0
    x[0, v - 3] = math.nan
    x[1] = x[1].flip(0)
    x[1, 5] = math.nan
    x[2, v // 2] = math.nan
    want = [True, True, True, False]
    lse = top_logits(x, 3)[2]
    idx = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    idx[1] = v - 1
    loss = topk_distill(x, idx, torch.zeros(4, 2, device="cuda"), reduction="none")
    assert (torch.isnan(lse).tolist(), torch.isnan(loss).tolist()) == (want, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [64, 1500, 40000])
def test_rows_without_a_teacher_may_hold_anything(v, dtype):
    x, idx, top, _ = _rand(8, v, 5, dtype, seed=21, pads=False)
    idx[[1, 3, 5]] = -1
    top[6] = -math.inf
    clean = topk_distill(x[[0, 2, 4, 7]], idx[[0, 2, 4, 7]], top[[0, 2, 4, 7]], reduction="none")
    x[1], x[3, v // 2], x[5, ::3], x[6, v - 1] = math.nan, math.nan, math.inf, math.nan
    for reduction in ("none", "sum", "mean"):
        leaf = x.detach().requires_grad_()
        loss = topk_distill(leaf, idx, top, reduction=reduction)
        dx, = torch.autograd.grad(loss.sum(), [leaf])
        assert not dx[[1, 3, 5, 6]].any() and torch.isfinite(dx).all()
        if reduction == "none":
            assert not loss[[1, 3, 5, 6]].any() and torch.equal(loss[[0, 2, 4, 7]], clean)
        else:      # summed in 64 bits and rounded; the division rounds once more
            want = float(clean.double().sum()) / (4 if reduction == "mean" else 1)
            assert abs(loss.item() - want) <= 2.0 ** -23 * abs(want)


def test_second_derivatives_of_the_loss_are_refused():
    x, idx, top, _ = _rand(4, 30, 3, torch.float32, seed=2)
    leaf = x.detach().requires_grad_()
    up = torch.ones(4, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(topk_distill(leaf, idx, top, reduction="none"), [leaf], up, create_graph=True)
    for t in (leaf, up):
        with pytest.raises(RuntimeError, match="differentiable twice"):
            torch.autograd.grad(g.sum() + t.sum(), t, retain_graph=True)


def test_views_with_a_pending_negation():
    neg = torch._neg_view
    x, idx, top, gen = _rand(6, 200, 4, torch.float32, seed=7)
    lse = torch.rand(6, device="cuda", generator=gen) + 4
    assert all(torch.equal(p, q) for p, q in zip(top_logits(neg(x), 5), top_logits(-x, 5)))
    for i in range(3):
        args, want = [x, top, lse], [x, top, lse]
        args[i], want[i] = neg(args[i]), -want[i]
        got, other = (topk_distill(t[0], idx, t[1], 1.0, t[2], reduction="none") for t in (args, want))
        assert torch.equal(got, other), i
    leaf = x.clone().requires_grad_()
    grads = [torch.autograd.grad(topk_distill(leaf, idx, top, reduction="none"), leaf, g)[0] for g in (neg(lse), -lse)]
    assert torch.equal(*grads)


def test_indices_of_every_type():
    x, idx, top, _ = _rand(4, 100, 3, torch.float32, seed=2, pads=False)
    want = topk_distill(x, idx, top, reduction="none")
    for dtype in (torch.int8, torch.uint8, torch.int16, torch.uint16, torch.uint32, torch.int64, torch.uint64):
        assert torch.equal(topk_distill(x, idx.to(dtype), top, reduction="none"), want), dtype
    for dtype, bad in ((torch.uint32, 2 ** 32 - 1), (torch.uint32, 2 ** 31 + 5), (torch.uint64, 2 ** 64 - 1), (torch.uint64, 2 ** 32 + 5),
                       (torch.uint64, 2 ** 63), (torch.int64, 2 ** 32 + 5), (torch.int64, -2 ** 32 - 1), (torch.int8, -2)):
        rows = idx.tolist()
        rows[1][2] = bad                                    # (unsigned, there is no -1 that could be padding)
        table = torch.tensor(rows, dtype=dtype).cuda()
        loss = topk_distill(x, table, top, reduction="none")
        assert torch.isnan(loss).tolist() == [False, True, False, False], (dtype, bad)
        assert torch.equal(loss[[0, 2, 3]], want[[0, 2, 3]])


def test_extreme_temperatures():
    """At the ends of the range: one class has all the weight, or all have the same."""
    x = torch.tensor([[3.0, -1.0, 2.0, 0.5], [0.0, 0.0, -7.0, -7.5]], device="cuda")
    idx = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device="cuda")
    top = torch.zeros(2, 2, device="cuda")
    _, order, lse = top_logits(x, 2, 2.0 ** -126)
    assert order.tolist() == [[0, 2], [0, 1]] and lse.tolist()[0] == 3 * 2.0 ** 126      # (below 2^128: a float32)
    assert abs(lse.tolist()[1] - math.log(2.0)) <= 2.0 ** -22
    lse = top_logits(x, 2, 3e38)[2]
    assert bool(((lse - math.log(4.0)).abs() <= 2.0 ** -22).all())
    leaf = x.clone().requires_grad_()
    loss = topk_distill(leaf, idx, top, 3e38, reduction="none")      # two of four equal classes: log 4 - log 2
    assert bool(((loss.detach() - math.log(2.0)).abs() <= 2.0 ** -20).all())
    assert torch.isfinite(torch.autograd.grad(loss.sum(), leaf)[0]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_euclidean_neighbors_of_large_embeddings(dtype):
    """A component of 300: its square is no float16, the score of -45 000 is one.  Bias and score are each rounded, by at most
    half a step of 2^15 .. 2^16 (16, 128, 2^-9), and the loss divides by the temperature."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    z, ref = (torch.randn(n, 8, device="cuda", generator=gen).to(dtype).requires_grad_() for n in (5, 7))
    with torch.no_grad():
        ref[3, 2] = 300.0
    idx = torch.full((5, 1), 3, dtype=torch.int32, device="cuda")
    loss = NeighborDistillLoss(64.0, 1.0, "euclidean", "none")(z, ref, idx, torch.zeros(5, 1, device="cuda"))
    a, b = z.detach().double(), ref.detach().double()
    want = -torch.log_softmax((a @ b.t() - 0.5 * (b * b).sum(1)) / 64.0, 1)[:, 3]
    step = {torch.float16: 16.0, torch.bfloat16: 128.0, torch.float32: 2.0 ** -9}[dtype]
    assert bool(((loss.detach().double() - want).abs() <= 2 * step / 64 + 2.0 ** -8).all()), (loss, want)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(loss.sum(), [z, ref]))


@pytest.mark.parametrize("dtype", TYPES)
def test_cosine_neighbors_with_rows_of_zeros(dtype):
    """A row of zeros has similarity 0 to everything: its own loss is log 9, and it is one class like any other.

    The other scores are products of two unit vectors of 16 components, each component and the product rounded to
    the type: 2^-8 (bfloat16) of at most 1 three times, over the temperature; the loss takes two of them."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    z, ref = (torch.randn(n, 16, device="cuda", generator=gen).to(dtype).requires_grad_() for n in (4, 9))
    with torch.no_grad():
        z[1], ref[2] = 0.0, 0.0
    idx = torch.tensor([[2], [5], [0], [8]], dtype=torch.int32, device="cuda")
    loss = NeighborDistillLoss(0.5, 1.0, "cosine", "none")(z, ref, idx, torch.zeros(4, 1, device="cuda"))
    a, b = (torch.nn.functional.normalize(t.detach().double(), dim=1) for t in (z, ref))
    want = -torch.log_softmax(a @ b.t() / 0.5, 1).gather(1, idx.long())[:, 0]
    assert abs(float(want[1]) - math.log(9.0)) < 1e-12
    u = torch.finfo(dtype).eps / 2
    assert bool(((loss.detach().double() - want).abs() <= 12 * u + 2.0 ** -18).all()), (loss, want)
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(loss.sum(), [z, ref]))
