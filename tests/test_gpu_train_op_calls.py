"""Calls of the training operators that their documentation allows beyond the plain ones: layouts and wanted gradients
at the sizes of every kernel, offsets past 32 bits, threads, several captured graphs at once.

Tolerances as in test_gpu_dense.py and test_gpu_distill.py, whose helpers these tests use; where two calls make the same sums
in the same order their results are equal bit for bit."""
import math
import threading

import pytest
import torch

from scmiac_amd.modeling import NeighborDistillLoss, linear_act, top_logits, topk_distill
from test_gpu_dense import TYPES, _check, _make
from test_gpu_distill import _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(1024, 512, 768), (2050, 1600, 328), (1032, 1003, 1047), (3400, 3391, 400)])
def test_relu_in_large_products(m, k, n, dtype):
    _check(m, k, n, dtype, "relu", seed=7)


# the large tiles (of 128 and of 256; float32 from 3 2^30 on), the small ones of both widths, split and not, and a few rows
KINDS = [(2056, 1048, 2000), (3400, 3392, 400), (9000, 3900, 136), (300, 200, 70), (2100, 1031, 29), (13, 10003, 16), (1, 4096, 4097),
         (4, 4096, 4104), (8, 4096, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", KINDS)
def test_each_gradient_alone(m, k, n, dtype):
    x, w, b, res, dy = _make(m, k, n, dtype, seed=2)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    full = torch.autograd.grad(linear_act(*leaves, "silu"), leaves, dy)
    for wanted in [(0,), (1,), (2,), (3,), (0, 2), (1, 2), (0, 1), (0, 3)]:
        t = [v.clone().requires_grad_(i in wanted) for i, v in enumerate((x, w, b, res))]
        grads = torch.autograd.grad(linear_act(*t, "silu"), [t[i] for i in wanted], dy)
        for i, g in zip(wanted, grads):
            assert torch.equal(g, full[i]), (wanted, i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", KINDS)
def test_layouts_of_the_inputs(m, k, n, dtype):
    """Rows apart by a multiple of 16 bytes, by an odd number, starting anywhere, columns apart, one row for all."""
    x, w, b, res, dy = _make(m, k, n, dtype, seed=4)

    def spread(t, before, behind):
        store = torch.full((t.shape[0], t.shape[1] + before + behind), math.nan, dtype=t.dtype, device="cuda")
        store[:, before:before + t.shape[1]] = t
        return store[:, before:before + t.shape[1]]

    def grads_of(*t):
        leaves = [v.detach().requires_grad_() for v in t]
        y = linear_act(leaves[0], leaves[1], b, leaves[2], "gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = grads_of(x, w, res)
    for lay in (lambda t: spread(t, 8, 8), lambda t: spread(t, 0, 1), lambda t: spread(t, 3, 2), lambda t: t.t().contiguous().t()):
        for got, other in zip(grads_of(lay(x), lay(w), lay(res)), want):
            assert torch.equal(got, other)
    one = x[:1].expand(m, k)
    assert torch.equal(linear_act(one, w, b, res), linear_act(one.contiguous(), w, b, res))


def test_more_than_32_bits_of_elements_in_a_layer():
    """36 million rows: the first and the last against 64 bits, the sums over all rows against sums of parts."""
    m, k, n = 36_000_000, 8, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, k, device="cuda", generator=g, dtype=torch.float32).bfloat16().requires_grad_()
    w = (torch.randn(n, k, device="cuda", generator=g) / 3).bfloat16().requires_grad_()
    b = torch.randn(n, device="cuda", generator=g).bfloat16().requires_grad_()
    assert m * n > 2 ** 31
    y = linear_act(x, w, b, activation="relu")
    dy = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(m, n).contiguous()
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    u = 2.0 ** -8
    total_w, total_b = torch.zeros(n, k, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    with torch.no_grad():
        for lo in range(0, m, 4_000_000):
            part = x[lo:lo + 4_000_000].float()
            on = (part @ w.float().t() + b.float() > 0).float()      # (near zero the sums' order may decide: a few of 10^9)
            total_w += (on.t() @ part).double()
            total_b += on.double().sum(0)
        for rows in (slice(0, 5000), slice(m - 5000, m)):
            z = x[rows].double() @ w.double().t() + b.double()
            assert bool(((y[rows].double() - z.clamp(min=0)).abs() <= u * z.abs() + 2.0 ** -18).all())
            sure = (z.abs() > 1e-4).all(1)
            want = (z > 0).double() @ w.double()
            size = (z > 0).double() @ w.double().abs()
            assert bool(((dx[rows].double() - want).abs() <= u * want.abs() + 2.0 ** -16 * size)[sure].all())
    # counts of up to 3.6e7 and sums of that many values in float32 parts: u of the result and 2^-10 of its size for both sides
    assert bool(((db.double() - total_b).abs() <= (u + 2.0 ** -10) * total_b).all())
    assert bool(((dw.double() - total_w).abs() <= u * total_w.abs() + 2.0 ** -10 * total_b[:, None]).all())


def test_more_than_32_bits_of_elements_in_the_logits():
    n, v, k = 30_000, 100_000, 8
    assert n * v > 2 ** 31
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    for lo in range(0, n, 2000):
        x[lo:lo + 2000] = torch.randn(2000, v, device="cuda", generator=g)
    values, idx, lse = top_logits(x, k)
    top = torch.randn(n, k, device="cuda", generator=g)
    leaf = x.requires_grad_()
    loss = topk_distill(leaf, idx, top, reduction="none")
    dx, = torch.autograd.grad(loss, leaf, torch.ones(n, device="cuda"))
    for rows in (slice(0, 3), slice(n // 2, n // 2 + 3), slice(n - 3, n)):
        a = x.detach()[rows].contiguous()
        part = top_logits(a, k)
        assert torch.equal(values[rows], part[0]) and torch.equal(idx[rows], part[1])
        assert bool(((lse[rows].double() - torch.logsumexp(a.double(), 1)).abs() <= 2.0 ** -17).all())
        logp = torch.log_softmax(a.double(), 1)
        t = torch.softmax(top[rows].double(), 1)
        want = (t * (t.log() - logp.gather(1, idx[rows].long()))).sum(1)
        assert bool(((loss.detach()[rows].double() - want).abs() <= 2.0 ** -17 * 20).all())
        p = logp.exp()
        grad = p.clone().scatter_add_(1, idx[rows].long(), -t)
        size = p.scatter_add(1, idx[rows].long(), t)
        assert bool(((dx[rows].double() - grad).abs() <= 2.0 ** -8 * grad.abs() + 2.0 ** -16 * size + 2.0 ** -126).all())


def test_rows_far_apart():
    """A row stride of 2^28 elements: offsets past 32 bits in a few rows, and too long for the large tiles' addresses."""
    store = torch.zeros(10 * 2 ** 28, dtype=torch.bfloat16, device="cuda")
    apart = store.as_strided((10, 3000), (2 ** 28, 1))
    x, w, b, _, _ = _make(10, 3000, 50, torch.bfloat16, seed=1)
    apart.copy_(x)
    assert torch.equal(linear_act(apart, w, b), linear_act(x, w, b))
    assert torch.equal(linear_act(w, apart, None), linear_act(w, x, None))
    assert all(torch.equal(p, q) for p, q in zip(top_logits(apart, 9), top_logits(x, 9)))
    idx, top = torch.randint(0, 3000, (10, 4), device="cuda"), torch.randn(10, 4, device="cuda")
    leaf, flat = apart.detach().requires_grad_(), x.clone().requires_grad_()
    grads = [torch.autograd.grad(topk_distill(t, idx, top), t)[0] for t in (leaf, flat)]
    assert torch.equal(*grads)


def test_batches_without_rows():
    w = torch.randn(5, 64, device="cuda", requires_grad=True)
    x = torch.empty(2, 0, 64, device="cuda", requires_grad=True)
    y = linear_act(x, w, None, torch.empty(2, 0, 5, device="cuda"), "silu")
    assert y.shape == (2, 0, 5)
    dx, dw = torch.autograd.grad(y.sum(), [x, w])
    assert dx.shape == x.shape and not dw.any()
    values, idx, lse = top_logits(x, 3)
    assert values.shape == idx.shape == (2, 0, 3) and lse.shape == (2, 0)
    loss = topk_distill(x, torch.empty(2, 0, 3, dtype=torch.int64, device="cuda"), torch.empty(2, 0, 3, device="cuda"), 1.0,
                        torch.empty(2, 0, device="cuda"), reduction="none")
    assert loss.shape == (2, 0) and torch.autograd.grad(loss.sum(), x)[0].shape == x.shape


def test_one_row_of_logits_for_all():
    x, idx, top, _ = _rand(6, 3000, 4, torch.float32, seed=1)
    leaf = x[:1].clone().requires_grad_()
    loss = topk_distill(leaf.expand(6, 3000), idx, top)
    got, = torch.autograd.grad(loss, leaf)
    flat = x[:1].expand(6, 3000).contiguous().requires_grad_()
    want, = torch.autograd.grad(topk_distill(flat, idx, top), flat)
    assert torch.equal(got, want.sum(0, keepdim=True))


def test_threads_at_once():
    """Calls from several threads, each on a stream of its own."""
    data = []
    for i, (m, k, n) in enumerate([(700, 1500, 40), (2056, 1048, 2000), (3, 4100, 4099), (300, 64, 20000)]):
        x, w, b, res, dy = _make(m, k, n, torch.bfloat16, seed=i)
        table = top_logits(dy, 7)
        data.append((x, w, b, res, dy, table))

    def work(x, w, b, res, dy, table):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, res)]
        y = linear_act(*leaves, "gelu")
        loss = topk_distill(y, table[1], table[0], 2.0)
        return [y.detach(), *torch.autograd.grad(loss, leaves), *top_logits(y, 5)]

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got[i] = [work(*data[i % len(data)]) for _ in range(10)]
            stream.synchronize()
        except Exception as e:      # noqa: BLE001 (shown below)
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i, runs in got.items():
        for one in runs:
            assert all(torch.equal(p, q) for p, q in zip(one, want[i % len(data)]))


def test_two_graphs_of_a_training_step_replayed_in_turn():
    """Encoder layer, scores and loss, forward and backward, captured twice and replayed alternately with eager work between."""
    g = torch.Generator(device="cuda").manual_seed(4)
    steps = []
    for m in (256, 1040):
        leaves = [torch.randn(*s, device="cuda", generator=g).requires_grad_() for s in ((m, 50), (128, 50), (128,), (3001, 128))]
        idx = torch.randint(0, 3001, (m, 12), device="cuda", generator=g, dtype=torch.int32)
        dist = torch.rand(m, 12, device="cuda", generator=g)

        def step(leaves=leaves, idx=idx, dist=dist):
            h = linear_act(leaves[0], leaves[1], leaves[2], activation="silu")
            loss = NeighborDistillLoss(0.5, 1.0, "euclidean")(h, leaves[3], idx, -dist)
            grads = torch.autograd.grad(loss, leaves)
            return [loss.detach(), *grads]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        steps.append((graph, out, step, leaves))
    for turn in range(4):
        for graph, _, _, leaves in steps:
            with torch.no_grad():
                leaves[0].normal_(generator=g)
            graph.replay()
        torch.cuda.synchronize()
        for _, out, step, _ in steps:
            eager = step()
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), turn
        torch.cuda.synchronize()


@pytest.mark.parametrize("start", [0, 1])
def test_rows_of_as_many_classes_as_there_may_be(start):
    """2^31 - 1 classes: positions of lanes behind the end of the row pass 31 bits."""
    v = 2 ** 31 - 1 - start
    x = torch.full((1, 2 ** 31 - 1), -2.0, dtype=torch.bfloat16, device="cuda")[:, start:]
    at = [v - 1, 0, 12345, v // 2, v - 2, v - 6, v - 9, 2 ** 30 + 1]
    for rank, j in enumerate(at):
        x[0, j] = 30.0 - 2 * rank
    values, idx, lse = top_logits(x, 10)
    assert idx[0, :8].tolist() == at and values[0, :8].tolist() == [30.0 - 2 * r for r in range(8)]
    assert idx[0, 8:].tolist() == [1, 2] and values[0, 8:].tolist() == [-2.0, -2.0]
    want = math.log(sum(math.exp(30.0 - 2 * r) for r in range(8)) + (v - 8) * math.exp(-2.0))
    # 2^31 equal terms: a lane adds up 2^31 / 2^16 of them, each addition off by up to 2^-24 of the sum
    assert abs(float(lse) - want) < 2.0 ** -9
    table = torch.tensor([[v - 1, 0, v, v // 2]], device="cuda")
    assert torch.isnan(topk_distill(x, table, torch.zeros(1, 4, device="cuda"), reduction="none")).all()      # v is no class
    table[0, 2] = v - 2
    leaf = x.requires_grad_()
    loss = topk_distill(leaf, table, torch.zeros(1, 4, device="cuda"), reduction="none")
    dx, = torch.autograd.grad(loss, leaf, torch.ones(1, device="cuda"))
    scores = [30.0, 28.0, 22.0, 24.0]
    assert abs(loss.item() - (want - sum(scores) / 4 - math.log(4.0))) < 2.0 ** -9
    for j, s in zip(table[0].tolist(), scores):
        p = math.exp(s - want)
        assert abs(float(dx[0, j]) - (p - 0.25)) <= 2.0 ** -8 * abs(p - 0.25) + 2.0 ** -9


@pytest.mark.parametrize("dtype,scale", [(torch.float16, 1e-6), (torch.bfloat16, 1e-39), (torch.float32, 1e-30), (torch.float32, 1e-36),
                                         (torch.float32, 1e-39)])
@pytest.mark.parametrize("m,k,n", [(2056, 1048, 2000), (300, 200, 70), (1, 4096, 4097), (4, 4096, 4104)])
def test_small_and_denormal_inputs_count(m, k, n, dtype, scale):
    """x and dy of numbers at or below the type's smallest normal one, w large: nothing is taken for zero.  In the large layer a
    float32 value is three bfloat16 planes, which end at 2^-133: off by half of that where its own digits go further."""
    g = torch.Generator(device="cuda").manual_seed(m)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g, dtype=torch.float64)  # noqa: E731
    x, dy = ((r(*s) * scale).to(dtype) for s in ((m, k), (m, n)))
    w = (r(n, k) * (1000.0 if dtype == torch.float16 else 1e12)).to(dtype)
    leaf = x.requires_grad_()
    y = linear_act(leaf, w)
    dx, = torch.autograd.grad(y, leaf, dy)
    u, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    large = dtype == torch.float32 and m > 1000
    for got, a, b in ((y.detach(), x.detach().double(), w.double().t().contiguous()), (dx, dy.double(), w.double())):
        want, size = a @ b, a.abs() @ b.abs()
        bound = u * want.abs() + tiny + a.shape[1] * 2.0 ** -23 * size + (2.0 ** -134 * b.abs().sum(0) if large else 0)
        assert bool(((got.double() - want).abs() <= bound).all())
        assert bool((got != 0)[want.abs() > 4 * bound].all())
