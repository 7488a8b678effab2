"""linear_act -- product, bias, activation and residual in one -- against the same formula in 64 bits.

Tolerances: a type's rounding is at most half a step, u = finfo.eps / 2 of the value.  A sum of c products in
float32 is off by at most c 2^-23 of the sum of their magnitudes (any order, any rounding of the additions).
Element by element the outputs may differ by that bound plus their own rounding.  dz = dy act'(z) also inherits
the error of z: the sum's, through |act''| <= 0.8, and in the half types the rounding of the kept z, which moves the
slope by at most u |z act''(z)| <= 0.3 u (gelu: |z phi(z) (2 - z^2)| peaks at 0.29, silu's at 0.24), each times |dy|;
that dz is then summed into dx, dweight and dbias.  Over a whole tensor the roundings do not add up in one
direction, so its error's norm is within u (y: the output's rounding), 2 u (dbias: z's, too) or 3 u (dx, dweight: z's,
dz's and the output's) of its own norm, and float32's 2^-21 for the sums."""
import math

import pytest
import torch

from scmiac_amd.modeling import LinearAct, linear_act

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "gelu", "silu"]


def _make(m, k, n, dtype, seed=0, bias=True, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 131 + k * 17 + n)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, w = r(m, k).to(dtype), (r(n, k) / math.sqrt(k)).to(dtype)
    b = r(n).to(dtype) if bias else None
    res = r(m, n).to(dtype) if residual else None
    return x, w, b, res, r(m, n).to(dtype)


def _wide(x, w, b, res, dy, act):
    """(outputs, bounds on the sums) in 64 bits."""
    d, x_type = torch.float64, x.dtype
    x, w, dy = x.to(d), w.to(d), dy.to(d)
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.to(d), size + b.to(d).abs()
    half = x_type != torch.float32
    drift = dy.abs() * (0.8 * (x.shape[1] + 2) * 2.0 ** -23 * size + 2.0 ** -21 + (0.3 * torch.finfo(x_type).eps / 2 if half else 0))
    if act in ("none", "relu"):
        drift = torch.zeros_like(drift)
    if act == "none":
        y, s = z, torch.ones_like(z)
    elif act == "relu":
        y, s = z.clamp(min=0), (z > 0).to(d)
    elif act == "gelu":
        p = torch.special.ndtr(z)
        y, s = z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        p = torch.sigmoid(z)
        y, s = z * p, p + z * p * (1 - p)
    if res is not None:
        y = y + res.to(d)
        size = size + res.to(d).abs()
    dz = dy * s
    out = {"y": y, "dx": dz @ w, "dw": dz.t() @ x, "db": dz.sum(0)}
    sizes = {"y": size, "dx": dz.abs() @ w.abs(), "dw": dz.abs().t() @ x.abs(), "db": dz.abs().sum(0)}
    drifts = {"y": torch.zeros_like(y), "dx": drift @ w.abs(), "dw": drift.t() @ x.abs(), "db": drift.sum(0)}
    return out, {name: (sizes[name], drifts[name]) for name in out}


def _compare(got, want, sizes, counts, dtype, label):
    u = torch.finfo(dtype).eps / 2
    for name, t in got.items():
        if t is None:
            continue
        assert t.dtype == dtype and t.shape == want[name].shape, (label, name)
        if t.numel() == 0:
            continue
        err = (t.double() - want[name]).abs()
        size, drift = sizes[name]
        roundings = {"y": 1, "db": 2}.get(name, 3)
        inner = u if roundings == 3 and dtype != torch.float32 else 0          # dz's own rounding
        # gelu and silu amplify an error of z by at most 1.13, and add a few float32 steps of their own
        bound = u * want[name].abs() + (1.13 * counts[name] * 2.0 ** -23 + 2.0 ** -21 + inner) * size + drift \
            + torch.finfo(dtype).smallest_normal
        assert bool((err <= bound).all()), (label, name, float((err / bound).max()))
        if t.numel() >= 256:
            assert float(err.norm()) <= (roundings * u + 2.0 ** -21) * float(want[name].norm()), (label, name)


def _check(m, k, n, dtype, act, bias=True, residual=True, seed=0):
    x, w, b, res, dy = _make(m, k, n, dtype, seed, bias, residual)
    if act == "relu":      # no pre-activation within a rounding of zero, where the slope jumps
        z = x.double() @ w.double().t() + (0 if b is None else b.double())
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    want, sizes = _wide(x, w, b, res, dy, act)
    leaves = [t.requires_grad_() for t in (x, w, b, res) if t is not None]
    y = linear_act(x, w, b, res, act)
    grads = list(torch.autograd.grad(y, leaves, dy))
    got = {"y": y.detach(), "dx": grads[0], "dw": grads[1], "db": grads[2] if bias else None}
    if residual:
        assert torch.equal(grads[-1], dy)
    _compare(got, want, sizes, {"y": k + 2, "dx": n, "dw": m, "db": m}, dtype, (m, k, n, dtype, act))
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, res, act), y)      # the same numbers without a graph
    again = torch.autograd.grad(linear_act(x, w, b, res, act), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))   # and bit for bit on a repeat


SHAPES = [(1, 1, 1), (1, 64, 7), (2, 8, 64), (3, 5, 129), (64, 64, 64), (65, 33, 63), (256, 50, 128), (257, 200, 70),
          (1, 4096, 300), (5, 1000, 1030), (16, 513, 2049), (300, 2000, 17), (2000, 30, 515), (4097, 64, 30),
          (2049, 31, 1030), (150001, 30, 29), (13, 100003, 16), (2100, 7, 1001), (2100, 1031, 29), (5000, 421, 32),
          (4, 1030, 1100), (3, 4100, 4099), (7, 4101, 4099), (8, 4096, 4096), (1, 4097, 4099), (2, 4096, 4100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_shapes(m, k, n, dtype):
    act = ACTS[(m + k + n) % 4]
    _check(m, k, n, dtype, act, bias=m % 2 == 1 or n % 2 == 0, residual=(m + n) % 3 != 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype):
    _check(130, 96, 100, dtype, act, seed=3)


# products large enough for the big tiles: whole tiles, a few rows over, odd widths that need padding
LARGE = [(1024, 512, 768), (1025, 511, 769), (2100, 320, 1000), (520, 1600, 514), (300, 4100, 1100),
         # ends of rows and columns within a step of 64 and a tile, read as they lie or packed
         (1003, 520, 1032), (1031, 1048, 1032), (777, 1032, 1352), (2050, 1600, 328), (1032, 1003, 1047),
         # large in float32, too; few splits and many; tiles of 256 x 256 forward, of dx and of dw
         (2056, 1048, 2001), (1100, 4100, 960), (9000, 3900, 130), (3390, 400, 3401), (3400, 3391, 400), (400, 3392, 3400)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", LARGE)
def test_large_products(m, k, n, dtype):
    _check(m, k, n, dtype, ["gelu", "none", "silu"][(m + n) % 3], seed=5)


def test_strides_leading_dimensions_and_offsets():
    for dtype in TYPES:
        big = torch.randn(40, 130, device="cuda").to(dtype)
        w_all = torch.randn(50, 99, device="cuda").to(dtype)
        b, res_all = torch.randn(50, device="cuda").to(dtype), torch.randn(40, 60, device="cuda").to(dtype)
        for x, w, res in [(big[:, 3:67], w_all[:, 1:65], res_all[:, 5:55]),          # rows apart, odd starts
                          (big[::2, :64], w_all[:, :64], res_all[:20, :50]),
                          (big[:64].t()[:64, :40], w_all[:, :40], None),             # columns apart
                          (big[:1, :64].expand(40, 64), w_all[:, :64], res_all[:, :50])]:
            got = linear_act(x, w, b, res, "silu")
            want = linear_act(x.contiguous(), w.contiguous(), b, None if res is None else res.contiguous(), "silu")
            assert torch.equal(got, want)
        x4 = torch.randn(2, 3, 5, 64, device="cuda").to(dtype)
        r4 = torch.randn(2, 3, 5, 50, device="cuda").to(dtype)
        y = linear_act(x4, w_all[:, :64], b, r4, "gelu")
        assert y.shape == (2, 3, 5, 50)
        assert torch.equal(y.view(30, 50), linear_act(x4.view(30, 64), w_all[:, :64], b, r4.view(30, 50), "gelu"))
        assert linear_act(x4[0, 0, 0], w_all[:, :64], b).shape == (50,)


def test_gradients_of_views_and_broadcast_inputs():
    base = torch.randn(1, 48, device="cuda", requires_grad=True)
    w = torch.randn(20, 48, device="cuda", requires_grad=True)
    b = torch.randn(20, device="cuda", requires_grad=True)
    y = linear_act(base.expand(33, 48), w, b, activation="silu")
    y.sum().backward()                                                   # an expanded gradient, too
    got = base.grad.clone(), w.grad.clone(), b.grad.clone()
    # against 64 bits.  dz = silu'(z) with z a sum of 49 terms, silu'' <= 0.5: off by at most d below; a gradient sums up to
    # 33 x 20 products with dz in float32, each addition off by 2^-23 of the magnitudes' sum
    x64, w64, b64 = (t.detach().double() for t in (base.expand(33, 48), w, b))
    z = x64 @ w64.t() + b64
    s = torch.sigmoid(z)
    dz = s + z * s * (1 - s)
    d = 0.5 * 50 * 2.0 ** -23 * (x64.abs() @ w64.abs().t() + b64.abs()) + 2.0 ** -21
    size = dz.abs() * 33 * 20 * 2.0 ** -23 + d
    for g, want, bound in zip(got, ((dz @ w64).sum(0, keepdim=True), dz.t() @ x64, dz.sum(0)),
                              ((size @ w64.abs()).sum(0, keepdim=True), size.t() @ x64.abs(), size.sum(0))):
        assert bool(((g - want).abs() <= bound).all())


def test_only_the_wanted_gradients():
    x, w, b, res, dy = _make(70, 40, 90, torch.float32)
    full = None
    for wanted in [(0, 1, 2, 3), (0,), (1,), (2,), (3,), (1, 2)]:
        t = [v.clone().requires_grad_(i in wanted) for i, v in enumerate((x, w, b, res))]
        grads = torch.autograd.grad(linear_act(*t, "gelu"), [t[i] for i in wanted], dy)
        full = full or grads
        for i, g in zip(wanted, grads):
            assert torch.equal(g, full[i])


def test_no_rows_and_not_finite_values():
    x = torch.empty(0, 6, device="cuda", requires_grad=True)
    w = torch.randn(4, 6, device="cuda", requires_grad=True)
    b = torch.randn(4, device="cuda", requires_grad=True)
    y = linear_act(x, w, b, activation="relu")
    assert y.shape == (0, 4)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 4, device="cuda"))
    assert dx.shape == (0, 6) and not dw.any() and not db.any() and dw.shape == (4, 6)
    for dtype in TYPES:      # a row that is not finite stays alone
        x, w, b, _, _ = _make(70, 64, 66, dtype)
        x[3, 5], x[9, 0] = math.inf, math.nan
        y = linear_act(x, w, b, activation="none")
        bad = ~torch.isfinite(y).all(1)
        assert bad.nonzero().flatten().tolist() == [3, 9]
        assert torch.isnan(y[9]).all() and not torch.isfinite(y[3]).any()
        assert torch.isnan(linear_act(x, w, b, activation="relu")[9]).all()


def test_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(6, 9, device="cuda", generator=g)
    w = torch.randn(5, 9, device="cuda", generator=g) / 3
    b = torch.randn(5, device="cuda", generator=g)
    dy = torch.randn(6, 5, device="cuda", generator=g)
    for act in ("gelu", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(linear_act(*leaves, activation=act), leaves, dy)
        h = 2.0 ** -6
        for i, t in enumerate((x, w, b)):
            flat = t.view(-1)
            for e in range(0, flat.numel(), 7):
                vals = []
                for sign in (1, -1):
                    moved = [v.clone() for v in (x, w, b)]
                    moved[i].view(-1)[e] += sign * h
                    vals.append(float((linear_act(*moved, activation=act).double() * dy.double()).sum()))
                # central differences: h^2 / 6 of a third derivative below 20 here, and float32 sums over 2 h
                assert abs((vals[0] - vals[1]) / (2 * h) - float(grads[i].view(-1)[e])) < 2e-3


def test_module_streams_and_capture():
    torch.manual_seed(0)
    layer = LinearAct(64, 48, activation="silu", device="cuda")
    plain = torch.nn.Linear(64, 48, device="cuda")
    plain.load_state_dict(layer.state_dict())
    x, res = torch.randn(300, 64, device="cuda"), torch.randn(300, 48, device="cuda")
    want = torch.nn.functional.silu(plain(x)) + res
    torch.testing.assert_close(layer(x, res), want, rtol=1e-5, atol=1e-5)
    assert "silu" in repr(layer)
    # two streams at once: no scratch in common
    big = [torch.randn(700, 1500, device="cuda") for _ in range(2)]
    w = torch.randn(40, 1500, device="cuda")
    want = [linear_act(t, w, activation="gelu") for t in big]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(linear_act(big[i], w, activation="gelu"))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])
    # forward and backward in a graph, replayed on new inputs with eager work in between
    leaves = [t.detach().clone().requires_grad_() for t in (big[0], w)]
    dy = torch.randn(700, 40, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(linear_act(*leaves, activation="gelu"), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear_act(*leaves, activation="gelu")
        grads = torch.autograd.grad(y, leaves, dy)
    y = y.detach()
    for step in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(700, 1500, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = [t.detach().clone().requires_grad_() for t in leaves]
        yy = linear_act(*eager, activation="gelu")
        assert torch.equal(y, yy)
        assert all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(yy, eager, dy)))
        torch.cuda.synchronize()


def test_half_precision_pre_activations_beyond_the_type():
    # z of +-70 000 and +-1e5 is no float16; the outputs are 0 or (rightly) infinite, and the slopes 0 or 1
    x = torch.tensor([[-300.0], [300.0], [-400.0], [1.0]], device="cuda", dtype=torch.float16)
    w = torch.full((3, 1), 250.0, device="cuda", dtype=torch.float16)
    for act in ("relu", "gelu", "silu"):
        xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = linear_act(xx, ww, activation=act)
        dx, dw = torch.autograd.grad(y, [xx, ww], torch.ones_like(y))
        assert not y[0].any() and not y[2].any() and torch.isinf(y[1]).all()
        assert dx.flatten().tolist() == [0.0, 750.0, 0.0, 750.0] and dw.flatten().tolist() == [301.0] * 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", [(40, 96, 70), (2056, 1048, 2001)])
def test_what_is_not_finite_stays_in_its_row(m, k, n, dtype):
    x, w, b, _, dy = _make(m, k, n, dtype, seed=11, residual=False)
    clean = linear_act(x, w, b)
    for bad in (math.inf, -math.inf, math.nan):
        spoilt = x.clone()
        spoilt[m // 2, k - 1] = bad
        y = linear_act(spoilt, w, b)
        hit = w[:, k - 1] != 0
        assert not torch.isfinite(y[m // 2][hit]).any()
        rest = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(y[rest], clean[rest])
        leaf = spoilt.requires_grad_()
        weight = w.clone().requires_grad_()
        dx, dw = torch.autograd.grad(linear_act(leaf, weight, b), (leaf, weight), dy)
        assert torch.isfinite(dx).all() and torch.isfinite(dw[:, :k - 1]).all()
        assert not torch.isfinite(dw[dy[m // 2] != 0, k - 1]).any()


@pytest.mark.parametrize("trained", ["w", "b", "wb", "x", "xw", "xwb"])
def test_second_derivatives_are_refused_whatever_is_trained(trained):
    t = {"x": torch.randn(6, 5, device="cuda"), "w": torch.randn(4, 5, device="cuda"), "b": torch.randn(4, device="cuda")}
    leaves = [t[name].requires_grad_() for name in trained]
    for act in ACTS:
        y = linear_act(t["x"], t["w"], t["b"], activation=act)
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
        for g, same in zip(grads, torch.autograd.grad(linear_act(t["x"], t["w"], t["b"], activation=act), leaves, torch.ones_like(y))):
            assert torch.equal(g, same)
        for g in grads:      # a penalty on a gradient, beside a term that has a derivative of its own
            for leaf in leaves:
                with pytest.raises(RuntimeError, match="differentiable twice"):
                    torch.autograd.grad(g.square().sum() + leaf.sum(), leaf, retain_graph=True)
    # a recorded pass is no harm where no second derivative is asked for
    y = linear_act(t["x"], t["w"], t["b"], activation="gelu")
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y.sum(), leaves, create_graph=True))


def test_the_gradient_of_the_residual_keeps_its_derivatives():
    x, w, dy = (torch.randn(*s, device="cuda", requires_grad=True) for s in ((6, 5), (4, 5), (6, 4)))
    res = torch.randn(6, 4, device="cuda", requires_grad=True)
    y = linear_act(x, w, None, res, "gelu")
    dx, dres = torch.autograd.grad(y, [x, res], dy, create_graph=True)
    assert torch.equal(dres, dy)
    g, = torch.autograd.grad((dres * 3).sum(), dy, retain_graph=True)      # dres is dy: a derivative of 1
    assert torch.equal(g, torch.full_like(dy, 3.0))
    with pytest.raises(RuntimeError, match="differentiable twice"):
        torch.autograd.grad(dx.sum(), dy)
    y = linear_act(x.detach(), w.detach(), None, res)
    dres, = torch.autograd.grad(y, res, dy, create_graph=True)
    assert torch.equal(torch.autograd.grad((dres * 2).sum(), dy)[0], torch.full_like(dy, 2.0))


def test_float32_gelu_keeps_its_digits_where_it_is_small():
    """z = x * 1 is exact here.  P(z) = exp(-z^2 / 2) times a smooth factor: the exponent (46 as a power of two at z = -8)
    carries three roundings, 46 x 0.7 x 3 x 2^-24 < 2^-17, the factor less than 2^-20: 2^-16 of gelu in all.  In the slope, P + z phi,
    the two terms of opposite sign add up to 1.3 times the sum at most: 2^-15."""
    z = torch.linspace(-8, -3, 501, device="cuda").reshape(-1, 1).requires_grad_()
    y = linear_act(z, torch.ones(1, 1, device="cuda"), activation="gelu")
    slope, = torch.autograd.grad(y, z, torch.ones_like(y))
    d = z.detach().double()
    p = torch.special.erfc(-d / math.sqrt(2)) / 2
    want = p + d * torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
    assert bool(((y.detach().double() - d * p).abs() <= 2.0 ** -16 * (d * p).abs()).all())
    assert bool(((slope.double() - want).abs() <= 2.0 ** -15 * want.abs()).all())


def test_views_with_a_pending_negation():
    neg = torch._neg_view
    x, w, b, res, dy = _make(70, 40, 90, torch.float32)
    for i in range(4):
        args, want = [x, w, b, res], [x, w, b, res]
        args[i], want[i] = neg(args[i]), -want[i]
        assert torch.equal(linear_act(*args, "silu"), linear_act(*want, "silu")), i
    # as they come about: the imaginary part of a conjugate
    z = torch.randn(70, 1, dtype=torch.complex64, device="cuda").conj().imag
    assert z.is_neg() and torch.equal(linear_act(z, w[:, :1]), linear_act(z.clone(), w[:, :1]))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = [torch.autograd.grad(linear_act(*leaves, activation="silu"), leaves, g) for g in (neg(dy), -dy)]
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    leaf = x.clone().requires_grad_()
    through, = torch.autograd.grad(linear_act(neg(leaf), w), leaf, dy)
    straight = (-x).requires_grad_()
    assert torch.equal(through, -torch.autograd.grad(linear_act(straight, w), straight, dy)[0])


def test_float32_gelu_over_its_range():
    """From -1 on P(z) is 1/2 + z r(z^2), or 1 - q with q < 0.16: fits of 4e-8 and 8e-8 and a few roundings of 2^-24, of at least
    0.159 at z = -1, so 2^-21 of gelu in all; of the slope, whose terms are at most 1.13, 2^-21."""
    z = torch.cat([torch.linspace(-1, 9, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-6, -1e-6, 40.0, 1e30])]).reshape(-1, 1).cuda()
    z.requires_grad_()
    y = linear_act(z, torch.ones(1, 1, device="cuda"), activation="gelu")
    slope, = torch.autograd.grad(y, z, torch.ones_like(y))
    d = z.detach().double()
    p = torch.special.erfc(-d / math.sqrt(2)) / 2
    assert bool(((y.detach().double() - d * p).abs() <= 2.0 ** -21 * (d * p).abs()).all())
    want = p + d * torch.exp(-d * d / 2) / math.sqrt(2 * math.pi)
    assert bool(((slope.double() - want).abs() <= 2.0 ** -21).all())
    assert linear_act(torch.full((1, 1), math.inf, device="cuda"), torch.ones(1, 1, device="cuda"), activation="gelu").item() == math.inf
