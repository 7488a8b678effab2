"""What the training-side operators refuse, without a GPU: the C ABI's argument checks (they come before
anything touches a device) and the Python layer's."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from scmiac_amd import _hip
from scmiac_amd.modeling import LinearAct, NeighborDistillLoss, linear_act, top_logits, topk_distill

F32, F16, BF16 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    return _hip.load_library()


def _error(lib):
    return lib.scmiac_last_error().decode()


def test_linear_sizes_and_refusals(lib):
    n = ctypes.c_size_t(0)
    size = lib.scmiac_linear_workspace_size
    for args in [(0, 1, 1, F32, 0, 0), (0, 1, 1, F32, 0, 1), (256, 128, 50, F32, 1, 1), (8192, 4096, 4096, BF16, 2, 1),
                 (1, 16384, 4096, F16, 3, 0), (2 ** 24, 30, 50, F32, 0, 1)]:
        assert size(*args, ctypes.byref(n)) == 0, _error(lib)
    for args, word in [((4, 0, 4, F32, 0, 0), "n=0"), ((4, 4, 0, F32, 0, 0), "k=0"), ((-1, 4, 4, F32, 0, 0), "m=-1"),
                       ((4, 4, 4, 3, 0, 0), "dtype=3"), ((4, 4, 4, F32, 4, 0), "act=4"), ((4, 4, 4, F32, -1, 0), "act=-1"),
                       ((2 ** 31, 4, 4, F32, 0, 0), "2^31"), ((2 ** 20, 2 ** 20, 4, F32, 0, 0), "tiles")]:
        assert size(*args, ctypes.byref(n)) == 1 and word in _error(lib), (args, _error(lib))
    assert size(4, 4, 4, F32, 0, 0, None) == 1
    p = 4096       # never read: every call below is refused first
    assert lib.scmiac_linear_forward(None, 4, p, 4, None, None, 0, 4, 4, 4, F32, 0, p, None, None, 0, None) == 1
    assert lib.scmiac_linear_forward(p, -4, p, 4, None, None, 0, 4, 4, 4, F32, 0, p, None, None, 0, None) == 1
    assert lib.scmiac_linear_backward(p, 4, p, 4, None, p, 4, 4, 4, F32, 2, p, p, p, None, 0, None) == 1    # gelu without z
    assert lib.scmiac_linear_backward(None, 4, p, 4, p, p, 4, 4, 4, F32, 2, p, p, p, None, 0, None) == 1    # dw without x
    assert size(64, 64, 65536, F32, 0, 0, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.scmiac_linear_forward(p, 65536, p, 65536, None, None, 0, 64, 64, 65536, F32, 0, p, None, p, n.value - 1, None) == 2
    assert "needed" in _error(lib)
    assert lib.scmiac_linear_forward(None, 0, None, 0, None, None, 0, 0, 4, 4, F32, 0, None, None, None, 0, None) == 0   # no rows


def test_top_logits_and_distill_refusals(lib):
    n = ctypes.c_size_t(0)
    top = lib.scmiac_top_logits_workspace_size
    assert top(0, 10, 5, F32, ctypes.byref(n)) == 0 and n.value == 0
    assert top(1, 1000000, 64, F32, ctypes.byref(n)) == 0 and n.value > 0
    for args in [(1, 10, 0, F32), (1, 10, 65, F32), (1, 0, 1, F32), (-1, 10, 1, F32), (2 ** 24, 10, 1, F32), (1, 2 ** 31, 1, F32),
                 (1, 10, 1, 7)]:
        assert top(*args, ctypes.byref(n)) == 1, args
    p = 4096
    assert lib.scmiac_top_logits(None, 10, 1, 10, F32, 4, 1.0, p, p, p, None, 0, None) == 1
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert lib.scmiac_top_logits(p, 10, 1, 10, F32, 4, bad, p, p, p, None, 0, None) == 1
        assert lib.scmiac_distill_forward(p, 10, 1, 10, F32, p, p, 4, None, bad, 1.0, 0, p, p, None, p, 999, None) == 1
        assert lib.scmiac_distill_forward(p, 10, 1, 10, F32, p, p, 4, None, 1.0, bad, 0, p, p, None, p, 999, None) == 1
        assert "temperature" in _error(lib)
    size = lib.scmiac_distill_workspace_size
    assert size(0, 10, F32, ctypes.byref(n)) == 0 and n.value == 0
    assert size(8192, 100000, BF16, ctypes.byref(n)) == 0
    assert size(1, 0, F32, ctypes.byref(n)) == 1 and size(2 ** 24, 4, F32, ctypes.byref(n)) == 1
    fwd = lib.scmiac_distill_forward
    assert fwd(p, 10, 1, 10, F32, p, p, 0, None, 1.0, 1.0, 0, p, p, None, p, 999, None) == 1
    assert fwd(p, 10, 1, 10, F32, p, p, 1025, None, 1.0, 1.0, 0, p, p, None, p, 999, None) == 1 and "1024" in _error(lib)
    assert fwd(p, 10, 1, 10, F32, p, p, 4, None, 1.0, 1.0, 3, p, p, p, p, 999, None) == 1 and "REDUCE" in _error(lib)
    assert fwd(p, 10, 1, 10, F32, p, p, 4, None, 1.0, 1.0, 1, p, p, None, p, 999, None) == 1      # mean without scale
    assert fwd(p, 10, 1, 10, F32, None, p, 4, None, 1.0, 1.0, 0, p, p, None, p, 999, None) == 1
    assert fwd(p, 10, 1, 10, F32, p, p, 4, None, 1.0, 1.0, 0, p, p, None, p, 4, None) == 2
    assert fwd(None, 0, 0, 10, F32, None, None, 4, None, 1.0, 1.0, 0, None, None, None, None, 0, None) == 0
    bwd = lib.scmiac_distill_backward
    assert bwd(p, 10, 2, 10, F32, p, p, 4, 1.0, 1.0, p, p, 0, None, p, 9, None) == 1 and "overlap" in _error(lib)
    assert bwd(p, 10, 2, 10, F32, p, p, 4, 1.0, 1.0, p, p, -1, None, p, 10, None) == 1
    assert bwd(p, 10, 2, 10, F32, p, p, 4, 1.0, 1.0, None, p, 0, None, p, 10, None) == 1


def test_host_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    idx, top = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for call in (lambda: linear_act(x, w), lambda: top_logits(x, 2), lambda: topk_distill(x, idx, top),
                 lambda: NeighborDistillLoss()(x, w, idx, top), lambda: LinearAct(8, 3)(x), lambda: top_logits([1.0], 1)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_constructor_refusals():
    with pytest.raises(ValueError, match="activation"):
        LinearAct(4, 4, activation="tanh")
    with pytest.raises(ValueError, match="metric"):
        NeighborDistillLoss(metric="dot")


@pytest.mark.gpu
def test_python_refusals_of_device_tensors():
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(3, 8, device="cuda")
    b, r = torch.zeros(3, device="cuda"), torch.zeros(4, 3, device="cuda")
    for args, kind in [((x.double(), w.double()), TypeError), ((x, w.half()), TypeError), ((x, w, b.half()), TypeError),
                       ((x, w, b, r.half()), TypeError), ((x, w[:, :7]), ValueError), ((x, w[0]), ValueError),
                       ((x, w, b[:2]), ValueError), ((x, w, b, r[:2]), ValueError), ((x, w, b, r[:1]), ValueError),
                       ((x, w, b.cpu()), ValueError), ((x, None), ValueError), ((x, w, b, r, "tanh"), ValueError),
                       ((x[:, :0], w[:, :0]), ValueError), ((x, w[:0]), ValueError)]:
        with pytest.raises(kind):
            linear_act(*args)
    for call in (lambda: top_logits(x.double(), 2), lambda: top_logits(x.int(), 2)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: top_logits(x, 0), lambda: top_logits(x, 65), lambda: top_logits(x[:, :0], 1),
                 lambda: top_logits(x, 2, temperature=0.0), lambda: top_logits(x, 2, temperature=float("nan"))):
        with pytest.raises(ValueError):
            call()
    idx, top, lse = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda"), torch.zeros(4, device="cuda")
    for args, kind in [((x.double(), idx, top), TypeError), ((x, top, top), TypeError), ((x, idx, idx), TypeError),
                       ((x, idx.bool(), top), TypeError), ((x, idx[:3], top[:3]), ValueError), ((x, idx, top[:, :1]), ValueError),
                       ((x, idx[:, :0], top[:, :0]), ValueError), ((x, idx.cpu(), top), ValueError), ((x, idx[0], top[0]), ValueError),
                       ((x, idx, top, 0.0), ValueError), ((x, idx, top, 1.0, lse[:3]), ValueError), ((x, idx, top, 1.0, lse, -1.0), ValueError),
                       ((x, idx, top, 1.0, None, None, "batchmean"), ValueError), ((x, idx, top.clone().requires_grad_()), ValueError),
                       ((x, idx, top, 1.0, lse.clone().requires_grad_()), ValueError)]:
        with pytest.raises(kind):
            topk_distill(*args)
    wide = torch.zeros(4, 1025, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        topk_distill(x, wide, wide.float())
    for leaf, out in ((x.clone().requires_grad_(), lambda t: linear_act(t, w).sum()),
                      (x.clone().requires_grad_(), lambda t: topk_distill(t, idx, top))):
        g, = torch.autograd.grad(out(leaf), [leaf], create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), [leaf])


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    x, w, b, r = (torch.randn(*s, device="cuda") for s in ((6, 5), (4, 5), (4,), (6, 4)))
    idx, top = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.zeros(6, 2, device="cuda")
    lse = torch.zeros(6, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: linear_act(dual(x), w, b, r), lambda: linear_act(x, dual(w), b, r), lambda: linear_act(x, w, dual(b), r),
                     lambda: linear_act(x, w, b, dual(r)), lambda: topk_distill(dual(x), idx, top),
                     lambda: topk_distill(x, idx, dual(top)), lambda: topk_distill(x, idx, top, 1.0, dual(lse)),
                     lambda: NeighborDistillLoss()(dual(x), w, idx, top)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        values, _, _ = top_logits(dual(x), 2)                       # a teacher is a constant
        assert forward_ad.unpack_dual(values).tangent is None
        linear_act(x, w, b, r), topk_distill(x, idx, top)           # without tangents as ever


@pytest.mark.gpu
def test_tracing_is_refused():
    x, w = torch.randn(6, 5, device="cuda"), torch.randn(4, 5, device="cuda")
    idx, top = torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.zeros(6, 2, device="cuda")
    for call in (lambda t: linear_act(t, w), lambda t: top_logits(t, 2), lambda t: topk_distill(t, idx, top)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (x,))
        for mode in ("real", "fake"):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                make_fx(call, tracing_mode=mode)(x)
        call(x)


def test_denormal_temperatures_are_refused(lib):
    """log2(e) / T is an infinity for them, and 0 times it would be NaN."""
    p = 4096       # never read
    for bad in (1e-39, 4e-39, 1.1e-38, 1e-45):
        assert lib.scmiac_top_logits(p, 10, 1, 10, F32, 4, bad, p, p, p, None, 0, None) == 1
        assert lib.scmiac_distill_forward(p, 10, 1, 10, F32, p, p, 4, None, bad, 1.0, 0, p, p, None, p, 999, None) == 1
        assert lib.scmiac_distill_forward(p, 10, 1, 10, F32, p, p, 4, None, 1.0, bad, 0, p, p, None, p, 999, None) == 1
        assert "temperature" in _error(lib)
        assert lib.scmiac_distill_backward(p, 10, 1, 10, F32, p, p, 4, bad, 1.0, p, p, 0, None, p, 10, None) == 1
