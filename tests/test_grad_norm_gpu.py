"""Multi-tensor gradient norm and clipping against the formula in 64 bits (run on an MI355X).

Tolerances: sums are held in 64 bits, so the norm is one fp32 rounding off (2^-24 relative, twice
that allowed for the root in 64 bits); the coefficient takes an fp32 addition and a division, its
product with a gradient one more fp32 rounding and half a step of the gradient's type."""
import math

import pytest
import torch

from determined_clone_amd import pytorch as det_pytorch
from determined_clone_amd.ops import _ext, _grad, optim

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
KINDS = [2.0, 1.0, math.inf]
# odd sizes and ones around vector (8), chunk (2048 .. 32768) and launch (192 tensors) borders
SIZES = [1, 7, 8, 9, 2047, 2048, 2049, 40001, 3, 16, 65536]


def _grads(sizes, dtypes, seed=0, scale=1.0, odd=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        x = (torch.randn(n + 1, generator=g, device="cuda") * scale).to(dt)
        out.append(x[1:] if odd else x[:n].clone())  # from an unaligned address, or an aligned one
    return out


def _exact_norm(grads, p):
    if p == math.inf:
        return max(float(g.double().abs().max()) for g in grads if g.numel())
    return math.fsum(float((g.double().abs() ** p).sum()) for g in grads) ** (1 / p)


def _params(grads):
    ps = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


def _check(before, after, norm, p, max_norm):
    want = _exact_norm(before, p)
    assert norm.dtype == torch.float32 and norm.shape == () and abs(float(norm) - want) <= 2 * U * want
    c = min(1.0, max_norm / (want + 1e-6))
    for a, b in zip(before, after):
        if c == 1.0:
            assert torch.equal(a, b)
            continue
        w, info = a.double() * c, torch.finfo(a.dtype)
        bound = w.abs() * (info.eps / 2 * 1.001 + 6 * U) + info.smallest_normal * info.eps
        assert ((b.double() - w).abs() <= bound).all()


@pytest.mark.parametrize("p", KINDS)
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16],
                                    [torch.bfloat16, torch.float32, torch.float16]])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("max_norm", [0.75, 1e9])
def test_norm_and_clip(p, dtypes, odd, max_norm):
    grads = _grads(SIZES, dtypes, odd=odd)
    before = [g.clone() for g in grads]
    assert torch.equal(optim.grad_norm(grads, p), optim.clip_grad_norm_(_params(grads), max_norm, p))
    norm = optim.grad_norm(before, p)
    _check(before, grads, norm, p, max_norm)


@pytest.mark.parametrize("count", [1, 191, 192, 193, 700])
def test_many_tensors(count):
    grads = _grads([1 + (i * 37) % 301 for i in range(count)], [torch.float32, torch.bfloat16])
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(_params(grads), 1.0)
    _check(before, grads, norm, 2.0, 1.0)


@pytest.mark.parametrize("n", [3_000_001, 150_000_003])
def test_large_tensors(n):
    grads = _grads([n, 5, n // 3], [torch.bfloat16, torch.float32], scale=0.01)
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(_params(grads), 1.0)
    _check(before, grads, norm, 2.0, 1.0)
    again = [g.clone() for g in before]
    assert torch.equal(optim.clip_grad_norm_(_params(again), 1.0), norm)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


def test_far_offsets():
    n = 2 ** 31 + 9
    g = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    g[0], g[-1], g[2 ** 31] = 3.0, 4.0, 12.0
    assert float(optim.clip_grad_norm_(_params([g]), 6.5)) == 13.0
    assert g[0] == 1.5 and g[-1] == 2.0 and g[2 ** 31] == 6.0


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_no_overflow_and_no_underflow(scale):
    g = _grads([1000], [torch.float32], scale=scale)
    want = _exact_norm(g, 2.0)
    assert abs(float(optim.grad_norm(g)) - want) <= 2 * U * want


@pytest.mark.parametrize("p", KINDS)
def test_nan_and_infinity(p):
    for bad in (float("nan"), float("inf"), float("-inf")):
        grads = _grads([5000, 7], [torch.float32, torch.bfloat16])
        grads[0][4321] = bad
        kept = [g.clone() for g in grads]
        with pytest.raises(RuntimeError, match="non-finite"):
            optim.clip_grad_norm_(_params(grads), 1.0, p, error_if_nonfinite=True)
        assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(grads, kept))
        norm = optim.clip_grad_norm_(_params(grads), 1.0, p)
        want = _params([g.cpu() for g in kept])
        ref = torch.nn.utils.clip_grad_norm_(want, 1.0, p)
        assert torch.equal(norm.cpu().nan_to_num(5, 6, 7), ref.nan_to_num(5, 6, 7))
        for g, w in zip(grads, want):
            assert torch.equal(g.cpu().nan_to_num(5), w.grad.nan_to_num(5))


def test_error_if_nonfinite_clips_finite_gradients():
    grads = _grads(SIZES, [torch.float32])
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(_params(grads), 0.5, error_if_nonfinite=True)
    _check(before, grads, norm, 2.0, 0.5)


def test_dense_layouts_and_empty_tensors():
    a = torch.randn(8, 16, 3, 3, device="cuda").to(memory_format=torch.channels_last)
    grads = [a, torch.randn(30, 50, device="cuda").t(), torch.zeros(0, device="cuda"), torch.randn((), device="cuda")]
    assert _ext.load().grad_list_norm(grads, 0) is not None
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(_params(grads), 0.5)
    _check(before, grads, norm, 2.0, 0.5)
    assert float(optim.grad_norm([torch.zeros(0, device="cuda")])) == 0.0


@pytest.mark.parametrize("kind", ["double", "strided", "overlap", "cpu", "order 3"])
def test_what_the_kernels_do_not_take_goes_to_torch(kind):
    def make():
        g = torch.Generator(device="cuda").manual_seed(1)
        x = torch.randn(40, 40, generator=g, device="cuda")
        if kind == "double":
            return [x.double()]
        if kind == "strided":
            return [x[:, ::2], x[:, 1::2]]
        if kind == "overlap":
            return [x.view(-1)[:1000], x.view(-1)[600:]]
        return [x, x.cpu()] if kind == "cpu" else [x]
    p = 3.0 if kind == "order 3" else 2.0
    a, b = make(), make()
    if kind != "order 3":
        assert _ext.load().grad_list_norm(a, 0, 1.0) is None
    def wrap(gs):  # parameters of the gradients' shapes and strides
        ps = [torch.nn.Parameter(g.detach().clone()) for g in gs]
        for q, g in zip(ps, gs):
            q.grad = g
        return ps
    got = optim.clip_grad_norm_(wrap(a), 0.5, p)
    want = torch.nn.utils.clip_grad_norm_(wrap(b), 0.5, p, foreach=False if kind == "overlap" else None)
    torch.testing.assert_close(got, want, rtol=0, atol=0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_side_stream_gradients_land_first():
    """A weight gradient still running on the side stream is waited for."""
    p = torch.nn.Parameter(torch.zeros(1 << 22, device="cuda"))
    p._dca_direct_grad = True
    p.grad = torch.zeros_like(p)
    side = _grad.side_stream_for(p)
    if side is None:
        pytest.skip("side stream is off")
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    _grad.fork(side, (a,))
    with torch.cuda.stream(side):
        for _ in range(10):
            a = a @ a * 1e-2
        p.grad.add_(1.0)
    assert float(optim.clip_grad_norm_([p], 1.0)) == 2048.0
    torch.testing.assert_close(p.grad, torch.full_like(p, 1 / 2048.0), rtol=1e-5, atol=0)


@pytest.mark.parametrize("refuse", [False, True])
def test_autograd_hears_of_the_scaling(refuse):
    """A gradient that another graph has saved: its backward raises after clipping rather than use it."""
    p, = _params(_grads([300], [torch.float32]))
    x = torch.randn(300, device="cuda", requires_grad=True)
    y = x * p.grad
    optim.grad_norm([p.grad])
    torch.autograd.grad(y.sum(), x, retain_graph=True)  # a norm changes nothing
    optim.clip_grad_norm_([p], 1e-3, error_if_nonfinite=refuse)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        q = torch.zeros(3, device="cuda")
        q.grad = torch.full((3,), 2.0, device="cuda")
        optim.clip_grad_norm_([q], 1.0, error_if_nonfinite=refuse)
        assert float(q.grad.square().sum()) < 1.001


@pytest.mark.parametrize("kind", ["order 3", "CPU first"])
def test_side_stream_gradients_land_before_torchs_clipping(kind):
    p = torch.nn.Parameter(torch.zeros(1 << 20, device="cuda"))
    p._dca_direct_grad = True
    p.grad = torch.zeros_like(p)
    side = _grad.side_stream_for(p)
    if side is None:
        pytest.skip("side stream is off")
    a = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    _grad.fork(side, (a,))
    with torch.cuda.stream(side):
        for _ in range(10):
            a = a @ a * 1e-2
        p.grad.add_(1.0)
    params, order = [p], 3.0
    if kind == "CPU first":
        params, order = [torch.nn.Parameter(torch.zeros(4)), p], 2.0
        params[0].grad = torch.zeros(4)
    want = float(1 << 20) ** (1 / order)
    # torch's norm: its own order of 2^20 fp32 additions of ones and a root; all of them exact but the root
    assert abs(float(optim.clip_grad_norm_(params, 1.0, order)) - want) <= 1e-5 * want
    torch.testing.assert_close(p.grad, torch.full_like(p, 1 / want), rtol=2e-5, atol=0)


def test_captured_graph_replays():
    grads = _grads([3001, 70000, 5] * 80, [torch.bfloat16, torch.float32])
    ps = _params(grads)
    optim.clip_grad_norm_(ps, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(ps, 1.0)
    for k in range(4):
        fresh = _grads([3001, 70000, 5] * 80, [torch.bfloat16, torch.float32], seed=k, scale=10.0 ** (k - 3))
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        want = optim.clip_grad_norm_(_params(fresh), 1.0)
        assert torch.equal(norm, want), k
        assert all(torch.equal(a, b) for a, b in zip(grads, fresh)), k


def test_the_trials_marker_uses_the_kernels():
    grads = _grads([100, 2000], [torch.float32])
    before = [g.clone() for g in grads]
    norm = det_pytorch.clip_grad_norm(0.5)(iter(_params(grads)))
    _check(before, grads, norm, 2.0, 0.5)
