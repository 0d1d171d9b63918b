"""Norm and clipping of separate gradients on the CPU: torch's results, and the trial's marker."""
import math

import pytest
import torch

from determined_clone_amd import pytorch as det_pytorch
from determined_clone_amd.ops import _ext, _grad, optim


def _params(empty=True):
    g = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter(torch.zeros(s)) for s in ((3, 4), (5,), (), (0,) if empty else (1,), (2, 3, 4))]
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g)
    return ps + [torch.nn.Parameter(torch.zeros(2))]  # one without a gradient


@pytest.mark.parametrize("norm_type", [2, 1, math.inf, 3])
@pytest.mark.parametrize("max_norm", [0.5, 1e3])
def test_is_torchs_clip(norm_type, max_norm):
    empty = norm_type != math.inf  # torch's max norm refuses tensors without elements
    a, b = _params(empty), _params(empty)
    got = optim.clip_grad_norm_(iter(a), max_norm, norm_type)
    want = torch.nn.utils.clip_grad_norm_(b, max_norm, norm_type)
    torch.testing.assert_close(got, want, rtol=0, atol=0)
    for p, q in zip(a, b):
        assert (p.grad is None) == (q.grad is None)
        if p.grad is not None:
            torch.testing.assert_close(p.grad, q.grad, rtol=0, atol=0)
    torch.testing.assert_close(optim.grad_norm([p.grad for p in _params(empty) if p.grad is not None], norm_type), want)


def test_the_trials_marker_clips():
    a, b = _params(), _params()
    det_pytorch.clip_grad_norm(0.25)(a)
    torch.nn.utils.clip_grad_norm_(b, 0.25)
    assert all(p.grad is None or torch.equal(p.grad, q.grad) for p, q in zip(a, b))


def test_empty_single_and_refusals():
    assert optim.clip_grad_norm_([], 1.0) == 0 and optim.grad_norm([]) == 0
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.full((4,), 3.0)
    assert optim.clip_grad_norm_(p, 3.0) == 6.0
    torch.testing.assert_close(p.grad, torch.full((4,), 1.5), rtol=1e-6, atol=0)
    p.grad[1] = float("nan")
    kept = p.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        optim.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad.nan_to_num(7), kept.nan_to_num(7))
    with pytest.raises((TypeError, ValueError)):
        optim.clip_grad_norm_([p], "a lot")


@pytest.mark.parametrize("norm_type", [2, 3])
@pytest.mark.parametrize("refuse", [False, True])
def test_side_stream_gradients_are_awaited_where_torch_clips(norm_type, refuse, monkeypatch):
    """What the kernels do not take goes to torch, which must not read gradients still being written."""
    calls = []
    monkeypatch.setattr(_grad, "join", lambda: calls.append("join"))
    for name in ("clip_grad_norm_", "get_total_norm"):
        plain = getattr(torch.nn.utils, name)
        monkeypatch.setattr(torch.nn.utils, name, lambda *a, f=plain, n=name, **k: (calls.append(n), f(*a, **k))[1])
    optim.clip_grad_norm_(_params(), 0.5, norm_type, error_if_nonfinite=refuse)
    assert calls[:2] == ["join", "clip_grad_norm_"]
    calls.clear()
    optim.grad_norm([p.grad for p in _params() if p.grad is not None], norm_type)
    assert calls[:2] == ["join", "get_total_norm"]


def test_overlap_is_asked_of_memory_only():
    """Wrapper subclasses (sharded tensors) and nested tensors have no address to compare."""
    from torch.testing._internal.two_tensor import TwoTensor

    overlaps = _ext.load().grad_list_overlaps
    x = torch.randn(100)
    wrapped = [TwoTensor(torch.randn(3), torch.randn(3)) for _ in range(2)]
    nested = [torch.nested.nested_tensor([torch.randn(2), torch.randn(3)]) for _ in range(2)]
    assert not overlaps(wrapped) and not overlaps(nested) and not overlaps(wrapped + nested + [x[:50], x[50:]])
    assert overlaps(wrapped + nested + [x[:51], x[50:]])
