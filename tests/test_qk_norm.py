"""Query / key norm + rotary on the CPU: the formula, gradients against finite differences, refusals."""
import pytest
import torch

from determined_clone_amd.ops import transformer as T
from determined_clone_amd.ops.qk_norm import qk_norm_attention_qkvpacked, qk_norm_rope


def _qk(b=2, s=5, h=4, hk=2, d=8, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(b, s, h, d, generator=g, dtype=dtype), torch.randn(b, s, hk, d, generator=g, dtype=dtype),
            torch.rand(d, generator=g, dtype=dtype) + 0.5, torch.rand(d, generator=g, dtype=dtype) + 0.5)


def test_is_norm_then_rope():
    q, k, wq, wk = _qk(dtype=torch.float32)
    cos, sin = T.rope_tables(9, 4)
    yq, yk = qk_norm_rope(q, k, wq, wk, cos, sin, rot_dim=4, eps=1e-5)
    for x, w, y in ((q, wq, yq), (k, wk, yk)):
        n = torch.nn.functional.rms_norm(x, (8,), w, 1e-5)
        torch.testing.assert_close(y, T.reference_rope(n, cos, sin, 4), rtol=1e-6, atol=1e-6)
    pos = torch.tensor([[8, 0, 1, 1, 3], [0, 1, 2, 3, 4]])
    zq, zk = qk_norm_rope(q, k, wq, wk, cos, sin, rot_dim=4, positions=pos, eps=1e-5)
    assert torch.equal(zq[1], yq[1]) and torch.equal(zk[1], yk[1])
    assert torch.equal(zq[0, 1], qk_norm_rope(q[:1, 1:2], k[:1, 1:2], wq, wk, cos, sin, 4, eps=1e-5)[0][0, 0])
    # tables wider than the rotated part, and no rotation at all
    wide_cos, wide_sin = torch.cat([cos, cos], 1), torch.cat([sin, sin], 1)
    assert torch.equal(qk_norm_rope(q, k, wq, wk, wide_cos, wide_sin, 4, eps=1e-5)[0], yq)
    plain, _ = qk_norm_rope(q, k, eps=1e-5)
    torch.testing.assert_close(plain, torch.nn.functional.rms_norm(q, (8,), None, 1e-5))


@pytest.mark.parametrize("rot", [0, 2, 4, 8])
def test_gradients_against_differences(rot):
    q, k, wq, wk = (t.requires_grad_(True) for t in _qk(b=1, s=3))
    cos, sin = (t.double() for t in T.rope_tables(6, 8))
    pos = torch.tensor([5, 0, 2])
    assert torch.autograd.gradcheck(
        lambda *a: qk_norm_rope(*a, cos if rot else None, sin if rot else None, rot, pos), (q, k, wq, wk))


def test_packed_attention_is_norm_rope_attention():
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2, 7, 3, 2, 8, generator=g)
    w = torch.rand(8, generator=g) + 0.5
    cos, sin = T.rope_tables(7, 8)
    q, k = qk_norm_rope(qkv[:, :, 0], qkv[:, :, 1], w, None, cos, sin)
    lengths = torch.tensor([7, 3])
    want = T.flash_attention(q, k, qkv[:, :, 2], causal=True, key_lengths=lengths)
    got = qk_norm_attention_qkvpacked(qkv, w, None, cos, sin, causal=True, key_lengths=lengths)
    assert torch.equal(got, want)


def test_refusals():
    q, k, wq, wk = _qk(dtype=torch.float32)
    cos, sin = T.rope_tables(5, 8)
    bad = [(dict(q=q[0]), "required"), (dict(k=k[:, :4]), "required"), (dict(k=k[..., :4]), "required"),
           (dict(k=k.double()), "share"), (dict(q=q.long(), k=k.long()), "share"),
           (dict(q_weight=wq[:4]), "weights"), (dict(sin=None), "go together"),
           (dict(rot_dim=3), "even"), (dict(rot_dim=10), "even"), (dict(rot_dim=-2), "even"),
           (dict(cos=None, sin=None, rot_dim=4), "without cos"), (dict(cos=cos[:, :2], sin=sin[:, :2]), "tables"),
           (dict(cos=cos[:4], sin=sin[:4]), "table rows"), (dict(positions=torch.zeros(5)), "int32 or int64"),
           (dict(positions=torch.zeros(4, dtype=torch.long)), "positions must be"),
           (dict(q=torch.randn(1, 1, 1, 1026), k=torch.randn(1, 1, 1, 1026), q_weight=None, k_weight=None), "1024")]
    for change, match in bad:
        kw = dict(q=q, k=k, q_weight=wq, k_weight=wk, cos=cos, sin=sin)
        kw.update(change)
        with pytest.raises(ValueError, match=match):
            qk_norm_rope(**kw)
    with pytest.raises(IndexError):
        qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.full((5,), 5))
    with pytest.raises(ValueError, match="3, H, D"):
        qk_norm_attention_qkvpacked(torch.randn(2, 5, 2, 4, 8))


@pytest.mark.parametrize("bad", [-1, -5, -6, 5])
def test_positions_outside_the_tables_raise(bad):
    q, k, wq, wk = _qk(dtype=torch.float32)
    cos, sin = T.rope_tables(5, 8)
    for dtype in (torch.int32, torch.int64):
        pos = torch.tensor([0, 4, bad, 1, 2], dtype=dtype)
        for p in (pos, pos.expand(2, 5)):
            with pytest.raises(IndexError):
                qk_norm_rope(q, k, wq, wk, cos, sin, positions=p)
        with pytest.raises(IndexError):
            qk_norm_attention_qkvpacked(torch.randn(1, 5, 3, 2, 8), wq, wk, cos, sin, positions=pos)
    assert qk_norm_rope(q, k, wq, wk, positions=pos)[0].shape == q.shape  # nothing turns: not looked at
