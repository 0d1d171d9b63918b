"""RMS norm of queries and keys per head, with the rotary position encoding in the same pass.

GPU path: ``ops/csrc/qk_norm.hip``; CPU path (and oracle of the GPU tests): plain PyTorch. Stands
beside ``ops.transformer.rope`` and ``flash_attention``: same layouts ([B, S, H, Dh], slices of a
fused QKV projection accepted as they are, grouped K/V heads) and the same rotate-half convention.
Norms of q and k keep attention logits bounded in long or large-learning-rate training (the
reference's GPT-NeoX example trains rotary models: examples/deepspeed/gpt_neox/gpt2_trial.py).
"""
import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from determined_clone_amd.ops import _ext, _grad
from determined_clone_amd.ops.transformer import _attn_gpu_ok, _f32, _kv_len, reference_attention

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_HEAD_DIM = 1024


def _reference_one(x, w, cos, sin, rot, positions, eps):
    wide = torch.promote_types(x.dtype, torch.float32)
    y = x.to(wide)
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.to(wide)
    if rot:
        half = rot // 2
        # (a lookup, not an index: those count negative positions from the end)
        c, s = (t[:x.shape[1]] if positions is None else F.embedding(positions.long(), t) for t in (cos, sin))
        c, s = c.to(wide).unsqueeze(-2), s.to(wide).unsqueeze(-2)
        a, b, rest = y[..., :half], y[..., half:rot], y[..., rot:]
        y = torch.cat([a * c - b * s, b * c + a * s, rest], dim=-1)
    return y.to(x.dtype)


def reference_qk_norm_rope(q, k, q_weight=None, k_weight=None, cos=None, sin=None, rot_dim=None,
                           positions=None, eps=1e-6):
    """The same operator in plain PyTorch (fp32 or wider arithmetic, rounded once)."""
    cos, sin, rot = _tables(cos, sin, rot_dim, q.shape[-1])
    return (_reference_one(q, q_weight, cos, sin, rot, positions, eps),
            _reference_one(k, k_weight, cos, sin, rot, positions, eps))


def _tables(cos, sin, rot_dim, D) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], int]:
    """(cos, sin [P, rot / 2], rot); rot 0 when there is nothing to rotate."""
    if (cos is None) != (sin is None):
        raise ValueError("qk_norm_rope: cos and sin go together")
    rot = (0 if cos is None else D) if rot_dim is None else rot_dim
    if rot < 0 or rot % 2 or rot > D:
        raise ValueError(f"qk_norm_rope: rot_dim must be even and at most the head dim {D}, got {rot}")
    if rot == 0:
        return None, None, 0
    if cos is None:
        raise ValueError("qk_norm_rope: rot_dim without cos and sin")
    half = rot // 2
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] < half:
        raise ValueError(f"qk_norm_rope: cos and sin must be [P, >= {half}] tables of one shape")
    return cos[:, :half], sin[:, :half], rot


def _check(q, k, q_weight, k_weight, cos, sin, rot_dim, positions):
    """Checked (cos, sin, rot, positions): fp32 contiguous tables, contiguous positions."""
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"qk_norm_rope: q [B, S, H, D] and k [B, S, Hkv, D] required, got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    if q.dtype != k.dtype or q.device != k.device or not q.is_floating_point():
        raise ValueError("qk_norm_rope: q and k must share a floating dtype and a device")
    B, S, _, D = q.shape
    if not 1 <= D <= MAX_HEAD_DIM:
        raise ValueError(f"qk_norm_rope: head dim must be 1 .. {MAX_HEAD_DIM}, got {D}")
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (D,) or w.device != q.device or not w.is_floating_point()):
            raise ValueError(f"qk_norm_rope: weights must be [{D}] on {q.device}")
    cos, sin, rot = _tables(cos, sin, rot_dim, D)
    if not rot:
        return None, None, 0, None
    if cos.device != q.device or sin.device != q.device:
        raise ValueError(f"qk_norm_rope: cos and sin must be on {q.device}")
    if positions is None:
        if S > cos.shape[0]:
            raise ValueError(f"qk_norm_rope: {S} tokens, {cos.shape[0]} table rows")
    else:
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"qk_norm_rope: positions must be int32 or int64, got {positions.dtype}")
        if positions.shape not in ((S,), (B, S)) or positions.device != q.device:
            raise ValueError(f"qk_norm_rope: positions must be [{S}] or [{B}, {S}] on {q.device}")
        positions = positions.contiguous()
    if q.is_cuda:
        if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
            raise ValueError("qk_norm_rope: the GPU path has no gradients for cos and sin")
        cos, sin = _f32(cos), _f32(sin)
    return cos, sin, rot, positions


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, rot_dim: Optional[int] = None,
                 positions: Optional[torch.Tensor] = None, eps: float = 1e-6
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``R(pos) (weight * x / sqrt(mean(x^2) + eps))`` over each head of q [B, S, H, D] and
    k [B, S, Hkv, D] (any strides) -> contiguous tensors of the same shapes and dtype; fp32
    arithmetic, rounded once. D up to 1024.

    ``q_weight`` / ``k_weight`` [D] are shared by the heads (None: no weight). ``cos`` / ``sin``
    [P, >= rot_dim / 2] are ``ops.transformer.rope_tables``; the first ``rot_dim`` features turn in
    pairs (i, i + rot_dim / 2) (None: all of them, or none without tables); the tables get no
    gradients on the GPU, which refuses ones that ask for it. Token s uses table row s,
    or ``positions`` [S] or [B, S] (int32 / int64): generation from an offset, packed documents. A
    position outside the tables raises ``IndexError`` on the CPU; the GPU path, which does not wait
    for the values, returns NaN in the rotated features of such rows. Their gradients are NaN, and so
    are the weights' in the rotated features, which are sums over all rows. Second derivatives raise
    on the GPU."""
    cos, sin, rot, positions = _check(q, k, q_weight, k_weight, cos, sin, rot_dim, positions)
    if not q.is_cuda:
        return reference_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, rot, positions, eps)
    if q.dtype not in _DTYPES:
        raise ValueError(f"qk_norm_rope: GPU path needs bf16, fp16 or fp32, got {q.dtype}")
    return tuple(_ext.load().qk_norm_rope_autograd(q, k, q_weight, k_weight, cos, sin, rot, positions, float(eps)))


class _NotTwice(torch.autograd.Function):
    """Gradients that cannot be differentiated again (under ``create_graph``): doing so raises."""

    @staticmethod
    def forward(ctx, *grads):
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("trying to differentiate twice a function whose backward is a kernel")


class _QKNormAttention(torch.autograd.Function):
    """qk_norm_rope + flash attention on a packed QKV projection. One function, so that the backward
    writes dq, dk and dv into one packed gradient: attention's dq and dk land there, and the norm's
    backward turns them into the projection's gradients in place."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, rot, positions, eps, causal, scale, kv_len):
        C = _ext.load()
        q, k, v = qkv.unbind(2)
        yq, yk = C.qk_norm_rope(q, k, _f32(q_weight), _f32(k_weight), cos, sin, rot, positions, eps)
        o, lse = C.attn_fwd(yq, yk, v, scale, causal, kv_len)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions, qkv, yq, yk, o, lse, kv_len)
        ctx.rot, ctx.eps, ctx.params = rot, eps, (q_weight, k_weight)
        ctx.causal, ctx.scale = causal, scale
        return o

    @staticmethod
    def backward(ctx, do):
        with torch.no_grad():
            grads = _QKNormAttention._gradients(ctx, do)
        if torch.is_grad_enabled():  # they depend on qkv and the weights, whether or not on a graph of `do`
            grads = _NotTwice.apply(*(None if g is None else g.detach().requires_grad_(True) for g in grads))
        return grads + (None,) * 8

    @staticmethod
    def _gradients(ctx, do):
        C = _ext.load()
        q, k, wq, wk, cos, sin, positions, qkv, yq, yk, o, lse, kv_len = ctx.saved_tensors
        dqkv = torch.empty_like(qkv)
        dq, dk, dv = dqkv.unbind(2)
        C.attn_bwd(do, yq, yk, qkv[:, :, 2], o, lse, ctx.scale, ctx.causal, dq, dk, dv, kv_len)
        need = ctx.needs_input_grad[1:3]
        acc = [_grad.target(p) if n else None for p, n in zip(ctx.params, need)]
        _, _, dwq, dwk = C.qk_norm_rope_bwd(dq, dk, q, k, _f32(wq), _f32(wk), cos, sin, ctx.rot, positions,
                                            ctx.eps, need[0], need[1], acc[0], acc[1], dq, dk)
        dw = tuple(None if d is None else d.to(p.dtype) for d, p in zip((dwq, dwk), ctx.params))
        return (dqkv,) + dw


def qk_norm_attention_qkvpacked(qkv: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                                k_weight: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None,
                                sin: Optional[torch.Tensor] = None, rot_dim: Optional[int] = None,
                                positions: Optional[torch.Tensor] = None, eps: float = 1e-6,
                                causal: bool = True, scale: Optional[float] = None,
                                key_lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``flash_attention`` over :func:`qk_norm_rope` of a packed [B, S, 3, H, D] QKV projection ->
    [B, S, H, D]; the arguments are those of the two. The backward fills one packed gradient."""
    if qkv.dim() != 5 or qkv.shape[2] != 3:
        raise ValueError(f"qk_norm_attention_qkvpacked: [B, S, 3, H, D] required, got {tuple(qkv.shape)}")
    q, k, v = qkv.unbind(2)
    cos, sin, rot, positions = _check(q, k, q_weight, k_weight, cos, sin, rot_dim, positions)
    scale = scale if scale is not None else 1.0 / math.sqrt(qkv.shape[-1])
    if not qkv.is_cuda:
        q, k = reference_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, rot, positions, eps)
        return reference_attention(q, k, v, causal, scale, key_lengths)
    if not _attn_gpu_ok(q, k, v):
        raise ValueError("qk_norm_attention_qkvpacked: GPU path needs bf16 [B,S,3,H,D] with D in "
                         "{64,128} and 16-byte aligned rows")
    if qkv.numel() == 0:  # no launches of nothing
        q, k = reference_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, rot, positions, eps)
        return reference_attention(q, k, v, causal, scale, key_lengths)
    return _QKNormAttention.apply(qkv, q_weight, k_weight, cos, sin, rot, positions, float(eps), causal,
                                  float(scale), _kv_len(key_lengths, qkv.shape[0], qkv.device))


__all__ = ["qk_norm_rope", "qk_norm_attention_qkvpacked", "reference_qk_norm_rope"]
