"""Token embedding for language models: table lookup with scaling, learned positions added in the
same pass, vocabulary shards, and the table gradients.

GPU path: ``ops/csrc/embedding.hip``; CPU path (and oracle of the GPU tests): plain PyTorch. The
reference's GPT-NeoX example gets these from Megatron's ``VocabParallelEmbedding`` and
``torch.nn.Embedding`` (reference: examples/deepspeed/gpt_neox/gpt2_trial.py).

The token gradient sums the rows of each token in token order (ids sorted on the GPU, no float
atomics), so it does not change from run to run. With a persistent ``.grad`` (``ops._grad``) only
the rows of tokens that occur are touched, added in place; otherwise a dense gradient is returned.
"""
from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

from determined_clone_amd.ops import _ext

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def reference_embedding(idx, weight, pos_weight=None, positions=None, scale=1.0, vocab_start=None):
    """The same operator in plain PyTorch (fp32 or wider arithmetic, rounded once)."""
    local = idx.long() - vocab_start if vocab_start else idx.long()
    # without a product the one sum is rounded once in the tables' own type
    wide = weight.dtype if scale == 1 else torch.promote_types(weight.dtype, torch.float32)
    if vocab_start is None:
        out = F.embedding(local, weight)
    else:
        outside = (local < 0) | (local >= weight.shape[0])
        out = F.embedding(local.masked_fill(outside, 0), weight)
    if scale != 1:
        out = out.to(wide) * scale
    if vocab_start is not None:
        out = out.masked_fill(outside.unsqueeze(-1), 0)
    if pos_weight is not None:
        if positions is None:
            out = out + pos_weight[:idx.shape[-1]].to(wide)
        else:
            out = out + F.embedding(positions.long(), pos_weight).to(wide)
    return out.to(weight.dtype)


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _kernel_takes(weight: torch.Tensor, pos_weight: Optional[torch.Tensor] = None) -> bool:
    """Whether the tables (of one dtype and device) are plain GPU tensors outside of function transforms
    (vmap, jvp, grad, ...) and forward-mode differentiation, which the kernels' node does not know."""
    return (weight.is_cuda and weight.dtype in _DTYPES and type(weight) in _PLAIN
            and (pos_weight is None or type(pos_weight) in _PLAIN)
            and forward_ad._current_level < 0 and torch._C._functorch.peek_interpreter_stack() is None)


def _check_index(t: torch.Tensor, what: str) -> None:
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"embedding: {what} must be int32 or int64, got {t.dtype}")


def embedding(idx: torch.Tensor, weight: torch.Tensor, pos_weight: Optional[torch.Tensor] = None,
              positions: Optional[torch.Tensor] = None, scale: float = 1.0,
              vocab_start: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[idx] (+ pos_weight[positions])`` for ``idx`` [...] and ``weight`` [V, E] ->
    [..., E] in the table's dtype, computed in fp32 and rounded once.

    ``pos_weight`` [P, E] adds learned positions: row ``s`` to the tokens at index ``s`` of the last
    dim of ``idx`` (at most P of them), or row ``positions[...]`` when ``positions`` (int32 / int64,
    broadcastable to ``idx``) is given: packed documents, generation from an offset.

    ``vocab_start`` makes ``weight`` a shard of a larger vocabulary, rows ``vocab_start`` and up: ids
    outside it look up zeros and have no gradient (sum the shards' outputs with an all-reduce).
    Without it every id has to lie in [0, V), and every position in [0, P): the CPU path raises
    ``IndexError`` for others, the GPU kernels, which do not wait for the values, return NaN rows
    for them and give them no gradient in the table that they miss.

    float64 tables, tensor subclasses, function transforms (``torch.func``) and forward-mode
    differentiation run as plain PyTorch on the GPU too, where a mistaken id ends the program.
    Second derivatives through the kernels raise."""
    _check_index(idx, "idx")
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("embedding: weight must be a floating-point [V, E] table")
    if vocab_start is not None and vocab_start < 0:
        raise ValueError(f"embedding: vocab_start must not be negative, got {vocab_start}")
    if idx.device != weight.device:
        raise ValueError(f"embedding: idx on {idx.device}, weight on {weight.device}")
    if positions is not None and pos_weight is None:
        raise ValueError("embedding: positions without pos_weight")
    if pos_weight is not None:
        if vocab_start is not None:
            raise ValueError("embedding: add positions after the vocabulary shards are summed")
        if pos_weight.dim() != 2 or pos_weight.shape[1] != weight.shape[1] or \
                pos_weight.dtype != weight.dtype or pos_weight.device != weight.device:
            raise ValueError("embedding: pos_weight must be [P, E] like weight (width, dtype, device)")
        if positions is not None:
            _check_index(positions, "positions")
            if positions.device != weight.device:
                raise ValueError(f"embedding: positions on {positions.device}, weight on {weight.device}")
            if positions.shape != idx.shape:
                positions = positions.expand(idx.shape)  # raises for shapes that do not broadcast
        elif idx.dim() == 0:
            raise ValueError("embedding: a single id needs its position")
        elif idx.shape[-1] > pos_weight.shape[0]:
            raise ValueError(f"embedding: {idx.shape[-1]} tokens, {pos_weight.shape[0]} positions")
    if not _kernel_takes(weight, pos_weight):
        return reference_embedding(idx, weight, pos_weight, positions, scale, vocab_start)
    return _ext.load().embedding(idx, weight, pos_weight, positions, float(scale), vocab_start or 0,
                                 vocab_start is not None)


__all__ = ["embedding", "reference_embedding"]
