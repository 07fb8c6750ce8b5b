"""Block operators on tensors ``[..., d]`` of any width: the norms around a block joined with its gate, residual scale and
residual, and the gated feed-forward; token operators: attention over tokens with a learned bias of their relative position, the
relative position added to the pair tensor, and dropout on a block's output (all forward and backward).

What the triangle update and the pair Transition have inside their kernels for the pair tensor, the other tensors of a trunk need as
operators: token and alignment tensors of other widths (the reference builds its Transition for each of them,
``src/miniworld/blocks/msa_module.py:94-122``). A stack of blocks ``f`` runs as

    h = block_norm(x, w, b)
    x, h = block_join(x, f(h), gate=..., scale=..., post=Norm(...), pre=Norm(...))     # for each block but the last
    x = block_join(x, f(h), gate=..., scale=..., post=Norm(...))

with ``block_dropout(None, f(h), key, p=...)`` in the place of ``f(h)`` in training, or ``block_dropout(x, f(h), key, p=...)`` where a
block is joined without a norm, gate and scale.

Inputs are CUDA tensors; nothing here falls back to PyTorch arithmetic. Layouts and, where it says so, float types are converted;
everything else is refused with a ``RuntimeError``, forward-mode derivatives and second derivatives among it.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import _lib

_KINDS = {"layer": 1, "rms": 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1}


class Norm(NamedTuple):
    """A norm over the last dimension: ``kind`` "layer" or "rms", fp32 ``weight`` and ``bias`` [d] (None: 1 and 0), ``eps``."""

    kind: str = "layer"
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-5


_ABSENT = (0, None, None, 0.0)


def _kind(kind: str) -> int:
    code = _KINDS.get(kind)
    if code is None:
        raise ValueError(f"norm kind must be one of {sorted(_KINDS)}, got {kind!r}")
    return code


def _spread(norm: Optional[Norm]) -> tuple:
    if norm is None:
        return _ABSENT
    kind, weight, bias, eps = norm
    return _kind(kind), weight, bias, eps


def block_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, kind: str = "layer",
               eps: float = 1e-5) -> torch.Tensor:
    """``norm(x)`` over the last dimension, ``x`` bf16, fp16 or fp32 (differentiable)."""
    return _lib.native().block_join(x, None, None, None, None, *_ABSENT, _kind(kind), weight, bias, eps)[1]


def block_join(x: torch.Tensor, u: torch.Tensor, *, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
               mask: Optional[torch.Tensor] = None, post: Optional[Norm] = None, pre: Optional[Norm] = None):
    """``y = x + mask * scale * sigmoid(gate) * post(u)`` and, with ``pre``, ``(y, pre(y))`` (differentiable).

    ``x`` bf16, fp16 or fp32 [..., d]; ``u`` of its shape; ``gate`` logits [..., d] of ``x``'s leading dimensions and then
    ones (a row each, one for the rows of a sample, one for all); ``scale`` fp32 [d]; ``mask`` over the rows, zero: ``y = x`` there
    whatever ``u`` and ``gate`` hold. ``u`` and ``gate`` of another float type are converted. ``pre`` sees ``y`` before it is rounded to ``x``'s type.
    """
    y, h = _lib.native().block_join(x, u, gate, scale, mask, *_spread(post), *_spread(pre))
    return y if pre is None else (y, h)


def gated_feed_forward(x: torch.Tensor, w_a: torch.Tensor, w_b: torch.Tensor, w_s: torch.Tensor, *, activation: str = "silu") -> torch.Tensor:
    """``(act(x w_a^T) * (x w_b^T)) w_s^T`` for ``x`` [..., d], ``w_a`` and ``w_b`` [hidden, d], ``w_s`` [d, hidden]; ``d`` and
    ``hidden`` multiples of 8; ``activation`` "silu" or "gelu" (differentiable).

    bf16 and fp16 run as they are, other float types of ``x`` through bf16. The weights are of the type that the products run in, or
    fp32 (rounded to it in each call; their gradients are fp32)."""
    code = _ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    return _lib.native().gated_feed_forward(x, w_a, w_b, w_s, code)


def _bucket_list(reach: int, exact: Optional[int] = None) -> list[int]:
    """The numbers of :func:`relative_buckets`."""
    if not 0 <= reach <= 256:
        raise ValueError(f"reach must be from 0 to 256, got {reach}")
    if exact is None:
        return list(range(2 * reach + 1))
    if not 1 <= exact < reach or 4 * exact > 512:
        raise ValueError(f"exact must be at least 1, less than reach = {reach} and at most 128, got {exact}")

    def bucket(distance: int) -> int:
        far = abs(distance)
        if far >= exact:
            far = min(2 * exact - 1, exact + int(math.log(far / exact) / math.log(reach / exact) * exact))
        return far + (2 * exact if distance > 0 else 0)

    return [bucket(d) for d in range(-reach, reach + 1)]


def relative_buckets(reach: int, exact: Optional[int] = None, device=None) -> torch.Tensor:
    """Buckets of the distances ``-reach .. reach`` (of a key from its query, of the pair's second token from its first), int32
    ``[2 reach + 1]``; greater distances count as the outermost. ``exact`` None: a bucket for each distance, ``distance + reach``.
    Else two halves of ``2 exact`` buckets, for distances up to 0 and above: one bucket for each distance shorter than ``exact``, the
    other ``exact`` of a half on a logarithmic scale that ends at ``reach``.
    """
    numbers = _bucket_list(reach, exact)
    return torch.arange(len(numbers), dtype=torch.int32, device=device) if exact is None else torch.tensor(numbers, dtype=torch.int32, device=device)


def token_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, offsets: Optional[torch.Tensor] = None,
                    mask: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                    table: Optional[torch.Tensor] = None, bucket_of: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale q k^T + bias) v`` among the tokens of each sequence (differentiable).

    ``q`` [..., tokens, heads, d], ``k`` and ``v`` [..., tokens, kv_heads, d], ``heads`` a multiple of ``kv_heads`` (query head ``h``
    reads head ``h // (heads / kv_heads)``), ``d`` a multiple of 8 up to 128; slices of one projection are read where they lie. With
    ``offsets`` (integers [sequences + 1], the first 0, non-decreasing) the tokens of ``q`` [tokens, heads, d] are packed sequences: the
    rows ``offsets[s] .. offsets[s + 1]`` are sequence ``s``, of any length; rows behind the last one come out zero. ``mask`` over the
    tokens: those with zero are not attended to and come out zero, whatever they hold, with zero gradients. ``causal``: a token attends
    to itself and the ones before it (a value that is not finite at a later token may reach earlier ones all the same). ``scale`` defaults to ``d ** -0.5``. ``table`` [buckets, heads] (q's type or fp32) with ``bucket_of``
    (:func:`relative_buckets`): ``table[bucket_of[clip(j - i, -reach, reach) + reach], head]`` is added to the score of query ``i`` and
    key ``j`` of a sequence; where it is -inf the pair does not count (rows without any pair come out zero), and finite biases beyond
    fp16's range (65504 either way) count as its ends.

    bf16 and fp16 run as they are, other float types through bf16; scores, their gradients and sums are fp32, the probabilities and
    the gradients of the scores are rounded to 16 bits as operands of the products."""
    return _lib.native().token_attention(q, k, v, offsets, mask, causal, scale, table, bucket_of)


def relative_position(z: torch.Tensor, table: torch.Tensor, index: torch.Tensor, *, bucket_of: torch.Tensor,
                      chain: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``z[..., i, j, :] + table[bucket]`` for the pair tensor ``z`` [..., tokens, tokens, c] (bf16, fp16 or fp32) and the fp32
    ``table`` [buckets, c] (differentiable; the table's gradient is fp32).

    The bucket is ``bucket_of[clip(index[..., j] - index[..., i], -reach, reach) + reach]`` (:func:`relative_buckets`), or the last
    row of the table for two tokens whose ``chain`` differs. ``index`` and ``chain``: int32 or int64 [..., tokens]."""
    return _lib.native().relative_position(z, table, index, bucket_of, chain)


def dropout_key(device=None) -> torch.Tensor:
    """A key for :func:`block_dropout` from PyTorch's generator of ``device``: int64 [2] (under graph capture a new one each replay)."""
    return torch.randint(-(2**63), 2**63 - 1, (2,), dtype=torch.int64, device="cuda" if device is None else device)


def block_dropout(x: Optional[torch.Tensor], u: torch.Tensor, key: torch.Tensor, *, p: float, shared: Optional[int] = None,
                  call: int = 0) -> torch.Tensor:
    """``x + keep * u / (1 - p)`` (``x`` None: without it), with a mask that is never stored (differentiable).

    ``keep`` follows from an element's place, ``key`` (int64 CUDA tensor of two elements, :func:`dropout_key`) and ``call``, which
    tells calls with one key apart; the backward draws it again, so the key must not change in between. ``p`` counts in 1/65536,
    and the scale is the inverse of exactly the share that stays. ``shared``: a dimension along which all use one mask (the triangle
    updates drop rows that way: 1 for a pair tensor [B, N, N, c]). Where an element is dropped ``y = x`` whatever ``u`` holds."""
    return _lib.native().block_dropout(x, u, key, p, shared, call)


def read_status(device=None) -> int:
    """Synchronises the current stream; 0, or the code of the first device-side wait of a block or token operator on ``device`` that
    gave up since the last call."""
    import ctypes

    codes = []
    with torch.cuda.device(device):
        for name in ("b200_blocks_read_status", "b200_tokens_read_status"):
            code = ctypes.c_int(0)
            _lib.check(getattr(_lib.load(), name)(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)), name)
            codes.append(code.value)
    return codes[0] or codes[1]


def check_status(device=None, what: str = "gated_feed_forward") -> None:
    code = read_status(device)
    if code != 0:
        raise RuntimeError(f"{what}: {_lib.strerror(code)} [{code}]")
