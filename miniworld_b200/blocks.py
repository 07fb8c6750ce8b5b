"""Block operators on tensors ``[..., d]`` of any width: the norms around a block joined with its gate, residual scale and
residual, and the gated feed-forward (forward and backward).

What the triangle update and the pair Transition have inside their kernels for the pair tensor, the other tensors of a trunk need as
operators: token and alignment tensors of other widths (the reference builds its Transition for each of them,
``src/miniworld/blocks/msa_module.py:94-122``). A stack of blocks ``f`` runs as

    h = block_norm(x, w, b)
    x, h = block_join(x, f(h), gate=..., scale=..., post=Norm(...), pre=Norm(...))     # for each block but the last
    x = block_join(x, f(h), gate=..., scale=..., post=Norm(...))

Inputs are CUDA tensors; nothing here falls back to PyTorch arithmetic. Layouts and, where it says so, float types are converted;
everything else is refused with a ``RuntimeError``, forward-mode derivatives and second derivatives among it.
"""

from __future__ import annotations

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


def read_status(device=None) -> int:
    """Synchronises the current stream; 0, or the code of the first device-side wait of a block operator on ``device`` that gave up
    since the last call."""
    import ctypes

    code = ctypes.c_int(0)
    with torch.cuda.device(device):
        _lib.check(_lib.load().b200_blocks_read_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(code)), "b200_blocks_read_status")
    return code.value


def check_status(device=None, what: str = "gated_feed_forward") -> None:
    code = read_status(device)
    if code != 0:
        raise RuntimeError(f"{what}: {_lib.strerror(code)} [{code}]")
