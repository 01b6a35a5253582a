"""The gated delta rule of the linear-attention layers.

  gated_delta_step(q, k, v, g, beta, state, slots)              one token per sequence
  gated_delta_chunk(q, k, v, g, beta, state, cu_seqlens, slots) packed prompts

Per sequence and value head, with an fp32 state S [key_dim, value_dim]:
  S <- exp(g) S;  S <- S + k (beta (v - S^T k))^T;  out = S^T (scale q)
The state pool [slots, value_heads, key_dim, value_dim] is updated in place.
The reference's layers have 16 key and 32 value heads of 128 and call SGLang's
kernels (src/drama3/gdn.py:8-195).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import call


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, slots: torch.Tensor | None = None, *, scale: float | None = None,
                     l2norm: bool = True, eps: float = 1e-6, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    """One token for each of n sequences: q, k bf16 [n, key_heads, key_dim], v
    bf16 [n, value_heads, value_dim], g (log decay) and beta f32 [n,
    value_heads]. Sequence i's state is state[slots[i]] (int32; None: state[i]),
    updated in place; a negative slot leaves the sequence out (zero row), and no
    two sequences of a call may share one. q and
    k are divided by sqrt(|x|^2 + eps) when l2norm; scale: key_dim**-0.5 by
    default. Returns out bf16 [n, value_heads, value_dim]."""
    return _lib.native().gated_delta_step(q, k, v, g, beta, state, slots, scale, l2norm, eps, out, status)


def gated_delta_chunk_workspace(tokens: int, sequences: int, value_heads: int, key_dim: int, value_dim: int,
                                device) -> torch.Tensor:
    """Scratch of gated_delta_chunk for up to these sizes, for a caller that keeps it."""
    nbytes = ctypes.c_size_t()
    call("d3_gated_delta_chunk_workspace_size", tokens, sequences, value_heads, key_dim, value_dim,
         ctypes.byref(nbytes))
    return torch.empty(nbytes.value, dtype=torch.uint8, device=device)


def gated_delta_chunk(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                      state: torch.Tensor, cu_seqlens: torch.Tensor, slots: torch.Tensor | None = None, *,
                      fresh: torch.Tensor | None = None, scale: float | None = None, l2norm: bool = True,
                      eps: float = 1e-6, out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None,
                      status: torch.Tensor | None = None) -> torch.Tensor:
    """Packed prompts: rows [cu_seqlens[i], cu_seqlens[i+1]) (int32 [n+1]) are
    sequence i's tokens. Each sequence starts from state[slots[i]] (None:
    state[i]), or from zero where fresh[i] (bool [n]), and leaves its state
    there. Other arguments and the result are those of gated_delta_step; out must
    not overlap q, k or v, and its rows of no sequence are not written. The lengths
    are read on the device, so the call can be captured.

    Chunks of 64 tokens are multiplied with two bf16 terms per factor: the fp32
    state is within 2**-16 of its norm of the rule (2e-6 to 5e-6 measured), where
    gated_delta_step, all in fp32, keeps 2**-20, and out is rounded once more than
    there (2.3e-3 of its norm against 1.7e-3)."""
    return _lib.native().gated_delta_chunk(q, k, v, g, beta, state, cu_seqlens, slots, fresh, scale, l2norm, eps, out,
                                           workspace, status)
