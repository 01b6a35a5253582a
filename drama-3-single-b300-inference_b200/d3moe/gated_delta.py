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

from ._lib import D3GatedDelta, call
from .attention import _index_ptr, _need_cuda, _status_ptr, _stream


def _operands(q, k, v, g, beta, state, slots, n, scale, l2norm, eps, out):
    dev = state.get_device()
    _need_cuda(dev)
    qs, vs, ss = q.shape, v.shape, state.shape
    if len(qs) != 3 or len(vs) != 3 or len(ss) != 4:
        raise ValueError("q, k, v must be [T, heads, dim] and state [slots, heads, key_dim, value_dim]")
    T, Hk, dk = qs
    _, Hv, dv = vs
    gates = (T, Hv)
    if k.shape != qs or vs[0] != T or g.shape != gates or beta.shape != gates:
        raise ValueError("k must have the shape of q, v its tokens, g and beta [T, value_heads]")
    if ss[1:] != (Hv, dk, dv):
        raise ValueError(f"state must be [slots, {Hv}, {dk}, {dv}]")
    bf16, f32 = torch.bfloat16, torch.float32
    if q.dtype is not bf16 or k.dtype is not bf16 or v.dtype is not bf16:
        raise ValueError("q, k and v must be bfloat16")
    if g.dtype is not f32 or beta.dtype is not f32 or state.dtype is not f32:
        raise ValueError("g, beta and state must be float32")
    if (q.get_device() != dev or k.get_device() != dev or v.get_device() != dev or g.get_device() != dev
            or beta.get_device() != dev):
        raise ValueError("all operands must be on one device")
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    s0, s1, s2, s3 = state.stride()
    g0, g1 = g.stride()
    b0, b1 = beta.stride()
    if T and (q2 != 1 or k2 != 1 or v2 != 1 or (q1 != dk or k1 != dk) and Hk > 1 or v1 != dv and Hv > 1):
        raise ValueError("heads and dims of q, k, v and out must be contiguous (tokens may be strided)")
    if out is None:
        out = torch.empty_like(v)
    elif out.shape != vs or out.dtype is not bf16 or out.get_device() != dev:
        raise ValueError("out must be bfloat16 with the shape and device of v")
    o0, o1, o2 = out.stride()
    if T and (o2 != 1 or o1 != dv and Hv > 1):
        raise ValueError("heads and dims of q, k, v and out must be contiguous (tokens may be strided)")
    if s3 != 1 or s2 != dv or s1 != dk * dv and Hv > 1:
        raise ValueError("each slot of state must be contiguous")
    if T and Hv > 1 and (g1 != 1 or b1 != 1):
        raise ValueError("heads of g and beta must be contiguous")
    if slots is None and n > ss[0]:
        raise ValueError("state has fewer slots than there are sequences")
    a = D3GatedDelta(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), out.data_ptr(),
                     state.data_ptr(), None if slots is None else _index_ptr(slots, n, dev, "slots"),
                     q0, k0, v0, g0, b0, o0, s0, ss[0], Hk, Hv, dk, dv,
                     1 if l2norm else 0, dk ** -0.5 if scale is None else scale, eps)
    return a, out, dev


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, slots: torch.Tensor | None = None, *, scale: float | None = None,
                     l2norm: bool = True, eps: float = 1e-6, out: torch.Tensor | None = None,
                     status: torch.Tensor | None = None) -> torch.Tensor:
    """One token for each of n sequences: q, k bf16 [n, key_heads, key_dim], v
    bf16 [n, value_heads, value_dim], g (log decay) and beta f32 [n,
    value_heads]. Sequence i's state is state[slots[i]] (int32; None: state[i]),
    updated in place; a negative slot leaves the sequence out (zero row). q and
    k are divided by sqrt(|x|^2 + eps) when l2norm; scale: key_dim**-0.5 by
    default. Returns out bf16 [n, value_heads, value_dim]."""
    n = q.shape[0]
    a, out, dev = _operands(q, k, v, g, beta, state, slots, n, scale, l2norm, eps, out)
    call("d3_gated_delta_step", ctypes.byref(a), n, _status_ptr(status, dev), _stream(dev))
    return out


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
    there. Other arguments and the result are those of gated_delta_step. The
    lengths are read on the device, so the call can be captured."""
    n = cu_seqlens.numel() - 1
    if n < 0:
        raise ValueError("cu_seqlens must hold n + 1 row starts")
    a, out, dev = _operands(q, k, v, g, beta, state, slots, n, scale, l2norm, eps, out)
    if fresh is not None and (fresh.dtype not in (torch.bool, torch.uint8) or fresh.shape != (n,)
                              or not fresh.is_contiguous() or fresh.get_device() != dev):
        raise ValueError(f"fresh must be contiguous bool [{n}] on the operands' device")
    T = q.shape[0]
    if workspace is None:
        workspace = gated_delta_chunk_workspace(T, n, a.value_heads, a.key_dim, a.value_dim, q.device)
    call("d3_gated_delta_chunk", ctypes.byref(a), _index_ptr(cu_seqlens, n + 1, dev, "cu_seqlens"), T, n,
         None if fresh is None else fresh.data_ptr(), workspace.data_ptr(), workspace.numel(), _status_ptr(status, dev), _stream(dev))
    return out
