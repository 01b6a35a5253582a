"""The path's operators registered with torch.library (namespace "d3moe").

Registered operators carry a schema and a fake (meta) implementation, so a
model that calls them can be traced (FakeTensor / meta tensors, torch.fx,
torch.export) and stays one opaque node per call. The reference registers its
own CUDA operators this way (src/drama3/ops/slot_attention.py:350-460). Each
operator runs the same C-ABI entry point as the function of the same name in
d3moe.ops; there is no CPU implementation.

Expert weights enter as tensors (w13, s13, w2, s2) with gate_up_order 0 for
w13 rows [gate | up] (the checkpoint order) and 1 for [up | gate]
(FlashInfer's order, src/drama3/model.py:196-201).
"""

from __future__ import annotations

import torch

from . import attention, cache, gated_delta, ops

FP8 = torch.float8_e4m3fn
_ORDERS = ("gate_up", "up_gate")


def _view(w13, s13, w2, s2, gate_up_order: int) -> ops.ExpertView:
    if gate_up_order not in (0, 1):
        raise ValueError("gate_up_order must be 0 (gate_up) or 1 (up_gate)")
    return ops.ExpertView(tensors=(w13, s13, w2, s2), gate_up_order=_ORDERS[gate_up_order])


@torch.library.custom_op("d3moe::quant_act_fp8", mutates_args=())
def quant_act_fp8(x: torch.Tensor, transposed: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """prepare_moe_input's activation quantiser (src/drama3/moe_input.py:24-27)."""
    return ops.quant_act_fp8(x, transposed=transposed)


@quant_act_fp8.register_fake
def _(x, transposed):
    T, H = x.shape
    s = (H // 128, T) if transposed else (T, H // 128)
    return x.new_empty((T, H), dtype=FP8), x.new_empty(s, dtype=torch.float32)


@torch.library.custom_op("d3moe::route_topk", mutates_args=())
def route_topk(logits: torch.Tensor, k: int, bias: torch.Tensor | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """route (src/drama3/kernels.py:360-383): (weights bf16 [T,k], ids int64 [T,k])."""
    return ops.route_topk(logits, k, bias=bias, weights_dtype=torch.bfloat16)


@route_topk.register_fake
def _(logits, k, bias=None):
    T = logits.shape[0]
    return (logits.new_empty((T, k), dtype=torch.bfloat16),
            logits.new_empty((T, k), dtype=torch.int64))


@torch.library.custom_op("d3moe::moe_experts", mutates_args=())
def moe_experts(x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                w13: torch.Tensor, s13: torch.Tensor, w2: torch.Tensor, s2: torch.Tensor,
                gate_up_order: int = 0) -> torch.Tensor:
    """Routed expert output bf16 [T,H] (small_batch_moe / native_moe,
    src/drama3/kernels.py:325-357, 702-779)."""
    routed, _ = ops.moe_experts(x, topk_ids, topk_weights, _view(w13, s13, w2, s2, gate_up_order))
    return routed


@moe_experts.register_fake
def _(x, topk_ids, topk_weights, w13, s13, w2, s2, gate_up_order=0):
    return x.new_empty(x.shape, dtype=torch.bfloat16)


@torch.library.custom_op("d3moe::moe_layer", mutates_args=())
def moe_layer(x: torch.Tensor, router_weight: torch.Tensor,
              w13: torch.Tensor, s13: torch.Tensor, w2: torch.Tensor, s2: torch.Tensor,
              sh_w13: torch.Tensor, sh_s13: torch.Tensor, sh_w2: torch.Tensor, sh_s2: torch.Tensor,
              k: int = 8, gate_up_order: int = 0) -> torch.Tensor:
    """Whole MoE layer (DramaModel.moe, src/drama3/model.py:485-541): router
    rows [E + 1, H] (the last row is the shared-expert gate), routed and shared
    experts, out = routed + bf16(shared * bf16(sigmoid(gate)))."""
    return ops.moe_layer(x, router_weight, _view(w13, s13, w2, s2, gate_up_order),
                         _view(sh_w13, sh_s13, sh_w2, sh_s2, gate_up_order), k)


@moe_layer.register_fake
def _(x, router_weight, w13, s13, w2, s2, sh_w13, sh_s13, sh_w2, sh_s2, k=8, gate_up_order=0):
    return x.new_empty(x.shape, dtype=torch.bfloat16)


@torch.library.custom_op("d3moe::fp8_gemv", mutates_args=())
def fp8_gemv(x: torch.Tensor, wq: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Weight-only FP8 projection y bf16 [T,N] (experimental_fp8.linear,
    src/drama3/experimental_fp8.py:56-79)."""
    return ops.fp8_gemv(x, wq, scales)


@fp8_gemv.register_fake
def _(x, wq, scales):
    return x.new_empty((x.shape[0], wq.shape[0]), dtype=torch.bfloat16)


@torch.library.custom_op("d3moe::combine_experts_add_norm", mutates_args=("residual",))
def combine_experts_add_norm(routed: torch.Tensor, shared: torch.Tensor, gate: torch.Tensor,
                             residual: torch.Tensor, weight: torch.Tensor, epsilon: float
                             ) -> torch.Tensor:
    """Layer exit (src/drama3/kernels.py:448-499): residual is updated in
    place and RMSNorm(residual) * (1 + weight) is returned."""
    return ops.combine_experts_add_norm(routed, shared, gate, residual, weight, epsilon)


@combine_experts_add_norm.register_fake
def _(routed, shared, gate, residual, weight, epsilon):
    return residual.new_empty(residual.shape, dtype=torch.bfloat16)


@torch.library.custom_op("d3moe::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, scale: float | None = None, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, window: int = 0,
                    max_seq_len: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, lse) of d3moe.attention.paged_attention."""
    return attention.paged_attention(q, k_cache, v_cache, page_table, seq_lens, scale, k_scale=k_scale,
                                     v_scale=v_scale, window=window, max_seq_len=max_seq_len, return_lse=True)


@paged_attention.register_fake
def _(q, k_cache, v_cache, page_table, seq_lens, scale=None, k_scale=None, v_scale=None, window=0, max_seq_len=None):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


@torch.library.custom_op("d3moe::kv_append", mutates_args=("k_cache", "v_cache"))
def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, positions: torch.Tensor, seq_ids: torch.Tensor | None = None,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None) -> None:
    """d3moe.attention.kv_append; the caches are declared as mutated."""
    attention.kv_append(k, v, k_cache, v_cache, page_table, positions, seq_ids, k_scale=k_scale, v_scale=v_scale)


@kv_append.register_fake
def _(k, v, k_cache, v_cache, page_table, positions, seq_ids=None, k_scale=None, v_scale=None):
    return None


@torch.library.custom_op("d3moe::copy_pages", mutates_args=("pool",))
def copy_pages(pool: torch.Tensor, src: torch.Tensor, dst: torch.Tensor, page_dim: int = 0) -> None:
    """d3moe.cache.copy_pages; the pool is declared as mutated."""
    cache.copy_pages(pool, src, dst, page_dim)


@copy_pages.register_fake
def _(pool, src, dst, page_dim=0):
    return None


@torch.library.custom_op("d3moe::gated_delta_step", mutates_args=("state",))
def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, slots: torch.Tensor | None = None, scale: float | None = None,
                     l2norm: bool = True, eps: float = 1e-6) -> torch.Tensor:
    """d3moe.gated_delta.gated_delta_step; the state is declared as mutated."""
    return gated_delta.gated_delta_step(q, k, v, g, beta, state, slots, scale=scale, l2norm=l2norm, eps=eps)


@gated_delta_step.register_fake
def _(q, k, v, g, beta, state, slots=None, scale=None, l2norm=True, eps=1e-6):
    return v.new_empty(v.shape)


@torch.library.custom_op("d3moe::gated_delta_chunk", mutates_args=("state",))
def gated_delta_chunk(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                      state: torch.Tensor, cu_seqlens: torch.Tensor, slots: torch.Tensor | None = None,
                      fresh: torch.Tensor | None = None, scale: float | None = None, l2norm: bool = True,
                      eps: float = 1e-6) -> torch.Tensor:
    """d3moe.gated_delta.gated_delta_chunk; the state is declared as mutated."""
    return gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu_seqlens, slots, fresh=fresh, scale=scale,
                                         l2norm=l2norm, eps=eps)


@gated_delta_chunk.register_fake
def _(q, k, v, g, beta, state, cu_seqlens, slots=None, fresh=None, scale=None, l2norm=True, eps=1e-6):
    return v.new_empty(v.shape)
