"""Plain 64-bit forms of the sequence-memory operators, and the error bounds the
tests hold the kernels to.

Bounds. A bf16 value has 8 significant bits, so rounding to nearest changes it
by at most U = 2**-8 of itself (f16: 2**-11); fp32 sums of n terms are off by
at most n * 2**-24 of the sum of their magnitudes."""

from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS32 = 2.0 ** -24


def gather_rows(cache, table, b, lo, hi, head, scale=None):
    """Rows [lo, hi) of one sequence's head as float64 [hi - lo, dim]."""
    page = cache.shape[1]
    t = torch.arange(lo, hi, device=cache.device)
    rows = cache[table[b, t // page].long(), t % page, head].double()
    return rows if scale is None else rows * scale[head].double()


def attention(q, k_cache, v_cache, table, lens, scale, window=0, k_scale=None, v_scale=None):
    """(out, lse, bound on out, bound on lse), float64. The bound on out: the
    output's own rounding, one rounding of each probability to 16 bits before
    it meets V, and the fp32 noise of the logits and sums."""
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    G = Hq // Hkv
    out = torch.zeros((B, Hq, D), dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    bo, bl = torch.zeros_like(out), torch.zeros((B, Hq), dtype=torch.float64, device=q.device)
    u_out, u_p = U[q.dtype], U[q.dtype if k_cache.dtype != torch.float8_e4m3fn else torch.float16]
    for b, n in enumerate(lens.tolist()):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        for h in range(Hkv):
            k = gather_rows(k_cache, table, b, lo, n, h, k_scale)
            v = gather_rows(v_cache, table, b, lo, n, h, v_scale)
            sl = slice(h * G, (h + 1) * G)
            qh = q[b, sl].double()
            x = qh @ k.T * scale
            p = torch.softmax(x, -1)
            noise = ((D + 8) * EPS32 * abs(scale) * (qh.abs() @ k.abs().T)).amax(-1)  # of one logit
            out[b, sl], lse[b, sl] = p @ v, torch.logsumexp(x, -1)
            spread = p @ v.abs()
            rel = 2 * noise + (n - lo + 64) * EPS32 + 2.0 ** -20
            bo[b, sl] = u_out * (p @ v).abs() + (u_p + rel)[:, None] * spread * (1 + u_out) + 1e-30
            bl[b, sl] = noise + (n - lo + 64) * EPS32 + 2.0 ** -21 * lse[b, sl].abs() + 2.0 ** -21
    return out, lse, bo, bl


def unit(x, l2norm=True, eps=1e-6):
    x = x.double()
    return x / torch.sqrt(x.square().sum(-1, keepdim=True) + eps) if l2norm else x


def delta(q, k, v, g, beta, state, spans, slots, scale, l2norm=True, eps=1e-6, fresh=None):
    """The recurrence token by token in float64: (out, new state pool)."""
    rep = v.shape[1] // q.shape[1]
    qn = unit(q, l2norm, eps).repeat_interleave(rep, 1) * scale
    kn = unit(k, l2norm, eps).repeat_interleave(rep, 1)
    state = state.double().clone()
    out = torch.zeros(v.shape, dtype=torch.float64, device=v.device)
    for i, (a, b) in enumerate(spans):
        if slots[i] < 0 or slots[i] >= state.shape[0]:
            continue
        S = state[slots[i]].clone()
        if fresh is not None and fresh[i]:
            S.zero_()
        for t in range(a, b):
            S = S * torch.exp(g[t].double())[:, None, None]
            d = beta[t].double()[:, None] * (v[t].double() - torch.einsum("hkv,hk->hv", S, kn[t]))
            S = S + kn[t][:, :, None] * d[:, None, :]
            out[t] = torch.einsum("hkv,hk->hv", S, qn[t])
        state[slots[i]] = S
    return out, state


def rel_l2(got, want):
    want = want.double()
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))
