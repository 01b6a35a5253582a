"""Operators between the projections and the MoE of a hybrid decoder layer, in plain form and through d3moe.

A decoder of this kind keeps two memories per sequence: pages of keys and values for its attention
layers, and one fp32 matrix per head for its gated-delta layers. The operators read, extend and move them:

  attention   one new token per sequence attends to its paged keys and values
  append      new keys and values are written to their pages
  copy        pages (or state slots) of every layer are copied to others: forks and compaction
  step        the gated delta rule for one new token per sequence
  chunk       the gated delta rule for packed prompts

`run` takes the elementary torch form where `own` is false and the package's operator where it is true.
Shapes follow the decoder the package serves (16 query and 2 key heads of 256, pages of 16 tokens; 16 key and
32 value heads of 128 for the delta rule; 10 attention and 30 delta layers), besides common other ones.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": FP8, "f32": torch.float32}
CHUNK = 64  # tokens per step of the plain chunked form


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "drama-3-single-b300-inference_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from d3moe import attention, cache, gated_delta

    return attention, cache, gated_delta


# ------------------------------------------------------------------ cases --


def listed():
    return [
        # one voice being generated, a few hundred audio tokens in: the latency of a single step
        dict(name="attention_one_short", op="attention", batch=1, heads=16, kv_heads=2, dim=256, page=16, longest=301, shortest=301, type="bf16", window=0),
        # a full decode bucket: 64 request slots at different points of their 2048-token limit
        dict(name="attention_64_ragged", op="attention", batch=64, heads=16, kv_heads=2, dim=256, page=16, longest=2048, shortest=0, type="bf16", window=0),
        # a few long documents: the cache's length has to be split over the whole GPU
        dict(name="attention_long", op="attention", batch=4, heads=16, kv_heads=2, dim=256, page=16, longest=131072, shortest=100003, type="bf16", window=0),
        # FP8 cache with more key heads and larger pages, mid-length contexts
        dict(name="attention_fp8", op="attention", batch=16, heads=32, kv_heads=8, dim=128, page=64, longest=16411, shortest=4000, type="e4m3", window=0),
        # the decode bucket's new keys and values
        dict(name="append_64", op="append", tokens=64, sequences=64, kv_heads=2, dim=256, page=16, type="bf16"),
        # a packed prefill's keys and values
        dict(name="append_prompts", op="append", tokens=15670, sequences=64, kv_heads=2, dim=256, page=16, type="bf16"),
        # 16 continuations fork: the half-filled last page of each, in all 10 attention layers (keys and values)
        dict(name="copy_fork", op="copy", planes=20, pages=600, move=16, elements=8192, type="bf16"),
        # a fragmented cache is compacted
        dict(name="copy_compact", op="copy", planes=20, pages=3600, move=1500, elements=8192, type="bf16"),
        # one voice's decode step through a gated-delta layer
        dict(name="step_one", op="step", batch=1, slots=8, key_heads=16, value_heads=32, key_dim=128, value_dim=128),
        # the full decode bucket's step
        dict(name="step_64", op="step", batch=64, slots=80, key_heads=16, value_heads=32, key_dim=128, value_dim=128),
        # one long prompt on its own: time to the first token
        dict(name="chunk_one_prompt", op="chunk", longest=2048, shortest=2048, sequences=1, key_heads=16, value_heads=32, key_dim=128, value_dim=128),
        # 64 ragged prompts packed into one prefill call
        dict(name="chunk_64_prompts", op="chunk", longest=512, shortest=16, sequences=64, key_heads=16, value_heads=32, key_dim=128, value_dim=128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "copy", "step", "chunk", "chunk"])
    if op == "attention":
        heads, kv_heads, dim = rng.choice([(16, 2, 256), (32, 8, 128), (16, 2, 128), (8, 8, 64), (24, 8, 64), (16, 1, 128), (20, 4, 128), (6, 2, 256)])
        batch = _log(rng, 1, 64)
        longest = _log(rng, 1, min(131072, 260_000_000 // (batch * kv_heads * dim)))
        shortest = rng.choice([0, longest, max(1, longest // 3)])
        window = rng.choice([0, 0, 0, max(1, longest // 2)])
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), longest=longest, shortest=shortest,
                    type=rng.choice(["bf16", "bf16", "f16", "e4m3"]), window=window)
    if op == "append":
        tokens = _log(rng, 1, 16384)
        kv_heads, dim = rng.choice([(2, 256), (8, 128), (4, 64), (1, 128)])
        return dict(op=op, tokens=tokens, sequences=rng.randint(1, min(64, tokens)), kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "f16"]))
    if op == "copy":
        planes = rng.randint(1, 30)
        elements = rng.choice([2048, 8192, 16384, 24584])
        kind = rng.choice(["bf16", "f16", "f32"])
        move = _log(rng, 1, min(1500, 480_000_000 // (planes * elements * (4 if kind == "f32" else 2))))
        return dict(op=op, planes=planes, pages=2 * move + rng.randint(1, 200), move=move, elements=elements, type=kind)
    heads = rng.choice([(16, 32), (16, 32), (4, 8), (6, 6), (2, 8)])
    key_dim, value_dim = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 64)])
    rest = dict(key_heads=heads[0], value_heads=heads[1], key_dim=key_dim, value_dim=value_dim)
    if op == "step":
        batch = _log(rng, 1, 96)
        return dict(op=op, batch=batch, slots=batch + rng.randint(1, 20), **rest)
    sequences = _log(rng, 1, 64)
    longest = _log(rng, 1, 16384 // sequences)
    return dict(op=op, longest=longest, shortest=rng.choice([1, longest, max(1, longest // 4)]), sequences=sequences, **rest)


def _lengths(case, seed):
    """Token counts of the sequences (those of the case alone decide how much work a pass is)."""
    n = case.get("batch", case.get("sequences"))
    g = torch.Generator().manual_seed(977 + n * 31 + case["longest"])
    lens = torch.randint(case["shortest"], case["longest"] + 1, (n,), generator=g)
    lens[0] = case["longest"]
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(int(seed)))
    return lens[perm]


# --------------------------------------------------------------- prepare --


def prepare(case, seed):
    return {"attention": _prepare_attention, "append": _prepare_append, "copy": _prepare_copy, "step": _prepare_step, "chunk": _prepare_chunk}[case["op"]](case, int(seed))


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 13)


def _randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _to_cache(x, scale, dtype):
    """Values [pages, page, heads, dim] as the cache holds them; an FP8 cache holds x / scale[head]."""
    return (x / scale[:, None]).clamp(-448, 448).to(dtype) if dtype == FP8 else x.to(dtype)


def _prepare_attention(case, seed):
    g, kind = _gen(seed), DTYPES[case["type"]]
    B, Hkv, D, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case, seed)
    need = [-(-int(n) // page) for n in lens]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1))
    width = max(1, -(-case["longest"] // page))
    table = torch.zeros((B, width), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    scales = (0.5 + torch.rand((2, Hkv), generator=g, device=DEV)) / 64 if kind == FP8 else None
    caches = [_to_cache(_randn(g, pages, page, Hkv, D), None if scales is None else scales[i], kind) for i in range(2)]
    # queries of a normalised projection; the logits' spread (about 3) gives some keys most of the weight
    q = _randn(g, B, case["heads"], D, scale=3.0).to(torch.bfloat16 if kind == FP8 else kind)
    return dict(case, q=q, k_cache=caches[0], v_cache=caches[1], table=table.to(DEV), lens=lens.int().to(DEV),
                k_scale=None if scales is None else scales[0].contiguous(), v_scale=None if scales is None else scales[1].contiguous())


def _prepare_append(case, seed):
    g, kind = _gen(seed), DTYPES[case["type"]]
    T, N, Hkv, D, page = case["tokens"], case["sequences"], case["kv_heads"], case["dim"], case["page"]
    new = torch.full((N,), T // N)
    new[: T % N] += 1
    r = torch.Generator().manual_seed(seed)
    before = torch.randint(0, 500, (N,), generator=r)  # tokens that each sequence has already
    need = (before + new + page - 1) // page
    pages = N * ((499 + int(new.max()) + page - 1) // page) + 4
    order = torch.randperm(pages, generator=r)
    table = torch.zeros((N, int(need.max())), dtype=torch.int32)
    at = 0
    for n in range(N):
        table[n, : need[n]] = order[at:at + need[n]].int()
        at += int(need[n])
    seq = torch.repeat_interleave(torch.arange(N), new)
    first = torch.cumsum(new, 0) - new
    pos = torch.arange(T) - first[seq] + before[seq]
    kv = _randn(g, T, 2 * Hkv * D).to(kind)  # the packed projection that holds the keys and the values
    return dict(case, k=kv[:, : Hkv * D].view(T, Hkv, D), v=kv[:, Hkv * D:].view(T, Hkv, D), table=table.to(DEV), seq=seq.int().to(DEV), pos=pos.int().to(DEV),
                k_cache=torch.zeros((pages, page, Hkv, D), dtype=kind, device=DEV), v_cache=torch.zeros((pages, page, Hkv, D), dtype=kind, device=DEV))


def _prepare_copy(case, seed):
    g = _gen(seed)
    pool = torch.empty((case["planes"], case["pages"], case["elements"]), dtype=DTYPES[case["type"]], device=DEV)
    for p in range(case["planes"]):
        pool[p] = _randn(g, case["pages"], case["elements"])
    order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed))
    src, dst = order[: case["move"]], order[case["move"]: 2 * case["move"]]
    return dict(case, pool=pool, src=src.int().to(DEV), dst=dst.int().to(DEV))


def _delta_inputs(case, g, T):
    """What a gated-delta layer's convolution and gate projections give: q | k | v of one packed row after SiLU, log decays and step sizes."""
    Hk, Hv, dk, dv = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    x = torch.nn.functional.silu(_randn(g, T, 2 * Hk * dk + Hv * dv, scale=1.5)).to(torch.bfloat16)
    q, k, v = x.split([Hk * dk, Hk * dk, Hv * dv], dim=1)
    rate = 1 + 15 * torch.rand((Hv,), generator=g, device=DEV)
    dt = torch.exp(torch.rand((Hv,), generator=g, device=DEV) * math.log(100) + math.log(1e-3))
    bias = dt + torch.log(-torch.expm1(-dt))
    decay = -rate * torch.nn.functional.softplus(_randn(g, T, Hv, scale=0.5) + bias)
    beta = torch.sigmoid(_randn(g, T, Hv))
    return dict(q=q.view(T, Hk, dk), k=k.view(T, Hk, dk), v=v.view(T, Hv, dv), g=decay, beta=beta)


def _prepare_step(case, seed):
    g = _gen(seed)
    ins = _delta_inputs(case, g, case["batch"])
    state = _randn(g, case["slots"], case["value_heads"], case["key_dim"], case["value_dim"], scale=0.3)
    slots = torch.randperm(case["slots"], generator=torch.Generator().manual_seed(seed))[: case["batch"]]
    return dict(case, **ins, state=state, slot=slots.int().to(DEV))


def _prepare_chunk(case, seed):
    g = _gen(seed)
    lens = _lengths(case, seed)
    cu = torch.zeros(len(lens) + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(lens, 0)
    ins = _delta_inputs(case, g, int(cu[-1]))
    n = case["sequences"]
    state = _randn(g, n + 2, case["value_heads"], case["key_dim"], case["value_dim"], scale=0.3)
    slots = torch.randperm(n + 2, generator=torch.Generator().manual_seed(seed))[:n]
    return dict(case, **ins, state=state, slot=slots.int().to(DEV), cu=cu.to(DEV), lens=lens.tolist())


# ------------------------------------------------------------------- run --


def run(s):
    if own:
        return _run_own(s)
    return {"attention": _plain_attention, "append": _plain_append, "copy": _plain_copy, "step": _plain_step, "chunk": _plain_chunk}[s["op"]](s)


def _run_own(s):
    attention, cache, gated_delta = _package()
    op = s["op"]
    if op == "attention":
        return attention.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], k_scale=s["k_scale"], v_scale=s["v_scale"], window=s["window"],
                                         max_seq_len=s["longest"], return_lse=True)
    if op == "append":
        attention.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["pos"], s["seq"])
        return s["k_cache"], s["v_cache"]
    if op == "copy":
        cache.copy_pages(s["pool"], s["src"], s["dst"], page_dim=1)
        return s["pool"]
    if op == "step":
        return gated_delta.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["slot"]), s["state"]
    return gated_delta.gated_delta_chunk(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["cu"], s["slot"]), s["state"]


def _plain_attention(s):
    q, table, lens = s["q"], s["table"].long(), s["lens"].long()
    B, Hq, D = q.shape
    Hkv = s["kv_heads"]
    L = s["longest"]
    pos = torch.arange(L, device=DEV)
    page, off = table[:, pos // s["page"]], (pos % s["page"]).expand(B, L)
    k = s["k_cache"][page, off].float()  # [B, L, Hkv, D]
    qs = (q.float() * D ** -0.5).view(B, Hkv, Hq // Hkv, D)
    if s["k_scale"] is not None:
        qs = qs * s["k_scale"][None, :, None, None]
    logits = qs @ k.permute(0, 2, 3, 1)  # [B, Hkv, G, L]
    del k
    begin = (lens - s["window"]).clamp(min=0) if s["window"] else torch.zeros_like(lens)
    keep = (pos < lens[:, None]) & (pos >= begin[:, None])
    logits = torch.where(keep[:, None, None], logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(logits - top)
    total = p.sum(-1, keepdim=True)
    o = (p @ s["v_cache"][page, off].float().transpose(1, 2)) / total.clamp(min=1e-30)
    if s["v_scale"] is not None:
        o = o * s["v_scale"][None, :, None, None]
    return o.view(B, Hq, D).to(q.dtype), (torch.log(total) + top).view(B, Hq)


def _plain_append(s):
    page = s["table"][s["seq"].long(), s["pos"].long() // s["page"]].long()
    off = s["pos"].long() % s["page"]
    s["k_cache"][page, off] = s["k"]
    s["v_cache"][page, off] = s["v"]
    return s["k_cache"], s["v_cache"]


def _plain_copy(s):
    s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    return s["pool"]


def _normed(x):
    x = x.float()
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_step(s):
    rep = s["value_heads"] // s["key_heads"]
    q = _normed(s["q"]).repeat_interleave(rep, 1) * s["key_dim"] ** -0.5
    k = _normed(s["k"]).repeat_interleave(rep, 1)
    slot = s["slot"].long()
    S = s["state"][slot] * torch.exp(s["g"])[:, :, None, None]
    delta = s["beta"][:, :, None] * (s["v"].float() - (k[:, :, None, :] @ S).squeeze(2))
    S = S + k[:, :, :, None] * delta[:, :, None, :]
    o = (q[:, :, None, :] @ S).squeeze(2)
    s["state"][slot] = S
    return o.to(torch.bfloat16), s["state"]


def _plain_chunk(s):
    """Prompts side by side in one padded batch; what of a chunk does not need the state is computed for all chunks at once, then the state goes from chunk to chunk."""
    N, Hv, dk, dv = s["sequences"], s["value_heads"], s["key_dim"], s["value_dim"]
    rep, C = Hv // s["key_heads"], CHUNK
    n = -(-s["longest"] // C)
    cu = s["cu"].long()
    at = cu[:-1, None] + torch.arange(n * C, device=DEV)
    keep = at < cu[1:, None]
    at = torch.where(keep, at, 0)

    def chunks(x):  # [T, H, ...] -> [N, H, n, C, ...], zero behind each prompt's end
        x = torch.where(keep.view(N, n * C, *[1] * (x.dim() - 1)), x[at], 0)
        return x.view(N, n, C, *x.shape[2:]).movedim(3, 1)

    q = chunks(_normed(s["q"]) * dk ** -0.5).repeat_interleave(rep, 1)
    k = chunks(_normed(s["k"])).repeat_interleave(rep, 1)
    v, beta = chunks(s["v"].float()), chunks(s["beta"])
    G = torch.cumsum(chunks(s["g"]), -1)
    lower = torch.ones((C, C), device=DEV).tril()
    decay = torch.exp(torch.where(lower > 0, G[..., :, None] - G[..., None, :], -math.inf))
    eye = torch.eye(C, device=DEV)
    A = beta[..., None] * (k @ k.transpose(-1, -2)) * decay * lower.tril(-1)
    A2 = A @ A
    A4 = A2 @ A2
    A8 = A4 @ A4
    A16 = A8 @ A8
    T = (eye - A) @ (eye + A2) @ (eye + A4) @ (eye + A8) @ (eye + A16) @ (eye + A16 @ A16)  # (I + A)^-1: A^64 = 0
    del A, A2, A4, A8, A16
    U, W = T @ (beta[..., None] * v), T @ ((beta * torch.exp(G))[..., None] * k)
    P = (q @ k.transpose(-1, -2)) * decay
    qg, kg = q * torch.exp(G)[..., None], (k * torch.exp(G[..., -1:] - G)[..., None]).transpose(-1, -2)
    end = torch.exp(G[..., -1])[..., None, None]
    slot = s["slot"].long()
    S = s["state"][slot]
    o = torch.empty((N, Hv, n, C, dv), device=DEV)
    for c in range(n):
        new = U[:, :, c] - W[:, :, c] @ S
        o[:, :, c] = qg[:, :, c] @ S + P[:, :, c] @ new
        S = S * end[:, :, c] + kg[:, :, c] @ new
    s["state"][slot] = S
    return o.movedim(1, 3).reshape(N, n * C, Hv, dv)[keep].to(torch.bfloat16), s["state"]


# ------------------------------------------------------------------ work --


def work(case):
    op = case["op"]
    if op == "attention":
        lens = _lengths(case, 0).tolist()
        keys = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        D, size = case["dim"], 1 if case["type"] == "e4m3" else 2
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * keys * case["kv_heads"] * D * size + case["batch"] * case["heads"] * (4 * D + 4) + 4 * pages + 4 * case["batch"],
                "flops": 4 * keys * case["heads"] * D}
    if op == "append":
        return {"bytes": 2 * 2 * case["tokens"] * case["kv_heads"] * case["dim"] * 2 + 12 * case["tokens"], "flops": 0}
    if op == "copy":
        return {"bytes": 2 * case["planes"] * case["move"] * case["elements"] * (4 if case["type"] == "f32" else 2) + 8 * case["move"], "flops": 0}
    Hk, Hv, dk, dv = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    n = case["batch"] if op == "step" else case["sequences"]
    T = n if op == "step" else int(_lengths(case, 0).sum())
    return {"bytes": 2 * T * (2 * Hk * dk + 2 * Hv * dv) + 8 * T * Hv + 8 * n * Hv * dk * dv + 4 * n, "flops": 6 * T * Hv * dk * dv}


# ----------------------------------------------------------------- exact --


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "append": _exact_append, "copy": _exact_copy, "step": _exact_step, "chunk": _exact_chunk}[case["op"]](s)


def _exact_attention(s):
    B, Hq, D = s["q"].shape
    Hkv, out, lse = s["kv_heads"], [], []
    for b, n in enumerate(s["lens"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == 0:
            out.append(torch.zeros((Hq, D), dtype=torch.float64, device=DEV))
            lse.append(torch.full((Hq,), -math.inf, dtype=torch.float64, device=DEV))
            continue
        ids = s["table"][b, : -(-n // s["page"])].long()
        heads = []
        for h in range(Hkv):
            k, v = (s[c][ids, :, h].reshape(-1, D)[lo:n].double() for c in ("k_cache", "v_cache"))
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            x = s["q"][b, h * (Hq // Hkv):(h + 1) * (Hq // Hkv)].double() @ k.T / math.sqrt(D)
            heads.append((torch.softmax(x, -1) @ v, torch.logsumexp(x, -1)))
        out.append(torch.cat([a for a, _ in heads]))
        lse.append(torch.cat([a for _, a in heads]))
    return torch.stack(out), torch.stack(lse)


def _exact_append(s):
    found = []
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        flat = cache.double().flatten(0, 1)
        row = s["table"].long()[s["seq"].long(), torch.div(s["pos"], s["page"], rounding_mode="floor").long()] * s["page"] + s["pos"] % s["page"]
        found.append(flat.index_copy(0, row, new.double()).view(cache.shape))
    return tuple(found)


def _exact_copy(s):
    pool = s["pool"].clone()
    for p in range(pool.shape[0]):
        pool[p].index_copy_(0, s["dst"].long(), pool[p].index_select(0, s["src"].long()))
    return pool


def _unit(x):
    x = x.double()
    return x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)


def _exact_token(S, q, k, v, g, beta):
    """One token: S [N, H, dk, dv] decays, then moves towards v along k; what q reads from it."""
    S.mul_(g.exp()[..., None, None])
    err = beta[..., None] * (v - torch.einsum("nhkv,nhk->nhv", S, k))
    S.addcmul_(k[..., :, None], err[..., None, :])
    return torch.einsum("nhkv,nhk->nhv", S, q)


def _exact_step(s):
    rep = s["value_heads"] // s["key_heads"]
    q, k = (_unit(s[x]).repeat_interleave(rep, 1) for x in ("q", "k"))
    state = s["state"].double()
    S = state[s["slot"].long()]
    o = _exact_token(S, q / math.sqrt(s["key_dim"]), k, s["v"].double(), s["g"].double(), s["beta"].double())
    state[s["slot"].long()] = S
    return o, state


def _exact_chunk(s):
    rep = s["value_heads"] // s["key_heads"]
    q, k = _unit(s["q"]) / math.sqrt(s["key_dim"]), _unit(s["k"])
    cu, lens = s["cu"].tolist(), s["lens"]
    state = s["state"].double()
    slot = s["slot"].long()
    order = sorted(range(len(lens)), key=lambda i: -lens[i])  # the longest first: those that go on are always a prefix
    S = state[slot[order]]
    start = torch.tensor([cu[i] for i in order], device=DEV)
    o = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
    for t in range(max(lens)):
        n = sum(lens[i] > t for i in order)
        at = start[:n] + t
        o[at] = _exact_token(S[:n], q[at].repeat_interleave(rep, 1), k[at].repeat_interleave(rep, 1), s["v"][at].double(), s["g"][at].double(), s["beta"][at].double())
    state[slot[order]] = S
    return o, state
