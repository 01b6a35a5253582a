"""A small hybrid decoder on d3moe's operators: prompts in, tokens out.

Layers alternate as in the decoder the package serves: gated-delta layers, and
an attention layer after every third of them, each followed by a mixture-of-
experts layer. Projections are the weight-only FP8 GEMV, weights are random.

  prefill   packed prompts: gated_delta_chunk, kv_append, causal attention of the
            prompt tokens by torch (the package has decode attention only)
  decode    one token per sequence: gated_delta_step, kv_append, paged_attention
  fork      PagedCache.fork for the pages, copy_pages for the recurrent state

    python examples/hybrid_decoder.py            # needs a B200 and the built library

Left out of the model, to keep it short: rotary positions, the short convolution
and the gates around the mixers.
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "drama-3-single-b300-inference_b200"))

from d3moe import attention, gated_delta, ops, synth  # noqa: E402
from d3moe.cache import PagedCache, copy_pages  # noqa: E402


class Projection:
    """y = x W^T with W [n, k] in FP8 blocks."""

    def __init__(self, n: int, k: int, gen: torch.Generator):
        w = (torch.randn((n, k), generator=gen, device="cuda") * k ** -0.5).to(torch.bfloat16)
        self.n, (self.q, self.s) = n, ops.fp8_quantize_weight(w)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return torch.cat([ops.fp8_gemv(part, self.q, self.s, n=self.n) for part in x.split(64)])


class Decoder:
    def __init__(self, layers: int = 4, hidden: int = 512, vocab: int = 1000, sequences: int = 8, max_len: int = 512,
                 heads: int = 4, kv_heads: int = 2, dim: int = 128, key_heads: int = 2, value_heads: int = 4,
                 experts: int = 16, expert_width: int = 256, seed: int = 0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.key_heads, self.value_heads = key_heads, value_heads
        self.embed = torch.randn((vocab, hidden), generator=gen, device="cuda").to(torch.bfloat16)
        self.head = torch.randn((vocab, hidden), generator=gen, device="cuda").to(torch.bfloat16)
        self.norm = torch.zeros(hidden, dtype=torch.bfloat16, device="cuda")
        self.kinds = ["attention" if i % 4 == 3 else "delta" for i in range(layers)]
        self.mixers, self.moes = [], []
        d, w = dim, 2 * key_heads * 128 + value_heads * 128
        for i, kind in enumerate(self.kinds):
            if kind == "attention":
                self.mixers.append((Projection((heads + 2 * kv_heads) * d, hidden, gen), Projection(hidden, heads * d, gen)))
            else:
                self.mixers.append((Projection(w + 2 * value_heads, hidden, gen), Projection(hidden, value_heads * 128, gen)))
            self.moes.append(synth.make_layer(experts, expert_width, hidden, seed=seed + i, device="cuda"))
        n_attn = self.kinds.count("attention")
        # every sequence may fill its length
        self.cache = PagedCache(n_attn, sequences * -(-max_len // 16), 16, kv_heads, d, sequences, max_len)
        self.state = torch.zeros((layers - n_attn, sequences, value_heads, 128, 128), device="cuda")

    # ------------------------------------------------------------- the mixers --
    def _delta(self, i: int, x: torch.Tensor):
        """(q, k, v, g, beta) of layer i."""
        Hk, Hv = self.key_heads, self.value_heads
        y = self.mixers[i][0](x)
        q, k, v, a, b = y.split([Hk * 128, Hk * 128, Hv * 128, Hv, Hv], dim=1)
        silu = torch.nn.functional.silu(y[:, :2 * Hk * 128 + Hv * 128])
        q, k, v = silu.split([Hk * 128, Hk * 128, Hv * 128], dim=1)
        g = -torch.nn.functional.softplus(a.float()) * 0.1
        return q.view(-1, Hk, 128), k.view(-1, Hk, 128), v.view(-1, Hv, 128), g, torch.sigmoid(b.float())

    def _qkv(self, i: int, x: torch.Tensor):
        H, Hkv, d = self.heads, self.kv_heads, self.dim
        q, k, v = self.mixers[i][0](x).split([H * d, Hkv * d, Hkv * d], dim=1)
        return q.view(-1, H, d), k.view(-1, Hkv, d), v.view(-1, Hkv, d)

    def _run(self, x: torch.Tensor, mix) -> torch.Tensor:
        """All layers over rows x; mix(kind, i, j, x) is layer i's mixer, the j-th of its kind. Returns logits."""
        seen = {"attention": 0, "delta": 0}
        residual = torch.zeros_like(x)
        for i, kind in enumerate(self.kinds):
            h = ops.add_norm(x, residual, self.norm, 1e-6)
            h = self.mixers[i][1](mix(kind, i, seen[kind], h).flatten(1))
            seen[kind] += 1
            h = ops.add_norm(h, residual, self.norm, 1e-6)
            lw = self.moes[i]
            x = ops.moe_layer(h, lw.router, lw.experts, lw.shared, 4)
        h = ops.add_norm(x, residual, self.norm, 1e-6)
        return h.float() @ self.head.float().T

    # --------------------------------------------------------------- the calls --
    def prefill(self, prompts: list[list[int]]) -> tuple[list[int], torch.Tensor]:
        """New sequences for the prompts: their numbers, and the logits of their last tokens."""
        i32 = dict(dtype=torch.int32, device="cuda")
        seqs = [self.cache.new() for _ in prompts]
        places = [self.cache.extend(s, len(p)) for s, p in zip(seqs, prompts)]
        ids = torch.tensor([t for p in prompts for t in p], device="cuda")
        pos = torch.tensor([t for r in places for t in r], **i32)
        owner = torch.tensor([s for s, p in zip(seqs, prompts) for _ in p], **i32)
        cu = torch.tensor([0] + [len(p) for p in prompts], **i32).cumsum(0, dtype=torch.int32)
        slots, fresh = torch.tensor(seqs, **i32), torch.ones(len(seqs), dtype=torch.bool, device="cuda")
        bounds = cu.tolist()

        def mix(kind, i, j, x):
            if kind == "delta":
                return gated_delta.gated_delta_chunk(*self._delta(i, x), self.state[j], cu, slots, fresh=fresh)
            q, k, v = self._qkv(i, x)
            attention.kv_append(k, v, self.cache.k(j), self.cache.v(j), self.cache.table, pos, owner)
            out = torch.empty_like(q)
            for a, b in zip(bounds, bounds[1:]):
                o = torch.nn.functional.scaled_dot_product_attention(
                    *(t[a:b].transpose(0, 1)[None] for t in (q, k, v)), is_causal=True, enable_gqa=True)
                out[a:b] = o[0].transpose(0, 1)
            return out

        return seqs, self._run(self.embed[ids], mix)[cu[1:].long() - 1]

    def decode(self, seqs: list[int], tokens: torch.Tensor) -> torch.Tensor:
        """One more token for each of the sequences: their next logits."""
        i32 = dict(dtype=torch.int32, device="cuda")
        pos = torch.tensor([self.cache.extend(s, 1)[0] for s in seqs], **i32)
        slots = torch.tensor(seqs, **i32)
        table = self.cache.table[slots.long()]
        longest = max(self.cache.lens[s] for s in seqs)

        def mix(kind, i, j, x):
            if kind == "delta":
                return gated_delta.gated_delta_step(*self._delta(i, x), self.state[j], slots)
            q, k, v = self._qkv(i, x)
            kc, vc = self.cache.k(j), self.cache.v(j)
            attention.kv_append(k, v, kc, vc, self.cache.table, pos, slots)
            return attention.paged_attention(q, kc, vc, table, pos + 1, max_seq_len=longest)

        return self._run(self.embed[tokens], mix)

    def fork(self, seq: int) -> int:
        """A second continuation of a sequence."""
        child = self.cache.fork(seq)
        one = dict(dtype=torch.int32, device="cuda")
        copy_pages(self.state, torch.tensor([seq], **one), torch.tensor([child], **one), 1)
        return child


def main() -> None:
    model = Decoder()
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (70, 5, 133)]
    seqs, logits = model.prefill(prompts)
    seqs.append(model.fork(seqs[2]))  # a second continuation of the longest prompt
    logits = torch.cat([logits, logits[2:]])
    second = logits.topk(2).indices[:, 1]
    tokens = logits.argmax(1)
    tokens[3] = second[3]  # ... that starts with its second-best token
    out = [[int(t)] for t in tokens]
    for _ in range(15):
        tokens = model.decode(seqs, tokens).argmax(1)
        for o, t in zip(out, tokens.tolist()):
            o.append(t)
    for s, o in zip(seqs, out):
        print(f"sequence {s}: {model.cache.lens[s]} tokens, continued with {o}")
    model.cache.free(seqs[0])
    print(f"{model.cache.compact()} pages moved after sequence {seqs[0]} ended, {model.cache.free_pages} are free")


if __name__ == "__main__":
    main()
