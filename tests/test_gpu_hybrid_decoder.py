"""The operators together, as examples/hybrid_decoder.py uses them: prompts taken at
once and token by token lead to the same logits, forks and compaction change
nothing, and the registered operators agree with the functions."""

from __future__ import annotations

import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from conftest import ROOT  # noqa: E402

sys.path.insert(0, str(ROOT / "examples"))


@pytest.fixture(scope="module")
def decoder():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import hybrid_decoder
    return hybrid_decoder


def _near(a, b):
    # bf16 activations through four layers, and FP8 requantisation between them: a last-bit
    # difference may move an FP8 value by 2**-4 of itself
    return float((a - b).norm() / b.norm()) < 2.0 ** -4


def test_prefill_equals_decoding_token_by_token(decoder):
    a, b = decoder.Decoder(), decoder.Decoder()
    prompts = [list(range(3, 73)), [9, 8, 7], list(range(500, 617))]
    seqs, logits = a.prefill(prompts)
    other, first = b.prefill([p[:1] for p in prompts])
    rows = [first[i] for i in range(3)]
    for t in range(1, max(map(len, prompts))):
        live = [i for i, p in enumerate(prompts) if t < len(p)]
        got = b.decode([other[i] for i in live], torch.tensor([prompts[i][t] for i in live], device="cuda"))
        for j, i in enumerate(live):
            rows[i] = got[j]
    for i in range(3):
        assert _near(rows[i], logits[i])
        assert torch.allclose(a.state[:, seqs[i]], b.state[:, other[i]], atol=float(a.state.abs().max()) * 2.0 ** -4)


def test_fork_and_compaction_change_no_logits(decoder):
    model = decoder.Decoder()
    seqs, _ = model.prefill([list(range(40)), list(range(100, 137)), list(range(7))])
    child = model.fork(seqs[1])
    step = torch.tensor([5, 5], device="cuda")
    got = model.decode([seqs[1], child], step)
    assert torch.equal(got[0], got[1])
    model.cache.free(seqs[0])
    before = model.cache.fork(child), model.cache.fork(child)  # two looks at the same place
    model.state[:, list(before)] = model.state[:, child][:, None]
    one = model.decode([before[0]], torch.tensor([11], device="cuda"))
    assert model.cache.compact() > 0
    assert torch.equal(model.decode([before[1]], torch.tensor([11], device="cuda")), one)


def test_example_runs(decoder, capsys):
    decoder.main()
    said = capsys.readouterr().out
    assert said.count("continued with") == 4 and "pages moved" in said


def test_registered_operators(decoder):
    from d3moe import attention, gated_delta, torch_ops  # noqa: F401
    g = torch.Generator(device="cuda").manual_seed(1)
    cache = torch.randn((2, 8, 16, 2, 64), generator=g, device="cuda").to(torch.bfloat16)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.tensor([50, 3], dtype=torch.int32, device="cuda")
    q = torch.randn((2, 4, 64), generator=g, device="cuda").to(torch.bfloat16)
    got = torch.ops.d3moe.paged_attention(q, cache[0], cache[1], table, lens)
    want = attention.paged_attention(q, cache[0], cache[1], table, lens, return_lse=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    both = ("test_schema", "test_faketensor")
    check = torch.library.opcheck
    check(torch.ops.d3moe.paged_attention.default, (q, cache[0].clone(), cache[1].clone(), table, lens), test_utils=both)
    check(torch.ops.d3moe.kv_append.default, (q[:, :2].contiguous(), q[:, 2:].contiguous(), cache[0].clone(), cache[1].clone(), table, lens), test_utils=both)
    pair = torch.tensor([[1], [5]], dtype=torch.int32, device="cuda")
    check(torch.ops.d3moe.copy_pages.default, (cache[0].clone(), pair[0], pair[1], 0), test_utils=both)
    k = torch.randn((3, 2, 64), generator=g, device="cuda").to(torch.bfloat16)
    v = torch.randn((3, 4, 64), generator=g, device="cuda").to(torch.bfloat16)
    gate = -torch.rand((3, 4), generator=g, device="cuda")
    state = torch.randn((3, 4, 64, 64), generator=g, device="cuda")
    a, b = state.clone(), state.clone()
    assert torch.equal(torch.ops.d3moe.gated_delta_step(k, k, v, gate, -gate, a), gated_delta.gated_delta_step(k, k, v, gate, -gate, b))
    assert torch.equal(a, b)
    check(torch.ops.d3moe.gated_delta_step.default, (k, k, v, gate, -gate, state), test_utils=both)
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda")
    check(torch.ops.d3moe.gated_delta_chunk.default, (k, k, v, gate, -gate, state, cu), test_utils=both)


def test_graph_capture(decoder):
    """A decode step's mixers replayed from a CUDA graph with other lengths than at capture."""
    from d3moe import attention, gated_delta
    g = torch.Generator(device="cuda").manual_seed(2)
    B = 3
    cache = torch.randn((2, 30, 16, 2, 128), generator=g, device="cuda").to(torch.bfloat16)
    table = torch.randperm(30, generator=g, device="cuda").int().view(B, 10)
    lens = torch.tensor([17, 1, 90], dtype=torch.int32, device="cuda")
    q = torch.randn((B, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    kv = torch.randn((2, B, 2, 128), generator=g, device="cuda").to(torch.bfloat16)
    state = torch.randn((B, 2, 128, 128), generator=g, device="cuda")
    gate = -torch.rand((B, 2), generator=g, device="cuda")

    def step(c, s):
        attention.kv_append(kv[0], kv[1], c[0], c[1], table, lens - 1)
        return attention.paged_attention(q, c[0], c[1], table, lens), gated_delta.gated_delta_step(kv[0], kv[0], kv[1], gate, -gate, s)

    step(cache.clone(), state.clone())  # first use outside the capture
    c, s = cache.clone(), state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(c, s)
    lens.copy_(torch.tensor([160, 33, 2], dtype=torch.int32))
    c.copy_(cache)
    s.copy_(state)
    graph.replay()
    c2, s2 = cache.clone(), state.clone()
    want = step(c2, s2)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert torch.equal(c, c2) and torch.equal(s, s2)
