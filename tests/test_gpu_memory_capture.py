"""Every sequence-memory operator replayed from a CUDA graph with other lengths, slots and pages
than at capture, and the states that prompts leave compared per layer, sequence and head."""

from __future__ import annotations

import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402
from conftest import ROOT  # noqa: E402
from test_gpu_attention import BF16, make_cache  # noqa: E402
from test_gpu_gated_delta import operands, pool  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _graph(call):
    call()  # first use outside the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    return graph, out


@pytest.mark.parametrize("limit", [90, 1000, 4200])  # units whole, by clusters, the line and its joining kernel
def test_attention(limit):
    from d3moe import attention
    k, v, table, _, _ = make_cache([4200, 4200, 4200], 2, 128, 16, BF16)
    q = torch.randn((3, 16, 128), device="cuda").to(BF16)
    lens = _i32([limit, 3, limit // 2])
    call = lambda: attention.paged_attention(q, k, v, table, lens, max_seq_len=limit)  # noqa: E731
    graph, out = _graph(call)
    for now in ([1, limit, 0], [limit - 1, limit // 3, limit], [0, 0, 0]):
        lens.copy_(_i32(now))
        graph.replay()
        assert torch.equal(out, call())


@pytest.mark.parametrize("n", [3, 40])  # pairs of warps, and without
def test_delta_chunk(n):
    from d3moe import gated_delta
    q, k, v, g, beta = operands(n * 50, 2, 4, 128, 128)
    first = pool(n + 2, 4, 128, 128)
    state, slots, fresh = first.clone(), _i32(list(range(n))), torch.zeros(n, dtype=torch.bool, device="cuda")
    cu = _i32([50 * i for i in range(n + 1)])
    graph, out = _graph(lambda: gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu, slots, fresh=fresh))
    cu.copy_(_i32([0, 130] + [130 + (i * (n * 50 - 130)) // (n - 1) for i in range(1, n)]))
    slots.copy_(_i32(list(range(n + 1, 1, -1))))
    fresh[1] = True
    state.copy_(first)
    graph.replay()
    again = first.clone()
    assert torch.equal(out, gated_delta.gated_delta_chunk(q, k, v, g, beta, again, cu, slots, fresh=fresh))
    assert torch.equal(state, again)


def test_copy_pages_and_append():
    from d3moe import attention, cache
    first = torch.randn((2, 12, 16, 2, 64), device="cuda").to(BF16)
    kv, new = first.clone(), torch.randn((2, 3, 2, 64), device="cuda").to(BF16)
    src, dst, pos, table = _i32([0, 1, -1]), _i32([4, 5, 6]), _i32([3, 17, 2]), _i32([[0, 1], [2, 3], [7, 8]])

    def call():
        cache.copy_pages(kv, src, dst, 1)
        attention.kv_append(new[0], new[1], kv[0], kv[1], table, pos)

    graph, _ = _graph(call)
    src.copy_(_i32([9, 2, 3]))
    dst.copy_(_i32([10, 5, 11]))
    pos.copy_(_i32([31, -1, 0]))
    kv.copy_(first)
    graph.replay()
    got = kv.clone()
    kv.copy_(first)
    call()
    assert torch.equal(got, kv) and not torch.equal(got, first)


def test_prompts_at_once_and_token_by_token_leave_the_same_states():
    # the bound of the logits, a FP8 value's last bit, for each layer, sequence and head on its own
    sys.path.insert(0, str(ROOT / "examples"))
    import hybrid_decoder
    a, b = hybrid_decoder.Decoder(), hybrid_decoder.Decoder()
    prompts = [list(range(3, 73)), [9, 8, 7], list(range(500, 617))]
    seqs, _ = a.prefill(prompts)
    other, _ = b.prefill([p[:1] for p in prompts])
    for t in range(1, max(map(len, prompts))):
        live = [i for i, p in enumerate(prompts) if t < len(p)]
        b.decode([other[i] for i in live], torch.tensor([prompts[i][t] for i in live], device="cuda"))
    for layer in range(a.state.shape[0]):
        for s, o in zip(seqs, other):
            for h in range(a.state.shape[2]):
                assert R.rel_l2(a.state[layer, s, h], b.state[layer, o, h]) < 2.0 ** -4, (layer, s, h)
