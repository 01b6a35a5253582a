"""What the sequence-memory operators take at the edges of sizes and strides."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention import BF16, make_cache  # noqa: E402
from test_gpu_gated_delta import operands, pool  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("shape,page_dim", [((0, 5, 8), 1), ((2, 0, 5, 8), 2), ((3, 2, 0, 5, 8), 3), ((5, 2, 0), 0), ((2, 0, 8), 1), ((4, 3, 0, 2), 1)])
def test_copy_pages_of_an_empty_pool(shape, page_dim):
    from d3moe import cache
    at = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    cache.copy_pages(torch.empty(shape, device="cuda"), at, at + 2, page_dim)
    with pytest.raises(ValueError, match="dst"):
        cache.copy_pages(torch.empty(shape, device="cuda"), at, at.long(), page_dim)


def test_strides_of_axes_with_one_entry():
    from d3moe import attention, gated_delta

    def odd(x):  # the same values, the first axis (one entry) with a stride that is not a multiple of 16 bytes
        wide = torch.zeros(x.numel() + 3, dtype=x.dtype, device="cuda")
        wide[:x.numel()] = x.flatten()
        return wide.as_strided(x.shape, (x.numel() + 3, *x.stride()[1:]))

    k, v, table, _, _ = make_cache([9], 1, 64, 16, BF16, spare=0)  # one page, one head
    ln = torch.tensor([9], dtype=torch.int32, device="cuda")
    q = torch.randn((1, 4, 64), device="cuda").to(BF16)
    want = attention.paged_attention(q, k, v, table, ln)
    narrow = torch.cat([table[:, :1], table[:, :1]], 1).t()[:1].t()[:, :1]  # width 1
    narrow = narrow.as_strided((1, 1), (1, 7))
    one = k.as_strided(k.shape, (k.numel() + 5, 64, 3, 1))
    assert torch.equal(attention.paged_attention(odd(q), one, v, narrow, ln, out=odd(torch.zeros_like(q))), want)
    new = torch.randn((1, 1, 64), device="cuda").to(BF16)
    pos = torch.tensor([4], dtype=torch.int32, device="cuda")
    attention.kv_append(odd(new), odd(new), k, v, narrow, pos)
    assert torch.equal(k[int(table[0, 0]), 4], new[0]) and torch.equal(v[int(table[0, 0]), 4], new[0])
    ops = operands(1, 2, 4, 128, 128)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for f, extra in ((gated_delta.gated_delta_step, ()), (gated_delta.gated_delta_chunk, (cu,))):
        a, b = pool(1, 4, 128, 128), odd(pool(1, 4, 128, 128))
        assert torch.equal(f(*ops, a, *extra), f(*map(odd, (x.contiguous() for x in ops)), b, *extra)) and torch.equal(a, b)
