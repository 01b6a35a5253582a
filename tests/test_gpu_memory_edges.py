"""What the sequence-memory operators take at the edges of sizes and strides."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


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
