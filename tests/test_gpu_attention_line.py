"""Paged attention where all units' tiles form one line that the CTAs share (bounds above 24
tiles of at most 128 keys), and clusters whose CTAs outnumber the tiles, against the 64-bit form."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402
from test_gpu_attention import BF16, F16, FP8, check_attention, make_cache  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


RAGGED = [4100, 1, 0, 63, 64, 65, 700, 3999, 128, 17, 0, 2050]


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,heads", [(16, 2), (8, 8), (16, 1), (5, 1), (24, 2), (20, 1)])
def test_ragged_sequences(dtype, dim, q_heads, heads):
    """8 and 16 heads per unit, part-filled and several units per key head, every type and dim."""
    check_attention(RAGGED, q_heads, heads, dim, 16, dtype, seed=dim + q_heads)


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_mid_length_sequences_of_the_fp8_kind(dtype):
    g = torch.Generator().manual_seed(1)
    check_attention([4203] + torch.randint(1000, 4200, (9,), generator=g).tolist(), 32, 8, 128, 64, dtype)


# the scan over the sequences takes several per thread from 129 on; 300 sequences of 4 heads are more rows than 8 per SM
@pytest.mark.parametrize("B", [100, 129, 300, 1500])
@pytest.mark.parametrize("dtype,q_heads,heads,dim", [(BF16, 4, 1, 64), (F16, 16, 1, 128), (FP8, 4, 2, 128)])
def test_many_sequences(B, dtype, q_heads, heads, dim):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    lens[B // 3], lens[-1] = 3500, 1
    check_attention(lens, q_heads, heads, dim, 16, dtype)


def test_many_long_sequences():
    """Shares that hold several whole units between two parts."""
    g = torch.Generator().manual_seed(6)
    lens = torch.randint(0, 400, (700,), generator=g).tolist()
    lens[0], lens[350] = 3301, 3400
    check_attention(lens, 8, 1, 64, 16, BF16)


@pytest.mark.parametrize("window", [3400, 3500, 4096])
@pytest.mark.parametrize("dtype,q_heads,heads,dim", [(BF16, 16, 2, 256), (FP8, 16, 2, 128), (F16, 16, 1, 64)])
def test_windows(window, dtype, q_heads, heads, dim):
    check_attention([9001, 3450, 3399, 100, 0, 5000], q_heads, heads, dim, 32, dtype, window=window)


@pytest.mark.parametrize("page,heads_first", [(1, False), (24, True), (128, False)])
def test_pages(page, heads_first):
    for dtype in (BF16, FP8):
        check_attention([3700, 90, 1500], 8, 2, 128, page, dtype, heads_first=heads_first)


@pytest.mark.parametrize("lens,window", [([700, 1, 30], 600), ([650], 500), ([64, 500, 0], 450)])
@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_clusters_with_fewer_tiles_than_ctas_under_a_window(lens, window, dtype):
    check_attention(lens, 16, 2, 256, 16, dtype, window=window)


def test_bad_page_on_the_line():
    from d3moe import _lib, attention
    k, v, table, _, _ = make_cache([5000, 40], 2, 128, 16, BF16)
    k.nan_to_num_()
    v.nan_to_num_()
    q = torch.randn((2, 4, 128), device="cuda").to(BF16)
    ln = torch.tensor([5000, 40], dtype=torch.int32, device="cuda")
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        t = table.clone()
        t[0, 200] = bad
        got = attention.paged_attention(q, k, v, t, ln, status=status)
        assert int(status) == _lib.D3_STATUS_BAD_ROW
        t[0, 200] = 0
        status.zero_()
        assert torch.equal(got, attention.paged_attention(q, k, v, t, ln, status=status)) and int(status) == 0


@pytest.mark.parametrize("dtype", [BF16, FP8])
def test_every_form_gives_equal_bits_again(dtype):
    from d3moe import attention
    for lens, limit in ((RAGGED, None), ([40, 130], 200), ([301], 1000)):
        k, v, table, ks, vs = make_cache(lens, 2, 128, 16, dtype)
        q = torch.randn((len(lens), 16, 128), generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        call = lambda: attention.paged_attention(q, k, v, table, ln, k_scale=ks, v_scale=vs, max_seq_len=limit, return_lse=True)  # noqa: E731
        want = call()
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(call(), want))


def test_the_forms_agree():
    """The same short sequence whole, by a cluster and on the line: only the bound on the host differs."""
    from d3moe import attention
    k, v, _, _, _ = make_cache([90], 2, 128, 16, BF16, spare=300)
    table = torch.arange(k.shape[0], dtype=torch.int32, device="cuda")[None]
    k.nan_to_num_()
    v.nan_to_num_()
    q = torch.randn((1, 16, 128), generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    ln = torch.tensor([90], dtype=torch.int32, device="cuda")
    want, wlse, bo, bl = R.attention(q, k, v, table, ln, 128 ** -0.5)
    for limit in (100, 128, 1000, 1536, 4000):
        got, lse = attention.paged_attention(q, k, v, table, ln, max_seq_len=limit, return_lse=True)
        assert ((got.double() - want).abs() <= bo).all() and ((lse.double() - wlse).abs() <= bl).all()
