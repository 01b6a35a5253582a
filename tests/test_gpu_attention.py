"""Paged attention and the cache's writes (append, page copies) on the GPU against
their plain 64-bit forms."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def make_cache(lens, heads, dim, page, dtype, seed=0, heads_first=False, spare=3):
    """A cache whose unused places hold NaN, its shuffled page table and scales."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need + [1]) + 1), 2 ** 30, dtype=torch.int32)  # unused entries lie outside
    filled = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = ids.int()
        t = torch.arange(n)
        filled[ids[t // page], t % page] = True
    scales = [torch.rand(heads, generator=g).cuda() / 32 + 0.01 for _ in range(2)] if dtype == FP8 else [None, None]
    caches = []
    for s in scales:
        x = torch.randn((pages, page, heads, dim), generator=g).cuda()
        if s is not None:
            x = (x / s[:, None]).clamp(-448, 448)
        x = torch.where(filled.cuda()[:, :, None, None], x, torch.full_like(x, math.nan)).to(dtype)
        if heads_first:
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        caches.append(x)
    return caches[0], caches[1], table.cuda(), scales[0], scales[1]


def check_attention(lens, q_heads, heads, dim, page, dtype, window=0, heads_first=False, seed=0, q_scale=2.0, **kw):
    from d3moe import attention
    k, v, table, ks, vs = make_cache(lens, heads, dim, page, dtype, seed, heads_first)
    qt = BF16 if dtype == FP8 else dtype
    q = (torch.randn((len(lens), q_heads, dim), generator=torch.Generator().manual_seed(seed + 1)) * q_scale).to(qt).cuda()
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = attention.paged_attention(q, k, v, table, ln, k_scale=ks, v_scale=vs, window=window, return_lse=True, status=status, **kw)
    want, wlse, bo, bl = R.attention(q, k, v, table, ln, dim ** -0.5, window, ks, vs)
    assert int(status) == 0
    assert torch.equal(torch.isinf(lse), torch.isinf(wlse))
    live = ~torch.isinf(wlse)
    assert ((lse.double() - wlse).abs()[live] <= bl[live]).all(), float((lse.double() - wlse).abs()[live].max())
    excess = (out.double() - want).abs() - bo
    assert (excess <= 0).all(), f"{float(excess.max())} above the bound"
    assert not torch.isnan(out).any()
    return out


LENS = [1, 0, 15, 16, 17, 63, 64, 65, 130, 301]


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,heads", [(16, 2), (4, 4), (6, 2), (24, 2), (5, 1)])
def test_attention(dtype, dim, q_heads, heads):
    check_attention(LENS, q_heads, heads, dim, 16, dtype, seed=dim + q_heads)


@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 128])
@pytest.mark.parametrize("heads_first", [False, True])
def test_page_sizes_and_layouts(page, heads_first):
    for dtype in (BF16, FP8):
        check_attention(LENS, 8, 2, 128, page, dtype, heads_first=heads_first, seed=page)


@pytest.mark.parametrize("window", [1, 16, 50, 64, 1000])
def test_window(window):
    check_attention(LENS, 16, 2, 256, 16, BF16, window=window)
    check_attention([5000, 4097, 1], 8, 1, 64, 32, F16, window=window)


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
def test_long_few_sequences(dtype):
    check_attention([70001], 16, 2, 256, 16, dtype)
    check_attention([33000, 1, 0, 9000], 8, 8, 64, 64, dtype)


@pytest.mark.parametrize("B", [1, 7, 300, 1500])
def test_many_sequences(B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 90, (B,), generator=g).tolist()
    check_attention(lens, 4, 1, 64, 16, BF16)


def test_all_empty():
    from d3moe import attention
    out = check_attention([0, 0, 0], 16, 2, 256, 16, BF16)
    assert (out == 0).all()
    k, v, table, _, _ = make_cache([4], 2, 64, 16, BF16)
    q = torch.empty((0, 4, 64), dtype=BF16, device="cuda")
    assert attention.paged_attention(q, k, v, table[:0], torch.empty(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


def test_large_logits_and_infinite_keys():
    check_attention(LENS, 8, 1, 128, 16, BF16, q_scale=300.0)
    # a key that is -inf along a positive query gives a logit of -inf: it takes no part
    from d3moe import attention
    k, v, table, _, _ = make_cache([40], 1, 64, 16, BF16)
    q = torch.rand((1, 1, 64), device="cuda").to(BF16) + 0.5
    k[table[0, 1].long(), 3] = -math.inf
    got, lse = attention.paged_attention(q, k, v, table, torch.tensor([40], dtype=torch.int32, device="cuda"), return_lse=True)
    rows = [R.gather_rows(c, table, 0, 0, 40, 0) for c in (k, v)]
    keep = torch.arange(40, device="cuda") != 19
    x = q[0].double() @ rows[0][keep].T / 8
    assert (got[0].double() - torch.softmax(x, -1) @ rows[1][keep]).abs().max() < 2 ** -6
    assert abs(float(lse) - float(torch.logsumexp(x, -1))) < 1e-4
    k[table[0, 1].long(), 3] = math.nan  # a NaN that is attended to is not hidden
    got = attention.paged_attention(q, k, v, table, torch.tensor([40], dtype=torch.int32, device="cuda"))
    assert torch.isnan(got).all()


def test_strided_operands_other_stream_and_determinism():
    from d3moe import attention
    lens = [301, 40, 2000]
    k, v, table, _, _ = make_cache(lens, 2, 128, 16, BF16)
    packed = torch.randn((3, 3 * 8 * 128), device="cuda").to(BF16)
    q = packed[:, 1024:2048].view(3, 8, 128)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((3, 2, 8, 128), 7.0, dtype=BF16, device="cuda")
    want = attention.paged_attention(q.contiguous(), k, v, table, ln)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ws = attention.paged_attention_workspace(3, 8, 2, 128, q.device)
        attention.paged_attention(q, k, v, table, ln, out=out[:, 1], workspace=ws, max_seq_len=2000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out[:, 1], want) and (out[:, 0] == 7).all()
    for _ in range(3):
        assert torch.equal(attention.paged_attention(q, k, v, table, ln), want)


def test_max_len_bounds_what_is_read():
    from d3moe import attention
    k, v, table, _, _ = make_cache([100], 2, 64, 16, F16)
    q = torch.randn((1, 4, 64), device="cuda").to(F16)
    long, short = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (100, 33))
    assert torch.equal(attention.paged_attention(q, k, v, table, long, max_seq_len=33),
                       attention.paged_attention(q, k, v, table, short, max_seq_len=33))
    neg = torch.tensor([-5], dtype=torch.int32, device="cuda")
    assert (attention.paged_attention(q, k, v, table, neg) == 0).all()


def test_bad_page_sets_status_and_stays_inside():
    from d3moe import _lib, attention
    k, v, table, _, _ = make_cache([64], 2, 64, 16, BF16)
    k.nan_to_num_()
    v.nan_to_num_()
    q = torch.randn((1, 4, 64), device="cuda").to(BF16)
    ln = torch.tensor([64], dtype=torch.int32, device="cuda")
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        t = table.clone()
        t[0, 2] = bad
        got = attention.paged_attention(q, k, v, t, ln, status=status)
        assert int(status) == _lib.D3_STATUS_BAD_ROW
        t[0, 2] = 0
        assert torch.equal(got, attention.paged_attention(q, k, v, t, ln))


def test_offsets_past_32_bits():
    """A cache of more than 2**32 bytes: pages at its far end are the ones read and written."""
    from d3moe import attention
    page, heads, dim = 64, 8, 256
    pages = (2 ** 32 + 2 ** 28) // (page * heads * dim)
    if torch.cuda.mem_get_info()[0] < 12 * 2 ** 30:
        pytest.skip("not enough free memory")
    cache = torch.zeros((pages, page, heads, dim), dtype=FP8, device="cuda")
    table = (pages - 1 - torch.arange(3)).int().view(1, 3).cuda()
    new = torch.randn((150, heads, dim), device="cuda").to(BF16)
    pos = torch.arange(150, dtype=torch.int32, device="cuda")
    seq = torch.zeros(150, dtype=torch.int32, device="cuda")
    attention.kv_append(new, new, cache, cache, table, pos, seq)
    tail = cache[pages - 3:].flip(0).reshape(-1, heads, dim)[:150]
    assert torch.equal(tail.view(torch.uint8), new.float().to(FP8).view(torch.uint8))
    q = torch.randn((1, 16, dim), device="cuda").to(BF16)
    ln = torch.tensor([150], dtype=torch.int32, device="cuda")
    got = attention.paged_attention(q, cache, cache, table, ln)
    small = cache[pages - 3:].clone()
    assert torch.equal(got, attention.paged_attention(q, small, small, 2 - torch.arange(3).int().view(1, 3).cuda(), ln))


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("heads,dim,page", [(2, 256, 16), (1, 64, 5), (8, 128, 64), (3, 80, 16)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append(dtype, heads, dim, page, heads_first):
    from d3moe import _lib, attention
    N, width, T = 4, 5, 37
    g = torch.Generator().manual_seed(dim)
    pages = N * width + 2
    table = torch.randperm(pages, generator=g)[:N * width].view(N, width).int().cuda()
    caches = [torch.randn((pages, page, heads, dim), generator=g).cuda().to(dtype) for _ in range(2)]
    if heads_first:
        caches = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in caches]
    src_t = BF16 if dtype == FP8 else dtype
    packed = (torch.randn((T, 2 * heads * dim + 8), generator=g) * 30).to(src_t).cuda()
    k, v = packed[:, :heads * dim].view(T, heads, dim), packed[:, heads * dim:2 * heads * dim].view(T, heads, dim)
    place = torch.randperm(N * width * page, generator=g)[:T]
    seq, pos = (place // (width * page)).int(), (place % (width * page)).int()
    seq[3], pos[4] = -1, -2
    scales = [torch.rand(heads, generator=g).cuda() + 0.05 for _ in range(2)] if dtype == FP8 else [None, None]
    want = [c.clone() for c in caches]
    for i in range(T):
        if i in (3, 4):
            continue
        for c, x, s in zip(want, (k, v), scales):
            row = x[i] if s is None else (x[i].float() / s[:, None]).clamp(-448, 448).to(FP8)
            c[int(table[seq[i], pos[i] // page]), int(pos[i]) % page] = row
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    args = (k, v, *caches, table)
    attention.kv_append(*args, pos.cuda(), seq.cuda(), k_scale=scales[0], v_scale=scales[1], status=status)
    for c, w in zip(caches, want):
        assert torch.equal(c.view(torch.uint8) if dtype == FP8 else c, w.view(torch.uint8) if dtype == FP8 else w)
    assert int(status) == 0
    # one token per sequence; past the table, and a page outside the cache: nothing is written
    bad = table.clone()
    bad[1, 0], bad[2, 0] = pages, -1
    far = torch.tensor([width * page, 0, 0, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    attention.kv_append(k[:N], v[:N], *caches, bad, far, k_scale=scales[0], v_scale=scales[1], status=status)
    assert int(status) == _lib.D3_STATUS_BAD_ROW
    for c, w in zip(caches, want):
        assert torch.equal(c.view(torch.uint8) if dtype == FP8 else c, w.view(torch.uint8) if dtype == FP8 else w)


@pytest.mark.parametrize("shape,page_dim,dtype", [
    ((6, 40, 16, 2, 256), 1, BF16), ((3, 2, 21, 5, 64), 2, F16), ((9, 2, 128, 128), 0, torch.float32),
    ((2, 33, 7), 1, torch.uint8), ((2, 33, 7), 1, torch.bfloat16), ((12, 4099), 0, torch.float32), ((1, 5, 1), 1, torch.int64)])
def test_copy_pages(shape, page_dim, dtype):
    from d3moe import _lib, cache
    g = torch.Generator().manual_seed(shape[page_dim])
    pool = torch.randint(0, 100, shape, generator=g).to(dtype).cuda()
    n = shape[page_dim] // 2
    order = torch.randperm(shape[page_dim], generator=g)
    src, dst = order[:n].int(), order[n:2 * n].int()
    want = pool.clone().movedim(page_dim, 0)
    want[dst.long().cuda()] = want[src.long().cuda()]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    # pairs that are left out: negative ones quietly, others with a status
    src2, dst2 = (torch.cat([x, torch.tensor([-1, 0], dtype=torch.int32)]).cuda() for x in (src, dst))
    dst2[-1] = -7
    cache.copy_pages(pool, src2, dst2, page_dim, status=status)
    assert torch.equal(pool.movedim(page_dim, 0), want) and int(status) == 0
    cache.copy_pages(pool, torch.tensor([shape[page_dim]], dtype=torch.int32, device="cuda"),
                     torch.zeros(1, dtype=torch.int32, device="cuda"), page_dim, status=status)
    assert torch.equal(pool.movedim(page_dim, 0), want) and int(status) == _lib.D3_STATUS_BAD_ROW
    cache.copy_pages(pool, src2[:0], dst2[:0], page_dim)


def test_copy_pages_of_a_view_and_one_source_to_many():
    from d3moe import cache
    whole = torch.arange(4 * 10 * 96, device="cuda", dtype=torch.float32).view(4, 10, 96)
    pool = whole[:, 1:9, 16:80]  # pages are parts of wider rows
    want = whole.clone()
    want[:, 1:9, 16:80][:, torch.tensor([5, 6, 7])] = want[:, 1:9, 16:80][:, torch.tensor([2, 2, 2])]
    cache.copy_pages(pool, torch.tensor([2, 2, 2], dtype=torch.int32, device="cuda"), torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda"), 1)
    assert torch.equal(whole, want)


def test_refusals():
    from d3moe import attention, cache
    k, v, table, _, _ = make_cache([20, 20], 2, 64, 16, BF16)
    q = torch.randn((2, 4, 64), device="cuda").to(BF16)
    ln = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    one = torch.ones(2, device="cuda")
    ok = dict(q=q, k_cache=k, v_cache=v, page_table=table, seq_lens=ln)
    for change, match in [
        (dict(q=q.half()), "q must be"), (dict(q=q[:, :, :32]), "q must be"), (dict(q=q[:, :3]), "multiple of key heads"),
        (dict(q=q[:1]), "one row per query"), (dict(seq_lens=ln.long()), "seq_lens"), (dict(page_table=table.long()), "page_table"),
        (dict(v_cache=v.half()), "k_cache and v_cache"), (dict(k_cache=k[:1]), "of one shape"), (dict(window=-1), "negative"),
        (dict(k_scale=one), "only an e4m3"), (dict(out=q.float()), "out must"), (dict(q=q.cpu()), "q must be"),
        (dict(k_cache=k.cpu(), v_cache=v.cpu()), "CUDA tensors"), (dict(k_cache=k[..., :40], v_cache=v[..., :40], q=q[..., :40]), "64, 128 or 256"),
        (dict(k_cache=k.transpose(2, 3), v_cache=v.transpose(2, 3)), "last axis"), (dict(seq_lens=ln[:1]), "seq_lens"),
    ]:
        with pytest.raises(ValueError, match=match):
            attention.paged_attention(**{**ok, **change})
    odd = torch.zeros(k.numel() + 4, dtype=BF16, device="cuda")[4:].view(k.shape)
    with pytest.raises(ValueError, match="16-byte aligned"):
        attention.paged_attention(**{**ok, "k_cache": odd})
    new = torch.zeros((2, 2, 64), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="k and v must be"):
        attention.kv_append(new.half(), new.half(), k, v, table, ln)
    with pytest.raises(ValueError, match="k and v must be"):
        attention.kv_append(new[:, :1], new[:, :1], k, v, table, ln)
    with pytest.raises(ValueError, match="positions"):
        attention.kv_append(new, new, k, v, table, ln[:1])
    with pytest.raises(ValueError, match="behind page_dim"):
        cache.copy_pages(k.transpose(1, 2), ln, ln, 0)
    with pytest.raises(ValueError, match="page_dim must"):
        cache.copy_pages(k, ln, ln, 4)
    with pytest.raises(ValueError, match="step evenly"):
        cache.copy_pages(torch.zeros((4, 3, 6, 8), device="cuda")[:, :2], ln, ln, 2)
    with pytest.raises(ValueError, match="dst"):
        cache.copy_pages(k, ln, ln.long(), 0)
