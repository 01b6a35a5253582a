"""Host side of the sequence-memory operators, without a GPU: argument checks of the
C ABI and of the Python functions, the registered operators on meta tensors, and
the page bookkeeping of PagedCache."""

from __future__ import annotations

import ctypes
import random

import pytest

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def test_c_abi_refuses_bad_arguments():
    from d3moe import _lib
    lib = _lib.load()
    n = ctypes.c_size_t()

    def refused(rc, text):
        assert rc == _lib.D3_EINVAL and text in lib.d3_last_error_string(), lib.d3_last_error_string()

    assert lib.d3_paged_attention_workspace_size(4, 16, 2, 256, ctypes.byref(n)) == 0 and n.value > 0
    refused(lib.d3_paged_attention_workspace_size(4, 16, 3, 256, ctypes.byref(n)), b"multiple of key heads")
    refused(lib.d3_paged_attention_workspace_size(4, 16, 2, 80, ctypes.byref(n)), b"64, 128 or 256")
    assert lib.d3_gated_delta_chunk_workspace_size(0, 0, 4, 128, 128, ctypes.byref(n)) == 0
    refused(lib.d3_gated_delta_chunk_workspace_size(10, 1, 4, 96, 128, ctypes.byref(n)), b"64 or 128")
    refused(lib.d3_gated_delta_chunk_workspace_size(-1, 1, 4, 128, 128, ctypes.byref(n)), b"negative")

    def cache(**kw):
        d = dict(k=4096, v=4096, k_page_stride=8192, k_token_stride=512, k_head_stride=256, v_page_stride=8192,
                 v_token_stride=512, v_head_stride=256, table=4096, table_stride=4, sequences=2, table_pages=4,
                 num_pages=8, page_size=16, heads=2, dim=256, dtype=_lib.D3_DTYPE_BF16)
        return ctypes.byref(_lib.D3KvCache(**{**d, **kw}))

    def append(c, dtype=_lib.D3_DTYPE_BF16, T=1, k=4096, stride=512):
        return lib.d3_kv_append(k, stride, 256, 4096, 512, 256, dtype, T, None, 4096, c, None, None)

    refused(append(None), b"NULL")
    refused(append(cache(dtype=_lib.D3_DTYPE_F32)), b"unsupported cache dtype")
    refused(append(cache(page_size=0)), b"geometry")
    refused(append(cache(v_head_stride=3)), b"16 bytes")
    refused(append(cache(k=4104)), b"16-byte aligned")
    refused(append(cache(k_scale=4096)), b"only an e4m3")
    refused(append(cache(), dtype=_lib.D3_DTYPE_F16), b"rows of dtype")
    refused(append(cache(), T=-1), b"negative")
    refused(append(cache(), k=None), b"NULL")
    refused(append(cache(), stride=513), b"16-byte aligned")
    assert append(cache(), T=0) == 0

    def attend(c, q_heads=16, lens=4096, max_len=64, window=0, ws=1 << 30, q=4096, dtype=_lib.D3_DTYPE_BF16, B=2):
        return lib.d3_paged_attention(q, 4096, 256, dtype, B, q_heads, c, lens, max_len, window, 1.0, 4096, 4096, 256,
                                      None, 4096, ws, None, None)

    refused(attend(cache(), q_heads=5), b"multiple of key heads")
    refused(attend(cache(), window=-1), b"negative")
    refused(attend(cache(), max_len=-1), b"negative")
    refused(attend(cache(), B=3), b"one row per query")
    refused(attend(cache(), q=None), b"NULL")
    refused(attend(cache(), q=4100), b"16-byte aligned")
    refused(attend(cache(num_pages=0)), b"empty cache")
    refused(attend(cache(), dtype=_lib.D3_DTYPE_F16), b"queries of dtype")
    assert attend(cache(), ws=16) == _lib.D3_EWORKSPACE
    assert attend(cache(sequences=0), B=0) == 0

    def copy(**kw):
        d = dict(pool=4096, planes=2, plane_stride=1 << 20, pages=8, page_stride=4096, page_bytes=4096, src=4096, dst=4096, n=1)
        return lib.d3_copy_pages(*{**d, **kw}.values(), None, None)

    refused(copy(n=-1), b"negative")
    refused(copy(page_stride=100), b"overlap")
    refused(copy(src=None), b"NULL")
    assert copy(n=0) == 0 and copy(planes=0) == 0 and copy(page_bytes=0) == 0

    def delta(n=1, **kw):
        d = dict(q=4096, k=4096, v=4096, g=4096, beta=4096, out=4096, state=4096, q_stride=256, k_stride=256, v_stride=512,
                 g_stride=4, beta_stride=4, out_stride=512, slot_stride=65536, slots=4, key_heads=2, value_heads=4,
                 key_dim=128, value_dim=128, l2norm=1, scale=1.0, eps=1e-6)
        return lib.d3_gated_delta_step(ctypes.byref(_lib.D3GatedDelta(**{**d, **kw})), n, None, None)

    refused(delta(key_dim=96), b"64 or 128")
    refused(delta(key_heads=3), b"multiple of key heads")
    refused(delta(n=5), b"5 sequences and 4 slots")
    refused(delta(q=4104), b"16-byte aligned")
    refused(delta(v_stride=513), b"16-byte aligned")
    refused(delta(state=4100), b"16-byte aligned")
    refused(delta(beta=None), b"NULL")
    assert delta(n=0) == 0


def test_c_abi_refuses_sizes_whose_counters_would_pass_32_bits():
    from d3moe import _lib
    lib = _lib.load()
    top = 2**31 - 1

    def refused(rc, text):
        assert rc == _lib.D3_EINVAL and text in lib.d3_last_error_string(), lib.d3_last_error_string()

    # pages of 2^20 tokens: a table of 2048 of them reaches 2^31
    c = _lib.D3KvCache(k=4096, v=4096, k_page_stride=0, k_token_stride=0, k_head_stride=64, v_page_stride=0, v_token_stride=0,
                       v_head_stride=64, table=4096, table_stride=2048, sequences=1, table_pages=2048, num_pages=1,
                       page_size=1 << 20, heads=1, dim=64, dtype=_lib.D3_DTYPE_BF16)
    refused(lib.d3_paged_attention(4096, 64, 64, _lib.D3_DTYPE_BF16, 1, 1, ctypes.byref(c), 4096, top, 0, 1.0, 4096, 64, 64,
                                   None, 4096, 1 << 30, None, None), b"too large for one call")
    refused(lib.d3_kv_append(4096, 64, 64, 4096, 64, 64, _lib.D3_DTYPE_BF16, top, None, 4096, ctypes.byref(c), None, None),
            b"too many tokens")
    refused(lib.d3_copy_pages(4096, 1, 0, 8, 4096, 4096, 4096, 4096, top, None, None), b"too many planes or pairs")
    refused(lib.d3_copy_pages(4096, top, 0, 8, 4096, 4096, 4096, 4096, 1, None, None), b"too many planes or pairs")


def test_python_functions_refuse_cpu_tensors_and_other_things():
    from d3moe import attention, cache, gated_delta
    c, i = torch.zeros((2, 16, 2, 64), dtype=BF16), torch.zeros((1, 2), dtype=torch.int32)
    q = torch.zeros((1, 4, 64), dtype=BF16)
    with pytest.raises(ValueError, match="CUDA tensors"):
        attention.paged_attention(q, c, c, i, i[0, :1])
    with pytest.raises(ValueError, match="CUDA tensors"):
        attention.kv_append(q[:, :2], q[:, :2], c, c, i, i[0, :1])
    with pytest.raises(ValueError, match="CUDA tensors"):
        cache.copy_pages(c, i[0], i[0])
    s = torch.zeros((1, 4, 64, 64))
    x, g = torch.zeros((1, 4, 64), dtype=BF16), torch.zeros((1, 4))
    with pytest.raises(ValueError, match="CUDA tensors"):
        gated_delta.gated_delta_step(x, x, x, g, g, s)
    with pytest.raises(ValueError, match="CUDA tensors"):
        gated_delta.gated_delta_chunk(x, x, x, g, g, s, i[0])
    with pytest.raises(ValueError, match="must be a tensor"):
        attention.paged_attention(None, c, c, i, i)
    with pytest.raises(ValueError, match="must be a tensor"):
        cache.copy_pages([1], i, i)


def test_registered_operators_on_meta_tensors():
    from d3moe import torch_ops  # noqa: F401

    def meta(shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device="meta")

    q, c = meta((3, 16, 256), BF16), meta((9, 16, 2, 256), BF16)
    t, i = meta((3, 4), torch.int32), meta((3,), torch.int32)
    out, lse = torch.ops.d3moe.paged_attention(q, c, c, t, i)
    assert (out.shape, out.dtype, lse.shape, lse.dtype) == ((3, 16, 256), BF16, (3, 16), torch.float32)
    torch.ops.d3moe.kv_append(meta((3, 2, 256), BF16), meta((3, 2, 256), BF16), c, meta((9, 16, 2, 256), BF16), t, i)
    torch.ops.d3moe.copy_pages(c, i, i, 0)
    k, v, g, s = meta((5, 2, 128), BF16), meta((5, 4, 128), BF16), meta((5, 4)), meta((5, 4, 128, 128))
    assert torch.ops.d3moe.gated_delta_step(k, k, v, g, g, s).shape == (5, 4, 128)
    assert torch.ops.d3moe.gated_delta_chunk(k, k, v, g, g, s, i).dtype == BF16
    for name, args in (("kv_append", ("k_cache", "v_cache")), ("copy_pages", ("pool",)), ("gated_delta_step", ("state",)),
                       ("gated_delta_chunk", ("state",))):
        schema = getattr(torch.ops.d3moe, name).default._schema
        assert tuple(a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write) == args


class HostCache:
    """PagedCache on the CPU, its copies done by indexing."""

    def __new__(cls, *a, **kw):
        from d3moe.cache import PagedCache

        class _Cache(PagedCache):
            def _copy(self, src, dst):
                assert len(src) == len(dst) and not set(src) & set(dst) and len(set(dst)) == len(dst)
                self.pool[:, :, dst] = self.pool[:, :, src]

        return _Cache(*a, device="cpu", **kw)


def _consistent(c, told):
    """Every sequence's table row leads to the values it was told; page counts agree."""
    held = [0] * c.pool.shape[2]
    for seq, values in told.items():
        pages = c.table[seq].tolist()
        assert c.lens[seq] == len(values)
        for t, x in enumerate(values):
            assert (c.pool[:, :, pages[t // c.page_size], t % c.page_size] == x).all()
        for p in pages[:-(-len(values) // c.page_size)]:
            held[p] += 1
    assert held == c._holders and c.free_pages == held.count(0)


def test_paged_cache_grows_forks_frees_and_compacts():
    rng = random.Random(3)
    c = HostCache(2, 60, 4, 1, 2, max_sequences=12, max_len=40)
    told, next_value = {}, 0
    for step in range(600):
        what = rng.random()
        if what < 0.2 and len(told) < 12:
            told[c.new()] = []
        elif what < 0.6 and told:
            seq = rng.choice(list(told))
            n = rng.randint(0, 5)
            try:
                places = c.extend(seq, n)
            except (RuntimeError, ValueError):
                continue
            for t in places:
                next_value += 1
                c.pool[:, :, int(c.table[seq, t // 4]), t % 4] = next_value
                told[seq].append(next_value)
        elif what < 0.75 and told:
            seq = rng.choice(list(told))
            try:
                child = c.fork(seq)
            except RuntimeError:
                continue
            told[child] = list(told[seq])
        elif what < 0.9 and told:
            seq = rng.choice(list(told))
            c.free(seq)
            del told[seq]
        else:
            c.compact()
            assert all(n == 0 for n in c._holders[len([n for n in c._holders if n]):])
        _consistent(c, told)


def test_paged_cache_refuses():
    c = HostCache(1, 3, 4, 1, 2, max_sequences=2, max_len=16)
    a = c.new()
    with pytest.raises(ValueError, match="at most"):
        c.extend(a, 17)
    with pytest.raises(ValueError, match="negative"):
        c.extend(a, -1)
    c.extend(a, 9)
    with pytest.raises(RuntimeError, match="free pages"):
        c.fork(a)  # the part-filled page has nowhere to go
    assert c.lens[1] is None and c.free_pages == 0
    b = c.new()
    with pytest.raises(RuntimeError, match="free pages"):
        c.extend(b, 1)
    assert c.lens[b] == 0
    with pytest.raises(RuntimeError, match="in use"):
        c.new()
    with pytest.raises(ValueError, match="no sequence"):
        c.free(7)
    c.free(a)
    with pytest.raises(ValueError, match="no sequence"):
        c.extend(a, 1)
    assert c.free_pages == 3 and c.compact() == 0
