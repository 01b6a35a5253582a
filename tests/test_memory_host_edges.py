"""Host side of the sequence-memory operators at the edges of what they take, without a GPU."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")


def _refused(rc, text):
    from d3moe import _lib
    lib = _lib.load()
    assert rc == _lib.D3_EINVAL and text in lib.d3_last_error_string(), (rc, lib.d3_last_error_string())


def test_attention_refuses_negative_cache_strides():
    """Row offsets below zero mark places past a sequence's end, so no key may have one."""
    from d3moe import _lib
    lib = _lib.load()
    ok = dict(k=1 << 20, v=1 << 20, k_page_stride=8192, k_token_stride=512, k_head_stride=256, v_page_stride=8192, v_token_stride=512,
              v_head_stride=256, table=4096, table_stride=4, sequences=2, table_pages=4, num_pages=8, page_size=16, heads=2, dim=256,
              dtype=_lib.D3_DTYPE_BF16)
    for name in ("k_page_stride", "k_token_stride", "v_page_stride", "v_token_stride"):
        c = _lib.D3KvCache(**{**ok, name: -ok[name]})
        _refused(lib.d3_paged_attention(4096, 4096, 256, _lib.D3_DTYPE_BF16, 2, 16, ctypes.byref(c), 4096, 64, 0, 1.0, 4096, 4096, 256,
                                        None, 4096, 1 << 30, None, None), b"negative")


def test_delta_chunk_refuses_tokens_whose_counter_would_pass_32_bits():
    from d3moe import _lib
    lib = _lib.load()
    a = _lib.D3GatedDelta(q=4096, k=4096, v=4096, g=4096, beta=4096, out=4096, state=4096, slots=1, key_heads=1, value_heads=1, key_dim=64,
                          value_dim=64, l2norm=1, scale=1.0, eps=1e-6)
    _refused(lib.d3_gated_delta_chunk(ctypes.byref(a), 4096, 2**31 - 1, 1, None, 4096, 1 << 60, None, None), b"too many tokens")


@pytest.mark.parametrize("room,written", [(10, 0), (10, 3), (10, 4), (10, 7), (10, 8), (10, 10), (3, 0), (8, 8), (0, 0)])
def test_a_fork_shares_no_page_that_is_still_to_be_written(room, written):
    """A fork between extend and the writes: parent and child then write tokens of their own."""
    from test_memory_host import HostCache
    c = HostCache(2, 16, 4, 1, 2, max_sequences=4, max_len=16)

    def put(seq, t, x):
        c.pool[:, :, int(c.table[seq, t // 4]), t % 4] = x

    def held(seq):
        return [float(c.pool[0, 0, int(c.table[seq, t // 4]), t % 4, 0, 0]) for t in range(c.lens[seq])]

    a = c.new()
    c.extend(a, room)
    for t in range(written):
        put(a, t, 1 + t)
    b = c.fork(a, written)
    for t in range(written, room):
        put(a, t, 100 + t)
        put(b, t, 200 + t)
    for seq, base in ((a, 100), (b, 200)):
        for t in c.extend(seq, 2):
            put(seq, t, base + t)
        assert held(seq) == [1 + t for t in range(written)] + [base + t for t in range(written, room + 2)]
    shared = set(c._pages[a]) & set(c._pages[b])
    assert len(shared) == written // 4 and sum(n > 0 for n in c._holders) == 2 * -(-(room + 2) // 4) - len(shared)
    c.free(a)
    c.free(b)
    assert c.free_pages == 16


def test_fork_refuses_more_written_tokens_than_there_are():
    from test_memory_host import HostCache
    c = HostCache(1, 8, 4, 1, 2, max_sequences=2, max_len=16)
    a = c.new()
    c.extend(a, 5)
    for n in (6, -1):
        with pytest.raises(ValueError, match="cannot have been written"):
            c.fork(a, n)
    assert c.lens[1] is None and c.free_pages == 6


def test_the_package_imports_without_the_binding():
    """Only a call of a sequence-memory operator needs _d3native.so; the others reach libd3moe.so by ctypes."""
    import subprocess
    import sys

    from conftest import PKG_DIR
    code = """
from d3moe import _lib
def missing():
    raise ImportError("no binding here")
_lib.native = missing
import torch
from d3moe import attention, cache, gated_delta, torch_ops
torch.ops.d3moe.moe_layer, torch.ops.d3moe.paged_attention
t = torch.zeros(1)
for f, a in ((attention.kv_append, (t,) * 6), (attention.paged_attention, (t,) * 5), (cache.copy_pages, (t,) * 3),
             (gated_delta.gated_delta_step, (t,) * 6), (gated_delta.gated_delta_chunk, (t,) * 7)):
    try:
        f(*a)
    except ImportError as e:
        assert "no binding here" in str(e)
    else:
        raise AssertionError(f)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=PKG_DIR, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.fixture
def builder(tmp_path, monkeypatch):
    """build.py with its outputs in a folder of their own, and a record of what it would link."""
    import importlib.util

    from conftest import PKG_DIR
    spec = importlib.util.spec_from_file_location("d3moe_build_edges", PKG_DIR / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    for name in ("LIB", "SELFTEST_LIB", "NATIVE_LIB"):
        monkeypatch.setattr(b, name, tmp_path / getattr(b, name).name)
    monkeypatch.setattr(b, "OUT_DIR", tmp_path)
    monkeypatch.setattr(b, "HERE", tmp_path)
    b.linked = []

    def link(cc, srcs, out, objdir, verbose):
        b.linked.append(out.name)
        out.write_bytes(b"")

    def binding(out, verbose):
        b.linked.append(out.name)
        out.write_bytes(f"...{b.binding_mark(b.torch_version())}...".encode())

    monkeypatch.setattr(b, "_link", link)
    monkeypatch.setattr(b, "_link_binding", binding)
    monkeypatch.setattr(b, "nvcc", lambda: "nvcc")
    return b


def test_the_binding_is_rebuilt_for_another_torch(builder, monkeypatch):
    monkeypatch.setattr(builder, "torch_version", lambda: "2.0+x")
    builder.build()
    assert builder.linked == ["libd3moe.so", "libd3moe_selftest.so", "_d3native.so"] and not builder.needs_build()
    monkeypatch.setattr(builder, "torch_version", lambda: "2.0")
    assert builder.needs_build()
    builder.linked.clear()
    builder.build()
    assert builder.linked == ["_d3native.so"] and not builder.needs_build()


def test_without_torch_the_library_is_built_alone(builder, monkeypatch, capsys):
    monkeypatch.setattr(builder, "torch_version", lambda: None)
    builder.build()
    assert builder.linked == ["libd3moe.so", "libd3moe_selftest.so"] and not builder.needs_build()
    assert "binding" in capsys.readouterr().err
    monkeypatch.setattr(builder, "torch_version", lambda: "2.0")  # torch came later
    assert builder.needs_build()


def test_the_binding_in_the_tree_names_the_torch_it_is_for():
    import importlib.util

    from conftest import PKG_DIR
    from d3moe import _lib
    spec = importlib.util.spec_from_file_location("d3moe_build_mark", PKG_DIR / "build.py")
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    assert _lib.native().built_for == b.binding_mark(b.torch_version())
