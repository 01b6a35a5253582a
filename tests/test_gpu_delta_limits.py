"""The chunked gated delta rule at its limits, against the 64-bit recurrence: many strong
decays in a chunk, and values that are not finite. Bounds as in test_gpu_gated_delta."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402
from test_gpu_gated_delta import OUT_TOL, STATE_TOL, operands, pool  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _run(q, k, v, g, beta, lens):
    """(out, state) of the kernel and of the recurrence."""
    from d3moe import gated_delta
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    n, (Hv, dv), dk = len(lens), v.shape[1:], q.shape[2]
    state = pool(n, Hv, dk, dv, 4)
    want, ws = R.delta(q, k, v, g, beta, state, list(zip(cu[:-1], cu[1:])), list(range(n)), dk ** -0.5)
    out = gated_delta.gated_delta_chunk(q, k, v, g, beta, state, torch.tensor(cu, dtype=torch.int32, device="cuda"))
    return out, want, state, ws


def _close(out, want, state, ws):
    for h in range(out.shape[1]):
        assert R.rel_l2(out[:, h], want[:, h]) <= OUT_TOL
        for i in range(state.shape[0]):
            assert R.rel_l2(state[i, h], ws[i, h]) <= STATE_TOL, (i, h, R.rel_l2(state[i, h], ws[i, h]))


@pytest.mark.parametrize("strong", [-40.0, -100.0, -1e4, -math.inf])
@pytest.mark.parametrize("shape", [(2, 4, 128, 128), (1, 4, 64, 128)])
def test_many_strong_decays_leave_the_mild_ones_behind_them_exact(shape, strong):
    lens = [64, 128, 101, 64 + 40]
    q, k, v, g, beta = operands(sum(lens), *shape, seed=11, decay=0.05)
    g[0:48] = strong                      # 48 in a row, then 16 mild ones to the end
    g[64 + 64:64 + 64 + 40:2] = strong    # every other one of the second chunk's first 40
    mild = torch.rand(101, generator=torch.Generator().manual_seed(3)) < 0.5
    g[192:293][mild.cuda()] = strong      # half of them anywhere, others in the next head
    g[192:293, 1][~mild.cuda()] = strong
    g[293 + 64:293 + 64 + 20] = strong    # 20 in a short last chunk
    _close(*_run(q, k, v, g, beta, lens))


# sequences on both sides of where pairs of warps and their columns change
@pytest.mark.parametrize("others", [0, 11, 45])
@pytest.mark.parametrize("shape", [(2, 4, 128, 128), (3, 3, 64, 64), (2, 2, 128, 64)])
@pytest.mark.parametrize("what,value", [("v", math.nan), ("v", math.inf), ("k", math.nan), ("g", math.nan), ("beta", math.nan),
                                        ("q", math.nan), ("beta", math.inf)])
def test_what_is_not_finite_reaches_no_token_before_it(others, shape, what, value):
    lens = [150] + [70] * others
    T, Hk, Hv, dv = sum(lens), shape[0], shape[1], shape[3]
    for at in (13, 127) if others else (0, 13, 47, 63, 75, 127, 149):
        q, k, v, g, beta = operands(T, *shape, seed=at, decay=0.3)
        place = {"v": (at, Hv - 1, dv - 5), "q": (at, Hk - 1, 3), "k": (at, Hk - 1, 60), "g": (at, 0), "beta": (at, Hv - 1)}[what]
        dict(q=q, k=k, v=v, g=g, beta=beta)[what][place] = value
        out, want, state, ws = _run(q, k, v, g, beta, lens)
        good, kept = torch.isfinite(want), torch.isfinite(ws)
        assert torch.equal(torch.isfinite(out), good), f"token {at}: {int((torch.isfinite(out) != good).sum())} outputs differ"
        assert torch.equal(torch.isfinite(state), kept)
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        assert R.rel_l2(torch.where(good, out.double(), zero), torch.where(good, want, zero)) <= OUT_TOL
        assert R.rel_l2(torch.where(kept, state.double(), zero), torch.where(kept, ws, zero)) <= STATE_TOL


def test_a_state_that_is_not_finite_keeps_to_its_column():
    from d3moe import gated_delta
    q, k, v, g, beta = operands(100, 2, 4, 128, 128, seed=2)
    state = pool(1, 4, 128, 128)
    state[0, 2, 7, 33] = math.nan
    want, ws = R.delta(q, k, v, g, beta, state, [(0, 100)], [0], 128 ** -0.5)
    out = gated_delta.gated_delta_chunk(q, k, v, g, beta, state, torch.tensor([0, 100], dtype=torch.int32, device="cuda"))
    assert torch.equal(torch.isfinite(out), torch.isfinite(want)) and torch.equal(torch.isfinite(state), torch.isfinite(ws))
