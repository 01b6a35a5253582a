"""Paged attention where logits or queries span a wide range, against the 64-bit form."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402
from test_gpu_attention import BF16, F16, FP8, make_cache  # noqa: E402


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _sink_case(lens, q_heads, heads, dim, page, dtype, gap, at):
    """One key per sequence lies `gap` above all others (which spread by a few tenths) and has a
    value of zero: the result is made of the small probabilities alone."""
    k, v, table, ks, vs = make_cache(lens, heads, dim, page, dtype, seed=int(gap) + dim)
    if dtype == FP8:
        ks, vs = torch.full_like(ks, 0.25), torch.ones_like(vs)
    unit = 1.0 if ks is None else 0.25
    q = torch.randn((len(lens), q_heads, dim), generator=torch.Generator().manual_seed(5)) * 0.3
    q[:, :, 0] = math.sqrt(dim)
    q = q.to(BF16 if dtype == FP8 else dtype).cuda()
    kf, vf = k.float().nan_to_num(0.0), v.float().nan_to_num(0.0)
    if dtype == FP8:
        kf, vf = kf.clamp(-2, 2) / unit * 0.5, vf.clamp(-2, 2)
    kf[..., 0] = 0
    vf = (vf.abs() + 0.5) * (2.0 if dtype == FP8 else 1024.0)  # of one sign, and far from f16's smallest
    for b, n in enumerate(lens):
        if n == 0:
            continue
        t = min(n - 1, int(at * n))
        p = int(table[b, t // page])
        kf[p, t % page] = 0
        kf[p, t % page, :, 0] = gap / unit
        vf[p, t % page] = 0
    return q, kf.to(dtype), vf.to(dtype), table, ks, vs


@pytest.mark.parametrize("dtype", [BF16, F16, FP8])
@pytest.mark.parametrize("gap", [14.0, 16.0, 18.0])
@pytest.mark.parametrize("lens,q_heads,heads,dim,at", [
    ([250, 97, 1, 0], 8, 2, 128, 0.0),   # units taken whole
    ([700], 16, 2, 256, 0.5),            # a cluster per unit
    ([9000, 3000], 16, 1, 64, 0.0),      # the line of tiles, 16 heads per unit
    ([20000], 8, 1, 128, 0.9),
])
def test_small_probabilities_beside_a_large_one(dtype, gap, lens, q_heads, heads, dim, at):
    from d3moe import attention
    q, k, v, table, ks, vs = _sink_case(lens, q_heads, heads, dim, 16, dtype, gap, at)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got, lse = attention.paged_attention(q, k, v, table, ln, k_scale=ks, v_scale=vs, return_lse=True)
    want, wlse, bo, bl = R.attention(q, k, v, table, ln, dim ** -0.5, 0, ks, vs)
    excess = (got.double() - want).abs() - bo
    assert (excess <= 0).all(), f"{float(((got.double() - want).abs() / want.abs().clamp(min=1e-30)).max())} of the result"
    live = ~torch.isinf(wlse)
    assert ((lse.double() - wlse).abs()[live] <= bl[live]).all()


@pytest.mark.parametrize("power", [-120, -60, 60, 122])
def test_queries_of_any_power_of_two_over_an_e4m3_cache(power):
    """Queries times 2^p with a scale of 2^-p are the same operands: no bit changes."""
    from d3moe import attention
    k, v, table, _, _ = make_cache([90, 40], 2, 64, 16, FP8)
    q = torch.randn((2, 8, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    ln = torch.tensor([90, 40], dtype=torch.int32, device="cuda")
    q = torch.where(q.abs() < 2.0 ** -5, torch.zeros_like(q), q)  # the others stay normal numbers
    want = attention.paged_attention(q, k, v, table, ln, 2.0 ** -3)
    got = attention.paged_attention((q.float() * 2.0 ** power).to(BF16), k, v, table, ln, 2.0 ** (-3 - power))
    assert torch.isfinite(want).all() and torch.equal(got, want)
