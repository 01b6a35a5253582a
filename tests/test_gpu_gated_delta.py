"""The gated delta rule on the GPU against its 64-bit recurrence.

Bounds. out is rounded to bf16 once (rms at most 2**-8 / sqrt(3) of the result);
the packed form may also round the state, the new values and the in-chunk
weights to bf16 once where they only form an output: four such roundings give
at most 4.6e-3 of the norm. The state is kept to two bf16 terms or better,
2**-16 of its norm; a single token is plain fp32."""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import mixer_reference as R  # noqa: E402

OUT_TOL, STATE_TOL = 2 * 2.0 ** -8 / math.sqrt(3), 2.0 ** -16
STEP_OUT_TOL, STEP_STATE_TOL = 2.0 ** -8 / math.sqrt(3) * 1.1, 2.0 ** -20
SHAPES = [(2, 4, 128, 128), (3, 3, 64, 64), (1, 4, 64, 128), (2, 2, 128, 64)]


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def operands(T, Hk, Hv, dk, dv, seed=0, decay=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.nn.functional.silu(torch.randn((T, 2 * Hk * dk + Hv * dv + 8), generator=g) * 1.5).to(torch.bfloat16).cuda()
    a, b = Hk * dk, 2 * Hk * dk
    q, k, v = x[:, :a].view(T, Hk, dk), x[:, a:b].view(T, Hk, dk), x[:, b:b + Hv * dv].view(T, Hv, dv)
    ld = (-decay * torch.rand((T, Hv), generator=g) ** 3).cuda()
    beta = torch.sigmoid(torch.randn((T, Hv), generator=g)).cuda()
    return q, k, v, ld, beta


def pool(slots, Hv, dk, dv, seed=0):
    return torch.randn((slots, Hv, dk, dv), generator=torch.Generator().manual_seed(seed + 9)).cuda() * 0.3


def chunk(spans_lens, shape, seed=0, decay=1.0, fresh=None, slots=None, l2norm=True, scale=None, pad=0):
    from d3moe import gated_delta
    Hk, Hv, dk, dv = shape
    n = len(spans_lens)
    cu = [pad]
    for x in spans_lens:
        cu.append(cu[-1] + x)
    T = cu[-1] + pad
    q, k, v, g, beta = operands(T, Hk, Hv, dk, dv, seed, decay)
    if not l2norm:
        q, k = (q.float() * 0.1).to(torch.bfloat16), (k.float() * 0.05).to(torch.bfloat16)
    state = pool(n + 2, Hv, dk, dv, seed)
    before = state.clone()
    slots = list(range(n, 0, -1)) if slots is None else slots
    fr = None if fresh is None else torch.tensor(fresh, device="cuda")
    out = torch.full((T, Hv, dv), 5.0, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gated_delta.gated_delta_chunk(q, k, v, g, beta, state, torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                  torch.tensor(slots, dtype=torch.int32, device="cuda"), fresh=fr, l2norm=l2norm, scale=scale, out=out, status=status)
    want, ws = R.delta(q, k, v, g, beta, before, list(zip(cu[:-1], cu[1:])), slots, dk ** -0.5 if scale is None else scale, l2norm, 1e-6, fresh)
    assert (out[:pad] == 5).all() and (out[T - pad:] == 5).all()
    return out[pad:T - pad], want[pad:T - pad], state, ws, int(status)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", [[1], [63, 1, 65, 64, 128, 2, 0, 17], [300], [200, 0, 0, 129]])
def test_chunk(shape, lens):
    out, want, state, ws, status = chunk(lens, shape, seed=len(lens))
    assert status == 0
    assert R.rel_l2(out, want) <= OUT_TOL
    assert R.rel_l2(state, ws) <= STATE_TOL
    for i in range(state.shape[0]):  # each slot on its own, those that no sequence names unchanged
        assert R.rel_l2(state[i], ws[i]) <= STATE_TOL


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", [14, 26, 60, 100])
def test_chunk_batches(shape, n):
    """Numbers of sequences on both sides of where the split over the SMs changes."""
    out, want, state, ws, status = chunk([(37 * i + 11) % 150 for i in range(n)], shape, seed=n)
    assert status == 0
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL


@pytest.mark.parametrize("decay", [0.0, 0.01, 30.0])
def test_chunk_decays(decay):
    """No decay, slow decay, and one that leaves nothing of a state."""
    out, want, state, ws, _ = chunk([150, 70], (2, 4, 128, 128), seed=3, decay=decay)
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL


def test_chunk_long():
    out, want, state, ws, _ = chunk([2500, 700], (1, 2, 128, 128), seed=4, decay=0.05)
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL


def test_chunk_fresh_left_out_and_scale():
    fresh = [True, False, True, False]
    out, want, state, ws, status = chunk([70, 5, 0, 64], (2, 4, 128, 128), fresh=fresh, slots=[2, -1, 0, 4], scale=0.7)
    assert status == 0 and (out[70:75] == 0).all()
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL
    assert (state[0] == 0).all()  # a fresh sequence without tokens
    out, want, state, ws, status = chunk([70, 5], (2, 4, 64, 64), slots=[4, 1])
    from d3moe import _lib
    assert status == _lib.D3_STATUS_BAD_ROW and (out[:70] == 0).all()
    assert R.rel_l2(state, ws) <= STATE_TOL


def test_chunk_without_norm_and_rows_of_no_sequence():
    out, want, state, ws, _ = chunk([100, 33], (2, 4, 128, 128), l2norm=False, pad=3)
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL


def test_chunk_zero_rows_and_zero_beta():
    """Keys of zero (padding) and beta of zero leave only the decay."""
    from d3moe import gated_delta
    q, k, v, g, beta = operands(100, 2, 4, 128, 128)
    k[:] = 0
    state = pool(1, 4, 128, 128)
    before = state.clone()
    cu = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu)
    assert R.rel_l2(state[0], before[0].double() * torch.exp(g.double().sum(0))[:, None, None]) <= STATE_TOL
    q, k, v, g, beta = operands(100, 2, 4, 128, 128)
    state = before.clone()
    gated_delta.gated_delta_chunk(q, k, v, g, beta * 0, state, cu)
    assert R.rel_l2(state[0], before[0].double() * torch.exp(g.double().sum(0))[:, None, None]) <= STATE_TOL


def test_chunk_resets():
    """A log decay of -infinity (or far below what fp32 holds) forgets everything before its token."""
    from d3moe import gated_delta
    q, k, v, g, beta = operands(150, 2, 4, 128, 128, seed=8)
    g[[20, 63, 64, 100], 1:3] = -math.inf
    g[[5, 90], 0] = -1e4
    state = pool(1, 4, 128, 128)
    before = state.clone()
    out = gated_delta.gated_delta_chunk(q, k, v, g, beta, state, torch.tensor([0, 150], dtype=torch.int32, device="cuda"))
    want, ws = R.delta(q, k, v, g, beta, before, [(0, 150)], [0], 128 ** -0.5)
    assert R.rel_l2(out, want) <= OUT_TOL and R.rel_l2(state, ws) <= STATE_TOL
    a, b = before.clone(), before.clone()
    gated_delta.gated_delta_step(q[20:21], k[20:21], v[20:21], g[20:21], beta[20:21], a)
    _, b = R.delta(q[20:21], k[20:21], v[20:21], g[20:21], beta[20:21], b, [(0, 1)], [0], 128 ** -0.5)
    assert R.rel_l2(a, b) <= STEP_STATE_TOL


def test_chunk_many_sequences_and_determinism():
    lens = [(7 * i) % 90 for i in range(150)]
    a = chunk(lens, (1, 2, 64, 64), seed=5)
    assert R.rel_l2(a[0], a[1]) <= OUT_TOL and R.rel_l2(a[2], a[3]) <= STATE_TOL
    b = chunk(lens, (1, 2, 64, 64), seed=5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", [1, 5, 67])
@pytest.mark.parametrize("l2norm", [True, False])
def test_step(shape, n, l2norm):
    from d3moe import gated_delta
    Hk, Hv, dk, dv = shape
    q, k, v, g, beta = operands(n, Hk, Hv, dk, dv, seed=n)
    if not l2norm:
        k = (k.float() * 0.1).to(torch.bfloat16)
    state = pool(n + 3, Hv, dk, dv)
    before = state.clone()
    slots = torch.randperm(n + 3, generator=torch.Generator().manual_seed(n))[:n].int()
    out = gated_delta.gated_delta_step(q, k, v, g, beta, state, slots.cuda(), l2norm=l2norm)
    want, ws = R.delta(q, k, v, g, beta, before, [(i, i + 1) for i in range(n)], slots.tolist(), dk ** -0.5, l2norm)
    assert R.rel_l2(out, want) <= STEP_OUT_TOL
    assert R.rel_l2(state, ws) <= STEP_STATE_TOL
    rest = torch.ones(n + 3, dtype=torch.bool)
    rest[slots.long()] = False
    assert torch.equal(state[rest.cuda()], before[rest.cuda()])


def test_step_slots_and_strides():
    from d3moe import _lib, gated_delta
    q, k, v, g, beta = operands(4, 2, 4, 128, 128)
    wide = pool(6, 4, 128, 256)
    state = torch.zeros((6, 4 * 128 * 128 + 64), device="cuda")[:, :4 * 128 * 128].view(6, 4, 128, 128)
    state.copy_(wide[..., :128])
    before = state.clone()
    slots = torch.tensor([5, -1, 6, 0], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    gates = torch.zeros((4, 24), device="cuda")
    gates[:, 2:6], gates[:, 13:17] = g, beta
    out = gated_delta.gated_delta_step(q, k, v, gates[:, 2:6], gates[:, 13:17], state, slots, status=status)
    want, ws = R.delta(q, k, v, g, beta, before, [(i, i + 1) for i in range(4)], slots.tolist(), 128 ** -0.5)
    assert int(status) == _lib.D3_STATUS_BAD_ROW and (out[1:3] == 0).all()
    assert R.rel_l2(out, want) <= STEP_OUT_TOL and R.rel_l2(state, ws) <= STEP_STATE_TOL
    empty = gated_delta.gated_delta_step(q[:0], k[:0], v[:0], g[:0], beta[:0], state, slots[:0])
    assert empty.shape == (0, 4, 128)


def test_steps_equal_a_chunk_and_run_on_another_stream():
    from d3moe import gated_delta
    q, k, v, g, beta = operands(20, 2, 4, 128, 128)
    a, b = pool(1, 4, 128, 128), pool(1, 4, 128, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = gated_delta.gated_delta_chunk(q, k, v, g, beta, a, torch.tensor([0, 20], dtype=torch.int32, device="cuda"))
    torch.cuda.current_stream().wait_stream(side)
    s = torch.cat([gated_delta.gated_delta_step(*(x[t:t + 1] for x in (q, k, v, g, beta)), b) for t in range(20)])
    assert R.rel_l2(o, s) <= OUT_TOL and R.rel_l2(a, b) <= STATE_TOL


def test_refusals():
    from d3moe import gated_delta
    q, k, v, g, beta = operands(3, 2, 4, 128, 128)
    state = pool(3, 4, 128, 128)
    ok = dict(q=q, k=k, v=v, g=g, beta=beta, state=state)
    for change, match in [
        (dict(q=q.half()), "bfloat16"), (dict(k=k[:, :1]), "shape of q"), (dict(g=g.half()), "float32"), (dict(beta=beta[:, :2]), "value_heads"),
        (dict(state=state[:, :, :64]), "state must be"), (dict(state=state.transpose(2, 3)), "contiguous"), (dict(state=state.cpu()), "CUDA tensors"),
        (dict(state=state[:2]), "fewer slots"), (dict(slots=torch.zeros(3, device="cuda")), "slots"), (dict(v=v.transpose(1, 2)), "value_heads|state must"),
        (dict(q=torch.zeros((3, 3, 128), dtype=torch.bfloat16, device="cuda"), k=torch.zeros((3, 3, 128), dtype=torch.bfloat16, device="cuda")), "multiple of key heads"),
    ]:
        with pytest.raises(ValueError, match=match):
            gated_delta.gated_delta_step(**{**ok, **change})
    small = operands(3, 2, 4, 32, 32)
    with pytest.raises(ValueError, match="64 or 128"):
        gated_delta.gated_delta_step(*small, pool(3, 4, 32, 32))
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu.long())
    with pytest.raises(ValueError, match="fresh"):
        gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu, fresh=torch.zeros(3, dtype=torch.bool, device="cuda"))
    from d3moe import _lib
    need = gated_delta.gated_delta_chunk_workspace(3, 2, 4, 128, 128, "cuda").numel()
    if need:
        with pytest.raises(_lib.D3Error, match="workspace"):
            gated_delta.gated_delta_chunk(q, k, v, g, beta, state, cu, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
