"""The prompt form of kv4_attention: queries that f16 does not hold, and ragged prompts over a pool at head_dim 128."""
from __future__ import annotations

import numpy as np
import pytest

from tests import _kv4
from tests.test_gpu_kv4 import F32_TOL, TC_TOL, dev, paged, poison, to_gpu

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def rounding_of_queries(q, k, v, n):
    """How far one query head's output [d] may move when its f32 queries are rounded to f16 (relative 2^-11 each): scores move by
    at most D = max_j scale sum_i |q_i k_ji| 2^-11, the weights by factors in [e^-D, e^D], and since sum p (v - o) = 0 the output
    by at most (e^(2 D) - 1) sum_j p_j |v_j - o|."""
    k, v, q = k[:n], v[:n], q.astype(np.float64)
    scale = 1 / np.sqrt(len(q))
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    top = np.max(np.abs(k) @ np.abs(q)) * scale * 2.0 ** -11
    return np.expm1(2 * top) * (p @ np.abs(v - p @ v))


@pytest.mark.parametrize("T", [8, 96, 128, 300])
@pytest.mark.parametrize("d,H,Hkv", [(64, 9, 3), (128, 8, 2)])
def test_f32_queries(cuda_lib, T, d, H, Hkv):
    """DECODE_SPLIT keeps f32 accuracy at every token count; PREFILL_TC is within its bound and the rounding of the queries; AUTO
    is one of the two, bit for bit."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(T + d)
    ctx = 1000 + T
    parts = _kv4.random_cache(rng, 1, Hkv, -(-ctx // 16) * 16, d)
    q = rng.standard_normal((1, T, H, d)).astype(np.float32)
    k, v = _kv4.values(*parts[:2])[0], _kv4.values(*parts[2:])[0]
    outs = {}
    for kind in ("DECODE_SPLIT", "PREFILL_TC", "AUTO"):
        out = torch.full(q.shape, float("nan"), device="cuda")
        desc = ab.kv4_attention(dev(q), to_gpu(parts), out, start_position=ctx - T, kind=ab.Kernel[kind])
        ab.device_status()
        outs[kind] = out[0].cpu().numpy()
    assert np.array_equal(outs["AUTO"], outs[ab.kv4_select(desc).name])
    for t in sorted({0, 1, T // 2, T - 1}):
        n = ctx - T + 1 + t
        want = _kv4.attention(q[0, t:t + 1], k, v, n)[0]
        assert np.max(np.abs(outs["DECODE_SPLIT"][t] - want)) <= F32_TOL
        for h in range(H):
            room = TC_TOL + rounding_of_queries(q[0, t, h], k[h * Hkv // H], v[h * Hkv // H], n)
            assert np.all(np.abs(outs["PREFILL_TC"][t, h] - want[h]) <= room)


@pytest.mark.parametrize("d,H,Hkv", [(64, 9, 3), (128, 8, 2)])
@pytest.mark.parametrize("block_rows", [16, 48, 128])
def test_ragged_prompts_over_a_pool(cuda_lib, d, H, Hkv, block_rows):
    """Ragged prompts whose pool rows past the contexts, and whose workspace, hold NaN."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(d + block_rows)
    counts, starts = [1, 200, 0, 129, 70, 2], [0, 300, 5, 0, 257, 127]
    S, max_ctx = len(counts), 512
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rng.standard_normal((int(offs[-1]), H, d)).astype(np.float16).astype(np.float32)
    parts = _kv4.random_cache(rng, S, Hkv, max_ctx, d)
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    poison(parts, [a + b for a, b in zip(counts, starts)])
    pool, table = paged(parts, block_rows, rng)
    out = torch.full(q.shape, float("nan"), device="cuda")
    qd, od, sd, td, cache = dev(q).half(), dev(offs), dev(np.array(starts, np.int32)), dev(table), to_gpu(pool)
    desc = ab.make_kv4_varlen_desc(qd, cache, out, od, sd, max_tokens=200, max_ctx_len=max_ctx, block_table=td)
    ws = torch.full((ab.kv4_workspace_bytes(desc),), 0xFF, dtype=torch.uint8, device="cuda")
    assert ws.numel() >= 4 * S * max_ctx * Hkv * d  # the f16 rows
    ab.kv4_attention_launch(desc, ws)
    ab.device_status()
    got = out.double().cpu().numpy()
    for s in range(S):
        if counts[s]:
            want = _kv4.attention(q[offs[s]:offs[s + 1]], k[s], v[s], starts[s] + counts[s])
            assert np.max(np.abs(got[offs[s]:offs[s + 1]] - want)) <= TC_TOL
