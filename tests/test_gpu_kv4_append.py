"""qkv_append: head norms at the ends of f32, one token per sequence into f16 / f32 rows, every head_dim, RoPE bases below 1."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from tests import _kv4
from tests.test_gpu_kv4 import DT, _norm, _rope64, dev

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 96, 128])
@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_where_the_sum_of_squares_overflows(cuda_lib, d, interleaved):
    """x * (1 / sqrt(mean(x^2) + eps)) * w in f32: a sum of squares past f32 gives 1 / sqrt(inf) = 0, zeros and no NaN."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(d)
    q = rng.standard_normal((2, 5, 3, d)).astype(np.float32)
    q[0, 1, 2] *= np.float32(1e25)
    q[1, 4, 0] *= np.float32(1e20)
    q[1, 2, 1] *= np.float32(1e-30)  # and one whose squares vanish: eps alone is left
    w = (1 + 0.2 * rng.standard_normal(d)).astype(np.float32)
    out = torch.full(q.shape, float("nan"), device="cuda")
    ab.qkv_append(dev(q), None, None, out, None, theta=1e4, start_position=3, interleaved=interleaved, q_norm=dev(w))
    ab.device_status()
    got = out.double().cpu().numpy()
    want = np.stack([_rope64(_norm(q[s], w, 1e-5), 3 + np.arange(5), 1e4, interleaved) for s in range(2)])
    want[0, 1, 2] = want[1, 4, 0] = 0.0
    assert not got[0, 1, 2].any() and not got[1, 4, 0].any()
    # the norm's factors and the rotation's products: a handful of f32 roundings of values up to max|.|
    assert np.max(np.abs(got - want)) <= 8 * 2.0 ** -24 * np.max(np.abs(want)) + 1e-7


@pytest.mark.parametrize("d,H,Hkv", [(64, 9, 3), (128, 32, 8), (96, 4, 2)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("in_kind", ["f16", "f32"])
def test_one_token_with_norms_into_rows(cuda_lib, d, H, Hkv, interleaved, kind, in_kind):
    """A decode step of a model with q / k norms over the ordinary cache: every sequence at its own position; nothing but the
    new row is written."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(d + H)
    S, rows, eps, theta = 37, 48, 1e-6, 10000.0
    cast = (lambda x: x.astype(np.float16).astype(np.float32)) if in_kind == "f16" else (lambda x: x)
    q, k, v = (cast(rng.standard_normal((S, 1, h, d)).astype(np.float32) * 2) for h in (H, Hkv, Hkv))
    qn, kn = ((1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    pos = rng.integers(0, rows, S).astype(np.int32)
    pos[:2] = 0, rows - 1
    cache = tuple(torch.full((S, rows, Hkv, d), 7.0, dtype=DT[kind], device="cuda") for _ in range(2))
    out = torch.empty((S, 1, H, d), dtype=DT[kind], device="cuda")
    ab.qkv_append(dev(q).to(DT[in_kind]), dev(k).to(DT[in_kind]), dev(v).to(DT[in_kind]), out, cache, theta=theta, positions=dev(pos),
                  interleaved=interleaved, q_norm=dev(qn), k_norm=dev(kn), eps=eps)
    ab.device_status()
    kc, vc, qo = (x.double().cpu().numpy() for x in (*cache, out))
    for s in range(S):
        at = pos[s:s + 1]
        for got, x in ((qo[s], _rope64(_norm(q[s], qn, eps), at, theta, interleaved)), (kc[s, at], _rope64(_norm(k[s], kn, eps), at, theta, interleaved)),
                       (vc[s, at], v[s].astype(np.float64))):
            # f32: the norm's factors and the rotation's products; f16 rounds once more
            bound = 8 * 2.0 ** -24 * np.max(np.abs(x)) + 1e-7 + (np.abs(x) * 2.0 ** -11 if kind == "f16" else 0)
            assert np.all(np.abs(got - x) <= bound)
        other = np.arange(rows) != pos[s]
        assert (kc[s, other] == 7).all() and (vc[s, other] == 7).all()


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("theta", [1e4, 1.0, 0.01])
def test_every_head_dim_bitwise(cuda_lib, d, interleaved, theta):
    """Queries as the oracle rotates them and cache rows as the format defines them, bit for bit; a base below 1 turns faster
    with the channel, up to 2^33 radians here."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(d)
    for start in (0, 1_000_003, 1 << 30 if theta >= 1 else 1 << 27):
        T = 7 if start < 1 << 30 else 1
        start -= T if start else 0
        q = rng.standard_normal((1, T, 3, d)).astype(np.float32)
        out = torch.empty(q.shape, device="cuda")
        ab.qkv_append(dev(q), None, None, out, None, theta=theta, start_position=start, interleaved=interleaved)
        ab.device_status()
        assert np.array_equal(out[0].cpu().numpy(), oracle.rope(q[0], start, theta, interleaved))
    k, v = (rng.standard_normal((2, 7, 3, d)).astype(np.float32) for _ in range(2))
    cache = ab.kv4_cache(2, 32, 3, d)
    ab.qkv_append(None, dev(k), dev(v), None, cache, theta=theta, start_position=20, interleaved=interleaved)
    ab.device_status()
    for s in range(2):
        for i, x in ((0, oracle.rope(k[s], 20, theta, interleaved)), (2, v[s])):
            codes, scales = _kv4.quantise(np.swapaxes(x, 0, 1))
            assert np.array_equal(cache[i][s, :, 20:27].cpu().numpy(), codes)
            assert np.array_equal(cache[i + 1][s, :, 20:27].cpu().numpy(), scales)
