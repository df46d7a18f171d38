"""qkv_append: head norms at the ends of f32."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_kv4 import _norm, _rope64, dev

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
