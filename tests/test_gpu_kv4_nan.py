"""NaN value blocks of the 4-bit cache and the causal mask: a token's outputs are NaN in a block's channels exactly where it
sees a row whose block reads as NaN. The call's later tokens' rows are hidden from its earlier tokens, and hidden means not
read into the result at all: 0 x NaN is NaN."""
from __future__ import annotations

import numpy as np
import pytest

from tests import _kv4
from tests.test_gpu_kv4 import F32_TOL, dev, to_gpu

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SHAPES = [  # T, H, Hkv, d: one to four columns folds, 4, 8 and 16 query rows a unit, units of several tokens and of one
    (2, 3, 3, 64),
    (2, 9, 3, 64),
    (3, 4, 4, 128),
    (4, 8, 4, 64),
    (5, 6, 2, 128),
    (9, 9, 3, 64),
    (7, 16, 2, 64),
    (2, 32, 2, 128),
]


def compare(got, want):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want).any() and not np.isnan(want).all()
    assert np.nanmax(np.abs(got - want)) <= F32_TOL


def make(rng, S, T, Hkv, d, rows, lens):
    """A cache whose own rows (the call's tokens') hold NaN blocks in V: the last token's, a middle one's, one block each."""
    parts = _kv4.random_cache(rng, S, Hkv, rows, d)
    scales = parts[3].view(np.uint16)
    nb = d // 32
    for s, L in enumerate(lens):
        for i, row in enumerate((L - 1, L - 1 - (T - 1) // 2)):
            if row >= 0:
                scales[s, (s + i) % Hkv, row, (s + 2 * i) % nb] = 0x7E00
        parts[2][s, :, max(L - 1, 0)] |= 1  # codes of any value
    return parts


@pytest.mark.parametrize("kind", ["DECODE_SPLIT", "GENERAL"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_hidden_nan_rows_reach_no_token(cuda_lib, shape, kind):
    import alpaca_b200 as ab
    T, H, Hkv, d = SHAPES[shape]
    rng = np.random.default_rng(100 + shape)
    lens = [T, 64 + T // 2, 65, 203, 130 + T, 33]  # the own rows inside a tile, over its end, and the whole context
    S, rows = len(lens), 224
    parts = make(rng, S, T, Hkv, d, rows, lens)
    q = rng.standard_normal((S, T, H, d)).astype(np.float32)
    out = torch.zeros((S, T, H, d), dtype=torch.float32, device="cuda")
    ab.kv4_attention(dev(q), to_gpu(parts), out, ctx_lens=dev(np.array(lens, np.int32)), max_ctx_len=max(lens), kind=ab.Kernel[kind])
    ab.device_status()
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    compare(out, np.stack([_kv4.attention(q[s], k[s], v[s], n) for s, n in enumerate(lens)]))


@pytest.mark.parametrize("T,H,Hkv,d", [(2, 8, 8, 64), (3, 8, 8, 128), (5, 24, 8, 64), (4, 16, 8, 128)])
def test_hidden_nan_rows_many_units(cuda_lib, T, H, Hkv, d):
    """More units than SMs: runs of tiles and records instead of one CTA per unit."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(T)
    S, rows = 24, 336
    lens = [int(x) for x in rng.integers(T, rows + 1, S)]
    parts = make(rng, S, T, Hkv, d, rows, lens)
    q = rng.standard_normal((S, T, H, d)).astype(np.float32)
    out = torch.zeros((S, T, H, d), dtype=torch.float32, device="cuda")
    ab.kv4_attention(dev(q), to_gpu(parts), out, ctx_lens=dev(np.array(lens, np.int32)), max_ctx_len=rows, kind=ab.Kernel.DECODE_SPLIT)
    ab.device_status()
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    compare(out, np.stack([_kv4.attention(q[s], k[s], v[s], n) for s, n in enumerate(lens)]))
