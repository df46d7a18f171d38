"""kv4_attention's split kernel where a warp works off a run of several tiles and units (records and the combine kernel), at
batches past one and two blocks of 32 sequences. Every shape states the plan it needs: more places (two per unit and one per
tile) than warps, several times over, so that a retuned plan cannot empty these cases."""
from __future__ import annotations

import numpy as np
import pytest

from tests import _kv4
from tests.test_gpu_kv4 import DT, F32_TOL, check, dev

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SMS, UNIT_PLACES = 148, 2


def plan(S, T, H, Hkv, d, lens, max_ctx):
    """(units, places of the call's contexts, chunks) as the split kernel's host side lays them out."""
    rows = T * (H // Hkv)
    nt = 1 if rows <= 4 else 2 if rows <= 8 else 4
    fold = (4 if d == 64 else 2) if rows == 1 else 2 if rows == 2 else 1
    groups = -(-rows // (4 * nt // fold))
    warps = {1: 16, 2: 12, 4: 8}[nt]
    tk = 4096 // d
    units = S * Hkv * groups
    chunks = min(units * (UNIT_PLACES + max(1, -(-max_ctx // tk))), SMS * warps)
    places = Hkv * groups * sum(UNIT_PLACES + max(1, -(-n // tk)) for n in lens)
    return units, places, chunks


def aliased(x, S, Hkv, rows):
    """[slabs, rows, w] as S x Hkv heads, head h of sequence s on slab s + h."""
    return x.as_strided((S, Hkv, rows, x.shape[2]), (rows * x.shape[2], rows * x.shape[2], x.shape[2], 1))


# S, T, H, Hkv, d, longest context, rows of a pool block (0: contiguous)
RUNS = [
    (70, 1, 32, 32, 64, 700, 0),     # four folds
    (130, 1, 32, 32, 64, 333, 16),
    (40, 1, 32, 32, 128, 700, 0),    # two folds
    (130, 1, 16, 16, 128, 500, 48),
    (130, 1, 16, 8, 64, 1100, 64),   # two query rows
    (70, 2, 16, 16, 64, 900, 0),
    (130, 1, 9, 3, 64, 3000, 64),    # four query rows
    (70, 1, 32, 8, 128, 900, 16),
    (512, 1, 9, 3, 64, 700, 0),
    (70, 2, 24, 8, 64, 1300, 48),     # eight
    (40, 3, 16, 8, 128, 1000, 0),
    (70, 5, 9, 3, 64, 1900, 64),     # sixteen, and a second group of query rows
    (40, 9, 24, 8, 64, 700, 0),
    (130, 3, 32, 4, 128, 300, 48),
]


def run(case, types, uniform=False):
    import alpaca_b200 as ab
    S, T, H, Hkv, d, longest, block_rows = case
    q_type, out_type = types.split()
    rng = np.random.default_rng(S + T + H + d)
    lens = [longest] * S if uniform else [0, 1, longest, T - 1, longest - 1] + [int(x) for x in rng.integers(0, longest + 1, S - 5)]
    units, places, chunks = plan(S, T, H, Hkv, d, lens, longest)
    assert units > SMS and places >= 3 * chunks, (units, places, chunks)
    q = rng.standard_normal((S, T, H, d)).astype(np.float32)
    if q_type == "f16":
        q = q.astype(np.float16).astype(np.float32)
    table = None
    if block_rows:  # a pool that the sequences share
        per, pool = -(-longest // block_rows), 97
        parts = _kv4.random_cache(rng, pool, Hkv, block_rows, d)
        table = rng.integers(0, pool, (S, per)).astype(np.int32)
        k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
        rows_of = lambda x, s: np.concatenate(x[table[s]], axis=1)  # noqa: E731
        cache = ab.Kv4Cache(*(dev(x) for x in parts))
    else:
        rows = -(-longest // 16) * 16
        parts = [x[:, 0] for x in _kv4.random_cache(rng, S + Hkv - 1, 1, rows, d)]
        k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
        rows_of = lambda x, s: x[s:s + Hkv]  # noqa: E731
        cache = ab.Kv4Cache(*(aliased(dev(x), S, Hkv, rows) for x in parts))
    out = torch.full((S, T, H, d), float("nan"), dtype=DT[out_type], device="cuda")
    where = dict(start_position=longest - T) if uniform else dict(ctx_lens=dev(np.array(lens, np.int32)), max_ctx_len=longest)
    ab.kv4_attention(dev(q).to(DT[q_type]), cache, out, block_table=dev(table) if block_rows else None, kind=ab.Kernel.DECODE_SPLIT, **where)
    ab.device_status()
    got = out.double().cpu().numpy()
    for s in range(S):
        check(got[s], _kv4.attention(q[s], rows_of(k, s), rows_of(v, s), lens[s]), F32_TOL, out_type)


@pytest.mark.parametrize("types", ["f32 f32", "f16 f16"])
@pytest.mark.parametrize("case", range(len(RUNS)))
def test_runs_of_tiles_and_units(cuda_lib, case, types):
    run(RUNS[case], types)


@pytest.mark.parametrize("case", [(40, 1, 32, 32, 64, 800, 0), (70, 1, 9, 3, 64, 3001, 16), (66, 5, 9, 3, 64, 1999, 0)])
def test_runs_at_one_position(cuda_lib, case):
    run(case, "f32 f32", uniform=True)
