"""kv4_attention's automatic choice against measured times (profiles/kv4_choice.csv): over calls that its estimates were not
fitted to, the kernel it names is on average within 2% of the better one and never 1.3 times as slow. Host only."""
from __future__ import annotations

import csv
from pathlib import Path

import pytest

DATA = Path(__file__).resolve().parent.parent / "profiles" / "kv4_choice.csv"
FAKE = 1 << 20  # a 16-byte aligned fake device address: validation never dereferences pointers


@pytest.fixture(scope="module")
def ab():
    from alpaca_b200 import build
    build.build()
    import alpaca_b200
    return alpaca_b200


def chosen(ab, seqs, tokens, heads, kv_heads, d, ctx):
    a, c = ab.Kv4AttnDesc(), ab.Kv4CacheDesc()
    c.rows = -(-ctx // 16) * 16
    c.k_codes = c.v_codes = c.k_scales = c.v_scales = FAKE
    c.code_head_stride, c.scale_head_stride = c.rows * d // 2, c.rows * d // 32
    c.code_unit_stride, c.scale_unit_stride = kv_heads * c.code_head_stride, kv_heads * c.scale_head_stride
    a.n_seqs, a.n_heads, a.n_kv_heads, a.head_dim, a.tokens, a.start_position = seqs, heads, kv_heads, d, tokens, ctx - tokens
    a.q_dtype = a.out_dtype = int(ab.DType.F16)
    a.q = a.out = FAKE
    a.q_token_stride = a.out_token_stride = heads * d
    a.q_seq_stride = a.out_seq_stride = tokens * heads * d
    a.cache = c
    return ab.kv4_select(a)


@pytest.mark.parametrize("which,calls,mean,worst", [("check", 200, 1.02, 1.3), ("fit", 200, 1.02, 1.3)])
def test_choice_is_near_the_better_kernel(ab, which, calls, mean, worst):
    ratios, kinds = [], set()
    for r in csv.DictReader(DATA.open()):
        if r["set"] != which:
            continue
        kind = chosen(ab, *(int(r[k]) for k in ("seqs", "tokens", "heads", "kv_heads", "head_dim", "context")))
        t = {ab.Kernel.DECODE_SPLIT: float(r["split_us"]), ab.Kernel.PREFILL_TC: float(r["prefill_us"])}
        kinds.add(kind)
        ratios.append(t[kind] / min(t.values()))
    print(f"{len(ratios)} calls, mean {sum(ratios) / len(ratios):.4f}, worst {max(ratios):.3f}")
    assert len(ratios) >= calls and len(kinds) == 2
    assert sum(ratios) / len(ratios) <= mean and max(ratios) <= worst
