"""The 4-bit KV cache on the GPU: rows written (head norms, RoPE, quantisation), read back, attended over.

Bounds. Reading back is exact. Written codes and scales equal the f32 definition bit for bit where no norm is applied (the
rotation is the library's bit-exact one); with a norm a value is within half a step of the f64 rows plus f32 rounding.
Attention: the split and general kernels keep f32 accuracy, 1e-5 max-abs on N(0, 1) rows (the bound of the f16 decode),
plus half an ulp where the output is f16; the tensor-core prefill rounds P to f16, 2e-3 max-abs (its bound)."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from tests import _kv4

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

F32_TOL, TC_TOL = 1e-5, 2e-3
DT = {"f16": torch.float16, "f32": torch.float32}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def to_gpu(parts):
    import alpaca_b200 as ab
    return ab.Kv4Cache(*(dev(x) for x in parts))


def paged(parts, block_rows, rng, extra=2):
    """Contiguous [S, H, rows, ..] parts as shuffled pool blocks and their table; spare blocks and rows hold NaN blocks."""
    S, H, rows = parts[0].shape[:3]
    per = -(-rows // block_rows)
    total = S * per + extra
    order = rng.permutation(total).astype(np.int32)
    table = order[: S * per].reshape(S, per)
    out = []
    for x in parts:
        pool = np.full((total, H, block_rows, x.shape[3]), 0x7E00 if x.dtype == np.int16 else 0xFF, x.dtype)
        for s in range(S):
            for b in range(per):
                rowsb = x[s, :, b * block_rows:(b + 1) * block_rows]
                pool[table[s, b], :, : rowsb.shape[1]] = rowsb
        out.append(pool)
    return out, table


def poison(parts, lens):
    """Rows past every sequence's context become NaN blocks with full codes."""
    for i, x in enumerate(parts):
        for s, n in enumerate(lens):
            x[s, :, n:] = 0x7E00 if x.dtype == np.int16 else 0xFF


def check(got, want, tol, out_type):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all()
    bound = tol + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if out_type == "f16" else 0)
    worst = np.max(np.abs(got - want) - bound)
    print(f"max-abs {np.max(np.abs(got - want)):.3e}")
    assert worst <= 0, worst


# ------------------------------------------------------------------------------------------------ read back

@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("block_rows", [0, 16, 48])
def test_read_is_exact(cuda_lib, d, block_rows):
    import alpaca_b200 as ab
    rng = np.random.default_rng(d + block_rows)
    S, H, rows = 3, 3, 80
    parts = _kv4.random_cache(rng, S, H, rows, d)
    parts[1].view(np.uint16)[0, 0, 5] = 0x0010 | 7   # the smallest step, 2^-20
    parts[1].view(np.uint16)[0, 1, 6] = 0x6C40 | 15  # the largest
    want = [np.swapaxes(_kv4.values(parts[i], parts[i + 1]), 1, 2) for i in (0, 2)]
    table = None
    if block_rows:
        parts, tb = paged(parts, block_rows, rng)
        table = dev(tb)
    cache = to_gpu(parts)
    starts = np.array([0, 7, 33], np.int32)
    for n, kw, first in [(rows, {}, [0, 0, 0]), (37, dict(start_row=11), [11] * 3), (29, dict(row_starts=dev(starts)), starts), (1, dict(start_row=79), [79] * 3)]:
        for kind in ("f16", "f32"):
            k, v = (torch.full((S, n, H, d), 7.0, dtype=DT[kind], device="cuda") for _ in range(2))
            ab.kv4_read(cache, k, v, block_table=table, **kw)
            ab.device_status()
            for got, w in ((k, want[0]), (v, want[1])):
                for s in range(S):
                    assert np.array_equal(got[s].double().cpu().numpy(), w[s, first[s]:first[s] + n])


def test_read_nan_block_and_strides(cuda_lib):
    import alpaca_b200 as ab
    rng = np.random.default_rng(4)
    parts = _kv4.random_cache(rng, 2, 4, 48, 64)
    parts[1].view(np.uint16)[1, 2, 9, 1] = 0x7E00
    big = to_gpu(parts)
    cache = ab.Kv4Cache(*(x[:, 1:3] for x in big))  # two heads of four
    buf = torch.zeros((2, 20, 3, 64), dtype=torch.float16, device="cuda")
    out = buf.as_strided((2, 20, 2, 64), (20 * 192, 192, 64, 1))
    out2 = torch.zeros_like(buf).as_strided((2, 20, 2, 64), (20 * 192, 192, 64, 1))
    ab.kv4_read(cache, out, out2)
    ab.device_status()
    want = np.swapaxes(_kv4.values(parts[0], parts[1])[:, 1:3, :20], 1, 2)
    assert np.array_equal(out.double().cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want).sum() == 32
    assert not buf[:, :, 2].any()  # between the rows nothing is written


def test_read_out_of_range_reads_zero_and_reports(cuda_lib):
    import alpaca_b200 as ab
    rng = np.random.default_rng(5)
    parts = _kv4.random_cache(rng, 2, 2, 32, 64)
    cache = to_gpu(parts)
    k, v = (torch.full((2, 8, 2, 64), 7.0, dtype=torch.float32, device="cuda") for _ in range(2))
    ab.kv4_read(cache, k, v, row_starts=dev(np.array([28, -3], np.int32)))
    with pytest.raises(ab.AlpacaCUDAError) as e:
        ab.device_status()
    assert e.value.status == ab.Status.INVALID_ARGUMENT
    want = np.swapaxes(_kv4.values(parts[0], parts[1]), 1, 2)
    assert np.array_equal(k[0, :4].double().cpu().numpy(), want[0, 28:])
    assert not k[0, 4:].any() and not k[1, :3].any()
    assert np.array_equal(k[1, 3:].double().cpu().numpy(), want[1, :5])


# ------------------------------------------------------------------------------------------------ append

@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_append_equals_definition_bitwise(cuda_lib, d, interleaved, kind):
    """No norms: queries as alpaca_rope_kv_append's, cache rows as the format's definition of the rotated rows."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(d)
    S, T, H, Hkv, start, theta = 2, 11, 3, 2, 21, 10000.0
    cast = (lambda x: x.astype(np.float16).astype(np.float32)) if kind == "f16" else (lambda x: x)
    q = cast(rng.standard_normal((S, T, H, d)).astype(np.float32))
    k, v = (cast(rng.standard_normal((S, T, Hkv, d)).astype(np.float32)) for _ in range(2))
    v[0, 1, 0, :32] = 0.0       # a block of zeros
    v[0, 2, 1, :32] = -3.0      # one-sided blocks
    v[0, 3, 1, :32] = 2.5
    v[1, 4, 0, 0] = 6e4         # a wide block
    v[1, 5, 0, 31] = np.nan
    v[1, 6, 1, 3] = np.inf
    v[1, 7, 1, :32] *= 1e-7 if kind == "f32" else 0.0
    cache = ab.kv4_cache(S, start + T, Hkv, d)
    out = torch.empty((S, T, H, d), dtype=torch.float32, device="cuda")
    ab.qkv_append(dev(q).to(DT[kind]), dev(k).to(DT[kind]), dev(v).to(DT[kind]), out, cache, theta=theta, start_position=start,
                  interleaved=interleaved)
    ab.device_status()
    for s in range(S):
        assert np.array_equal(out[s].cpu().numpy(), oracle.rope(q[s], start, theta, interleaved))
        kr = oracle.rope(k[s], start, theta, interleaved)
        for i, x in ((0, kr), (2, v[s])):
            codes, scales = _kv4.quantise(np.swapaxes(x, 0, 1))
            assert np.array_equal(cache[i][s, :, start:start + T].cpu().numpy(), codes)
            assert np.array_equal(cache[i + 1][s, :, start:start + T].cpu().numpy(), scales)
    assert not cache.k_codes[:, :, :start].any() and not cache.k_codes[:, :, start + T:].any()


def _norm(x, w, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def _rope64(x, pos, theta, interleaved):
    d = x.shape[-1]
    ang = np.asarray(pos, np.float64)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    out = np.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., : d // 2], x[..., d // 2:])
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, d // 2), slice(d // 2, None))
    out[..., lo], out[..., hi] = a * c - b * s, a * s + b * c
    return out


@pytest.mark.parametrize("d,H,Hkv", [(64, 9, 3), (128, 8, 2), (96, 2, 1), (32, 5, 5)])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("which", ["both", "q", "k"])
@pytest.mark.parametrize("cache_kind", ["kv4", "f16", "f32"])
def test_append_with_norms(cuda_lib, d, H, Hkv, interleaved, which, cache_kind):
    import alpaca_b200 as ab
    rng = np.random.default_rng(7)
    S, T, eps, theta = 3, 5, 1e-5, 500000.0
    pos = np.array([0, 4001, 12], np.int32)
    q, k, v = (rng.standard_normal((S, T, h, d)).astype(np.float32) * 3 for h in (H, Hkv, Hkv))
    qn, kn = ((1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2))
    rows = 4016
    cache = ab.kv4_cache(S, rows, Hkv, d) if cache_kind == "kv4" else \
        tuple(torch.zeros((S, rows, Hkv, d), dtype=DT[cache_kind], device="cuda") for _ in range(2))
    out = torch.empty((S, T, H, d), dtype=torch.float32, device="cuda")
    ab.qkv_append(dev(q), dev(k), dev(v), out, cache, theta=theta, positions=dev(pos), interleaved=interleaved, eps=eps,
                  q_norm=dev(qn) if which != "k" else None, k_norm=dev(kn) if which != "q" else None)
    ab.device_status()
    if cache_kind == "kv4":
        kv = [torch.empty((S, T, Hkv, d), dtype=torch.float32, device="cuda") for _ in range(2)]
        ab.kv4_read(cache, *kv, row_starts=dev(pos))
        ab.device_status()
    else:
        kv = [torch.stack([x[s, p:p + T] for s, p in enumerate(pos)]).float() for x in cache]
    for s in range(S):
        at = pos[s] + np.arange(T)
        qr = _rope64(_norm(q[s], qn, eps) if which != "k" else q[s].astype(np.float64), at, theta, interleaved)
        kr = _rope64(_norm(k[s], kn, eps) if which != "q" else k[s].astype(np.float64), at, theta, interleaved)
        # f32: the norm's factors and the rotation's products, a handful of roundings of values up to max|.|
        assert np.max(np.abs(out[s].cpu().numpy() - qr)) <= 8 * 2.0 ** -24 * np.max(np.abs(qr)) + 1e-7
        for x, got in ((kr, kv[0][s]), (v[s].astype(np.float64), kv[1][s])):
            got = got.double().cpu().numpy()
            slack = 8 * 2.0 ** -24 * np.max(np.abs(x)) + 1e-7
            if cache_kind == "kv4":
                y = x.reshape(*x.shape[:-1], -1, 32)
                span = np.maximum(y.max(-1), 0) - np.minimum(y.min(-1), 0)
                half = np.repeat(span / 15 * (1 + 2.0 ** -6) / 2, 32, -1)  # half a step, at most one ulp of 7 bits above the span
                assert np.all(np.abs(got - x) <= half + slack)
            else:
                assert np.all(np.abs(got - x) <= slack + (np.abs(x) * 2.0 ** -11 if cache_kind == "f16" else 0))


def test_append_in_place_strided_equals_rope(cuda_lib):
    """Without norms: queries in place and f16 rows equal alpaca_rope_kv_append, from a fused [q | k | v] projection."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(9)
    S, T, H, Hkv, d, start = 2, 13, 9, 3, 64, 5
    qkv = dev(rng.standard_normal((S, T, (H + 2 * Hkv) * d)).astype(np.float32))
    W = (H + 2 * Hkv) * d

    def view(buf, first, heads):
        return buf.as_strided((S, T, heads, d), (T * W, W, d, 1), first * d)
    ref = qkv.clone()
    caches = [torch.zeros((S, 32, Hkv, d), dtype=torch.float16, device="cuda") for _ in range(4)]
    ab.rope_kv_append(view(ref, 0, H), view(ref, H, Hkv), view(ref, H + Hkv, Hkv), caches[0], caches[1], theta=1e4, start_position=start)
    q = view(qkv, 0, H)
    ab.qkv_append(q, view(qkv, H, Hkv), view(qkv, H + Hkv, Hkv), q, (caches[2], caches[3]), theta=1e4, start_position=start)
    ab.device_status()
    assert torch.equal(qkv, ref)
    assert torch.equal(caches[2], caches[0]) and torch.equal(caches[3], caches[1])


@pytest.mark.parametrize("block_rows", [16, 80])
def test_append_paged_and_bad_positions(cuda_lib, block_rows):
    import alpaca_b200 as ab
    rng = np.random.default_rng(11)
    S, T, Hkv, d = 3, 20, 2, 64
    k, v = (rng.standard_normal((S, T, Hkv, d)).astype(np.float32) for _ in range(2))
    per = -(-96 // block_rows)
    pool = ab.kv4_cache(S * per, block_rows, Hkv, d)
    table = rng.permutation(S * per).astype(np.int32).reshape(S, per)
    pos = np.array([0, 70, 33], np.int32)
    ab.qkv_append(None, dev(k), dev(v), None, pool, theta=1e4, positions=dev(pos), block_table=dev(table))
    ab.device_status()
    got = [torch.empty((S, T, Hkv, d), dtype=torch.float32, device="cuda") for _ in range(2)]
    ab.kv4_read(pool, *got, row_starts=dev(pos), block_table=dev(table))
    ab.device_status()
    for s in range(S):
        want = _kv4.values(*_kv4.quantise(v[s]))
        assert np.array_equal(got[1][s].double().cpu().numpy(), want)
        assert np.array_equal(got[0][s].double().cpu().numpy(), _kv4.values(*_kv4.quantise(oracle.rope(k[s], int(pos[s]), 1e4, True))))
    before = [x.clone() for x in pool]
    ab.qkv_append(None, dev(k), dev(v), None, pool, theta=1e4, positions=dev(np.array([-20, 96 * block_rows, 1 << 30], np.int32)),
                  block_table=dev(table))
    with pytest.raises(ab.AlpacaCUDAError):
        ab.device_status()
    assert all(torch.equal(x, y) for x, y in zip(pool, before))


# ------------------------------------------------------------------------------------------------ attention

ATTN = [
    # S, T, H, Hkv, d, contexts, block_rows
    (4, 1, 9, 3, 64, [1, 17, 64, 65], 0),
    (4, 1, 9, 3, 64, [0, 255, 256, 257], 64),
    (2, 1, 32, 32, 64, [511, 700], 0),
    (3, 1, 16, 2, 64, [5, 300, 1030], 16),
    (2, 1, 5, 1, 64, [64, 999], 48),
    (3, 1, 8, 2, 128, [1, 129, 515], 0),
    (3, 1, 32, 8, 128, [0, 31, 640], 16),
    (2, 1, 16, 1, 128, [33, 400], 32),
    (3, 2, 9, 3, 64, [1, 2, 300], 0),
    (2, 3, 6, 6, 64, [0, 77], 64),
    (3, 7, 8, 4, 64, [3, 64, 520], 0),
    (2, 5, 8, 1, 128, [4, 200], 0),
    (2, 33, 4, 2, 64, [20, 150], 0),
    (1, 9, 6, 2, 128, [9], 0),
    # one and two query rows per KV head (folded columns), contexts past one tile a warp, paged
    (3, 1, 4, 4, 128, [1, 40, 700], 48),
    (3, 1, 4, 4, 64, [16, 65, 1300], 16),
    (3, 2, 3, 3, 64, [1, 130, 999], 0),
    (2, 1, 4, 2, 128, [100, 601], 128),
    # one CTA per unit with several tiles a warp (32 and 96 units or more), and its limits
    (17, 1, 6, 2, 64, [7 * i * i for i in range(17)], 0),
    (49, 1, 4, 2, 64, [60 + 70 * i for i in range(49)], 64),
    (33, 3, 8, 4, 128, [40 * i for i in range(33)], 0),
]


def run_attention(case, kind, q_type, out_type, rng, scale=0.0, q_scale=1.0):
    import alpaca_b200 as ab
    S, T, H, Hkv, d, ctx, block_rows = case
    cap = -(-max(max(ctx), 1) // 16) * 16 + 16
    q = (rng.standard_normal((S, T, H, d)) * q_scale).astype(np.float32)
    if q_type == "f16":
        q = q.astype(np.float16).astype(np.float32)
    parts = _kv4.random_cache(rng, S, Hkv, cap, d)
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    want = np.stack([_kv4.attention(q[s], k[s], v[s], ctx[s], scale or None) for s in range(S)])
    poison(parts, ctx)
    table = None
    if block_rows:
        parts, tb = paged(parts, block_rows, rng)
        table = dev(tb)
    out = torch.full((S, T, H, d), float("nan"), dtype=DT[out_type], device="cuda")
    ab.kv4_attention(dev(q).to(DT[q_type]), to_gpu(parts), out, ctx_lens=dev(np.array(ctx, np.int32)), max_ctx_len=max(ctx),
                     block_table=table, kind=kind, scale=scale)
    ab.device_status()
    return out.double().cpu().numpy(), want


@pytest.mark.parametrize("kind", ["DECODE_SPLIT", "GENERAL"])
@pytest.mark.parametrize("types", ["f32 f32", "f16 f16", "f16 f32"])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(cuda_lib, case, types, kind):
    import alpaca_b200 as ab
    q_type, out_type = types.split()
    got, want = run_attention(ATTN[case], ab.Kernel[kind], q_type, out_type, np.random.default_rng(case))
    check(got, want, F32_TOL, out_type)


@pytest.mark.parametrize("d", [32, 96, 160, 256])
def test_attention_other_head_dims(cuda_lib, d):
    import alpaca_b200 as ab
    got, want = run_attention((3, 2, 6, 3, d, [0, 40, 131], 16), ab.Kernel.AUTO, "f32", "f32", np.random.default_rng(d))
    check(got, want, F32_TOL, "f32")


@pytest.mark.parametrize("d,H,Hkv,ctx", [(64, 3, 1, 20000), (128, 4, 1, 9000), (64, 4, 4, 3001)])
def test_attention_many_splits(cuda_lib, d, H, Hkv, ctx):
    import alpaca_b200 as ab
    got, want = run_attention((1, 1, H, Hkv, d, [ctx], 0), ab.Kernel.DECODE_SPLIT, "f32", "f32", np.random.default_rng(d))
    check(got, want, F32_TOL, "f32")


@pytest.mark.parametrize("q_scale,scale", [(1e4, 1e-5), (1e-6, 0.0), (30.0, 0.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_query_ranges(cuda_lib, d, q_scale, scale):
    """Large and tiny queries; at 30 the softmax is nearly one-hot: scores reach 2^8, whose f32 rounding the bound allows."""
    import alpaca_b200 as ab
    got, want = run_attention((2, 1, 4, 2, d, [200, 900], 0), ab.Kernel.DECODE_SPLIT, "f32", "f32", np.random.default_rng(3),
                              scale=scale, q_scale=q_scale)
    # a score of magnitude S carries about S * 2^-21, which moves p by that much and the output by |v| (4) times it, twice
    check(got, want, F32_TOL + (2 * 4 * 300 * 2.0 ** -21 if q_scale == 30.0 else 0), "f32")


def test_attention_nan_block_stays_in_its_rows(cuda_lib):
    import alpaca_b200 as ab
    rng = np.random.default_rng(13)
    S, H, Hkv, d, n = 2, 6, 2, 64, 150
    parts = _kv4.random_cache(rng, S, Hkv, 160, d)
    parts[3].view(np.uint16)[0, 1, 70, 1] = 0x7E00  # V, sequence 0, head 1, second block
    parts[1].view(np.uint16)[1, 0, 149, 0] = 0x7E00  # K, sequence 1, head 0
    q = rng.standard_normal((S, 1, H, d)).astype(np.float32)
    for kind in (ab.Kernel.DECODE_SPLIT, ab.Kernel.GENERAL):
        out = torch.zeros((S, 1, H, d), dtype=torch.float32, device="cuda")
        ab.kv4_attention(dev(q), to_gpu(parts), out, start_position=n - 1, kind=kind)
        ab.device_status()
        bad = torch.isnan(out[:, 0]).cpu().numpy()
        want = np.zeros_like(bad)
        want[0, 3:, 32:] = True
        want[1, :3] = True
        assert np.array_equal(bad, want)


def test_attention_strides_stream_and_workspace_reuse(cuda_lib):
    """Queries inside a fused projection, an output with room between tokens, heads of a wider cache, on its own stream."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(17)
    S, T, H, Hkv, d, ctx = 2, 3, 4, 2, 64, 333
    parts = _kv4.random_cache(rng, S, Hkv + 3, 336, d)
    q = rng.standard_normal((S, T, H + 4, d)).astype(np.float32)
    stream = torch.cuda.Stream()
    buf, obuf = dev(q), torch.zeros((S, T, H + 1, d), dtype=torch.float32, device="cuda")
    cache = ab.Kv4Cache(*(x[:, 1:1 + Hkv] for x in to_gpu(parts)))
    qv = buf.as_strided((S, T, H, d), buf.stride())
    ov = obuf.as_strided((S, T, H, d), obuf.stride())
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        ab.kv4_attention(qv, cache, ov, start_position=ctx - T, kind=ab.Kernel.DECODE_SPLIT, stream=stream)
    ab.device_status(stream)
    k, v = _kv4.values(*parts[:2])[:, 1:3], _kv4.values(*parts[2:])[:, 1:3]
    want = np.stack([_kv4.attention(q[s][:, :H], k[s], v[s], ctx) for s in range(S)])
    check(ov.cpu().numpy(), want, F32_TOL, "f32")
    assert not obuf[:, :, H].any()


def test_attention_reports_bad_lengths_and_tables(cuda_lib):
    import alpaca_b200 as ab
    rng = np.random.default_rng(19)
    parts = _kv4.random_cache(rng, 3, 2, 64, 64)
    pool, table = paged(parts, 16, rng)
    q = dev(rng.standard_normal((3, 1, 4, 64)).astype(np.float32))
    for kind in (ab.Kernel.DECODE_SPLIT, ab.Kernel.GENERAL):
        out = torch.zeros((3, 1, 4, 64), dtype=torch.float32, device="cuda")
        for lens, bad in (([64, 65, 3], False), ([1, -1, 3], False), ([64, 64, 64], True)):
            tb = table.copy()
            if bad:
                tb[1, 2], tb[2, 0] = len(pool[0]), -1
            ab.kv4_attention(q, to_gpu(pool), out, ctx_lens=dev(np.array(lens, np.int32)), max_ctx_len=64, block_table=dev(tb), kind=kind)
            with pytest.raises(ab.AlpacaCUDAError) as e:
                ab.device_status()
            assert e.value.status == ab.Status.INVALID_ARGUMENT
            ab.device_status()
        assert torch.isfinite(out).all()


# ------------------------------------------------------------------------------------------------ prompt chunks

@pytest.mark.parametrize("d,H,Hkv", [(64, 9, 3), (128, 4, 2)])
@pytest.mark.parametrize("T,ctx", [(8, 8), (100, 100), (129, 400), (300, 1111)])
@pytest.mark.parametrize("block_rows", [0, 48])
@pytest.mark.parametrize("types", ["f16 f16", "f32 f32"])
def test_prefill(cuda_lib, d, H, Hkv, T, ctx, block_rows, types):
    import alpaca_b200 as ab
    q_type, out_type = types.split()
    rng = np.random.default_rng(T + ctx)
    S, cap = 2, -(-ctx // 16) * 16 + 32
    q = rng.standard_normal((S, T, H, d)).astype(np.float16).astype(np.float32)
    parts = _kv4.random_cache(rng, S, Hkv, cap, d)
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    poison(parts, [ctx] * S)
    table = None
    if block_rows:
        parts, tb = paged(parts, block_rows, rng)
        table = dev(tb)
    out = torch.full((S, T, H, d), float("nan"), dtype=DT[out_type], device="cuda")
    cache = to_gpu(parts)
    ab.kv4_attention(dev(q).to(DT[q_type]), cache, out, start_position=ctx - T, block_table=table, kind=ab.Kernel.PREFILL_TC)
    ab.device_status()
    rows = sorted({0, 1, T // 2, T - 1})
    for s in range(S):
        got = out[s].double().cpu().numpy()
        assert np.isfinite(got).all()
        for t in rows:
            want = _kv4.attention(q[s, t:t + 1], k[s], v[s], ctx - T + 1 + t)
            check(got[t:t + 1], want, TC_TOL, out_type)


@pytest.mark.parametrize("block_rows", [0, 64])
def test_prefill_ragged(cuda_lib, block_rows):
    import alpaca_b200 as ab
    rng = np.random.default_rng(23)
    H, Hkv, d = 6, 2, 64
    counts, starts = [130, 0, 1, 300, 47], [0, 10, 512, 77, 3]
    S, max_ctx = len(counts), 544
    offs = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rng.standard_normal((offs[-1], H, d)).astype(np.float16).astype(np.float32)
    parts = _kv4.random_cache(rng, S, Hkv, max_ctx, d)
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    poison(parts, [a + b for a, b in zip(counts, starts)])
    table = None
    if block_rows:
        parts, tb = paged(parts, block_rows, rng)
        table = dev(tb)
    out = torch.full((int(offs[-1]), H, d), float("nan"), dtype=torch.float32, device="cuda")
    ab.kv4_prefill_varlen(dev(q).half(), to_gpu(parts), out, dev(offs), dev(np.array(starts, np.int32)), max_tokens=300,
                          max_ctx_len=max_ctx, block_table=table)
    ab.device_status()
    got = out.double().cpu().numpy()
    for s in range(S):
        if counts[s]:
            want = _kv4.attention(q[offs[s]:offs[s + 1]], k[s], v[s], starts[s] + counts[s])
            check(got[offs[s]:offs[s + 1]], want, TC_TOL, "f32")


def test_rotation_at_long_positions(cuda_lib):
    """Angles far out: cos and sin keep double accuracy before their one rounding, as the oracle's."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(29)
    for start in (100_000, 12_345_678, (1 << 30) - 8):
        for d in (64, 96):
            q = rng.standard_normal((1, 4, 2, d)).astype(np.float32)
            out = torch.empty((1, 4, 2, d), dtype=torch.float32, device="cuda")
            ab.qkv_append(dev(q), None, None, out, None, theta=500000.0, start_position=start, interleaved=bool(d == 64))
            ab.device_status()
            assert np.array_equal(out[0].cpu().numpy(), oracle.rope(q[0], start, 500000.0, bool(d == 64)))


def test_example_session(cuda_lib, capsys):
    """The session of examples/kv4_session.py: the caches' bytes, and 4-bit context vectors near the f16 cache's.
    A value is off by at most half a step, uniform over it: 1 / sqrt(12) of a step of about 4.1 / 15 standard deviations, 8%; the
    scores' and the values' errors together stay below twice that."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "kv4_session.py"
    spec = importlib.util.spec_from_file_location("kv4_session", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    r = mod.main(["--prompt", "300", "--tokens", "5", "--chunk", "128", "--layers", "2"])
    rows = 305  # 2 layers, K and V, 3 heads of 64: 128 bytes a head row, and 36 with the rows rounded up to 16
    assert r["bytes"] == {"f16": 2 * 2 * 3 * 128 * rows, "4-bit": 2 * 2 * 3 * 36 * 320}
    assert r["relative_error"] < 0.16


@pytest.mark.parametrize("d", [64, 96, 128])
def test_offsets_past_32_bits(cuda_lib, d):
    """Two sequences whose caches lie more than 2^32 bytes (and 2^31 scales) apart: append, read-back and every attention form."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(31)
    S, T, H, Hkv, rows = 2, 40, 4, 2, 48
    far = (1 << 32) + 4096
    codes, scales = torch.zeros(far + 2 * Hkv * rows * d, dtype=torch.uint8, device="cuda"), \
        torch.zeros(far + 2 * Hkv * rows * (d // 32) + 4096, dtype=torch.int16, device="cuda")

    def view(buf, width, first):
        return buf.as_strided((S, Hkv, rows, width), (far, rows * width, width, 1), first)
    cache = ab.Kv4Cache(view(codes, d // 2, 0), view(scales, d // 32, 0), view(codes, d // 2, Hkv * rows * d // 2),
                        view(scales, d // 32, Hkv * rows * (d // 32)))
    q, k, v = (rng.standard_normal((S, T, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
    rot = torch.empty((S, T, H, d), dtype=torch.float32, device="cuda")
    ab.qkv_append(dev(q), dev(k), dev(v), rot, cache, theta=1e4)
    ko, vo = (torch.empty((S, T, Hkv, d), dtype=torch.float32, device="cuda") for _ in range(2))
    ab.kv4_read(cache, ko, vo)
    ab.device_status()
    want_v = _kv4.values(*_kv4.quantise(v))
    assert np.array_equal(vo.double().cpu().numpy(), want_v)
    kd, qd = ko.double().cpu().numpy(), rot.cpu().numpy()
    for kind in (["DECODE_SPLIT", "PREFILL_TC", "GENERAL"] if d != 96 else ["GENERAL"]):
        out = torch.empty((S, T, H, d), dtype=torch.float32, device="cuda")
        ab.kv4_attention(rot, cache, out, kind=ab.Kernel[kind])
        ab.device_status()
        for s in range(S):
            want = _kv4.attention(qd[s], np.swapaxes(kd[s], 0, 1), np.swapaxes(want_v[s], 0, 1), T)
            check(out[s].cpu().numpy(), want, TC_TOL if kind == "PREFILL_TC" else F32_TOL, "f32")


@pytest.mark.parametrize("tokens,start,kind", [(1, 900, "DECODE_SPLIT"), (5, 900, "DECODE_SPLIT"), (1, 6, "DECODE_SPLIT"),
                                               (100, 1500, "PREFILL_TC"), (300, 0, "PREFILL_TC"), (3, 50, "GENERAL")])
@pytest.mark.parametrize("d", [64, 128])
def test_graph_behind_other_work(cuda_lib, tokens, start, kind, d):
    """Append, attention and read-back as a captured graph, replayed on a cleared workspace behind queued work: every launch
    waits for what the one before it wrote, and a replay takes the inputs that stand there then."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(41 + tokens + d)
    S, H, Hkv, n = 3, 6, 2, start + tokens
    parts = _kv4.random_cache(rng, S, Hkv, -(-n // 16) * 16, d)
    cache = to_gpu(parts)
    q, k, v = (torch.empty((S, tokens, h, d), device="cuda") for h in (H, Hkv, Hkv))
    rot, out = torch.empty_like(q), torch.empty_like(q)
    ko, vo = torch.empty((S, n, Hkv, d), device="cuda"), torch.empty((S, n, Hkv, d), device="cuda")
    desc = ab.make_kv4_attn_desc(rot, cache, out, start_position=start)
    ws = torch.zeros(max(16, ab.kv4_workspace_bytes(desc, ab.Kernel[kind])), dtype=torch.uint8, device="cuda")
    busy = torch.zeros(1 << 26, device="cuda")

    def step():
        ab.qkv_append(q, k, v, rot, cache, start_position=start, theta=1e4)
        ab.kv4_attention(rot, cache, out, start_position=start, kind=ab.Kernel[kind], workspace=ws)
        ab.kv4_read(cache, ko, vo)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x in (q, k, v):
            x.zero_()
        step()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(2):
            for x in (q, k, v):
                x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
            ws.zero_()
            for x in (out, ko, vo):
                x.fill_(7.0)
            stream.synchronize()
            for _ in range(4):
                busy.mul_(1.0)
            graph.replay()
            stream.synchronize()
            ab.device_status(stream)
            kd, vd = ko.double().cpu().numpy(), vo.double().cpu().numpy()
            want_v = _kv4.values(*parts[2:])[:, :, :n].swapaxes(1, 2).copy()
            want_v[:, start:] = _kv4.values(*_kv4.quantise(v.cpu().numpy()))
            assert np.array_equal(vd, want_v)
            for s in range(S):
                want = _kv4.attention(rot[s].cpu().numpy(), kd[s].swapaxes(0, 1), vd[s].swapaxes(0, 1), n)
                check(out[s].cpu().numpy(), want, TC_TOL if kind == "PREFILL_TC" else F32_TOL, "f32")
    del graph


@pytest.mark.parametrize("d", [64, 128])
def test_varlen_behind_other_work(cuda_lib, d):
    """The ragged form on a cleared workspace behind queued work."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(43 + d)
    H, Hkv, lens, starts = 6, 2, [100, 1, 300], [700, 50, 0]
    parts = _kv4.random_cache(rng, 3, Hkv, 800, d)
    cache = to_gpu(parts)
    q = rng.standard_normal((sum(lens), H, d)).astype(np.float32)
    offs = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    qd, od, sd = dev(q), dev(offs), dev(np.array(starts, np.int32))
    out = torch.full(q.shape, 7.0, device="cuda")
    desc = ab.make_kv4_varlen_desc(qd, cache, out, od, sd, max_tokens=300, max_ctx_len=800)
    ws = torch.zeros(ab.kv4_workspace_bytes(desc), dtype=torch.uint8, device="cuda")
    busy = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    for _ in range(4):
        busy.mul_(1.0)
    ab.kv4_attention_launch(desc, ws)
    ab.device_status()
    k, v = _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    for s, (n, p) in enumerate(zip(lens, starts)):
        want = _kv4.attention(q[offs[s]:offs[s + 1]], k[s], v[s], n + p)
        check(out[offs[s]:offs[s + 1]].cpu().numpy(), want, TC_TOL, "f32")


@pytest.mark.parametrize("d,H,Hkv", [(64, 2, 1), (64, 9, 3), (96, 2, 1), (128, 3, 1)])
@pytest.mark.parametrize("S,T", [(1, 1003), (3, 739), (1, 4099), (2, 2501)])
@pytest.mark.parametrize("by_positions", [False, True])
def test_append_prompts_equal_definition_bitwise(cuda_lib, d, H, Hkv, S, T, by_positions):
    """Prompts long enough for every number of tokens per CTA, none of them a divisor of the prompt."""
    import alpaca_b200 as ab
    rng = np.random.default_rng(S * T + d)
    theta, starts = 10000.0, ([5, 130, 0][:S] if by_positions else [21] * S)
    q, k, v = (rng.standard_normal((S, T, h, d)).astype(np.float32) for h in (H, Hkv, Hkv))
    cache = ab.kv4_cache(S, max(starts) + T, Hkv, d)
    out = torch.empty((S, T, H, d), dtype=torch.float32, device="cuda")
    where = dict(positions=dev(np.array(starts, np.int32))) if by_positions else dict(start_position=21)
    ab.qkv_append(dev(q), dev(k), dev(v), out, cache, theta=theta, **where)
    ab.device_status()
    for s, p in enumerate(starts):
        assert np.array_equal(out[s].cpu().numpy(), oracle.rope(q[s], p, theta, True))
        for i, x in ((0, oracle.rope(k[s], p, theta, True)), (2, v[s])):
            codes, scales = _kv4.quantise(np.swapaxes(x, 0, 1))
            assert np.array_equal(cache[i][s, :, p:p + T].cpu().numpy(), codes)
            assert np.array_equal(cache[i + 1][s, :, p:p + T].cpu().numpy(), scales)
        assert not cache.k_codes[s, :, :p].any() and not cache.k_codes[s, :, p + T:].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,H,Hkv", [(1, 4, 4), (1, 6, 2), (1, 16, 2), (2, 9, 3), (7, 9, 3), (18, 9, 3)])
@pytest.mark.parametrize("ctx", [1, 20, 31, 65, 300, 1000])
def test_attention_of_few_units(cuda_lib, d, T, H, Hkv, ctx):
    """One CTA per unit: fewer tiles than warps, more, and a last group of query rows that is not full; f16 and f32 out."""
    import alpaca_b200 as ab
    if T > ctx:
        ctx += T
    rng = np.random.default_rng(ctx + T + H)
    S = 2
    parts = _kv4.random_cache(rng, S, Hkv, -(-ctx // 16) * 16, d)
    q = rng.standard_normal((S, T, H, d)).astype(np.float32)
    lens = np.array([ctx, max(0, ctx - 3)], np.int32)
    cache, k, v = to_gpu(parts), _kv4.values(*parts[:2]), _kv4.values(*parts[2:])
    for out_type in ("f32", "f16"):
        out = torch.full(q.shape, 7.0, dtype=DT[out_type], device="cuda")
        ab.kv4_attention(dev(q), cache, out, ctx_lens=dev(lens), max_ctx_len=ctx, kind=ab.Kernel.DECODE_SPLIT)
        ab.device_status()
        for s in range(S):
            check(out[s].float().cpu().numpy(), _kv4.attention(q[s], k[s], v[s], int(lens[s])), F32_TOL, out_type)
