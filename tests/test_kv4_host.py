"""The 4-bit KV cache without a GPU: the format's plain form, the library's refusals, kernel choice and workspace sizes. No
call here launches a kernel."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from tests import _kv4

FAKE = 1 << 20  # a 16-byte aligned fake device address: validation never dereferences pointers


@pytest.fixture(scope="module")
def lib():
    from alpaca_b200 import build
    build.build()
    import alpaca_b200
    return alpaca_b200.load()


def cache_desc(rows=256, heads=3, d=64, units=4, **kw):
    import alpaca_b200 as ab
    c = ab.Kv4CacheDesc()
    c.k_codes = c.v_codes = c.k_scales = c.v_scales = FAKE
    c.code_head_stride, c.scale_head_stride = rows * d // 2, rows * d // 32
    c.code_unit_stride, c.scale_unit_stride = heads * rows * d // 2, heads * rows * d // 32
    c.rows = rows
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn_desc(cache=None, **kw):
    import alpaca_b200 as ab
    a = ab.Kv4AttnDesc()
    a.n_seqs, a.n_heads, a.n_kv_heads, a.head_dim, a.tokens, a.start_position = 4, 9, 3, 64, 1, 199
    a.q_dtype = a.out_dtype = int(ab.DType.F32)
    a.q = a.out = FAKE
    a.q_token_stride = a.out_token_stride = a.q_seq_stride = a.out_seq_stride = 9 * 64
    for k, v in kw.items():
        setattr(a, k, v)
    a.cache = cache if cache is not None else cache_desc(d=a.head_dim)
    return a


def qkv_desc(cache=None, **kw):
    import alpaca_b200 as ab
    a = ab.QkvDesc()
    a.n_seqs, a.n_heads, a.n_kv_heads, a.head_dim, a.tokens, a.start_position = 4, 9, 3, 64, 2, 100
    a.theta, a.eps, a.interleaved, a.cache_kind = 1e4, 1e-5, 1, int(ab.CacheKind.KV4)
    a.q = a.q_out = a.k = a.v = FAKE
    a.q_token_stride = a.q_out_token_stride = 9 * 64
    a.q_seq_stride = a.q_out_seq_stride = 2 * 9 * 64
    a.kv_token_stride, a.kv_seq_stride = 3 * 64, 2 * 3 * 64
    a.kv4 = cache if cache is not None else cache_desc()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def read_desc(cache=None, **kw):
    import alpaca_b200 as ab
    a = ab.Kv4ReadDesc()
    a.n_seqs, a.n_kv_heads, a.head_dim, a.n_rows, a.start_row, a.out_dtype = 4, 3, 64, 10, 20, int(ab.DType.F16)
    a.k_out = a.v_out = FAKE
    a.out_row_stride, a.out_seq_stride = 3 * 64, 10 * 3 * 64
    a.cache = cache if cache is not None else cache_desc()
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_struct_sizes_match_header(tmp_path):
    """sizeof and the last field's offset of every structure, from the C compiler."""
    import shutil
    import subprocess
    from pathlib import Path

    import alpaca_b200 as ab
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    inc = Path(__file__).resolve().parent.parent / "include"
    names = {"alpaca_kv4_cache": (ab.Kv4CacheDesc, "reserved0"), "alpaca_qkv_desc": (ab.QkvDesc, "reserved0"),
             "alpaca_kv4_read_desc": (ab.Kv4ReadDesc, "reserved0"), "alpaca_kv4_attn_desc": (ab.Kv4AttnDesc, "cache")}
    src = tmp_path / "s.c"
    src.write_text('#include "alpaca_cuda.h"\n#include <stdio.h>\nint main(void) {\n' + "".join(
        f'printf("%zu %zu\\n", sizeof({n}), offsetof({n}, {last}));\n' for n, (_, last) in names.items()) + "return 0;}\n")
    subprocess.run([cc, "-I", str(inc), str(src), "-o", str(tmp_path / "s")], check=True)
    out = subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()
    for i, (n, (t, last)) in enumerate(names.items()):
        assert (int(out[2 * i]), int(out[2 * i + 1])) == (ctypes.sizeof(t), getattr(t, last).offset), n


# ------------------------------------------------------------------------------------------------ plain form

@pytest.mark.parametrize("scale", [1e-5, 1.0, 300.0, 1e5])
def test_quantised_values_within_half_a_step(scale):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 64)) * scale).astype(np.float32)
    x[:40] = np.abs(x[:40])
    x[40:80] = -np.abs(x[40:80])
    codes, scales = _kv4.quantise(x)
    y = _kv4.values(codes, scales)
    step = np.repeat((scales.view(np.uint16) & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64), 32, -1)
    blocks = x.reshape(200, 2, 32).astype(np.float64)
    span = np.maximum(blocks.max(-1), 0) - np.minimum(blocks.min(-1), 0)
    inside = np.repeat(span <= 65280, 32, -1)  # a wider block saturates
    assert np.all((np.abs(y - x) <= step / 2 * (1 + 2.0 ** -20))[inside])
    assert np.array_equal(y, y.astype(np.float16).astype(np.float64))  # every value is exact in f16


def test_values_exact_in_f16_for_every_header():
    for zero in range(16):
        bits = (np.arange(0x10, 0x6C50, 16) | zero).astype(np.uint16)
        scales = bits.view(np.int16).reshape(-1, 1)
        codes = np.tile(np.arange(16, dtype=np.uint8) * 17, (len(bits), 1))
        y = _kv4.values(codes, scales)
        assert np.array_equal(y, y.astype(np.float16).astype(np.float64))


def test_special_blocks():
    x = np.zeros((6, 32), np.float32)
    x[1, 3], x[2, 4], x[3, 5], x[4] = np.nan, np.inf, -np.inf, 3.4e38
    x[5, 0] = 1e-12
    codes, scales = _kv4.quantise(x)
    y = _kv4.values(codes, scales)
    assert not y[0].any() and np.isnan(y[1:4]).all()
    assert np.array_equal(y[4], np.full(32, 65280.0))
    assert not y[5].any()


# ------------------------------------------------------------------------------------------------ refusals

def status(lib, kind, d):
    import alpaca_b200 as ab
    if kind == "attn":
        n = ctypes.c_size_t(0)
        return ab.Status(lib.alpaca_kv4_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(n)))
    # refused before anything is enqueued: these descriptors never reach a launch
    f = lib.alpaca_qkv_append if kind == "qkv" else lib.alpaca_kv4_read
    return ab.Status(f(ctypes.byref(d), None))


BAD_CACHE = [dict(k_codes=0), dict(v_scales=0), dict(k_codes=FAKE + 8), dict(v_scales=FAKE + 4), dict(rows=0), dict(rows=24),
             dict(code_head_stride=256 * 32 - 16), dict(code_head_stride=256 * 32 + 8), dict(scale_head_stride=256 * 2 + 4),
             dict(scale_head_stride=256 * 2 - 8), dict(code_unit_stride=16), dict(code_unit_stride=-16), dict(rows=96),
             dict(block_table=FAKE, max_blocks=0, pool_blocks=9), dict(block_table=FAKE, max_blocks=4, pool_blocks=0),
             dict(block_table=FAKE, max_blocks=1, pool_blocks=9, rows=16)]


@pytest.mark.parametrize("i", range(len(BAD_CACHE)))
def test_bad_caches_are_refused(lib, i):
    import alpaca_b200 as ab
    for kind, make in (("attn", attn_desc), ("qkv", qkv_desc), ("read", read_desc)):
        kw = dict(start_row=150) if kind == "read" else {}
        assert status(lib, kind, make(cache=cache_desc(**BAD_CACHE[i]), **kw)) == ab.Status.INVALID_ARGUMENT, (kind, BAD_CACHE[i])
        assert b"4-bit cache" in lib.alpaca_cuda_last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_seqs=65536), dict(n_heads=8), dict(n_kv_heads=0), dict(tokens=0),
                                dict(start_position=-1), dict(head_dim=48), dict(head_dim=288), dict(q_dtype=2), dict(out_dtype=-1),
                                dict(flags=2), dict(scale=-1.0), dict(scale=float("nan")), dict(q=0), dict(out=FAKE + 4),
                                dict(q_token_stride=9 * 64 - 4), dict(q_seq_stride=0), dict(out_seq_stride=9 * 64 + 2),
                                dict(start_position=256), dict(start_position=(1 << 30) + 1), dict(ctx_lens=FAKE, max_ctx_len=-1),
                                dict(ctx_lens=FAKE, max_ctx_len=257), dict(flags=1), dict(flags=1, q_offsets=FAKE, start_positions=FAKE),
                                dict(flags=1, q_offsets=FAKE, start_positions=FAKE, total_tokens=5, max_ctx_len=9, ctx_lens=FAKE)])
def test_bad_attention_calls_are_refused(lib, kw):
    import alpaca_b200 as ab
    assert status(lib, "attn", attn_desc(**kw)) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_cuda_last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(tokens=0), dict(n_heads=0, n_kv_heads=0), dict(head_dim=40), dict(theta=0.0),
                                dict(theta=float("inf")), dict(interleaved=2), dict(flags=1), dict(in_dtype=5), dict(q_out_dtype=9),
                                dict(cache_kind=3), dict(q_norm=FAKE, eps=0.0), dict(k_norm=FAKE + 4), dict(q=FAKE + 8), dict(q_out=0),
                                dict(k=0), dict(v=FAKE + 2), dict(kv_token_stride=3 * 64 - 4), dict(kv_seq_stride=0),
                                dict(q_out_token_stride=9 * 64 + 2), dict(q_out_dtype=1), dict(start_position=255),
                                dict(cache_kind=1), dict(cache_kind=0, k_cache=FAKE, v_cache=FAKE, cache_row_stride=3 * 64, cache_seq_stride=64 * 192, cache_rows=64)])
def test_bad_appends_are_refused(lib, kw):
    import alpaca_b200 as ab
    assert status(lib, "qkv", qkv_desc(**kw)) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_cuda_last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(n_rows=-1), dict(start_row=-1), dict(head_dim=20), dict(out_dtype=3), dict(k_out=0),
                                dict(v_out=FAKE + 8), dict(out_row_stride=128), dict(out_seq_stride=0), dict(out_row_stride=3 * 64 + 4),
                                dict(start_row=247), dict(flags=1)])
def test_bad_reads_are_refused(lib, kw):
    import alpaca_b200 as ab
    assert status(lib, "read", read_desc(**kw)) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_cuda_last_error()


def test_null_descriptors(lib):
    import alpaca_b200 as ab
    n = ctypes.c_size_t(0)
    assert lib.alpaca_qkv_append(None, None) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_read(None, None) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_attention(None, 0, None, 0, None) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_workspace_bytes(None, 0, ctypes.byref(n)) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_workspace_bytes(ctypes.byref(attn_desc()), 0, None) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_select(ctypes.byref(attn_desc()), None) == ab.Status.INVALID_ARGUMENT
    assert lib.alpaca_kv4_workspace_bytes(ctypes.byref(attn_desc()), 9, ctypes.byref(n)) == ab.Status.INVALID_ARGUMENT


def test_an_empty_read_is_ok(lib):
    import alpaca_b200 as ab
    assert status(lib, "read", read_desc(n_rows=0)) == ab.Status.OK


def test_kernel_choice(lib):
    import alpaca_b200 as ab
    K = ab.Kernel
    wide = dict(q_seq_stride=128 * 9 * 64, out_seq_stride=128 * 9 * 64)
    assert ab.kv4_select(attn_desc()) == K.DECODE_SPLIT
    assert ab.kv4_select(attn_desc(tokens=7, start_position=100, **wide)) == K.DECODE_SPLIT
    assert ab.kv4_select(attn_desc(tokens=128, start_position=100, **wide)) == K.PREFILL_TC
    # 4 sequences of 4000 rows: a few tokens on the split kernel, a chunk on the prefill
    for tokens, kind in ((8, K.DECODE_SPLIT), (32, K.DECODE_SPLIT), (128, K.PREFILL_TC), (512, K.PREFILL_TC)):
        big = dict(tokens=tokens, start_position=4000 - tokens, q_seq_stride=tokens * 576, out_seq_stride=tokens * 576)
        assert ab.kv4_select(attn_desc(cache=cache_desc(rows=4000), **big)) == kind, tokens
    assert ab.kv4_select(attn_desc(tokens=128, ctx_lens=FAKE, max_ctx_len=200, **wide)) == K.DECODE_SPLIT
    assert ab.kv4_select(attn_desc(head_dim=96, q_token_stride=864, out_token_stride=864, q_seq_stride=864, out_seq_stride=864)) == K.GENERAL
    varlen = attn_desc(flags=1, q_offsets=FAKE, start_positions=FAKE, total_tokens=5, max_ctx_len=9)
    assert ab.kv4_select(varlen) == K.PREFILL_TC
    n = ctypes.c_size_t(0)
    for d, kind in ((varlen, K.DECODE_SPLIT), (varlen, K.GENERAL), (attn_desc(ctx_lens=FAKE, max_ctx_len=9), K.PREFILL_TC),
                    (attn_desc(head_dim=96, q_token_stride=864, out_token_stride=864, q_seq_stride=864, out_seq_stride=864), K.DECODE_SPLIT)):
        assert lib.alpaca_kv4_workspace_bytes(ctypes.byref(d), int(kind), ctypes.byref(n)) == ab.Status.UNSUPPORTED


def test_workspace_too_small_is_refused(lib):
    import alpaca_b200 as ab
    d = attn_desc(n_seqs=1, start_position=20000, cache=cache_desc(rows=20016))
    need = ab.kv4_workspace_bytes(d)
    assert need > 0
    for ws, n in ((None, need), (FAKE, need - 1), (None, 0)):
        assert lib.alpaca_kv4_attention(ctypes.byref(d), 0, ws, n, None) == ab.Status.WORKSPACE_TOO_SMALL
    assert lib.alpaca_kv4_attention(ctypes.byref(d), 0, FAKE + 4, need, None) == ab.Status.INVALID_ARGUMENT
    assert ab.kv4_workspace_bytes(d, ab.Kernel.GENERAL) == 0


def test_host_tensors_are_refused(lib):
    """The kernels follow raw addresses, so a call with a host tensor must not reach them."""
    import torch

    import alpaca_b200 as ab
    cache = ab.kv4_cache(2, 32, 2, 64, device="cpu")
    q, k = torch.zeros((2, 3, 4, 64)), torch.zeros((2, 3, 2, 64))
    for call in (lambda: ab.qkv_append(q, k, k.clone(), torch.empty_like(q), cache, theta=1e4),
                 lambda: ab.qkv_append(q, None, None, torch.empty_like(q), None, theta=1e4),
                 lambda: ab.qkv_append(None, k, k.clone(), None, (torch.empty(2, 8, 2, 64), torch.empty(2, 8, 2, 64)), theta=1e4),
                 lambda: ab.kv4_read(cache, k, k.clone()),
                 lambda: ab.kv4_attention(q, cache, torch.empty_like(q))):
        with pytest.raises(ab.AlpacaCUDAError, match="one CUDA device") as e:
            call()
        assert e.value.status == ab.Status.INVALID_ARGUMENT
