"""The 4-bit KV cache operators as measured work: writing rows (q / k norms, RoPE, quantisation), reading them back, and
attention over the cache. Each has a plain form in elementary torch operations and, with `own`, the library's calls.

The 4-bit cache (one tensor pair for K, one for V; unit = sequence, or block of a pool):
  codes   uint8 [units][kv heads][rows][d / 2]    eight 4-bit codes per 32-bit word; with d / 32 blocks of 32 channels,
                                                  word t * (d / 32) + b holds channels 32 b + 8 t .. + 7, low nibble first
  scales  int16 [units][kv heads][rows][d / 32]   f16 bits of the block's step d; the low 4 mantissa bits are its zero point z
  value = (code - z) * d
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
THETA = 10000.0
DTYPES = {"f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases

def _append(name, seqs, tokens, heads, kv_heads, head_dim, start, norm, interleaved, in_type, q_type, cache="kv4"):
    return dict(name=name, op="append", seqs=seqs, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                start=start, norm=norm, interleaved=interleaved, in_type=in_type, q_type=q_type, cache=cache)


def _read(name, seqs, rows, kv_heads, head_dim, out_type):
    return dict(name=name, op="read", seqs=seqs, rows=rows, kv_heads=kv_heads, head_dim=head_dim, out_type=out_type)


def _attend(name, seqs, tokens, heads, kv_heads, head_dim, ctx, ragged, block_rows, q_type, out_type):
    return dict(name=name, op="attend", seqs=seqs, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                ctx=ctx, ragged=ragged, block_rows=block_rows, q_type=q_type, out_type=out_type)


def listed():
    return [
        # One decode step's append for a serving batch of the SmolLM2-135M shape: the f32 rows of the decode
        # projections, every sequence at its own position. Latency counts.
        _append("append_decode", 64, 1, 9, 3, 64, 4095, False, True, "f32", "f32"),
        # A whole prompt of the SmolLM2-135M shape written in one pass, with q / k norms in front of the rotation.
        _append("append_prompt_norm", 1, 4096, 9, 3, 64, 0, True, False, "f32", "f16"),
        # Prompts of a batch at head_dim 128 with q / k norms, f16 projections, into the 4-bit cache.
        _append("append_batch_norm_d128", 8, 2048, 32, 8, 128, 777, True, False, "f16", "f16"),
        # The same pass for a caller who keeps an f16 cache.
        _append("append_prompt_norm_f16", 2, 2011, 15, 5, 64, 301, True, True, "f32", "f16", "f16"),
        # One session's rows back as f16, as before handing the cache to an f16 consumer.
        _read("read_session", 1, 1357, 3, 64, "f16"),
        # A batch of caches read back whole (SmolLM2-360M shape, 8 sequences of 4096 tokens).
        _read("read_batch", 8, 4096, 5, 64, "f16"),
        # One chat session's decode step with a short odd context: latency.
        _attend("decode_one", 1, 1, 9, 3, 64, 517, False, 0, "f32", "f32"),
        # Decode of 64 sequences with contexts of 1..4096 (SmolLM2-135M shape), f32 in and out.
        _attend("decode_batch", 64, 1, 9, 3, 64, 4096, True, 0, "f32", "f32"),
        # Decode of 64 sequences with contexts of 1..8192 (SmolLM2-1.7B shape): a GPU's share of 512 sequences on 8 GPUs.
        _attend("decode_mha_long", 64, 1, 32, 32, 64, 8192, True, 0, "f16", "f16"),
        # Grouped heads at head_dim 128 over a paged pool of 64-row blocks, long ragged contexts.
        _attend("decode_paged_d128", 48, 1, 32, 8, 128, 16000, True, 64, "f16", "f16"),
        # A prompt's last 512-token chunk over the cache of the tokens before it (SmolLM2-135M shape).
        _attend("chunk_512", 1, 512, 9, 3, 64, 4096, False, 0, "f16", "f16"),
        # Whole prompts of 4096 tokens in one call (SmolLM2-360M shape, two sequences).
        _attend("prompt_4096", 2, 4096, 15, 5, 64, 4096, False, 0, "f16", "f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(9, 3, 64), (15, 5, 64), (32, 32, 64), (16, 2, 64), (32, 8, 128), (8, 8, 128)])
    op = rng.choice(["append", "append", "read", "attend", "attend", "attend"])
    if op == "append":
        seqs = _log_int(rng, 1, 64)
        tokens = 1 if rng.random() < 0.3 else _log_int(rng, 2, max(2, 12000 // seqs))
        return _drop_name(_append("", seqs, tokens, heads, kv_heads, head_dim, rng.randrange(0, 5000), rng.random() < 0.6,
                                  rng.random() < 0.5, rng.choice(["f16", "f32"]), rng.choice(["f16", "f32"]),
                                  "kv4" if tokens == 1 or rng.random() < 0.7 else "f16"))
    if op == "read":
        seqs = _log_int(rng, 1, 32)
        return _drop_name(_read("", seqs, _log_int(rng, 1, 160000 // (seqs * kv_heads)), kv_heads, head_dim, rng.choice(["f16", "f32"])))
    kind = rng.choice(["decode", "decode", "few", "chunk"])
    if kind == "chunk":
        seqs = _log_int(rng, 1, 4)
        tokens = _log_int(rng, 16, 2000 // seqs)
        ctx = tokens + rng.randrange(0, 2000)
        block = rng.choice([0, 0, 64, 128])
        return _drop_name(_attend("", seqs, tokens, heads, kv_heads, head_dim, ctx, False, block, "f16", "f16"))
    seqs = _log_int(rng, 1, 64)
    tokens = 1 if kind == "decode" else rng.randrange(2, 8)
    rows = 8_000_000 * 64 // (seqs * kv_heads * head_dim)
    ctx = _log_int(rng, 16, min(16000, rows))
    return _drop_name(_attend("", seqs, tokens, heads, kv_heads, head_dim, ctx, rng.random() < 0.7, rng.choice([0, 0, 16, 64, 128]),
                              rng.choice(["f16", "f32"]), rng.choice(["f16", "f32"])))


def _drop_name(case):
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ plain form

def _quantise(x):
    """f32 [..., d] -> (codes uint8 [..., d / 2], scales int16 [..., d / 32])."""
    blocks = x.shape[-1] // 32
    y = x.reshape(*x.shape[:-1], blocks, 32)
    lo, hi = y.amin(-1).clamp(max=0.0), y.amax(-1).clamp(min=0.0)
    # divided by a tensor: torch multiplies by a rounded 1 / 15 when the divisor is a number
    step = ((hi - lo) / torch.full_like(hi, 15.0)).clamp(max=4352.0)
    half = step.half()
    bits = half.view(torch.int16).to(torch.int32) + (half.float() < step).to(torch.int32)
    bits = (bits + 15) // 16 * 16
    d = bits.to(torch.int16).view(torch.float16).float()
    safe = torch.where(d > 0, d, torch.ones_like(d))  # an all-zero block has step 0
    z = torch.round(-lo / safe).clamp(0, 15)
    c = (torch.round(y / safe.unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0, 15).to(torch.uint8)
    scales = (bits + z.to(torch.int32)).to(torch.int16)
    c = c.reshape(*x.shape[:-1], blocks, 4, 4, 2).transpose(-4, -3)  # [t][block][byte][nibble]
    codes = (c[..., 0] | (c[..., 1] << 4)).reshape(*x.shape[:-1], x.shape[-1] // 2)
    return codes.contiguous(), scales.contiguous()


def _values(codes, scales):
    """The f32 values [..., d] that 4-bit rows stand for."""
    blocks = scales.shape[-1]
    d = (scales & -16).view(torch.float16).float().unsqueeze(-1)
    z = (scales & 15).float().unsqueeze(-1)
    b = codes.reshape(*codes.shape[:-1], 4, blocks, 4).transpose(-3, -2)  # [block][t][byte]
    c = torch.stack((b & 15, b >> 4), -1).reshape(*scales.shape, 32).float()
    return ((c - z) * d).reshape(*codes.shape[:-1], blocks * 32)


def _rotate(x, cos, sin, interleaved):
    """x [S, T, H, d] rotated by cos, sin [S, T, 1, d / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _norm(x, w):
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w


def _plain_append(s, c):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if c["norm"]:
        q, k = _norm(q, s["q_norm"]), _norm(k, s["k_norm"])
    q, k = (_rotate(x, s["cos"], s["sin"], c["interleaved"]) for x in (q, k))
    if c["cache"] == "kv4":
        k, v = _values(*_quantise(k)), _values(*_quantise(v))
    return {"q": q.to(DTYPES[c["q_type"]]), "k": k.half(), "v": v.half()}


def _rows(codes, scales, table):
    """Pool blocks [blocks][heads][rows][..] -> [seqs][heads][rows][..] through the block table."""
    if table is None:
        return codes, scales
    return tuple(x[table.long()].transpose(1, 2).flatten(2, 3) for x in (codes, scales))


def _plain_attend(s, c):
    group = c["heads"] // c["kv_heads"]
    q = s["q"].float().transpose(1, 2).reshape(c["seqs"], c["kv_heads"], group * c["tokens"], c["head_dim"])
    k = _values(*_rows(s["k_codes"], s["k_scales"], s["table"]))[:, :, : c["ctx"]]
    score = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(c["head_dim"]))
    del k
    score = score.reshape(c["seqs"], c["heads"], c["tokens"], c["ctx"])
    row = torch.arange(c["ctx"], device=DEV)
    last = s["lens"][:, None] - c["tokens"] + torch.arange(c["tokens"], device=DEV)  # newest row that token t sees
    seen = (row <= last[..., None])[:, None]
    score = score.masked_fill(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)  # a token that sees nothing gives zeros
    p = torch.exp(score - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    del score
    v = _values(*_rows(s["v_codes"], s["v_scales"], s["table"]))[:, :, : c["ctx"]]
    # rows past a context may hold anything
    v = v.masked_fill((row >= s["lens"][:, None])[:, None, :, None], 0.0)
    o = p.reshape(c["seqs"], c["kv_heads"], group * c["tokens"], c["ctx"]) @ v
    o = o.reshape(c["seqs"], c["heads"], c["tokens"], c["head_dim"]).transpose(1, 2)
    return o.to(DTYPES[c["out_type"]]).contiguous()


# ------------------------------------------------------------------------------------------------ inputs

def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEV, dtype=dtype)


def _random_cache(gen, units, heads, rows, head_dim):
    """Codes and scales of N(0, 1) rows, made in slices to keep the f32 rows small."""
    codes = torch.empty((units, heads, rows, head_dim // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((units, heads, rows, head_dim // 32), dtype=torch.int16, device=DEV)
    step = max(1, (1 << 27) // (heads * rows * head_dim))
    for i in range(0, units, step):
        n = min(step, units - i)
        codes[i:i + n], scales[i:i + n] = _quantise(_normal(gen, n, heads, rows, head_dim))
    return codes, scales


def _up(n, m):
    return (n + m - 1) // m * m


def prepare(case, seed):
    """The tensors in hand before the call and, with `own`, the descriptor and workspace that a program keeps for them."""
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "append":
        S, T, D = c["seqs"], c["tokens"], c["head_dim"]
        kind = DTYPES[c["in_type"]]
        s["q"] = _normal(gen, S, T, c["heads"], D).to(kind)
        s["k"] = _normal(gen, S, T, c["kv_heads"], D).to(kind)
        s["v"] = _normal(gen, S, T, c["kv_heads"], D).to(kind)
        if c["norm"]:
            s["q_norm"] = 1.0 + 0.1 * _normal(gen, D)
            s["k_norm"] = 1.0 + 0.1 * _normal(gen, D)
        # one token: every sequence at its own position up to `start`; longer runs: all from `start`
        if T == 1:
            start = torch.randint(0, c["start"] + 1, (S,), generator=gen, device=DEV, dtype=torch.int32)
        else:
            start = torch.full((S,), c["start"], device=DEV, dtype=torch.int32)
        s["positions"] = start
        # the cos / sin table of the positions, as a program without a fused pass keeps it
        angle = (start[:, None] + torch.arange(T, device=DEV)).double()[..., None] * _frequencies(D)
        s["cos"], s["sin"] = angle.cos().float().unsqueeze(2), angle.sin().float().unsqueeze(2)
    elif c["op"] == "read":
        rows = _up(c["rows"], 16)
        s["k_codes"], s["k_scales"] = _random_cache(gen, c["seqs"], c["kv_heads"], rows, c["head_dim"])
        s["v_codes"], s["v_scales"] = _random_cache(gen, c["seqs"], c["kv_heads"], rows, c["head_dim"])
    else:
        S, D, block = c["seqs"], c["head_dim"], c["block_rows"]
        s["q"] = _normal(gen, S, c["tokens"], c["heads"], D).to(DTYPES[c["q_type"]])
        if c["ragged"]:
            s["lens"] = torch.randint(1, c["ctx"] + 1, (S,), generator=gen, device=DEV, dtype=torch.int32)
        else:
            s["lens"] = torch.full((S,), c["ctx"], device=DEV, dtype=torch.int32)
        s["table"], units, rows = None, S, _up(c["ctx"], 16)
        if block:
            per = -(-c["ctx"] // block)
            units, rows = S * per, block
            s["table"] = torch.randperm(units, generator=gen, device=DEV).to(torch.int32).reshape(S, per)
        s["k_codes"], s["k_scales"] = _random_cache(gen, units, c["kv_heads"], rows, D)
        s["v_codes"], s["v_scales"] = _random_cache(gen, units, c["kv_heads"], rows, D)
    if own:
        _plan(s, c)
    return s


def _plan(s, c):
    """Outputs, descriptors and workspace of the library's calls, which a serving loop makes once and calls with each step."""
    import alpaca_b200 as ab

    if c["op"] == "append":
        S, T, D = c["seqs"], c["tokens"], c["head_dim"]
        s["q_out"] = torch.empty(s["q"].shape, dtype=DTYPES[c["q_type"]], device=DEV)
        rows = _up(c["start"] + T, 16)
        rope = dict(theta=THETA, interleaved=c["interleaved"], q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=EPS)
        if T == 1:
            rope["positions"] = s["positions"]
        else:
            rope["start_position"] = c["start"]
        if c["cache"] == "kv4":
            s["cache"] = ab.kv4_cache(S, rows, c["kv_heads"], D, device=DEV)
            s["k_out"], s["v_out"] = (torch.empty((S, T, c["kv_heads"], D), dtype=torch.float16, device=DEV) for _ in range(2))
            at = dict(row_starts=s["positions"]) if T == 1 else dict(start_row=c["start"])
            s["read"] = ab.make_kv4_read_desc(s["cache"], s["k_out"], s["v_out"], **at)
        else:
            s["cache"] = tuple(torch.zeros((S, rows, c["kv_heads"], D), dtype=torch.float16, device=DEV) for _ in range(2))
            s["k_out"], s["v_out"] = (x[:, c["start"]:c["start"] + T] for x in s["cache"])
        s["desc"] = ab.make_qkv_desc(s["q"], s["k"], s["v"], s["q_out"], s["cache"], **rope)
    elif c["op"] == "read":
        s["cache"] = ab.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
        s["k_out"], s["v_out"] = (torch.empty((c["seqs"], c["rows"], c["kv_heads"], c["head_dim"]), dtype=DTYPES[c["out_type"]], device=DEV)
                                  for _ in range(2))
        s["desc"] = ab.make_kv4_read_desc(s["cache"], s["k_out"], s["v_out"], start_row=0)
    else:
        s["cache"] = ab.Kv4Cache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
        s["out"] = torch.empty(s["q"].shape, dtype=DTYPES[c["out_type"]], device=DEV)
        where = dict(ctx_lens=s["lens"], max_ctx_len=c["ctx"]) if c["ragged"] else dict(start_position=c["ctx"] - c["tokens"])
        s["desc"] = ab.make_kv4_attn_desc(s["q"], s["cache"], s["out"], block_table=s["table"], **where)
        n = ab.kv4_workspace_bytes(s["desc"])
        s["ws"] = torch.empty(n, dtype=torch.uint8, device=DEV) if n else None


def _frequencies(head_dim):
    return THETA ** (-2.0 * torch.arange(head_dim // 2, device=DEV, dtype=torch.float64) / head_dim)


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    s, c = state, state["case"]
    if own:
        import alpaca_b200 as ab

        if c["op"] == "append":
            ab.qkv_launch(s["desc"])
            if c["cache"] == "kv4":
                ab.kv4_read_launch(s["read"])  # the rows just written, as the values they stand for
            return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}
        if c["op"] == "read":
            ab.kv4_read_launch(s["desc"])
            return {"k": s["k_out"], "v": s["v_out"]}
        ab.kv4_attention_launch(s["desc"], s["ws"])
        return s["out"]
    if c["op"] == "append":
        return _plain_append(s, c)
    if c["op"] == "read":
        kind = DTYPES[c["out_type"]]
        k, v = (_values(s[x + "_codes"], s[x + "_scales"])[:, :, : c["rows"]].transpose(1, 2).to(kind).contiguous() for x in "kv")
        return {"k": k, "v": v}
    return _plain_attend(s, c)


def work(case):
    c = case
    D = c["head_dim"]
    size = {"f16": 2, "f32": 4}
    row4 = D // 2 + D // 16  # bytes of one 4-bit head row
    if c["op"] == "append":
        n, kv = c["seqs"] * c["tokens"], 2 * c["kv_heads"]
        moved = n * D * (c["heads"] * (size[c["in_type"]] + size[c["q_type"]]) + kv * (size[c["in_type"]] + 2))
        if c["cache"] == "kv4":
            moved += n * kv * row4
        return {"bytes": moved, "flops": n * (c["heads"] + kv) * D * 10}
    if c["op"] == "read":
        n = 2 * c["seqs"] * c["rows"] * c["kv_heads"]
        return {"bytes": n * (row4 + D * size[c["out_type"]]), "flops": 2 * n * D}
    T, L = c["tokens"], c["ctx"]
    rows = c["seqs"] * ((L + 1) / 2 if c["ragged"] else L)  # ragged contexts are uniform in 1 .. ctx
    pairs = c["seqs"] * (T * (L + 1) / 2 if c["ragged"] else T * L - T * (T - 1) / 2)
    moved = rows * 2 * c["kv_heads"] * row4 + c["seqs"] * T * c["heads"] * D * (size[c["q_type"]] + size[c["out_type"]])
    return {"bytes": moved, "flops": 4.0 * pairs * c["heads"] * D}


# ------------------------------------------------------------------------------------------------ in 64 bits

def _exact_values(codes, scales):
    """Row values in f64, word by word and nibble by nibble."""
    blocks = scales.shape[-1]
    word = codes.contiguous().view(torch.int32)
    out = torch.empty((*codes.shape[:-1], blocks * 32), dtype=torch.float64, device=codes.device)
    for b in range(blocks):
        header = scales[..., b].to(torch.int32) & 0xFFFF
        zero = (header & 15).double()
        power, mantissa = (header >> 10) & 31, (header & 0x3F0).double()
        step = torch.where(power > 0, torch.ldexp(1.0 + mantissa / 1024.0, power - 15), mantissa * 2.0 ** -24)
        for t in range(4):
            for n in range(8):
                code = (word[..., t * blocks + b] >> (4 * n)) & 15
                out[..., 32 * b + 8 * t + n] = (code.double() - zero) * step
    return out


def _exact_quantised(x):
    """What f64 rows [..., d] become in the 4-bit cache."""
    y = x.unflatten(-1, (-1, 32))
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    lo, hi = torch.minimum(y.min(-1, keepdim=True).values, zero), torch.maximum(y.max(-1, keepdim=True).values, zero)
    step = torch.minimum((hi - lo) / 15, zero + 4352)
    unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -14))) - 6)  # 7 significant bits
    step = torch.ceil(step / unit) * unit
    safe = torch.where(step > 0, step, torch.ones_like(step))
    z = torch.round(-lo / safe).clamp(0, 15)
    return ((torch.round(y / safe) + z).clamp(0, 15).sub(z) * step).flatten(-2)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "append":
        q, k, v = (s[x].double() for x in "qkv")
        if c["norm"]:
            q = q / (q.square().mean(-1, keepdim=True) + EPS).sqrt() * s["q_norm"].double()
            k = k / (k.square().mean(-1, keepdim=True) + EPS).sqrt() * s["k_norm"].double()
        half = c["head_dim"] // 2
        position = s["positions"].double()[:, None] + torch.arange(c["tokens"], device=DEV)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), position[..., None] * _frequencies(c["head_dim"]))[:, :, None]
        done = []
        for x in (q, k):
            pair = x.unflatten(-1, (half, 2)) if c["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            done.append((y if c["interleaved"] else y.transpose(-1, -2)).flatten(-2))
        q, k = done
        if c["cache"] == "kv4":
            k, v = _exact_quantised(k), _exact_quantised(v)
        return {"q": q, "k": k, "v": v}
    if c["op"] == "read":
        return {x: _exact_values(s[x + "_codes"], s[x + "_scales"])[:, :, : c["rows"]].transpose(1, 2).contiguous() for x in "kv"}
    T, group = c["tokens"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lens = s["lens"].tolist()
    for i, n in enumerate(lens):
        if s["table"] is None:
            part = [s[x][i] for x in ("k_codes", "k_scales", "v_codes", "v_scales")]
        else:
            part = [torch.cat([s[x][j] for j in s["table"][i].tolist()], 1) for x in ("k_codes", "k_scales", "v_codes", "v_scales")]
        k, v = _exact_values(part[0][:, :n], part[1][:, :n]), _exact_values(part[2][:, :n], part[3][:, :n])
        hidden = torch.arange(n, device=DEV)[None] > (n - T + torch.arange(T, device=DEV))[:, None]
        first = max(0, T - n)  # tokens before this one see no row
        for h in range(c["heads"]):
            score = s["q"][i, :, h].double() @ k[h // group].T / math.sqrt(c["head_dim"])
            weight = score.masked_fill(hidden, -torch.inf)[first:].softmax(-1)
            out[i, first:, h] = weight @ v[h // group]
    return out
