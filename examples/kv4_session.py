"""A chat session's attention over the 4-bit KV cache, step by step, next to the same session over the f16 cache.

Per layer and step a model does: new tokens' projections -> head norms + RoPE + cache append (one pass) -> attention over the
cache. Here the projections are seeded random numbers of a SmolLM2-135M layer's shape; the prompt goes through in chunks, then
tokens one by one. Prints the caches' bytes, the time of a decode step as this loop issues it (at these sizes mostly the host's:
descriptors and launches), and how far the 4-bit session's context vectors are from the f16 session's.

    python examples/kv4_session.py [--prompt 1000] [--tokens 32] [--chunk 512] [--layers 4]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import alpaca_b200 as ab  # noqa: E402

HEADS, KV_HEADS, HEAD_DIM, THETA = 9, 3, 64, 10000.0


class Session:
    """One sequence's caches of `layers` layers, 4-bit or f16, and the two calls that advance it."""

    def __init__(self, layers: int, rows: int, four_bit: bool, norms):
        self.four_bit, self.norms = four_bit, norms
        if four_bit:
            self.caches = [ab.kv4_cache(1, rows, KV_HEADS, HEAD_DIM) for _ in range(layers)]
        else:
            self.caches = [tuple(torch.zeros((1, rows, KV_HEADS, HEAD_DIM), dtype=torch.float16, device="cuda") for _ in range(2))
                           for _ in range(layers)]
        self.position = 0
        self.workspace = None  # of the attention calls: the largest asked for so far, shared by the layers

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for c in self.caches for t in c)

    def step(self, qkv):
        """Appends the new tokens' rows of every layer and attends: qkv[layer] = (q, k, v) f32 -> context vectors f16."""
        outs = []
        for cache, (q, k, v) in zip(self.caches, qkv):
            q_rot = torch.empty(q.shape, dtype=torch.float16, device="cuda")
            ab.qkv_append(q, k, v, q_rot, cache, theta=THETA, start_position=self.position, q_norm=self.norms[0], k_norm=self.norms[1])
            out = torch.empty_like(q_rot)
            if self.four_bit:
                desc = ab.make_kv4_attn_desc(q_rot, cache, out, start_position=self.position)
                need = ab.kv4_workspace_bytes(desc)
                if self.workspace is None or self.workspace.nbytes < need:
                    self.workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
                ab.kv4_attention_launch(desc, self.workspace)
            else:
                ab.attention_device(q_rot, cache[0], cache[1], out, start_position=self.position)
            outs.append(out)
        self.position += qkv[0][0].shape[1]
        return outs


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--prompt", type=int, default=1000)
    p.add_argument("--tokens", type=int, default=32)
    p.add_argument("--chunk", type=int, default=512)
    p.add_argument("--layers", type=int, default=4)
    a = p.parse_args(argv)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)

    def rows(n, heads):
        return torch.randn((1, n, heads, HEAD_DIM), generator=gen, device="cuda")

    norms = [1 + 0.1 * torch.randn(HEAD_DIM, generator=gen, device="cuda") for _ in range(2)]
    total = a.prompt + a.tokens
    sessions = {"4-bit": Session(a.layers, total, True, norms), "f16": Session(a.layers, total, False, norms)}
    error = norm = 0.0
    start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    spent = dict.fromkeys(sessions, 0.0)
    at = 0
    while at < total:
        n = min(a.chunk, a.prompt - at) if at < a.prompt else 1
        qkv = [(rows(n, HEADS), rows(n, KV_HEADS), rows(n, KV_HEADS)) for _ in range(a.layers)]
        outs = {}
        for name, s in sessions.items():
            start.record()
            outs[name] = s.step(qkv)
            stop.record()
            stop.synchronize()
            if at > a.prompt:  # the first decode step warms up
                spent[name] += start.elapsed_time(stop)
        for x, y in zip(outs["4-bit"], outs["f16"]):
            error += float((x.float() - y.float()).square().sum())
            norm += float(y.float().square().sum())
        at += n
    ab.device_status()
    result = {"relative_error": (error / norm) ** 0.5, "bytes": {n: s.bytes() for n, s in sessions.items()}}
    for name, s in sessions.items():
        print(f"{name:>6}: {s.bytes() / 2 ** 20:.2f} MiB of cache, {1e3 * spent[name] / max(1, a.tokens - 1) / a.layers:.1f} us a layer and decode step")
    print(f"4-bit against f16 context vectors: relative error {result['relative_error']:.3f}")
    return result


if __name__ == "__main__":
    main()
