"""Prefill calls enqueued behind other work: the work list and the partial records that one launch of a call writes
and the next one reads are read after they are written, whatever the workspace held before."""
from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

H, HKV = 8, 2


def _behind_other_work(launch, workspace, out, busy):
    """`out` of a call that is enqueued on a cleared workspace while the device is still busy with earlier work."""
    workspace.zero_()
    out.fill_(7.0)
    torch.cuda.synchronize()
    for _ in range(4):
        busy.mul_(1.0)
    launch()
    torch.cuda.synchronize()
    return out.clone()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("lens,starts", [([300, 1, 128, 129, 700, 512, 37], [0, 517, 128, 1000, 33, 1536, 0]),  # unsplit
                                         ([100, 60], [1500, 900])])  # split KV and its merge
def test_ragged(cuda_lib, d, q_dtype, lens, starts):
    from alpaca_b200 import Kernel, device_status, ops
    gen = torch.Generator(device="cuda").manual_seed(5 + d)
    ctx, total = max(a + b for a, b in zip(lens, starts)), sum(lens)
    q = torch.randn((total, H, d), generator=gen, device="cuda").to(q_dtype)
    k, v = (torch.randn((len(lens), ctx, HKV, d), generator=gen, device="cuda").half() for _ in range(2))
    offs = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    first = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out = torch.empty((total, H, d), dtype=torch.float32, device="cuda")
    desc = ops.make_varlen_desc(q, k, v, out, offs, first, max_tokens=max(lens), max_ctx_len=ctx)
    ws = torch.zeros(ops.workspace_bytes(desc, Kernel.PREFILL_TC), dtype=torch.uint8, device="cuda")
    busy = torch.zeros(1 << 26, device="cuda")
    got = [_behind_other_work(lambda: ops.launch(desc, Kernel.PREFILL_TC, ws), ws, out, busy) for _ in range(3)]
    device_status()
    o = 0
    for s, (n, p) in enumerate(zip(lens, starts)):  # 64-bit: queries rounded to f16 as the kernel takes them
        qs = q[o:o + n].half().double().transpose(0, 1)
        ks, vs = (x[s, :p + n].double().repeat_interleave(H // HKV, 1).transpose(0, 1) for x in (k, v))
        scores = qs @ ks.transpose(1, 2) / d ** 0.5
        later = torch.arange(p + n, device="cuda")[None, :] > p + torch.arange(n, device="cuda")[:, None]
        want = (scores.masked_fill(later, float("-inf")).softmax(-1) @ vs).transpose(0, 1)
        for g in got:
            assert (g[o:o + n].double() - want).abs().max().item() < 2e-3, f"sequence {s}"
        o += n


@pytest.mark.parametrize("d", [64, 128])
def test_uniform_split(cuda_lib, d):
    """A chunk with few work items: KV parts and their merge."""
    from alpaca_b200 import Kernel, device_status, ops
    gen = torch.Generator(device="cuda").manual_seed(9 + d)
    n, p = 128, 2000
    q = torch.randn((1, n, H, d), generator=gen, device="cuda").half()
    k, v = (torch.randn((1, p + n, HKV, d), generator=gen, device="cuda").half() for _ in range(2))
    out = torch.empty((1, n, H, d), dtype=torch.float32, device="cuda")
    desc = ops.make_desc(q, k, v, out, start_position=p)
    ws = torch.zeros(ops.workspace_bytes(desc, Kernel.PREFILL_TC), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    busy = torch.zeros(1 << 26, device="cuda")
    got = [_behind_other_work(lambda: ops.launch(desc, Kernel.PREFILL_TC, ws), ws, out, busy) for _ in range(3)]
    device_status()
    qs = q[0].double().transpose(0, 1)
    ks, vs = (x[0].double().repeat_interleave(H // HKV, 1).transpose(0, 1) for x in (k, v))
    later = torch.arange(p + n, device="cuda")[None, :] > p + torch.arange(n, device="cuda")[:, None]
    want = ((qs @ ks.transpose(1, 2) / d ** 0.5).masked_fill(later, float("-inf")).softmax(-1) @ vs).transpose(0, 1)
    for g in got:
        assert (g[0].double() - want).abs().max().item() < 2e-3
