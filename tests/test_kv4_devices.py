"""The 4-bit cache calls and the device that their tensors live on, without a GPU: the kernels follow raw addresses, so a
descriptor of host tensors must not be made and a launch with a workspace elsewhere must not reach the library."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class Library:
    """Stands for the loaded library: counts the calls that reach it."""
    calls = 0

    def __getattr__(self, name):
        def call(*args):
            Library.calls += 1
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    from alpaca_b200 import ops
    Library.calls = 0
    monkeypatch.setattr(ops, "load", Library)
    return Library


def refused(call, match):
    import alpaca_b200 as ab
    with pytest.raises(ab.AlpacaCUDAError, match=match) as e:
        call()
    assert e.value.status == ab.Status.INVALID_ARGUMENT


def test_descriptors_of_host_tensors_are_refused():
    import alpaca_b200 as ab
    cache = ab.kv4_cache(2, 32, 2, 64, device="cpu")
    rows = tuple(torch.empty(2, 8, 2, 64) for _ in range(2))
    q, k = torch.zeros((2, 3, 4, 64)), torch.zeros((2, 3, 2, 64))
    for call in (lambda: ab.make_qkv_desc(q, k, k.clone(), torch.empty_like(q), cache, theta=1e4),
                 lambda: ab.make_qkv_desc(q, None, None, torch.empty_like(q), None, theta=1e4),
                 lambda: ab.make_qkv_desc(None, k, k.clone(), None, rows, theta=1e4),
                 lambda: ab.make_kv4_read_desc(cache, k, k.clone()),
                 lambda: ab.make_kv4_attn_desc(q, cache, torch.empty_like(q))):
        refused(call, "one CUDA device")


def test_a_workspace_elsewhere_is_refused(library):
    import alpaca_b200 as ab
    desc = ab.Kv4AttnDesc()
    desc.device = 0  # as made from tensors on cuda:0
    refused(lambda: ab.kv4_attention_launch(desc, torch.empty(64, dtype=torch.uint8)), "workspace")
    assert library.calls == 0


class Stream:
    """What the launches read of a torch.cuda.Stream."""
    def __init__(self, device):
        self.device_index, self.cuda_stream = device, 77


def launches():
    import alpaca_b200 as ab
    return [(ab.QkvDesc, ab.qkv_launch), (ab.Kv4ReadDesc, ab.kv4_read_launch),
            (ab.Kv4AttnDesc, lambda d, stream=None: ab.kv4_attention_launch(d, stream=stream))]


@pytest.mark.parametrize("i", range(3))
def test_a_call_away_from_its_tensors_is_refused(library, monkeypatch, i):
    """The library launches on the current device; the device index is stubbed."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 55, raising=False)
    make, launch = launches()[i]
    desc = make()
    desc.device = 1
    refused(lambda: launch(desc), "cuda:0 is current")
    refused(lambda: launch(desc, stream=Stream(1)), "cuda:0 is current")
    desc.device = 0
    refused(lambda: launch(desc, stream=Stream(1)), "stream on cuda:1")
    assert library.calls == 0
    launch(desc)
    launch(desc, stream=Stream(0))
    launch(make())  # a descriptor filled by hand names no device
    assert library.calls == 3


def test_no_workspace_is_allocated_for_a_refused_call(library, monkeypatch):
    from alpaca_b200 import ops
    import alpaca_b200 as ab
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(ops, "kv4_workspace_bytes", lambda *a: 1 / 0)
    desc = ab.Kv4AttnDesc()
    desc.device = 1
    refused(lambda: ops._kv4_run(desc, ab.Kernel.AUTO, None, "cuda:1", None), "cuda:0 is current")
    assert library.calls == 0
