"""CPU tests of what nsq_linear, the experts' layer and their Python calls
promise about workspaces, devices, overlapping ranges and shapes."""
import os

import pytest

from planejaja_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from planejaja_b200.build import build
        build()
    return _lib.load()


# ---------------------------------------------------------------- workspaces
@pytest.mark.parametrize("k", [32, 256, 896, 4096, 14336, 1 << 20])
def test_linear_workspace_never_shrinks_with_the_tokens(lib, k):
    """A workspace of m tokens serves every smaller call."""
    sizes = [lib.nsq_linear_workspace_size(m, k) for m in range(1, _lib.GEMV_MAX_M + 1)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])), sizes


def test_linear_workspace_never_shrinks_with_k(lib):
    ks = [32 * i for i in range(1, 80)] + [1 << i for i in range(12, 25)]
    for m in range(1, _lib.GEMV_MAX_M + 1):
        sizes = [lib.nsq_linear_workspace_size(m, k) for k in ks]
        assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:])), m


def test_linear_workspace_of_a_prompt_serves_decode_calls(lib):
    """CudaEngine.linear_workspace: calls of up to m tokens, prompts (which need none) among them."""
    import torch
    from planejaja_b200.engine import CudaEngine
    eng = object.__new__(CudaEngine)
    eng.lib, eng.device = lib, torch.device("cpu")
    for m in (17, 512):
        assert eng.linear_workspace(m, 64, 1024).numel() >= lib.nsq_linear_workspace_size(16, 1024)
    for m in range(1, 17):
        assert eng.linear_workspace(m, 64, 1024).numel() == lib.nsq_linear_workspace_size(m, 1024)


def moe_size(lib, m, top_k, e=8, d=512, f=512):
    import ctypes
    mo = _lib.Moe(0x10000, 0x10000, 0x10000, 12, 0, 12, 0, 1, e, d, f)
    return lib.nsq_moe_workspace_size(ctypes.addressof(mo), m, top_k)


@pytest.mark.parametrize("e", [1, 2, 7, 8, 60, 512])
def test_moe_workspace_never_shrinks(lib, e):
    """With the tokens and with the picks of each: one made for the largest call serves the others."""
    for top_k in range(1, _lib.MOE_MAX_TOP_K + 1):
        sizes = [moe_size(lib, m, top_k, e) for m in range(1, _lib.MOE_MAX_TOKENS + 1)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), (top_k, sizes)
    for m in range(1, _lib.MOE_MAX_TOKENS + 1):
        sizes = [moe_size(lib, m, top_k, e) for top_k in range(1, _lib.MOE_MAX_TOP_K + 1)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), (m, sizes)


# ---------------------------------------------------------------- devices
class Bytes:
    """GGUF bytes on a GPU that this machine need not have: what the host checks look at, and nothing behind it."""

    def __init__(self, device, n=1 << 20):
        import torch
        self.dtype, self.device, self.is_cuda, self.n = torch.uint8, torch.device("cuda", device), True, n

    def get_device(self):
        return self.device.index

    def is_contiguous(self):
        return True

    def numel(self):
        return self.n

    def data_ptr(self):
        return 0x10000


class NoCalls:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


def engine_on(device, lib=None):
    import torch
    from planejaja_b200.engine import CudaEngine
    eng = object.__new__(CudaEngine)
    eng.lib, eng.device = lib or NoCalls(), torch.device(device)
    return eng


def status_of(fn, *a, **kw):
    with pytest.raises(_lib.NsqError) as e:
        fn(*a, **kw)
    return e.value.status


def experts_of(gate=0, up=0, down=0):
    from planejaja_b200.engine import MoeExperts
    return MoeExperts(Bytes(gate), Bytes(up), Bytes(down), 2, 256, 256, 12, 12)


def test_linear_refuses_weights_on_another_device():
    import torch
    x = torch.zeros(2, 256)  # its own refusal (no CUDA tensor) comes after the weights'
    assert status_of(engine_on("cuda:0").linear, x, Bytes(1), 12, 16, 256) == _lib.ERR_DEVICE
    assert status_of(engine_on("cuda:1").linear, x, Bytes(0), 12, 16, 256) == _lib.ERR_DEVICE
    assert status_of(engine_on("cuda:1").linear, x, Bytes(1), 12, 16, 256) == _lib.ERR_TYPE


def test_an_engine_of_no_device_runs_on_the_current_one(monkeypatch):
    import torch
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    x = torch.zeros(2, 256)
    assert status_of(engine_on("cuda").linear, x, Bytes(0), 12, 16, 256) == _lib.ERR_DEVICE
    assert status_of(engine_on("cuda").linear, x, Bytes(1), 12, 16, 256) == _lib.ERR_TYPE
    other = Bytes(0, 512)
    other.dtype = torch.float32
    assert status_of(engine_on("cuda")._tensor, other, 512, torch.float32, "x") == _lib.ERR_DEVICE


@pytest.mark.parametrize("where", [(0, 1, 0), (0, 0, 1), (1, 0, 0)])
def test_experts_lie_on_one_device(where):
    assert status_of(experts_of, *where) == _lib.ERR_DEVICE


def test_experts_of_another_device_are_refused(lib):
    import torch
    x, ids, wts, router = torch.zeros(2, 256), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1), torch.zeros(2, 256)
    here, there = experts_of(), experts_of(1, 1, 1)
    eng = engine_on("cuda:0")
    for call in (lambda m: eng.moe_ffn(m, x, ids, wts), lambda m: eng.moe_layer(m, router, x, 1)):
        assert status_of(call, there) == _lib.ERR_DEVICE
        assert status_of(call, here) == _lib.ERR_TYPE  # x is no CUDA tensor
    assert status_of(eng.moe_workspace, there, 2, 1) == _lib.ERR_DEVICE
