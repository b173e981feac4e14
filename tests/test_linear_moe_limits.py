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
