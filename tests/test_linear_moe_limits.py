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


# ---------------------------------------------------------------- overlapping ranges
# Addresses that are never dereferenced: a range of A bytes for each tensor.
A = 1 << 32
NAMES = ["gate", "up", "down", "router", "bias", "x", "res", "y", "ids", "wts", "ws"]
PLACES = {n: (i + 1) * A for i, n in enumerate(NAMES)}
M, K, E, D, F = 3, 2, 8, 512, 256
ROW_IN, ROW_DOWN = 2 * 144, 210  # bytes of a row: Q4_K of 512, Q6_K of 256
SIZES = dict(gate=E * F * ROW_IN, up=E * F * ROW_IN, down=E * D * ROW_DOWN, router=E * D * 4, bias=E * 4, x=M * D * 4,
             res=M * D * 4, y=M * D * 4, ids=M * K * 4, wts=M * K * 4)


def moe_call(lib, given=False, **at):
    import ctypes
    a = dict(PLACES, **at)
    mo = _lib.Moe(a["gate"], a["up"], a["down"], 12, 0, 14, 0, 1, E, D, F)
    ref = ctypes.addressof(mo)
    size = lib.nsq_moe_workspace_size(ref, M, K)
    if given:
        return lib.nsq_moe_ffn(ref, a["x"], a["ids"], a["wts"], a["res"], a["y"], M, K, a["ws"], size, None)
    return lib.nsq_moe_layer(ref, a["router"], 0, a["bias"], 1.0, a["x"], a["res"], a["y"], a["ids"], a["wts"], M, K,
                             a["ws"], size, None)


def ends(lib, name):
    import ctypes
    mo = _lib.Moe(A, A, A, 12, 0, 14, 0, 1, E, D, F)
    size = SIZES.get(name) or lib.nsq_moe_workspace_size(ctypes.addressof(mo), M, K)
    return PLACES[name], PLACES[name] + (size - 1) // 16 * 16


# what a call writes, against everything else that it has: y may lie on x and on all of residual
PAIRS = [(w, o) for w in ("y", "ids", "wts", "ws") for o in NAMES if o != w and (w, o) != ("y", "x")]


@pytest.mark.parametrize("written,other", PAIRS)
def test_moe_layer_refuses_outputs_over_other_tensors(lib, written, other):
    """On the first and on the last 16 bytes of the other tensor."""
    first, last = ends(lib, other)
    for at in ((last,) if (written, other) == ("y", "res") else (first, last)):
        assert moe_call(lib, **{written: at}) == _lib.ERR_SHAPE, (written, other, at)


@pytest.mark.parametrize("other", [n for n in NAMES if n not in ("ws", "router", "bias")])
def test_moe_ffn_refuses_its_workspace_and_output_over_other_tensors(lib, other):
    for at in ends(lib, other):
        assert moe_call(lib, given=True, ws=at) == _lib.ERR_SHAPE, other
        if other not in ("x", "y") and (other, at) != ("res", PLACES["res"]):
            assert moe_call(lib, given=True, y=at) == _lib.ERR_SHAPE, other


def passes(status):
    return status in (_lib.ERR_CUDA, _lib.ERR_DEVICE)


def test_moe_allowed_overlaps_pass_the_checks(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not the device's")
    p = PLACES
    for kw in (dict(), dict(y=p["x"]), dict(y=p["x"] + 16), dict(y=p["res"]), dict(res=p["x"], y=p["x"]), dict(res=None),
               dict(res=p["x"]), dict(bias=None), dict(bias=p["router"]), dict(gate=p["up"]), dict(x=p["router"])):
        assert passes(moe_call(lib, **kw)), kw
    for kw in (dict(), dict(y=p["x"]), dict(y=p["res"]), dict(ids=p["x"]), dict(wts=p["x"]), dict(wts=p["res"])):
        assert passes(moe_call(lib, given=True, **kw)), kw


def linear_call(lib, m=1, n=512, k=512, t=12, dtype=0, **at):
    a = dict(w=A, x=2 * A, bias=3 * A, res=4 * A, y=5 * A, ws=6 * A)
    a.update(at)
    return lib.nsq_linear(a["w"], t, 0, a["x"], a["bias"], 0, a["res"], a["y"], dtype, m, n, k, a["ws"],
                          lib.nsq_linear_workspace_size(min(m, 16), k), None)


def test_linear_refuses_outputs_over_its_weights(lib):
    import torch
    last = A + 512 * ROW_IN - 16
    for at in (A, last):
        assert linear_call(lib, ws=at) == _lib.ERR_SHAPE
        for m, dtype in ((1, 0), (16, 1), (17, 1)):
            assert linear_call(lib, m, dtype=dtype, y=at) == _lib.ERR_SHAPE, (m, at)
    if not torch.cuda.is_available():
        assert passes(linear_call(lib)) and passes(linear_call(lib, ws=last + 16)) and passes(linear_call(lib, y=last + 16))
        assert passes(linear_call(lib, 17, dtype=1, ws=A))  # no workspace is used


# ---------------------------------------------------------------- shapes
class Dev(Bytes):
    """A tensor on a GPU as the host checks see it."""

    def __init__(self, *shape, dtype=None):
        import torch
        n = 1
        for s in shape:
            n *= s
        super().__init__(0, n)
        self.shape, self.dtype = torch.Size(shape), dtype or torch.float32

    def dim(self):
        return len(self.shape)

    def new_empty(self, shape, dtype=None):
        return Dev(*shape, dtype=dtype or self.dtype)


class Calls:
    """libnsq that takes every call and does nothing."""

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def fake(monkeypatch):
    import torch
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    return engine_on("cuda:0", Calls()), dict(workspace=Dev(1 << 20, dtype=torch.uint8), sync=False)


def test_linear_refuses_transposed_tensors(fake):
    eng, kw = fake
    w, k, n = Bytes(0), 256, 16

    def call(x=Dev(3, 256), residual=None, out=None, n=n):
        return eng.linear(x, w, 12, n, k, residual=residual, out=out, **kw)
    for bad in (dict(x=Dev(256, 3)), dict(x=Dev(2, 256, 3)), dict(residual=Dev(16, 3)), dict(out=Dev(16, 3)),
                dict(residual=Dev(4, 3, 4)), dict(x=Dev(6, 128))):
        assert status_of(call, **bad) == _lib.ERR_SHAPE, list(bad.values())[0].shape
    for good in (dict(), dict(x=Dev(768)), dict(x=Dev(3, 1, 256)), dict(x=Dev(3, 2, 128)), dict(residual=Dev(3, 16)),
                 dict(residual=Dev(3, 4, 4)), dict(residual=Dev(1, 48)), dict(residual=Dev(48)),
                 dict(residual=Dev(1, 3, 16), out=Dev(48)), dict(x=Dev(256)), dict(x=Dev(256, 1), residual=Dev(16, 1)),
                 dict(x=Dev(1, 256), residual=Dev(1, 16)), dict(n=1, residual=Dev(1, 3)), dict(x=Dev(256), n=1, residual=Dev())):
        call(**good)


def test_moe_refuses_transposed_tensors(fake):
    import torch
    eng, kw = fake
    moe = experts_of()
    ids = Dev(4, 2, dtype=torch.int32)

    def ffn(x=Dev(4, 256), weights=Dev(4, 2), residual=None, out=None, ids=ids):
        return eng.moe_ffn(moe, x, ids, weights, residual=residual, out=out, **kw)

    def layer(x=Dev(4, 256), router=Dev(2, 256), residual=None, out=None):
        return eng.moe_layer(moe, router, x, 2, residual=residual, out=out, **kw)
    for call in (ffn, layer):
        for bad in (dict(x=Dev(256, 4)), dict(residual=Dev(256, 4)), dict(out=Dev(256, 4)), dict(out=Dev(2, 512))):
            assert status_of(call, **bad) == _lib.ERR_SHAPE, bad
        for good in (dict(), dict(x=Dev(2, 2, 256)), dict(x=Dev(1024)), dict(residual=Dev(1024), out=Dev(4, 1, 256))):
            call(**good)
    assert status_of(ffn, weights=Dev(2, 4)) == _lib.ERR_SHAPE
    assert status_of(layer, router=Dev(256, 2)) == _lib.ERR_SHAPE
    ffn(weights=Dev(8))
    ffn(weights=Dev(4, 2, dtype=torch.float32))
    layer(router=Dev(512))
    ffn(x=Dev(256), ids=Dev(1, 2, dtype=torch.int32), weights=Dev(2))
