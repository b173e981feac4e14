"""CPU tests of nsq_linear and nsq_moe_*: sizes, refusals before any launch,
and the plain reference that the GPU tests compare with."""
import ctypes
import os
import re

import pytest

from planejaja_b200 import _lib
from planejaja_b200.formats import Q4_0, Q4_K, Q5_K, Q6_K, Q8_0

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AL = 0x10000  # never dereferenced: every call below fails validation first
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from planejaja_b200.build import build
        build()
    return _lib.load()


def linear(lib, **kw):
    a = dict(w=AL, t=Q4_K, layout=0, x=AL, bias=AL, act=0, res=AL, y=AL, dtype=0, m=1, n=16, k=256, ws=AL, wsb=BIG)
    a.update(kw)
    return lib.nsq_linear(a["w"], a["t"], a["layout"], a["x"], a["bias"], a["act"], a["res"], a["y"], a["dtype"],
                          a["m"], a["n"], a["k"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("want,kw", [
    (_lib.ERR_TYPE, dict(t=3)), (_lib.ERR_TYPE, dict(t=Q5_K, layout=2)), (_lib.ERR_TYPE, dict(t=Q6_K, layout=-1)),
    (_lib.ERR_TYPE, dict(act=5)), (_lib.ERR_TYPE, dict(act=-1)), (_lib.ERR_TYPE, dict(dtype=2)),
    (_lib.ERR_NULL, dict(w=None)), (_lib.ERR_NULL, dict(x=None)), (_lib.ERR_NULL, dict(y=None)),
    (_lib.ERR_ALIGN, dict(w=AL + 8)), (_lib.ERR_ALIGN, dict(x=AL + 2)), (_lib.ERR_ALIGN, dict(y=AL + 1)),
    (_lib.ERR_ALIGN, dict(res=AL + 2)), (_lib.ERR_ALIGN, dict(bias=AL + 2)), (_lib.ERR_ALIGN, dict(ws=AL + 8)),
    (_lib.ERR_ALIGN, dict(dtype=1, x=AL + 1)),
    (_lib.ERR_SHAPE, dict(m=0)), (_lib.ERR_SHAPE, dict(m=-1)), (_lib.ERR_SHAPE, dict(m=17)),
    (_lib.ERR_SHAPE, dict(n=0)), (_lib.ERR_SHAPE, dict(n=1 << 25)), (_lib.ERR_SHAPE, dict(k=128)),
    (_lib.ERR_SHAPE, dict(t=Q8_0, k=48)), (_lib.ERR_SHAPE, dict(k=0)),
    (_lib.ERR_WORKSPACE, dict(ws=None)), (_lib.ERR_WORKSPACE, dict(m=3, k=512, wsb=3 * 2 * 880)),
])
def test_linear_refusals(lib, want, kw):
    assert linear(lib, **kw) == want


@pytest.mark.parametrize("kw", [
    dict(res=4 * AL - 4), dict(bias=4 * AL + 60), dict(ws=4 * AL), dict(x=8 * AL, ws=8 * AL), dict(ws=2 * AL, res=2 * AL),
    dict(m=17, dtype=1, x=4 * AL), dict(m=17, dtype=1, x=4 * AL + 512), dict(m=17, dtype=1, res=4 * AL + 2),
])
def test_linear_overlaps_are_refused(lib, kw):
    """Ranges that the product reads while it writes y: y [16] at 4 AL, everything else apart."""
    a = dict(x=AL, bias=2 * AL, res=None, y=4 * AL, ws=16 * AL, wsb=lib.nsq_linear_workspace_size(1, 256))
    a.update(kw)
    assert linear(lib, **a) == _lib.ERR_SHAPE


def test_linear_allowed_overlaps_pass_the_checks(lib):
    apart = dict(x=AL, bias=2 * AL, res=None, y=4 * AL, ws=16 * AL, wsb=lib.nsq_linear_workspace_size(1, 256))
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not the device's")
    for kw in (dict(), dict(res=4 * AL), dict(x=4 * AL), dict(res=4 * AL + 64), dict(m=17, dtype=1, res=4 * AL)):
        assert linear(lib, **dict(apart, **kw)) in (_lib.ERR_CUDA, _lib.ERR_DEVICE), kw


def test_linear_workspace_size(lib):
    # one record of 880 bytes per token and 256 of K (rounded up to 256), 8 tickets
    # and two parts of 8 row tiles of 32 (16 beyond 8 tokens) rows for 320 CTAs
    def size(m, k):
        return -(-m * -(-k // 256) * 880 // 256) * 256 + 320 * 8 * 4 + 320 * 2 * 8 * (16 if m > 8 else 32) * m * 4
    for m, k in ((1, 256), (4, 896), (5, 896), (16, 14336)):
        assert lib.nsq_linear_workspace_size(m, k) == size(m, k)
    assert lib.nsq_linear_workspace_size(17, 256) == 0
    assert lib.nsq_linear_workspace_size(0, 256) == 0


def moe(**kw):
    a = dict(w_gate=AL, w_up=AL, w_down=AL, type_in=Q4_K, layout_in=0, type_down=Q6_K, layout_down=0, act=1,
             n_expert=8, n_embd=512, n_ff=256)
    a.update(kw)
    return _lib.Moe(**a)


def ffn(lib, mo, **kw):
    a = dict(x=AL, ids=AL, wts=AL, res=AL, y=AL, m=2, k=2, ws=AL, wsb=BIG)
    a.update(kw)
    return lib.nsq_moe_ffn(ctypes.addressof(mo) if mo is not None else None, a["x"], a["ids"], a["wts"], a["res"],
                           a["y"], a["m"], a["k"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("want,mo,kw", [
    (_lib.ERR_TYPE, dict(type_in=3), {}), (_lib.ERR_TYPE, dict(type_down=0), {}), (_lib.ERR_TYPE, dict(act=9), {}),
    (_lib.ERR_TYPE, dict(layout_down=7), {}),
    (_lib.ERR_NULL, dict(w_gate=None), {}), (_lib.ERR_NULL, dict(w_up=None), {}), (_lib.ERR_NULL, dict(w_down=None), {}),
    (_lib.ERR_ALIGN, dict(w_up=AL + 4), {}),
    (_lib.ERR_SHAPE, dict(n_expert=0), {}), (_lib.ERR_SHAPE, dict(n_expert=513), {}), (_lib.ERR_SHAPE, dict(n_embd=300), {}),
    (_lib.ERR_SHAPE, dict(n_ff=96), {}), (_lib.ERR_SHAPE, dict(n_ff=0), {}),
    (_lib.ERR_SHAPE, {}, dict(m=0)), (_lib.ERR_SHAPE, {}, dict(m=65)), (_lib.ERR_SHAPE, {}, dict(k=0)),
    (_lib.ERR_SHAPE, {}, dict(k=9)), (_lib.ERR_SHAPE, dict(n_expert=64), dict(k=17)),
    (_lib.ERR_NULL, {}, dict(x=None)), (_lib.ERR_NULL, {}, dict(y=None)), (_lib.ERR_NULL, {}, dict(ids=None)),
    (_lib.ERR_NULL, {}, dict(wts=None)),
    (_lib.ERR_ALIGN, {}, dict(x=AL + 2)), (_lib.ERR_ALIGN, {}, dict(ids=AL + 1)), (_lib.ERR_ALIGN, {}, dict(ws=AL + 4)),
    (_lib.ERR_WORKSPACE, {}, dict(ws=None)), (_lib.ERR_WORKSPACE, {}, dict(wsb=100)),
])
def test_moe_refusals(lib, want, mo, kw):
    assert ffn(lib, moe(**mo), **kw) == want


@pytest.mark.parametrize("kw", [dict(res=4 * AL + 4), dict(wts=2 * AL + 4), dict(ids=4 * AL), dict(wts=4 * AL + 64),
                                dict(ws=AL), dict(ws=4 * AL), dict(ws=2 * AL), dict(ws=3 * AL), dict(res=64 * AL)])
def test_moe_overlaps_are_refused(lib, kw):
    a = dict(x=AL, ids=2 * AL, wts=3 * AL, res=None, y=4 * AL, ws=64 * AL)
    a.update(kw)
    assert ffn(lib, moe(), **a) == _lib.ERR_SHAPE


def test_moe_null_and_layer_refusals(lib):
    assert ffn(lib, None) == _lib.ERR_NULL
    m = moe()
    ref = ctypes.addressof(m)

    def layer(router=AL, score=0, bias=None):
        return lib.nsq_moe_layer(ref, router, score, bias, 1.0, AL, None, AL, AL, AL, 2, 2, AL, 100, None)
    assert layer(router=None) == _lib.ERR_NULL
    assert layer(score=3) == _lib.ERR_TYPE and layer(score=-1) == _lib.ERR_TYPE
    assert layer(router=AL + 2) == _lib.ERR_ALIGN and layer(bias=AL + 2) == _lib.ERR_ALIGN
    assert layer() == _lib.ERR_WORKSPACE


def test_moe_workspace_grows_with_every_size(lib):
    def size(m=2, k=2, **kw):
        mo = moe(**kw)
        return lib.nsq_moe_workspace_size(ctypes.addressof(mo), m, k)
    base = size()
    assert base > 0 and base % 256 == 0
    assert size(m=9) > base and size(k=8) > base and size(n_ff=1024) > base and size(n_embd=4096) > base
    assert size(m=65) == 0 and size(k=0) == 0 and size(n_expert=0) == 0
    assert lib.nsq_moe_workspace_size(None, 1, 1) == 0


def test_structs_and_constants_agree():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "nsq.h")).read(), flags=re.S)
    body = re.search(r"typedef struct nsq_moe\s*\{(.*?)\}", src, flags=re.S).group(1)
    fields = [f for line in body.split(";") for f in re.findall(r"\*?(\w+)\s*(?:,|$)", line.strip())]
    assert fields == [f for f, _ in _lib.Moe._fields_]
    rs = open(os.path.join(ROOT, "nodestor-cuda", "src", "ffi.rs")).read()
    assert fields == re.findall(r"pub (\w+):", re.search(r"pub struct NsqMoe\s*\{(.*?)\}", rs, flags=re.S).group(1))
    consts = {m.group(1): int(m.group(2)) for m in re.finditer(r"#define\s+(NSQ_[A-Z0-9_]+)\s+(-?\d+)\b", src)}
    for name, v in _lib.ACTS.items():
        assert consts["NSQ_ACT_" + name.upper()] == v
    for name, v in _lib.SCORES.items():
        assert consts["NSQ_SCORE_" + name.upper()] == v
    assert (consts["NSQ_MOE_MAX_TOKENS"], consts["NSQ_MOE_MAX_EXPERTS"], consts["NSQ_MOE_MAX_TOP_K"]) == (
        _lib.MOE_MAX_TOKENS, _lib.MOE_MAX_EXPERTS, _lib.MOE_MAX_TOP_K)
