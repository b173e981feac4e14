"""GPU tests of nsq_linear and the mixture-of-experts layer against a plain
implementation in 64 bits over the oracle's dequantised weights.

Tolerances (up to 16 tokens).  An activation is an integer below 2^23 times
one scale per 256 of K: off by at most 2^-24 of the largest of its 256; the
formats' integers are exact, sums are s32 and then f32.  With A = sum_k |x_k|
(|w_k| + 2 o_k), o the offset part of a weight (the weight whose quant bits
are 0), the f32 part passes at most 17 additions within a unit, nsb units and
16 joins, each off by at most 2^-23 of a partial sum <= A:
  |y - r| <= (2 * 2^-22 + 2^-23 (17 + nsb + 16)) A                (element)
The activations' roundings are independent.  Here (normal values, one in a
hundred 50 times as large: largest <= 200, mean size of all >= 1) they add up
to a deviation of 2^-24 * 200 sqrt(256 / 3) = 2^-24 * 1850 of a weight per
unit, a ninth of the bound's 2^-24 * (8 + 66) * 246 of a weight.  As a norm
that is 2^-24 * 1850 / (16 * 5) = 1.4e-6 of the result, and the f32 part
2^-23 sqrt(33 + nsb) / 2 <= 6e-7 of parts up to 3 times the result: 5e-6 is
asked of one product, 1e-5 of the two of an expert.  A bf16 result adds half
a step, at most 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

from planejaja_b200 import _lib
from planejaja_b200 import quantize as Q
from planejaja_b200.formats import FORMATS, Q4_0, Q4_K, Q5_K, Q6_K, Q8_0

pytestmark = pytest.mark.gpu

ALL = [(Q4_0, 0), (Q8_0, 0), (Q4_K, 0), (Q5_K, 0), (Q5_K, 1), (Q6_K, 0), (Q6_K, 1)]
IDS = ["Q4_0", "Q8_0", "Q4_K", "Q5_K", "Q5_K_nodestor", "Q6_K", "Q6_K_nodestor"]
ONE, TWO = 5e-6, 1e-5


@pytest.fixture(scope="module")
def eng():
    from planejaja_b200.engine import CudaEngine
    e = CudaEngine(0)
    yield e
    assert e.device_status() == 0


def blocks(n, k, t, seed, std=0.02):
    """Random block bytes with scales of every sign and size the formats hold."""
    f = FORMATS[t]
    r = np.random.default_rng(seed)
    b = r.integers(0, 256, (n * k // f.block_weights, f.block_bytes), np.uint8)

    def half(lo, hi):
        return (r.uniform(lo, hi, b.shape[0]) * std).astype(np.float16).view(np.uint8).reshape(-1, 2)
    if t == Q6_K:
        b[:, 208:210] = half(-1 / 900, 1 / 900)
    elif t in (Q4_K, Q5_K):
        b[:, 0:2] = half(0, 1 / 80)
        b[:, 2:4] = half(0, 1 / 20)
    else:
        b[:, 0:2] = half(-0.4, 0.4) if t == Q4_0 else half(0, 0.03)
    return b.reshape(-1)


def offsets(raw, t):
    """The same blocks with quant bits of value 0."""
    b = raw.reshape(-1, FORMATS[t].block_bytes).copy()
    if t == Q8_0:
        b[:, 2:] = 0x80
    elif t == Q4_0:
        b[:, 2:] = 0
    elif t == Q6_K:
        b[:, :192] = 0
    else:
        b[:, 16:] = 0
    return b.reshape(-1)


def dequant(oracle, raw, t, layout, n, k):
    return oracle.dequant(raw, t, layout).reshape(n, k).astype(np.float64)


def act64(v, name):
    if name == "silu":
        return v / (1 + np.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(torch.from_numpy(v / np.sqrt(2))).numpy())
    if name == "gelu_tanh":
        return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    return np.maximum(v, 0) if name == "relu" else v


def norm_err(y, r):
    return float(np.linalg.norm(y - r) / max(np.linalg.norm(r), 1e-300))


def activations(m, k, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((m, k)).astype(np.float32)
    x[:, r.random(k) < 0.01] *= 50
    x *= 10.0 ** r.integers(-3, 4, (m, 1))
    return x.astype(np.float32)


# ---------------------------------------------------------------- linear
@pytest.mark.parametrize("m", [1, 2, 4, 5, 11, 16])
@pytest.mark.parametrize("t,layout", ALL, ids=IDS)
def test_linear_plain_product(eng, oracle, t, layout, m):
    for n, k in ((37, 256), (200, 2048), (5, 4864), (300, 416 if t in (Q4_0, Q8_0) else 768)):
        raw, x = blocks(n, k, t, 7 * m + k), activations(m, k, k + m)
        y = eng.linear(torch.from_numpy(x).cuda(), eng.upload(raw), t, n, k, q6k_layout=layout).double().cpu().numpy()
        w = dequant(oracle, raw, t, layout, n, k)
        o = np.abs(dequant(oracle, offsets(raw, t), t, layout, n, k))
        r = x.astype(np.float64) @ w.T
        a = np.abs(x).astype(np.float64) @ (np.abs(w) + 2 * o).T
        nsb = -(-k // 256)
        assert np.all(np.abs(y - r) <= (2 * 2.0 ** -22 + 2.0 ** -23 * (33 + nsb)) * a), (n, k)
        for i in range(m):  # tokens differ by orders of magnitude: each on its own
            assert norm_err(y[i], r[i]) <= ONE, (n, k, i, norm_err(y[i], r[i]))


@pytest.mark.parametrize("t,layout", ALL, ids=IDS)
def test_linear_one_hot_reads_every_weight(eng, oracle, t, layout):
    """x = unit vectors: y is the dequantised column, exact but for the last roundings."""
    n, k = 19, 512
    raw = blocks(n, k, t, 3)
    w = dequant(oracle, raw, t, layout, n, k)
    o = np.abs(dequant(oracle, offsets(raw, t), t, layout, n, k))
    wd = eng.upload(raw)
    for k0 in range(0, k, 16):
        x = np.zeros((16, k), np.float32)
        x[np.arange(16), k0 + np.arange(16)] = 1.0
        y = eng.linear(torch.from_numpy(x).cuda(), wd, t, n, k, q6k_layout=layout).double().cpu().numpy()
        c = slice(k0, k0 + 16)
        # two parts, each exact, one f32 subtraction and the token scale: a few half steps
        assert np.all(np.abs(y - w[:, c].T) <= 2.0 ** -22 * (np.abs(w[:, c]) + 2 * o[:, c]).T), k0


@pytest.mark.parametrize("act", sorted(_lib.ACTS))
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_linear_epilogue(eng, oracle, act, dtype):
    dt = torch.float32 if dtype == "f32" else torch.bfloat16
    for m, n, k, t, bias, res in ((1, 77, 1024, Q4_K, True, True), (7, 130, 896, Q8_0, True, False),
                                  (16, 48, 512, Q6_K, False, True)):
        r = np.random.default_rng(m)
        raw = blocks(n, k, t, 5)
        x = torch.from_numpy(r.standard_normal((m, k)).astype(np.float32)).to(dt)
        b = torch.from_numpy(r.standard_normal(n).astype(np.float32)) if bias else None
        s = torch.from_numpy(r.standard_normal((m, n)).astype(np.float32)).to(dt) if res else None
        cuda = lambda v: None if v is None else v.cuda()  # noqa: E731
        y = eng.linear(x.cuda(), eng.upload(raw), t, n, k, bias=cuda(b), act=act, residual=cuda(s))
        assert y.dtype == dt
        v = x.double().numpy() @ dequant(oracle, raw, t, 0, n, k).T
        v = act64(v if b is None else v + b.double().numpy(), act)
        v = v if s is None else v + s.double().numpy()
        err = np.abs(y.double().cpu().numpy() - v)
        # f32: the product's 5e-6 of its norm (rms ~ |v|), the activation's own 4 * 2^-24 and its slope <= 1.13
        tol = 2e-5 * max(1.0, float(np.sqrt(np.mean(v * v))))
        assert np.all(err <= tol + (2.0 ** -8 * np.abs(v) if dtype == "bf16" else 0)), (m, act, err.max())


def test_linear_in_place_residual_out_and_strides(eng, oracle):
    m, n, k = 3, 64, 512
    raw = blocks(n, k, Q4_K, 9)
    w = eng.upload(raw)
    big = torch.randn(m, 2 * k, device="cuda")
    x = big[:, ::2]  # not contiguous
    res = torch.randn(m, n, device="cuda")
    want = eng.linear(x.contiguous(), w, Q4_K, n, k, residual=res)
    y = res.clone()
    got = eng.linear(x, w, Q4_K, n, k, residual=y, out=y)
    assert got.data_ptr() == y.data_ptr() and torch.equal(got, want)
    # pointers that are only 4-byte aligned
    xs = torch.empty(m * k + 1, device="cuda")[1:].copy_(x.reshape(-1)).reshape(m, k)
    out = torch.empty(m * n + 1, device="cuda")[1:].reshape(m, n)
    assert xs.data_ptr() % 16 == 4
    assert torch.equal(eng.linear(xs, w, Q4_K, n, k, residual=res, out=out), want)


def test_linear_extreme_activations(eng, oracle):
    """Zeros, the largest and smallest floats, and a token of NaN or infinity that leaves the others alone."""
    n, k = 40, 512
    raw = blocks(n, k, Q4_K, 1)
    w = dequant(oracle, raw, Q4_K, 0, n, k)
    r = np.random.default_rng(0)
    x = r.standard_normal((8, k)).astype(np.float32)
    x[1] = 0
    x[2] *= np.float32(1e34)
    x[3] *= np.float32(1e-34)
    x[4, 7] = np.nan
    x[5, 300] = np.inf
    x[6, 1:] = 0
    y = eng.linear(torch.from_numpy(x).cuda(), eng.upload(raw), Q4_K, n, k).double().cpu().numpy()
    assert np.all(y[1] == 0)
    assert not np.isfinite(y[4]).any() and not np.isfinite(y[5]).any()
    for i in (0, 2, 3, 6, 7):
        assert norm_err(y[i], x[i].astype(np.float64) @ w.T) <= ONE, i


def test_linear_repeats_bit_for_bit_and_other_streams(eng):
    raw = blocks(4096, 4096, Q4_K, 2)
    w = eng.upload(raw)
    x = torch.randn(5, 4096, device="cuda")
    y = eng.linear(x, w, Q4_K, 4096, 4096)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = [eng.linear(x, w, Q4_K, 4096, 4096, sync=False) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(v, y) for v in z)


@pytest.mark.parametrize("m,n,k,t", [(1, 896, 896, Q8_0), (3, 512, 512, Q4_K), (16, 4096, 4096, Q4_K), (2, 2048, 2048, Q6_K)])
def test_linear_output_over_its_input(eng, m, n, k, t):
    w = eng.upload(blocks(n, k, t, 4))
    x = torch.randn(m, k, device="cuda")
    want = eng.linear(x, w, t, n, k, act="silu", residual=x)
    got = eng.linear(x, w, t, n, k, act="silu", residual=x, out=x)
    assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)


def test_linear_calls_side_by_side(eng):
    """Four streams, their kernels on the GPU at once: small, divided and whole tasks, prompts; each its own workspace."""
    calls = []
    for i, (m, n, k, t) in enumerate(((1, 1152, 896, Q8_0), (1, 4096, 14336, Q6_K), (16, 2048, 4096, Q4_K), (40, 512, 1024, Q5_K))):
        w = eng.upload(blocks(n, k, t, i))
        x = torch.randn(m, k, device="cuda")
        x = x.bfloat16() if m > 16 else x
        calls.append((torch.cuda.Stream(), x, w, t, n, k, eng.linear(x, w, t, n, k, act="gelu")))
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, x, w, t, n, k, want in calls:
            with torch.cuda.stream(s):
                got.append((eng.linear(x, w, t, n, k, act="gelu", sync=False), want))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y, want in got)


def test_linear_captured_with_one_workspace(eng):
    """Two graphs that share a workspace, replayed in turn over changing inputs."""
    n, k = 512, 1024
    ws = eng.linear_workspace(16, n, k)
    sides = []
    for t, m in ((Q4_K, 2), (Q8_0, 16)):
        w, x = eng.upload(blocks(n, k, t, t)), torch.randn(m, k, device="cuda")
        res = torch.randn(m, n, device="cuda")
        eng.linear(x, w, t, n, k, residual=res, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = eng.linear(x, w, t, n, k, residual=res, act="silu", workspace=ws, sync=False)
        sides.append((g, w, x, res, t, y))
    for i in range(6):
        g, w, x, res, t, y = sides[i % 2]
        x.copy_(torch.randn_like(x))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eng.linear(x, w, t, n, k, residual=res, act="silu"))


def bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a)).float().bfloat16().double().numpy()


def prompt_bound(x, w, bias, act, residual):
    """The product over weights rounded to bf16, in 64 bits, and what a bf16 result may be off by: the f32 sums
    truncate at most once per 16 products and once per joined part (2^-23 of at most A = |x| . |w| each), the
    activation's slope is at most 1.13 and its own error below 2^-20 of the sum, and the result is rounded once."""
    v = x @ w.T
    b = np.zeros(w.shape[0]) if bias is None else bias
    e = 1.13 * 2.0 ** -23 * (x.shape[1] / 16 + 4) * (np.abs(x) @ np.abs(w).T + np.abs(b))
    e = e + 2.0 ** -20 * np.abs(v + b)
    v = act64(v + b, act)
    v = v if residual is None else v + residual
    return v, e + 2.0 ** -8 * (np.abs(v) + e)


@pytest.mark.parametrize("t,layout", ALL, ids=IDS)
@pytest.mark.parametrize("m,n,k", [
    (17, 1, 256),        # one output row, one column of K
    (100, 129, 1280),    # a tile of one row; K splits of unequal length
    (129, 300, 512),     # 256-token tiles, two of them
    (600, 257, 2304),    # 256-token tiles again (few weight rows), split K
])
def test_linear_of_prompts(eng, oracle, t, layout, m, n, k):
    r = np.random.default_rng(m + n)
    raw = blocks(n, k, t, m)
    x, b, s = (bf16(r.standard_normal(sh) * sc) for sh, sc in (((m, k), 1.0), (n, 1.0), ((m, n), 1.0)))
    c = lambda a: torch.from_numpy(a).cuda().bfloat16()  # noqa: E731
    act = ("none", "silu", "gelu", "gelu_tanh", "relu")[(m + t) % 5]
    wd = eng.upload(raw)
    w = bf16(dequant(oracle, raw, t, layout, n, k))
    y = eng.linear(c(x), wd, t, n, k, bias=torch.from_numpy(b).float().cuda(), act=act, residual=c(s),
                   q6k_layout=layout).double().cpu().numpy()
    v, tol = prompt_bound(x, w, b, act, s)
    assert np.all(np.abs(y - v) <= tol), (act, float((np.abs(y - v) / tol).max()))
    # without an epilogue: nsq_gemm_bf16's product (K may be split at other places)
    v, tol = prompt_bound(x, w, None, "none", None)
    for y in (eng.linear(c(x), wd, t, n, k, q6k_layout=layout), eng.gemm_bf16(wd, t, c(x), n, k, q6k_layout=layout)):
        assert np.all(np.abs(y.reshape(m, n).double().cpu().numpy() - v) <= tol)


@pytest.mark.parametrize("act", sorted(_lib.ACTS))
def test_linear_of_prompts_every_epilogue(eng, oracle, act):
    """512-token tiles without a K split and small ones with: each activation, with and without bias and residual."""
    for m, n, k in ((513, 4900, 256), (40, 70, 1536)):
        r = np.random.default_rng(m)
        raw = blocks(n, k, Q4_K, m)
        wd, w = eng.upload(raw), bf16(dequant(oracle, raw, Q4_K, 0, n, k))
        x, b, s = bf16(3 * r.standard_normal((m, k))), bf16(r.standard_normal(n)), bf16(r.standard_normal((m, n)))
        for bias, res in ((b, s), (b, None), (None, s), (None, None)):
            t = lambda a, d: None if a is None else torch.from_numpy(a).cuda().to(d)  # noqa: E731
            y = eng.linear(t(x, torch.bfloat16), wd, Q4_K, n, k, bias=t(bias, torch.float32), act=act,
                           residual=t(res, torch.bfloat16)).double().cpu().numpy()
            v, tol = prompt_bound(x, w, bias, act, res)
            assert np.all(np.abs(y - v) <= tol), (m, act, float((np.abs(y - v) / tol).max()))


def test_linear_of_prompts_in_place_rows_behind_and_captured(eng):
    m, n, k = 333, 1003, 2816
    wd = eng.upload(blocks(n, k, Q8_0, 6))
    x = torch.randn(m, k, device="cuda").bfloat16()
    bias = torch.randn(n, device="cuda")
    big = torch.randn(m + 8, n, device="cuda").bfloat16()
    before = big.clone()
    want = eng.linear(x, wd, Q8_0, n, k, bias=bias, act="relu", residual=before[:m].contiguous())
    eng.linear(x, wd, Q8_0, n, k, bias=bias, act="relu", residual=big[:m], out=big[:m])
    assert torch.equal(big[:m], want) and torch.equal(big[m:], before[m:])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = eng.linear(x, wd, Q8_0, n, k, bias=bias, act="relu", residual=before[:m], sync=False)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    x[7, 3] = float("nan")
    z = eng.linear(x, wd, Q8_0, n, k, bias=bias, act="relu", residual=before[:m])
    keep = [i for i in range(m) if i != 7]
    assert torch.equal(z[keep], want[keep]) and torch.isnan(z[7]).all()
    for kw, status in ((dict(x=x.float()), _lib.ERR_SHAPE), (dict(x=x.reshape(-1)[1:1 + 32 * k].reshape(32, k)), _lib.ERR_ALIGN),
                       (dict(k=2784, x=x[:, :2784].contiguous()), _lib.ERR_SHAPE)):
        a = dict(x=x, w=wd, ggml_type=Q8_0, n=n, k=k)
        a.update(kw)
        with pytest.raises(_lib.NsqError) as e:
            eng.linear(**a)
        assert e.value.status == status, list(kw)


def test_linear_refusals(eng):
    w = eng.upload(blocks(16, 256, Q4_K, 0))
    x = torch.zeros(2, 256, device="cuda")
    for kw, status in ((dict(x=x.half()), _lib.ERR_TYPE), (dict(act="tanh"), _lib.ERR_TYPE), (dict(ggml_type=3), _lib.ERR_TYPE),
                       (dict(bias=torch.zeros(15, device="cuda")), _lib.ERR_SHAPE), (dict(n=17), _lib.ERR_SHAPE),
                       (dict(bias=torch.zeros(16, device="cuda").bfloat16()), _lib.ERR_TYPE),
                       (dict(residual=torch.zeros(2, 16, device="cuda").bfloat16()), _lib.ERR_TYPE),
                       (dict(residual=torch.zeros(16, device="cuda")), _lib.ERR_SHAPE), (dict(x=x.cpu()), _lib.ERR_TYPE),
                       (dict(out=torch.zeros(16, 2, device="cuda").t()), _lib.ERR_SHAPE),
                       (dict(x=torch.zeros(17, 256, device="cuda")), _lib.ERR_SHAPE),
                       (dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")), _lib.ERR_WORKSPACE)):
        a = dict(x=x, w=w, ggml_type=Q4_K, n=16, k=256)
        a.update(kw)
        with pytest.raises(_lib.NsqError) as e:
            eng.linear(**a)
        assert e.value.status == status, kw


# ---------------------------------------------------------------- mixture of experts
class Layer:
    def __init__(self, eng, oracle, e, d, f, t_in, t_down, lay_in=0, lay_down=0, act="silu", seed=1):
        from planejaja_b200.engine import MoeExperts
        self.e, self.d, self.f, self.act = e, d, f, act
        raws = [blocks(e * f, d, t_in, seed), blocks(e * f, d, t_in, seed + 1), blocks(e * d, f, t_down, seed + 2)]
        self.wg, self.wu = (dequant(oracle, r, t_in, lay_in, e * f, d).reshape(e, f, d) for r in raws[:2])
        self.wd = dequant(oracle, raws[2], t_down, lay_down, e * d, f).reshape(e, d, f)
        self.moe = MoeExperts(*(eng.upload(r) for r in raws), e, d, f, t_in, t_down, layout_in=lay_in,
                              layout_down=lay_down, act=act)

    def ffn(self, x, ids, wts, residual=None):
        y = np.zeros((x.shape[0], self.d)) if residual is None else residual.astype(np.float64).copy()
        x = x.astype(np.float64)
        for m in range(x.shape[0]):
            for j, e in enumerate(ids[m]):
                if 0 <= e < self.e:
                    h = act64(self.wg[e] @ x[m], self.act) * (self.wu[e] @ x[m])
                    y[m] += float(wts[m, j]) * (self.wd[e] @ h)
        return y


def picks(e, m, k, seed):
    r = np.random.default_rng(seed)
    ids = np.stack([r.permutation(e)[:k] for _ in range(m)]).astype(np.int32)
    return ids, r.random((m, k)).astype(np.float32) + 0.1


@pytest.mark.parametrize("t,layout", ALL, ids=IDS)
@pytest.mark.parametrize("m", [1, 3, 17])
def test_moe_ffn_every_format(eng, oracle, t, layout, m):
    e, k = 5, 3
    d, f = (352, 288) if t in (Q4_0, Q8_0) else (512, 768)
    ly = Layer(eng, oracle, e, d, f, t, t, layout, layout)
    ids, wts = picks(e, m, k, m)
    x = np.random.default_rng(m).standard_normal((m, d)).astype(np.float32)
    y = eng.moe_ffn(ly.moe, *(torch.from_numpy(v).cuda() for v in (x, ids, wts))).double().cpu().numpy()
    r = ly.ffn(x, ids, wts)
    for i in range(m):
        assert norm_err(y[i], r[i]) <= TWO, (i, norm_err(y[i], r[i]))


@pytest.mark.parametrize("e,m,k,d,f,t_in,t_down,act", [
    (1, 1, 1, 256, 32, Q4_K, Q8_0, "silu"),       # one expert, one block of K
    (2, 64, 2, 256, 256, Q8_0, Q4_K, "gelu"),     # every expert for the most tokens: groups of 16
    (16, 64, 16, 288, 96, Q4_0, Q4_0, "relu"),    # the most picks
    (512, 6, 8, 256, 256, Q4_0, Q6_K, "silu"),    # the most experts
    (7, 33, 1, 1024, 1376, Q5_K, Q8_0, "gelu_tanh"),
    (3, 2, 2, 2048, 3840, Q6_K, Q5_K, "none"),
    (512, 64, 16, 256, 256, Q5_K, Q4_K, "silu"),  # the most of everything
])
def test_moe_ffn_sizes(eng, oracle, e, m, k, d, f, t_in, t_down, act):
    ly = Layer(eng, oracle, e, d, f, t_in, t_down, act=act)
    ids, wts = picks(e, m, k, 11)
    x = np.random.default_rng(3).standard_normal((m, d)).astype(np.float32)
    res = np.random.default_rng(4).standard_normal((m, d)).astype(np.float32) * 1e-3
    y = eng.moe_ffn(ly.moe, *(torch.from_numpy(v).cuda() for v in (x, ids, wts, res))).double().cpu().numpy()
    r = ly.ffn(x, ids, wts, res)
    for i in range(m):
        assert norm_err(y[i], r[i]) <= TWO, (i, norm_err(y[i], r[i]))


def test_moe_ffn_unused_slots_empty_tokens_and_repeats(eng, oracle):
    ly = Layer(eng, oracle, 6, 256, 256, Q4_K, Q4_K)
    m, k = 9, 4
    ids, wts = picks(6, m, k, 2)
    ids[0] = -1                      # a token without experts
    ids[1, 2:] = -1
    ids[2] = [6, 99, -5, 2 ** 30]    # none of them an expert
    ids[3] = [4, 4, 4, 4]            # one expert four times
    ids[4] = [1, 0, 1, 0]
    x = np.random.default_rng(3).standard_normal((m, 256)).astype(np.float32)
    dev = [torch.from_numpy(v).cuda() for v in (x, ids, wts)]
    y = eng.moe_ffn(ly.moe, *dev)
    r = ly.ffn(x, ids, wts)
    got = y.double().cpu().numpy()
    assert np.all(got[0] == 0) and np.all(got[2] == 0)
    for i in (1, 3, 4, 5, 6, 7, 8):
        assert norm_err(got[i], r[i]) <= TWO, i
    res = torch.randn(m, 256, device="cuda")
    out = res.clone()
    eng.moe_ffn(ly.moe, *dev, residual=out, out=out)
    assert torch.equal(out[0], res[0]) and torch.equal(out[2], res[2])
    # nobody has an expert
    dev[1].fill_(-1)
    assert torch.equal(eng.moe_ffn(ly.moe, *dev, residual=res), res)


def test_moe_ffn_bad_token_stays_alone(eng, oracle):
    ly = Layer(eng, oracle, 4, 256, 256, Q4_K, Q6_K)
    ids, wts = picks(4, 6, 2, 5)
    x = np.random.default_rng(3).standard_normal((6, 256)).astype(np.float32)
    dev = [torch.from_numpy(v).cuda() for v in (x, ids, wts)]
    y = eng.moe_ffn(ly.moe, *dev).clone()
    dev[0][2, 5] = float("nan")
    z = eng.moe_ffn(ly.moe, *dev)
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(y[keep], z[keep]) and not torch.isfinite(z[2]).any()


def reference_route(x, wr, score, bias, scale, k):
    l = x.astype(np.float64) @ wr.astype(np.float64).T
    if score == "sigmoid_norm":
        s = 1 / (1 + np.exp(-l))
    else:
        s = np.exp(l - l.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
    by = s if bias is None else s + bias.astype(np.float64)
    ids = np.argsort(-by, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(s, ids, 1)
    if score != "softmax":
        w = w / w.sum(1, keepdims=True)
    return ids.astype(np.int32), w * scale


@pytest.mark.parametrize("score", sorted(_lib.SCORES))
@pytest.mark.parametrize("bias", [False, True])
def test_moe_layer_routes_and_computes(eng, oracle, score, bias):
    for e, m, k, scale in ((8, 1, 2, 1.0), (60, 13, 6, 2.5), (100, 40, 4, 1.0)):
        ly = Layer(eng, oracle, e, 256, 256, Q4_0, Q4_K)
        r = np.random.default_rng(e)
        x = r.standard_normal((m, 256)).astype(np.float32)
        wr = (r.standard_normal((e, 256)) / 16).astype(np.float32)
        b = (0.1 * r.standard_normal(e)).astype(np.float32) if bias else None
        cuda = lambda v: None if v is None else torch.from_numpy(v).cuda()  # noqa: E731
        y, ids, wts = eng.moe_layer(ly.moe, cuda(wr), cuda(x), k, score=score, sel_bias=cuda(b), scale=scale)
        ri, rw = reference_route(x, wr, score, b, scale, k)
        assert np.array_equal(ids.cpu().numpy(), ri)
        # f64 inside, rounded once
        assert np.all(np.abs(wts.double().cpu().numpy() - rw) <= 2.0 ** -23 * rw)
        want = ly.ffn(x, ri, rw)
        got = y.double().cpu().numpy()
        for i in range(m):
            assert norm_err(got[i], want[i]) <= TWO, i
        assert torch.equal(y, eng.moe_ffn(ly.moe, cuda(x), ids, wts))


def test_moe_layer_ties_go_to_the_lowest_id(eng, oracle):
    ly = Layer(eng, oracle, 40, 256, 256, Q4_0, Q4_0)
    wr = np.zeros((40, 256), np.float32)
    wr[33] = wr[7] = 0.1
    x = np.abs(np.random.default_rng(0).standard_normal((3, 256))).astype(np.float32)
    x[2] = 0  # every logit the same
    for score in _lib.SCORES:
        _, ids, _ = eng.moe_layer(ly.moe, torch.from_numpy(wr).cuda(), torch.from_numpy(x).cuda(), 4, score=score)
        assert ids.cpu().tolist() == [[7, 33, 0, 1], [7, 33, 0, 1], [0, 1, 2, 3]], score


def test_moe_layer_close_logits(eng, oracle):
    """Router rows that differ in the last bit of one entry: f64 sums tell them apart."""
    ly = Layer(eng, oracle, 4, 1024, 256, Q4_0, Q4_0)
    r = np.random.default_rng(1)
    row = r.standard_normal(1024).astype(np.float32)
    x = r.standard_normal((1, 1024)).astype(np.float32)
    x[0, 500] = 0.25
    row[500] = 0.5
    wr = np.stack([row] * 4)
    for e, up in ((0, 1), (1, 3), (2, 0), (3, 2)):
        for _ in range(up):
            wr[e, 500] = np.nextafter(wr[e, 500], np.float32(1))
    _, ids, _ = eng.moe_layer(ly.moe, torch.from_numpy(wr).cuda(), torch.from_numpy(x).cuda(), 4)
    assert ids.cpu().tolist() == [[1, 3, 0, 2]]


def test_moe_layer_nan_scores_still_pick_experts(eng, oracle):
    ly = Layer(eng, oracle, 8, 256, 256, Q4_0, Q4_0)
    x = torch.randn(3, 256, device="cuda")
    wr = torch.randn(8, 256, device="cuda")
    x[1] = float("nan")
    for score in _lib.SCORES:
        y, ids, wts = eng.moe_layer(ly.moe, wr, x, 3, score=score)
        assert sorted(set(ids[1].tolist())) == [0, 1, 2]
        assert torch.isfinite(y[[0, 2]]).all() and not torch.isfinite(y[1]).any()


def test_moe_layer_captured_and_on_another_stream(eng, oracle):
    ly = Layer(eng, oracle, 8, 512, 512, Q4_K, Q6_K)
    x, wr = torch.randn(4, 512, device="cuda"), torch.randn(8, 512, device="cuda")
    res = torch.randn(4, 512, device="cuda")
    ws = eng.moe_workspace(ly.moe, 4, 2)
    eng.moe_layer(ly.moe, wr, x, 2, residual=res, workspace=ws)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, ids, wts = eng.moe_layer(ly.moe, wr, x, 2, residual=res, workspace=ws, sync=False)
    for i in range(4):
        x.copy_(torch.randn_like(x))
        g.replay()
        torch.cuda.synchronize()
        want = eng.moe_layer(ly.moe, wr, x, 2, residual=res)
        assert torch.equal(y, want[0]) and torch.equal(ids, want[1]) and torch.equal(wts, want[2])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        z = eng.moe_layer(ly.moe, wr, x, 2, residual=res, sync=False)[0]
    torch.cuda.synchronize()
    assert torch.equal(z, y)


def test_moe_calls_side_by_side(eng, oracle):
    """A layer on two streams at once, each call with a workspace of its own."""
    ly = Layer(eng, oracle, 16, 512, 1024, Q4_K, Q4_K)
    wr = torch.randn(16, 512, device="cuda")
    xs = [torch.randn(m, 512, device="cuda") for m in (1, 24)]
    want = [eng.moe_layer(ly.moe, wr, x, 4) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, eng.moe_layer(ly.moe, wr, xs[i], 4, sync=False)))
    torch.cuda.synchronize()
    for i, g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_a_decoder_block_of_these_operators(eng, oracle):
    """Attention's output projection with bias and residual, then the layer on the stream, then the next q|k|v."""
    d, e, k, f, m = 512, 8, 2, 768, 6
    r = np.random.default_rng(8)
    raw_o, raw_q = blocks(d, d, Q4_K, 31), blocks(d + 256, d, Q8_0, 32)
    ly = Layer(eng, oracle, e, d, f, Q4_K, Q6_K, seed=40)
    att, stream = (r.standard_normal((m, d)).astype(np.float32) for _ in range(2))
    bo, bq = r.standard_normal(d).astype(np.float32), r.standard_normal(d + 256).astype(np.float32)
    wr = (r.standard_normal((e, d)) / 30).astype(np.float32)
    c = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    s = c(stream)
    eng.linear(c(att), eng.upload(raw_o), Q4_K, d, d, bias=c(bo), residual=s, out=s, sync=False)
    y, ids, wts = eng.moe_layer(ly.moe, c(wr), s, k, residual=s, sync=False)
    q = eng.linear(y, eng.upload(raw_q), Q8_0, d + 256, d, bias=c(bq))
    s64 = stream + att.astype(np.float64) @ dequant(oracle, raw_o, Q4_K, 0, d, d).T + bo
    ri, rw = reference_route(s64, wr, "softmax_norm", None, 1.0, k)
    assert np.array_equal(ids.cpu().numpy(), ri)
    y64 = ly.ffn(s64, ri, rw, s64)
    q64 = y64 @ dequant(oracle, raw_q, Q8_0, 0, d + 256, d).T + bq
    assert norm_err(s.double().cpu().numpy(), s64) <= ONE
    # errors pass on through weights of norm <~ 1 per product
    assert norm_err(y.double().cpu().numpy(), y64) <= 2 * TWO
    assert norm_err(q.double().cpu().numpy(), q64) <= 3 * TWO


def test_moe_refusals(eng, oracle):
    from planejaja_b200.engine import MoeExperts
    ly = Layer(eng, oracle, 4, 256, 256, Q4_0, Q4_0)
    x, ids = torch.zeros(2, 256, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    wts = torch.zeros(2, 2, device="cuda")
    for a, status in (((x.bfloat16(), ids, wts), _lib.ERR_TYPE), ((x, ids.long(), wts), _lib.ERR_TYPE),
                      ((x[:1], ids, wts), _lib.ERR_SHAPE), ((x, ids, wts[:1]), _lib.ERR_SHAPE),
                      ((x, ids[0], wts), _lib.ERR_SHAPE), ((x.cpu(), ids, wts), _lib.ERR_TYPE)):
        with pytest.raises(_lib.NsqError) as err:
            eng.moe_ffn(ly.moe, *a)
        assert err.value.status == status
    for kw, status in ((dict(top_k=5), _lib.ERR_SHAPE), (dict(top_k=0), _lib.ERR_SHAPE), (dict(score="max"), _lib.ERR_TYPE),
                       (dict(sel_bias=torch.zeros(5, device="cuda")), _lib.ERR_SHAPE),
                       (dict(workspace=torch.empty(64, dtype=torch.uint8, device="cuda")), _lib.ERR_WORKSPACE)):
        a = dict(top_k=2)
        a.update(kw)
        with pytest.raises(_lib.NsqError) as err:
            eng.moe_layer(ly.moe, torch.zeros(4, 256, device="cuda"), x, **a)
        assert err.value.status == status, kw
    w = ly.moe
    for a, status in (((w.w_gate[:-1], w.w_up, w.w_down, 4, 256, 256, Q4_0, Q4_0), _lib.ERR_SHAPE),
                      ((w.w_gate, w.w_up, w.w_down, 4, 250, 256, Q4_0, Q4_0), _lib.ERR_SHAPE),
                      ((w.w_gate, w.w_up, w.w_down, 4, 256, 256, 7, Q4_0), _lib.ERR_TYPE),
                      ((w.w_gate.cpu(), w.w_up, w.w_down, 4, 256, 256, Q4_0, Q4_0), _lib.ERR_TYPE)):
        with pytest.raises(_lib.NsqError) as err:
            MoeExperts(*a)
        assert err.value.status == status
