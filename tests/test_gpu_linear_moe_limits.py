"""GPU tests of nsq_linear and the experts' layer at the limits of what their
documentation allows: kept workspaces, odd edges, routers of every size,
alignments, and the launch-planning switches."""
import numpy as np
import pytest
import torch

from planejaja_b200 import _lib
from planejaja_b200 import quantize as Q
from planejaja_b200.formats import FORMATS, Q4_0, Q4_K, Q5_K, Q6_K, Q8_0
from test_gpu_linear_moe import act64, bf16, reference_route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from planejaja_b200.engine import CudaEngine
    e = CudaEngine(0)
    yield e
    assert e.device_status() == 0


@pytest.mark.parametrize("t", [Q4_K, Q8_0])
def test_linear_kept_workspace_serves_smaller_calls(eng, t):
    """A workspace made for m tokens and k, used by every smaller call: with divided tasks (512 rows) and without."""
    for n, k in ((512, 1024), (4096, 512)):
        w = eng.upload(Q.synthetic_weights(n, k, t, seed=n))
        x = torch.randn(16, k, device="cuda")
        want = [eng.linear(x[:m].contiguous(), w, t, n, k) for m in range(1, 17)]
        for made_for in (9, 12, 15, 16, 40):
            ws = eng.linear_workspace(made_for, n, k)
            for m in range(1, min(made_for, 16) + 1):
                y = eng.linear(x[:m].contiguous(), w, t, n, k, workspace=ws)
                assert torch.equal(y, want[m - 1]), (made_for, m)



def prompt_reference(oracle, raw, t, n, k, x, bias, act, residual, parts):
    """nsq_linear for prompts in 64 bits over weights rounded to bf16, and what a bf16 result may be off by.

    The f32 sums truncate at most once per 16 products and once per joined part, 2^-23 of at most A = |x| . |w|
    each; the activations' slopes are at most 1.13 and their own errors below 2^-20 of the sum; the result is
    rounded once, by at most 2^-8 of itself."""
    w = bf16(oracle.dequant(raw, t, 0).reshape(n, k))
    v = x @ w.T + bias
    e = 1.13 * 2.0 ** -23 * (k / 16 + parts) * (np.abs(x) @ np.abs(w).T + np.abs(bias)) + 2.0 ** -20 * np.abs(v)
    v = act64(v, act) + residual
    return v, e + 2.0 ** -8 * (np.abs(v) + e)


@pytest.mark.parametrize("tok", [128, 256, 512])
@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
def test_prompts_with_lanes_behind_the_last_row(eng, oracle, tuning, tok, split):
    """N that ends inside a warp's 32 rows, every activation: warps meet again before each load and barrier of theirs."""
    tuning.set("NSQ_GEMM_TOK", tok)
    tuning.set("NSQ_GEMM_SPLIT", split)
    m, k = 70, 2048
    for n in (1, 45, 129, 1003):
        r = np.random.default_rng(n + split)
        raw = Q.synthetic_weights(n, k, Q4_K, seed=n)
        w = eng.upload(raw)
        x, b, s = bf16(r.standard_normal((m, k))), bf16(r.standard_normal(n)), bf16(r.standard_normal((m, n)))
        xd, sd = torch.from_numpy(x).cuda().bfloat16(), torch.from_numpy(s).cuda().bfloat16()
        bd = torch.from_numpy(b).cuda().float()
        for act in sorted(_lib.ACTS):
            y = eng.linear(xd, w, Q4_K, n, k, bias=bd, act=act, residual=sd).double().cpu().numpy()
            v, tol = prompt_reference(oracle, raw, Q4_K, n, k, x, b, act, s, split)
            assert np.all(np.abs(y - v) <= tol), (n, act, float((np.abs(y - v) / tol).max()))
        y = eng.gemm_bf16(w, Q4_K, xd, n, k).double().cpu().numpy()
        v, tol = prompt_reference(oracle, raw, Q4_K, n, k, x, 0 * b, "none", 0 * s, split)
        assert np.all(np.abs(y - v) <= tol), n


# ---------------------------------------------------------------- mixture of experts
def experts(eng, e, d, f, t_in, t_down, seed=0):
    from planejaja_b200.engine import MoeExperts
    w = [eng.upload(Q.synthetic_weights(e * n, k, t, seed=seed + i))
         for i, (n, k, t) in enumerate(((f, d, t_in), (f, d, t_in), (d, f, t_down)))]
    return MoeExperts(*w, e, d, f, t_in, t_down)


def test_moe_kept_workspace_serves_smaller_calls(eng):
    """One made for 17 tokens of 2 picks: groups of 16 there, of up to 8 for fewer tokens."""
    e, d, f = 8, 512, 768
    moe = experts(eng, e, d, f, Q4_K, Q4_K)
    x, wr = torch.randn(17, d, device="cuda"), torch.randn(e, d, device="cuda")
    ws = eng.moe_workspace(moe, 17, 2)
    for m, k in ((17, 2), (16, 2), (9, 1), (17, 1), (8, 2), (1, 1), (16, 1)):
        want = eng.moe_layer(moe, wr, x[:m].contiguous(), k)
        got = eng.moe_layer(moe, wr, x[:m].contiguous(), k, workspace=ws)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (m, k)


def test_divided_tasks_joined_by_many_ctas_repeat(eng, tuning):
    """Every task divided, its parts and rows of h read by the last CTA to arrive: the same bits each time."""
    tuning.set("NSQ_QMM_SPLIT", 1)
    for t, m, e, d, f in ((Q4_K, 24, 8, 512, 2048), (Q8_0, 5, 4, 1056, 992), (Q6_K, 2, 16, 768, 1280)):
        moe = experts(eng, e, d, f, t, Q8_0 if t == Q8_0 else Q4_K)
        x, wr = torch.randn(m, d, device="cuda"), torch.randn(e, d, device="cuda")
        ws = eng.moe_workspace(moe, m, 3)
        want = eng.moe_layer(moe, wr, x, 3, workspace=ws)
        got = [eng.moe_layer(moe, wr, x, 3, workspace=ws, sync=False)[0] for _ in range(50)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[0]) for y in got), t
        n = 640
        w = eng.upload(Q.synthetic_weights(n, d, t, seed=9))
        x = x[:16].contiguous()
        want = eng.linear(x, w, t, n, d)
        got = [eng.linear(x, w, t, n, d, sync=False) for _ in range(50)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in got), t


def test_shapes_that_hold_the_rows_otherwise(eng):
    """Flat tensors, heads x size for a row, and the refusals of transposed ones, on the GPU's own tensors."""
    n, k = 48, 512
    w = eng.upload(Q.synthetic_weights(n, k, Q4_K, seed=2))
    x, res = torch.randn(6, k, device="cuda"), torch.randn(6, n, device="cuda")
    want = eng.linear(x, w, Q4_K, n, k, residual=res)
    for a, b in ((x.reshape(-1), res.reshape(-1)), (x.reshape(6, 4, 128), res.reshape(6, 3, 16)),
                 (x.reshape(2, 3, k), res.reshape(2, 3, n))):
        assert torch.equal(eng.linear(a, w, Q4_K, n, k, residual=b), want)
    heads = torch.randn(4, 6, 128, device="cuda").transpose(0, 1)  # not contiguous
    assert torch.equal(eng.linear(heads, w, Q4_K, n, k), eng.linear(heads.reshape(6, k), w, Q4_K, n, k))
    for bad in (dict(x=x.t().contiguous()), dict(residual=res.t().contiguous()), dict(residual=res.t()),
                dict(out=torch.empty(n, 6, device="cuda"))):
        with pytest.raises(_lib.NsqError) as e:
            eng.linear(**dict(dict(x=x, w=w, ggml_type=Q4_K, n=n, k=k), **bad))
        assert e.value.status == _lib.ERR_SHAPE, list(bad)


# ---------------------------------------------------------------- launch-planning switches
@pytest.mark.parametrize("split", [0, 1])
@pytest.mark.parametrize("kw", [1, 2, 4, 8])
def test_switches_change_the_plan_and_not_the_result(eng, oracle, tuning, kw, split):
    """Columns of K and the division of tasks set by hand, where the rings of 8 columns fit and where they do not
    (9 to 16 tokens).  5e-6 and 1e-5 of the norm, as for the planner's own choices: the sums only meet in another
    order, at most 8 columns and one part per unit."""
    tuning.set("NSQ_QMM_KW", kw)
    tuning.set("NSQ_QMM_SPLIT", split)
    for t, k in ((Q4_K, 2048), (Q5_K, 1280), (Q6_K, 768), (Q4_0, 992), (Q8_0, 4096)):
        n = 150
        raw = Q.synthetic_weights(n, k, t, seed=k)
        w, w64 = eng.upload(raw), oracle.dequant(raw, t, 0).reshape(n, k).astype(np.float64)
        for m in (1, 3, 8, 16):
            x = np.random.default_rng(m).standard_normal((m, k)).astype(np.float32)
            y = eng.linear(torch.from_numpy(x).cuda(), w, t, n, k).double().cpu().numpy()
            r = x.astype(np.float64) @ w64.T
            assert np.linalg.norm(y - r) <= 5e-6 * np.linalg.norm(r), (t, m)
    for m, e, d, f, t in ((2, 4, 512, 768, Q4_K), (40, 4, 256, 1024, Q8_0), (11, 6, 1056, 352, Q4_0)):
        moe = experts(eng, e, d, f, t, t)
        g, u, dn = (oracle.dequant(v.cpu().numpy()[:], t, 0).astype(np.float64) for v in (moe.w_gate, moe.w_up, moe.w_down))
        g, u, dn = g.reshape(e, f, d), u.reshape(e, f, d), dn.reshape(e, d, f)
        r = np.random.default_rng(m)
        x = r.standard_normal((m, d)).astype(np.float32)
        ids = np.stack([r.permutation(e)[:2] for _ in range(m)]).astype(np.int32)
        wts = r.random((m, 2)).astype(np.float32)
        y = eng.moe_ffn(moe, *(torch.from_numpy(v).cuda() for v in (x, ids, wts))).double().cpu().numpy()
        want = np.zeros((m, d))
        for i in range(m):
            for j in range(2):
                xe, c = x[i].astype(np.float64), ids[i, j]
                want[i] += float(wts[i, j]) * (dn[c] @ (act64(g[c] @ xe, "silu") * (u[c] @ xe)))
        assert np.linalg.norm(y - want) <= 1e-5 * np.linalg.norm(want), (t, m)


# ---------------------------------------------------------------- routers
def cuda(v):
    return None if v is None else torch.from_numpy(v).cuda()


def check_route(eng, moe, x, wr, k, score, bias, scale=1.5):
    y, ids, wts = eng.moe_layer(moe, cuda(wr), cuda(x), k, score=score, sel_bias=cuda(bias), scale=scale)
    ri, rw = reference_route(x, wr, score, bias, scale, k)
    assert np.array_equal(ids.cpu().numpy(), ri)
    assert np.all(np.abs(wts.double().cpu().numpy() - rw) <= 2.0 ** -23 * rw)  # f64 inside, rounded once
    assert torch.equal(y, eng.moe_ffn(moe, cuda(x), ids, wts))


@pytest.mark.parametrize("score", sorted(_lib.SCORES))
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("e", [33, 128, 129, 300, 512])
def test_routers_of_many_experts(eng, e, with_bias, score):
    """Up to 16 experts of a lane, with the last lanes' part filled and empty."""
    moe = experts(eng, e, 256, 32, Q4_K, Q8_0)
    r = np.random.default_rng(e)
    wr = (r.standard_normal((e, 256)) / 16).astype(np.float32)
    bias = (0.1 * r.standard_normal(e)).astype(np.float32) if with_bias else None
    for m, k in ((1, 8), (21, 16), (64, 1)):
        x = r.standard_normal((m, 256)).astype(np.float32)
        check_route(eng, moe, x, wr, k, score, bias)
    wr[:] = 0  # ties over all lanes: the lowest ids, or the order of the bias
    check_route(eng, moe, x[:2].copy(), wr, 16, score, bias)
    x, wr = np.ones((1, 256), np.float32), np.zeros((e, 256), np.float32)
    wr[[e - 1, e // 2], 0] = 1.0
    check_route(eng, moe, x, wr, 3, score, None)


@pytest.mark.parametrize("d", [4064, 4096, 4128, 8192, 12320])
@pytest.mark.parametrize("off", [0, 1])
def test_routers_over_wide_rows(eng, d, off):
    """Rows of one, two and four turns of the logits' CTA, whole and begun, with and without 16-byte alignment."""
    moe = experts(eng, 5, d, 32, Q8_0, Q8_0)
    r = np.random.default_rng(d)
    wr = (r.standard_normal((5, d)) / np.sqrt(d)).astype(np.float32)
    for m in (1, 11):
        x = r.standard_normal((m, d)).astype(np.float32)
        xd, wd = (torch.empty(v.size + 1, device="cuda")[off:off + v.size].copy_(cuda(v.reshape(-1))).reshape(v.shape)
                  for v in (x, wr))
        assert (xd.data_ptr() % 16 != 0) == bool(off)
        y, ids, wts = eng.moe_layer(moe, wd, xd, 2)
        ri, rw = reference_route(x, wr, "softmax_norm", None, 1.0, 2)
        assert np.array_equal(ids.cpu().numpy(), ri)
        assert np.all(np.abs(wts.double().cpu().numpy() - rw) <= 2.0 ** -23 * rw)
        assert torch.equal(y, eng.moe_layer(moe, cuda(wr), cuda(x), 2)[0])


def test_softmax_picks_go_by_the_logits(eng):
    """Scores far below the largest round to 0 and keep their logits' order; a NaN logit comes last, alone."""
    e = 40
    moe = experts(eng, e, 256, 32, Q4_K, Q8_0)
    x = np.zeros((1, 256), np.float32)
    x[0, 0] = 1.0
    wr = np.zeros((e, 256), np.float32)
    wr[:, 0] = -2000.0 - np.arange(e)[::-1]
    wr[7, 0] = 0.0
    for score in ("softmax", "softmax_norm"):
        _, ids, wts = eng.moe_layer(moe, cuda(wr), cuda(x), 4, score=score)
        assert ids.tolist() == [[7, 39, 38, 37]] and wts.tolist() == [[1.0, 0.0, 0.0, 0.0]]
    wr[39, 0] = np.nan
    _, ids, wts = eng.moe_layer(moe, cuda(wr), cuda(x), 4, score="softmax_norm")
    assert ids.tolist() == [[7, 38, 37, 36]] and wts.tolist() == [[1.0, 0.0, 0.0, 0.0]]
    _, ids, _ = eng.moe_layer(moe, cuda(wr), cuda(x), 16, score="sigmoid_norm")
    assert 39 not in ids.tolist()[0]


# ---------------------------------------------------------------- tensors beyond 32-bit offsets, long and short shapes
def device_blocks(rows, k, t, seed):
    """Random GGUF blocks made on the GPU, their f16 scales small and finite."""
    f = FORMATS[t]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = rows * k // f.block_weights
    b = torch.randint(0, 256, (n, f.block_bytes), generator=g, device="cuda", dtype=torch.uint8)
    places = {Q6_K: (208,), Q4_K: (0, 2), Q5_K: (0, 2)}.get(t, (0,))
    for at in places:
        scale = (torch.rand(n, generator=g, device="cuda") * 1e-3 + 1e-4).to(torch.float16)
        b[:, at:at + 2] = scale.view(torch.uint8).reshape(n, 2)
    return b.reshape(-1)


@pytest.mark.parametrize("t,k", [(Q8_0, 8192), (Q6_K, 7936), (Q4_0, 8224)], ids=["aligned", "unaligned_q6k", "unaligned_q40"])
def test_linear_rows_beyond_4_gb(eng, t, k):
    """The last rows of a tensor of more than 4 GB against the same rows as a tensor of their own."""
    rb = FORMATS[t].row_bytes(k)
    n, last = (4 << 30) // rb + 3000, 259
    w = device_blocks(n, k, t, 1)
    tail = w[(n - last) * rb:].clone()
    for m in (1, 6, 16):
        x = torch.randn(m, k, device="cuda")
        y = eng.linear(x, w, t, n, k)[:, -last:].double()
        r = eng.linear(x, tail, t, last, k).double()
        assert torch.linalg.norm(y - r) <= 1e-5 * torch.linalg.norm(r), m  # two results, each 5e-6 off
    if k % 256 == 0:
        x = torch.randn(40, k, device="cuda").bfloat16()
        y, r = eng.linear(x, w, t, n, k)[:, -last:].double(), eng.linear(x, tail, t, last, k).double()
        assert torch.linalg.norm(y - r) <= 2.0 ** -7 * torch.linalg.norm(r)  # both rounded to bf16


@pytest.mark.parametrize("t,d,f", [(Q4_K, 4096, 4096), (Q6_K, 3584, 4352), (Q4_0, 4128, 4064)])
def test_moe_experts_beyond_4_gb(eng, t, d, f):
    """The last of many experts against a layer that has it alone (gate and up are one tensor here)."""
    from planejaja_b200.engine import MoeExperts
    up, down = f * FORMATS[t].row_bytes(d), d * FORMATS[t].row_bytes(f)
    e = (33 << 27) // min(up, down) + 1
    assert e <= 512
    wu, wd = device_blocks(e * f, d, t, 2), device_blocks(e * d, f, t, 3)
    assert min(wu.numel(), wd.numel()) > (4 << 30) + min(up, down)
    many = MoeExperts(wu, wu, wd, e, d, f, t, t)
    g, dn = wu[(e - 1) * up:].clone(), wd[(e - 1) * down:].clone()
    one = MoeExperts(g, g, dn, 1, d, f, t, t)
    for m in (1, 7, 33):
        x = torch.randn(m, d, device="cuda")
        wts = torch.rand(m, 1, device="cuda")
        ids = torch.full((m, 1), e - 1, dtype=torch.int32, device="cuda")
        y, r = eng.moe_ffn(many, x, ids, wts).double(), eng.moe_ffn(one, x, ids * 0, wts).double()
        assert torch.linalg.norm(y - r) <= 2e-5 * torch.linalg.norm(r), m  # two results, each 1e-5 off


def test_prompt_outputs_beyond_2_to_31_elements(eng):
    m, n, k = 65600, 33000, 256
    w = eng.upload(Q.synthetic_weights(n, k, Q4_K, seed=4))
    x = torch.randn(m, k, device="cuda").bfloat16()
    b = torch.randn(n, device="cuda")
    y = eng.linear(x, w, Q4_K, n, k, bias=b, act="silu")
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 200), slice(m - 200, m), slice(m // 2, m // 2 + 200)):
        r = eng.linear(x[rows], w, Q4_K, n, k, bias=b, act="silu").double()
        assert torch.linalg.norm(y[rows].double() - r) <= 2.0 ** -7 * torch.linalg.norm(r)


@pytest.mark.parametrize("m", [1, 4, 9])
@pytest.mark.parametrize("n,k,t", [(1, 1 << 20, Q8_0), (3, 1 << 20, Q6_K), (1 << 20, 32, Q4_0), (1 << 18, 256, Q5_K)])
def test_linear_long_and_flat(eng, oracle, m, n, k, t):
    """One row of a million, a million rows of one block.  With independent roundings (2^-24 of the partial sums, up
    to 3 times the result, at each of nsb units and 33 joins; 1.4e-6 for the activations) an output is off by
    3 * 2^-24 sqrt(33 + nsb) + 1.4e-6 of its terms' root sum of squares; 5e-6 at least is allowed."""
    w = device_blocks(n, k, t, n + k)
    x = torch.randn(m, k, device="cuda")
    y = eng.linear(x, w, t, n, k).double()
    w64 = torch.from_numpy(oracle.dequant(w.cpu().numpy(), t, 0).reshape(n, k)).cuda().double()
    r = x.double() @ w64.t()
    size = torch.sqrt((x.double() ** 2) @ (w64 ** 2).t())
    tol = max(5e-6, 1.4e-6 + 3 * 2.0 ** -24 * (33 + -(-k // 256)) ** 0.5)
    assert torch.linalg.norm(y - r) <= tol * torch.linalg.norm(size)


@pytest.mark.parametrize("act", sorted(_lib.ACTS))
@pytest.mark.parametrize("m,dtype", [(2, torch.float32), (2, torch.bfloat16), (17, torch.bfloat16)])
def test_activations_over_all_values(eng, m, dtype, act):
    """x = 0, so that bias is what the activation gets: small, large, infinite and NaN values against the formula in
    64 bits, written without the cancellation of 1 + erf and 1 + tanh far below 0.

    In half steps of f32 (2^-24): gelu's argument v / sqrt 2 has 2 roundings, and erfc falls by 2 x^2 of itself per
    relative change of x, x^2 <= 88; the argument of gelu_tanh's exponential, up to 88, has 7 (4 of them in the
    cube); the functions and what follows them at most 12.  A bf16 result adds its rounding (2^-8 here, twice the
    half step, which leaves room for the fast exponential of prompts: 2 + 1.16 * 88 steps of f32).  An exponential
    below 1e-30 may be lost."""
    v = np.concatenate([s * np.float32(10.0) ** np.arange(-30, 31, 3) for s in (-1, 1)] + [np.linspace(-100, 100, 401)])
    v = np.concatenate([v, [0.0, -0.0, np.inf, -np.inf, np.nan, 3e38, -3e38]]).astype(np.float32)
    n, k = v.size, 256
    w = eng.upload(Q.synthetic_weights(n, k, Q4_K, seed=0))
    x = torch.zeros(m, k, device="cuda", dtype=dtype)
    y = eng.linear(x, w, Q4_K, n, k, bias=torch.from_numpy(v).cuda(), act=act).double().cpu()
    d = torch.from_numpy(v).double()
    r = {"none": d, "silu": d * torch.sigmoid(d), "gelu": 0.5 * d * torch.erfc(-d / 2 ** 0.5),
         "gelu_tanh": d * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (d + 0.044715 * d ** 3)),
         "relu": torch.where(d < 0, 0.0, d)}[act]  # (-inf * 0 is NaN)
    eps = 2.0 ** -24 * (12 + 88 * {"gelu": 4, "gelu_tanh": 7}.get(act, 0)) + (2.0 ** -8 if dtype is torch.bfloat16 else 0)
    for i in range(m):
        assert torch.equal(y[i].isnan(), r.isnan())
        # (in bf16 3e38 may round to infinity)
        ok = r.isfinite() if dtype is torch.float32 else r.abs() < 3e38
        over = (y[i][ok] - r[ok]).abs() / (eps * r[ok].abs() + 1e-30)
        worst = int(over.argmax())
        assert float(over[worst]) <= 1, (float(d[ok][worst]), float(y[i][ok][worst]), float(r[ok][worst]))
        assert torch.equal(y[i][r.isinf()], r[r.isinf()])


# ---------------------------------------------------------------- captures
def test_captured_behind_copies_and_between_streams(eng):
    """One graph: inputs copied from the host, two branches of products that meet in a layer, its output copied back."""
    d, e, f = 512, 8, 768
    moe = experts(eng, e, d, f, Q4_K, Q6_K)
    w = [eng.upload(Q.synthetic_weights(d, d, t, seed=t)) for t in (Q4_K, Q8_0)]
    wr = torch.randn(e, d, device="cuda")
    host, back = torch.empty(3, d).pin_memory(), torch.empty(3, d).pin_memory()
    x = torch.empty(3, d, device="cuda")
    ws = [eng.linear_workspace(3, d, d), eng.linear_workspace(3, d, d), eng.moe_workspace(moe, 3, 2)]

    def step(sync):
        side, main = torch.cuda.Stream(), torch.cuda.current_stream()
        x.copy_(host, non_blocking=True)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            b = eng.linear(x, w[1], Q8_0, d, d, act="silu", workspace=ws[1], sync=sync)
        a = eng.linear(x, w[0], Q4_K, d, d, workspace=ws[0], sync=sync)
        main.wait_stream(side)
        y, _, _ = eng.moe_layer(moe, wr, a, 2, residual=b, workspace=ws[2], sync=sync)
        z = eng.linear(y, w[0], Q4_K, d, d, residual=a, workspace=ws[0], sync=sync)
        back.copy_(z, non_blocking=True)
        b.record_stream(main)
        return z
    host.normal_()
    step(True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        z = step(False)
    for _ in range(5):
        host.normal_()
        g.replay()
        torch.cuda.synchronize()
        got = z.clone()
        assert torch.equal(back, got.cpu())
        assert torch.equal(step(True), got)
