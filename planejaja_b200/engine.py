"""Host-side mirror of the reference engine's matmul / dequant operators.

`CudaEngine` keeps the shape of NodeStor's `VulkanEngine`
(nodestor/crates/nodestor-vulkan/src/lib.rs:38-271) for the hot path:

  upload(bytes)                 -> device buffer       (lib.rs:221-224)
  download_f32(buf)             -> host f32 array      (lib.rs:236-239)
  matmul(a, b, m, k, n)         -> C = A[m,k] . B[k,n] (lib.rs:117-122, dense f32)
  matmul_quant(x, w, t, m, k, n)-> y = x . W^T over GGUF blocks (the quantized
                                   branch of TensorOp::Matmul,
                                   src/operator_registry.rs:43-49, 246-259)
  dequant(w, t, n)              -> f32 / bf16 weights (DequantDispatcher::dequantize,
                                   crates/nodestor-inference/src/dequant/mod.rs:142-191)
  linear(x, w, t, n, k, ...)    -> y = act(x . W^T + bias) + residual, the
                                   matmul, add and activation calls of a
                                   projection (transformer.rs:241-321) as one
  moe_layer / moe_ffn           -> a mixture-of-experts feed-forward layer over
                                   GGUF experts, with or without its router
  zipgemm(w, x, m, k, n)        -> y = x . W^T from an NSZ (TCA-TBE) tensor,
                                   decompressed in registers (lib.rs:124-151)
  nsz_decode(w)                 -> the NSZ tensor's original weights, bit-exact
                                   (nsz_decoder.rs:19-196)

Device memory, streams and the output buffers come from PyTorch; every
computation is a call into libnsq.so.  Like the reference, calls are
synchronous by default (the reference waits for queue idle after every
dispatch, src/pipeline.rs:486-487); pass `sync=False` to stay asynchronous on
the current CUDA stream.  Errors raise NsqError (the reference returns
NodeStorError, crates/nodestor-core/src/error.rs:1-38).

Kernel choice for matmul_quant: M <= 16 uses the decode GEMV (fp32
activations and output); larger M uses the tcgen05 prefill GEMM (bf16
operands, fp32 accumulate, bf16 output widened back to f32).  The
environment variable NSQ_MATMUL_PATH=gemv|gemm forces one of them.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

import numpy as np
import torch

from . import _lib
from .formats import FORMATS, Q6K_GGML, fmt
from ._lib import NsqError, check


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream_handle(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class MoeExperts:
    """The experts of a mixture-of-experts layer: three GGUF tensors on one
    device, as they lie in the file (ffn_gate_exps and ffn_up_exps
    [n_expert x n_ff rows of n_embd], ffn_down_exps [n_expert x n_embd rows of
    n_ff])."""

    def __init__(self, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, n_expert: int, n_embd: int,
                 n_ff: int, type_in: int, type_down: int, layout_in: int = Q6K_GGML, layout_down: int = Q6K_GGML,
                 act: str = "silu"):
        for name, w, t, n, k in (("w_gate", w_gate, type_in, n_ff, n_embd), ("w_up", w_up, type_in, n_ff, n_embd),
                                 ("w_down", w_down, type_down, n_embd, n_ff)):
            if t not in FORMATS:
                raise NsqError(_lib.ERR_TYPE, f"MoeExperts: {name} has ggml type {t}")
            if min(n_expert, n, k) < 1 or k % FORMATS[t].block_weights:
                raise NsqError(_lib.ERR_SHAPE, f"MoeExperts: {name} [{n_expert} x {n} x {k}]")
            _check_bytes(w, n_expert * FORMATS[t].tensor_bytes(n, k), f"MoeExperts: {name}", w_gate.get_device())
        if act not in _lib.ACTS:
            raise NsqError(_lib.ERR_TYPE, f"MoeExperts: activation {act!r}")
        self.w_gate, self.w_up, self.w_down = w_gate, w_up, w_down
        self.n_expert, self.n_embd, self.n_ff = n_expert, n_embd, n_ff
        self.device_index = w_gate.get_device()
        self._c = _lib.Moe(_ptr(w_gate), _ptr(w_up), _ptr(w_down), type_in, layout_in, type_down, layout_down,
                           _lib.ACTS[act], n_expert, n_embd, n_ff)
        self._ref = ctypes.addressof(self._c)


def _check_bytes(w: torch.Tensor, nbytes: int, what: str, device: int) -> None:
    if w.dtype != torch.uint8 or not w.is_cuda or not w.is_contiguous():
        raise NsqError(_lib.ERR_TYPE, f"{what}: GGUF bytes are a contiguous uint8 CUDA tensor")
    if w.get_device() != device:  # the kernels would read memory that the GPU need not have mapped
        raise NsqError(_lib.ERR_DEVICE, f"{what}: on {w.device}, cuda:{device} is wanted")
    if w.numel() < nbytes:
        raise NsqError(_lib.ERR_SHAPE, f"{what}: {w.numel()} bytes, {nbytes} needed")


def _has_rows(shape, row: int) -> bool:
    """Whether a tensor of this shape is a list of rows of `row` elements: its last dimensions make one up
    ([tokens, heads, size] holds rows of heads x size), or it is one run of elements."""
    dims = [s for s in shape if s != 1]
    size = 1
    for s in reversed(dims):
        if size == row:
            return True
        size *= s
    return size == row or len(dims) <= 1


class CudaEngine:
    """Engine facade over libnsq for one CUDA device."""

    def __init__(self, device: int | str | torch.device = 0):
        if not torch.cuda.is_available():
            raise NsqError(_lib.ERR_DEVICE, "no CUDA device")
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        self.lib = _lib.load()
        self._ws: Optional[torch.Tensor] = None

    # ---- buffers ---------------------------------------------------------
    def upload(self, data) -> torch.Tensor:
        """Copy host bytes (bytes / numpy array) to a new device uint8 buffer."""
        arr = np.frombuffer(data, np.uint8) if isinstance(data, (bytes, bytearray, memoryview)) else \
            np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        return torch.from_numpy(arr.copy()).to(self.device)

    def upload_f32(self, data) -> torch.Tensor:
        return torch.as_tensor(np.ascontiguousarray(data, np.float32)).to(self.device)

    def download_f32(self, buf: torch.Tensor) -> np.ndarray:
        return buf.detach().float().cpu().numpy()

    def workspace(self, nbytes: int) -> torch.Tensor:
        """Scratch for prepared activations; grown outside the hot calls."""
        if self._ws is None or self._ws.numel() < nbytes:
            self._ws = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=self.device)
        return self._ws

    def _stream(self) -> int:
        return _stream_handle(self.device)

    def _sync(self, sync: bool):
        if sync:
            torch.cuda.synchronize(self.device)

    # ---- operators ---------------------------------------------------------
    def dequant(self, w: torch.Tensor, ggml_type: int, n_elems: int, out_dtype: str = "f32",
                q6k_layout: int = Q6K_GGML, out: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        od = _lib.OUT_F32 if out_dtype == "f32" else _lib.OUT_BF16
        if out is None:
            out = torch.empty(n_elems, dtype=torch.float32 if od == _lib.OUT_F32 else torch.bfloat16,
                              device=self.device)
        check(self.lib.nsq_dequant(_ptr(w), ggml_type, q6k_layout, od, _ptr(out), n_elems, self._stream()),
              "nsq_dequant")
        self._sync(sync)
        return out

    def gemv(self, w: torch.Tensor, ggml_type: int, x: torch.Tensor, n: int, k: int,
             q6k_layout: int = Q6K_GGML, y: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        m = x.numel() // k
        if y is None:
            y = torch.empty((m, n), dtype=torch.float32, device=self.device)
        wsb = self.lib.nsq_gemv_workspace_size(m, k)
        ws = self.workspace(wsb)
        check(self.lib.nsq_gemv(_ptr(w), ggml_type, q6k_layout, _ptr(x), _ptr(y), m, n, k, _ptr(ws), ws.numel(),
                                self._stream()), "nsq_gemv")
        self._sync(sync)
        return y

    def gemv_multi(self, segments, x: torch.Tensor, k: int, sync: bool = True):
        """Fused GEMV over matrices sharing `x` (q|k|v, gate|up).

        segments: list of (w, ggml_type, n) or (w, ggml_type, n, q6k_layout);
        returns the list of outputs [m, n_s] (f32)."""
        m = x.numel() // k
        segs = (_lib.Segment * len(segments))()
        outs = []
        for i, sg in enumerate(segments):
            w, t, n = sg[0], sg[1], sg[2]
            layout = sg[3] if len(sg) > 3 else Q6K_GGML
            y = torch.empty((m, n), dtype=torch.float32, device=self.device)
            outs.append(y)
            segs[i] = _lib.Segment(_ptr(w), t, layout, n, _ptr(y))
        wsb = self.lib.nsq_gemv_workspace_size(m, k)
        ws = self.workspace(wsb)
        check(self.lib.nsq_gemv_multi(ctypes.cast(segs, ctypes.c_void_p), len(segments), _ptr(x), m, k, _ptr(ws),
                                      ws.numel(), self._stream()), "nsq_gemv_multi")
        self._sync(sync)
        return outs

    def gemv_swiglu(self, w_gate: torch.Tensor, w_up: torch.Tensor, ggml_type: int, x: torch.Tensor, n: int, k: int,
                    q6k_layout: int = Q6K_GGML, out: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        """h[m, n] = silu(x . Wg^T) * (x . Wu^T) in one launch (the FFN input
        projection with the reference's silu + mul fused in)."""
        m = x.numel() // k
        h = out if out is not None else torch.empty(m, n, dtype=torch.float32, device=self.device)
        x = x.contiguous().float()
        ws = self.workspace(self.lib.nsq_gemv_workspace_size(m, k))
        check(self.lib.nsq_gemv_swiglu(_ptr(w_gate), _ptr(w_up), ggml_type, q6k_layout, _ptr(x), _ptr(h), m, n, k,
                                       _ptr(ws), ws.numel(), self._stream()), "nsq_gemv_swiglu")
        self._sync(sync)
        return h

    def gemv_residual(self, w: torch.Tensor, ggml_type: int, x: torch.Tensor, residual: torch.Tensor, n: int, k: int,
                      q6k_layout: int = Q6K_GGML, out: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        """y = residual + x . W^T in one launch; `out` may be `residual` (in place)."""
        m = x.numel() // k
        y = out if out is not None else torch.empty(m, n, dtype=torch.float32, device=self.device)
        x = x.contiguous().float()
        residual = residual.contiguous().float()
        ws = self.workspace(self.lib.nsq_gemv_workspace_size(m, k))
        check(self.lib.nsq_gemv_residual(_ptr(w), ggml_type, q6k_layout, _ptr(x), _ptr(residual), _ptr(y), m, n, k,
                                         _ptr(ws), ws.numel(), self._stream()), "nsq_gemv_residual")
        self._sync(sync)
        return y

    def prepare(self, x: torch.Tensor, k: int, ws: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Prepare activations once for several GEMVs (q|k|v, gate|up)."""
        m = x.numel() // k
        nbytes = self.lib.nsq_gemv_workspace_size(m, k)
        if ws is None:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        check(self.lib.nsq_prepare_activations(_ptr(x), m, k, _ptr(ws), ws.numel(), self._stream()),
              "nsq_prepare_activations")
        return ws

    def gemv_prepared(self, w: torch.Tensor, ggml_type: int, ws: torch.Tensor, m: int, n: int, k: int,
                      q6k_layout: int = Q6K_GGML, y: Optional[torch.Tensor] = None) -> torch.Tensor:
        if y is None:
            y = torch.empty((m, n), dtype=torch.float32, device=self.device)
        check(self.lib.nsq_gemv_prepared(_ptr(w), ggml_type, q6k_layout, _ptr(ws), _ptr(y), m, n, k,
                                         self._stream()), "nsq_gemv_prepared")
        return y

    def gemm_bf16(self, w: torch.Tensor, ggml_type: int, x: torch.Tensor, n: int, k: int,
                  q6k_layout: int = Q6K_GGML, y: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        if x.dtype != torch.bfloat16:
            raise NsqError(_lib.ERR_TYPE, "gemm_bf16 expects bf16 activations")
        m = x.numel() // k
        if y is None:
            y = torch.empty((m, n), dtype=torch.bfloat16, device=self.device)
        check(self.lib.nsq_gemm_bf16(_ptr(w), ggml_type, q6k_layout, _ptr(x), _ptr(y), m, n, k, self._stream()),
              "nsq_gemm_bf16")
        self._sync(sync)
        return y

    def matmul(self, a: torch.Tensor, b: torch.Tensor, m: int, k: int, n: int, sync: bool = True) -> torch.Tensor:
        """Dense f32 C[m, n] = A[m, k] . B[k, n] (the reference operator's layout)."""
        c = torch.empty((m, n), dtype=torch.float32, device=self.device)
        check(self.lib.nsq_matmul_f32(_ptr(a), _ptr(b), _ptr(c), m, k, n, self._stream()), "nsq_matmul_f32")
        self._sync(sync)
        return c

    def matmul_quant(self, x: torch.Tensor, w: torch.Tensor, ggml_type: int, m: int, k: int, n: int,
                     q6k_layout: int = Q6K_GGML, sync: bool = True) -> torch.Tensor:
        """y[m, n] f32 = x[m, k] . W^T with W[n, k] in GGUF blocks of `ggml_type`."""
        if ggml_type not in FORMATS:
            raise NsqError(_lib.ERR_TYPE, f"matmul_quant: ggml type {ggml_type}")
        if w.numel() < fmt(ggml_type).tensor_bytes(n, k):
            raise NsqError(_lib.ERR_SHAPE, "matmul_quant: weight buffer smaller than N*row_bytes")
        path = os.environ.get("NSQ_MATMUL_PATH", "")
        if path == "gemv" or (path != "gemm" and m <= _lib.GEMV_MAX_M):
            return self.gemv(w, ggml_type, x.reshape(m, k).float().contiguous(), n, k, q6k_layout, sync=sync)
        xb = x.reshape(m, k).to(torch.bfloat16).contiguous()
        return self.gemm_bf16(w, ggml_type, xb, n, k, q6k_layout, sync=sync).float()

    # ---- products with an epilogue, and mixture-of-experts layers -----------
    def _index(self) -> int:
        """The device that calls run on: the engine's, or the current one where the engine names none."""
        index = self.device.index
        return torch._C._cuda_getDevice() if index is None else index

    def _check_experts(self, moe: MoeExperts, what: str) -> None:
        if moe.device_index != self._index():
            raise NsqError(_lib.ERR_DEVICE, f"{what}: the experts are on cuda:{moe.device_index}, the engine is on "
                                            f"{self.device}")

    def _tensor(self, t: Optional[torch.Tensor], numel: int, dtype: torch.dtype, what: str,
                row: int = 0) -> Optional[torch.Tensor]:
        """`t` as the library reads it: contiguous, of this dtype and size, on the engine's device, its last
        dimensions making up rows of `row` elements (where it has rows)."""
        if t is None:
            return None
        if (t.dtype is dtype and t.device == self.device and t.numel() == numel
                and (not row or numel == row or t.shape[-1] == row) and t.is_contiguous()):
            return t  # small calls are bound by the host: the usual case first
        if t.dtype != dtype or not t.is_cuda:
            raise NsqError(_lib.ERR_TYPE, f"{what}: a {dtype} CUDA tensor is wanted, not {t.dtype} on {t.device}")
        if t.device.index != self._index():
            raise NsqError(_lib.ERR_DEVICE, f"{what}: on {t.device}, the engine is on {self.device}")
        if t.numel() != numel:
            raise NsqError(_lib.ERR_SHAPE, f"{what}: {t.numel()} elements, not {numel}")
        if row and not _has_rows(t.shape, row):
            raise NsqError(_lib.ERR_SHAPE, f"{what}: {list(t.shape)} has no rows of {row}")
        return t if t.is_contiguous() else t.contiguous()

    def _out(self, out: Optional[torch.Tensor], shape, dtype: torch.dtype, what: str, like: torch.Tensor) -> torch.Tensor:
        if out is None:
            return like.new_empty(shape)
        if not out.is_contiguous():
            raise NsqError(_lib.ERR_SHAPE, f"{what}: the output has to be contiguous")
        return self._tensor(out, shape[0] * shape[1], dtype, what, shape[1])

    def _call(self, fn, what: str, nbytes, workspace: Optional[torch.Tensor], args, sync: bool) -> None:
        """fn(*args, workspace, bytes, stream) with the engine's device current.  Without a workspace of the
        caller's, the call takes one of nbytes() from PyTorch's allocator, which keeps it from other streams and
        graphs."""
        if workspace is None:
            workspace = torch.empty(nbytes() or 16, dtype=torch.uint8, device=self.device)
        elif workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
            raise NsqError(_lib.ERR_TYPE, f"{what}: a workspace is contiguous uint8, not {workspace.dtype}")
        else:
            self._tensor(workspace, workspace.numel(), torch.uint8, f"{what}: workspace")
        index = self.device.index
        current = torch._C._cuda_getDevice()
        if index is None or index == current:
            rc = fn(*args, workspace.data_ptr(), workspace.numel(), torch._C._cuda_getCurrentRawStream(current))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, workspace.data_ptr(), workspace.numel(), _stream_handle(self.device))
        if rc:
            raise NsqError(rc, what)
        if sync:
            torch.cuda.synchronize(self.device)

    def linear_workspace(self, m: int, n: int, k: int) -> torch.Tensor:
        """Workspace of `linear` calls of up to this size; one call at a time may use it.  (Calls of more than 16
        tokens use none: one made for them serves those of up to 16.)"""
        size = self.lib.nsq_linear_workspace_size(min(m, _lib.GEMV_MAX_M), k)
        return torch.empty(size or 16, dtype=torch.uint8, device=self.device)

    def linear(self, x: torch.Tensor, w: torch.Tensor, ggml_type: int, n: int, k: int,
               bias: Optional[torch.Tensor] = None, act: str = "none", residual: Optional[torch.Tensor] = None,
               q6k_layout: int = Q6K_GGML, out: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        """y[m, n] = act(x . W^T + bias) + residual in one product (nsq_linear).

        x [m, k], residual and y are f32 (m <= 16) or bf16; bias [n] f32; act one of "none", "silu", "gelu",
        "gelu_tanh", "relu".  `out` may be `residual`.

        Up to 16 tokens k is a multiple of the format's block and the weights enter unrounded; more tokens want bf16,
        k % 256 == 0 and 16-byte aligned x and out, and round the weights to bf16 as gemm_bf16 does: the same bf16
        call is off by 1.7e-3 of its norm with 16 tokens and by about 2.3e-3 with 17.  A token with an infinity gives
        NaN up to 16 tokens and IEEE results beyond."""
        dtype = x.dtype
        if dtype is not torch.float32 and dtype is not torch.bfloat16:
            raise NsqError(_lib.ERR_TYPE, f"linear: activations are f32 or bf16, not {dtype}")
        if ggml_type not in FORMATS or act not in _lib.ACTS:
            raise NsqError(_lib.ERR_TYPE, f"linear: ggml type {ggml_type}, activation {act!r}")
        f = FORMATS[ggml_type]
        size = x.numel()
        if k < 1 or n < 1 or size % k or k % f.block_weights:
            raise NsqError(_lib.ERR_SHAPE, f"linear: {size} activations, n = {n}, k = {k}")
        m = size // k
        _check_bytes(w, n * k // f.block_weights * f.block_bytes, "linear: w", self._index())
        x = self._tensor(x, size, dtype, "linear: x", k)
        bias = self._tensor(bias, n, torch.float32, "linear: bias")
        residual = self._tensor(residual, m * n, dtype, "linear: residual", n)
        y = self._out(out, (m, n), dtype, "linear: out", x)
        self._call(self.lib.nsq_linear, "nsq_linear", lambda: self.lib.nsq_linear_workspace_size(m, k), workspace,
                   (_ptr(w), ggml_type, q6k_layout, _ptr(x), _ptr(bias), _lib.ACTS[act], _ptr(residual), _ptr(y),
                    _lib.OUT_F32 if dtype is torch.float32 else _lib.OUT_BF16, m, n, k), sync)
        return y

    def moe_workspace(self, moe: MoeExperts, m: int, top_k: int) -> torch.Tensor:
        """Workspace of `moe_ffn` / `moe_layer` calls of up to this size; one call at a time may use it."""
        self._check_experts(moe, "moe_workspace")
        return torch.empty(self.lib.nsq_moe_workspace_size(moe._ref, m, top_k) or 16, dtype=torch.uint8,
                           device=self.device)

    def moe_ffn(self, moe: MoeExperts, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                workspace: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        """y[m] = residual[m] + sum_j weights[m, j] * expert ids[m, j] of x[m] (nsq_moe_ffn).

        x [m, n_embd] f32; ids [m, top_k] int32, -1 for an unused slot; weights [m, top_k] f32.  `out` may be
        `residual`."""
        self._check_experts(moe, "moe_ffn")
        if ids.dim() != 2:
            raise NsqError(_lib.ERR_SHAPE, "moe_ffn: ids are [tokens, top_k]")
        m, top_k = ids.shape
        x = self._tensor(x, m * moe.n_embd, torch.float32, "moe_ffn: x", moe.n_embd)
        ids = self._tensor(ids, m * top_k, torch.int32, "moe_ffn: ids")
        weights = self._tensor(weights, m * top_k, torch.float32, "moe_ffn: weights", top_k)
        residual = self._tensor(residual, m * moe.n_embd, torch.float32, "moe_ffn: residual", moe.n_embd)
        y = self._out(out, (m, moe.n_embd), torch.float32, "moe_ffn: out", x)
        self._call(self.lib.nsq_moe_ffn, "nsq_moe_ffn", lambda: self.lib.nsq_moe_workspace_size(moe._ref, m, top_k),
                   workspace, (moe._ref, _ptr(x), _ptr(ids), _ptr(weights), _ptr(residual), _ptr(y), m, top_k), sync)
        return y

    def moe_layer(self, moe: MoeExperts, w_router: torch.Tensor, x: torch.Tensor, top_k: int,
                  score: str = "softmax_norm", sel_bias: Optional[torch.Tensor] = None, scale: float = 1.0,
                  residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  workspace: Optional[torch.Tensor] = None, sync: bool = True):
        """Router, picks and experts (nsq_moe_layer): (y [m, n_embd], ids [m, top_k] int32, weights [m, top_k]).

        w_router [n_expert, n_embd] f32 (GGUF ffn_gate_inp); score one of "softmax", "softmax_norm",
        "sigmoid_norm"; sel_bias [n_expert] enters the choice alone."""
        self._check_experts(moe, "moe_layer")
        if score not in _lib.SCORES:
            raise NsqError(_lib.ERR_TYPE, f"moe_layer: score {score!r}")
        if x.numel() % moe.n_embd:
            raise NsqError(_lib.ERR_SHAPE, f"moe_layer: {x.numel()} activations, n_embd = {moe.n_embd}")
        m = x.numel() // moe.n_embd
        x = self._tensor(x, m * moe.n_embd, torch.float32, "moe_layer: x", moe.n_embd)
        w_router = self._tensor(w_router, moe.n_expert * moe.n_embd, torch.float32, "moe_layer: w_router", moe.n_embd)
        sel_bias = self._tensor(sel_bias, moe.n_expert, torch.float32, "moe_layer: sel_bias")
        residual = self._tensor(residual, m * moe.n_embd, torch.float32, "moe_layer: residual", moe.n_embd)
        y = self._out(out, (m, moe.n_embd), torch.float32, "moe_layer: out", x)
        ids = x.new_empty((m, max(top_k, 0)), dtype=torch.int32)
        weights = x.new_empty((m, max(top_k, 0)))
        self._call(self.lib.nsq_moe_layer, "nsq_moe_layer",
                   lambda: self.lib.nsq_moe_workspace_size(moe._ref, m, top_k), workspace,
                   (moe._ref, _ptr(w_router), _lib.SCORES[score], _ptr(sel_bias), scale, _ptr(x), _ptr(residual),
                    _ptr(y), _ptr(ids), _ptr(weights), m, top_k), sync)
        return y, ids, weights

    # ---- NSZ (TCA-TBE) tensors and ZipGEMM --------------------------------
    def nsz_upload(self, stream, num_weights: int, dtype: int = _lib.NSZ_FP32, shape=()) -> "NszTensor":
        """One-time upload of an NSZ tile stream and its validated offset table."""
        from .nsz import NszTensor, index
        stream = np.ascontiguousarray(stream, np.uint8).reshape(-1)
        off = index(stream, num_weights, dtype)
        tiles = torch.from_numpy(stream.copy()).to(self.device) if stream.size else \
            torch.empty(16, dtype=torch.uint8, device=self.device)
        offsets = torch.from_numpy(off.view(np.int32)).to(self.device)
        return NszTensor(tiles, offsets, int(num_weights), int(dtype), tuple(shape))

    def nsz_decode(self, t, out: Optional[torch.Tensor] = None, sync: bool = True) -> torch.Tensor:
        """Lossless decode: float32 / float16 / bfloat16 weights, bit-exact."""
        dt = {_lib.NSZ_FP32: torch.float32, _lib.NSZ_FP16: torch.float16, _lib.NSZ_BF16: torch.bfloat16}[t.dtype]
        if out is None:
            out = torch.empty(max(t.count, 1), dtype=dt, device=self.device)[:t.count]
        check(self.lib.nsq_nsz_decode(_ptr(t.tiles), _ptr(t.offsets), t.count, t.dtype, _ptr(out),
                                      self._stream()), "nsq_nsz_decode")
        self._sync(sync)
        return out

    def zipgemm(self, w, x: torch.Tensor, m: int, k: int, n: int, out: Optional[torch.Tensor] = None,
                sync: bool = True) -> torch.Tensor:
        """ZipGEMM (VulkanEngine::zipgemm, lib.rs:124-151): y[m, n] f32 =
        x[m, k] . W^T, W [n x k] decompressed on the fly from an NszTensor."""
        if w.count != n * k:
            raise NsqError(_lib.ERR_SHAPE, f"zipgemm: tensor holds {w.count} weights, not {n} x {k}")
        x = x.reshape(m, k)
        if x.dtype != torch.float32 or not x.is_contiguous():
            x = x.float().contiguous()
        if out is None:
            out = torch.empty((m, n), dtype=torch.float32, device=self.device)
        check(self.lib.nsq_zipgemm(_ptr(w.tiles), _ptr(w.offsets), w.dtype, _ptr(x), _ptr(out), m, n, k,
                                   self._stream()), "nsq_zipgemm")
        self._sync(sync)
        return out

    def device_status(self, clear: bool = True) -> int:
        """NSQ_ERR_TIMEOUT if a bounded device-side wait gave up, else 0."""
        return self.lib.nsq_device_status(1 if clear else 0)
