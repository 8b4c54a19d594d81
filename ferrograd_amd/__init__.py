"""ferrograd_amd -- MI355X (gfx950) backend for ferrograd's fused training path.

The product is the C-ABI library ``libferrograd_hip.so`` (declared in
``include/ferrograd_hip.h``): hand-written HIP kernels for gfx950 and the C++
host runtime around them.  This package is the thin Python face of that ABI:

* ``Context`` / direct-kernel helpers below take device pointers (``int``) or
  any object with ``data_ptr()`` (e.g. a torch tensor used purely as device
  memory);
* ``graph`` mirrors ferrograd's Graph / GpuContext API (build, lower,
  schedule, dispatch_forward / loss / backward / optim) on top of the
  library's planner.

Nothing here computes on the CPU: every call goes to the library, and the
import fails loudly when the library has not been built.
"""
from __future__ import annotations

import ctypes
import weakref
from typing import Optional, Sequence

import numpy as np

from . import _lib
from ._lib import FgError, call, load

NN, NT, TN = 0, 1, 2
ACT_NONE, ACT_RELU, ACT_GELU = 0, 1, 2
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
ELTWISE_INTERPRET, ELTWISE_COMPILE_LARGE, ELTWISE_COMPILE_ALL = 0, 1, 2

__all__ = [
    "NN", "NT", "TN", "ACT_NONE", "ACT_RELU", "ACT_GELU", "FgError", "Context",
    "MultiTensor", "load", "rng_uniform", "rng_normal", "rng_int", "torch_context",
    "eltwise_mode", "eltwise_stats",
]


def _ptr(x) -> Optional[int]:
    """Device address of x: None, an int address, or an object with data_ptr()."""
    if x is None or isinstance(x, int):
        return x
    return int(x.data_ptr())


class Context:
    """An fg_ctx bound to ``device`` and a HIP stream.

    ``stream`` is a raw hipStream_t address (e.g. ``torch.cuda.current_stream()
    .cuda_stream``) or None for a private stream."""

    def __init__(self, device: int = 0, stream: Optional[int] = None):
        h = ctypes.c_void_p()
        call("fg_ctx_create", device, stream, ctypes.byref(h))
        self.handle = h
        arch = ctypes.create_string_buffer(64)
        flags = ctypes.c_uint32()
        cus = ctypes.c_int()
        call("fg_ctx_target", h, arch, 64, ctypes.byref(flags), ctypes.byref(cus))
        self.arch = arch.value.decode()
        self.flags = flags.value
        self.cu_count = cus.value
        # Plans and tensor lists made on this context (they keep a pointer to
        # it): closed before it, whatever order the garbage collector picks.
        self._dependents = weakref.WeakSet()

    def adopt(self, obj) -> None:
        """Close `obj` (anything with close()) before this context closes."""
        self._dependents.add(obj)

    @property
    def stream(self) -> int:
        s = ctypes.c_void_p()
        call("fg_ctx_stream", self.handle, ctypes.byref(s))
        return int(s.value or 0)

    def sync(self) -> None:
        call("fg_sync", self.handle)

    def is_ready(self) -> bool:
        r = ctypes.c_int()
        call("fg_is_ready", self.handle, ctypes.byref(r))
        return bool(r.value)

    def reserve_workspace(self, nbytes: int) -> None:
        call("fg_ctx_reserve_workspace", self.handle, nbytes)

    def close(self) -> None:
        if self.handle:
            for d in list(getattr(self, "_dependents", ())):
                d.close()
            call("fg_ctx_destroy", self.handle)
            self.handle = None

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------ direct kernels
    def gemm(self, layout: int, M: int, N: int, K: int, A, lda: int, B, ldb: int, C, ldc: int,
             bias=None, act: int = ACT_NONE, Z=None, ldz: int = 0,
             accumulate: bool = False) -> None:
        call("fg_gemm_f32", self.handle, layout, M, N, K, _ptr(A), lda, _ptr(B), ldb, _ptr(bias),
             act, _ptr(C), ldc, _ptr(Z), ldz, int(accumulate))

    def gemm_bwd(self, layout: int, M: int, N: int, K: int, A, lda: int, B, ldb: int, C,
                 ldc: int, act: int = ACT_NONE, Zs=None, ldzs: int = 0,
                 accumulate: bool = False) -> None:
        call("fg_gemm_bwd_f32", self.handle, layout, M, N, K, _ptr(A), lda, _ptr(B), ldb, act,
             _ptr(Zs), ldzs, _ptr(C), ldc, int(accumulate))

    def gemm_dw(self, M: int, N: int, K: int, A, lda: int, B, ldb: int, C, ldc: int,
                accumulate: bool = False, colsum=None, colsum_accumulate: bool = False) -> None:
        """C (=|+=) A^T.B and colsum (=|+=) column sums of B in one launch."""
        call("fg_gemm_dw_f32", self.handle, M, N, K, _ptr(A), lda, _ptr(B), ldb, _ptr(C), ldc,
             int(accumulate), _ptr(colsum), int(colsum_accumulate))

    def linear_bwd(self, act: int, M: int, N: int, K: int, X, ldx: int, W, ldw: int, Zs,
                   ldzs: int, dC, lddc: int, dX=None, lddx: int = 0, dW=None, lddw: int = 0,
                   dbias=None, accumulate: bool = False, dZ=None, lddz: int = 0) -> None:
        """Backward of C = act(X.W + bias): dZ = dC * act'(Zs), dX = dZ.W^T,
        dW = X^T.dZ, dbias = colsum(dZ) (any output may be None).  With a dZ
        buffer, dZ is materialised by one pass; without, act' is applied to
        the dC tiles as the GEMMs load them."""
        call("fg_linear_bwd_f32", self.handle, act, M, N, K, _ptr(X), ldx, _ptr(W), ldw,
             _ptr(Zs), ldzs, _ptr(dC), lddc, _ptr(dX), lddx or K, _ptr(dW), lddw or N,
             _ptr(dbias), int(accumulate), _ptr(dZ), lddz or N)

    def matmul_bwd(self, M: int, N: int, K: int, X, ldx: int, W, ldw: int, dZ, lddz: int, dX,
                   lddx: int, dW, lddw: int, dbias=None, act: int = ACT_NONE, Zs=None,
                   ldzs: int = 0, accumulate: bool = False) -> None:
        """A matmul node's gradients from dZ: dW = X^T.dZ (+ dbias = colsum(dZ))
        and dX = (dZ.W^T) * act'(Zs), in one launch when their kernels pair."""
        call("fg_matmul_bwd_f32", self.handle, M, N, K, _ptr(X), ldx, _ptr(W), ldw, _ptr(dZ),
             lddz, act, _ptr(Zs), ldzs, _ptr(dX), lddx, _ptr(dW), lddw, _ptr(dbias),
             int(accumulate))

    def matmul_bwd_x16(self, dtype: int, M: int, N: int, K: int, X, ldx: int, W, ldw: int, dZ,
                       lddz: int, dX, lddx: int, dW, lddw: int, dbias=None, act: int = ACT_NONE,
                       Zs=None, ldzs: int = 0, accumulate: bool = False) -> None:
        """matmul_bwd with 16-bit tensors (dtype DTYPE_F16 / DTYPE_BF16)."""
        call("fg_matmul_bwd_x16", self.handle, dtype, M, N, K, _ptr(X), ldx, _ptr(W), ldw,
             _ptr(dZ), lddz, act, _ptr(Zs), ldzs, _ptr(dX), lddx, _ptr(dW), lddw, _ptr(dbias),
             int(accumulate))

    def gemm_dw_x16(self, dtype: int, M: int, N: int, K: int, A, lda: int, B, ldb: int, C,
                    ldc: int, accumulate: bool = False, colsum=None,
                    colsum_accumulate: bool = False) -> None:
        """16-bit C (=|+=) A^T.B and colsum (=|+=) column sums of B in one launch."""
        call("fg_gemm_dw_x16", self.handle, dtype, M, N, K, _ptr(A), lda, _ptr(B), ldb, _ptr(C),
             ldc, int(accumulate), _ptr(colsum), int(colsum_accumulate))

    def gemm_x16(self, dtype: int, layout: int, M: int, N: int, K: int, A, lda: int, B,
                 ldb: int, C, ldc: int, bias=None, act: int = ACT_NONE, Z=None, ldz: int = 0,
                 accumulate: bool = False) -> None:
        """16-bit GEMM (dtype DTYPE_F16 / DTYPE_BF16 for every operand)."""
        call("fg_gemm_x16", self.handle, dtype, layout, M, N, K, _ptr(A), lda, _ptr(B), ldb,
             _ptr(bias), act, _ptr(C), ldc, _ptr(Z), ldz, int(accumulate))

    def gemm_bwd_x16(self, dtype: int, layout: int, M: int, N: int, K: int, A, lda: int, B,
                     ldb: int, C, ldc: int, act: int = ACT_NONE, Zs=None, ldzs: int = 0,
                     accumulate: bool = False) -> None:
        call("fg_gemm_bwd_x16", self.handle, dtype, layout, M, N, K, _ptr(A), lda, _ptr(B),
             ldb, act, _ptr(Zs), ldzs, _ptr(C), ldc, int(accumulate))

    def bias_grad(self, M: int, N: int, dZ, ld: int, dbias, accumulate: bool = False,
                  dtype: int = DTYPE_F32) -> None:
        call("fg_bias_grad", self.handle, dtype, M, N, _ptr(dZ), ld, _ptr(dbias),
             int(accumulate))

    def act_bwd(self, act: int, n: int, dH, Z, dZ) -> None:
        call("fg_act_bwd_f32", self.handle, act, n, _ptr(dH), _ptr(Z), _ptr(dZ))

    def softmax_ce(self, logits, ldx: int, labels, R: int, C: int, grad_scale: float = 1.0,
                   row_loss=None, mean_loss=None, dlogits=None, ldd: int = 0,
                   argmax=None, dtype: int = DTYPE_F32) -> None:
        call("fg_softmax_ce", self.handle, dtype, _ptr(logits), ldx, _ptr(labels), R, C,
             grad_scale, _ptr(row_loss), _ptr(mean_loss), _ptr(dlogits), ldd or C, _ptr(argmax))

    def softmax(self, x, R: int, C: int, y, dtype: int = DTYPE_F32) -> None:
        call("fg_softmax", self.handle, dtype, _ptr(x), R, C, _ptr(y))

    def softmax_bwd(self, y, dy, R: int, C: int, dx, accumulate: bool = False,
                    dtype: int = DTYPE_F32) -> None:
        call("fg_softmax_bwd", self.handle, dtype, _ptr(y), _ptr(dy), R, C, _ptr(dx),
             int(accumulate))

    def layer_norm(self, x, ldx: int, R: int, C: int, y, ldy: int, gamma=None, beta=None,
                   eps: float = 1e-5, mean=None, rstd=None, dtype: int = DTYPE_F32) -> None:
        """y = (x - mean) * rstd * gamma + beta per row; mean and rstd (fp32,
        one per row) are kept when given."""
        call("fg_layer_norm", self.handle, dtype, _ptr(x), ldx, _ptr(gamma), _ptr(beta), eps, R, C,
             _ptr(y), ldy, _ptr(mean), _ptr(rstd))

    def layer_norm_bwd(self, x, ldx: int, dy, lddy: int, mean, rstd, R: int, C: int, gamma=None,
                       dx=None, lddx: int = 0, dgamma=None, dbeta=None, accumulate: bool = False,
                       dgamma_accumulate: bool = False, dbeta_accumulate: bool = False,
                       dtype: int = DTYPE_F32) -> None:
        """dx, dgamma and dbeta (any may be None) from x, dy and the forward's
        mean and rstd."""
        call("fg_layer_norm_bwd", self.handle, dtype, _ptr(x), ldx, _ptr(dy), lddy, _ptr(gamma),
             _ptr(mean), _ptr(rstd), R, C, _ptr(dx), lddx or C, int(accumulate), _ptr(dgamma),
             int(dgamma_accumulate), _ptr(dbeta), int(dbeta_accumulate))

    def rms_norm(self, x, ldx: int, R: int, C: int, y=None, ldy: int = 0, r=None, ldr: int = 0,
                 s=None, lds: int = 0, gamma=None, eps: float = 1e-5, q=None, ldq: int = 0, e=None,
                 lde: int = 0, rstd=None, dtype: int = DTYPE_F32) -> None:
        """s = x + r (without r: x), y = s * rstd * gamma per row; y in 8 bits
        too when q and e are given, rstd (fp32, one per row) kept when given."""
        call("fg_rms_norm", self.handle, dtype, _ptr(x), ldx, _ptr(r), ldr or C, _ptr(gamma), eps,
             R, C, _ptr(s), lds or C, _ptr(y), ldy or C, _ptr(q), ldq or C, _ptr(e),
             lde or (C + 31) // 32, _ptr(rstd))

    def rms_norm_bwd(self, s, lds: int, dy, lddy: int, rstd, R: int, C: int, gamma=None, ds=None,
                     ldds: int = 0, dx=None, lddx: int = 0, dgamma=None,
                     dgamma_accumulate: bool = False, dtype: int = DTYPE_F32) -> None:
        """dx (the norm's, plus ds) and dgamma (either may be None) from s, dy
        and the forward's rstd."""
        call("fg_rms_norm_bwd", self.handle, dtype, _ptr(s), lds, _ptr(dy), lddy, _ptr(gamma),
             _ptr(rstd), R, C, _ptr(ds), ldds or C, _ptr(dx), lddx or C, _ptr(dgamma),
             int(dgamma_accumulate))

    def attention(self, q, ldq: int, k, ldk: int, v, ldv: int, q_starts, k_starts, n: int, Tq: int,
                  Tk: int, heads: int, kv_heads: int, D: int, out, ldo: int, k_lens=None,
                  scale: Optional[float] = None, causal: bool = True, lse=None,
                  dtype: int = DTYPE_F32) -> None:
        """Attention over n packed sequences (u32 starts of their rows and keys,
        n + 1 each; k_lens: the keys used of a cache's).  scale None: 1/sqrt(D).
        lse (fp32, [heads][Tq]) is kept when given."""
        call("fg_attention", self.handle, dtype, _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv,
             _ptr(q_starts), _ptr(k_starts), _ptr(k_lens), n, Tq, Tk, heads, kv_heads, D,
             D ** -0.5 if scale is None else scale, int(causal), _ptr(out), ldo, _ptr(lse))

    def attention_bwd(self, q, ldq: int, k, ldk: int, v, ldv: int, out, ldo: int, dout, lddo: int,
                      lse, q_starts, k_starts, n: int, Tq: int, Tk: int, heads: int, kv_heads: int,
                      D: int, dq, lddq: int, dk, lddk: int, dv, lddv: int,
                      scale: Optional[float] = None, causal: bool = True, accumulate: bool = False,
                      dtype: int = DTYPE_F32) -> None:
        """dq, dk and dv from dout and the forward's out and lse."""
        call("fg_attention_bwd", self.handle, dtype, _ptr(q), ldq, _ptr(k), ldk, _ptr(v), ldv,
             _ptr(out), ldo, _ptr(dout), lddo, _ptr(lse), _ptr(q_starts), _ptr(k_starts), n, Tq, Tk,
             heads, kv_heads, D, D ** -0.5 if scale is None else scale, int(causal), _ptr(dq), lddq,
             _ptr(dk), lddk, _ptr(dv), lddv, int(accumulate))

    def token_logprobs(self, logits, ldx: int, tokens, R: int, C: int, logp=None, entropy=None,
                       lse=None, top: int = 0, top_ids=None, top_logp=None, scale: float = 1.0,
                       dtype: int = DTYPE_F32) -> None:
        """Per row of softmax(scale * logits): the log probability of its token,
        the entropy, the log of the sum and the `top` most probable columns with
        theirs."""
        call("fg_token_logprobs", self.handle, dtype, _ptr(logits), ldx, _ptr(tokens), R, C, scale,
             _ptr(logp), _ptr(entropy), _ptr(lse), top, _ptr(top_ids), _ptr(top_logp))

    def token_logprobs_bwd(self, logits, ldx: int, tokens, R: int, C: int, lse, dlogits, ldd: int,
                           entropy=None, dlogp=None, dentropy=None, scale: float = 1.0,
                           dtype: int = DTYPE_F32) -> None:
        """dlogits from the gradients of logp and entropy (either may be None)
        and the forward's lse and entropy."""
        call("fg_token_logprobs_bwd", self.handle, dtype, _ptr(logits), ldx, _ptr(tokens), R, C,
             scale, _ptr(lse), _ptr(entropy), _ptr(dlogp), _ptr(dentropy), _ptr(dlogits), ldd)

    def embedding(self, tokens, T: int, V: int, C: int, table, ldt: int, out, ldo: int,
                  scale: float = 1.0, dtype: int = DTYPE_F32) -> None:
        """out[t] = scale * table[tokens[t]] (u32 tokens; a row of NaN for a
        token outside the table)."""
        call("fg_embedding", self.handle, dtype, _ptr(tokens), T, V, C, _ptr(table), ldt, scale,
             _ptr(out), ldo)

    def embedding_bwd(self, tokens, T: int, V: int, C: int, dout, lddo: int, dtable, lddt: int,
                      scale: float = 1.0, accumulate: bool = False,
                      dtype: int = DTYPE_F32) -> None:
        """dtable[v] (=|+=) scale * sum of dout[t] over the t with tokens[t] = v."""
        call("fg_embedding_bwd", self.handle, dtype, _ptr(tokens), T, V, C, _ptr(dout), lddo,
             scale, _ptr(dtable), lddt, int(accumulate))

    def ckpt8_save(self, x, ldx: int, R: int, C: int, q, ldq: int, e, lde: int,
                   dtype: int = DTYPE_F32) -> None:
        """x in 8 bits: int8 q[R][C] and a uint8 exponent e[R][ceil(C / 32)]
        per 32 columns of a row."""
        call("fg_ckpt8_save", self.handle, dtype, _ptr(x), ldx, R, C, _ptr(q), ldq, _ptr(e), lde)

    def ckpt8_load(self, q, ldq: int, e, lde: int, R: int, C: int, z=None, ldz: int = 0, h=None,
                   ldh: int = 0, act: int = ACT_NONE, dtype: int = DTYPE_F32) -> None:
        """z = the values kept by ckpt8_save, h = act(z) (either may be None)."""
        call("fg_ckpt8_load", self.handle, dtype, act, _ptr(q), ldq, _ptr(e), lde, R, C, _ptr(z),
             ldz or C, _ptr(h), ldh or C)

    def act_bwd_ckpt8(self, act: int, dH, lddh: int, q, ldq: int, e, lde: int, R: int, C: int, dZ,
                      lddz: int, dtype: int = DTYPE_F32) -> None:
        """dZ = dH * act'(z) with the pre-activation z kept by ckpt8_save."""
        call("fg_act_bwd_ckpt8", self.handle, dtype, act, _ptr(dH), lddh, _ptr(q), ldq, _ptr(e),
             lde, R, C, _ptr(dZ), lddz)

    def matmul_bwd_ckpt8(self, M: int, N: int, K: int, q, ldq: int, e, lde: int, W, ldw: int, dZ,
                         lddz: int, Xr, dX, lddx: int, dW, lddw: int, Zr=None, dbias=None,
                         act: int = ACT_NONE, accumulate: bool = False,
                         dtype: int = DTYPE_F32) -> None:
        """matmul_bwd of X.W with X = act(z) and z[M][K] kept by ckpt8_save:
        dW = act(z)^T.dZ (+ dbias = colsum(dZ)), dX = (dZ.W^T) * act'(z).  Xr
        and (for GELU) Zr are scratch of M x K elements."""
        call("fg_matmul_bwd_ckpt8", self.handle, dtype, M, N, K, act, _ptr(q), ldq, _ptr(e), lde,
             _ptr(W), ldw, _ptr(dZ), lddz, _ptr(Zr), _ptr(Xr), _ptr(dX), lddx, _ptr(dW), lddw,
             _ptr(dbias), int(accumulate))

    def fill_u32(self, dst, value: int, count: int) -> None:
        call("fg_fill_u32", self.handle, _ptr(dst), value, count)

    def rng_uniform(self, seed, tensor_id, lo, hi, dst, n) -> None:
        call("fg_rng_uniform_dev", self.handle, seed, tensor_id, lo, hi, _ptr(dst), n)

    def rng_normal(self, seed, tensor_id, mean, std, dst, n) -> None:
        call("fg_rng_normal_dev", self.handle, seed, tensor_id, mean, std, _ptr(dst), n)

    def rng_int(self, seed, tensor_id, bound, dst, n) -> None:
        call("fg_rng_int_dev", self.handle, seed, tensor_id, bound, _ptr(dst), n)


def torch_context(device: int = 0):
    """A Context sharing a fresh default-priority torch stream, made current.

    torch's default stream has the handle 0, which fg_ctx_create reads as
    "create a private stream"; binding an explicit stream instead keeps
    torch ops (allocation, copies, events) and library launches in one
    ordered queue.  Returns (context, torch stream)."""
    import torch

    torch.cuda.init()
    s = torch.cuda.Stream(device)
    torch.cuda.set_stream(s)
    return Context(device, s.cuda_stream), s


class MultiTensor:
    """A device-resident tensor list for the one-launch SGD / Adam updates."""

    def __init__(self, ctx: Context, params: Sequence, grads: Sequence,
                 m: Optional[Sequence] = None, v: Optional[Sequence] = None,
                 sizes: Optional[Sequence[int]] = None, dtypes: Optional[Sequence[int]] = None):
        """dtypes: element type per tensor (DTYPE_*) of params / grads; m and
        v are always fp32."""
        n = len(params)
        if sizes is None:
            sizes = [int(p.numel()) for p in params]
        arr = ctypes.c_void_p * n
        P = arr(*[_ptr(p) for p in params])
        G = arr(*[_ptr(g) for g in grads])
        Mv = arr(*[_ptr(x) for x in m]) if m is not None else None
        Vv = arr(*[_ptr(x) for x in v]) if v is not None else None
        S = (ctypes.c_uint64 * n)(*sizes)
        h = ctypes.c_void_p()
        D = (ctypes.c_int * n)(*dtypes) if dtypes is not None else None
        call("fg_mt_create_x", ctx.handle, n, D, P, G, Mv, Vv, S, ctypes.byref(h))
        self.ctx = ctx
        self.handle = h
        ctx.adopt(self)

    def sgd(self, lr: float, zero_grad: bool = True) -> None:
        call("fg_sgd_step", self.ctx.handle, self.handle, lr, int(zero_grad))

    def adam(self, lr: float, b1: float, b2: float, eps: float, step: int,
             zero_grad: bool = False) -> None:
        call("fg_adam_step", self.ctx.handle, self.handle, lr, b1, b2, eps, step, int(zero_grad))

    def adam_scalars(self, b1: float, b2: float, eps: float, step_size: float,
                     inv_sqrt_bc2: float, zero_grad: bool = False) -> None:
        call("fg_adam_step_scalars", self.ctx.handle, self.handle, b1, b2, eps, step_size,
             inv_sqrt_bc2, int(zero_grad))

    def close(self) -> None:
        if self.handle:
            call("fg_mt_destroy", self.handle)
            self.handle = None

    def __del__(self):  # pragma: no cover - best effort
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------ synthetic data
def rng_uniform(seed: int, tensor_id: int, shape, lo: float = 0.0, hi: float = 1.0) -> np.ndarray:
    out = np.empty(shape, dtype=np.float32)
    call("fg_rng_uniform_host", seed, tensor_id, lo, hi, out.ctypes.data, out.size)
    return out


def rng_normal(seed: int, tensor_id: int, shape, mean: float = 0.0,
               std: float = 1.0) -> np.ndarray:
    out = np.empty(shape, dtype=np.float32)
    call("fg_rng_normal_host", seed, tensor_id, mean, std, out.ctypes.data, out.size)
    return out


def rng_int(seed: int, tensor_id: int, shape, bound: int) -> np.ndarray:
    out = np.empty(shape, dtype=np.uint32)
    call("fg_rng_int_host", seed, tensor_id, bound, out.ctypes.data, out.size)
    return out


# ------------------------------------------------ compiled elementwise kernels
def eltwise_mode(mode: int) -> int:
    """Sets how plans run elementwise programs (ELTWISE_INTERPRET,
    ELTWISE_COMPILE_LARGE -- the default -- or ELTWISE_COMPILE_ALL), process-wide;
    returns the previous mode."""
    prev = ctypes.c_int32(0)
    call("fg_eltwise_set_mode", mode, ctypes.byref(prev))
    return prev.value


def eltwise_stats() -> dict:
    """Process-wide counts: kernels compiled, launches of compiled kernels,
    launches of the interpreter."""
    c, j, i = ctypes.c_uint64(0), ctypes.c_uint64(0), ctypes.c_uint64(0)
    call("fg_eltwise_stats", ctypes.byref(c), ctypes.byref(j), ctypes.byref(i))
    return {"compiled": c.value, "compiled_launches": j.value, "interpreted_launches": i.value}
