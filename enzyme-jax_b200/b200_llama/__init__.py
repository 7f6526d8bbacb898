"""Host-side driver of the B200 llama path.

Thin ``ctypes`` layer over ``libb200_llama.so`` (the C ABI declared in
``include/b200_llama.h``).  PyTorch supplies device memory, streams and
``torch.distributed``; every computation runs in the library's own sm_100a
kernels.  There is no CPU fallback: loading fails loudly when the library has
not been built, and every entry point raises :class:`B200Error` on a non-zero
status.
"""
from __future__ import annotations

import ctypes
import functools
import os
from ctypes import POINTER, byref, c_char_p, c_float, c_int32, c_size_t, c_uint32, c_void_p
from typing import Dict, Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "lib", "libb200_llama.so")

F32, BF16 = 0, 1
LEAF_ORDER = (
    "rms_att_weight", "rms_ffn_weight", "rms_final_weight", "token_embedding_table",
    "w1", "w2", "w3", "wcls", "wk", "wo", "wq", "wv",
)
CONFIG_KEYS = ("dim", "hidden_dim", "n_layers", "n_heads", "n_kv_heads", "vocab_size", "seq_len")

EXPORTS = (
    "b200_last_error", "b200_version", "b200_device_status", "b200_plan_create", "b200_plan_destroy",
    "b200_packed_weight_bytes", "b200_pack_weights", "b200_workspace_bytes", "b200_saved_bytes", "b200_forward",
    "b200_backward", "b200_packed_grad_bytes", "b200_unpack_grads", "b200_allreduce_f32", "b200_decode_step",
    "b200_gemm", "b200_rmsnorm", "b200_attention", "b200_comm_unique_id", "b200_comm_init_rank",
    "b200_comm_destroy", "b200_launch_count", "b200_profile_enable", "b200_profile_read",
    "b200_attention_decode_scratch_bytes", "b200_attention_decode", "b200_attention_decode_static",
    "b200_attention_backward", "b200_comm_peer_memory", "b200_selftest_bounded_wait", "b200_argmax",
    "b200_selftest_peer_wait", "b200_plan_cached", "b200_ffi_available", "b200_ffi_handler",
    "b200_token_vjp_workspace_bytes", "b200_token_vjp", "b200_comm_init_rank_ex", "b200_comm_setup_peer_memory",
    "b200_comm_attach_memory", "b200_tp_exchange_buffers", "b200_tp_reduce_norm", "b200_token_forward",
    "b200_static_sizes", "b200_jvp_workspace_bytes", "b200_forward_jvp", "b200_token_jvp_workspace_bytes",
    "b200_token_jvp", "b200_plan_set_option", "b200_plan_get_option", "b200_attention_packed",
    "b200_attention_packed_backward", "b200_kv4_append", "b200_kv4_read", "b200_attention_decode_kv4_scratch_bytes",
    "b200_attention_decode_kv4_scratch_bytes_for", "b200_attention_decode_kv4", "b200_copy_pages",
)


class B200Error(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"b200 status {status}: {message}")
        self.status = status


class _Config(ctypes.Structure):
    _fields_ = [(k, c_int32) for k in CONFIG_KEYS] + [("dtype", c_int32), ("rope_theta", c_float), ("rms_eps", c_float)]


_lib = None


def lib() -> ctypes.CDLL:
    """Loads the CUDA library; raises if it has not been built."""
    global _lib
    if _lib is None:
        path = os.environ.get("B200_LLAMA_LIB", LIB_PATH)  # another build of the same ABI, e.g. to compare two kernels
        if not os.path.exists(path):
            raise RuntimeError(
                f"{path} is missing: build it with `python enzyme-jax_b200/build.py` "
                "(there is no fallback implementation)")
        l = ctypes.CDLL(path)
        l.b200_last_error.restype = c_char_p
        l.b200_version.restype = c_char_p
        for name in EXPORTS:
            fn = getattr(l, name)
            if name not in ("b200_last_error", "b200_version", "b200_ffi_handler"):
                fn.restype = c_int32
        l.b200_ffi_handler.restype = c_void_p
        l.b200_ffi_handler.argtypes = [c_char_p]
        l.registerEnzymeJaXB200FFI.restype = c_int32
        l.b200_plan_cached.argtypes = [POINTER(_Config), c_int32, c_int32, c_void_p, POINTER(c_void_p)]
        l.b200_selftest_peer_wait.argtypes = [ctypes.c_int64, c_void_p, c_void_p]
        l.b200_token_vjp_workspace_bytes.argtypes = [c_void_p, c_int32, POINTER(c_size_t)]
        l.b200_token_forward.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                         c_size_t, c_void_p]
        l.b200_jvp_workspace_bytes.argtypes = [c_void_p, c_int32, c_int32, POINTER(c_size_t)]
        l.b200_forward_jvp.argtypes = [c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p,
                                       c_void_p, c_size_t, c_void_p]
        l.b200_token_jvp_workspace_bytes.argtypes = [c_void_p, c_int32, POINTER(c_size_t)]
        l.b200_token_jvp.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]
        l.b200_static_sizes.argtypes = [POINTER(_Config), c_int32, c_int32, POINTER(c_size_t), POINTER(c_size_t),
                                        POINTER(c_size_t)]
        l.b200_token_vjp.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                     c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]
        l.b200_launch_count.restype = ctypes.c_int64
        l.b200_profile_enable.argtypes = [c_int32]
        l.b200_profile_read.argtypes = [c_int32, POINTER(ctypes.c_double), POINTER(ctypes.c_double),
                                        POINTER(ctypes.c_int64)]
        l.b200_plan_create.argtypes = [POINTER(_Config), c_int32, c_int32, c_void_p, POINTER(c_void_p)]
        l.b200_plan_destroy.argtypes = [c_void_p]
        l.b200_plan_set_option.argtypes = [c_void_p, c_char_p, c_int32]
        l.b200_plan_get_option.argtypes = [c_void_p, c_char_p, POINTER(c_int32)]
        l.b200_packed_weight_bytes.argtypes = [c_void_p, c_int32, POINTER(c_size_t)]
        l.b200_packed_grad_bytes.argtypes = [c_void_p, POINTER(c_size_t)]
        l.b200_pack_weights.argtypes = [c_void_p, POINTER(c_void_p), c_int32, c_int32, c_void_p, c_void_p]
        l.b200_workspace_bytes.argtypes = [c_void_p, c_int32, c_int32, c_int32, POINTER(c_size_t)]
        l.b200_saved_bytes.argtypes = [c_void_p, c_int32, c_int32, POINTER(c_size_t)]
        l.b200_forward.argtypes = [c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p,
                                   c_void_p, c_size_t, c_void_p]
        l.b200_backward.argtypes = [c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p,
                                    c_int32, c_void_p, c_size_t, c_void_p]
        l.b200_unpack_grads.argtypes = [c_void_p, c_void_p, POINTER(c_void_p), c_void_p]
        l.b200_allreduce_f32.argtypes = [c_void_p, c_void_p, c_size_t, c_void_p]
        l.b200_decode_step.argtypes = [c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
                                       c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]
        l.b200_gemm.argtypes = [c_void_p, c_void_p, c_void_p] + [c_int32] * 12 + [c_void_p]
        l.b200_rmsnorm.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32, c_float, c_int32,
                                   c_void_p]
        l.b200_attention.argtypes = [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p] + [c_int32] * 9 + [c_void_p]
        l.b200_attention_decode_scratch_bytes.argtypes = [c_int32] * 4 + [POINTER(c_size_t)]
        l.b200_attention_decode.argtypes = [c_void_p] * 5 + [c_size_t] + [c_int32] * 10 + [c_void_p]
        l.b200_attention_decode_static.argtypes = [c_void_p] * 4 + [c_int32] * 10 + [c_void_p]
        l.b200_attention_backward.argtypes = [c_void_p] * 10 + [c_int32] * 9 + [c_void_p]
        l.b200_selftest_bounded_wait.argtypes = [ctypes.c_int64, c_void_p, c_void_p]
        l.b200_argmax.argtypes = [c_void_p, c_int32, c_int32, c_int32, c_void_p, c_void_p]
        l.b200_device_status.argtypes = [c_void_p, POINTER(c_uint32)]
        l.b200_comm_unique_id.argtypes = [c_void_p]
        l.b200_comm_init_rank.argtypes = [c_void_p, c_int32, c_int32, POINTER(c_void_p)]
        l.b200_comm_init_rank_ex.argtypes = [c_void_p, c_int32, c_int32, c_int32, POINTER(c_void_p)]
        l.b200_comm_setup_peer_memory.argtypes = [c_void_p]
        l.b200_comm_attach_memory.argtypes = [c_void_p, c_size_t, POINTER(c_void_p), c_void_p]
        l.b200_tp_exchange_buffers.argtypes = [c_void_p, c_size_t, POINTER(c_void_p), POINTER(c_void_p)]
        l.b200_tp_reduce_norm.argtypes = [c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_float,
                                          c_void_p]
        l.b200_comm_destroy.argtypes = [c_void_p]
        l.b200_comm_peer_memory.argtypes = [c_void_p, POINTER(c_int32)]
        l.b200_attention_packed.argtypes = [c_void_p] * 6 + [c_int32] * 11 + [c_void_p]
        l.b200_attention_packed_backward.argtypes = [c_void_p] * 11 + [c_int32] * 15 + [c_void_p]
        l.b200_kv4_append.argtypes = [c_void_p] * 7 + [c_int32] * 10 + [c_void_p]
        l.b200_kv4_read.argtypes = [c_void_p] * 7 + [c_int32] * 10 + [c_void_p]
        l.b200_attention_decode_kv4_scratch_bytes.argtypes = [c_int32] * 4 + [POINTER(c_size_t)]
        l.b200_attention_decode_kv4_scratch_bytes_for.argtypes = [c_int32] * 7 + [POINTER(c_size_t)]
        l.b200_attention_decode_kv4.argtypes = [c_void_p] * 7 + [c_size_t] + [c_int32] * 11 + [c_void_p]
        l.b200_copy_pages.argtypes = [c_void_p] + [c_int32] * 5 + [c_void_p] * 3 + [c_int32, c_void_p, ctypes.c_int64,
                                                                                  c_void_p, c_void_p]
        _lib = l
    return _lib


def check(status: int) -> None:
    if status != 0:
        raise B200Error(status, lib().b200_last_error().decode("utf-8", "replace"))


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dt(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return F32
    if dtype == torch.bfloat16:
        return BF16
    raise B200Error(3, f"unsupported dtype {dtype}")


def static_sizes(config: Dict[str, int], dtype: torch.dtype = torch.float32, with_transposed: bool = False,
                 pos: int = 0, rope_theta: float = 10000.0, rms_eps: float = 1e-5) -> Dict[str, int]:
    """Byte sizes of the packed weights, the packed gradients and the workspace of the reference-shaped call for a
    model on one GPU, computed without a device (``b200_static_sizes``)."""
    c = _Config(*[int(config[k]) for k in CONFIG_KEYS], _dt(dtype), rope_theta, rms_eps)
    a, b, w = c_size_t(0), c_size_t(0), c_size_t(0)
    check(lib().b200_static_sizes(byref(c), int(with_transposed), pos, byref(a), byref(b), byref(w)))
    return {"packed_bytes": a.value, "grad_bytes": b.value, "token_workspace_bytes": w.value}


def device_status() -> int:
    """Reads and clears the device status word (synchronises the stream)."""
    code = c_uint32(0)
    check(lib().b200_device_status(_stream(), byref(code)))
    return code.value


def launch_count() -> int:
    return int(lib().b200_launch_count())


PROFILE_CLASSES = ("gemm_tcgen05", "gemm_ffma", "attention_fwd", "attention_bwd", "attention_decode", "allreduce",
                   "gemm_tcgen05_pair")


def profile_enable(on: bool) -> None:
    check(lib().b200_profile_enable(int(on)))


def profile_read() -> Dict[str, Dict[str, float]]:
    """Per kernel class: summed ms, summed algorithmic work, launches (synchronises the recorded events)."""
    out = {}
    for i, name in enumerate(PROFILE_CLASSES):
        ms, work, n = ctypes.c_double(0), ctypes.c_double(0), ctypes.c_int64(0)
        check(lib().b200_profile_read(i, byref(ms), byref(work), byref(n)))
        out[name] = {"ms": ms.value, "work": work.value, "launches": int(n.value)}
    return out


# --------------------------------------------------------------------------
# single kernels
# --------------------------------------------------------------------------

def gemm(a: torch.Tensor, b: torch.Tensor, *, ta=False, tb=False, out_dtype=None, impl=0,
         out: Optional[torch.Tensor] = None, accumulate=False) -> torch.Tensor:
    """Y = op(a) @ op(b)^T with fp32 accumulation.  a is [M,K] ([K,M] with ta), b is [N,K] ([K,N] with tb)."""
    M, K = (a.shape[1], a.shape[0]) if ta else (a.shape[0], a.shape[1])
    N = b.shape[1] if tb else b.shape[0]
    out_dtype = out_dtype or a.dtype
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
    check(lib().b200_gemm(a.data_ptr(), b.data_ptr(), out.data_ptr(), M, N, K, a.stride(0), b.stride(0),
                          out.stride(0), int(ta), int(tb), _dt(a.dtype), _dt(out.dtype), int(accumulate), impl,
                          _stream()))
    return out


def rmsnorm(x: torch.Tensor, gain: torch.Tensor, eps: float = 1e-5, out_dtype=torch.float32):
    rows, dim = x.shape
    y = torch.empty(rows, dim, dtype=out_dtype, device=x.device)
    rinv = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib().b200_rmsnorm(x.data_ptr(), gain.data_ptr(), y.data_ptr(), rinv.data_ptr(), rows, dim, eps,
                             _dt(out_dtype), _stream()))
    return y, rinv


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: int, seq: int, n_heads: int, impl=0):
    """Causal attention; q,k,v are [batch*seq, n_heads*head_size] (possibly strided row views)."""
    T, d = q.shape
    hs = d // n_heads
    o = torch.empty(T, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(batch, n_heads, seq, dtype=torch.float32, device=q.device)
    check(lib().b200_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), batch, seq,
                               n_heads, hs, q.stride(0), k.stride(0), o.stride(0), _dt(q.dtype), impl, _stream()))
    return o, lse


def attention_backward(qkv: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, d_o: torch.Tensor, batch: int, seq: int,
                       n_heads: int, impl=0) -> torch.Tensor:
    """Backward of causal attention for a packed qkv [batch*seq, 3*d]; returns dqkv of the same shape."""
    T, d3 = qkv.shape
    d = d3 // 3
    es = qkv.element_size()
    dqkv = torch.empty_like(qkv)
    delta = torch.empty(batch * n_heads * seq, dtype=torch.float32, device=qkv.device)
    base, dbase = qkv.data_ptr(), dqkv.data_ptr()
    check(lib().b200_attention_backward(base, base + d * es, base + 2 * d * es, o.data_ptr(), lse.data_ptr(),
                                        d_o.data_ptr(), dbase, dbase + d * es, dbase + 2 * d * es, delta.data_ptr(),
                                        batch, seq, n_heads, d // n_heads, d3, d3, o.stride(0), _dt(qkv.dtype), impl,
                                        _stream()))
    return dqkv


def attention_decode(q: torch.Tensor, kv_layer: torch.Tensor, page_table: torch.Tensor, ctx: int, n_heads: int,
                     scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention of q [batch, n_heads*hs] over one layer of a paged cache [2, n_pages, n_heads, page_size, hs]."""
    batch, d = q.shape
    hs = d // n_heads
    n_pages, page_size = kv_layer.shape[1], kv_layer.shape[3]
    o = torch.empty(batch, d, dtype=q.dtype, device=q.device)
    if scratch is None:
        n = c_size_t(0)
        check(lib().b200_attention_decode_scratch_bytes(batch, n_heads, hs, ctx, byref(n)))
        scratch = torch.empty(n.value, dtype=torch.uint8, device=q.device)
    check(lib().b200_attention_decode(q.data_ptr(), kv_layer.data_ptr(), page_table.data_ptr(), o.data_ptr(),
                                      scratch.data_ptr(), scratch.numel(), batch, ctx, n_heads, hs, q.stride(0),
                                      o.stride(0), n_pages, page_size, page_table.shape[1], _dt(q.dtype), _stream()))
    return o


def attention_decode_static(q: torch.Tensor, kv_layer: torch.Tensor, page_table: torch.Tensor, ctx: int,
                            n_heads: int, out: torch.Tensor) -> torch.Tensor:
    """Decode attention that allocates nothing: the caller passes the output, the scratch is the
    library's built-in 4 MiB array.  For callers that cannot allocate device memory (no scratch
    operand to give, fixed memory pool, cudaMalloc not permitted where they run).  Calls that may
    overlap on the GPU race on the shared scratch; make the first call outside stream capture."""
    batch, d = q.shape
    hs = d // n_heads
    check(lib().b200_attention_decode_static(q.data_ptr(), kv_layer.data_ptr(), page_table.data_ptr(),
                                             out.data_ptr(), batch, ctx, n_heads, hs, q.stride(0), out.stride(0),
                                             kv_layer.shape[1], kv_layer.shape[3], page_table.shape[1],
                                             _dt(q.dtype), _stream()))
    return out


# --------------------------------------------------------------------------
# packed prompts, the 4-bit cache, page copies
# --------------------------------------------------------------------------

def _device_of(what: str, names: str, *tensors) -> torch.device:
    """The one CUDA device all given tensors (None: left out) are on; ``names``: their names, for the message."""
    first = None
    try:
        for t in tensors:
            if t is None:
                continue
            d = t.get_device()
            if first is None:
                first = d
            if d != first or d < 0:
                break
        else:
            return _DEVICES[first]
    except AttributeError:
        pass
    except IndexError:
        return torch.device("cuda", first)
    for name, t in zip(names.split(), tensors):
        if t is not None and (not isinstance(t, torch.Tensor) or not t.is_cuda):
            raise B200Error(1, f"{what}: {name} must be a CUDA tensor")
    raise B200Error(1, f"{what}: the tensors {names} are not all on one device")


_DEVICES = [torch.device("cuda", i) for i in range(16)]


def _call(dev: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` with ``dev`` current, on its current stream (the raw handle: building the Stream object
    costs more than the launch)."""
    if dev.index == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if status != 0:
        check(status)


_INT32_MAX = 0x7FFFFFFF


def _rows(what: str, name: str, t: torch.Tensor, cols: int, rows: Optional[int] = None,
          dtype: Optional[torch.dtype] = None) -> int:
    """Row pitch of a [rows, cols] tensor with unit column stride."""
    shape = t.shape
    if len(shape) != 2 or shape[1] != cols or (rows is not None and shape[0] != rows):
        raise B200Error(2, f"{what}: {name} has shape {tuple(shape)}, expected "
                           f"[{'rows' if rows is None else rows}, {cols}]")
    if dtype is not None and t.dtype != dtype:
        raise B200Error(3, f"{what}: {name} is {t.dtype}, expected {dtype}")
    ld, unit = t.stride()
    if shape[0] <= 1:
        if cols > 1 and shape[0] == 1 and unit != 1:
            raise B200Error(2, f"{what}: {name} needs unit column stride")
        return max(cols, 1)
    if unit != 1 or ld < cols:
        raise B200Error(2, f"{what}: {name} needs unit column stride and rows that do not overlap")
    if ld > _INT32_MAX or shape[0] > _INT32_MAX:  # (a foreign call takes the low 32 bits without a word)
        raise B200Error(2, f"{what}: {name} has {shape[0]} rows of pitch {ld}, more than 32 bits hold")
    return ld


def _rows_or_new(what: str, name: str, t: Optional[torch.Tensor], cols: int, rows: int, dtype: torch.dtype, dev):
    """The caller's tensor, checked, or a new one, with its row pitch."""
    if t is None:
        return torch.empty(rows, cols, dtype=dtype, device=dev), cols
    return t, _rows(what, name, t, cols, rows, dtype)


def _index(what: str, name: str, t: torch.Tensor, dim: int = 1) -> None:
    if t.dtype is not torch.int32 or t.dim() != dim or not t.is_contiguous():
        raise B200Error(3, f"{what}: {name} must be a contiguous int32 tensor of {dim} dimension(s)")


def _heads(what: str, q: torch.Tensor, n_heads: int, n_kv_heads: int) -> int:
    if n_heads <= 0 or n_kv_heads <= 0 or n_heads % n_kv_heads or q.dim() != 2 or q.shape[1] % n_heads:
        raise B200Error(2, f"{what}: {n_heads} query heads over {n_kv_heads} key heads do not fit q {tuple(q.shape)}")
    return q.shape[1] // n_heads


def attention_packed(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor, n_heads: int,
                     n_kv_heads: Optional[int] = None, *, impl: int = 0, out: Optional[torch.Tensor] = None,
                     lse: Optional[torch.Tensor] = None):
    """Causal attention over packed sequences of different lengths, with grouped heads.

    ``q`` [rows, n_heads*hs], ``k`` and ``v`` [rows, n_kv_heads*hs] (strided row views are fine); ``cu_seqlens`` int32
    [n_seqs + 1] on the device: sequence s owns rows cu_seqlens[s] .. cu_seqlens[s+1]-1.  Returns ``(o, lse)`` with lse
    fp32 [n_heads, rows].  Rows of no sequence are not written: give ``out`` / ``lse`` to choose what stands there."""
    what = "attention_packed"
    n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
    dev = _device_of(what, "q k v cu_seqlens out lse", q, k, v, cu_seqlens, out, lse)
    hs = _heads(what, q, n_heads, n_kv_heads)
    rows, dt = q.shape[0], q.dtype
    ldq = _rows(what, "q", q, n_heads * hs)
    ldk = _rows(what, "k", k, n_kv_heads * hs, rows, dt)
    ldv = _rows(what, "v", v, n_kv_heads * hs, rows, dt)
    _index(what, "cu_seqlens", cu_seqlens)
    if cu_seqlens.numel() < 1:
        raise B200Error(2, f"{what}: cu_seqlens holds n_seqs + 1 entries, at least one")
    out, ldo = _rows_or_new(what, "out", out, n_heads * hs, rows, dt, dev)
    if lse is None:
        lse = torch.empty(n_heads, rows, dtype=torch.float32, device=dev)
    elif lse.dtype != torch.float32 or tuple(lse.shape) != (n_heads, rows) or not lse.is_contiguous():
        raise B200Error(2, f"{what}: lse must be a contiguous fp32 [{n_heads}, {rows}]")
    _call(dev, lib().b200_attention_packed, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
          cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, rows, n_heads, n_kv_heads, hs, ldq, ldk, ldv, ldo, _dt(dt),
          impl)
    return out, lse


def attention_packed_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                              d_o: torch.Tensor, cu_seqlens: torch.Tensor, n_heads: int,
                              n_kv_heads: Optional[int] = None, *, impl: int = 0, dq: Optional[torch.Tensor] = None,
                              dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None):
    """Reverse mode of :func:`attention_packed`: returns ``(dq, dk, dv)`` of the layouts and dtype of q, k, v; dk and dv
    are summed over the query heads of a group.  Rows of no sequence are not written."""
    what = "attention_packed_backward"
    n_kv_heads = n_heads if n_kv_heads is None else n_kv_heads
    dev = _device_of(what, "q k v o lse d_o cu_seqlens dq dk dv",
                     q, k, v, o, lse, d_o, cu_seqlens, dq, dk, dv)
    hs = _heads(what, q, n_heads, n_kv_heads)
    rows, dt = q.shape[0], q.dtype
    wq, wk = n_heads * hs, n_kv_heads * hs
    ldq = _rows(what, "q", q, wq)
    ldk = _rows(what, "k", k, wk, rows, dt)
    ldv = _rows(what, "v", v, wk, rows, dt)
    ldo = _rows(what, "o", o, wq, rows, dt)
    lddo = _rows(what, "d_o", d_o, wq, rows, dt)
    if lse.dtype != torch.float32 or tuple(lse.shape) != (n_heads, rows) or not lse.is_contiguous():
        raise B200Error(2, f"{what}: lse must be a contiguous fp32 [{n_heads}, {rows}]")
    _index(what, "cu_seqlens", cu_seqlens)
    if cu_seqlens.numel() < 1:
        raise B200Error(2, f"{what}: cu_seqlens holds n_seqs + 1 entries, at least one")
    dq, lddq = _rows_or_new(what, "dq", dq, wq, rows, dt, dev)
    dk, lddk = _rows_or_new(what, "dk", dk, wk, rows, dt, dev)
    dv, lddv = _rows_or_new(what, "dv", dv, wk, rows, dt, dev)
    delta = torch.empty(n_heads * rows, dtype=torch.float32, device=dev)
    _call(dev, lib().b200_attention_packed_backward, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
          lse.data_ptr(), d_o.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr(),
          cu_seqlens.data_ptr(), cu_seqlens.numel() - 1, rows, n_heads, n_kv_heads, hs, ldq, ldk, ldv, ldo, lddo,
          lddq, lddk, lddv, _dt(dt), impl)
    return dq, dk, dv


def new_kv4_pages(n_layers: int, n_pages: int, n_kv_heads: int, page_size: int, head_size: int, device="cuda"):
    """Pools of a 4-bit key/value cache: ``codes`` uint8 [n_layers, 2, n_pages, n_kv_heads, page_size, head_size/2] and
    ``params`` bf16 [n_layers, 2, n_pages, n_kv_heads, page_size, 2] (scale, minimum).  A row stands for
    minimum + scale * code.  ``codes[l], params[l]`` is one layer, what the kv4 functions take."""
    if head_size % 2:
        raise B200Error(2, f"head size {head_size} is odd")
    codes = torch.zeros(n_layers, 2, n_pages, n_kv_heads, page_size, head_size // 2, dtype=torch.uint8, device=device)
    params = torch.zeros(n_layers, 2, n_pages, n_kv_heads, page_size, 2, dtype=torch.bfloat16, device=device)
    return codes, params


def _kv4_layer(what: str, codes: torch.Tensor, params: torch.Tensor):
    shape = codes.shape
    if len(shape) != 5 or shape[0] != 2 or codes.dtype is not torch.uint8 or not codes.is_contiguous():
        raise B200Error(2, f"{what}: codes must be a contiguous uint8 [2, n_pages, n_kv_heads, page_size, hs/2]")
    _, n_pages, n_kv_heads, page_size, half = shape
    want = (2, n_pages, n_kv_heads, page_size, 2)
    if params.dtype is not torch.bfloat16 or params.shape != want or not params.is_contiguous():
        raise B200Error(2, f"{what}: params must be a contiguous bf16 {want}")
    return n_pages, n_kv_heads, page_size, 2 * half


def _kv4_rows(what: str, page_table: torch.Tensor, cu_seqlens: torch.Tensor, ctx_before: Optional[torch.Tensor]) -> int:
    _index(what, "page_table", page_table, 2)
    _index(what, "cu_seqlens", cu_seqlens)
    n_seqs = page_table.shape[0]
    if cu_seqlens.numel() != n_seqs + 1:
        raise B200Error(2, f"{what}: cu_seqlens has {cu_seqlens.numel()} entries for {n_seqs} page-table rows")
    if ctx_before is not None:
        _index(what, "ctx_before", ctx_before)
        if ctx_before.numel() != n_seqs:
            raise B200Error(2, f"{what}: ctx_before has {ctx_before.numel()} entries for {n_seqs} sequences")
    return n_seqs


def kv4_append(k: torch.Tensor, v: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, page_table: torch.Tensor,
               cu_seqlens: torch.Tensor, ctx_before: Optional[torch.Tensor] = None) -> None:
    """Quantises the packed rows k, v [rows, n_kv_heads*hs] into one layer of a 4-bit cache.  Row t of sequence s becomes
    its cached row ``ctx_before[s] + t - cu_seqlens[s]`` (``ctx_before`` None: the sequences start empty).  No two rows of
    a call may have the same place: sequences that share pages append behind them.  Rows without a place (behind the page
    table, or a page id outside the pool) are skipped and make :func:`device_status` raise."""
    what = "kv4_append"
    dev = _device_of(what, "k v codes params page_table cu_seqlens ctx_before",
                     k, v, codes, params, page_table, cu_seqlens, ctx_before)
    n_pages, n_kv_heads, page_size, hs = _kv4_layer(what, codes, params)
    n_seqs = _kv4_rows(what, page_table, cu_seqlens, ctx_before)
    ldk = _rows(what, "k", k, n_kv_heads * hs)
    ldv = _rows(what, "v", v, n_kv_heads * hs, k.shape[0], k.dtype)
    _call(dev, lib().b200_kv4_append, k.data_ptr(), v.data_ptr(), codes.data_ptr(), params.data_ptr(),
          page_table.data_ptr(), cu_seqlens.data_ptr(), _ptr(ctx_before), n_seqs, k.shape[0], n_kv_heads, hs, ldk,
          ldv, n_pages, page_size, page_table.shape[1], _dt(k.dtype))


def kv4_read(codes: torch.Tensor, params: torch.Tensor, page_table: torch.Tensor, cu_seqlens: torch.Tensor,
             ctx_before: Optional[torch.Tensor], rows: int, *, dtype: torch.dtype = torch.bfloat16,
             k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None):
    """Reads cached rows back as packed k, v [rows, n_kv_heads*hs]: the way back of :func:`kv4_append` with the same
    ``cu_seqlens`` and ``ctx_before``.  Rows without a place are not written.  (:func:`attention_packed` takes as many
    queries as keys: it attends to rows read back only where every one of them has a query; a single query per sequence
    is :func:`attention_decode_kv4`.)"""
    what = "kv4_read"
    dev = _device_of(what, "codes params page_table cu_seqlens ctx_before k v",
                     codes, params, page_table, cu_seqlens, ctx_before, k, v)
    n_pages, n_kv_heads, page_size, hs = _kv4_layer(what, codes, params)
    n_seqs = _kv4_rows(what, page_table, cu_seqlens, ctx_before)
    if rows < 0:
        raise B200Error(2, f"{what}: {rows} rows")
    k, ldk = _rows_or_new(what, "k", k, n_kv_heads * hs, rows, dtype, dev)
    v, ldv = _rows_or_new(what, "v", v, n_kv_heads * hs, rows, dtype, dev)
    _call(dev, lib().b200_kv4_read, k.data_ptr(), v.data_ptr(), codes.data_ptr(), params.data_ptr(),
          page_table.data_ptr(), cu_seqlens.data_ptr(), _ptr(ctx_before), n_seqs, rows, n_kv_heads, hs, ldk, ldv,
          n_pages, page_size, page_table.shape[1], _dt(dtype))
    return k, v


@functools.lru_cache(maxsize=256)
def _kv4_scratch_bytes(device: int, *sizes: int) -> int:
    """Scratch of a step on one device: the shares of a step go by its number of SMs."""
    n = c_size_t(0)
    with torch.cuda.device(device):
        check(lib().b200_attention_decode_kv4_scratch_bytes_for(*sizes, byref(n)))
    return n.value


def attention_decode_kv4(q: torch.Tensor, codes: torch.Tensor, params: torch.Tensor, page_table: torch.Tensor,
                         ctx_lens: torch.Tensor, n_heads: int, *, impl: int = 0, out: Optional[torch.Tensor] = None,
                         scratch: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention of q [batch, n_heads*hs] over one layer of a 4-bit cache.  Sequence b attends to its first
    ``ctx_lens[b]`` (int32 [batch] on the device) cached rows; zero rows give a zero output.  Query head h reads key head
    h / (n_heads / n_kv_heads).  bf16 heads of 64 and 128 on pages of a multiple of 16 rows take the tensor cores, where
    query elements are held to 2^-16 of their head's largest and weights to 2^-16 of the largest of 32 neighbouring keys;
    ``impl=2`` keeps both in fp32."""
    what = "attention_decode_kv4"
    dev = _device_of(what, "q codes params page_table ctx_lens out scratch",
                     q, codes, params, page_table, ctx_lens, out, scratch)
    n_pages, n_kv_heads, page_size, hs = _kv4_layer(what, codes, params)
    if n_heads <= 0 or n_heads % n_kv_heads:
        raise B200Error(2, f"{what}: {n_heads} query heads over {n_kv_heads} key heads")
    ldq = _rows(what, "q", q, n_heads * hs)
    batch = q.shape[0]
    _index(what, "page_table", page_table, 2)
    _index(what, "ctx_lens", ctx_lens)
    if page_table.shape[0] != batch or ctx_lens.numel() != batch:
        raise B200Error(2, f"{what}: page_table {tuple(page_table.shape)} and ctx_lens {tuple(ctx_lens.shape)} for a "
                           f"batch of {batch}")
    out, ldo = _rows_or_new(what, "out", out, n_heads * hs, batch, q.dtype, dev)
    max_pages, dt = page_table.shape[1], _dt(q.dtype)
    if scratch is None:
        size = _kv4_scratch_bytes(dev.index, batch, n_heads, n_kv_heads, hs, page_size, max_pages, dt)
        at = None
        if size:
            scratch = torch.empty(size, dtype=torch.uint8, device=dev)
            at = scratch.data_ptr()
    else:
        size, at = scratch.numel() * scratch.element_size(), scratch.data_ptr()
    _call(dev, lib().b200_attention_decode_kv4, q.data_ptr(), codes.data_ptr(), params.data_ptr(),
          page_table.data_ptr(), ctx_lens.data_ptr(), out.data_ptr(), at, size, batch, n_heads, n_kv_heads, hs, ldq,
          ldo, n_pages, page_size, max_pages, dt, impl)
    return out


def _check_copies(what: str, n_pages: int, src, dst) -> None:
    if len(src) != len(dst):
        raise B200Error(2, f"{what}: {len(src)} sources for {len(dst)} destinations")
    for p in list(src) + list(dst):
        if not 0 <= int(p) < n_pages:
            raise B200Error(1, f"{what}: page {p} is not a page of this pool of {n_pages}")
    if len(set(dst)) != len(dst):
        raise B200Error(1, f"{what}: a destination page is named twice")
    sources = {}
    for s, d in zip(src, dst):
        sources.setdefault(s, set()).add(d)
    for d in dst:
        if sources.get(d, set()) - {d}:
            raise B200Error(1, f"{what}: destination page {d} is the source of another copy")


def _page_list(what: str, name: str, x, dev) -> torch.Tensor:
    if isinstance(x, torch.Tensor):
        if not x.is_cuda:
            raise B200Error(1, f"{what}: {name} must be a CUDA tensor or a list of page numbers")
        _index(what, name, x)
        return x
    return torch.tensor([int(i) for i in x], dtype=torch.int32, device=dev)


def _check_pool(what, pool, src, dst, rows, page_table, page_map) -> None:
    """Everything that can be refused about one pool of a call, before any of its pools is touched."""
    if pool.dim() < 4 or not pool.is_contiguous():
        raise B200Error(2, f"{what}: the pool must be contiguous [..., n_pages, n_heads, page_size, row]")
    n_pages, n_heads, page_size, row = pool.shape[-4:]
    if max(n_pages, page_size * n_heads * row * pool.element_size()) > _INT32_MAX:
        raise B200Error(2, f"{what}: {n_pages} pages of [{n_heads}, {page_size}, {row}] {pool.dtype}: a page exceeds 2 GiB")
    if src.numel() != dst.numel() or (rows is not None and rows.numel() != src.numel()):
        raise B200Error(2, f"{what}: src, dst and rows must have one entry per copy")
    if page_map is not None and page_map.numel() != n_pages:
        raise B200Error(2, f"{what}: page_map has {page_map.numel()} entries for {n_pages} pages")
    _device_of(what, "pool src dst rows page_table page_map", pool, src, dst, rows, page_table, page_map)


def _copy_pages(what, pool, src, dst, rows, page_table, page_map) -> None:
    n_pages, n_heads, page_size, row = pool.shape[-4:]
    planes = 1
    for d in pool.shape[:-4]:
        planes *= d
    n = src.numel()
    if pool.numel() == 0:  # nothing to copy, but the table may have to follow the pages
        if page_table is None:
            return
        planes = n_heads = page_size = row = 1
        n = 0
    _call(pool.device, lib().b200_copy_pages, pool.data_ptr(), planes, n_pages, n_heads, page_size, row * pool.element_size(),
          src.data_ptr(), dst.data_ptr(), _ptr(rows), n, _ptr(page_table),
          0 if page_table is None else page_table.numel(), _ptr(page_map))


def copy_pages(pool: torch.Tensor, src, dst, rows=None) -> None:
    """Copies page ``src[i]`` to page ``dst[i]`` in every plane of a pool [..., n_pages, n_heads, page_size, row] (the
    pools of ``Plan.new_kv_pages`` and both pools of :func:`new_kv4_pages`), the first ``rows[i]`` rows of each head when
    ``rows`` is given.  Lists of page numbers are checked on the host; int32 CUDA tensors are taken as they are, and
    their destinations must be distinct and no copy's source."""
    what = "copy_pages"
    _device_of(what, "pool", pool)
    lists = [not isinstance(x, torch.Tensor) for x in (src, dst)]
    if all(lists):
        src, dst = [int(p) for p in src], [int(p) for p in dst]
        _check_copies(what, pool.shape[-4] if pool.dim() >= 4 else 0, src, dst)
    elif any(lists):
        raise B200Error(1, f"{what}: give src and dst both as lists or both as CUDA tensors")
    rows = None if rows is None else _page_list(what, "rows", rows, pool.device)
    src, dst = _page_list(what, "src", src, pool.device), _page_list(what, "dst", dst, pool.device)
    _check_pool(what, pool, src, dst, rows, None, None)
    _copy_pages(what, pool, src, dst, rows, None, None)


def compact_pages(pools, src, dst, page_table: torch.Tensor, page_map) -> None:
    """Moves pages ``src[i]`` to ``dst[i]`` in one pool, or in every pool of a list that shares the page table (codes and
    params of a 4-bit cache), and rewrites the int32 ``page_table`` in place: entry p becomes ``page_map[p]``.
    ``PageAllocator.compact`` returns the three lists."""
    what = "compact_pages"
    pools = list(pools) if isinstance(pools, (list, tuple)) else [pools]
    if not pools:
        raise B200Error(1, f"{what}: no pool")
    _device_of(what, "page_table pools", page_table, *pools)
    if page_table.dtype != torch.int32 or not page_table.is_contiguous():
        raise B200Error(3, f"{what}: page_table must be a contiguous int32 tensor")
    dev = page_table.device
    if len({p.shape[-4] if p.dim() >= 4 else 0 for p in pools}) != 1:
        raise B200Error(2, f"{what}: the pools differ in their number of pages")
    if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
        src, dst = [int(p) for p in src], [int(p) for p in dst]
        _check_copies(what, pools[0].shape[-4] if pools[0].dim() >= 4 else 0, src, dst)
    src, dst = _page_list(what, "src", src, dev), _page_list(what, "dst", dst, dev)
    page_map = _page_list(what, "page_map", page_map, dev)
    for pool in pools:
        _check_pool(what, pool, src, dst, None, page_table, page_map)
    moved = [p for p in pools if p.numel()] or pools[-1:]
    for i, pool in enumerate(moved):  # the table follows in the last pool's launch
        last = i == len(moved) - 1
        _copy_pages(what, pool, src, dst, None, page_table if last else None, page_map if last else None)


# --------------------------------------------------------------------------
# communicator
# --------------------------------------------------------------------------

def argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Row-wise argmax of fp32 logits [rows, cols] on the device (lowest index among equal maxima) -> int32 [rows]."""
    if logits.dtype != torch.float32 or logits.dim() != 2 or logits.stride(1) != 1:
        raise B200Error(3, "argmax takes fp32 [rows, cols] logits with unit column stride")
    if out is None:
        out = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    check(lib().b200_argmax(logits.data_ptr(), logits.shape[0], logits.shape[1], logits.stride(0), out.data_ptr(),
                            _stream()))
    return out


class PageAllocator:
    """Free list over the pages of one KV pool (host side).  Sequences take whole pages; a page table row lists a
    sequence's pages in position order, as ``b200_decode_step`` reads it.  A page may be shared by several sequences
    (:meth:`share`, :meth:`fork`); it is free again when the last of them gave it back."""

    def __init__(self, n_pages: int):
        self.n_pages = int(n_pages)
        self._free = list(range(self.n_pages - 1, -1, -1))
        self._refs: Dict[int, int] = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def refs(self, page: int) -> int:
        """Number of holders of a page (0: free)."""
        return self._refs.get(int(page), 0)

    def alloc(self, n: int):
        if n > len(self._free):
            raise B200Error(5, f"KV pool exhausted: {n} pages wanted, {len(self._free)} free")
        pages = [self._free.pop() for _ in range(n)]
        for p in pages:
            self._refs[p] = 1
        return pages

    @staticmethod
    def _numbers(pages):
        """Page numbers as plain ints: elements of a tensor or an array count as the numbers they hold."""
        return [int(p) for p in pages]

    def _held(self, pages) -> None:
        counts: Dict[int, int] = {}
        for p in pages:
            counts[p] = counts.get(p, 0) + 1
        for p, n in counts.items():
            if self._refs.get(p, 0) < n:
                raise B200Error(1, f"page {p} is not an allocated page of this pool")

    def free(self, pages) -> None:
        """Gives pages back, once per entry; all of them or, when one is not held, none."""
        pages = self._numbers(pages)
        self._held(pages)
        gone = []
        for p in pages:
            self._refs[p] -= 1
            if self._refs[p] == 0:
                del self._refs[p]
                gone.append(p)
        self._free.extend(reversed(gone))

    def share(self, pages) -> None:
        """Adds one holder to each of the pages."""
        pages = self._numbers(pages)
        for p in pages:
            if p not in self._refs:
                raise B200Error(1, f"page {p} is not an allocated page of this pool")
        for p in pages:
            self._refs[p] += 1

    def fork(self, pages, length: int, page_size: int):
        """Pages of a second sequence that begins with the first ``length`` rows of the sequence on ``pages``: full pages
        are shared, a partly filled last one gets a page of its own.  Returns ``(new_pages, copies)``; ``copies`` is a
        list of at most one ``(src, dst, rows)`` for :func:`copy_pages`."""
        pages = self._numbers(pages)
        if length < 0 or page_size <= 0 or length > len(pages) * page_size:
            raise B200Error(2, f"{length} rows do not fit {len(pages)} pages of {page_size}")
        full, rest = divmod(length, page_size)
        for p in pages[:full + (1 if rest else 0)]:
            if p not in self._refs:
                raise B200Error(1, f"page {p} is not an allocated page of this pool")
        own = self.alloc(1) if rest else []
        self.share(pages[:full])
        return pages[:full] + own, [(pages[full], own[0], rest)] if rest else []

    def compact(self):
        """Moves the pages in use to the lowest numbers.  Returns ``(src, dst, page_map)`` for :func:`compact_pages`:
        page src[i] moves to dst[i], and page_map[p] is where page p is found afterwards (itself unless it moves).  Page
        numbers the caller keeps elsewhere have to be sent through ``page_map`` too."""
        live = len(self._refs)
        src = sorted(p for p in self._refs if p >= live)
        dst = sorted(p for p in range(live) if p not in self._refs)
        page_map = list(range(self.n_pages))
        for s, d in zip(src, dst):
            page_map[s] = d
            self._refs[d] = self._refs.pop(s)
        if src:
            self._free = list(range(self.n_pages - 1, live - 1, -1))
        return src, dst, page_map


def _new_unique_id() -> bytes:
    ident = ctypes.create_string_buffer(128)
    check(lib().b200_comm_unique_id(ident))
    return ident.raw


def share_unique_id(rank: int, world: int, make_id, group=None) -> bytes:
    """Host-side hand-off of the 128-byte communicator id: rank 0 makes it, every rank receives it, and every rank
    then confirms to every other that it is there.  A rank that died or never joined makes the hand-off fail on the
    others within the process group's timeout; that surfaces as ``B200Error`` with the NCCL status code, before any
    GPU work that would wait for the missing rank has been launched."""
    import torch.distributed as dist
    box = [make_id() if rank == 0 else None]
    try:
        dist.broadcast_object_list(box, src=0, group=group)
        present = [None] * world
        dist.all_gather_object(present, rank, group=group)
    except Exception as exc:  # a timeout or a closed connection: some rank is not there
        raise B200Error(8, f"the communicator id did not reach every rank (rank {rank} of {world}): {exc}") from exc
    if sorted(present) != list(range(world)) or not isinstance(box[0], (bytes, bytearray)) or len(box[0]) != 128:
        raise B200Error(8, f"communicator hand-off incomplete: ranks present {present}")
    return bytes(box[0])


class Comm:
    """NCCL communicator created from a unique id that rank 0 shares through
    ``torch.distributed`` (any backend: the id is 128 bytes of host data)."""

    def __init__(self, rank: int, world: int, group=None, symmetric: Optional[bool] = None):
        raw = share_unique_id(rank, world, _new_unique_id, group)
        ident = ctypes.create_string_buffer(raw, 128)
        handle = c_void_p()
        if symmetric is None:
            symmetric = os.environ.get("B200_SYMM_MEM", "1") != "0"
        symmetric = bool(symmetric) and world > 1
        check(lib().b200_comm_init_rank_ex(ident, rank, world, 0 if symmetric else 1, byref(handle)))
        self.handle, self.rank, self.world = handle, rank, world
        self._symm = None
        if symmetric and not self._attach_symmetric(group):
            check(lib().b200_comm_setup_peer_memory(handle))  # the library's own CUDA-IPC buffers instead

    def _attach_symmetric(self, group) -> bool:
        """Exchange memory from torch.distributed's symmetric-memory allocator: one block per rank, mapped into every
        rank, and (on NVSwitch systems) bound to a multicast object, which lets the tensor-parallel exchange reduce
        inside the switch.  Every rank reaches ``b200_comm_attach_memory`` whatever happened before it, so that the
        ranks agree on the outcome; False means that no rank attached."""
        import torch.distributed as dist
        nbytes = (int(os.environ.get("B200_P2P_MB", "136")) << 20) + 4096
        ptrs = (c_void_p * self.world)()
        mc = None
        keep = None
        try:
            import torch.distributed._symmetric_memory as symm_mem
            dev = torch.device("cuda", torch.cuda.current_device())
            block = symm_mem.empty(nbytes, dtype=torch.uint8, device=dev)
            hdl = symm_mem.rendezvous(block, group=group if group is not None else dist.group.WORLD)
            for r, p in enumerate(hdl.buffer_ptrs):
                ptrs[r] = p
            mc = int(hdl.multicast_ptr) or None
            keep = (block, hdl)
        except Exception:  # no symmetric memory here: attach nothing, but still take part in the agreement
            ptrs = (c_void_p * self.world)()
            mc = None
        status = lib().b200_comm_attach_memory(self.handle, nbytes, ptrs, mc)
        if status == 0:
            self._symm = keep  # the library never frees it; it lives as long as this object
            return True
        if status != 10:
            check(status)
        return False

    def peer_memory(self) -> int:
        """0: tensor-parallel partial sums travel through NCCL; 1: through peer-mapped memory (plain loads and stores
        over NVLink); 2: through peer-mapped memory bound to a multicast object (summed inside the NVLink switch)."""
        on = c_int32(0)
        check(lib().b200_comm_peer_memory(self.handle, byref(on)))
        return int(on.value)

    def exchange_buffers(self, rows_total: int, dim: int, dtype: torch.dtype):
        """(part, gathered): views of this rank's exchange memory, [rows_total, dim] of ``dtype`` each (see
        ``b200_tp_exchange_buffers``).  They alias library-managed device memory: valid while the communicator lives."""
        es = 2 if dtype == torch.bfloat16 else 4
        n = rows_total * dim * es
        part, gath = c_void_p(), c_void_p()
        check(lib().b200_tp_exchange_buffers(self.handle, n, byref(part), byref(gath)))

        def view(ptr):
            class _Raw:  # __cuda_array_interface__ lets torch wrap device memory it does not own
                __cuda_array_interface__ = {"shape": (n,), "typestr": "|u1", "data": (ptr.value, False), "version": 2}
            return torch.as_tensor(_Raw(), device="cuda").view(dtype).view(rows_total, dim)

        return view(part), view(gath)

    def reduce_norm(self, rows_total: int, dim: int, dtype: torch.dtype, x_own: torch.Tensor, gain: torch.Tensor,
                    eps: float = 1e-5, reduce: bool = True) -> None:
        check(lib().b200_tp_reduce_norm(self.handle, rows_total, dim, _dt(dtype), int(reduce), x_own.data_ptr(),
                                        gain.data_ptr(), eps, _stream()))

    def allreduce_f32(self, t: torch.Tensor) -> None:
        check(lib().b200_allreduce_f32(self.handle, t.data_ptr(), t.numel(), _stream()))

    def destroy(self) -> None:
        if self.handle:
            check(lib().b200_comm_destroy(self.handle))
            self.handle = None
            self._symm = None


# --------------------------------------------------------------------------
# plan
# --------------------------------------------------------------------------

class Plan:
    """A model on the current CUDA device: config, packed weights, buffers."""

    def __init__(self, config: Dict[str, int], dtype: torch.dtype = torch.bfloat16, *, tp_rank: int = 0,
                 tp_size: int = 1, comm: Optional[Comm] = None, rope_theta: float = 10000.0, rms_eps: float = 1e-5):
        if not torch.cuda.is_available():
            raise RuntimeError("the B200 llama path needs a CUDA device; there is no CPU implementation")
        self.config = dict(config)
        self.dtype = dtype
        self.tp_rank, self.tp_size, self.comm = tp_rank, tp_size, comm
        self.device = torch.device("cuda", torch.cuda.current_device())
        c = _Config(*[int(config[k]) for k in CONFIG_KEYS], _dt(dtype), rope_theta, rms_eps)
        self._h = c_void_p()
        check(lib().b200_plan_create(byref(c), tp_rank, tp_size, comm.handle if comm else None, byref(self._h)))
        self.packed: Optional[torch.Tensor] = None
        self.with_transposed = False
        self._ws: Optional[torch.Tensor] = None
        self._ws_pinned_by_graphs = []  # workspaces that captured graphs point into: kept alive with the plan
        self.vocab_local = config["vocab_size"] // tp_size
        self.d_local = config["dim"] // tp_size

    def close(self) -> None:
        if self._h:
            lib().b200_plan_destroy(self._h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- buffers ---------------------------------------------------------
    def _bytes(self, fn, *args) -> int:
        n = c_size_t(0)
        check(fn(self._h, *args, byref(n)))
        return n.value

    def workspace(self, mode: int, batch: int, seq: int) -> torch.Tensor:
        need = self._bytes(lib().b200_workspace_bytes, mode, batch, seq)
        if self._ws is None or self._ws.numel() < need:
            if not any(self._ws is t for t in self._ws_pinned_by_graphs):
                self._ws = None  # free before the larger allocation, unless a captured graph still points into it
            self._ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        return self._ws

    def _check_capturable(self) -> None:
        if self.tp_size > 1:
            raise B200Error(10, "a tensor-parallel plan cannot be captured into a CUDA graph: the peer exchange "
                                "numbers its rounds from the host; launch its steps eagerly")

    def saved_bytes(self, batch: int, seq: int) -> int:
        return self._bytes(lib().b200_saved_bytes, batch, seq)

    def grad_bytes(self) -> int:
        return self._bytes(lib().b200_packed_grad_bytes)

    # ---- weights ---------------------------------------------------------
    def pack_weights(self, weights: Dict[str, torch.Tensor], with_transposed: bool = False) -> None:
        """``weights``: the reference's weight dict (full, unsharded leaves) on this device."""
        leaves = []
        dts = set()
        for name in LEAF_ORDER:
            t = weights[name]
            if not t.is_cuda or not t.is_contiguous():
                raise B200Error(1, f"leaf {name} must be a contiguous CUDA tensor")
            leaves.append(t)
            dts.add(t.dtype)
        if len(dts) != 1:
            raise B200Error(3, "all leaves must share one dtype")
        n = self._bytes(lib().b200_packed_weight_bytes, int(with_transposed))
        self.packed = torch.empty(n, dtype=torch.uint8, device=self.device)
        arr = (c_void_p * len(leaves))(*[t.data_ptr() for t in leaves])
        check(lib().b200_pack_weights(self._h, arr, _dt(dts.pop()), int(with_transposed), self.packed.data_ptr(),
                                      _stream()))
        self.with_transposed = with_transposed

    def pack_tangents(self, tangents: Dict[str, torch.Tensor]) -> torch.Tensor:
        """Packs a dict of weight-leaf tangents (same names and shapes as the weights; missing leaves count as zero)
        into the layout of the weights, for ``forward_jvp``."""
        cfg = self.config
        L, d, h, V = cfg["n_layers"], cfg["dim"], cfg["hidden_dim"], cfg["vocab_size"]
        shapes = {"rms_att_weight": (L, d), "rms_ffn_weight": (L, d), "rms_final_weight": (d,),
                  "token_embedding_table": (V, d), "w1": (L, h, d), "w2": (L, d, h), "w3": (L, h, d), "wcls": (V, d),
                  "wk": (L, d, d), "wo": (L, d, d), "wq": (L, d, d), "wv": (L, d, d)}
        leaves = []
        for name in LEAF_ORDER:
            t = tangents.get(name)
            t = torch.zeros(shapes[name], dtype=self.dtype, device=self.device) if t is None else \
                t.to(self.device, self.dtype).contiguous()
            if tuple(t.shape) != shapes[name]:
                raise B200Error(2, f"tangent of {name} has shape {tuple(t.shape)}, expected {shapes[name]}")
            leaves.append(t)
        n = self._bytes(lib().b200_packed_weight_bytes, 0)
        packed = torch.empty(n, dtype=torch.uint8, device=self.device)
        arr = (c_void_p * len(leaves))(*[t.data_ptr() for t in leaves])
        check(lib().b200_pack_weights(self._h, arr, _dt(self.dtype), 0, packed.data_ptr(), _stream()))
        return packed

    def forward_jvp(self, tokens: torch.Tensor, tangents: Dict[str, torch.Tensor]):
        """``jax.jvp``-shaped: returns ``(logits, dlogits)`` for the tangents of the weight leaves."""
        B, S = tokens.shape
        tok = tokens.to(self.device, torch.int32).contiguous()
        saved = self.new_saved(B, S)
        logits = self.forward(tok, saved=saved)
        packed_dw = self.pack_tangents(tangents)
        dlogits = torch.empty(B, S, self.vocab_local, dtype=torch.float32, device=self.device)
        need = self._bytes(lib().b200_jvp_workspace_bytes, B, S)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        check(lib().b200_forward_jvp(self._h, tok.data_ptr(), B, S, self.packed.data_ptr(), packed_dw.data_ptr(),
                                     saved.data_ptr(), dlogits.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
        return logits, dlogits

    # ---- run-time options -------------------------------------------------
    def set_option(self, name: str, value: int) -> None:
        """Sets a run-time option of the plan (``b200_plan_set_option``), e.g. ``"tp_pipeline"``; every rank of a
        tensor-parallel plan must set the same value."""
        check(lib().b200_plan_set_option(self._h, name.encode(), int(value)))

    def get_option(self, name: str) -> int:
        v = c_int32(0)
        check(lib().b200_plan_get_option(self._h, name.encode(), byref(v)))
        return int(v.value)

    def tune_tensor_parallel(self, tokens: torch.Tensor, logits: Optional[torch.Tensor] = None, reps: int = 2,
                             group=None) -> Dict[str, float]:
        """Times the tensor-parallel prefill of ``tokens`` both ways - one batch with the exchange between the
        kernels, and two halves with the exchange of one beside the compute of the other - and keeps the faster one
        (``"tp_pipeline"``).  Which one wins depends on the rank count and on the NVLink fabric of the moment, so it is
        measured, during warm-up, and not assumed.  Collective: every rank calls it with the same shapes; the ranks
        agree through a MAX all-reduce of their device times over ``group`` (default: the world group), so they all
        keep the same choice.  Returns the two times in ms and the choice."""
        if self.tp_size < 2:
            return {"one_batch_ms": 0.0, "two_halves_ms": 0.0, "tp_pipeline": 0}
        import torch.distributed as dist
        times = []
        for mode in (0, 1):
            self.set_option("tp_pipeline", mode)
            self.forward(tokens, logits=logits)  # first call of a variant: kernel attributes, workspace
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            dist.barrier(group=group)
            a.record()
            for _ in range(reps):
                self.forward(tokens, logits=logits)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) / reps)
        t = torch.tensor(times, dtype=torch.float64, device=self.device)
        dist.all_reduce(t, op=dist.ReduceOp.MAX, group=group)
        one, two = float(t[0]), float(t[1])
        choice = 1 if two < one else 0
        self.set_option("tp_pipeline", choice)
        return {"one_batch_ms": one, "two_halves_ms": two, "tp_pipeline": choice}

    # ---- forward / backward ---------------------------------------------
    def forward(self, tokens: torch.Tensor, *, saved: Optional[torch.Tensor] = None,
                kv_out: Optional[torch.Tensor] = None, logits: Optional[torch.Tensor] = None) -> torch.Tensor:
        """tokens int32 [B,S] on the device -> fp32 logits [B,S,V/tp]."""
        B, S = tokens.shape
        if tokens.dtype != torch.int32 or not tokens.is_cuda:
            raise B200Error(3, "tokens must be an int32 CUDA tensor")
        if logits is None:
            logits = torch.empty(B, S, self.vocab_local, dtype=torch.float32, device=self.device)
        ws = self.workspace(1 if saved is not None else 0, B, S)
        check(lib().b200_forward(self._h, tokens.data_ptr(), B, S, self.packed.data_ptr(), logits.data_ptr(),
                                 _ptr(saved), _ptr(kv_out), ws.data_ptr(), ws.numel(), _stream()))
        return logits

    def capture_forward(self, tokens: torch.Tensor, logits: torch.Tensor) -> "torch.cuda.CUDAGraph":
        """Captures one forward over fixed token / logits buffers into a CUDA graph (the kernel sequence of a
        plan is static, so a replay costs one launch instead of 1 + 7L + 2).  Run one eager forward first so that
        the workspace exists and every kernel attribute is set outside the capture.  The graph points into the plan's
        workspace of this moment, which the plan keeps alive from here on even when a later, larger call replaces it."""
        self._check_capturable()
        self.forward(tokens, logits=logits)
        torch.cuda.synchronize()
        self._ws_pinned_by_graphs.append(self._ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self.forward(tokens, logits=logits)
        return graph

    def capture_prefill_step(self, host_tokens: torch.Tensor, tokens: torch.Tensor, logits: torch.Tensor,
                             last_logits: torch.Tensor, host_last_logits: torch.Tensor) -> "torch.cuda.CUDAGraph":
        """One serving step as a single CUDA graph: upload `host_tokens` (pinned) into `tokens`, run the forward,
        gather the last-position logits of every sequence into `last_logits` and copy them to
        `host_last_logits` (pinned).  Copies inside the graph keep consecutive replays back to back; separate
        copy calls between replays cost more than the copies themselves."""
        if not (host_tokens.is_pinned() and host_last_logits.is_pinned()):
            raise B200Error(1, "host buffers of a captured step must be pinned")
        self._check_capturable()
        self.forward(tokens, logits=logits)
        torch.cuda.synchronize()
        self._ws_pinned_by_graphs.append(self._ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tokens.copy_(host_tokens, non_blocking=True)
            self.forward(tokens, logits=logits)
            last_logits.copy_(logits[:, -1, :])
            host_last_logits.copy_(last_logits, non_blocking=True)
        return graph

    def new_saved(self, batch: int, seq: int) -> torch.Tensor:
        return torch.empty(self.saved_bytes(batch, seq), dtype=torch.uint8, device=self.device)

    def new_grads(self) -> torch.Tensor:
        return torch.zeros(self.grad_bytes() // 4, dtype=torch.float32, device=self.device)

    def backward(self, tokens: torch.Tensor, dlogits: torch.Tensor, saved: torch.Tensor, grads: torch.Tensor,
                 accumulate: bool = False) -> torch.Tensor:
        if not self.with_transposed:
            raise B200Error(1, "backward needs weights packed with with_transposed=True")
        B, S = tokens.shape
        ws = self.workspace(2, B, S)
        check(lib().b200_backward(self._h, tokens.data_ptr(), B, S, self.packed.data_ptr(), dlogits.data_ptr(),
                                  saved.data_ptr(), grads.data_ptr(), int(accumulate), ws.data_ptr(), ws.numel(),
                                  _stream()))
        return grads

    def unpack_grads(self, grads: torch.Tensor) -> Dict[str, torch.Tensor]:
        cfg = self.config
        L, d, h, V = cfg["n_layers"], cfg["dim"], cfg["hidden_dim"], cfg["vocab_size"]
        shapes = {
            "rms_att_weight": (L, d), "rms_ffn_weight": (L, d), "rms_final_weight": (d,),
            "token_embedding_table": (V, d), "w1": (L, h, d), "w2": (L, d, h), "w3": (L, h, d), "wcls": (V, d),
            "wk": (L, d, d), "wo": (L, d, d), "wq": (L, d, d), "wv": (L, d, d),
        }
        out = {k: torch.empty(shapes[k], dtype=torch.float32, device=self.device) for k in LEAF_ORDER}
        arr = (c_void_p * len(LEAF_ORDER))(*[out[k].data_ptr() for k in LEAF_ORDER])
        check(lib().b200_unpack_grads(self._h, grads.data_ptr(), arr, _stream()))
        return out

    def token_forward(self, x: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor) -> torch.Tensor:
        """The reference's call over flat caches: ``forward(x, weights, key_cache, value_cache) -> hidden`` with
        ``x`` fp32 [d] and caches [L, pos, d]."""
        L, d = self.config["n_layers"], self.config["dim"]
        pos = int(key_cache.shape[1])
        if tuple(key_cache.shape) != (L, pos, d) or tuple(value_cache.shape) != (L, pos, d):
            raise B200Error(2, f"caches must be [{L}, pos, {d}], got {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
        dev = self.device
        xin = x.to(dev, torch.float32).reshape(d).contiguous()
        kc = key_cache.to(dev, self.dtype).contiguous()
        vc = value_cache.to(dev, self.dtype).contiguous()
        hidden = torch.empty(d, dtype=torch.float32, device=dev)
        need = self._bytes(lib().b200_token_vjp_workspace_bytes, pos)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        check(lib().b200_token_forward(self._h, xin.data_ptr(), kc.data_ptr() if pos else None,
                                       vc.data_ptr() if pos else None, pos, self.packed.data_ptr(), hidden.data_ptr(),
                                       ws.data_ptr(), ws.numel(), _stream()))
        return hidden

    def token_jvp(self, x, key_cache, value_cache, dx, dweights: Dict[str, torch.Tensor], d_key_cache, d_value_cache):
        """Forward mode of the reference's own call with tangents for all of its inputs (``jax.jvp(fn, ins, dins)``).
        Returns ``(hidden, d_hidden)``, both fp32 [d]."""
        L, d = self.config["n_layers"], self.config["dim"]
        pos = int(key_cache.shape[1])
        for name, c in (("key_cache", key_cache), ("value_cache", value_cache), ("d_key_cache", d_key_cache),
                        ("d_value_cache", d_value_cache)):
            if tuple(c.shape) != (L, pos, d):
                raise B200Error(2, f"{name} must be [{L}, {pos}, {d}], got {tuple(c.shape)}")
        dev = self.device
        f32 = lambda t: t.to(dev, torch.float32).reshape(d).contiguous()
        cd = lambda t: t.to(dev, self.dtype).contiguous()
        xin, dxin = f32(x), f32(dx)
        kc, vc, dkc, dvc = cd(key_cache), cd(value_cache), cd(d_key_cache), cd(d_value_cache)
        packed_dw = self.pack_tangents(dweights)
        hidden = torch.empty(d, dtype=torch.float32, device=dev)
        d_hidden = torch.empty(d, dtype=torch.float32, device=dev)
        need = self._bytes(lib().b200_token_jvp_workspace_bytes, pos)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        ptr = lambda t: t.data_ptr() if pos else None
        check(lib().b200_token_jvp(self._h, xin.data_ptr(), ptr(kc), ptr(vc), pos, self.packed.data_ptr(),
                                   dxin.data_ptr(), packed_dw.data_ptr(), ptr(dkc), ptr(dvc), hidden.data_ptr(),
                                   d_hidden.data_ptr(), ws.data_ptr(), ws.numel(), _stream()))
        return hidden, d_hidden

    def token_vjp(self, x: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, d_hidden: torch.Tensor):
        """Reverse mode of the reference's own call ``forward(x, weights, key_cache, value_cache) -> hidden`` with
        respect to all of its inputs.  ``x`` fp32 [d]; caches [L, pos, d]; ``d_hidden`` fp32 [d].  Returns
        ``(hidden, dx, packed_grads, d_key_cache, d_value_cache)``; ``unpack_grads`` turns the packed gradients into
        the per-leaf dict (``wcls`` and the embedding come out exactly zero: the result does not depend on them)."""
        if not self.with_transposed:
            raise B200Error(1, "token_vjp needs weights packed with with_transposed=True")
        L, d = self.config["n_layers"], self.config["dim"]
        pos = int(key_cache.shape[1])
        if tuple(key_cache.shape) != (L, pos, d) or tuple(value_cache.shape) != (L, pos, d):
            raise B200Error(2, f"caches must be [{L}, pos, {d}], got {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
        dev = self.device
        xin = x.to(dev, torch.float32).reshape(d).contiguous()
        dh = d_hidden.to(dev, torch.float32).reshape(d).contiguous()
        kc = key_cache.to(dev, self.dtype).contiguous()
        vc = value_cache.to(dev, self.dtype).contiguous()
        hidden = torch.empty(d, dtype=torch.float32, device=dev)
        dx = torch.empty(d, dtype=torch.float32, device=dev)
        dkc = torch.zeros(L, pos, d, dtype=torch.float32, device=dev)
        dvc = torch.zeros(L, pos, d, dtype=torch.float32, device=dev)
        grads = torch.empty(self.grad_bytes() // 4, dtype=torch.float32, device=dev)
        need = self._bytes(lib().b200_token_vjp_workspace_bytes, pos)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        check(lib().b200_token_vjp(self._h, xin.data_ptr(), kc.data_ptr() if pos else None,
                                   vc.data_ptr() if pos else None, pos, self.packed.data_ptr(), dh.data_ptr(),
                                   hidden.data_ptr(), dx.data_ptr(), grads.data_ptr(),
                                   dkc.data_ptr() if pos else None, dvc.data_ptr() if pos else None, ws.data_ptr(),
                                   ws.numel(), _stream()))
        return hidden, dx, grads, dkc, dvc

    # ---- decode ----------------------------------------------------------
    def new_kv_pages(self, n_pages: int, page_size: int) -> torch.Tensor:
        L = self.config["n_layers"]
        hs = self.config["dim"] // self.config["n_heads"]
        return torch.zeros(L, 2, n_pages, self.d_local // hs, page_size, hs, dtype=self.dtype, device=self.device)

    def decode_step(self, pos: int, kv_pages: torch.Tensor, page_table: torch.Tensor, *,
                    tokens: Optional[torch.Tensor] = None, x: Optional[torch.Tensor] = None,
                    want_hidden: bool = False, want_logits: bool = True,
                    logits: Optional[torch.Tensor] = None):
        B = (tokens if tokens is not None else x).shape[0]
        n_pages, page_size = kv_pages.shape[2], kv_pages.shape[4]
        hidden = torch.empty(B, self.config["dim"], dtype=torch.float32, device=self.device) if want_hidden else None
        if want_logits and logits is None:
            logits = torch.empty(B, self.vocab_local, dtype=torch.float32, device=self.device)
        ws = self.workspace(3, B, pos + 1)
        check(lib().b200_decode_step(self._h, _ptr(tokens), _ptr(x), B, pos, self.packed.data_ptr(),
                                     kv_pages.data_ptr(), page_table.data_ptr(), n_pages, page_size,
                                     page_table.shape[1], _ptr(hidden), _ptr(logits) if want_logits else None,
                                     ws.data_ptr(), ws.numel(), _stream()))
        return hidden, (logits if want_logits else None)

    def generate(self, prompt: torch.Tensor, n_new: int, *, page_size: int = 64,
                 kv_pages: Optional[torch.Tensor] = None, allocator: Optional["PageAllocator"] = None) -> torch.Tensor:
        """Greedy decoding: prefill the int32 prompts [B, S0], then ``n_new`` decode steps whose next token is the
        on-device argmax of the step's logits (no logits leave the GPU).  KV rows live in pages taken from
        ``allocator`` (a pool of ``kv_pages``; both are created when absent) and are returned to it at the end.
        Returns int32 [B, S0 + n_new].  One GPU (the vocabulary is not sharded)."""
        if self.tp_size != 1:
            raise B200Error(10, "generate needs the whole vocabulary on one GPU")
        B, S0 = prompt.shape
        total = S0 + n_new
        if total > self.config["seq_len"]:
            raise B200Error(2, f"{total} positions exceed the plan's seq_len={self.config['seq_len']}")
        per_seq = (total + page_size - 1) // page_size
        if kv_pages is None:
            kv_pages = self.new_kv_pages(B * per_seq, page_size)
        if allocator is None:
            allocator = PageAllocator(kv_pages.shape[2])
        owned = []
        try:
            for _ in range(B):
                owned.append(allocator.alloc(per_seq))
            table = torch.tensor(owned, dtype=torch.int32, device=self.device)
            # prefill: logits of every prompt position and the rotated K / V rows, scattered into the pages
            L, H = self.config["n_layers"], self.config["n_heads"]
            hs = self.config["dim"] // H
            kv_flat = torch.empty(L, 2, B, S0, H * hs, dtype=self.dtype, device=self.device)
            logits = self.forward(prompt, kv_out=kv_flat)
            pos = torch.arange(S0, device=self.device)
            pg = table.long()[:, pos // page_size].reshape(-1)            # [B*S0] page of every (sequence, position)
            off = (pos % page_size).repeat(B)
            # advanced indices on the page and row dimensions come first in the indexed view: [B*S0, L, 2, H, hs]
            kv_pages[:, :, pg, :, off, :] = kv_flat.view(L, 2, B * S0, H, hs).permute(2, 0, 1, 3, 4)
            out = torch.empty(B, total, dtype=torch.int32, device=self.device)
            out[:, :S0] = prompt
            cur = argmax(logits[:, -1, :])
            step_logits = torch.empty(B, self.vocab_local, dtype=torch.float32, device=self.device)
            for i in range(n_new):
                out[:, S0 + i] = cur
                if i + 1 == n_new:
                    break
                self.decode_step(S0 + i, kv_pages, table, tokens=cur, logits=step_logits)
                cur = argmax(step_logits)
            return out
        finally:
            for pages in owned:
                allocator.free(pages)
