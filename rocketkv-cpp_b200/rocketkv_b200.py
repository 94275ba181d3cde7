"""Python front end of librkv_b200.so (the C ABI in include/rkv.h).

This module mirrors the reference's rocket.h interface for Python callers
(tests, benchmark, torch.distributed drivers): ``compute_rocket_params``,
``compute_prefill_eviction`` and ``compute_hybrid_sparse_decode`` with the
reference's argument meaning, plus the device-resident batched entry points
that take torch CUDA tensors.  Every call goes through the CUDA library; if
the library is missing, loading raises -- there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import os
from dataclasses import dataclass, fields

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "librkv_b200.so")

RKV_OK = 0
RKV_ERR_INVALID_ARG = 1
RKV_ERR_UNSUPPORTED = 2
RKV_ERR_CUDA = 3
RKV_ERR_WORKSPACE = 4
RKV_ERR_DEVICE_TIMEOUT = 5
RKV_ERR_NO_DEVICE = 6

F32, BF16, Q8_0, F16 = 0, 1, 2, 3
ENGINE_AUTO, ENGINE_SIMT, ENGINE_TENSOR, ENGINE_TENSOR_TILES = 0, 1, 2, 3

# Every symbol include/rkv.h declares.
EXPORTS = [
    "rkv_abi_version", "rkv_status_string", "rkv_config_init", "rkv_compute_params",
    "rkv_evict_max_kept", "rkv_evict_workspace_size", "rkv_evict", "rkv_evict_pool_heads",
    "rkv_evict_select_pooled", "rkv_prefill_eviction_host", "rkv_hsa_sel_capacity",
    "rkv_hsa_workspace_size", "rkv_hsa_decode", "rkv_hybrid_sparse_decode_host",
    "rkv_hsa_decode_host_ex", "rkv_workspace_status", "rkv_hsa_decode_noalloc", "rkv_hsa_decode_noalloc_status",
    "rkv_selftest_wait_timeout", "rkv_compact_kv", "rkv_hsa_summary_size", "rkv_hsa_build_summary",
    "rkv_hsa_decode_summary", "rkv_capture_rows", "rkv_evict_compact", "rkv_paged_append",
    "rkv_paged_decode_workspace_size", "rkv_paged_decode", "rkv_weight_evict",
    "rkv_sink_attention_workspace_size", "rkv_sink_attention",
]


class RkvError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {status_string(status)} (status {status})")


class _Config(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in (
        "num_heads", "num_heads_kv", "dim_head", "window_size", "kernel_size",
        "prompt_budget", "topk_decode", "chunk_size", "r_dim")] + [("compression_ratio", ctypes.c_float)]


class _Budget(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in (
        "token_budget", "sequence_length", "max_new_tokens", "capacity_budget",
        "prompt_budget", "chunk_size", "r", "k")] + [("compression_ratio", ctypes.c_float)]


class _PagedCache(ctypes.Structure):
    _fields_ = ([("K", ctypes.c_void_p), ("V", ctypes.c_void_p)]
                + [(n, ctypes.c_int) for n in ("dtype", "num_heads_kv", "dim_head", "page_size", "num_pages",
                                               "table_stride")]
                + [(n, ctypes.c_longlong) for n in ("page_stride", "head_stride", "token_stride")]
                + [("block_table", ctypes.c_void_p), ("lens", ctypes.c_void_p)])


class _RowStrides(ctypes.Structure):
    _fields_ = [(n, ctypes.c_longlong) for n in ("item", "head", "token")]


@dataclass
class RocketConfig:
    """Mirror of the reference RocketConfig (rocket.h:18-34); same defaults."""

    num_heads: int = 0
    num_heads_kv: int = 0
    dim_head: int = 0
    window_size: int = 32
    kernel_size: int = 63
    prompt_budget: int = 0
    topk_decode: int = 0
    chunk_size: int = 0
    r_dim: int = 0
    compression_ratio: float = 0.0

    def c(self) -> _Config:
        return _Config(*[getattr(self, f.name) for f in fields(self)])


@dataclass
class RocketBudgetParams:
    """Mirror of the reference RocketBudgetParams (rocket.h:5-15)."""

    token_budget: int
    sequence_length: int
    max_new_tokens: int
    capacity_budget: int
    prompt_budget: int
    chunk_size: int
    r: int
    k: int
    compression_ratio: float


_lib = None
_VP = ctypes.c_void_p
_I = ctypes.c_int
_LL = ctypes.c_longlong
_SZ = ctypes.c_size_t
_CFGP = ctypes.POINTER(_Config)
_PCP = ctypes.POINTER(_PagedCache)
_RSP = ctypes.POINTER(_RowStrides)


def lib() -> ctypes.CDLL:
    """Loads librkv_b200.so (raises if it was not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise FileNotFoundError(
            f"{LIB_PATH} is missing; build it with `make -C rocketkv-cpp_b200` "
            "(the CUDA library is required, there is no CPU fallback)")
    L = ctypes.CDLL(LIB_PATH)
    sig = {
        "rkv_abi_version": ([], _I),
        "rkv_status_string": ([_I], ctypes.c_char_p),
        "rkv_config_init": ([_CFGP], None),
        "rkv_compute_params": ([_I, _I, _I, _I, _I, ctypes.POINTER(_Budget)], _I),
        "rkv_evict_max_kept": ([_CFGP, _I, _I], _I),
        "rkv_evict_workspace_size": ([_CFGP, _I, _I, _I, _I, ctypes.POINTER(_SZ)], _I),
        "rkv_evict": ([_VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _VP, _I, _VP, _VP, _SZ, _I, _VP], _I),
        "rkv_evict_pool_heads": ([_VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _I, _I, _VP, _VP, _SZ, _I, _VP], _I),
        "rkv_evict_select_pooled": ([_VP, _I, _I, _I, _CFGP, _VP, _I, _VP, _VP, _SZ, _VP], _I),
        "rkv_prefill_eviction_host": ([_VP, _VP, _I, _I, _CFGP, _VP, _I, ctypes.POINTER(_I)], _I),
        "rkv_hsa_sel_capacity": ([_CFGP, _I, _I], _I),
        "rkv_hsa_workspace_size": ([_CFGP, _I, _I, _I, _I, ctypes.POINTER(_SZ)], _I),
        "rkv_hsa_decode": ([_VP, _VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _I, _I, _VP, _VP, _I, _VP,
                            _VP, _SZ, _VP], _I),
        "rkv_hybrid_sparse_decode_host": ([_VP, _VP, _VP, _I, _CFGP, _VP], _I),
        "rkv_hsa_decode_host_ex": ([_VP, _VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _VP, _VP, _I, _VP], _I),
        "rkv_workspace_status": ([_VP, _VP], _I),
        "rkv_selftest_wait_timeout": ([_VP, _VP], _I),
        "rkv_hsa_decode_noalloc": ([_VP, _VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _I, _I, _VP, _VP, _I, _VP,
                                    _VP], _I),
        "rkv_hsa_decode_noalloc_status": ([_VP], _I),
        "rkv_capture_rows": ([_VP, _I, _I, _I, _I, _LL, _LL, _I, _VP, _I, _I, _I, _LL, _I, _VP], _I),
        "rkv_evict_compact": ([_VP, _VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _VP, _I, _VP, _VP, _VP, _I, _LL,
                               _VP, _SZ, _I, _VP], _I),
        "rkv_compact_kv": ([_VP, _VP, _I, _I, _I, _I, _I, _LL, _VP, _VP, _I, _VP, _VP, _I, _LL, _VP], _I),
        "rkv_hsa_summary_size": ([_CFGP, _I, _I, _I, _I, ctypes.POINTER(_SZ)], _I),
        "rkv_hsa_build_summary": ([_VP, _I, _I, _I, _I, _LL, _CFGP, _VP, _VP], _I),
        "rkv_hsa_decode_summary": ([_VP, _VP, _VP, _VP, _I, _I, _I, _I, _LL, _LL, _CFGP, _I, _I, _VP, _VP, _I,
                                    _VP, _VP, _SZ, _VP], _I),
        "rkv_paged_append": ([_PCP, _VP, _VP, _I, _I, _LL, _LL, _LL, _VP, _VP], _I),
        "rkv_paged_decode_workspace_size": ([_I, _I, _I, _I, _I, _I, ctypes.POINTER(_SZ)], _I),
        "rkv_paged_decode": ([_VP, _LL, _I, _PCP, _I, _I, _I, _I, _VP, _VP, _VP, _I, _VP, _SZ, _VP], _I),
        "rkv_weight_evict": ([_PCP, _VP, _I, _I, _I, _I, _I, _I, _PCP, _VP, _VP, _I, _VP, _VP], _I),
        "rkv_sink_attention_workspace_size": ([_I, _I, _I, _I, _I, _I, _I, ctypes.POINTER(_SZ)], _I),
        "rkv_sink_attention": ([_VP, _VP, _VP, _I, _I, _I, _I, _I, _I, _I, _RSP, _RSP, _VP, _I, _I, _VP, _RSP, _VP,
                                _VP, _SZ, _VP], _I),
    }
    for name, (args, res) in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = res
    _lib = L
    return L


def status_string(st: int) -> str:
    return lib().rkv_status_string(st).decode()


def _check(st: int, what: str) -> None:
    if st != RKV_OK:
        raise RkvError(st, what)


def _ptr(a) -> int:
    """Address of a numpy array or torch tensor (0 for None)."""
    if a is None:
        return 0
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    return a.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return int(stream)


_raw_stream = None


def _current_stream(index: int) -> int:
    """The device's current stream as a number; torch's Stream object, which
    costs microseconds to make, only where torch lacks the direct query."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda i: torch.cuda.current_stream(i).cuda_stream)
    return _raw_stream(index)


# ---------------------------------------------------------------------------
# rocket.h mirror (host buffers, synchronous)
# ---------------------------------------------------------------------------
def compute_rocket_params(token_budget: int, sequence_length: int, max_new_tokens: int,
                          head_dim: int, window_size: int = 32) -> RocketBudgetParams:
    """rocket.h:36-41."""
    b = _Budget()
    _check(lib().rkv_compute_params(token_budget, sequence_length, max_new_tokens, head_dim,
                                    window_size, ctypes.byref(b)), "compute_rocket_params")
    return RocketBudgetParams(*[getattr(b, n) for n, _ in _Budget._fields_])


def compute_prefill_eviction(Q: np.ndarray, K: np.ndarray, len_q: int, len_k: int,
                             cfg: RocketConfig) -> np.ndarray:
    """rocket.h:43-46: fp32 host Q [H, len_q, D], K [HK, len_k, D] -> kept indices."""
    Q = np.ascontiguousarray(Q, np.float32)
    K = np.ascontiguousarray(K, np.float32)
    c = cfg.c()
    cap = lib().rkv_evict_max_kept(ctypes.byref(c), len_q, len_k)
    if cap < 0:
        raise RkvError(-cap, "compute_prefill_eviction")
    out = np.zeros(cap, np.int32)
    n = _I(0)
    _check(lib().rkv_prefill_eviction_host(_ptr(Q), _ptr(K), len_q, len_k, ctypes.byref(c),
                                           _ptr(out), cap, ctypes.byref(n)),
           "compute_prefill_eviction")
    return out[: n.value].copy()


def compute_hybrid_sparse_decode(Q: np.ndarray, K: np.ndarray, V: np.ndarray, len_k: int,
                                 cfg: RocketConfig) -> np.ndarray:
    """rocket.h:48-50: fp32 host Q [H, D], K/V [HK, len_k, D] -> O [H * D]."""
    Q = np.ascontiguousarray(Q, np.float32)
    K = np.ascontiguousarray(K, np.float32)
    V = np.ascontiguousarray(V, np.float32)
    O = np.zeros(cfg.num_heads * cfg.dim_head, np.float32)
    c = cfg.c()
    _check(lib().rkv_hybrid_sparse_decode_host(_ptr(Q), _ptr(K), _ptr(V), len_k, ctypes.byref(c),
                                               _ptr(O)), "compute_hybrid_sparse_decode")
    return O


def hsa_decode_host(Q: np.ndarray, K: np.ndarray, V: np.ndarray, dtype: int, len_k: int,
                    cfg: RocketConfig, recent_window: int = 0, with_sel: bool = False):
    """Host-buffer stage 2, any dtype and batch.  Q [B, H, D], K/V [B, HK, len_k, D]
    as float32 or uint16 (bf16 bits).  Returns O [B, H, D] (and sel, n_sel)."""
    B = Q.shape[0]
    c = cfg.c()
    O = np.zeros((B, cfg.num_heads, cfg.dim_head), np.float32)
    cap = lib().rkv_hsa_sel_capacity(ctypes.byref(c), len_k, recent_window)
    sel = np.zeros((B, cfg.num_heads_kv, cap), np.int32) if with_sel else None
    nsel = np.zeros((B, cfg.num_heads_kv), np.int32) if with_sel else None
    _check(lib().rkv_hsa_decode_host_ex(_ptr(Q), _ptr(K), _ptr(V), dtype, len_k, recent_window, B,
                                        Q[0].nbytes, K[0].nbytes, ctypes.byref(c), _ptr(O),
                                        _ptr(sel), cap, _ptr(nsel)), "hsa_decode_host")
    return (O, sel, nsel) if with_sel else O


# ---------------------------------------------------------------------------
# Device-resident batched entry points (torch CUDA tensors)
# ---------------------------------------------------------------------------
def evict_max_kept(cfg: RocketConfig, len_q: int, len_k: int) -> int:
    c = cfg.c()
    n = lib().rkv_evict_max_kept(ctypes.byref(c), len_q, len_k)
    if n < 0:
        raise RkvError(-n, "evict_max_kept")
    return n


def evict_workspace_size(cfg: RocketConfig, dtype: int, len_q: int, len_k: int, batch: int) -> int:
    c = cfg.c()
    b = _SZ(0)
    _check(lib().rkv_evict_workspace_size(ctypes.byref(c), dtype, len_q, len_k, batch, ctypes.byref(b)),
           "evict_workspace_size")
    return b.value


def hsa_sel_capacity(cfg: RocketConfig, len_k: int, recent_window: int = 0) -> int:
    c = cfg.c()
    n = lib().rkv_hsa_sel_capacity(ctypes.byref(c), len_k, recent_window)
    if n < 0:
        raise RkvError(-n, "hsa_sel_capacity")
    return n


def hsa_workspace_size(cfg: RocketConfig, len_k: int, recent_window: int, batch: int,
                       head_count: int) -> int:
    c = cfg.c()
    b = _SZ(0)
    _check(lib().rkv_hsa_workspace_size(ctypes.byref(c), len_k, recent_window, batch, head_count,
                                        ctypes.byref(b)), "hsa_workspace_size")
    return b.value


def _dtype_of(t) -> int:
    import torch
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    if t.dtype == torch.float16:
        return F16
    if t.dtype == torch.uint8:
        return Q8_0
    raise TypeError(f"unsupported tensor dtype {t.dtype}")


def _workspace(nbytes: int, device):
    import torch
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


class Evictor:
    """Stage 1 on device tensors.  Q [B, H, len_q, D*], K [B, HK, len_k, D*]
    (float32, bfloat16, or uint8 q8_0 rows), one workspace reused across calls."""

    def __init__(self, cfg: RocketConfig, len_q: int, len_k: int, batch: int, dtype: int, device):
        import torch
        self.cfg, self.len_q, self.len_k, self.batch, self.dtype = cfg, len_q, len_k, batch, dtype
        self.c = cfg.c()
        self.max_kept = evict_max_kept(cfg, len_q, len_k)
        self.ws_bytes = evict_workspace_size(cfg, dtype, len_q, len_k, batch)
        self.ws = _workspace(self.ws_bytes, device)
        self.kept = torch.zeros((batch, self.max_kept), dtype=torch.int32, device=device)
        self.n_kept = torch.zeros(batch, dtype=torch.int32, device=device)

    def __call__(self, Q, K, stream=None, engine: int = ENGINE_AUTO):
        assert Q.is_contiguous() and K.is_contiguous() and Q.shape[0] == K.shape[0] == self.batch
        _check(lib().rkv_evict(_ptr(Q), _ptr(K), self.dtype, self.len_q, self.len_k, self.batch,
                               Q[0].nbytes if self.batch else 0, K[0].nbytes if self.batch else 0,
                               ctypes.byref(self.c), _ptr(self.kept), self.max_kept, _ptr(self.n_kept),
                               _ptr(self.ws), self.ws_bytes, engine, _stream(stream)), "rkv_evict")
        return self.kept, self.n_kept

    def evict_compact(self, Q, K, V=None, K_out=None, V_out=None, stream=None, engine: int = ENGINE_AUTO):
        """Stage 1 on Q and the cache's K, then the cache compacted to the kept
        rows in the same call (rkv_evict_compact): in place without K_out /
        V_out, else into K_out / V_out [B, HK, out_len, D*].  Returns (kept, n_kept)."""
        assert Q.is_contiguous() and K.is_contiguous() and (V is None or V.is_contiguous())
        if K_out is None:
            K_out, V_out = K, V
        _check(lib().rkv_evict_compact(_ptr(Q), _ptr(K), _ptr(V) if V is not None else None, self.dtype, self.len_q,
                                       self.len_k, self.batch, Q[0].nbytes if self.batch else 0,
                                       K[0].nbytes if self.batch else 0, ctypes.byref(self.c), _ptr(self.kept),
                                       self.max_kept, _ptr(self.n_kept), _ptr(K_out),
                                       _ptr(V_out) if V_out is not None else None, K_out.shape[2],
                                       K_out[0].nbytes if self.batch else 0, _ptr(self.ws), self.ws_bytes, engine,
                                       _stream(stream)), "rkv_evict_compact")
        return self.kept, self.n_kept

    def pool_heads(self, Q, K, head_begin: int, head_count: int, pooled, stream=None, engine: int = ENGINE_AUTO):
        _check(lib().rkv_evict_pool_heads(_ptr(Q), _ptr(K), self.dtype, self.len_q, self.len_k,
                                          self.batch, Q[0].nbytes, K[0].nbytes, ctypes.byref(self.c),
                                          head_begin, head_count, _ptr(pooled), _ptr(self.ws),
                                          self.ws_bytes, engine, _stream(stream)),
               "rkv_evict_pool_heads")
        return pooled

    def select_pooled(self, pooled, stream=None):
        _check(lib().rkv_evict_select_pooled(_ptr(pooled), self.len_q, self.len_k, self.batch,
                                             ctypes.byref(self.c), _ptr(self.kept), self.max_kept,
                                             _ptr(self.n_kept), _ptr(self.ws), self.ws_bytes,
                                             _stream(stream)), "rkv_evict_select_pooled")
        return self.kept, self.n_kept


def compact_kv(K, V, kept, n_kept, dim_head: int, K_out=None, V_out=None, stream=None):
    """Applies kept token indices to a KV cache on the device (rkv_compact_kv).

    K, V: [B, HK, len_k, D*] (float32, bfloat16, or uint8 q8_0 rows of
    dim_head values); V may be None.  kept [B, >=n] int32 ascending, n_kept
    [B] int32 (an Evictor's outputs).  Without K_out / V_out the cache is
    compacted in place (row i of every head becomes row kept[i]); with them,
    K_out / V_out [B, HK, out_len, D*] receive the kept rows.  Returns the
    tensors written."""
    assert K.is_contiguous() and (V is None or V.is_contiguous())
    dtype = _dtype_of(K)
    B, HK, len_k = K.shape[0], K.shape[1], K.shape[2]
    if K_out is None:
        K_out, V_out = K, V
    assert K_out.is_contiguous() and (V_out is None or V_out.is_contiguous())
    _check(lib().rkv_compact_kv(_ptr(K), _ptr(V) if V is not None else None, dtype, dim_head, HK, len_k, B,
                                K[0].nbytes if B else 0, _ptr(kept), _ptr(n_kept), kept.shape[1], _ptr(K_out),
                                _ptr(V_out) if V_out is not None else None, K_out.shape[2],
                                K_out[0].nbytes if B else 0, _stream(stream)), "rkv_compact_kv")
    return K_out, V_out


def capture_rows(src, dst, token_offset: int, dst_first: int = 0, item: int = 0, stream=None):
    """The capture side on the device (rkv_capture_rows): one micro-batch of
    post-RoPE rows src [n_tokens, n_heads, dim_head] (float32, float16 or
    bfloat16, any strides along tokens and heads, unit stride along dim_head),
    global tokens token_offset .., scattered into item `item` of dst
    [items, n_heads, dst_tokens, dim_head] (float32, or bfloat16 from a
    bfloat16 source), row token - dst_first.  Returns dst."""
    assert src.dim() == 3 and src.stride(2) == 1 and dst.is_contiguous()
    n_tokens, n_heads, dim_head = src.shape
    es = src.element_size()
    _check(lib().rkv_capture_rows(_ptr(src), _dtype_of(src), n_tokens, n_heads, dim_head, src.stride(0) * es,
                                  src.stride(1) * es, token_offset, _ptr(dst), _dtype_of(dst), dst_first,
                                  dst.shape[2], dst[0].nbytes if dst.shape[0] else 0, item, _stream(stream)),
           "rkv_capture_rows")
    return dst


class HsaDecoder:
    """Stage 2 on device tensors.  Q [B, H, D], K/V [B, HK, len_k, D] (float32
    or bfloat16); KV heads [head_begin, head_begin + head_count)."""

    def __init__(self, cfg: RocketConfig, len_k: int, batch: int, device, recent_window: int = 0,
                 head_begin: int = 0, head_count: int | None = None):
        import torch
        self.cfg, self.len_k, self.batch, self.w = cfg, len_k, batch, recent_window
        self.head_begin = head_begin
        self.head_count = cfg.num_heads_kv if head_count is None else head_count
        self.c = cfg.c()
        self.sel_cap = hsa_sel_capacity(cfg, len_k, recent_window)
        self.ws_bytes = hsa_workspace_size(cfg, len_k, recent_window, batch, self.head_count)
        self.ws = _workspace(self.ws_bytes, device)
        self.O = torch.zeros((batch, cfg.num_heads, cfg.dim_head), dtype=torch.float32, device=device)
        self.sel = torch.zeros((batch, self.head_count, self.sel_cap), dtype=torch.int32, device=device)
        self.n_sel = torch.zeros((batch, self.head_count), dtype=torch.int32, device=device)

    def build_summary(self, K, stream=None, out=None):
        """Page summaries of K (every KV head) for this decoder's geometry:
        later calls with summary=... read them instead of scanning every K row.
        out: a buffer from an earlier call to rebuild into (no allocation)."""
        import torch
        dt = _dtype_of(K)
        n = ctypes.c_size_t(0)
        _check(lib().rkv_hsa_summary_size(ctypes.byref(self.c), dt, self.len_k, self.w, self.batch, ctypes.byref(n)),
               "rkv_hsa_summary_size")
        S = out if out is not None else torch.empty(max(n.value, 16), dtype=torch.uint8, device=K.device)
        assert S.numel() >= n.value
        _check(lib().rkv_hsa_build_summary(_ptr(K), dt, self.len_k, self.w, self.batch, K[0].nbytes if self.batch else 0,
                                           ctypes.byref(self.c), _ptr(S), _stream(stream)), "rkv_hsa_build_summary")
        return S

    def __call__(self, Q, K, V, stream=None, want_sel: bool = True, summary=None):
        assert Q.is_contiguous() and K.is_contiguous() and V.is_contiguous()
        assert K.shape == V.shape and Q.shape[0] == K.shape[0] == self.batch
        dt = _dtype_of(K)
        common = (dt, self.len_k, self.w, self.batch, Q[0].nbytes, K[0].nbytes, ctypes.byref(self.c), self.head_begin,
                  self.head_count, _ptr(self.O), _ptr(self.sel) if want_sel else 0, self.sel_cap,
                  _ptr(self.n_sel) if want_sel else 0, _ptr(self.ws), self.ws_bytes, _stream(stream))
        if summary is None:
            _check(lib().rkv_hsa_decode(_ptr(Q), _ptr(K), _ptr(V), *common), "rkv_hsa_decode")
        else:
            _check(lib().rkv_hsa_decode_summary(_ptr(Q), _ptr(K), _ptr(V), _ptr(summary), *common),
                   "rkv_hsa_decode_summary")
        return self.O

    def status(self, stream=None) -> int:
        return lib().rkv_workspace_status(_ptr(self.ws), _stream(stream))


# ---------------------------------------------------------------------------
# Paged KV cache: append, dense decode, eviction by accumulated weight
# ---------------------------------------------------------------------------
def _handle(device, stream) -> int:
    return _current_stream(device.index) if stream is None else int(stream)


def _stream_object(device, handle: int):
    import torch
    return torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)


def _launch(device, stream, what, fn, *args, owner=None) -> None:
    """fn(*args, stream) with the tensors' device current (a stream belongs to one)."""
    import torch
    h = _handle(device, stream)
    if owner is not None and h not in owner._streams:
        # the object's buffers belong to the stream they were made on; dropped with it while this call runs on
        # another one, they would be handed out again at once (the mark lasts, but not one set under a capture)
        other = _stream_object(device, h)
        for t in owner._buffers():
            t.record_stream(other)
        if not torch.cuda.is_current_stream_capturing():
            owner._streams.add(h)
    if device.index == torch.cuda.current_device():
        st = fn(*args, h)
    else:
        with torch.cuda.device(device):
            st = fn(*args, h)
    if st != RKV_OK:
        raise RkvError(st, what)


def _on_stream(device, stream):
    """What a call allocates and fills belongs to its stream, not to the current one."""
    import contextlib
    import torch
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(_stream_object(device, int(stream)))


def _int32(t, device, what):
    import torch
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        raise TypeError(f"{what}: a contiguous int32 tensor on {device} is needed")


class PagedCache:
    """K and V pages [num_pages, HK, page_size, D] (float32, bfloat16 or
    float16; unit stride along D, any 16-byte multiple along the others, so a
    [num_pages, page_size, HK, D] pool is passed as pool.transpose(1, 2)),
    block_table [B, table_stride] int32 and lens [B] int32, all on one device.
    Holds the tensors; lens may be replaced or updated in place between calls."""

    def __init__(self, K, V, block_table, lens):
        if K.shape != V.shape or K.stride() != V.stride() or K.dtype != V.dtype or K.dim() != 4:
            raise ValueError("K and V: [num_pages, HK, page_size, D], of one layout and type")
        if not K.is_cuda or V.device != K.device:
            raise TypeError("K and V: CUDA tensors on one device")
        pages, hk, page, d = K.shape
        if d > 1 and K.stride(3) != 1:
            raise ValueError("unit stride along the last dimension is needed")
        dt = _dtype_of(K)
        if dt == Q8_0:
            raise TypeError("a paged cache holds float32, bfloat16 or float16")
        _int32(block_table, K.device, "block_table")
        if block_table.dim() != 2:
            raise ValueError("block_table: [batch, pages per sequence]")
        self.K, self.V, self.block_table = K, V, block_table
        es = K.element_size()
        # the stride of a dimension of one entry is never used: any value passes
        st = [K.stride(i) * es if K.shape[i] > 1 else 16 * ((d * es + 15) // 16) for i in range(3)]
        self.c = _PagedCache(_ptr(K), _ptr(V), dt, hk, d, page, pages, block_table.shape[1], st[0], st[1], st[2],
                             _ptr(block_table), None)
        self.ref = ctypes.byref(self.c)
        self.batch = block_table.shape[0]
        self.lens = lens

    @property
    def lens(self):
        return self._lens

    @lens.setter
    def lens(self, t):
        if t is not None:
            _int32(t, self.K.device, "lens")
            if t.numel() != self.batch:
                raise ValueError("lens: one entry per row of block_table")
        self._lens = t
        self.c.lens = _ptr(t)


def paged_append(cache: PagedCache, k, v, n_new=None, stream=None):
    """Newest rows into the pages (rkv_paged_append).  k, v: [B, n_rows, HK, D]
    (or [B, HK, D] for one row) of the cache's type, unit stride along D, equal
    strides; cache.lens already counts them, and n_new [B] int32 (nullable)
    says how many of the n_rows each sequence has."""
    if k.dim() == 3:
        k, v = k[:, None], v[:, None]
    if k.shape != v.shape or k.stride() != v.stride() or k.dtype != cache.K.dtype or v.dtype != k.dtype:
        raise ValueError("k and v: one shape, layout and the cache's type")
    B, n, hk, d = k.shape
    if B != cache.batch or hk != cache.K.shape[1] or d != cache.K.shape[3] or (d > 1 and k.stride(3) != 1):
        raise ValueError("k, v: [B, n_rows, HK, D] of the cache's geometry, unit stride along D")
    if k.device != cache.K.device or v.device != k.device:
        raise TypeError("k and v: on the cache's device")
    if n_new is not None:
        _int32(n_new, k.device, "n_new")
        if n_new.numel() != B:
            raise ValueError("n_new: one entry per sequence")
    es = k.element_size()
    si, st, sh, _ = k.stride()
    _launch(k.device, stream, "rkv_paged_append", lib().rkv_paged_append, cache.ref, k.data_ptr(), v.data_ptr(), n, B,
            si * es, st * es, sh * es, _ptr(n_new))


class PagedDecoder:
    """One new token per sequence attended over a paged cache
    (rkv_paged_decode), with its outputs O [B, H, D] and lse [B, H] float32 and
    its workspace.  window > 0: only the first `sinks` and the last `window`
    tokens are seen.  weights=True reserves what a call that accumulates
    attention weights needs."""

    def __init__(self, num_heads: int, num_heads_kv: int, dim_head: int, max_len: int, batch: int, device, sinks: int = 0,
                 window: int = 0, weights: bool = False):
        import torch
        b = _SZ(0)
        _check(lib().rkv_paged_decode_workspace_size(num_heads, num_heads_kv, dim_head, max_len, batch, int(weights),
                                                     ctypes.byref(b)), "rkv_paged_decode_workspace_size")
        self.num_heads, self.num_heads_kv, self.dim_head = num_heads, num_heads_kv, dim_head
        self.max_len, self.batch, self.sinks, self.window = max_len, batch, sinks, window
        self.ws_bytes = b.value
        self.ws = _workspace(b.value, device)
        # each call writes all of them; a fill on this stream could run after a call on another
        self.O = torch.empty((batch, num_heads, dim_head), dtype=torch.float32, device=device)
        self.lse = torch.empty((batch, num_heads), dtype=torch.float32, device=device)
        self._streams = {_handle(self.ws.device, None)}  # whose work its buffers outlive

    def _buffers(self):
        return self.ws, self.O, self.lse

    def __call__(self, Q, cache: PagedCache, weights=None, stream=None):
        """Q [B, H, D] of the cache's type.  weights (nullable): float32
        [B, HK, >= max_len]; every visible token's attention weight, summed over
        its KV head's query heads, is added.  Returns O."""
        if Q.shape != self.O.shape or not Q.is_contiguous():
            raise ValueError("Q: contiguous [B, H, D] of the decoder's sizes")
        dev = Q.device
        if (Q.dtype != cache.K.dtype or dev != cache.K.device or dev != self.ws.device
                or cache.batch != self.batch or cache._lens is None):
            raise ValueError("Q, the cache and the decoder: one type, device and batch, and the cache's lens set")
        if (cache.c.num_heads_kv, cache.c.dim_head) != (self.num_heads_kv, self.dim_head):
            raise ValueError("the cache's heads are not the decoder's")
        wstride = _check_weights(weights, self.batch, self.num_heads_kv, self.max_len, dev)
        _launch(dev, stream, "rkv_paged_decode", lib().rkv_paged_decode, Q.data_ptr(),
                self.num_heads * self.dim_head * Q.element_size(), self.num_heads, cache.ref, self.max_len, self.batch,
                self.sinks, self.window, self.O.data_ptr(), self.lse.data_ptr(), _ptr(weights), wstride,
                self.ws.data_ptr(), self.ws_bytes, owner=self)
        return self.O


def _check_weights(w, batch, heads, max_len, device) -> int:
    """Row stride of accumulated weights [B, HK, >= max_len] (0 for None)."""
    import torch
    if w is None:
        return 0
    if (w.dtype != torch.float32 or w.device != device or not w.is_contiguous() or w.dim() != 3
            or w.shape[0] != batch or w.shape[1] != heads or w.shape[2] < max_len):
        raise ValueError("weights: contiguous float32 [B, HK, >= max_len] on the cache's device")
    return w.shape[2]


class WeightEvictor:
    """Eviction by accumulated attention weight (rkv_weight_evict): every
    (sequence, KV head) keeps its first `sinks`, its last `recent` and the
    heaviest of its other tokens, `budget` in all."""

    def __init__(self, num_heads_kv: int, max_len: int, batch: int, budget: int, device, sinks: int = 0, recent: int = 0):
        import torch
        self.num_heads_kv, self.max_len, self.batch = num_heads_kv, max_len, batch
        self.budget, self.sinks, self.recent = budget, sinks, recent
        # each call writes all of them; a fill on this stream could run after a call on another
        self.kept = torch.empty((batch, num_heads_kv, max(0, min(budget, max_len))), dtype=torch.int32, device=device)
        self.new_lens = torch.empty(batch, dtype=torch.int32, device=device)
        self._streams = {_handle(self.kept.device, None)}

    def _buffers(self):
        return self.kept, self.new_lens

    def __call__(self, cache: PagedCache, weights, out: PagedCache | None = None, weights_out=None, stream=None):
        """In place without out / weights_out.  Returns (kept [B, HK, min(budget,
        max_len)] int32 ascending with -1 behind, new_lens [B] int32), which the
        next call overwrites: copy new_lens to where the cache's lens is kept.
        A cache whose lens is this evictor's new_lens is refused."""
        dev = cache.K.device
        if cache.batch != self.batch or cache.c.num_heads_kv != self.num_heads_kv or cache._lens is None or weights is None:
            raise ValueError("the evictor's batch and KV heads, lens and weights are needed")
        if out is not None and (out.batch != self.batch or out.K.device != dev):
            raise ValueError("out: the same batch, on the cache's device")
        if self.kept.device != dev:
            raise ValueError("the cache is not on the evictor's device")
        if self.batch and cache.c.lens == self.new_lens.data_ptr():
            raise ValueError("the cache's lens is this evictor's new_lens, which the call overwrites: copy it")
        ws = _check_weights(weights, self.batch, self.num_heads_kv, self.max_len, dev)
        if weights_out is not None and _check_weights(weights_out, self.batch, self.num_heads_kv, self.max_len, dev) != ws:
            raise ValueError("weights_out: the layout of weights")
        _launch(dev, stream, "rkv_weight_evict", lib().rkv_weight_evict, cache.ref, weights.data_ptr(), ws, self.max_len,
                self.batch, self.budget, self.sinks, self.recent, out.ref if out is not None else None, _ptr(weights_out),
                self.kept.data_ptr(), self.kept.shape[2], self.new_lens.data_ptr(), owner=self)
        return self.kept, self.new_lens


def _row_strides(t, what):
    """(item, head, token) byte strides of [B, H, len, D] with unit stride along D."""
    if t.dim() != 4 or (t.shape[3] > 1 and t.stride(3) != 1):
        raise ValueError(f"{what}: [B, heads, len, D] with unit stride along D")
    es = t.element_size()
    (i, h, n, d), (si, sh, sn, _) = t.shape, t.stride()
    row = 16 * ((d * es + 15) // 16)  # the stride of a dimension of one entry is never used
    return _RowStrides(si * es if i > 1 else row, sh * es if h > 1 else row, sn * es if n > 1 else row)


class SinkAttention:
    """Causal prefill attention over a sliding window and a few first tokens
    that stay visible (rkv_sink_attention); window 0: every key up to the
    query.  Holds the workspace, which grows with the calls' sizes, at least to
    twice what it was, so that what is kept of outgrown ones stays below the
    largest: calls that may run at the same time need an object each."""

    def __init__(self, sinks: int = 0, window: int = 0, device="cuda"):
        self.sinks, self.window = sinks, window
        self.ws, self._outgrown = _workspace(0, device), []
        self._streams = {_handle(self.ws.device, None)}  # whose work its buffers outlive
        self._ran = False  # a call with work to do has used ws (and each of _outgrown), and written its error word

    def reserve(self, dtype: int, num_heads: int, num_heads_kv: int, dim_head: int, len_q: int, len_k: int, batch: int = 1,
                stream=None) -> None:
        """Makes room for calls of these sizes, under any sinks and window, as
        each call does for its own.  Few queries take more than many: their keys
        are split."""
        need = _SZ(0)
        _check(lib().rkv_sink_attention_workspace_size(dtype, len_q, len_k, batch, num_heads, num_heads_kv, dim_head,
                                                       ctypes.byref(need)), "rkv_sink_attention_workspace_size")
        if self.ws.numel() < need.value:
            if self._ran:
                self._outgrown.append(self.ws)  # calls in flight and captured graphs may still use it
            with _on_stream(self.ws.device, stream):
                self.ws = _workspace(max(need.value, 2 * self.ws.numel()), self.ws.device)
            self._streams, self._ran = {_handle(self.ws.device, stream)}, False

    def _buffers(self):
        return (self.ws,)

    def __call__(self, Q, K, V, lens=None, out=None, lse=None, stream=None):
        """Q [B, H, len_q, D], K, V [B, HK, len_k, D] (float32, bfloat16 or
        float16; unit stride along D, K and V strided alike); lens (nullable) [B]
        int32: valid keys of each item, query rows at positions from lens[b] on
        are left as they were.  out: as Q (a fresh one without, 0 in the rows left
        out); lse: float32 [B, H, len_q].  Returns out."""
        import torch
        if K.shape != V.shape or K.stride() != V.stride() or not (Q.dtype == K.dtype == V.dtype):
            raise ValueError("K and V: one shape and layout; Q, K, V: one type")
        if not (Q.device == K.device == V.device == self.ws.device):
            raise ValueError("Q, K, V and the workspace: one device")
        if out is None:
            with _on_stream(Q.device, stream):
                # without lens every row is written
                out = (torch.empty if lens is None else torch.zeros)(Q.shape, dtype=Q.dtype, device=Q.device)
        if out.shape != Q.shape or out.dtype != Q.dtype or out.device != Q.device:
            raise ValueError("out: Q's shape, type and device")
        B, H, Lq, D = Q.shape
        if K.shape[0] != B or K.shape[3] != D:
            raise ValueError("K, V: [B, HK, len_k, D] of Q's batch and D")
        dt = _dtype_of(Q)
        if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, Lq) or not lse.is_contiguous()
                                or lse.device != Q.device):
            raise ValueError("lse: contiguous float32 [B, H, len_q] on Q's device")
        if lens is not None:
            _int32(lens, Q.device, "lens")
            if lens.numel() != B:
                raise ValueError("lens: one entry per item")
        self.reserve(dt, H, K.shape[1], D, Lq, K.shape[2], B, stream)
        qs, ks, os_ = _row_strides(Q, "Q"), _row_strides(K, "K, V"), _row_strides(out, "out")
        _launch(Q.device, stream, "rkv_sink_attention", lib().rkv_sink_attention, Q.data_ptr(), K.data_ptr(), V.data_ptr(),
                dt, Lq, K.shape[2], B, H, K.shape[1], D, ctypes.byref(qs), ctypes.byref(ks), _ptr(lens), self.sinks,
                self.window, out.data_ptr(), ctypes.byref(os_), _ptr(lse), self.ws.data_ptr(), self.ws.numel(), owner=self)
        self._ran |= B > 0 and Lq > 0
        return out

    def status(self, stream=None) -> int:
        """Waits for `stream`; the first error that a call recorded in any
        workspace since the last look, or RKV_OK."""
        import torch
        found = RKV_OK
        with torch.cuda.device(self.ws.device):
            for ws in self._outgrown + [self.ws] * self._ran:
                st = lib().rkv_workspace_status(_ptr(ws), _stream(stream))
                found = found or st
        return found
