"""One-byte ring KV caches through libgtmoe (include/gtmoe_attention.h): written by the pass that
norms and rotates a step's queries and keys, read back as fp32, and attended by a step's rows with
one shared prefix. Host arrays (positions, sequence indices) are sequences of ints or contiguous
numpy uint32 arrays; the latter are passed without a copy.
"""
from __future__ import annotations

import ctypes as C

from . import ERR_INVALID, ERR_UNSUPPORTED, GtmError, KvCacheDesc, _stream, check, lib, ptr

INT8, E4M3 = 0, 1
FORMATS = {"int8": INT8, "e4m3": E4M3}


def _u32(vals, n: int | None = None):
    """(pointer, owner) of a host array of uint32; n: the length it must have."""
    import numpy as np
    if not (isinstance(vals, np.ndarray) and vals.dtype == np.uint32 and vals.flags.c_contiguous):
        vals = np.asarray(vals)
        if vals.size and (vals.dtype.kind not in "iu" or vals.min() < 0 or vals.max() > 0xFFFFFFFF):
            raise GtmError(ERR_INVALID, "positions and sequence indices are integers in [0, 2^32)")
        vals = np.ascontiguousarray(vals, dtype=np.uint32)
    if n is not None and vals.size != n:
        raise GtmError(ERR_INVALID, f"{vals.size} positions or sequence indices for {n} rows")
    return C.c_void_p(vals.ctypes.data), vals


def _f32(t, name: str, device, shape=None) -> None:
    """The checks a raw pointer cannot make."""
    import torch
    if t.dtype != torch.float32 or t.device != device:
        raise GtmError(ERR_INVALID, f"{name} must be float32 on {device}, not {t.dtype} on {t.device}")
    if shape is not None and (tuple(t.shape) != tuple(shape) or not t.is_contiguous()):
        raise GtmError(ERR_INVALID, f"{name} must be contiguous {tuple(shape)}, not {tuple(t.shape)}")


def _row_stride(t, name: str, device, n: int, width: int) -> int:
    _f32(t, name, device)
    if t.dim() != 2 or t.shape[0] != n or t.shape[1] != width or t.stride(1) != 1:
        raise GtmError(ERR_INVALID, f"{name} must be [{n}, {width}] with contiguous rows, not {tuple(t.shape)}")
    return width if n <= 1 else t.stride(0)


def _bf16(t, name: str, device, n: int) -> None:
    if t is not None and (t.element_size() != 2 or t.numel() != n or not t.is_contiguous() or t.device != device):
        raise GtmError(ERR_INVALID, f"{name} must be {n} contiguous bf16 values on {device}")


class KvCache:
    """num_seqs ring caches of `capacity` positions: codes [num_seqs, capacity, kv_heads, head_dim]
    (torch.int8 or torch.float8_e4m3fn) and scales [num_seqs, kv_heads, capacity] (fp32) for keys
    and values; a value is code * scale."""

    def __init__(self, num_seqs: int, capacity: int, kv_heads: int, head_dim: int, fmt: str = "int8", device: str = "cuda"):
        import torch
        if fmt not in FORMATS:
            raise GtmError(ERR_UNSUPPORTED, f"cache format {fmt!r} (one of {sorted(FORMATS)})")
        dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
        shape = (num_seqs, capacity, kv_heads, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(dt) for _ in range(2))
        ks, vs = (torch.zeros(num_seqs, kv_heads, capacity, dtype=torch.float32, device=device) for _ in range(2))
        self._over(k, v, ks, vs)

    @classmethod
    def over(cls, k, v, k_scale, v_scale) -> "KvCache":
        """A cache over the caller's tensors, which it keeps alive."""
        c = cls.__new__(cls)
        c._over(k, v, k_scale, v_scale)
        return c

    def _over(self, k, v, k_scale, v_scale) -> None:
        import torch
        if k.dtype not in (torch.int8, torch.float8_e4m3fn) or v.dtype != k.dtype or k.dim() != 4 or v.shape != k.shape:
            raise GtmError(ERR_INVALID, "codes must be two int8 or float8_e4m3fn tensors [num_seqs, capacity, kv_heads, head_dim]")
        num_seqs, capacity, kv_heads, head_dim = k.shape
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _f32(t, name, k.device, (num_seqs, kv_heads, capacity))
        if not (k.is_contiguous() and v.is_contiguous()) or v.device != k.device:
            raise GtmError(ERR_INVALID, "codes must be contiguous and on one device")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, k.device
        self.num_seqs, self.capacity, self.kv_heads, self.head_dim = num_seqs, capacity, kv_heads, head_dim
        self.fmt = "int8" if k.dtype == torch.int8 else "e4m3"
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), FORMATS[self.fmt], num_seqs,
                                capacity, kv_heads, head_dim, 0)

    def write(self, q, k, v, q_out, positions, seqs, *, q_w=None, k_w=None, eps: float = 1e-6, rotated_pairs: int = 0,
              theta: float = 10000.0, stream=None) -> None:
        """gtm_qkv_cache_rows: q [n, q_heads * head_dim], k and v [n, kv_heads * head_dim] (rows may be
        strided, v may be k); q_out contiguous like q, or q itself; q_w, k_w bf16 [head_dim] or None."""
        n, width = q.shape[0], self.kv_heads * self.head_dim
        if q.dim() != 2 or q.shape[1] % self.head_dim:
            raise GtmError(ERR_INVALID, f"q must be [n, q_heads * {self.head_dim}], not {tuple(q.shape)}")
        qs = _row_stride(q, "q", self.device, n, q.shape[1])
        ks, vs = (_row_stride(t, name, self.device, n, width) for name, t in (("k", k), ("v", v)))
        _f32(q_out, "q_out", self.device, (n, q.shape[1]))
        _bf16(q_w, "q_w", self.device, self.head_dim)
        _bf16(k_w, "k_w", self.device, self.head_dim)
        pos, _p = _u32(positions, n)
        sq, _s = _u32(seqs, n)
        check(lib().gtm_qkv_cache_rows(C.byref(self.desc), q.shape[1] // self.head_dim, n, ptr(q), ptr(k), ptr(v), qs, ks, vs,
                                       ptr(q_w), ptr(k_w), eps, rotated_pairs, theta, pos, sq, ptr(q_out), _stream(stream)))

    def read(self, seq: int, first: int, count: int, k_out=None, v_out=None, stream=None):
        """gtm_kv_read: positions [first, first + count) of `seq` as fp32 [count, kv_heads * head_dim];
        (k_out, v_out), allocated where both are None."""
        import torch
        shape = (count, self.kv_heads * self.head_dim)
        if k_out is None and v_out is None:
            k_out, v_out = (torch.empty(shape, dtype=torch.float32, device=self.device) for _ in range(2))
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is not None:
                _f32(t, name, self.device, shape)
        check(lib().gtm_kv_read(C.byref(self.desc), seq, first, count, ptr(k_out), ptr(v_out), _stream(stream)))
        return k_out, v_out


class KvAttention:
    """Attention of up to max_rows rows over KvCache caches (gtm_attention_kv_rows), with its workspace;
    one object serves one stream at a time."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, max_rows: int, device: str = "cuda"):
        import torch
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        n = lib().gtm_attention_kv_workspace_bytes(q_heads, kv_heads, head_dim, max_rows)
        if n == 0:
            raise GtmError(ERR_UNSUPPORTED, f"attention of {q_heads} / {kv_heads} heads of {head_dim}, {max_rows} rows")
        self.workspace = torch.empty(n, dtype=torch.uint8, device=device)
        self.ws_ptr, self.ws_bytes = C.c_void_p(self.workspace.data_ptr()), n

    def __call__(self, q, cache: KvCache, seqs, positions, ctx, *, window: int = 0, prefix: KvCache | None = None,
                 prefix_seq: int = 0, prefix_len: int = 0, stream=None) -> None:
        n, width = q.shape[0], self.q_heads * self.head_dim
        _f32(q, "q", cache.device, (n, width))
        _f32(ctx, "ctx", cache.device, (n, width))
        if (cache.kv_heads, cache.head_dim) != (self.kv_heads, self.head_dim) or self.workspace.device != cache.device:
            raise GtmError(ERR_INVALID, "the cache's heads or device are not the attention's")
        if prefix is not None and prefix.device != cache.device:
            raise GtmError(ERR_INVALID, "cache and prefix must be on one device")
        pos, _p = _u32(positions, n)
        sq, _s = _u32(seqs, n)
        check(lib().gtm_attention_kv_rows(C.byref(cache.desc), C.byref(prefix.desc) if prefix is not None else None, prefix_seq,
                                          prefix_len, self.q_heads, n, window, ptr(q), sq, pos, ptr(ctx), self.ws_ptr,
                                          self.ws_bytes, _stream(stream)))
