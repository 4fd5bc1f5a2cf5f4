"""One-byte ring KV caches through libgtmoe (include/gtmoe_attention.h): written by the pass that
norms and rotates a step's queries and keys, read back as fp32, and attended by a step's rows with
one shared prefix. Host arrays (positions, sequence indices) are sequences of ints or contiguous
numpy uint32 arrays; the latter are passed without a copy.
"""
from __future__ import annotations

import ctypes as C

from . import ERR_INVALID, ERR_UNSUPPORTED, GtmError, KvCacheDesc, check, lib

INT8, E4M3 = 0, 1
FORMATS = {"int8": INT8, "e4m3": E4M3}


def _u32(vals, n: int | None = None):
    """(address, owner) of a host array of uint32; n: the length it must have."""
    import numpy as np
    if not (type(vals) is np.ndarray and vals.dtype == np.uint32 and vals.flags.c_contiguous):
        vals = np.asarray(vals)
        if vals.size and (vals.dtype.kind not in "iu" or vals.min() < 0 or vals.max() > 0xFFFFFFFF):
            raise GtmError(ERR_INVALID, "positions and sequence indices are integers in [0, 2^32)")
        vals = np.ascontiguousarray(vals, dtype=np.uint32)
    if n is not None and vals.size != n:
        raise GtmError(ERR_INVALID, f"{vals.size} positions or sequence indices for {n} rows")
    # the address by the shortest way (a few tenths of a microsecond), which takes writable arrays with elements only
    return C.addressof(C.c_char.from_buffer(vals)) if vals.size and vals.flags.writeable else vals.ctypes.data, vals


def _raw_stream(stream, device):
    """The stream to launch on, as an integer: the caller's, or torch's current one, on the tensors' device,
    which has to be the current device. (Without a GPU the library refuses the call itself.)"""
    import torch
    if device.type != "cuda":
        if torch.cuda.is_available():
            raise GtmError(ERR_INVALID, f"the tensors are on {device}, not on a GPU")
        return None
    if torch.cuda.current_device() != device.index:
        raise GtmError(ERR_INVALID, f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device.index)   # current_stream() makes an object: 3 us more a call
    if stream.device_index != device.index:
        raise GtmError(ERR_INVALID, f"the tensors are on {device}, the stream on cuda:{stream.device_index}")
    return stream.cuda_stream


def _uint(**vals) -> None:
    """Refuses what would not survive the way into a uint32."""
    for name, x in vals.items():
        if not 0 <= x <= 0xFFFFFFFF:
            raise GtmError(ERR_INVALID, f"{name} {x} is not in [0, 2^32)")


def _f32(t, name: str, device, shape=None) -> int:
    """The checks a raw pointer cannot make, and the pointer."""
    import torch
    if t.dtype is not torch.float32 or t.device != device:
        raise GtmError(ERR_INVALID, f"{name} must be float32 on {device}, not {t.dtype} on {t.device}")
    if shape is not None and (t.shape != shape or not t.is_contiguous()):
        raise GtmError(ERR_INVALID, f"{name} must be contiguous {tuple(shape)}, not {tuple(t.shape)}")
    return t.data_ptr()


def _rows(t, name: str, device, n: int, width: int):
    """(pointer, row stride) of n rows of `width` floats."""
    p = _f32(t, name, device)
    if t.shape != (n, width):
        raise GtmError(ERR_INVALID, f"{name} must be [{n}, {width}], not {tuple(t.shape)}")
    stride = t.stride()
    if stride[1] != 1:
        raise GtmError(ERR_INVALID, f"{name} must have contiguous rows")
    return p, width if n <= 1 else stride[0]


def _bf16(t, name: str, device, n: int):
    """A bfloat16 tensor, or one of its bits as int16 or uint16 (an fp16 one would be read as what it is not)."""
    import torch
    if t is None:
        return None
    if t.dtype not in (torch.bfloat16, torch.int16, torch.uint16) or t.numel() != n or not t.is_contiguous() or t.device != device:
        raise GtmError(ERR_INVALID, f"{name} must be {n} contiguous bf16 values on {device}")
    return t.data_ptr()


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
        self._ref = C.byref(self.desc)

    def write(self, q, k, v, q_out, positions, seqs, *, q_w=None, k_w=None, eps: float = 1e-6, rotated_pairs: int = 0,
              theta: float = 10000.0, stream=None) -> None:
        """gtm_qkv_cache_rows: q [n, q_heads * head_dim], k and v [n, kv_heads * head_dim] (rows may be
        strided, v may be k); q_out contiguous like q, or q itself; q_w, k_w bf16 [head_dim] or None."""
        if q.dim() != 2 or q.shape[1] % self.head_dim:
            raise GtmError(ERR_INVALID, f"q must be [n, q_heads * {self.head_dim}], not {tuple(q.shape)}")
        shape, dev, width = q.shape, self.device, self.kv_heads * self.head_dim
        n = shape[0]
        _uint(rotated_pairs=rotated_pairs)
        qp, qs = _rows(q, "q", dev, n, shape[1])
        kp, ks = _rows(k, "k", dev, n, width)
        vp, vs = _rows(v, "v", dev, n, width)
        out = _f32(q_out, "q_out", dev, shape)
        qw, kw = _bf16(q_w, "q_w", dev, self.head_dim), _bf16(k_w, "k_w", dev, self.head_dim)
        pos, _p = _u32(positions, n)
        sq, _s = _u32(seqs, n)
        check(lib().gtm_qkv_cache_rows(self._ref, shape[1] // self.head_dim, n, qp, kp, vp, qs, ks, vs, qw, kw, eps,
                                       rotated_pairs, theta, pos, sq, out, _raw_stream(stream, dev)))

    def read(self, seq: int, first: int, count: int, k_out=None, v_out=None, stream=None):
        """gtm_kv_read: positions [first, first + count) of `seq` as fp32 [count, kv_heads * head_dim];
        (k_out, v_out), allocated where both are None, as memory of the stream that writes them."""
        _uint(seq=seq, first=first, count=count)
        shape = (count, self.kv_heads * self.head_dim)
        if k_out is None and v_out is None:
            import contextlib

            import torch
            # memory that the current stream has given up may still be read by what is queued there
            with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
                k_out, v_out = (torch.empty(shape, dtype=torch.float32, device=self.device) for _ in range(2))
        kp = None if k_out is None else _f32(k_out, "k_out", self.device, shape)
        vp = None if v_out is None else _f32(v_out, "v_out", self.device, shape)
        check(lib().gtm_kv_read(self._ref, seq, first, count, kp, vp, _raw_stream(stream, self.device)))
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
        self.workspace[:4].zero_()   # the error word
        self.ws_ptr, self.ws_bytes, self.device = self.workspace.data_ptr(), n, self.workspace.device

    def __call__(self, q, cache: KvCache, seqs, positions, ctx, *, window: int = 0, prefix: KvCache | None = None,
                 prefix_seq: int = 0, prefix_len: int = 0, stream=None) -> None:
        dev, shape = cache.device, (q.shape[0], self.q_heads * self.head_dim)
        n = shape[0]
        _uint(window=window, prefix_seq=prefix_seq, prefix_len=prefix_len)
        qp, out = _f32(q, "q", dev, shape), _f32(ctx, "ctx", dev, shape)
        if cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim or self.device != dev:
            raise GtmError(ERR_INVALID, "the cache's heads or device are not the attention's")
        if prefix is not None and prefix.device != dev:
            raise GtmError(ERR_INVALID, "cache and prefix must be on one device")
        pos, _p = _u32(positions, n)
        sq, _s = _u32(seqs, n)
        check(lib().gtm_attention_kv_rows(cache._ref, None if prefix is None else prefix._ref, prefix_seq, prefix_len, self.q_heads, n,
                                          window, qp, sq, pos, out, self.ws_ptr, self.ws_bytes, _raw_stream(stream, dev)))

    def check(self, stream=None) -> None:
        """gtm_attention_kv_check: raises GtmError (ERR_TIMEOUT) where a wait of an earlier call ran out."""
        check(lib().gtm_attention_kv_check(self.ws_ptr, _raw_stream(stream, self.device)))
