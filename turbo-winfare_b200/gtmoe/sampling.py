"""Token sampling through libgtmoe (include/gtmoe_sampling.h), named after the reference's
include/gturbo/sampling.hpp: ``SamplingParams``, ``validate_sampling``, ``splitmix64``,
``seed_for``, ``apply_repetition_penalty`` and ``sample_token``, with the logits in device
memory. Invalid parameters raise ``GtmError`` carrying the reference's message, where the
reference throws GTurboFormatError.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import NamedTuple

from . import ERR_INVALID, GtmError, Sampling, SamplingRow, _stream, check, lib, ptr

MAX_TOP_K = 256
DEGENERATE, NEAR_CUT, NEAR_DRAW = 1, 2, 4   # bits of the device status word


@dataclass
class SamplingParams:
    """include/gturbo/sampling.hpp:21-30 (same defaults: greedy, no truncation, no penalty)."""
    temperature: float = 0.0
    top_p: float = 1.0
    top_k: int = 0
    repetition_penalty: float = 1.0
    has_seed: bool = False
    seed: int = 0

    def is_greedy(self) -> bool:
        return self.temperature <= 0.0 and self.repetition_penalty == 1.0

    def c(self) -> Sampling:
        return Sampling(self.temperature, self.top_p, self.top_k, self.repetition_penalty, int(self.has_seed), 0,
                        self.seed)


def validate_sampling(p: SamplingParams) -> None:
    """sampling.cpp:32-54; raises GtmError(ERR_INVALID) with the reference's message."""
    c = p.c()
    check(lib().gtm_sampling_validate(C.byref(c)))


def splitmix64(x: int) -> int:
    return lib().gtm_sampling_splitmix64(x)


def seed_for(p: SamplingParams, position: int) -> int:
    c = p.c()
    return lib().gtm_sampling_seed_for(C.byref(c), position)


def softcap(logits, cap: float, out=None, stream=None) -> None:
    """cap * tanh(z / cap) on fp32 device logits, in place unless out is given."""
    check(lib().gtm_softcap(logits.numel(), ptr(logits), cap, ptr(logits if out is None else out), _stream(stream)))


class Sampler:
    """Device sampling over a vocabulary of `vocab` ids, with its own workspace."""

    def __init__(self, vocab: int, device: str = "cuda"):
        import torch
        self.vocab = vocab
        n = lib().gtm_sample_workspace_bytes(vocab)
        if n == 0:
            raise GtmError(ERR_INVALID, f"sampling workspace size query failed for vocab {vocab}")
        self.workspace = torch.empty(n + 256, dtype=torch.uint8, device=device)
        self.ws_ptr = C.c_void_p((self.workspace.data_ptr() + 255) // 256 * 256)
        self.ws_bytes = n
        self.token = torch.zeros(2, dtype=torch.int32, device=device)   # [token, status]

    def apply_repetition_penalty(self, logits, history, penalty: float, softcap: float, stream=None) -> None:
        """sampling.cpp:74-90, in place on fp32 device logits; history: int32/uint32 device ids."""
        n = 0 if history is None else history.numel()
        check(lib().gtm_repetition_penalty(ptr(logits), self.vocab, ptr(history) if n else None, n, penalty, softcap,
                                           self.ws_ptr, self.ws_bytes, _stream(stream)))

    def sample_token(self, logits, p: SamplingParams, seed: int, stream=None):
        """sampling.cpp:92-169 on fp32 device logits. Returns the device tensor [token, status]
        (asynchronous); status carries DEGENERATE / NEAR_CUT / NEAR_DRAW bits."""
        c = p.c()
        check(lib().gtm_sample_token(ptr(logits), self.vocab, C.byref(c), seed, ptr(self.token[0:1]),
                                     ptr(self.token[1:2]), self.ws_ptr, self.ws_bytes, _stream(stream)))
        return self.token


# ---- one token for each row of a batch (gtm_sample_rows) ------------------------------------------

@dataclass
class RowParams:
    """A row's settings (GtmSamplingRow): temperature 0 = greedy, top_p 1, min_p 0 and top_k 0 = no cut."""
    temperature: float = 0.0
    top_p: float = 1.0
    min_p: float = 0.0
    top_k: int = 0


def sampling_rows(params):
    """The rows of a call, from RowParams; kept by a caller whose settings do not change."""
    for p in params:
        if not 0 <= p.top_k <= 0x7FFFFFFF:
            raise GtmError(ERR_INVALID, f"top_k {p.top_k} is not in [0, 2^31)")
    return (SamplingRow * max(1, len(params)))(*[SamplingRow(p.temperature, p.top_p, p.min_p, p.top_k) for p in params])


class RowTokens(NamedTuple):
    """Views of the sampler's buffers, overwritten by its next call: int32 tokens (-1: the row has none),
    int32 counts of the ids the cuts kept, fp32 log probabilities."""
    tokens: object
    kept: object
    logprobs: object


class RowSampler:
    """Tokens for up to max_rows rows of logits over a vocabulary of `vocab` ids."""

    def __init__(self, vocab: int, max_rows: int, device: str = "cuda"):
        import torch
        self.vocab, self.max_rows = vocab, max_rows
        self.tokens, self.kept = (torch.zeros(max_rows, dtype=torch.int32, device=device) for _ in range(2))
        self.logprobs = torch.zeros(max_rows, dtype=torch.float32, device=device)
        self._out = tuple(t.data_ptr() for t in (self.tokens, self.kept, self.logprobs))

    def __call__(self, logits, rows, uniforms=None, stream=None) -> RowTokens:
        """logits: fp32 [n, vocab], rows contiguous but possibly strided; rows: sampling_rows(...) or a
        list of RowParams, n of them; uniforms: float64 [n] on the device, None where every row is greedy."""
        import torch
        from .kvcache import _raw_stream
        dev, shape, stride = self.tokens.device, logits.shape, logits.stride()
        if len(shape) != 2 or shape[1] != self.vocab or logits.dtype is not torch.float32 or stride[1] != 1 or logits.device != dev:
            raise GtmError(ERR_INVALID, f"logits must be float32 [n, {self.vocab}] on {dev} with contiguous rows")
        n = shape[0]
        if n > self.max_rows:
            raise GtmError(ERR_INVALID, f"{n} rows for a sampler of {self.max_rows}")
        u = None
        if uniforms is not None:
            if uniforms.dtype is not torch.float64 or uniforms.numel() != n or not uniforms.is_contiguous() or uniforms.device != dev:
                raise GtmError(ERR_INVALID, f"uniforms must be {n} contiguous float64 values on {dev}")
            u = uniforms.data_ptr()
        if isinstance(rows, (list, tuple)):
            if len(rows) != n:
                raise GtmError(ERR_INVALID, f"{len(rows)} settings for {n} rows")
            rows = sampling_rows(rows)
        elif len(rows) < n:
            raise GtmError(ERR_INVALID, f"{len(rows)} settings for {n} rows")
        check(lib().gtm_sample_rows(logits.data_ptr(), n, self.vocab, self.vocab if n <= 1 else stride[0], rows, u, *self._out,
                                    _raw_stream(stream, dev)))
        return RowTokens(self.tokens[:n], self.kept[:n], self.logprobs[:n])
