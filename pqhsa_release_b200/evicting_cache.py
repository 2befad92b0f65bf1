"""Decode attention over a cache that stays within a budget by dropping the keys that have gathered the least attention
weight: the other way, next to the IVF-PQ index, of bounding what a long context costs per step.  Exact attention over
the keys that are left, no approximation of the others.

Same call forms as :class:`~pqhsa_release_b200.decode_adapter.IVFPQDecodeAttentionAdapter`:

    keys / values : [batch, kv_heads, seq, 128]         queries : [batch, query_heads, 128]

``ValueError`` for shapes, ``RuntimeError`` for use before ``build_cache``.  The reference has no counterpart.
"""

from __future__ import annotations

import torch

from . import _lib
from .decode_adapter import DecodeAttentionOutput, _squeeze_decode_token
from .paged_attention import MAX_QUERY_LEN, MAX_ROWS, PagedAttention


def _rows(x: torch.Tensor) -> torch.Tensor:
    """Rows that the kernels can read: as they are where they lie in one piece on 16-byte boundaries, else a copy."""
    fit = 16 // x.element_size()
    if x.stride(-1) == 1 and not (x.data_ptr() & 15 or any(s % fit for s in x.stride()[:-1])):
        return x
    return x.clone(memory_format=torch.contiguous_format)


class EvictingCacheAdapter:
    """Up to ``budget + interval`` keys per (request, KV head); once that many are there, an eviction keeps ``budget``:
    the first ``sink_tokens`` and last ``recent`` positions and those of the largest accumulated weight.  ``softcap``,
    ``alibi_slopes`` and ``window`` as for :class:`PagedAttention`.

    Which step evicts is counted on the host, so ``build_cache`` and ``append`` refuse to be captured into a CUDA graph
    (``RuntimeError``); ``forward`` can be, and so can a loop of :class:`PagedAttention`'s own calls."""

    def __init__(self, *, num_query_heads: int, num_kv_heads: int, budget: int, interval: int = 256, sink_tokens: int = 4,
                 recent: int = 128, scale: float | None = None, softcap: float = 0.0,
                 alibi_slopes: torch.Tensor | None = None, window: int = 0) -> None:
        if num_kv_heads < 1 or num_query_heads < 1 or num_query_heads % num_kv_heads != 0:
            raise ValueError("GQA requires num_query_heads % num_kv_heads == 0")
        if budget < 1 or interval < 1 or sink_tokens < 0 or recent < 0 or sink_tokens + recent > budget:
            raise ValueError("need budget >= 1, interval >= 1 and sink_tokens + recent <= budget")
        self.num_query_heads, self.num_kv_heads = int(num_query_heads), int(num_kv_heads)
        self.budget, self.interval, self.recent = int(budget), int(interval), int(recent)
        self._kw = dict(scale=scale, softcap=softcap, alibi_slopes=alibi_slopes, window=window, sink_tokens=int(sink_tokens))
        self.attention: PagedAttention | None = None
        self.length = 0      # keys held per (request, KV head)
        self.position = 0    # tokens seen
        self.evictions = 0

    # ---- cache -------------------------------------------------------------------------------------------
    @staticmethod
    def _not_captured(call: str) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{call} counts on the host when to evict and cannot be captured into a CUDA graph")

    def _layer(self, keys: torch.Tensor, values: torch.Tensor, tokens: int = 1) -> PagedAttention:
        """A layer over these contiguous buffers; positions and weights are [batch, kv_heads, capacity] as they."""
        B, H, cap, _ = keys.shape
        layer = PagedAttention(num_query_heads=self.num_query_heads, num_kv_heads=H, max_requests=B, token_capacity=cap,
                               dtype=keys.dtype, device=keys.device, max_query_len=tokens, **self._kw)
        layer.bind_kv_contiguous(keys, values)
        return layer

    def build_cache(self, keys: torch.Tensor, values: torch.Tensor, queries: torch.Tensor | None = None) -> "EvictingCacheAdapter":
        """The prompt's keys and values (copied).  ``queries`` ``[batch, query_heads, W, 128]``: those of its last W
        tokens, whose attention weights choose what a prompt longer than the budget keeps; without them only the last
        and the first positions are told apart from the rest, of which the lowest stay."""
        if keys.ndim != 4 or values.ndim != 4 or keys.shape != values.shape or keys.shape[1] != self.num_kv_heads or keys.shape[3] != _lib.HEAD_DIM:
            raise ValueError(f"keys and values must be [batch, {self.num_kv_heads}, seq, 128]")
        B, H, S, D = keys.shape
        if S < 1:
            raise ValueError("the prompt is empty")
        if queries is not None and (queries.ndim != 4 or queries.shape[:2] != (B, self.num_query_heads) or queries.shape[3] != D
                                    or not 1 <= queries.shape[2] <= S or queries.dtype != keys.dtype):
            raise ValueError(f"queries must be [{B}, {self.num_query_heads}, 1..{S}, 128] in the keys' dtype")
        if keys.is_cuda:
            self._not_captured("build_cache")
        dev, room = keys.device, self.budget + self.interval

        def buffers(cap):
            k, v = (torch.zeros(B, H, cap, D, dtype=keys.dtype, device=dev) for _ in range(2))
            return k, v, torch.zeros(B, H, cap, dtype=torch.int32, device=dev), torch.zeros(B, H, cap, device=dev)

        # the adapter takes all of it over at the end: a prompt that is refused leaves the cache there was
        k, v, positions, weights = buffers(max(S, room))
        k[:, :, :S], v[:, :, :S] = keys, values
        positions[:] = torch.arange(k.shape[2], dtype=torch.int32, device=dev)
        layer = self._layer(k, v)
        lens = torch.full((B,), S, dtype=torch.int32, device=dev)
        query_pos = torch.full((B,), S - 1, dtype=torch.int32, device=dev)
        length, evictions = S, 0
        if queries is not None:
            # A few tokens at a time, each seeing what lies before it; a layer of their own, whose scores (8 tokens'
            # against the one of a decode step) go with it.
            queries = _rows(queries)
            W, step = queries.shape[2], min(MAX_QUERY_LEN, MAX_ROWS // (self.num_query_heads // H))
            vote = self._layer(k, v, step)
            for lo in range(0, W, step):
                hi = min(lo + step, W)
                at = torch.full_like(query_pos, S - W + hi - 1)
                vote.forward(queries[:, :, lo:hi].transpose(1, 2), lens, key_pos=positions, query_pos=at, mass=weights)
            del vote
        if S >= room:
            layer.evict(lens, mass=weights, key_pos=positions, query_pos=query_pos, budget=self.budget, recent=self.recent)
            length, evictions = self.budget, 1
            if S > room:  # the long buffers are not needed any more
                small = buffers(room)
                for big, to in zip((k, v, positions, weights), small):
                    to[:, :, :length] = big[:, :, :length]
                k, v, positions, weights = small
                layer = self._layer(k, v)
        self.attention, self.keys, self.values, self.positions, self.weights = layer, k, v, positions, weights
        self.lens, self.query_pos = lens, query_pos
        self.length, self.position, self.evictions = length, S, evictions
        return self

    def _evict(self) -> None:
        self.attention.evict(self.lens, mass=self.weights, key_pos=self.positions, query_pos=self.query_pos, budget=self.budget,
                             recent=self.recent)
        self.length = min(self.length, self.budget)
        self.evictions += 1

    def _ready(self) -> PagedAttention:
        if self.attention is None:
            raise RuntimeError("build_cache must be called before the cache is used")
        return self.attention

    # ---- decode -------------------------------------------------------------------------------------------
    def append(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """One token per request, ``[batch, kv_heads, 128]`` (or with a token dimension of one)."""
        att = self._ready()
        keys, values = _squeeze_decode_token(keys, "keys"), _squeeze_decode_token(values, "values")
        if keys.shape != (self.keys.shape[0], self.num_kv_heads, _lib.HEAD_DIM) or values.shape != keys.shape:
            raise ValueError(f"keys and values must be [{self.keys.shape[0]}, {self.num_kv_heads}, 128]")
        for x in (keys, values):  # before anything is counted or moved
            if x.dtype != self.keys.dtype or x.device != self.keys.device:
                raise ValueError(f"keys and values must be {self.keys.dtype} tensors on {self.keys.device}, got {x.dtype} on {x.device}")
        self._not_captured("append")
        keys, values = _rows(keys.contiguous()), _rows(values.contiguous())
        if self.length >= self.budget + self.interval:
            self._evict()
        self.query_pos.add_(1)
        att.append(keys, values, self.lens, key_pos=self.positions, query_pos=self.query_pos, mass=self.weights)
        self.length += 1
        self.position += 1

    def _queries(self, queries: torch.Tensor) -> torch.Tensor:
        """Checked, and as rows that the attention can read."""
        if queries.ndim != 3 or queries.shape != (self.keys.shape[0], self.num_query_heads, _lib.HEAD_DIM):
            raise ValueError(f"queries must be [{self.keys.shape[0]}, {self.num_query_heads}, 128]")
        if queries.dtype != self.keys.dtype or queries.device != self.keys.device:
            raise ValueError(f"queries must be a {self.keys.dtype} tensor on {self.keys.device}, got {queries.dtype} on {queries.device}")
        return _rows(queries)

    def forward(self, queries: torch.Tensor) -> DecodeAttentionOutput:
        """The last token's attention; its weights are accumulated."""
        att = self._ready()
        return DecodeAttentionOutput(context=att.forward(self._queries(queries), self.lens, key_pos=self.positions,
                                                         query_pos=self.query_pos, mass=self.weights))

    def decode_step(self, queries: torch.Tensor, keys: torch.Tensor | None = None, values: torch.Tensor | None = None, *,
                    append_kv: bool = True) -> DecodeAttentionOutput:
        if append_kv:
            if keys is None or values is None:
                raise ValueError("keys and values are required when append_kv=True")
            self._ready()
            queries = self._queries(queries)  # a refused step appends nothing
            self.append(keys, values)
        return self.forward(queries)
