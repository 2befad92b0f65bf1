"""Dense attention of a step's tokens over a paged KV cache, the append of their rows, and eviction from the cache by
accumulated attention weight: thin wrappers over ``pqhsa_paged_*`` (include/pqhsa.h has the formulas).

The exact counterpart of :class:`~pqhsa_release_b200.device_index.DeviceIndexPool`'s decode step, for requests without
an index.  The reference leaves it to the serving engine
(benchmarks/vllm_backend/pq_hsa_decode_runtime.py:790-822).  Lengths, positions and block tables are read on the
device: nothing here synchronises, and a captured call follows the lengths of its replays.
"""

from __future__ import annotations

import ctypes as C
import threading
import weakref
from math import isfinite, sqrt

import torch

from . import _lib
from .device_index import _DTYPE_CODE

MAX_QUERY_LEN, MAX_GROUP, MAX_ROWS = 8, 16, 64
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_is_capturing = torch._C._cuda_isCurrentStreamCapturing


class _Scratch:
    """Scratch memory of one stream of execution.  Whoever uses it holds ``lock`` from ``take`` until the call's launches
    are made: those of another thread may not come between them."""

    __slots__ = ("now", "kept", "lock", "__weakref__")

    def __init__(self):
        self.now, self.kept, self.lock = None, [], threading.Lock()

    def take(self, nbytes: int, device: torch.device, counters: bool, capturing: bool) -> int:
        t = self.now
        if t is None or t.numel() < nbytes:
            if capturing and t is not None:
                self.kept.append(t)  # launches recorded before still use it
            t = self.now = torch.empty(nbytes, dtype=torch.uint8, device=device)
            if counters:
                t[:4096].zero_()
        return t.data_ptr()


# (kind, device, stream, capture) -> _Scratch, as long as a layer holds it: the calls made on one stream, or recorded into
# one capture, run in order, whichever layer makes them.
_SCRATCH: weakref.WeakValueDictionary = weakref.WeakValueDictionary()


class PagedAttention:
    """The settings of one attention layer, a bound cache, and the workspaces its calls need.

    ``softcap``: scores become ``softcap * tanh(score / softcap)``.  ``alibi_slopes`` ``[num_query_heads]``: minus slope
    times distance (copied).  ``window`` / ``sink_tokens``: a token sees the last ``window`` positions (itself included) and the
    first ``sink_tokens`` of its document; 0 = everything.  ``token_capacity``: most slots of a request, the last
    dimension of ``mass`` and ``key_pos``.

    Calls on one stream run in order and share a workspace, those of a model's other layers among them; every other
    stream, and every CUDA-graph capture, gets its own (kept as long as a layer that used it), so two streams or two
    graphs may run at once.  A graph replayed twice at the same time shares its own.  One object is used by one host
    thread at a time."""

    def __init__(self, *, num_query_heads: int, num_kv_heads: int, max_requests: int, token_capacity: int, dtype: torch.dtype,
                 device: torch.device | str, max_query_len: int = 1, scale: float | None = None, softcap: float = 0.0,
                 alibi_slopes: torch.Tensor | None = None, window: int = 0, sink_tokens: int = 0):
        if dtype not in _DTYPE_CODE:
            raise ValueError(f"unsupported dtype {dtype}: need float32, bfloat16 or float16")
        if num_kv_heads < 1 or num_query_heads < 1 or num_query_heads % num_kv_heads:
            raise ValueError("GQA requires num_query_heads % num_kv_heads == 0")
        self.Hq, self.H = int(num_query_heads), int(num_kv_heads)
        self.G = self.Hq // self.H
        if self.G > MAX_GROUP:
            raise ValueError(f"at most {MAX_GROUP} query heads per KV head, got {self.G}")
        if not 1 <= max_query_len <= MAX_QUERY_LEN or self.G * max_query_len > MAX_ROWS:
            raise ValueError(f"max_query_len must be in 1..{MAX_QUERY_LEN} with group * max_query_len <= {MAX_ROWS}")
        if max_requests < 1 or token_capacity < 1:
            raise ValueError("max_requests and token_capacity must be positive")
        scale = 1.0 / sqrt(_lib.HEAD_DIM) if scale is None else float(scale)
        kept = [C.c_float(x).value for x in (scale, softcap)]  # as the kernels get them
        if not all(map(isfinite, kept)) or softcap < 0 or (kept[1] == 0.0) != (softcap == 0.0):
            raise ValueError("scale must be finite and softcap finite and non-negative, in 32 bits too")
        if window < 0 or sink_tokens < 0:
            raise ValueError("window and sink_tokens must be non-negative")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("PagedAttention needs a CUDA device: there is no CPU path")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._index = self.device.index
        self.dtype = dtype
        self.max_requests, self.token_capacity, self.max_query_len = int(max_requests), int(token_capacity), int(max_query_len)
        self.alibi_slopes = None
        if alibi_slopes is not None:
            if tuple(alibi_slopes.shape) != (self.Hq,):
                raise ValueError(f"alibi_slopes must have one entry per query head, got {tuple(alibi_slopes.shape)}")
            self.alibi_slopes = self._slopes(alibi_slopes.detach())
        # one argument block per operator (each keeps the sizes of its last call), the cache's part the same in all
        self.p, self._append_p, self._evict_p = _lib.PagedParams(), _lib.PagedParams(), _lib.PagedParams()
        for p in (self.p, self._append_p, self._evict_p):
            p.abi_version, p.dtype, p.head_dim = _lib.ABI_VERSION, _DTYPE_CODE[dtype], _lib.HEAD_DIM
            p.requests, p.kv_heads, p.group, p.query_len = self.max_requests, self.H, self.G, self.max_query_len
            p.slot_capacity = self.token_capacity
            p.scale, p.softcap, p.window, p.sink_tokens = scale, float(softcap), int(window), int(sink_tokens)
        self.p.alibi_slopes = self.alibi_slopes.data_ptr() if self.alibi_slopes is not None else None
        self._ref, self._append_ref, self._evict_ref = C.byref(self.p), C.byref(self._append_p), C.byref(self._evict_p)
        self._sizes: dict = {}  # (requests, tokens) of a call -> workspace bytes without and with weights
        if 0 in self._workspace_bytes(self.max_requests, self.max_query_len):
            raise ValueError(_lib.lib.pqhsa_last_error_string().decode("utf-8", "replace"))
        self._ws: dict = {}  # the shared scratch memory this layer has used
        self._kv_keepalive = None
        self._rows = 0  # requests the bound cache addresses
        self._forward_shape = self._append_shape = None  # shapes the blocks are set for (contiguous rows), or None

    # ---- cache ----------------------------------------------------------------------------------------
    def bind_kv_paged(self, kv_cache: torch.Tensor, block_table: torch.Tensor) -> None:
        """vLLM FLASH_ATTN pages, either layout (benchmarks/vllm_backend/paged_kv_fa.py:44-58): 5-D
        ``[2, blocks, block_size, Hkv, 128]`` or 4-D ``[blocks, Hkv, block_size, 256]``, and the block table, int32
        ``[requests, max_blocks]``.  Both are read when a call runs: their contents may change between calls."""
        self._check(kv_cache, "kv_cache", self.dtype)
        self._check(block_table, "block_table", torch.int32)
        if block_table.dim() != 2 or not block_table.is_contiguous() or block_table.numel() == 0:
            raise ValueError("block_table must be a contiguous int32 [requests, max_blocks] tensor")
        D = _lib.HEAD_DIM
        if kv_cache.dim() == 5:
            if kv_cache.shape[0] != 2 or kv_cache.shape[4] != D or kv_cache.shape[3] != self.H or kv_cache.stride(4) != 1:
                raise ValueError(f"5-D KV pages must be [2, blocks, block_size, {self.H}, 128] with contiguous rows")
            base, off, nb, bs = kv_cache.data_ptr(), kv_cache.stride(0) * kv_cache.element_size(), kv_cache.shape[1], kv_cache.shape[2]
            strides = kv_cache.stride(1), kv_cache.stride(3), kv_cache.stride(2)
        elif kv_cache.dim() == 4:
            if kv_cache.shape[3] != 2 * D or kv_cache.shape[1] != self.H or kv_cache.stride(3) != 1:
                raise ValueError(f"4-D KV pages must be [blocks, {self.H}, block_size, 2*128] with contiguous rows")
            base, off, nb, bs = kv_cache.data_ptr(), D * kv_cache.element_size(), kv_cache.shape[0], kv_cache.shape[2]
            strides = kv_cache.stride(0), kv_cache.stride(1), kv_cache.stride(2)
        else:
            raise ValueError(f"unsupported FLASH_ATTN kv_cache shape {tuple(kv_cache.shape)}")
        self._bind(base, base + off, nb, bs, strides, block_table.data_ptr(), block_table.shape[1])
        self._rows = block_table.shape[0]
        self._kv_keepalive = (kv_cache, block_table)

    def bind_kv_contiguous(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """keys / values: ``[B, Hkv, capacity, 128]`` (any strides that keep rows contiguous), request r in row r."""
        self._check(keys, "keys", self.dtype)
        self._check(values, "values", self.dtype)
        if keys.dim() != 4 or keys.shape[1] != self.H or keys.shape[3] != _lib.HEAD_DIM:
            raise ValueError(f"keys and values must be [B, {self.H}, capacity, 128]")
        if keys.shape != values.shape or keys.stride() != values.stride() or keys.stride(-1) != 1:
            raise ValueError("keys and values must have the same shape and strides with contiguous rows")
        self._bind(keys.data_ptr(), values.data_ptr(), keys.shape[0], keys.shape[2],
                   (keys.stride(0), keys.stride(1), keys.stride(2)), None, 0)
        self._rows = keys.shape[0]
        self._kv_keepalive = (keys, values)

    def _bind(self, k: int, v: int, blocks: int, block_size: int, strides, table, max_blocks: int) -> None:
        if blocks < 1 or block_size < 1:
            raise ValueError("the KV cache is empty")
        a = 4 if self.dtype == torch.float32 else 8
        if (k | v) & 15 or any(s % a for s in strides):
            raise ValueError("KV rows must be 16-byte aligned")
        for p in (self.p, self._append_p, self._evict_p):
            p.k_base, p.v_base, p.num_blocks, p.block_size = k, v, blocks, block_size
            p.stride_block, p.stride_head, p.stride_row = strides
            p.block_table, p.max_blocks = table, max_blocks
        self._forward_shape = self._append_shape = None

    def _slopes(self, given: torch.Tensor) -> torch.Tensor:
        """A copy that every stream may read.  During a capture a copy would only be there once the graph has run: then the
        tensor itself."""
        slopes = given.to(device=self.device, dtype=torch.float32).contiguous()
        with torch.cuda.device(self._index):
            if not _is_capturing():
                slopes = slopes.clone()
                torch.cuda.current_stream().synchronize()
            elif slopes.data_ptr() != given.data_ptr():
                raise RuntimeError(f"a layer made during a CUDA-graph capture needs its alibi_slopes as a contiguous float32 tensor on {self.device}")
        return slopes

    # ---- checks and scratch ------------------------------------------------------------------------------
    def _check(self, t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
        if t.dtype != dtype or t.device != self.device:
            raise ValueError(f"{name} must be a {dtype} tensor on {self.device}, got {t.dtype} on {t.device}")

    def _per_request(self, t: torch.Tensor, name: str, B: int) -> int:
        if t.dtype is not torch.int32 or t.get_device() != self._index or t.shape != (B,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of {B} entries on {self.device}")
        return t.data_ptr()

    def _per_slot(self, t: torch.Tensor, name: str, dtype: torch.dtype, B: int) -> int:
        shape = t.shape
        if (t.dtype is not dtype or t.get_device() != self._index or len(shape) != 3 or shape[0] < B
                or shape[1:] != (self.H, self.token_capacity) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dtype} [>= {B}, {self.H}, {self.token_capacity}] tensor on {self.device}")
        return t.data_ptr()

    def _tokens(self, shape, name: str, heads: int) -> tuple[int, int]:
        """(requests, tokens) of a ``[B, heads, 128]`` or ``[B, T, heads, 128]`` shape this layer can serve."""
        if len(shape) not in (3, 4):
            raise ValueError(f"{name} must be [requests, heads, 128] or [requests, tokens, heads, 128]")
        B, T = shape[0], shape[1] if len(shape) == 4 else 1
        if shape[-2] != heads or shape[-1] != _lib.HEAD_DIM:
            raise ValueError(f"{name} must have {heads} heads of 128 elements, got {tuple(shape)}")
        if B > self.max_requests or B > self._rows:
            raise ValueError(f"{B} requests: the layer was made for {self.max_requests}, the bound cache addresses {self._rows}")
        if not 1 <= T <= self.max_query_len:
            raise ValueError(f"{T} query tokens per request: the layer was made for 1..{self.max_query_len}")
        return B, T

    def _rows_at(self, t: torch.Tensor, name: str) -> int:
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise ValueError(f"{name} must be a {self.dtype} tensor on {self.device}, got {t.dtype} on {t.device}")
        a = t.data_ptr()
        if a & 15:
            raise ValueError(f"rows of {name} must be 16-byte aligned")
        return a

    def _strides_of(self, t: torch.Tensor, name: str) -> tuple[int, int, int]:
        """Element strides from one request, token and head to the next."""
        shape, st = t.shape, t.stride()
        s = (st[0], 0, st[1]) if len(shape) == 3 else (st[0], st[1], st[2])
        s = tuple(x if n > 1 else 0 for x, n in zip(s, (shape[0], shape[1] if len(shape) == 4 else 1, shape[-2])))  # one row has no stride
        if st[-1] != 1 or (s[0] | s[1] | s[2]) & (3 if self.dtype is torch.float32 else 7):
            raise ValueError(f"rows of {name} must be contiguous and 16-byte aligned")
        return s

    def _workspace_bytes(self, requests: int, tokens: int) -> tuple[int, int]:
        """Workspace of the attention at this size, without and with weights."""
        got = self._sizes.get((requests, tokens))
        if got is None:
            p = _lib.PagedParams.from_buffer_copy(self.p)
            p.requests, p.query_len, got = requests, tokens, []
            for mass in (None, 1):
                p.mass = mass
                got.append(int(_lib.lib.pqhsa_paged_workspace_bytes(C.byref(p))))
            got = self._sizes[requests, tokens] = tuple(got)
        return got

    def _scratch(self, kind: str) -> tuple[_Scratch, int, bool]:
        """The scratch memory of that kind of this stream (or this capture), the stream, and whether it is being captured."""
        stream = _raw_stream(self._index)
        capturing = _is_capturing()
        key = (kind, self._index, stream, _lib.lib.pqhsa_stream_capture_id(stream) if capturing else 0)
        scratch = self._ws.get(key)
        if scratch is None:
            scratch = self._ws[key] = _SCRATCH.setdefault(key, _Scratch())
        return scratch, stream, capturing

    def _positions(self, p, B: int, key_pos, query_pos, mass) -> None:
        p.key_pos = None if key_pos is None else self._per_slot(key_pos, "key_pos", torch.int32, B)
        p.query_pos = None if query_pos is None else self._per_request(query_pos, "query_pos", B)
        p.mass = None if mass is None else self._per_slot(mass, "mass", torch.float32, B)

    def _call(self, name: str, *args) -> None:
        """A library call with this layer's device current; the last argument of every entry point is the stream."""
        rc = getattr(_lib.lib, name)(*args)
        if rc != 0:
            raise _lib.PqhsaError(name, rc, _lib.lib.pqhsa_last_error_string().decode("utf-8", "replace"))

    # ---- calls ---------------------------------------------------------------------------------------------
    def forward(self, q: torch.Tensor, seq_lens: torch.Tensor, *, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                first_key: torch.Tensor | None = None, key_pos: torch.Tensor | None = None,
                query_pos: torch.Tensor | None = None, mass: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of ``q`` ``[B, Hq, 128]`` or ``[B, T, Hq, 128]`` (any strides with contiguous, aligned rows) over
        the first ``seq_lens[r]`` slots of every request, the T new tokens' own rows among them; rows 0 .. B - 1 of the
        bound block table.  Returns ``out`` (same shape as q; made if not given).

        ``lse``: float32 ``q.shape[:-1]``, receives ln of the row's exp-sum.  ``first_key`` int32 ``[B]``: first
        position of the request's current document.  ``key_pos`` int32 ``[>= B, Hkv, token_capacity]`` with ``query_pos``
        int32 ``[B]`` (position of the last query token): the slots' positions, after an eviction.  ``mass`` float32, same shape as
        key_pos: every slot's attention weights of this call are added to it."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.forward(q, seq_lens, out=out, lse=lse, first_key=first_key, key_pos=key_pos, query_pos=query_pos, mass=mass)
        if self._kv_keepalive is None:
            raise RuntimeError("bind_kv_paged or bind_kv_contiguous must be called first")
        p, shape = self.p, q.shape
        if out is None:
            out = torch.empty(shape, dtype=self.dtype, device=self.device)
        elif out.shape != shape:
            raise ValueError("out must match q in shape")
        p.q, p.out = self._rows_at(q, "q"), self._rows_at(out, "out")
        even = q.is_contiguous() and out.is_contiguous()
        if not even or shape != self._forward_shape:
            self._forward_shape = None  # what follows may refuse the call with the block half set
            p.requests, p.query_len = self._tokens(shape, "q", self.Hq)
            self._bytes = self._workspace_bytes(p.requests, p.query_len)
            p.q_stride_request, p.q_stride_token, p.q_stride_head = self._strides_of(q, "q")
            if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
                raise ValueError("rows of out must not lie on one another")
            p.out_stride_request, p.out_stride_token, p.out_stride_head = self._strides_of(out, "out")
            self._forward_shape = shape if even else None
        B = shape[0]
        p.seq_lens = self._per_request(seq_lens, "seq_lens", B)
        if lse is None:
            p.lse = None
        else:
            if lse.dtype is not torch.float32 or lse.get_device() != self._index or lse.shape != shape[:-1] or not lse.is_contiguous():
                raise ValueError(f"lse must be a contiguous float32 tensor of shape {tuple(shape[:-1])} on {self.device}")
            p.lse = lse.data_ptr()
        p.first_key = None if first_key is None else self._per_request(first_key, "first_key", B)
        if key_pos is not None and query_pos is None:
            raise ValueError("key_pos needs query_pos")
        self._positions(p, B, key_pos, query_pos, mass)
        p.workspace_bytes = n = self._bytes[0 if mass is None else 1]
        scratch, stream, capturing = self._scratch("attention")
        with scratch.lock:
            p.workspace = scratch.take(n, self.device, True, capturing)
            self._call("pqhsa_paged_attention", self._ref, stream)
        return out

    def append(self, keys: torch.Tensor, values: torch.Tensor, seq_lens: torch.Tensor, *, new_lens: torch.Tensor | None = None,
               key_pos: torch.Tensor | None = None, query_pos: torch.Tensor | None = None,
               mass: torch.Tensor | None = None) -> torch.Tensor:
        """Write T new rows ``[B, Hkv, 128]`` or ``[B, T, Hkv, 128]`` per request to slots ``seq_lens[r]`` and on, with
        their positions (``query_pos`` is that of the last; without it, the slots) in ``key_pos`` and no weight yet in
        ``mass``.  Returns ``new_lens`` = lengths + T, ``seq_lens`` itself if not given.  A negative length is an idle
        request; rows that do not fit are dropped."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.append(keys, values, seq_lens, new_lens=new_lens, key_pos=key_pos, query_pos=query_pos, mass=mass)
        if self._kv_keepalive is None:
            raise RuntimeError("bind_kv_paged or bind_kv_contiguous must be called first")
        p, shape = self._append_p, keys.shape
        k, v = self._rows_at(keys, "keys"), self._rows_at(values, "values")
        if values.shape != shape:
            raise ValueError("keys and values must have the same shape")
        even = keys.is_contiguous() and values.is_contiguous()
        if not even or shape != self._append_shape:
            self._append_shape = None
            p.requests, p.query_len = self._tokens(shape, "keys", self.H)
            s = self._strides_of(keys, "keys")
            if self._strides_of(values, "values") != s:
                raise ValueError("keys and values must have the same strides")
            p.q_stride_request, p.q_stride_token, p.q_stride_head = s
            self._append_shape = shape if even else None
        B = shape[0]
        p.seq_lens = at = self._per_request(seq_lens, "seq_lens", B)
        to = at if new_lens is None else self._per_request(new_lens, "new_lens", B)
        self._positions(p, B, key_pos, query_pos, mass)
        self._call("pqhsa_paged_append", self._append_ref, k, v, to, _raw_stream(self._index))
        return seq_lens if new_lens is None else new_lens

    def evict(self, seq_lens: torch.Tensor, *, mass: torch.Tensor, key_pos: torch.Tensor, query_pos: torch.Tensor, budget: int,
              recent: int = 0, new_lens: torch.Tensor | None = None, new_mass: torch.Tensor | None = None,
              new_pos: torch.Tensor | None = None, source: torch.Tensor | None = None) -> torch.Tensor:
        """Bring every request down to ``budget`` slots per KV head: the first ``sink_tokens`` and last ``recent``
        positions and the slots of the largest ``mass`` stay (ties: the lower slot; NaN goes first), packed into the
        first ``budget`` slots with as few moves as possible (K and V rows in place; ``mass`` and ``key_pos`` in place
        too unless ``new_mass`` / ``new_pos`` are given).  Returns ``new_lens``, ``seq_lens`` itself if not given.
        ``source`` int32 ``[B, Hkv, budget]`` receives the former slot of every kept slot (-1 past the end).  The pages
        of a request must be its own; whole pages behind the new length may be freed.  A slot on a page that the block
        table does not have is never moved or filled: below the budget it takes one of its places, behind it it goes."""
        if _current_device() != self._index:
            with torch.cuda.device(self._index):
                return self.evict(seq_lens, mass=mass, key_pos=key_pos, query_pos=query_pos, budget=budget, recent=recent,
                                  new_lens=new_lens, new_mass=new_mass, new_pos=new_pos, source=source)
        if self._kv_keepalive is None:
            raise RuntimeError("bind_kv_paged or bind_kv_contiguous must be called first")
        p = self._evict_p
        if not 1 <= budget <= 1 << 24 or recent < 0 or p.sink_tokens + recent > budget:
            raise ValueError(f"need budget >= 1 and sink_tokens + recent <= budget, got {budget}, {p.sink_tokens} + {recent}")
        B = seq_lens.shape[0]
        if B > self.max_requests or B > self._rows:
            raise ValueError(f"{B} requests: the layer was made for {self.max_requests}, the bound cache addresses {self._rows}")
        p.requests, p.query_len = B, 1
        p.seq_lens = at = self._per_request(seq_lens, "seq_lens", B)
        to = at if new_lens is None else self._per_request(new_lens, "new_lens", B)
        self._positions(p, B, key_pos, query_pos, mass)
        nm = p.mass if new_mass is None else self._per_slot(new_mass, "new_mass", torch.float32, B)
        npos = p.key_pos if new_pos is None else self._per_slot(new_pos, "new_pos", torch.int32, B)
        n = 4 * B * self.H * (2 * budget + 8)
        if source is not None and (source.dtype is not torch.int32 or source.get_device() != self._index
                                   or source.shape != (B, self.H, budget) or not source.is_contiguous()):
            raise ValueError(f"source must be a contiguous int32 [{B}, {self.H}, {budget}] tensor on {self.device}")
        scratch, stream, capturing = self._scratch("evict")
        with scratch.lock:
            lists = scratch.take(n + 4 * B * self.H * budget, self.device, False, capturing)
            src = lists + n if source is None else source.data_ptr()
            self._call("pqhsa_paged_evict", self._evict_ref, int(budget), int(recent), to, nm, npos, src, lists, stream)
        return seq_lens if new_lens is None else new_lens
