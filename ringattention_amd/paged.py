"""Serving from a paged K/V cache: PagedAttention, on top of the C ABI (ringattn_paged_* in include/ringattn.h).

The calls of a step of a serving loop, for a ragged batch of sequences with some new tokens each:

    plan.append(k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores)      the new tokens' rows into the cache
    plan.forward(q, k_cache, v_cache, page_table, kv_lens, q_starts)                their attention over it: (out, lse)
    plan.weights(q, lse, k_cache, page_table, kv_lens, q_starts, scores)            what they gave to each cached token
    plan.evict(k_cache, v_cache, scores, page_table, kv_lens, kept_table, budget)   now and then: the tokens that drew most stay

Tensors (device): k_cache, v_cache [pages, kv_heads, page_size, dim] (any strides that keep a row together, both alike); page_table int32
[batch, pages of a sequence], -1 where there is none; kv_lens int32 [batch], tokens in the cache, the new ones among them; q_starts int32
[batch + 1], where a sequence's new tokens begin; q, out [tokens, heads, dim], k, v [tokens, kv_heads, dim] (any strides that
keep a row together); lse float32 [heads, tokens]; scores float32 [pages, kv_heads, page_size].  Lengths, starts and tables are read
on the device, by captured graphs at every replay.
"""
import ctypes

import torch

from . import _lib
from ._lib import RingattnPagedCache, RingattnPagedParams, check
from .api import DTYPE_CODE, TORCH_DTYPE, _check_tensors, _stream_ptr

FLAG_PAGED_PARTIALS = 1
FLAG_PAGED_KEEP_PRESENT = 4


def _check_rows(*specs):
    """specs: (tensor, name, dtype, shape): as api._check_tensors, for tensors of any strides that keep a row together in 16-byte steps."""
    for t, name, dtype, shape in specs:
        if tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
        if t.dtype != dtype:
            raise ValueError(f"{name} must have dtype {dtype}")
    for t, name, dtype, _ in specs:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a device tensor")
        step = 16 // t.element_size()
        if t.stride(-1) != 1 or any(n > 1 and (s < 0 or s % step) for n, s in zip(t.shape[:-1], t.stride()[:-1])) or t.data_ptr() % 16:
            raise ValueError(f"{name} must have contiguous rows that begin at multiples of 16 bytes")


def _strides(t):
    """Strides of all dimensions but the last, those of length one as if the tensor were contiguous."""
    made, step = [], t.shape[-1]
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        made.append(s if n > 1 else step)
        step = made[-1] * n
    return made[::-1]


class PagedAttention:
    """A plan for `heads` query heads on `kv_heads` KV heads of `dim`, pages of `page_size` tokens (16, 32, ... 1024), calls of up to
    `max_batch` sequences and `max_tokens` new tokens.

    `window` > 0: a token sees the last `window` tokens up to itself and the first `sinks` of the sequence.  `causal=False`:
    it sees every cached token; `partials`: out is float32, a partial (O, LSE) for api.merge -- together, for a sequence whose cache is
    spread over several pools or GPUs.  `keep_present`: evict() keeps no token whose page is not there.  `workspace`: a (device
    address, bytes) pair the caller owns and keeps alive, instead of an allocation by the plan.  It holds zeros when the plan is made
    (torch.zeros, not torch.empty): workgroups that share a row count themselves in it, and leave it at 0.  One call at a time, and replays
    of captured calls in turn: they share the plan's workspace."""

    def __init__(self, heads, dim, kv_heads=0, dtype="fp16", page_size=64, max_batch=64, max_tokens=8192, causal=True, softmax_scale=0.0,
                 window=0, sinks=0, partials=False, workspace=None, keep_present=False):
        self.lib = _lib.load()
        self.heads, self.dim, self.kv_heads, self.page_size = int(heads), int(dim), int(kv_heads) or int(heads), int(page_size)
        self.max_batch, self.max_tokens = int(max_batch), int(max_tokens)
        for name, x in (("heads", heads), ("dim", dim), ("kv_heads", kv_heads), ("page_size", page_size), ("max_batch", max_batch),
                        ("max_tokens", max_tokens), ("window", window), ("sinks", sinks)):
            if not -2 ** 31 <= int(x) < 2 ** 31:   # (a field of the struct would take what is left of it)
                raise ValueError(f"{name} must fit 32 bits")
        code = DTYPE_CODE[dtype]
        self.torch_dtype = TORCH_DTYPE[code]
        self.out_dtype = torch.float32 if partials else self.torch_dtype
        self.params = RingattnPagedParams(self.dim, self.heads, int(kv_heads), code, float(softmax_scale), self.page_size, self.max_batch,
                                          self.max_tokens, int(bool(causal)), int(window), int(sinks),
                                          (FLAG_PAGED_PARTIALS if partials else 0) | (FLAG_PAGED_KEEP_PRESENT if keep_present else 0))
        self.handle = ctypes.c_void_p()
        self.device = torch.cuda.current_device() if workspace is None and torch.cuda.is_available() else None
        ws_ptr, ws_bytes = (None, 0) if workspace is None else (ctypes.c_void_p(int(workspace[0])), int(workspace[1]))
        check(self.lib.ringattn_paged_plan_create(ctypes.byref(self.params), ws_ptr, ws_bytes, ctypes.byref(self.handle)),
              "ringattn_paged_plan_create")
        # Checks and launch of a call with tensors of the caller's in native code (csrc/ringattn_calls.cpp), made when first asked for; it
        # gives None where something is unusual, and the call then goes the general way.
        calls = _lib.load_calls()
        self._call_type = calls.Paged if calls and self.device is not None else None
        self._native = {}

    def _made(self, kind):
        entry = self.lib.addresses[("ringattn_paged_append", "ringattn_paged_fwd", "ringattn_paged_weights", "ringattn_paged_evict")[kind]]
        self._native[kind] = call = self._call_type(entry, self.handle.value, kind, self.heads, self.kv_heads, self.dim, self.page_size,
                                                    self.max_batch, self.max_tokens, self.device, self.torch_dtype, self.out_dtype)
        return call

    def close(self):
        self._call_type, self._native = None, {}
        if self.handle:
            check(self.lib.ringattn_paged_plan_destroy(self.handle), "ringattn_paged_plan_destroy")
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def workspace_bytes(self):
        return self.lib.ringattn_paged_workspace_bytes(ctypes.byref(self.params))

    # ---- what every call has
    def _cache(self, k_cache, v_cache, page_table, kv_lens, q_starts):
        """The checked sequences of a call as struct ringattn_paged_cache."""
        if k_cache.dim() != 4 or page_table.dim() != 2:
            raise ValueError("k_cache must be [pages, kv_heads, page_size, dim] and page_table [batch, pages of a sequence]")
        shape = (k_cache.shape[0], self.kv_heads, self.page_size, self.dim)
        batch = page_table.shape[0]
        if batch > self.max_batch:
            raise ValueError(f"the plan takes up to {self.max_batch} sequences, not {batch}")
        ints = [(kv_lens, "kv_lens", torch.int32, (batch,))]
        if q_starts is not None:
            ints.append((q_starts, "q_starts", torch.int32, (batch + 1,)))
        rows = [(k_cache, "k_cache", self.torch_dtype, shape)]
        if v_cache is not None:
            rows.append((v_cache, "v_cache", self.torch_dtype, shape))
        if page_table.dtype != torch.int32:
            raise ValueError("page_table must have dtype torch.int32")
        _check_tensors(*ints)
        _check_rows(*rows)
        if not page_table.is_cuda:
            raise ValueError("page_table must be a device tensor")
        if page_table.shape[1] > 1 and page_table.stride(1) != 1 or batch > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("page_table must have contiguous rows")
        strides = _strides(k_cache)
        if v_cache is not None and _strides(v_cache) != strides:
            raise ValueError("k_cache and v_cache must have the same strides")
        self._same_device(k_cache, v_cache, page_table, kv_lens, q_starts)
        return RingattnPagedCache(k_cache.data_ptr(), v_cache.data_ptr() if v_cache is not None else None, *strides, k_cache.shape[0],
                                  page_table.shape[1], page_table.stride(0) if batch > 1 else page_table.shape[1], page_table.data_ptr(),
                                  kv_lens.data_ptr(), q_starts.data_ptr() if q_starts is not None else None, batch)

    def _same_device(self, first, *others):
        for t in others:
            if t is not None and t.device != first.device:
                raise ValueError("the tensors of a call must be on one device")
        if self.device is not None and first.device.index != self.device:
            raise ValueError(f"the plan's workspace is on device {self.device}")

    def _tokens(self, t, name, heads):
        if t.dim() != 3:
            raise ValueError(f"{name} must be [tokens, {heads}, {self.dim}]")
        if t.shape[0] > self.max_tokens:
            raise ValueError(f"the plan takes up to {self.max_tokens} new tokens, not {t.shape[0]}")
        return (t.shape[0], heads, self.dim)

    def _call(self, name, device, stream, *args):
        """A launch on the tensors' own device, whichever is the current one."""
        if device.index == torch.cuda.current_device():
            check(getattr(self.lib, name)(self.handle, *args, _stream_ptr(stream)), name)
        else:
            with torch.cuda.device(device):
                check(getattr(self.lib, name)(self.handle, *args, _stream_ptr(stream)), name)

    @staticmethod
    def _new(shape, dtype, device, stream):
        """An output of a call on `stream`, whose memory is that stream's."""
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=device)

    def append(self, k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores=None, stream=None):
        """Rows k, v [tokens, kv_heads, dim] of the new tokens into the cache, as the last of each sequence's kv_lens tokens; their scores to 0."""
        if self._call_type:
            rc = (self._native.get(0) or self._made(0))(k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores, stream)
            if rc is not None:
                return check(rc, "ringattn_paged_append")
        shape = self._tokens(k, "k", self.kv_heads)
        cache = self._cache(k_cache, v_cache, page_table, kv_lens, q_starts)
        _check_rows((k, "k", self.torch_dtype, shape), (v, "v", self.torch_dtype, shape))
        if _strides(k) != _strides(v):
            raise ValueError("k and v must have the same strides")
        if scores is not None:
            _check_tensors((scores, "scores", torch.float32, k_cache.shape[:3]))
        self._same_device(k_cache, k, v, scores)
        if shape[0] == 0 or cache.batch == 0:
            return
        self._call("ringattn_paged_append", k.device, stream, ctypes.byref(cache), k.data_ptr(), v.data_ptr(), shape[0], *_strides(k),
                   scores.data_ptr() if scores is not None else None)

    def forward(self, q, k_cache, v_cache, page_table, kv_lens, q_starts, out=None, lse=None, stream=None):
        """Attention of the new tokens q [tokens, heads, dim] over the cache (their own rows are in it).  Returns (out, lse)."""
        if out is not None and lse is not None and self._call_type:
            rc = (self._native.get(1) or self._made(1))(q, k_cache, v_cache, page_table, kv_lens, q_starts, out, lse, stream)
            if rc is not None:
                check(rc, "ringattn_paged_fwd")
                return out, lse
        shape = self._tokens(q, "q", self.heads)
        cache = self._cache(k_cache, v_cache, page_table, kv_lens, q_starts)
        _check_rows((q, "q", self.torch_dtype, shape))
        if out is None:   # head by head where q is
            by_head = shape[0] > 1 and self.heads > 1 and q.stride(1) > q.stride(0)
            out = self._new((self.heads, shape[0], self.dim) if by_head else shape, self.out_dtype, q.device, stream)
            out = out.transpose(0, 1) if by_head else out
        if lse is None:
            lse = self._new((self.heads, shape[0]), torch.float32, q.device, stream)
        _check_rows((out, "out", self.out_dtype, shape))
        _check_tensors((lse, "lse", torch.float32, (self.heads, shape[0])))
        self._same_device(k_cache, q, out, lse)
        if shape[0] == 0 or cache.batch == 0:
            return out, lse
        self._call("ringattn_paged_fwd", q.device, stream, ctypes.byref(cache), q.data_ptr(), shape[0], *_strides(q), out.data_ptr(), *_strides(out),
                   lse.data_ptr())
        return out, lse

    def weights(self, q, lse, k_cache, page_table, kv_lens, q_starts, scores, stream=None):
        """Adds to scores what forward(q, ...) that returned `lse` gave to every cached token: the sum of its attention weights over the
        new tokens and the query heads of each KV head.  Returns scores."""
        if self._call_type:
            rc = (self._native.get(2) or self._made(2))(q, lse, k_cache, page_table, kv_lens, q_starts, scores, stream)
            if rc is not None:
                check(rc, "ringattn_paged_weights")
                return scores
        shape = self._tokens(q, "q", self.heads)
        cache = self._cache(k_cache, None, page_table, kv_lens, q_starts)
        _check_rows((q, "q", self.torch_dtype, shape))
        _check_tensors((lse, "lse", torch.float32, (self.heads, shape[0])), (scores, "scores", torch.float32, k_cache.shape[:3]))
        self._same_device(k_cache, q, lse, scores)
        if shape[0] == 0 or cache.batch == 0:
            return scores
        self._call("ringattn_paged_weights", q.device, stream, ctypes.byref(cache), q.data_ptr(), shape[0], *_strides(q), lse.data_ptr(),
                   scores.data_ptr())
        return scores

    def evict(self, k_cache, v_cache, scores, page_table, kv_lens, kept_table, budget, keep_first=0, keep_last=0, kept=None, kept_lens=None,
              stream=None):
        """Copies `budget` tokens of every sequence -- its first keep_first, its last keep_last, and between them those of the largest
        scores, for each KV head its own -- with their scores to the pages of kept_table, which are in none of page_table.
        Returns (kept, kept_lens): the places the tokens had [batch, kv_heads, budget], -1 behind the last, and the lengths that go with
        kept_table (may be the tensor kv_lens itself).

        A token that stays although its page is not there -- of a short sequence, or of the first or last -- is not copied: its row of the
        kept pages holds what it held, and would be seen.  Where pages have been given away, make the plan with keep_present: kept_lens is
        then what is left of min(kv_lens, budget) without such tokens."""
        if kept is not None and kept_lens is not None and self._call_type:
            rc = (self._native.get(3) or self._made(3))(k_cache, v_cache, scores, page_table, kv_lens, kept_table, budget, keep_first, keep_last,
                                                        kept, kept_lens, stream)
            if rc is not None:
                check(rc, "ringattn_paged_evict")
                return kept, kept_lens
        batch, budget = page_table.shape[0], int(budget)
        if kept_table.dim() != 2 or kept_table.shape[0] != batch or kept_table.shape[1] * self.page_size < budget:
            raise ValueError(f"kept_table must be [{batch}, pages for {budget} tokens]")
        if budget < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
            raise ValueError("budget must be positive and hold the first and the last tokens")
        cache = self._cache(k_cache, v_cache, page_table, kv_lens, None)
        if kept is None:
            kept = self._new((batch, self.kv_heads, budget), torch.int32, k_cache.device, stream)
        if kept_lens is None:
            kept_lens = self._new((batch,), torch.int32, k_cache.device, stream)
        _check_tensors((scores, "scores", torch.float32, k_cache.shape[:3]), (kept_table, "kept_table", torch.int32, kept_table.shape),
                       (kept, "kept", torch.int32, (batch, self.kv_heads, budget)), (kept_lens, "kept_lens", torch.int32, (batch,)))
        self._same_device(k_cache, scores, kept_table, kept, kept_lens)
        if cache.batch == 0:
            return kept, kept_lens
        self._call("ringattn_paged_evict", k_cache.device, stream, ctypes.byref(cache), scores.data_ptr(), kept_table.data_ptr(), kept_table.shape[1],
                   kept_table.shape[1], budget, int(keep_first), int(keep_last), kept.data_ptr(), kept_lens.data_ptr())
        return kept, kept_lens
