"""Serving from a paged K/V cache: PagedAttention, on top of the C ABI (ringattn_paged_* in include/ringattn.h).

The calls of a step of a serving loop, for a ragged batch of sequences with some new tokens each:

    plan.append(k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores)      the new tokens' rows into the cache
    plan.forward(q, k_cache, v_cache, page_table, kv_lens, q_starts)                their attention over it: (out, lse)
    plan.weights(q, lse, k_cache, page_table, kv_lens, q_starts, scores)            what they gave to each cached token
    plan.evict(k_cache, v_cache, scores, page_table, kv_lens, kept_table, budget)   now and then: the tokens that drew most stay

Of models with rotary positions, plan.append_rotary(rotary, q, k, v, ...) in place of append().  Capped scores and slopes of distance are a plan's
(softcap, slopes), prefixes that all tokens see and documents one behind the other a call's (prefix_lens, first_keys).  PagePool keeps the page table
on the device: forks, growth, releases, compaction.

Tensors (device): k_cache, v_cache [pages, kv_heads, page_size, dim] (any strides that keep a row together, both alike); page_table int32
[batch, pages of a sequence], -1 where there is none; kv_lens int32 [batch], tokens in the cache, the new ones among them; q_starts int32
[batch + 1], where a sequence's new tokens begin; q, out [tokens, heads, dim], k, v [tokens, kv_heads, dim] (any strides that
keep a row together); lse float32 [heads, tokens]; scores float32 [pages, kv_heads, page_size].  Lengths, starts and tables are read
on the device, by captured graphs at every replay.
"""
import ctypes

import torch

from . import _lib
from ._lib import RingattnPagedCache, RingattnPagedParams, RingattnPagedPool, RingattnPagedScoring, RingattnPages, check
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
    spread over several pools or GPUs.  `softcap` > 0, up to 1024: a score x becomes softcap tanh(x / softcap); `slopes`, float32 [heads] on the device: less
    slopes[head] times the distance of query and key (causal plans); for forward() and weights().  `keep_present`: evict() keeps no token whose page is not there.  `workspace`: a (device
    address, bytes) pair the caller owns and keeps alive, instead of an allocation by the plan.  It holds zeros when the plan is made
    (torch.zeros, not torch.empty): workgroups that share a row count themselves in it, and leave it at 0.  One call at a time, and replays
    of captured calls in turn: they share the plan's workspace."""

    def __init__(self, heads, dim, kv_heads=0, dtype="fp16", page_size=64, max_batch=64, max_tokens=8192, causal=True, softmax_scale=0.0,
                 window=0, sinks=0, partials=False, workspace=None, keep_present=False, softcap=0.0, slopes=None):
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
        self._softcap, self._slopes = ctypes.c_float(softcap).value, slopes
        if not 0 <= float(softcap) <= 1024 or (softcap and not self._softcap):   # (what is nothing in 32 bits would be no cap)
            raise ValueError("softcap must be 0 or a positive number up to 1024")
        if slopes is not None:
            if not causal:
                raise ValueError("slopes are for causal plans")
            _check_tensors((slopes, "slopes", torch.float32, (self.heads,)))
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

    # (calls that are made in native code hold the one, and the other has been checked: a plan's own, not to be replaced)
    softcap = property(lambda self: self._softcap)
    slopes = property(lambda self: self._slopes)

    def _made(self, kind):
        entry = self.lib.addresses[("ringattn_paged_append", "ringattn_paged_fwd", "ringattn_paged_weights", "ringattn_paged_evict",
                                    "ringattn_paged_fwd_scored", "ringattn_paged_weights_scored", "ringattn_paged_append_rotary")[kind]]
        self._native[kind] = call = self._call_type(entry, self.handle.value, kind if kind < 4 else 12 + kind, self.heads, self.kv_heads, self.dim, self.page_size,
                                                    self.max_batch, self.max_tokens, self.device, self.torch_dtype, self.out_dtype, self.softcap)
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

    def _scoring(self, prefix_lens, first_keys, batch, tokens):
        """What a call does with its scores as struct ringattn_paged_scoring."""
        if (prefix_lens is not None or first_keys is not None) and not self.params.causal:
            raise ValueError("prefixes and first keys are for causal plans")
        if prefix_lens is not None:
            _check_tensors((prefix_lens, "prefix_lens", torch.int32, (batch,)))
        if first_keys is not None:
            _check_tensors((first_keys, "first_keys", torch.int32, (tokens,)))
        return RingattnPagedScoring(self.softcap, *(t.data_ptr() if t is not None else None for t in (self.slopes, prefix_lens, first_keys)))

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

    @staticmethod
    def _like(t, stream):
        """A tensor that lies in memory as t does, of a call on `stream`."""
        if stream is None:
            return torch.empty_like(t)
        with torch.cuda.stream(stream):
            return torch.empty_like(t)

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

    def append_rotary(self, rotary, q, k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores=None, positions=None, q_out=None, stream=None):
        """append() with rotary positions on the way (rotary.Rotary): K turned and V as it is into the cache, q [tokens, heads, dim] turned into q_out
        (q itself for in place; not on rows of k or v, between which it may lie).  `positions` int32 [tokens]; None: a token's place in its sequence.
        Returns q_out."""
        rotary.check(self.dim, self.torch_dtype)
        if q_out is not None and self._call_type:
            rc = (self._native.get(6) or self._made(6))(q, k, v, k_cache, v_cache, page_table, kv_lens, q_starts, scores, positions, q_out, rotary.address,
                                                        rotary.turns, stream)
            if rc is not None:
                check(rc, "ringattn_paged_append_rotary")
                return q_out
        shape, kv_shape = self._tokens(q, "q", self.heads), self._tokens(k, "k", self.kv_heads)
        if kv_shape[0] != shape[0]:
            raise ValueError("q and k must have as many tokens")
        cache = self._cache(k_cache, v_cache, page_table, kv_lens, q_starts)
        _check_rows((q, "q", self.torch_dtype, shape), (k, "k", self.torch_dtype, kv_shape), (v, "v", self.torch_dtype, kv_shape))
        if _strides(k) != _strides(v):
            raise ValueError("k and v must have the same strides")
        if q_out is None:
            q_out = self._like(q, stream)
        _check_rows((q_out, "q_out", self.torch_dtype, shape))
        if scores is not None:
            _check_tensors((scores, "scores", torch.float32, k_cache.shape[:3]))
        if positions is not None:
            _check_tensors((positions, "positions", torch.int32, (shape[0],)))
        self._same_device(k_cache, q, q_out, k, v, scores, positions, rotary.turns)
        if shape[0] == 0 or cache.batch == 0:
            return q_out
        self._call("ringattn_paged_append_rotary", k.device, stream, ctypes.byref(cache), ctypes.byref(rotary.params(False)),
                   positions.data_ptr() if positions is not None else None, q.data_ptr(), *_strides(q), q_out.data_ptr(), *_strides(q_out), k.data_ptr(),
                   v.data_ptr(), shape[0], *_strides(k), scores.data_ptr() if scores is not None else None)
        return q_out

    def forward(self, q, k_cache, v_cache, page_table, kv_lens, q_starts, out=None, lse=None, stream=None, prefix_lens=None, first_keys=None):
        """Attention of the new tokens q [tokens, heads, dim] over the cache (their own rows are in it).  Returns (out, lse).

        `prefix_lens`, int32 [batch]: all new tokens of a sequence see so many first tokens, also those that come behind them.  `first_keys`, int32
        [tokens]: a token sees no key in front of this place (the first token of its document), but for the prefix and the sinks."""
        plain = prefix_lens is None and first_keys is None and self.slopes is None and not self.softcap
        if plain and out is not None and lse is not None and self._call_type:
            rc = (self._native.get(1) or self._made(1))(q, k_cache, v_cache, page_table, kv_lens, q_starts, out, lse, stream)
            if rc is not None:
                check(rc, "ringattn_paged_fwd")
                return out, lse
        elif out is not None and lse is not None and self._call_type and (self.params.causal or prefix_lens is None and first_keys is None):
            rc = (self._native.get(4) or self._made(4))(q, k_cache, v_cache, page_table, kv_lens, q_starts, out, lse, self.slopes, prefix_lens, first_keys, stream)
            if rc is not None:
                check(rc, "ringattn_paged_fwd_scored")
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
        scoring = self._scoring(prefix_lens, first_keys, cache.batch, shape[0])
        self._same_device(k_cache, q, out, lse, prefix_lens, first_keys, self.slopes)
        if shape[0] == 0 or cache.batch == 0:
            return out, lse
        self._call("ringattn_paged_fwd_scored", q.device, stream, ctypes.byref(cache), ctypes.byref(scoring), q.data_ptr(), shape[0], *_strides(q), out.data_ptr(), *_strides(out),
                   lse.data_ptr())
        return out, lse

    def weights(self, q, lse, k_cache, page_table, kv_lens, q_starts, scores, stream=None, prefix_lens=None, first_keys=None):
        """Adds to scores what forward(q, ...) that returned `lse` gave to every cached token: the sum of its attention weights over the
        new tokens and the query heads of each KV head.  prefix_lens and first_keys as forward() had them.  Returns scores."""
        plain = prefix_lens is None and first_keys is None and self.slopes is None and not self.softcap
        if plain and self._call_type:
            rc = (self._native.get(2) or self._made(2))(q, lse, k_cache, page_table, kv_lens, q_starts, scores, stream)
            if rc is not None:
                check(rc, "ringattn_paged_weights")
                return scores
        elif self._call_type and (self.params.causal or prefix_lens is None and first_keys is None):
            rc = (self._native.get(5) or self._made(5))(q, lse, k_cache, page_table, kv_lens, q_starts, scores, self.slopes, prefix_lens, first_keys, stream)
            if rc is not None:
                check(rc, "ringattn_paged_weights_scored")
                return scores
        shape = self._tokens(q, "q", self.heads)
        cache = self._cache(k_cache, None, page_table, kv_lens, q_starts)
        _check_rows((q, "q", self.torch_dtype, shape))
        _check_tensors((lse, "lse", torch.float32, (self.heads, shape[0])), (scores, "scores", torch.float32, k_cache.shape[:3]))
        scoring = self._scoring(prefix_lens, first_keys, cache.batch, shape[0])
        self._same_device(k_cache, q, lse, scores, prefix_lens, first_keys, self.slopes)
        if shape[0] == 0 or cache.batch == 0:
            return scores
        self._call("ringattn_paged_weights_scored", q.device, stream, ctypes.byref(cache), ctypes.byref(scoring), q.data_ptr(), shape[0], *_strides(q), lse.data_ptr(),
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


def _pool(k_cache, v_cache, scores, page_size):
    """The checked pool of a call as struct ringattn_paged_pool."""
    if k_cache.dim() != 4 or k_cache.dtype not in TORCH_DTYPE.values():
        raise ValueError("k_cache must be [pages, kv_heads, page_size, dim] of 16-bit floats")
    if k_cache.shape[2] != page_size:
        raise ValueError(f"k_cache must have pages of {page_size} tokens")
    _check_rows((k_cache, "k_cache", k_cache.dtype, k_cache.shape), (v_cache, "v_cache", k_cache.dtype, k_cache.shape))
    strides = _strides(k_cache)
    if _strides(v_cache) != strides:
        raise ValueError("k_cache and v_cache must have the same strides")
    if scores is not None:
        _check_tensors((scores, "scores", torch.float32, k_cache.shape[:3]))
    for t in (v_cache, scores):
        if t is not None and t.device != k_cache.device:
            raise ValueError("the tensors of a call must be on one device")
    return RingattnPagedPool(k_cache.data_ptr(), v_cache.data_ptr(), scores.data_ptr() if scores is not None else None, *strides, k_cache.shape[1], k_cache.shape[3])


def _on(device, stream, fn, *args):
    """A launch on the tensors' own device, whichever is the current one."""
    if device.index == torch.cuda.current_device():
        return fn(*args, _stream_ptr(stream))
    with torch.cuda.device(device):
        return fn(*args, _stream_ptr(stream))


def copy_pages(k_from, v_from, k_to, v_to, pairs, scores_from=None, scores_to=None, stream=None):
    """K, V (and scores) of pages from one pool to another of as many heads, or within one: pairs int32 [n, 2], from which page to which.  A page that
    is written to is in no other pair; pairs outside the pools are left out."""
    page = k_from.shape[2] if k_from.dim() == 4 else 0
    source, target = _pool(k_from, v_from, scores_from, page), _pool(k_to, v_to, scores_to, page)
    if k_from.dtype != k_to.dtype or k_from.shape[1:] != k_to.shape[1:]:
        raise ValueError("the two pools must have pages of the same shape and dtype")
    if (scores_from is None) != (scores_to is None):
        raise ValueError("scores of both pools, or of none")
    if pairs.dim() != 2:
        raise ValueError("pairs must be [n, 2]")
    _check_tensors((pairs, "pairs", torch.int32, (pairs.shape[0], 2)))
    for t in (k_to, pairs):
        if t.device != k_from.device:
            raise ValueError("the tensors of a call must be on one device")
    if pairs.shape[0]:
        check(_on(k_from.device, stream, _lib.load().ringattn_pages_copy, ctypes.byref(source), k_from.shape[0], ctypes.byref(target), k_to.shape[0], page,
                  pairs.data_ptr(), pairs.shape[0]), "ringattn_pages_copy")


class PagePool:
    """Which rows of a page table own and share which of `pages` pages, on the device: `page_table` int32 [rows, table_pages], `lens` int32 [rows],
    `refs` int32 [pages], how many entries of the table name a page (0: free).  They are a PagedAttention call's page_table and kv_lens as
    they are, or rows of theirs.  They are written in place, not replaced.  A caller may count entries of its own in refs (a prompt that is kept): those pages are not given out, and not written on.

        pool.update(k_cache, v_cache, parents, add)      rows become forks of others, or begin anew, and grow: before a step's append()
        pool.compact(k_cache, v_cache)                   the pages in use to the front of the pool

    The same calls give the same tables in every run.  Nothing waits for the host; calls may be captured.  One call at a time."""

    def __init__(self, pages, rows, table_pages, page_size=64, device=None):
        self.lib = _lib.load()
        self.pages, self.rows, self.table_pages, self.page_size = int(pages), int(rows), int(table_pages), int(page_size)
        for name, x in (("pages", self.pages), ("rows", self.rows), ("table_pages", self.table_pages)):
            if not 0 < x < 2 ** 31:
                raise ValueError(f"{name} must be positive and fit 32 bits")
        if self.page_size not in (16, 32, 64, 128, 256, 512, 1024) or self.table_pages * self.page_size > 2 ** 30:
            raise ValueError("page_size must be 16, 32, ... 1024, and a row of the table have room for 2^30 tokens at most")
        bytes_ = self.lib.ringattn_pages_scratch_bytes(self.pages, self.rows, self.table_pages)
        if bytes_ == 0:
            raise ValueError("up to 4096 rows, and 2^30 entries of the table")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        ints = dict(dtype=torch.int32, device=device)
        self._refs, self._lens = torch.zeros(self.pages, **ints), torch.zeros(self.rows, **ints)
        self._table = torch.full((self.rows, self.table_pages), -1, **ints)
        self._scratch = torch.empty(bytes_, dtype=torch.uint8, device=device)
        calls = _lib.load_calls()
        self._native = None
        self._struct = RingattnPages(self.refs.data_ptr(), self.page_table.data_ptr(), self.lens.data_ptr(), self.table_pages, self.pages, self.rows,
                                     self.table_pages, self.page_size, self._scratch.data_ptr(), bytes_)
        if calls and device.type == "cuda":   # checks and launches in native code, as PagedAttention's
            self._native = [calls.Pages(self.lib.addresses[name], ctypes.addressof(self._struct), kind, self.refs.device.index)
                            for kind, name in enumerate(("ringattn_pages_update", "ringattn_pages_compact"))]

    # (tensors of the pool's own, whose addresses its calls hold: written in place, not replaced)
    refs = property(lambda self: self._refs)
    lens = property(lambda self: self._lens)
    page_table = property(lambda self: self._table)

    def _checked(self, k_cache, v_cache, scores, pairs, *ints):
        """The checked pool of a call, None where there is none and the caller copies by `pairs`, (tensor, name, shape)."""
        pool = None
        if k_cache is not None:
            pool = _pool(k_cache, v_cache, scores, self.page_size)
            if k_cache.shape[0] != self.pages:
                raise ValueError(f"k_cache must have {self.pages} pages")
        elif pairs[0] is None or v_cache is not None or scores is not None:
            raise ValueError(f"without a cache, {pairs[1]} are needed")
        for t, name, shape in (pairs,) + ints:
            if t is not None:
                _check_tensors((t, name, torch.int32, shape))
        for t in (k_cache, pairs[0]) + tuple(t for t, _, _ in ints):
            if t is not None and t.device != self.refs.device:
                raise ValueError(f"the tensors of a call must be on {self.refs.device}, where the table is")
        return ctypes.byref(pool) if pool is not None else None

    def update(self, k_cache, v_cache, parents=None, add=None, scores=None, short=None, copies=None, stream=None):
        """All rows at once, from what they are before the call: row b begins with the tokens of row parents[b] (int32 [rows]; outside of [0, rows): with
        none), sharing their pages, and has add[b] more (int32 [rows]; negative: fewer).  Rows that grow take free pages, lowest first, in the order of
        the rows while there are enough; a page that is written on from within and that others name too is copied (K, V and `scores`).
        Returns short, int32 [rows]: 1 where a row was to grow and did not -- it then has what it began with.

        Several caches (a model's layers) go by one table: `copies`, int32 [rows, 2], gets the pairs for copy_pages in the others; with None for k_cache and
        v_cache nothing is copied here."""
        if short is not None and copies is None and self._native:
            rc = self._native[0](k_cache, v_cache, scores, parents, add, short, stream)
            if rc is not None:
                check(rc, "ringattn_pages_update")
                return short
        rows = (self.rows,)
        pool = self._checked(k_cache, v_cache, scores, (copies, "copies", (self.rows, 2)), (parents, "parents", rows), (add, "add", rows), (short, "short", rows))
        if short is None:
            short = PagedAttention._new(rows, torch.int32, self.refs.device, stream)
        check(_on(self.refs.device, stream, self.lib.ringattn_pages_update, ctypes.byref(self._struct), pool,
                  *(t.data_ptr() if t is not None else None for t in (parents, add, short, copies))), "ringattn_pages_update")
        return short

    def compact(self, k_cache, v_cache, scores=None, used=None, moved=None, moves=None, stream=None):
        """The n pages that something names to the first n places of the pool, their counts and the table with them; the others are free.  `moved`,
        int32 [pages]: where the page of a place is now, -1 for free ones.  `moves`, int32 [pages, 2]: the pairs for copy_pages in other caches that go by
        this table, as update()'s copies.  Returns used, int32 [1]: n."""
        if used is not None and moves is None and self._native:
            rc = self._native[1](k_cache, v_cache, scores, moved, None, used, stream)
            if rc is not None:
                check(rc, "ringattn_pages_compact")
                return used
        pool = self._checked(k_cache, v_cache, scores, (moves, "moves", (self.pages, 2)), (used, "used", (1,)), (moved, "moved", (self.pages,)))
        if used is None:
            used = PagedAttention._new((1,), torch.int32, self.refs.device, stream)
        check(_on(self.refs.device, stream, self.lib.ringattn_pages_compact, ctypes.byref(self._struct), pool,
                  *(t.data_ptr() if t is not None else None for t in (used, moved, moves))), "ringattn_pages_compact")
        return used
