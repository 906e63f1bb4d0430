"""Rotary positions on top of the C ABI (ringattn_rotary_* in include/ringattn.h): Rotary, for the Q and K of a ring
(apply), gradients by what apply() returned to those by what it was given (apply with inverse=True, called by hand: no call here is part of autograd's
graph), and the new tokens of a paged cache (paged.PagedAttention.append_rotary).

    rotary = Rotary(128, scaling="yarn", factor=8, trained=4096, dtype="bf16")
    q, k = rotary.apply(q, k, positions)                                    [batch, heads, tokens, dim], or [tokens, heads, dim]
    positions = torch.from_numpy(zigzag_order(plan.seqlen)).int().cuda()    of a ring in the zigzag layout
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import RingattnRotary, RingattnRows, check
from .api import DTYPE_CODE, TORCH_DTYPE, _check_tensors, _stream_ptr

MAX_POSITIONS = 2 ** 30   # tokens of a call


def frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, trained=0):
    """(radians per position of every pair, what turned columns are multiplied by), as Python floats.

    base^(-2 i / rotary_dim), for contexts `factor` times as long as those a model was trained on
      "linear"  divided by the factor: positions are interpolated;
      "ntk"     with a base so much larger that the slowest pair is divided by the factor and the fastest stays;
      "yarn"    pair by pair: those that turn more than 32 times within `trained` tokens stay, those that turn less than once are divided, a linear
                ramp between; and the columns are multiplied by 0.1 ln(factor) + 1."""
    half, base, factor = rotary_dim // 2, float(base), float(factor)
    if rotary_dim < 2 or rotary_dim % 2 or not (math.isfinite(base) and base > 1) or not (math.isfinite(factor) and factor >= 1):
        raise ValueError("rotary_dim must be even, base above 1 and factor at least 1")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', not {scaling!r}")
    if scaling is None and factor != 1:
        raise ValueError("a factor needs a scaling")
    if scaling == "ntk" and half > 1:
        base *= factor ** (half / (half - 1))
    f = [base ** (-i / half) for i in range(half)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling != "yarn":
        return f, 1.0
    if trained < 1:
        raise ValueError("'yarn' needs the tokens that the model was trained on")
    pair = lambda turns: half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)   # noqa: E731
    low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rotary_dim - 1)
    ramp = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(half)]
    return [x / factor * r + x * (1 - r) for x, r in zip(f, ramp)], 0.1 * math.log(factor) + 1


def _rows(t, name, dtype, dim):
    """Strides (batch, head, token) of [batch, heads, tokens, dim] or [tokens, heads, dim], 0 where there is one."""
    if t.dim() not in (3, 4) or t.shape[-1] != dim:
        raise ValueError(f"{name} must be [batch, heads, tokens, {dim}] or [tokens, heads, {dim}]")
    if t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.stride(-1) != 1 or any(n > 1 and (s < 0 or s % 8) for n, s in zip(t.shape[:-1], t.stride()[:-1])) or t.data_ptr() % 16:
        raise ValueError(f"{name} must have contiguous rows that begin at multiples of 16 bytes")
    s = [x if n > 1 else 0 for n, x in zip(t.shape, t.stride())]
    return (s[0], s[1], s[2]) if t.dim() == 4 else (0, s[1], s[0])


class Rotary:
    """Rotary positions of rows of `dim` (64 or 128) columns, the first `rotary_dim` of which turn (0: all; a multiple of 16).

    `interleaved`: columns 2 i and 2 i + 1 are a pair, else i and i + rotary_dim / 2.  `base`, `scaling`, `factor`, `trained`: see frequencies().
    `radians`: rotary_dim / 2 frequencies of the caller's in their place, radians per position; `scale`: what turned columns are multiplied by,
    in the place of what the scaling says.  The angles of any 32-bit position are exact to 2^-26 of a turn."""

    def __init__(self, dim, rotary_dim=0, base=10000.0, interleaved=False, scaling=None, factor=1.0, trained=0, dtype="fp16", radians=None, scale=None,
                 device=None):
        self.lib = _lib.load()
        self.dim, self.rotary_dim, self.interleaved = int(dim), int(rotary_dim) or int(dim), bool(interleaved)
        if self.dim not in (64, 128):
            raise ValueError("dim must be 64 or 128")
        if self.rotary_dim % 16 or not 16 <= self.rotary_dim <= self.dim:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to {self.dim}")
        self.dtype_code = DTYPE_CODE[dtype]
        self.torch_dtype = TORCH_DTYPE[self.dtype_code]
        if radians is None:
            radians, said = frequencies(self.rotary_dim, base, scaling, factor, trained)
        elif scaling is not None:
            raise ValueError("frequencies of the caller's are not scaled")
        else:
            radians, said = [float(x) for x in radians], 1.0
        if len(radians) != self.rotary_dim // 2 or not all(math.isfinite(x) for x in radians):
            raise ValueError(f"radians must be {self.rotary_dim // 2} finite numbers")
        self.scale = said if scale is None else float(scale)
        if not (math.isfinite(self.scale) and self.scale > 0 and math.isfinite(ctypes.c_float(self.scale).value) and ctypes.c_float(self.scale).value > 0):
            raise ValueError("scale must be a positive number")
        self.radians = radians
        n = len(radians)
        made = (ctypes.c_uint64 * n)()
        check(self.lib.ringattn_rotary_turns((ctypes.c_double * n)(*radians), n, made), "ringattn_rotary_turns")
        turns = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in made], dtype=torch.int64)
        if device is None:
            device = f"cuda:{torch.cuda.current_device()}" if torch.cuda.is_available() else "cpu"
        self._turns = turns.to(device)
        self._params = [RingattnRotary(self.rotary_dim, int(self.interleaved), back, self.scale, self.turns.data_ptr()) for back in (0, 1)]
        self.address = ctypes.addressof(self._params[0])   # for calls that are made in native code
        calls = _lib.load_calls()
        self._native = None
        if calls and self.turns.is_cuda:
            self._native = calls.Turn(self.lib.addresses["ringattn_rotary_apply"], self.address, ctypes.addressof(self._params[1]), self.dim, self.dtype_code,
                                      self.turns.device.index, self.torch_dtype)

    turns = property(lambda self: self._turns)   # (its address is the structs')

    def params(self, inverse):
        """struct ringattn_rotary."""
        return self._params[1 if inverse else 0]

    def check(self, dim, dtype):
        if dim != self.dim or dtype != self.torch_dtype:
            raise ValueError(f"the rotary is for rows of {self.dim} columns of {self.torch_dtype}")
        if not self.turns.is_cuda:
            raise ValueError("the rotary's frequencies must be on a device")

    def apply(self, q, k=None, positions=None, q_out=None, k_out=None, inverse=False, stream=None):
        """q, k: [batch, heads, tokens, dim] or both [tokens, heads, dim], of any strides that keep a row together.  `positions`: int32 [tokens] or
        [batch, tokens], of any sign; None: a token's number.  q_out, k_out: the tensor itself for in place; neither
        has rows of the other tensor, between whose rows it may lie.  `inverse`: turned back -- of
        gradients by the outputs the gradients by the inputs.  Returns (q_out, k_out), k_out None without k.  Autograd does not see the call: what it
        returns has no history, also where q and k require gradients, and tensors that it writes count no new version."""
        if q_out is not None and (k is None or k_out is not None) and self._native:
            rc = self._native(q, k, positions, q_out, k_out, inverse, stream)
            if rc is not None:
                check(rc, "ringattn_rotary_apply")
                return q_out, k_out
        given = [(q, "q", q_out)] + ([(k, "k", k_out)] if k is not None else [])
        if k is None and k_out is not None:
            raise ValueError("k_out without k")
        made, outs = [], []
        for t, name, out in given:
            strides = _rows(t, name, self.torch_dtype, self.dim)
            if out is None:
                out = self._like(t, stream)
            if out.shape != t.shape:
                raise ValueError(f"{name}_out must have shape {tuple(t.shape)}")
            out_strides = _rows(out, f"{name}_out", self.torch_dtype, self.dim)
            if t.shape[1]:   # (a tensor of no heads has no rows; the other one's turn all the same)
                made.append(RingattnRows(t.data_ptr(), out.data_ptr(), t.shape[1], *strides, *out_strides))
            outs.append(out)
        four = q.dim() == 4
        batch, tokens = (q.shape[0], q.shape[2]) if four else (1, q.shape[0])
        if k is not None and (k.dim() != q.dim() or ((k.shape[0], k.shape[2]) if four else (1, k.shape[0])) != (batch, tokens)):
            raise ValueError("q and k must have the same batch and as many tokens")
        if tokens > MAX_POSITIONS or batch > 65535 or sum(t.shape[1] for t, _, _ in given) > 65535:
            raise ValueError("a call takes up to 2^30 tokens, 65535 heads of q and k together, and 65535 batches")
        stride = 0
        if positions is not None:
            shape = (batch, tokens) if positions.dim() == 2 and four else (tokens,)
            _check_tensors((positions, "positions", torch.int32, shape))
            stride = tokens if len(shape) == 2 else 0
        self.check(self.dim, self.torch_dtype)
        for t in outs + [k, positions, self.turns]:
            if t is not None and t.device != q.device:
                raise ValueError("the tensors of a call must be on one device")
        if batch and tokens and made:
            self._call(q.device, stream, made, batch, tokens, positions.data_ptr() if positions is not None else None, stride, inverse)
        return outs[0], outs[1] if len(outs) > 1 else None

    def _call(self, device, stream, rows, batch, tokens, positions, stride, inverse):
        """A launch on the tensors' own device, whichever is the current one."""
        if device.index != torch.cuda.current_device():
            with torch.cuda.device(device):
                return self._call(device, stream, rows, batch, tokens, positions, stride, inverse)
        check(self.lib.ringattn_rotary_apply(ctypes.byref(self.params(inverse)), self.dim, self.dtype_code, (RingattnRows * len(rows))(*rows), len(rows),
                                             batch, tokens, positions, stride, _stream_ptr(stream)), "ringattn_rotary_apply")

    @staticmethod
    def _like(t, stream):
        if stream is None:
            return torch.empty_like(t)
        with torch.cuda.stream(stream):
            return torch.empty_like(t)
