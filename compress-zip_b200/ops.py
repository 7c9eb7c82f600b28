"""Operators on device tensors: ctypes binding of include/czg_ops.h (libczg.so).

The int8 product with scales for each token and channel (``quantize_rows``,
``linear_i8``), and a key/value cache held in 4 bits (``KV4Cache``) with attention
over it and eviction from it by accumulated attention weight.

Every call queues its work on the current stream of its tensors' device and returns
without waiting; nothing is allocated but the results, a workspace and, in ``linear_i8``, a
copy of an x whose leading dimensions cannot be viewed as rows, all by torch.
Shapes and types are checked here (ValueError) and again by the library (CzgError).
What only the device can see -- slots and lengths out of range -- sets bits that
``KV4Cache.check`` reads.  No fallback: tensors must be on a CUDA device.

There is no backward pass.  ``linear_i8`` and ``KV4Cache.attend`` refuse (ValueError) an
input that requires a gradient while torch records them: call them under
``torch.no_grad()``, or detach the input.  ``quantize_rows`` and ``KV4Cache.append`` store codes,
which have no gradient.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import engine as _engine
from .engine import CZG_OK, CzgError

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT32 = torch.int32

# The exported symbols of include/czg_ops.h, checked by the CPU test suite.
EXPORTS = ["czg_ops_last_error", "czg_ops_check", "czg_quantize_rows", "czg_linear_i8", "czg_linear_i8_workspace",
           "czg_linear_i8_dynamic_workspace", "czg_linear_i8_dynamic", "czg_kv4_append", "czg_kv4_read", "czg_kv4_attend_workspace",
           "czg_kv4_attend", "czg_kv4_evict"]

STATUS_BITS = {1: "a slot beyond the cache", 2: "a length or entry outside its range",
               4: "a slot named twice in one call"}


class _KV4(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("scales", C.c_void_p), ("weights", C.c_void_p),
                ("status", C.c_void_p), ("n_slots", C.c_int32), ("n_heads", C.c_int32),
                ("capacity", C.c_int32), ("head_dim", C.c_int32)]


_bound = None


def lib() -> C.CDLL:
    global _bound
    if _bound is None:
        L = _engine.lib()
        P, I, L64, U64 = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64
        K = C.POINTER(_KV4)
        sig = {
            "czg_quantize_rows": [P, I, L64, L64, L64, P, L64, P, P],
            "czg_linear_i8": [P, L64, P, P, L64, P, P, L64, L64, L64, P, I, L64, P],
            "czg_linear_i8_dynamic": [P, I, L64, P, L64, P, P, L64, L64, L64, P, I, L64, P, U64, P],
            "czg_kv4_append": [K, P, L64, L64, L64, P, L64, L64, L64, I, P, P, I, I, P],
            "czg_kv4_read": [K, P, P, I, I, P, P, I, P],
            "czg_kv4_attend": [K, P, L64, L64, L64, I, P, P, I, I, I, I, C.c_float, P, L64, L64, L64, P, U64, P],
            "czg_kv4_evict": [K, P, P, I, I, I, I, P, P, P],
        }
        for name, args in sig.items():
            fn = getattr(L, name)
            fn.argtypes, fn.restype = args, C.c_int
        L.czg_linear_i8_workspace.argtypes, L.czg_linear_i8_workspace.restype = [L64, L64], U64
        L.czg_linear_i8_dynamic_workspace.argtypes, L.czg_linear_i8_dynamic_workspace.restype = [L64, L64, L64], U64
        L.czg_kv4_attend_workspace.argtypes, L.czg_kv4_attend_workspace.restype = [K, I, I, I, I], U64
        L.czg_ops_check.argtypes, L.czg_ops_check.restype = [], C.c_int
        L.czg_ops_last_error.argtypes, L.czg_ops_last_error.restype = [], C.c_char_p
        _bound = L
    return _bound


def _raise(status: int) -> None:
    raise CzgError(status, lib().czg_ops_last_error().decode())


def _dtype(t: torch.Tensor, what: str) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _same_device(dev: torch.device, **tensors) -> None:
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {dev}")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the others on {dev}")


_current_device = torch.cuda.current_device
_recording = torch.is_grad_enabled


def _no_gradient(what: str) -> None:
    raise ValueError(f"{what} requires a gradient, which this operator does not have: use torch.no_grad() or detach it")


# the handle of a device's current stream, without a Stream object around it where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) on the current stream of dev, with dev current."""
    if dev.index == _current_device():
        st = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _raw_stream(dev.index))
    if st != CZG_OK:
        _raise(st)


def check(device=None) -> None:
    """Wait for the device and raise CzgError if a kernel of an operator gave up a bounded wait."""
    with torch.cuda.device(device):
        st = lib().czg_ops_check()
    if st != CZG_OK:
        _raise(st)


# ---- int8 product --------------------------------------------------------------


class QRows:
    """Rows of int8 codes [n, k] (beginning on 16-byte boundaries) and their float32 scales [n]."""
    __slots__ = ("codes", "scales", "n", "k", "ld", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.int8 or codes.dim() != 2 or (codes.stride(1) != 1 and codes.shape[1] > 1):
            raise ValueError("codes must be a 2-D int8 tensor with adjacent columns")
        self.n, self.k = codes.shape
        if scales.dtype != torch.float32 or scales.shape != (self.n,) or (self.n > 1 and scales.stride(0) != 1):
            raise ValueError("scales must be a contiguous float32 vector, one scale a row")
        # a single row may have any stride: the library's rule is met with the row's own length
        self.ld = codes.stride(0) if self.n > 1 else (self.k + 15) // 16 * 16
        if codes.data_ptr() % 16 or self.ld % 16:
            raise ValueError("rows of codes must begin on 16-byte boundaries (quantize_rows lays them out so)")
        if scales.device != codes.device:
            raise ValueError(f"scales are on {scales.device}, codes on {codes.device}")
        self.codes, self.scales, self.device = codes, scales, codes.device


def _rows(x: torch.Tensor, what: str) -> None:
    if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError(f"{what} must be 2-D with adjacent columns")


def quantize_rows(x: torch.Tensor) -> QRows:
    """Rows of x as int8 codes with one scale each: scale = max |x| / 127, code =
    round-half-even(127 x / max |x|).  For activations, one scale a token; for a weight
    [n, k], one scale an output channel."""
    code = _dtype(x, "x")
    _rows(x, "x")
    _same_device(x.device)
    m, k = x.shape
    ld = max((k + 15) // 16 * 16, 16)
    codes = torch.empty((m, ld), dtype=torch.int8, device=x.device)
    scales = torch.empty(m, dtype=torch.float32, device=x.device)
    if m and k:
        _call(x.device, lib().czg_quantize_rows, x.data_ptr(), code, x.stride(0), m, k, codes.data_ptr(), ld,
              scales.data_ptr())
    elif m:
        scales.zero_()
    return QRows(codes[:, :k], scales)


def linear_i8(x, w: QRows, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ w.T from int8 codes: exact int32 sums, times the token's and the channel's
    scale, plus ``bias`` (float32 [n]), rounded once to ``out_dtype``.

    x: a QRows, or a float tensor [..., k] whose rows are quantised in the same call.
    out_dtype defaults to x's type (bfloat16 for a QRows); ``out``, if given, has
    adjacent columns and is returned."""
    n, k, dev = w.n, w.k, w.device
    quantised = isinstance(x, QRows)
    if quantised:
        m, width, x2, lead = x.n, x.k, x.codes, None
    else:
        code = _dtype(x, "x")
        shape = x.shape
        if len(shape) == 2:
            x2, lead = x, None
        elif len(shape) == 0:
            raise ValueError("x must have a last dimension of k")
        else:
            lead = shape[:-1]
            x2 = x.reshape(lead.numel(), shape[-1])
        m, width = x2.shape
        if x2.stride(1) != 1 and width > 1:
            raise ValueError("x must have adjacent columns")
    if width != k:
        raise ValueError(f"x has rows of {width}, w of {k}")
    if x2.device != dev:
        raise ValueError(f"x is on {x2.device}, w on {dev}")
    if out is None:
        kind = out_dtype if out_dtype is not None else torch.bfloat16 if quantised else x.dtype
        out_code = DTYPES.get(kind)
        if out_code is None:
            raise ValueError(f"out_dtype must be float32, bfloat16 or float16, not {kind}")
    else:
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"out is of {out.dtype}, out_dtype {out_dtype}")
        out_code = _dtype(out, "out")
        if out.shape != ((m, n) if lead is None else (*lead, n)):
            raise ValueError(f"out must have shape {(*(lead or (m,)), n)}, not {tuple(out.shape)}")
        if out.device != dev:
            raise ValueError(f"out is on {out.device}, w on {dev}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or (n > 1 and bias.stride(0) != 1)
                             or bias.device != dev):
        raise ValueError(f"bias must be a contiguous float32 vector of {n} on {dev}")
    if _recording() and (x2.requires_grad or w.scales.requires_grad or (bias is not None and bias.requires_grad)
                         or (quantised and x.scales.requires_grad) or (out is not None and out.requires_grad)):
        _no_gradient("an input or out")
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {dev}")
    if out is None:
        out2 = x2.new_empty((m, n)) if x2.dtype is kind else x2.new_empty((m, n), dtype=kind)
        out = out2 if lead is None else out2.view(*lead, n)
    else:
        out2 = out if lead is None else out.view(m, n)
        _rows(out2, "out")
    if m == 0 or n == 0:
        return out
    if k == 0:
        out2.copy_(torch.zeros((), device=dev) if bias is None else bias)
        return out
    L = _bound or lib()
    bias_ptr = 0 if bias is None else bias.data_ptr()
    ldo = out2.stride(0) if m > 1 else n
    if quantised:
        _call(dev, L.czg_linear_i8, x2.data_ptr(), x.ld, x.scales.data_ptr(), w.codes.data_ptr(), w.ld, w.scales.data_ptr(),
              bias_ptr, m, n, k, out2.data_ptr(), out_code, ldo)
    else:
        need = L.czg_linear_i8_dynamic_workspace(m, n, k)
        ws = w.codes.new_empty(need) if need else None
        _call(dev, L.czg_linear_i8_dynamic, x2.data_ptr(), code, x2.stride(0) if m > 1 else k, w.codes.data_ptr(), w.ld,
              w.scales.data_ptr(), bias_ptr, m, n, k, out2.data_ptr(), out_code, ldo, ws.data_ptr() if need else 0, need)
    return out


# ---- key/value cache in 4 bits ----------------------------------------------------


class KV4Cache:
    """A key/value cache of 4-bit entries over the caller's tensors.

    k, v     uint8 [n_slots, n_heads, capacity, head_dim / 2]
    scales   bfloat16 [n_slots, n_heads, capacity, 4] (k step, k lo, v step, v lo)
    weights  None, or float32 [n_slots, n_heads, capacity]: sums of attention weights, grown by
             ``attend`` and ranked by ``evict``

    ``KV4Cache.empty`` allocates them.  Calls name sequences by ``slots`` (int32 [b]; a
    negative one is a padded place of the batch) and ``lengths`` (int32 [b], entries of
    each sequence, the rows of the call among them), both on the device.  Slots of a
    call that writes (append, evict, attend with weights) are distinct."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor, weights: Optional[torch.Tensor] = None):
        if k.dim() != 4 or k.dtype != torch.uint8 or v.shape != k.shape or v.dtype != torch.uint8:
            raise ValueError("k and v must be uint8 tensors [n_slots, n_heads, capacity, head_dim / 2]")
        if k.shape[3] not in (32, 64):
            raise ValueError(f"head_dim must be 64 or 128, not {2 * k.shape[3]}")
        if scales.shape != (*k.shape[:3], 4) or scales.dtype != torch.bfloat16:
            raise ValueError("scales must be a bfloat16 tensor [n_slots, n_heads, capacity, 4]")
        if weights is not None and (weights.shape != k.shape[:3] or weights.dtype != torch.float32):
            raise ValueError("weights must be a float32 tensor [n_slots, n_heads, capacity]")
        for name, t in (("k", k), ("v", v), ("scales", scales), ("weights", weights)):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError(f"{name} must be contiguous and begin on a 16-byte boundary")
        if k.numel() == 0:
            raise ValueError("a cache has at least one slot, head and entry")
        _same_device(k.device, v=v, scales=scales, weights=weights)
        self.k, self.v, self.scales, self.weights = k, v, scales, weights
        self.device = k.device
        self.n_slots, self.n_heads, self.capacity = k.shape[:3]
        self.head_dim = 2 * k.shape[3]
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._c = _KV4(k.data_ptr(), v.data_ptr(), scales.data_ptr(), 0 if weights is None else weights.data_ptr(),
                       self.status.data_ptr(), self.n_slots, self.n_heads, self.capacity, self.head_dim)
        self._needs = {}   # workspace bytes by a call's sizes
        self._ref, self._lib, self._index = C.byref(self._c), lib(), k.get_device()

    @classmethod
    def empty(cls, n_slots: int, n_heads: int, capacity: int, head_dim: int, track_weights: bool = False,
              device="cuda") -> "KV4Cache":
        """A cache of its own tensors: entries are zeros, no sequence holds any."""
        shape = (n_slots, n_heads, capacity)
        kv = [torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*kv, torch.zeros(*shape, 4, dtype=torch.bfloat16, device=device),
                   torch.zeros(shape, dtype=torch.float32, device=device) if track_weights else None)

    def _sequences(self, slots: torch.Tensor, counts: torch.Tensor, name: str) -> int:
        shape = slots.shape
        if (slots.dtype is not _INT32 or counts.dtype is not _INT32 or len(shape) != 1 or counts.shape != shape
                or not slots.is_contiguous() or not counts.is_contiguous()):
            raise ValueError(f"slots and {name} must be contiguous int32 vectors, one number a sequence")
        if slots.get_device() != self._index or counts.get_device() != self._index:
            raise ValueError(f"slots and {name} are on {slots.device} and {counts.device}, the cache on {self.device}")
        return shape[0]

    def _call(self, fn, *args) -> None:
        if self._index == _current_device():
            st = fn(self._ref, *args, _raw_stream(self._index))
        else:
            with torch.cuda.device(self._index):
                st = fn(self._ref, *args, _raw_stream(self._index))
        if st != CZG_OK:
            _raise(st)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, lengths: torch.Tensor) -> None:
        """Quantise rows k, v [b, t, n_heads, head_dim] into entries lengths - t .. lengths - 1
        of their slots; rows before entry 0 are padding.  Their weights become 0."""
        b = self._sequences(slots, lengths, "lengths")
        shape, code = k.shape, DTYPES.get(k.dtype)
        if len(shape) != 4 or shape[0] != b or shape[2] != self.n_heads or shape[3] != self.head_dim or v.shape != shape:
            raise ValueError(f"k and v must be [{b}, t, {self.n_heads}, {self.head_dim}]")
        if code is None or v.dtype is not k.dtype:
            raise ValueError(f"k and v must both be float32, bfloat16 or float16, not {k.dtype} and {v.dtype}")
        ks, vs = k.stride(), v.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("the last dimension of k and v must be adjacent")
        if k.get_device() != self._index or v.get_device() != self._index:
            raise ValueError(f"k and v are on {k.device} and {v.device}, the cache on {self.device}")
        if b and shape[1]:
            self._call(self._lib.czg_kv4_append, k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], code,
                       slots.data_ptr(), lengths.data_ptr(), b, shape[1])

    def read(self, slots: torch.Tensor, starts: torch.Tensor, count: int, dtype: torch.dtype = torch.bfloat16):
        """Entries starts .. starts + count - 1 of each slot as values: (k, v), each
        [b, count, n_heads, head_dim]; 0 for places outside the slot."""
        b = self._sequences(slots, starts, "starts")
        code = DTYPES.get(dtype)
        if code is None:
            raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
        if count < 0:
            raise ValueError("count must not be negative")
        k = self.k.new_empty((b, count, self.n_heads, self.head_dim), dtype=dtype)
        v = torch.empty_like(k)
        if b and count:
            self._call(self._lib.czg_kv4_read, slots.data_ptr(), starts.data_ptr(), b, count, k.data_ptr(), v.data_ptr(), code)
        return k, v

    def attend(self, q: torch.Tensor, slots: torch.Tensor, lengths: torch.Tensor, max_len: Optional[int] = None,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [b, t, hq, head_dim] (bfloat16 or float16) over the sequences'
        entries, row i seeing the first lengths - (t - 1 - i); rows that see none give 0.
        hq is a multiple of n_heads.  max_len (default: the capacity) bounds the lengths,
        scale defaults to head_dim ** -0.5.  With weights, each entry's grows by its
        probabilities, summed over the rows and query heads of its key head, and the workspace
        takes 4 bytes a row, query head and entry of max_len: give it where the capacity is far
        above the lengths.  A row's last bits may differ between calls of other t."""
        b = self._sequences(slots, lengths, "lengths")
        shape, qs = q.shape, q.stride()
        if len(shape) != 4 or shape[0] != b or shape[3] != self.head_dim or shape[2] % self.n_heads:
            raise ValueError(f"q must be [{b}, t, a multiple of {self.n_heads}, {self.head_dim}]")
        _, t, hq, _ = shape
        if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
            raise ValueError(f"q must be bfloat16 or float16, not {q.dtype}")
        if qs[3] != 1:
            raise ValueError("the last dimension of q must be adjacent")
        if q.get_device() != self._index:
            raise ValueError(f"q is on {q.device}, the cache on {self.device}")
        if _recording() and (q.requires_grad or (out is not None and out.requires_grad)):
            _no_gradient("q or out")
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != shape or out.dtype is not q.dtype or out.get_device() != self._index:
            raise ValueError("out must have q's shape, type and device")
        os = out.stride()
        if os[3] != 1:
            raise ValueError("the last dimension of out must be adjacent")
        if not (b and t and hq):
            return out
        n = self.capacity if max_len is None else min(max_len, self.capacity)
        need = self._needs.get((b, t, hq, n))
        if need is None:
            if len(self._needs) > 4096:
                self._needs.clear()
            need = self._needs[b, t, hq, n] = self._lib.czg_kv4_attend_workspace(self._ref, b, t, hq, n)
        ws = self.k.new_empty(need) if need else None
        self._call(self._lib.czg_kv4_attend, q.data_ptr(), qs[0], qs[1], qs[2], DTYPES[q.dtype], slots.data_ptr(),
                   lengths.data_ptr(), b, t, hq, n, self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(),
                   os[0], os[1], os[2], ws.data_ptr() if need else 0, need)
        return out

    def evict(self, slots: torch.Tensor, lengths: torch.Tensor, budget: int, recent: int = 0,
              max_len: Optional[int] = None):
        """Cut sequences longer than ``budget`` to it: of each head the last ``recent``
        entries stay and the budget - recent others with the largest weights (ties: the
        first), in order, moved to the front of the slot.  Returns (kept, new lengths):
        int32 [b, n_heads, budget] former places (-1 behind a shorter end) and int32 [b]."""
        b = self._sequences(slots, lengths, "lengths")
        if self.weights is None:
            raise ValueError("the cache keeps no weights to rank entries by")
        if not 1 <= budget < 1 << 31 or not 0 <= recent <= budget:
            raise ValueError("1 <= budget < 2^31 and 0 <= recent <= budget are needed")
        kept = slots.new_empty((b, self.n_heads, budget))
        new = torch.empty_like(slots)
        if b:
            self._call(self._lib.czg_kv4_evict, slots.data_ptr(), lengths.data_ptr(), b,
                       self.capacity if max_len is None else min(max_len, self.capacity), budget, recent, kept.data_ptr(), new.data_ptr())
        return kept, new

    def check(self) -> None:
        """Wait for the device and raise CzgError if a call met slots or lengths out of
        range, or a kernel gave up a bounded wait; the bits are cleared."""
        check(self.device)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise CzgError(1, ", ".join(text for bit, text in STATUS_BITS.items() if bits & bit))
