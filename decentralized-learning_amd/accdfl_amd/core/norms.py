"""Norms over many tensors, and what is bounded by them (include/dlagg.h, csrc/bound.hip).

A training step clips its gradient by the global norm over every parameter; a round bounds what one peer may move
the average by.  The reference does neither (its trainer steps at accdfl/core/model_trainer.py:18-121, its
aggregator averages whatever arrived, accdfl/core/gradient_aggregation/fedavg.py:20-25); both read every element
of a model once before the first element can be written, which is what these operators are built around::

    global_norm(tensors)                         one number over a list of tensors
    clip_global_norm(tensors, max_norm)          the list scaled to at most that norm, into new or given tensors
    clip_global_norm_(tensors, max_norm)         the same in place
    clip_grad_norm_(parameters, max_norm)        the same on parameters' gradients
    update_norms(models, center)                 how far each model lies from a centre
    wsum_bounded(peers, weights, center, R)      center + sum_k w_k min(1, R / n_k) (peer_k - center), flat peers
    wsum_bounded_multi(...)                      the same over the tensors of whole models

Tensors are float32 / bfloat16 / float16 / float64, mixed freely within a list, on one HIP device, empty ones
included.  Dense tensors are read where they are whatever the order of their axes and wherever they start; others
(a slice with gaps, an expanded tensor) are copied first.  Outputs that overlap each other, themselves or another tensor
are refused whatever their strides.  Norms and products are carried in 64 bits, averages in 64 (32 for the 16-bit
types, where they hold every term), and rounded once; a norm beyond float32's range is returned as infinity by
float32, but is finite for what is scaled by it.  Results are on the device and nothing synchronises; nothing here is
differentiable.  Work is enqueued on ``stream`` or the current stream of the tensors' device (tensors of another
stream are the caller's to keep until it has passed), workspaces come from torch's caching allocator for each call, and
launches take their tables by value (those of large rounds from a slot of page-locked memory that the call owns until
the GPU has read it; under capture by value too): calls on several streams or threads do not meet, and a call captured
into a graph replays.
"""
from __future__ import annotations

import bisect
import contextlib
import ctypes
import itertools
import math
from typing import Dict, Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch
from torch import nn

from accdfl_amd import _lib
from accdfl_amd.core import wsum as _wsum

Tensors = Union[nn.Module, torch.Tensor, Iterable[torch.Tensor]]

CLIP_EPS = 1e-6  # the norm is raised by this before the bound is divided by it (torch.nn.utils.clip_grad_norm_)
MAX_PEERS = 2048  # include/dlagg.h dla_peer_workspace


# ------------------------------------------------------------------------------------------- tables of tensors
class _Tables:
    """The walk extension's DenseTables (csrc/walk.cpp: what a call hands to the library, and the calls) in Python,
    for when the extension is absent: ``n`` tensors on HIP device ``device``; dtype codes, counts, the addresses of
    the first lists, and those of the other lists tensor-major."""

    def __init__(self, device: int, lists: List[List[torch.Tensor]], lead: int, written: Sequence[torch.Tensor]):
        n, rest = len(lists[0]), lists[lead:]
        address = lambda t: t.data_ptr() if t.numel() else 0  # noqa: E731
        self.n = n
        self.device = device
        self.written = [t for t in written if not t.is_inference()]
        self.wide = any(t.dtype == torch.float64 for t in lists[0])
        self.codes = (ctypes.c_int * n)(*[_wsum.dtype_code(t.dtype) for t in lists[0]])
        self.numels = (ctypes.c_int64 * n)(*[t.numel() for t in lists[0]])
        self.lead = [(ctypes.c_void_p * n)(*[address(t) for t in ts]) for ts in lists[:lead]]
        self.rest = (ctypes.c_void_p * (n * len(rest)))(*[address(ts[i]) for i in range(n) for ts in rest])

    def _result(self, size, double: bool):
        return torch.empty(size, dtype=torch.float64 if double else torch.float32, device=self.device)

    def _call(self, name: str, out, *args, written: Sequence[torch.Tensor] = ()):
        rc = getattr(_lib.lib().so, name)(self.n, self.codes, *args)
        if rc >= 0:  # not refused
            torch.autograd.graph.increment_version(written)
        return rc, out

    def norm(self, fn, code, counter, nbytes, stream):
        out, ws = self._result((), self.wide), _workspace(nbytes, self.device)
        return self._call("dla_norm", out, self.lead[0], self.numels, code, 3 * self.wide, out.data_ptr(), counter,
                          ws.data_ptr(), nbytes, stream)

    def clip(self, fn, code, max_norm, eps, counter, nbytes, stream):
        out, ws = self._result((), self.wide), _workspace(nbytes, self.device)
        return self._call("dla_norm_clip", out, self.lead[0], self.lead[1], self.numels, code, max_norm, eps,
                          3 * self.wide, out.data_ptr(), counter, ws.data_ptr(), nbytes, stream, written=self.written)

    def peer_norms(self, fn, n, squared, counters, table, table_bytes, nbytes, stream):
        out, ws = self._result(n, squared or self.wide), _workspace(nbytes, self.device)
        return self._call("dla_peer_norms", out, self.rest, self.lead[0], self.numels, n, out.data_ptr() if squared else 0,
                          3 * self.wide, 0 if squared else out.data_ptr(), counters, table, table_bytes, ws.data_ptr(),
                          nbytes, stream)

    def bounded(self, fn, outs, weights, max_norm, sq, counters, table, table_bytes, nbytes, stream):
        out, ws = self._result(len(weights), self.wide), _workspace(nbytes, self.device)
        return self._call("dla_wsum_bounded", out, self.rest, self.lead[0], self.lead[1], self.numels,
                          _lib._dbl_array(weights), len(weights), max_norm, sq, 3 * self.wide, out.data_ptr(), counters,
                          table, table_bytes, ws.data_ptr(), nbytes, stream, written=self.written)


def _pack(lists: List[List[torch.Tensor]], lead: int, out: int = -1):
    """The tables of lists whose tensors the kernels take as they are (walk.cpp dense_lists), else None.  ``out``: the
    list that the call writes (its tensors' version counters then move on, unless the call is refused)."""
    mod = _lib.walk_module()
    return None if mod is None else mod.dense_lists(lists, lead, out)


def _dense(t: torch.Tensor) -> bool:
    """Every element of the tensor's memory span is one element of the tensor (any order of its axes)."""
    if t.numel() < 2:
        return True
    expect = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _held(t: torch.Tensor) -> bool:
    """The tensor's storage holds every one of its elements (one that was resized under it may not)."""
    if t.numel() == 0:
        return True
    last = t.storage_offset() + sum((size - 1) * stride for size, stride in zip(t.shape, t.stride()))
    return t.untyped_storage().nbytes() >= (last + 1) * t.element_size()


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.stride() == b.stride() or (a.is_contiguous() and b.is_contiguous())


def _check(lists: List[List[torch.Tensor]], names: Sequence[str]) -> torch.device:
    """Raises for lists that no copy makes fit: types, devices, dtypes, counts, sizes."""
    first = lists[0]
    device = None
    for name, ts in zip(names, lists):
        if len(ts) != len(first):
            raise ValueError("%s has %d tensors, %s has %d" % (name, len(ts), names[0], len(first)))
        for i, t in enumerate(ts):
            what = "%s tensor %d" % (name, i)
            if not isinstance(t, torch.Tensor):
                raise TypeError("%s is a %s, not a tensor" % (what, type(t).__name__))
            if t.layout is not torch.strided:
                raise TypeError("%s is %s: only dense (strided) tensors are supported" % (what, t.layout))
            _wsum.dtype_code(t.dtype)
            if device is None:
                device = _wsum.require_device(t.device if t.is_cuda else None)
            if t.device != device:
                raise ValueError("%s is on %s, expected %s" % (what, t.device, device))
            if not _held(t):
                raise ValueError("%s lies outside its storage (%d bytes)" % (what, t.untyped_storage().nbytes()))
            if t.dtype != first[i].dtype or t.shape != first[i].shape:
                raise ValueError("%s is %s %s, %s has %s %s there" % (what, t.dtype, tuple(t.shape), names[0],
                                                                      first[i].dtype, tuple(first[i].shape)))
    return device


# Overlaps of outputs that are not dense: the library checks the memory that it is given, which for them is a copy.
_OVERLAP_WORK = 1_000_000  # candidates NumPy may try for two views whose spans meet; beyond it they count as overlapping


class _Elements:
    """Where the elements of a tensor lie: ``axes`` (stride, size) in elements of ``size`` bytes from ``begin`` on, all
    before ``end``.  NumPy takes it for an array; the memory is not touched."""

    def __init__(self, begin: int, axes: List[Tuple[int, int]], size: int):
        self.begin, self.axes, self.size = begin, axes, size
        self.end = begin + (sum(st * (n - 1) for st, n in axes) + 1) * size
        self.step = math.gcd(*[st for st, _ in axes]) * size

    @classmethod
    def of(cls, t: torch.Tensor) -> "_Elements":
        return cls(t.data_ptr(), [(st, n) for st, n in zip(t.stride(), t.shape) if n != 1], t.element_size())

    def same(self, other: "_Elements") -> bool:
        return self.begin == other.begin and self.axes == other.axes

    @property
    def __array_interface__(self):
        return {"version": 3, "typestr": "|V%d" % self.size, "data": (self.begin, True),
                "shape": tuple(n for _, n in self.axes), "strides": tuple(st * self.size for st, _ in self.axes)}

    def meet(self, other: "_Elements") -> bool:
        """Is there a byte that both have?"""
        if self.end <= other.begin or other.end <= self.begin:
            return False
        step = math.gcd(self.step, other.step)
        # both are periodic in `step` bytes: side by side in each period (columns of one matrix) they do not meet
        if step and self.size <= (other.begin - self.begin) % step <= step - other.size:
            return False
        try:
            return np.shares_memory(np.asarray(self), np.asarray(other), max_work=_OVERLAP_WORK)
        except np.exceptions.TooHardError:
            return True

    def meets_itself(self) -> bool:
        """Do two elements share memory?  Axis by axis, the smallest step first: what the axes so far reach, moved by any
        number of steps of the next one that stays within that reach, may not meet itself."""
        reach, inner = 0, []
        for stride, n in sorted(self.axes):
            if stride == 0:
                return True
            for k in range(1, min(n - 1, reach // stride) + 1):
                if _Elements(self.begin, inner, self.size).meet(_Elements(self.begin + k * stride * self.size, inner, self.size)):
                    return True
            inner.append((stride, n))
            reach += (n - 1) * stride
        return False


def _span(t: torch.Tensor) -> Tuple[int, int]:
    if t.is_contiguous():
        begin = t.data_ptr()
        return begin, begin + t.numel() * t.element_size()
    place = _Elements.of(t)
    return place.begin, place.end


def _refuse_overlaps(lists: List[List[torch.Tensor]], names: Sequence[str], out: int) -> None:
    """The library's rule for any strides: no element of lists[out] is written twice, and none is an element of another
    tensor, but for the tensor in its own place of another list."""
    own = [_Elements.of(t) if t.numel() else None for t in lists[out]]
    outs = sorted(((p, i) for i, p in enumerate(own) if p), key=lambda o: o[0].begin)
    for p, i in outs:
        if p.meets_itself():
            raise ValueError("%s tensor %d: an output has elements that share memory" % (names[out], i))
    begins = [p.begin for p, _ in outs]
    reach = list(itertools.accumulate((p.end for p, _ in outs), max))  # of outs[:j + 1]

    def refuse(l, i, t, begin, end, stop):
        """Raises if tensor i of list l meets one of outs[:stop]."""
        place = None
        j = min(stop, bisect.bisect_left(begins, end)) - 1
        while j >= 0 and reach[j] > begin:
            if outs[j][0].end > begin:
                if place is None:
                    place = _Elements.of(t)
                    if l != out and place.same(own[i]):
                        return
                if outs[j][0].meet(place):
                    raise _lib.DlaggError("%s tensor %d overlaps %s tensor %d" % (names[l], i, names[out], outs[j][1]))
            j -= 1

    for q, (p, i) in enumerate(outs):
        refuse(out, i, lists[out][i], p.begin, p.end, q)
    for l, ts in enumerate(lists):
        for i, t in enumerate(ts):
            if l != out and t is not lists[out][i] and own[i]:
                refuse(l, i, t, *_span(t), len(outs))


def _pack_checked(lists: List[List[torch.Tensor]], names: Sequence[str], lead: int, out: int = -1):
    """(tables, copies to write back) for any lists that _check accepts: tensors that are not dense, or whose
    element order differs within their place, are replaced by contiguous copies; lists[out]'s replacements are
    returned as (tensor, its copy) to be copied back after the call.  Outputs that overlap are refused."""
    device = _check(lists, names)
    lists = [list(ts) for ts in lists]
    back = []
    if out >= 0:
        _refuse_overlaps(lists, names, out)
    for i in range(len(lists[0])):
        place = [ts[i] for ts in lists]
        if all(_dense(t) and not t.is_neg() and _same_order(t, place[0]) for t in place):
            continue
        for ts, t in zip(lists, place):
            ts[i] = t.detach().resolve_neg().contiguous()
        if out >= 0:
            if lists[out][i].data_ptr() != place[out].data_ptr():
                lists[out][i] = torch.empty(place[out].shape, dtype=place[out].dtype, device=device)
                back.append((place[out], lists[out][i]))
    tables = _pack(lists, lead, out)
    if tables is None:
        tables = _Tables(device.index, lists, lead, lists[out] if out >= 0 else ())
    return tables, back, lists  # the lists keep the copies alive until the call is enqueued


def _write_back(pairs) -> None:
    with torch.no_grad():
        for t, copy in pairs:
            t.copy_(copy)


def _tensors_of(what: Tensors) -> List[torch.Tensor]:
    if isinstance(what, torch.Tensor):
        return [what]
    if isinstance(what, nn.Module):
        return list(what.parameters())
    return what if type(what) is list else list(what)


def _norm_code(norm_type: float) -> int:
    code = _lib.NORM_CODES.get(float(norm_type))
    if code is None:
        raise ValueError("norm_type must be 1, 2 or inf, got %r" % (norm_type,))
    return code


def _bound(max_norm: float) -> float:
    r = float(max_norm)
    if not r >= 0.0:
        raise ValueError("max_norm must be >= 0, got %r" % (max_norm,))
    return r


@contextlib.contextmanager
def _placed(device: torch.device, stream: torch.cuda.Stream):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


def _place(device: torch.device, stream: Optional[torch.cuda.Stream]):
    """The device, and the stream when one is given, made current for a call: allocations and launches of the
    call belong to them."""
    if stream is None:
        if device.index == torch.cuda.current_device():
            return contextlib.nullcontext()
        return torch.cuda.device(device)
    if stream.device != device:
        raise ValueError("stream is on %s, the tensors are on %s" % (stream.device, device))
    return _placed(device, stream)


def _raw_stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)


def _device_of(tensors: List[torch.Tensor], stream: Optional[torch.cuda.Stream]) -> torch.device:
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            return t.device
    return stream.device if stream is not None else _wsum.require_device(None)


def _workspace(nbytes: int, device: int) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


# Counters of the library's last-workgroup joins (include/dlagg.h): zero before and after every call, so the calls of
# one stream share one set — (device, stream handle) -> tensor.  A captured call takes none (a replay may run on
# another stream): it joins in a launch of its own.  Nor does hipStreamPerThread, one handle for many streams.
_counters: Dict[Tuple[int, int], torch.Tensor] = {}
_STREAM_PER_THREAD = 2


def _counter(device: int, raw_stream: int) -> int:
    """The address of the stream's counters, or 0."""
    if raw_stream == _STREAM_PER_THREAD or torch.cuda.is_current_stream_capturing():
        return 0
    t = _counters.get((device, raw_stream))
    if t is None:
        t = _counters.setdefault((device, raw_stream), torch.zeros(_lib.COUNTER_BYTES // 4, dtype=torch.int32,
                                                                   device=device))
    return t.data_ptr()


def _refuse_nonfinite(norm: torch.Tensor, norm_type: float) -> None:
    if not bool(torch.isfinite(norm)):
        raise RuntimeError("the total norm of order %s is not finite, so it cannot be clipped by; pass "
                           "error_if_nonfinite=False to scale by it anyway" % float(norm_type))


def _refuse_capture() -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("error_if_nonfinite=True reads the norm on the host, which a captured call cannot")


# --------------------------------------------------------------------------------- a list of tensors: the norm
def global_norm(tensors: Tensors, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The norm of all elements of ``tensors`` (tensors, a module's parameters, or one tensor) as if they were one
    vector: ``norm_type`` 2, 1 or inf.  A scalar on their device, float32 (float64 if any tensor is); 0 for no
    elements.  NaN anywhere gives NaN; ``error_if_nonfinite`` raises where the norm, as it is returned, is NaN or
    infinite (it waits for the GPU)."""
    code = _norm_code(norm_type)
    tensors = _tensors_of(tensors)
    with _place(_device_of(tensors, stream), stream):
        if error_if_nonfinite:
            _refuse_capture()
        if not tensors:
            return torch.zeros((), dtype=torch.float32, device=_device_of(tensors, stream))
        tables, keep = _pack([tensors], 1), None
        if tables is None:
            tables, _, keep = _pack_checked([tensors], ["tensors"], 1)
        raw = _raw_stream(tables.device)
        rc, out = tables.norm(_lib.entry("dla_norm"), code, _counter(tables.device, raw), _lib.norm_workspace(tables.n), raw)
        if rc:
            _lib.lib().check(rc, "dla_norm")
        del keep
        if error_if_nonfinite:
            _refuse_nonfinite(out, norm_type)
        return out


def clip_global_norm(tensors: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                     outs: Optional[Sequence[torch.Tensor]] = None,
                     stream: Optional[torch.cuda.Stream] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """(``tensors`` times ``min(1, max_norm / (norm + 1e-6))``, their norm): what a list of tensors becomes under a
    largest global norm, the products rounded once to each tensor's dtype.  ``outs``: tensors of the same sizes
    and dtypes to write (``outs[i]`` may be ``tensors[i]``; no other overlap), else new ones.  A NaN norm makes
    everything NaN and one that is infinite in 64 bits multiplies by 0, as torch.nn.utils.clip_grad_norm_ does;
    ``error_if_nonfinite`` raises before anything is written where the norm, as it is returned, is not finite (it waits
    for the GPU)."""
    code = _norm_code(norm_type)
    bound = _bound(max_norm)
    tensors = _tensors_of(tensors)
    with _place(_device_of(tensors, stream), stream):
        if error_if_nonfinite:
            _refuse_capture()
        if outs is None:
            outs = [torch.empty_like(t, requires_grad=False) if isinstance(t, torch.Tensor) else t for t in tensors]
        else:
            outs = _tensors_of(outs)
        if len(outs) != len(tensors):
            raise ValueError("clip_global_norm: %d outs for %d tensors" % (len(outs), len(tensors)))
        if not tensors:
            return list(outs), torch.zeros((), dtype=torch.float32, device=_device_of(tensors, stream))
        tables, back, keep = _pack([tensors, outs], 2, out=1), (), None
        if tables is None:
            tables, back, keep = _pack_checked([tensors, outs], ["tensors", "outs"], 2, out=1)
        raw = _raw_stream(tables.device)
        counter, nbytes = _counter(tables.device, raw), _lib.norm_workspace(tables.n)
        if error_if_nonfinite:
            rc, norm = tables.norm(_lib.entry("dla_norm"), code, counter, nbytes, raw)
            if rc:
                _lib.lib().check(rc, "dla_norm")
            _refuse_nonfinite(norm, norm_type)
        rc, norm = tables.clip(_lib.entry("dla_norm_clip"), code, bound, CLIP_EPS, counter, nbytes, raw)
        if rc:
            _lib.lib().check(rc, "dla_norm_clip")
        if back:
            _write_back(back)
        del keep
        return list(outs), norm


def clip_global_norm_(tensors: Tensors, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                      stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """clip_global_norm in place; returns the norm before it.  Tensors that overlap are refused."""
    tensors = _tensors_of(tensors)
    return clip_global_norm(tensors, max_norm, norm_type, error_if_nonfinite, outs=tensors, stream=stream)[1]


def clip_grad_norm_(parameters: Tensors, max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """What torch.nn.utils.clip_grad_norm_ does: the gradients of ``parameters`` (parameters, or a module) clipped in
    place by their global norm, which is returned.  Parameters without a gradient are skipped.  Narrower than torch's:
    the gradients are on one HIP device, dense and distinct, ``norm_type`` is 1, 2 or inf, and there is no ``foreach``
    to choose by."""
    grads = [p.grad for p in _tensors_of(parameters)]
    return clip_global_norm_([g for g in grads if g is not None], max_norm, norm_type, error_if_nonfinite)


# ----------------------------------------------------------------------------------------- peers around a centre
def _pack_round(lists: List[List[torch.Tensor]], names, lead: int, out: int = -1):
    tables = _pack(lists, lead, out)
    if tables is not None:
        return tables, (), None
    return _pack_checked(lists, names() if callable(names) else names, lead, out=out)


def _check_peers(n: int) -> None:
    if n < 1:
        raise IndexError("list index out of range")
    if n > MAX_PEERS:
        raise ValueError("%d peers: at most %d in one call" % (n, MAX_PEERS))


@contextlib.contextmanager
def _ring_slot(nbytes: int, device: int):
    """(address, bytes) of page-locked memory for a round's table, or (0, 0): the table is small enough to go with
    the launches, the call is being captured (its launches then carry the table by value), or every slot of the
    device's ring is in use."""
    slot = None
    if nbytes and not torch.cuda.is_current_stream_capturing():
        ring = _wsum.table_ring(torch.device("cuda", device))
        slot = ring.take(nbytes, wait=False)
    if slot is None:
        yield 0, 0
        return
    try:
        yield slot[1].data_ptr(), nbytes
    finally:
        ring.done(slot[0], torch.cuda.current_stream(device), fence=True)


_NO_TABLE = contextlib.nullcontext((0, 0))


def _table_host(n_tensors: int, n: int, device: int):
    nbytes = _lib.peer_table(n_tensors, n)
    return _ring_slot(nbytes, device) if nbytes else _NO_TABLE


def update_norms(models: Sequence[Tensors], center: Tensors, stream: Optional[torch.cuda.Stream] = None,
                 squared: bool = False) -> torch.Tensor:
    """``|| model_k - center ||_2`` over all tensors of each model (lists of tensors, modules' parameters, or flat
    tensors, all with the centre's sizes and dtypes): [len(models)], float32 (float64 if any tensor is).
    ``squared``: the float64 squares instead, which ranks that hold one bucket of every model each add up."""
    lists = [_tensors_of(center)] + [_tensors_of(m) for m in models]
    n = len(lists) - 1
    _check_peers(n)
    device = _device_of(lists[0], stream)
    with _place(device, stream):
        if not lists[0] and not any(lists):
            return torch.zeros(n, dtype=torch.float64 if squared else torch.float32, device=device)
        tables, _, keep = _pack_round(lists, lambda: ["center"] + ["model %d" % k for k in range(n)], 1)
        raw = _raw_stream(tables.device)
        with _table_host(tables.n, n, tables.device) as (table, table_bytes):
            rc, out = tables.peer_norms(_lib.entry("dla_peer_norms"), n, squared, _counter(tables.device, raw), table,
                                        table_bytes, _lib.peer_workspace(tables.n, n), raw)
            if rc:
                _lib.lib().check(rc, "dla_peer_norms")
        del keep
        return out


def wsum_bounded_tables(tables, outs, weights: Sequence[float], max_norm: float,
                        sq_norms: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dla_wsum_bounded on packed tables (the centre first, then the outputs unless ``outs`` has their addresses, then
    the peers) on the current stream; returns the update norms [n]."""
    n = len(weights)
    raw = _raw_stream(tables.device)
    with _table_host(tables.n, n, tables.device) as (table, table_bytes):
        rc, norms = tables.bounded(_lib.entry("dla_wsum_bounded"), outs, weights, max_norm,
                                   0 if sq_norms is None else sq_norms.data_ptr(), _counter(tables.device, raw), table,
                                   table_bytes, _lib.peer_workspace(tables.n, n), raw)
        if rc:
            _lib.lib().check(rc, "dla_wsum_bounded")
    return norms


def wsum_bounded_multi(peer_params: Sequence[Tensors], weights: Sequence[float], center_params: Tensors, max_norm: float,
                       outs: Sequence[torch.Tensor], stream: Optional[torch.cuda.Stream] = None,
                       sq_norms: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The average of norm-bounded updates over the tensors of whole models::

        n_k     = || peer_k - center ||_2  over all its tensors
        outs[i] = center[i] + sum_k weights[k] * min(1, max_norm / n_k) * (peer_k[i] - center[i])

    in list order, carried in 64 bits (32 for the 16-bit types, where they hold every term) and rounded once.  A peer
    whose update is not finite (n_k, in 64 bits, is NaN or infinite) adds nothing.  ``outs[i]`` may be the i-th tensor of
    the centre or of a peer; no other overlap.  ``sq_norms``: float64 squared norms [n] on the device to bound by, when
    the tensors are one bucket of models whose norms are known (update_norms(squared=True), added up).  At most 2 048
    peers.  Returns the norms [n], float32 (float64 if any tensor is)."""
    bound = _bound(max_norm)
    outs = _tensors_of(outs)
    lists = [_tensors_of(center_params), outs] + [_tensors_of(p) for p in peer_params]
    n = len(lists) - 2
    _check_peers(n)
    if len(weights) != n:
        raise AssertionError("len(weights) != len(peers)")
    device = _device_of(lists[0], stream)
    with _place(device, stream):
        if not any(lists):
            return torch.zeros(n, dtype=torch.float32, device=device) if sq_norms is None else sq_norms.sqrt().float()
        tables, back, keep = _pack_round(lists, lambda: ["center", "outs"] + ["peer %d" % k for k in range(n)], 2, out=1)
        if sq_norms is not None and (sq_norms.dtype != torch.float64 or sq_norms.numel() != n
                                     or sq_norms.device != device or not sq_norms.is_contiguous()
                                     or sq_norms.is_neg() or not _held(sq_norms)):
            raise ValueError("sq_norms must be %d contiguous float64 values on %s" % (n, device))
        norms = wsum_bounded_tables(tables, None, [float(w) for w in weights], bound, sq_norms)
        if back:
            _write_back(back)
        del keep
        return norms


def wsum_bounded(peers: Sequence[torch.Tensor], weights: Sequence[float], center: torch.Tensor, max_norm: float,
                 out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None,
                 sq_norms: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """wsum_bounded_multi of one buffer per peer (wsum's flat peers): (the bounded average, the norms).  ``out``
    may be the centre or a peer.  With one peer of weight 1 it is that model pulled back to within ``max_norm`` of
    the centre: what a client that bounds its own update sends."""
    max_norm = _bound(max_norm)
    if out is None:
        with _place(_device_of([center], stream), stream):
            out = torch.empty_like(center, requires_grad=False)
    return out, wsum_bounded_multi([[p] for p in peers], weights, [center], max_norm, [out], stream, sq_norms)
