"""Training stages: hand-written kernels for what a per-sample kernel cannot
hold in one lane.

* :func:`recurrence`       a gated linear recurrence along a long axis;
* :func:`token_logp`       the log-probability of each row's target;
* :func:`policy_loss`      the clipped policy loss with a KL term;
* :func:`preference_loss`  the loss of pairs of sequences;
* :func:`dropout`          dropout from a counter-based generator, no mask stored;
* :func:`layer_norm`       layer norm over rows, its derivative with the weights' sums;
* :func:`linear_attention` linear attention with a decay for each head;
* :func:`sample`           a token drawn from each row of logits.

A stage is run as a loaded kernel is: ``hawk.run(stage, **planes)`` writes the
caller's output planes in place, on the current HIP stream or ``stream=``, and
``stage.prepare(**planes)`` returns a launcher that is one crossing a call.
``stage.vjp`` (also ``hawk.diff.vjp(stage)``) is its reverse-mode derivative:
a stage whose planes are the primal's with ``bar_`` names for adjoints::

    scan = hawk.stages.recurrence(gate="sigmoid")
    hawk.run(scan, gate=z, x=x, h=h)
    hawk.run(scan.vjp, gate=z, x=x, h=h, bar_h=bar_h, bar_gate=bar_z, bar_x=bar_x)

A stage is no traced kernel: it has no ``hawk.diff.jvp`` and is no member of a
``hawk.chain`` or ``hawk.steps``; it takes the planes that kernels write and read.

Planes are PyTorch-ROCm tensors, bound by address.  An output that may be an input is
that tensor: one address with other strides is refused.  Scratch belongs to a stream,
or to the graph a call is captured in: calls on several streams and replays of
several graphs may run at once (a launcher's own run one after another).  Nothing
synchronises.
"""

from __future__ import annotations

import ctypes
import math
import numbers
import threading

import torch

from . import _core
from .ir import HawkError
from .runtime import Stage, _on, _stream_of, _Workspace

_Tensor = torch.Tensor

__all__ = ["recurrence", "token_logp", "policy_loss", "preference_loss", "dropout", "layer_norm", "linear_attention",
           "sample"]

def _current_device() -> int:
    raw = getattr(torch._C, "_cuda_getDevice", None)
    if raw is None or not torch.cuda.is_initialized():
        return torch.cuda.current_device() if torch.cuda.is_available() else -1
    return raw()


def _current_raw(device: int) -> int:
    """The current HIP stream's handle on ``device``."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return torch.cuda.current_stream(device).cuda_stream if raw is None else raw(device)


#: Plans a stage keeps (one a set of shapes, strides and types); past this the
#: oldest half is dropped.
PLANS = 256


class _Plan:
    """One set of shapes, strides and types, checked: the job's fields that do
    not move between calls, and where the pointers go."""

    __slots__ = ("job", "slots", "fn", "entry", "scratch", "state", "cells", "apart", "spaces", "call")

    def __init__(self, job, slots: dict, fn, scratch: int, state=None, cells=(), apart=(), entry=None):
        self.job, self.fn, self.scratch = job, fn, scratch
        self.entry = entry                  # the entry of a stage without scratch
        self.slots = slots                  # plane -> word of the job that holds its address
        self.state = state                  # the job's word for the stream's zeroed state
        self.cells = cells                  # by-value words: (name, word)
        self.apart = apart                  # planes that may not start at one address
        self.spaces: dict = {}              # stream -> _Space
        self.call = None

    def bind(self, arrays: dict, values: tuple, device: int) -> None:
        """``call``: what checks a call's planes against these ones and runs it."""
        names = list(arrays)
        cells = dict(self.cells)
        planes = tuple((n, None, cells[n]) if n in values else (n, x, self.slots[n]) if x is not None else (n, None, -1)
                       for n, x in arrays.items())
        apart = tuple((names.index(a), names.index(b)) for a, b in self.apart
                      if arrays.get(a) is not None and arrays.get(b) is not None)
        entry = ctypes.cast(self.entry or self.fn, ctypes.c_void_p).value
        self.call = _core.bind().Call(entry, self.entry is not None, bool(self.scratch), device, bytes(self.job),
                                      -1 if self.state is None else self.state, planes, apart,
                                      _core.stream_capturing_entry())


def _word(job_type, *path) -> int:
    """The 64-bit word of ``job_type`` that field ``path`` begins at."""
    at = 0
    for name in path:
        field = getattr(job_type, name)
        at += field.offset
        job_type = dict(job_type._fields_)[name]
    return at // 8


_spaces: dict = {}
_spaces_lock = threading.Lock()


class _Space:
    """What a stage's calls on a stream work in: scratch, shared by every stage
    on it (a stream's calls run one after another), and zeroed state that every
    call leaves at zero."""

    __slots__ = ("scratch", "state", "held")

    def __init__(self, scratch, state):
        self.held = scratch, state
        self.scratch, self.state = scratch.data_ptr(), state.data_ptr()


def _space(device: int, stream: int, nbytes: int, state: bool) -> tuple:
    """``(space, kept)``: what the calls on ``stream`` work in.  A captured call's is
    its own: the memory is the graph's, which may be replayed on another stream
    beside calls on this one, and its state is cleared by the graph's replays."""
    with _spaces_lock, _on(stream):
        if _core.stream_capturing(stream):
            clear = torch.zeros if state else torch.empty
            return _Space(torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{device}"),
                          clear(_core.STATE_BYTES if state else 0, dtype=torch.uint8, device=f"cuda:{device}")), False
        found = _spaces.get((device, stream))
        if found is None:
            found = _spaces[device, stream] = _Workspace(torch.device("cuda", device))
        return _Space(found.bytes(("stage", "scratch", nbytes), nbytes),
                      found.bytes(("stage", "state"), _core.STATE_BYTES, zero=True)), True


class _Stage(Stage):
    """A stage: its planes by name, a plan a set of shapes."""

    #: Planes the stage reads, may read, writes (or may write).
    reads: tuple = ()
    may_read: tuple = ()
    writes: tuple = ()
    values: tuple = ()                      # by-value arguments
    vjp_of = None

    def __init__(self):
        self._plans: dict = {}
        self._last = None                   # the plan of the call before
        self._lock = threading.Lock()

    @property
    def planes(self) -> tuple:
        """Every plane's name."""
        return self.reads + self.may_read + self.writes

    def _refuse(self, text: str):
        raise HawkError(f"{self.name}: {text}")

    def _names(self, arrays: dict) -> None:
        for name in arrays:
            if name not in self.planes and name not in self.values:
                self._refuse(f"no plane is named {name!r} (planes: {', '.join(self.planes + self.values)})")
        for name in self.reads + self.values:
            if arrays.get(name) is None:
                self._refuse(f"the plane {name!r} is not given")
        if not any(arrays.get(name) is not None for name in self.writes):
            self._refuse(f"no output is given (one of {', '.join(self.writes)})")

    def _placed(self, arrays: dict) -> dict:
        """The planes that are given: tensors of the current device, outputs that
        repeat no memory."""
        tensors = {n: x for n, x in arrays.items() if x is not None and n in self.planes}
        for n, x in tensors.items():
            if not isinstance(x, torch.Tensor):
                self._refuse(f"the plane {n!r} is a torch tensor, got {type(x).__name__}")
            if not x.is_cuda:
                self._refuse(f"the plane {n!r} is on {x.device}, not on a ROCm device")
        devices = {x.get_device() for x in tensors.values()}
        if len(devices) != 1:
            self._refuse(f"its planes are on several devices: {sorted(devices)}")
        if devices != {torch.cuda.current_device()}:
            self._refuse(f"its planes are on cuda:{devices.pop()}, the current device is cuda:"
                         f"{torch.cuda.current_device()}")
        for n in self.writes:
            x = tensors.get(n)
            if x is not None and x.numel() and any(d > 1 and st == 0 for d, st in zip(x.shape, x.stride())):
                self._refuse(f"the output {n!r} repeats memory (strides {tuple(x.stride())})")
        return tensors

    def _crossed(self, tensors: dict) -> tuple:
        """The pairs of an output and another plane that lie differently: at one address
        an element of the one would be written over others of the other."""
        def lies(x):
            return [(d, st) for d, st in zip(x.shape, x.stride()) if d > 1]
        return tuple((out, n) for out in self.writes if out in tensors for n, x in tensors.items()
                     if n != out and x.shape == tensors[out].shape and lies(x) != lies(tensors[out]))

    def _plan(self, key, arrays: dict, device: int) -> _Plan:
        """A plan of ``key``, made, checked and bound before another thread may
        find it."""
        self._names(arrays)
        tensors = self._placed(arrays)
        plan = self._make(tensors)
        plan.apart += self._crossed(tensors)
        if key is None:
            self._refuse("a plane is no dense tensor")
        plan.bind(arrays, self.values, device)
        with self._lock:
            if len(self._plans) >= PLANS:
                for old in list(self._plans)[:PLANS // 2]:
                    del self._plans[old]
            self._plans[key] = plan
        return plan

    def _make(self, tensors: dict) -> _Plan:
        raise NotImplementedError

    def _value(self, name: str, x) -> int:
        raise NotImplementedError

    def _found(self, arrays: dict):
        """``(plan, [(word, value)], device)`` of a call."""
        device = _current_device()
        key = [device]
        try:
            for name, x in arrays.items():
                if x is None or name in self.values:
                    key.append((name, x is None))
                    continue
                key.append((name, x.dtype, x.shape, x.stride(), x.get_device()))
            key = tuple(key)
            plan = self._plans.get(key)
        except (AttributeError, RuntimeError, TypeError):
            plan, key = None, None
        if plan is None:
            plan = self._plan(key, arrays, device)
        self._last = plan if all(x is not None for x in arrays.values()) else None
        bound = [(plan.slots[name], x.data_ptr()) for name, x in arrays.items()
                 if x is not None and name not in self.values]
        return self._finish(plan, bound, arrays, device)

    def _finish(self, plan, bound: list, arrays: dict, device: int):
        for one, two in plan.apart:
            a, b = arrays.get(one), arrays.get(two)
            if a is not None and b is not None and a.data_ptr() == b.data_ptr() and a.numel():
                other = a.shape == b.shape and a.stride() != b.stride()
                self._refuse(f"the output {one!r} and {two!r} are one tensor" + other * ", which lies in two ways")
        for name, word in plan.cells:
            bound.append((word, self._value(name, arrays.get(name))))
        return plan, bound, device

    def run(self, arrays: dict, stream=None) -> None:
        """Bind ``arrays`` and run once, in place (``hawk.run``)."""
        device = _current_device()
        raw = 0 if device < 0 else _current_raw(device) if stream is None else _stream_of(stream)
        plan = self._last
        rc = -1 if plan is None else plan.call.run(arrays, device, raw)      # the planes of the call before, most often
        if rc < 0:
            plan, bound, device = self._found(arrays)
            space = None
            if plan.scratch:
                space = None if _core.stream_capturing(raw) else plan.spaces.get(raw)
                if space is None:
                    space, kept = _space(device, raw, plan.scratch, plan.state is not None)
                    if kept:
                        plan.spaces[raw] = space
                        plan.call.space(raw, space.scratch, space.state)
                if plan.state is not None:
                    bound.append((plan.state, space.state))
            rc = plan.call.launch(bound, 0 if space is None else space.scratch, raw)
        if rc:
            _core.check(rc)

    def prepare(self, *, stream=None, **arrays):
        """Bind the planes once: a launcher whose call is one crossing.  It
        keeps its planes and its scratch."""
        plan, bound, device = self._found(arrays)
        stream = _stream_of(stream)
        job = type(plan.job).from_buffer_copy(plan.job)
        words = (ctypes.c_uint64 * (ctypes.sizeof(job) // 8)).from_buffer(job)
        scratch = state = None
        if plan.scratch:
            with _on(stream):
                scratch = torch.empty(plan.scratch, dtype=torch.uint8, device=f"cuda:{device}")
                # under capture the clearing would wait for a replay: an entry does without
                if plan.state is not None and not _core.stream_capturing(stream):
                    state = torch.zeros(_core.STATE_BYTES, dtype=torch.uint8, device=f"cuda:{device}")
                    bound.append((plan.state, state.data_ptr()))
        for word, value in bound:
            words[word] = value
        return Launcher(plan.fn, job, (scratch, state), stream, dict(arrays))


class Launcher:
    """A stage with its planes bound (:meth:`prepare <_Stage.prepare>`)."""

    def __init__(self, fn, job, scratch: tuple, stream: int, arrays: dict):
        self._held = job, scratch, arrays
        self._args = fn, ctypes.byref(job), None if scratch[0] is None else scratch[0].data_ptr(), stream or None

    def __call__(self) -> None:
        fn, job, scratch, stream = self._args
        rc = fn(job, scratch, stream)
        if rc:
            _core.check(rc)


def _element(stage, dtype, allowed) -> int:
    code = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}.get(dtype)
    if code is None or code not in allowed:
        names = ", ".join(n for c, n in ((0, "float32"), (1, "float64"), (2, "bfloat16"), (3, "float16"))
                          if c in allowed)
        stage._refuse(f"its planes are {names}, got {dtype}")
    return code


def _integer(stage, name: str, x) -> int:
    """1 for a contiguous 1-D int64 plane, 0 for an int32 one."""
    if x.dtype not in (torch.int32, torch.int64) or x.dim() != 1 or not x.is_contiguous():
        stage._refuse(f"{name!r} is a contiguous 1-D int32 or int64 tensor, got {x.dtype} {tuple(x.shape)}")
    return int(x.dtype == torch.int64)


def _vector(stage, name: str, x, count: int) -> None:
    """A contiguous float32 plane of ``count`` numbers (a cell may have no axis)."""
    fits = x.dim() == 1 and x.shape[0] == count or count == 1 and x.dim() == 0
    if x.dtype != torch.float32 or not fits or not x.is_contiguous():
        stage._refuse(f"{name!r} is a contiguous float32 tensor of {count}, got {x.dtype} {tuple(x.shape)}")


# -- the recurrence ------------------------------------------------------------------------

class _Recurrence(_Stage):
    def __init__(self, gate: str, reverse: bool, derivative: bool):
        super().__init__()
        self.gate, self.reverse, self.derivative = gate, reverse, derivative
        self.name = "recurrence_vjp" if derivative else "recurrence"
        if derivative:
            self.reads = ("gate", "h", "bar_h") + (("x",) if gate == "sigmoid" else ())
            self.may_read = ("h0", "bar_last", "offsets") + (() if gate == "sigmoid" else ("x",))
            self.writes = ("bar_gate", "bar_x", "bar_h0")
        else:
            self.reads = ("gate", "x")
            self.may_read = ("h0", "offsets")
            self.writes = ("h", "last")
            self.vjp = _Recurrence(gate, reverse, True)
            self.vjp.vjp_of = self

    def _names(self, arrays: dict) -> None:
        super()._names(arrays)
        if not self.derivative and arrays.get("h") is None:
            self._refuse("the plane 'h' is not given")

    def _make(self, t: dict) -> _Plan:
        first = t["gate"]
        packed = t.get("offsets")
        job = _core.RecurrenceJob()
        job.dtype = _element(self, first.dtype, (0, 1, 2, 3))
        state = torch.float64 if job.dtype == 1 else torch.float32
        slots = {}
        if packed is None and first.dim() != 3:
            self._refuse(f"dense planes are (sequences, steps, channels), got gate {tuple(first.shape)}; packed ones "
                         "(rows, channels) come with offsets")
        if packed is not None:
            if first.dim() != 2:
                self._refuse(f"packed planes are (rows, channels), got gate {tuple(first.shape)}")
            job.offsets64 = _integer(self, "offsets", packed)
            if packed.numel() < 1:
                self._refuse("offsets holds one number more than there are sequences")
            job.seqs = packed.numel() - 1
            job.steps, job.chans = first.shape
        else:
            job.seqs, job.steps, job.chans = first.shape
        job.sigmoid, job.reverse = int(self.gate == "sigmoid"), int(self.reverse)
        for n in ("gate", "x", "h", "bar_h", "bar_gate", "bar_x"):
            x = t.get(n)
            if x is None:
                continue
            if x.shape != first.shape or x.dtype != first.dtype:
                self._refuse(f"{n!r} is {x.dtype} {tuple(x.shape)}, gate is {first.dtype} {tuple(first.shape)}")
            plane = getattr(job, n)
            strides = x.stride()
            plane.seq = 0 if packed is not None else strides[0]
            # an axis of one element has no stride of its own
            plane.step = strides[-2] if job.steps > 1 else 1
            plane.chan = strides[-1] if job.chans > 1 else 1
            slots[n] = _word(_core.RecurrenceJob, n, "data")
            plane.data = 8                  # any address: which planes there are decides how the call is cut
        for n in ("h0", "bar_last", "last", "bar_h0"):
            x = t.get(n)
            if x is None:
                continue
            if x.dtype != state or tuple(x.shape) != (job.seqs, job.chans) or not x.is_contiguous():
                self._refuse(f"the state {n!r} is a contiguous {state} tensor ({job.seqs}, {job.chans}), got "
                             f"{x.dtype} {tuple(x.shape)}")
            slots[n] = _word(_core.RecurrenceJob, n)
            setattr(job, n, 8)
        if packed is not None:
            slots["offsets"] = _word(_core.RecurrenceJob, "offsets")
            job.offsets = 8
        L = _core.lib()
        fn = L.hk_recurrence_vjp if self.derivative else L.hk_recurrence
        scratch = int(L.hk_recurrence_scratch_bytes(ctypes.byref(job), int(self.derivative)))
        apart = (("bar_gate", "h"), ("bar_x", "h"), ("bar_gate", "bar_x")) if self.derivative else ()
        return _Plan(job, slots, fn, scratch, apart=apart)


def recurrence(gate: str = "value", reverse: bool = False) -> Stage:
    """The gated linear recurrence ``h_t = a_t h_{t-1} + b_t`` along the steps.

    ``gate="value"``: ``a = gate``, ``b = x``.  ``gate="sigmoid"``:
    ``a = sigma(gate)``, ``b = (1 - a) x``.  ``reverse=True`` runs from the last
    step to the first (discounted sums: advantages with
    ``gate = discount * lambda * (1 - done)``).

    Planes: ``gate``, ``x``, ``h`` (written), all ``(sequences, steps,
    channels)`` of one type (float64, float32, bfloat16, float16), any strides,
    fastest where the channels or the steps are contiguous; or packed ``(rows,
    channels)`` with ``offsets``, the sequences' bounds (int32 or int64, one more
    than there are sequences, ascending from 0 to the rows; a sequence may be
    empty).  ``h0`` (state that enters, 0 if not given) and ``last`` (state that
    leaves, written) are ``(sequences, channels)`` in float32, float64 for
    float64 planes; ``last`` may be ``h0``, and ``.vjp``'s ``bar_h0`` ``bar_last``.
    ``h`` may be ``x`` or ``gate``.
    One token of running sequences is the same call with one step, ``h0`` and
    ``last``.

    A gate of exactly 0 cuts: nothing before it reaches the state, not even an
    infinity or a NaN.  A sigmoid gate is 0 below -86.6 (-745 in float64).  Finite
    gates of any size are taken: their products are held past the type's range.  Runs of
    steps are joined, so where gates grow, a run's own sum from a zero state has to
    stay in that range, and rounding errors grow as the gates' product does.

    ``.vjp`` reads ``gate``, ``h``, ``bar_h`` (``x`` too for the sigmoid gate),
    ``h0``, ``bar_last``, ``offsets`` and writes those given of ``bar_gate``,
    ``bar_x``, ``bar_h0``.  A plane that was expanded along an axis gets its
    full gradient; its own is the sum along that axis."""
    if gate not in ("value", "sigmoid"):
        raise HawkError(f"recurrence: gate= is 'value' or 'sigmoid', got {gate!r}")
    return _Recurrence(gate, bool(reverse), False)


# -- rows of logits ------------------------------------------------------------------------

class _Rows(_Stage):
    #: The planes of one number a row.
    per_row = ("logp", "lse", "bar_logp", "old_logp", "ref_logp", "advantage")
    entry = ""

    def __init__(self, scale: float, **options):
        super().__init__()
        if not isinstance(scale, (int, float)) or not scale > 0 or not math.isfinite(scale):
            raise HawkError(f"{self.name}: scale= is a positive number, got {scale!r}")
        self.options = dict(scale=float(scale), **options)

    def _make(self, t: dict) -> _Plan:
        job, slots = _core.RowLossJob(), {}
        logits, target = t["logits"], t["target"]
        if logits.dim() != 2:
            self._refuse(f"logits are (rows, vocabulary), got {tuple(logits.shape)}")
        job.dtype = _element(self, logits.dtype, (0, 2, 3))
        job.rows, job.vocab = logits.shape
        job.target64 = _integer(self, "target", target)
        if target.shape[0] != job.rows:
            self._refuse(f"target has {target.shape[0]} rows, logits {job.rows}")
        for n in ("logits", "bar_logits"):
            x = t.get(n)
            if x is None:
                continue
            if x.shape != logits.shape or x.dtype != logits.dtype:
                self._refuse(f"{n!r} is {x.dtype} {tuple(x.shape)}, logits are {logits.dtype} {tuple(logits.shape)}")
            if job.vocab > 1 and x.stride(1) != 1:
                self._refuse(f"a row of {n!r} is contiguous, got strides {tuple(x.stride())}")
            if n == "bar_logits" and job.rows > 1 and x.stride(0) < job.vocab:
                self._refuse(f"the rows of 'bar_logits' overlap (strides {tuple(x.stride())})")
            setattr(job, "row_stride" if n == "logits" else "bar_stride", x.stride(0))
        for n in self.per_row:
            if t.get(n) is not None:
                _vector(self, n, t[n], job.rows)
        for n in ("loss", "bar_loss"):
            if t.get(n) is not None:
                _vector(self, n, t[n], 1)
        self._more(t, job)
        for n, v in self.options.items():
            setattr(job, n, v)
        for n in t:
            slots[n] = _word(_core.RowLossJob, n)
        L = _core.lib()
        if self.vjp_of is not None:         # a derivative works in registers
            return _Plan(job, slots, getattr(L, self.entry), 0)
        scratch = int(L.hk_row_loss_scratch_bytes(ctypes.byref(job))) if "loss" in self.writes else min(job.rows, 1)
        return _Plan(job, slots, getattr(L, self.entry), scratch, state=_word(_core.RowLossJob, "state"))

    def _more(self, t: dict, job) -> None:
        if t.get("weight") is not None:
            _vector(self, "weight", t["weight"], job.rows)


class _TokenLogp(_Rows):
    def __init__(self, derivative: bool = False, **options):
        self.name = "token_logp_vjp" if derivative else "token_logp"
        self.entry = "hk_token_logp_vjp" if derivative else "hk_token_logp"
        super().__init__(**options)
        if derivative:
            self.reads, self.writes = ("logits", "target", "lse", "bar_logp"), ("bar_logits",)
        else:
            self.reads, self.writes = ("logits", "target"), ("logp", "lse")
            self.vjp = _TokenLogp(True, **options)
            self.vjp.vjp_of = self


def token_logp(scale: float = 1.0) -> Stage:
    """The log-probability of each row's target under ``softmax(scale * logits)``.

    Planes: ``logits`` ``(rows, vocabulary)`` in float32, bfloat16 or float16,
    a row contiguous, rows any distance apart; ``target`` int32 or int64;
    ``logp`` and ``lse`` (the row's log-sum-exp) float32, those given are
    written.  A target below 0 leaves its row out (``logp`` and ``lse`` 0, the
    logits not read); one past the vocabulary gives a NaN.  A logit of +inf makes
    ``lse`` +inf: the other logits have probability 0, its own is a NaN.

    ``.vjp`` reads ``logits``, ``target``, ``lse``, ``bar_logp`` and writes
    ``bar_logits`` (it may be ``logits``)."""
    return _TokenLogp(scale=scale)


class _PolicyLoss(_Rows):
    def __init__(self, derivative: bool = False, **options):
        self.name = "policy_loss_vjp" if derivative else "policy_loss"
        self.entry = "hk_policy_loss_vjp" if derivative else "hk_policy_loss"
        super().__init__(**options)
        needed = ("logits", "target", "old_logp", "advantage") + (("ref_logp",) if options["kl"] else ())
        more = ("weight", "bar_loss") + (() if options["kl"] else ("ref_logp",))
        if derivative:
            self.reads, self.may_read, self.writes = needed + ("logp", "lse"), more, ("bar_logits",)
        else:
            self.reads, self.may_read, self.writes = needed, more, ("loss", "logp", "lse", "bar_logits")
            self.vjp = _PolicyLoss(True, **options)
            self.vjp.vjp_of = self


def policy_loss(clip=0.2, kl: float = 0.0, scale: float = 1.0) -> Stage:
    """The clipped policy loss over rows of logits, with a KL term:
    ``sum_n weight_n (-min(r A, clamp(r, 1 - low, 1 + high) A) + kl (e^d - d - 1))``
    with ``r = exp(logp - old_logp)`` and ``d = ref_logp - logp``.

    ``clip``: ``low = high``, or ``(low, high)``.  Planes: ``logits`` and
    ``target`` as :func:`token_logp`; ``old_logp``, ``advantage``, ``ref_logp``
    (read if ``kl``), ``weight`` (1 / rows if not given; a weight of 0 leaves the
    row out whatever its other values) float32, one a row.  Written where given:
    ``loss`` (one cell, summed in a fixed order), ``logp``, ``lse``, and
    ``bar_logits``, the gradient of the loss (times ``bar_loss``, one cell, if
    given) in the same pass over the logits.

    ``.vjp`` takes ``logp`` and ``lse`` from an earlier call and writes
    ``bar_logits``.  The clipped term has a gradient where ``r A`` is at most the
    clipped product (at the bounds too)."""
    low, high = clip if isinstance(clip, (tuple, list)) and len(clip) == 2 else (clip, clip)
    if not all(isinstance(c, (int, float)) and c >= 0 and math.isfinite(c) for c in (low, high)):
        raise HawkError(f"policy_loss: clip= is a number from 0 or a pair of them, got {clip!r}")
    if not isinstance(kl, (int, float)) or not math.isfinite(kl):
        raise HawkError(f"policy_loss: kl= is a finite number, got {kl!r}")
    return _PolicyLoss(clip_low=float(low), clip_high=float(high), kl=float(kl), scale=scale)


class _PreferenceLoss(_Rows):
    def __init__(self, derivative: bool = False, **options):
        self.name = "preference_loss_vjp" if derivative else "preference_loss"
        self.entry = "hk_preference_loss_vjp" if derivative else "hk_preference_loss"
        super().__init__(**options)
        if derivative:
            self.reads, self.may_read = ("logits", "target", "offsets", "margin", "lse"), ("weight", "bar_loss")
            self.writes = ("bar_logits",)
        else:
            self.reads, self.may_read = ("logits", "target", "offsets"), ("ref_logp", "weight")
            self.writes = ("loss", "margin", "logp", "lse")
            self.vjp = _PreferenceLoss(True, **options)
            self.vjp.vjp_of = self

    def _more(self, t: dict, job) -> None:
        job.offsets64 = _integer(self, "offsets", t["offsets"])
        cuts = t["offsets"].numel()
        if cuts % 2 != 1:
            self._refuse(f"offsets holds 2 * pairs + 1 numbers, got {cuts}")
        job.pairs = cuts // 2
        for n in ("margin", "weight"):
            if t.get(n) is not None:
                _vector(self, n, t[n], job.pairs)


def preference_loss(beta: float = 0.1, smoothing: float = 0.0, scale: float = 1.0) -> Stage:
    """The loss of pairs of sequences by their log ratios against a reference:
    ``sum_p weight_p (-(1 - smoothing) log sigma(z_p) - smoothing log sigma(-z_p))``,
    ``z_p = beta margin_p``, ``margin_p`` the preferred sequence's sum of
    ``logp - ref_logp`` minus the other's.

    Planes: ``logits`` and ``target`` as :func:`token_logp`, the rows of all
    sequences in turn; ``offsets`` (int32 or int64, ``2 * pairs + 1``) bounds
    them: pair p prefers sequence 2p to 2p + 1; ``ref_logp`` float32, one a row
    (0 if not given); ``weight``, one a pair (1 / pairs if not given).  Rows with
    a target below 0 (a prompt's) are left out of the sums.  Written where given:
    ``loss`` (one cell), ``margin`` (one a pair), ``logp``, ``lse``.

    ``.vjp`` reads ``logits``, ``target``, ``offsets``, ``margin``, ``lse``,
    ``weight``, ``bar_loss`` and writes ``bar_logits``."""
    if not isinstance(beta, (int, float)) or not math.isfinite(beta):
        raise HawkError(f"preference_loss: beta= is a finite number, got {beta!r}")
    if not isinstance(smoothing, (int, float)) or not 0 <= smoothing <= 1:
        raise HawkError(f"preference_loss: smoothing= is in [0, 1], got {smoothing!r}")
    return _PreferenceLoss(beta=float(beta), smoothing=float(smoothing), scale=scale)


# -- dropout -------------------------------------------------------------------------------

def _row_stride(stage, name: str, x) -> int:
    """The distance of rows that lie evenly apart, each contiguous."""
    if not x.numel():
        return 0
    dims = [(d, st) for d, st in zip(x.shape[:-1], x.stride()[:-1]) if d != 1]
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        stage._refuse(f"a row of {name!r} is contiguous, got strides {tuple(x.stride())}")
    for (_, outer), (d, inner) in zip(dims, dims[1:]):
        if outer != d * inner:
            stage._refuse(f"the rows of {name!r} are not evenly apart (shape {tuple(x.shape)}, strides "
                          f"{tuple(x.stride())})")
    return dims[-1][1] if dims else 0


class _Dropout(_Stage):
    values = ("seed", "offset")

    def __init__(self, p: float, derivative: bool):
        super().__init__()
        self.p, self.derivative = p, derivative
        self.cut = int(round(p * 65536))
        self.name = "dropout_vjp" if derivative else "dropout"
        if derivative:
            self.source, self.target = "bar_y", "bar_x"
            self.reads, self.writes = ("bar_y",), ("bar_x",)
        else:
            self.source, self.target = "x", "y"
            self.reads, self.may_read, self.writes = ("x",), ("residual",), ("y",)
            self.vjp = _Dropout(p, True)
            self.vjp.vjp_of = self

    def _names(self, arrays: dict) -> None:
        super()._names({"offset": 0, **arrays})

    def _make(self, t: dict) -> _Plan:
        job, first = _core.DropoutJob(), t[self.source]
        job.dtype = _element(self, first.dtype, (0, 1, 2, 3))
        job.cut = self.cut
        shape = first.shape
        used = [n for n in (self.source, "residual", self.target) if t.get(n) is not None]
        for n in used:
            if t[n].shape != shape or t[n].dtype != first.dtype:
                self._refuse(f"{n!r} is {t[n].dtype} {tuple(t[n].shape)}, {self.source} is {first.dtype} "
                             f"{tuple(shape)}")
        whole = all(t[n].is_contiguous() for n in used)
        if whole:
            job.rows, job.cols = 1, first.numel()
        else:
            job.cols = shape[-1]
            job.rows = first.numel() // shape[-1] if shape[-1] else 0
        field = {self.source: "x", "residual": "residual", self.target: "y"}
        slots = {}
        for n in used:
            if not whole:                   # one row alone is read as contiguous too
                setattr(job, field[n] + "_stride", _row_stride(self, n, t[n]))
            slots[n] = _word(_core.DropoutJob, field[n])
        slots["offset"] = _word(_core.DropoutJob, "offset_cell")
        cells = (("seed", _word(_core.DropoutJob, "seed")), ("offset", _word(_core.DropoutJob, "offset")))
        fn = _core.lib().hk_dropout
        return _Plan(job, slots, lambda ref, scratch, stream: fn(ref, stream), 0, cells=cells, entry=fn)

    def _value(self, name: str, x) -> int:
        if name == "offset" and (x is None or isinstance(x, torch.Tensor)):
            return 0                        # none, or a cell on the device, bound by address
        number = int(x) if isinstance(x, numbers.Integral) and not isinstance(x, bool) else -1
        if not 0 <= number < 1 << 64:
            self._refuse(f"{name}= is an int in [0, 2^64), got {x!r}")
        return number

    def _found(self, arrays: dict):
        cell = arrays.get("offset")
        if isinstance(cell, torch.Tensor) and (cell.dtype != torch.int64 or cell.numel() != 1
                                               or not cell.is_cuda or cell.get_device() != _current_device()):
            self._refuse("offset= is an int or an int64 cell on the device")
        plan, bound, device = super()._found(arrays)
        bound.append((plan.slots["offset"], cell.data_ptr() if isinstance(cell, torch.Tensor) else 0))
        return plan, bound, device


def dropout(p: float) -> Stage:
    """Dropout at rate ``p`` (to the nearest 2^-16), ``y = kept ? x / (1 - p) : 0``
    plus ``residual`` if given, with no mask stored.

    Planes: ``x``, ``residual``, ``y`` (written) of one shape and type (float64,
    float32, bfloat16, float16), contiguous or with contiguous rows evenly apart;
    ``y`` may be ``x`` or ``residual``.  ``seed`` and ``offset`` (0 if not given)
    are ints (numpy's too) below 2^64: an element's number comes from them and its index in
    row-major order alone, so the mask does not depend on strides.  ``offset`` may
    be an int64 cell on the device, read by the kernel: a captured call then
    draws a new mask a replay.  Philox4x32-10 gives the numbers.

    ``.vjp`` (``bar_y``, ``bar_x``, the same ``seed`` and ``offset``) applies the
    same mask; the residual's gradient is ``bar_y``."""
    if isinstance(p, bool) or not isinstance(p, (int, float)) or not 0 <= p <= 1:
        raise HawkError(f"dropout: p= is in [0, 1], got {p!r}")
    cut = int(round(p * 65536))
    if (cut == 0) != (p == 0) or (cut == 65536) != (p == 1):
        raise HawkError(f"dropout: p={p!r} rounds to {cut // 65536} at the generator's resolution of 2^-16")
    return _Dropout(float(p), False)


# -- layer norm ----------------------------------------------------------------------------

def _float32(x) -> float:
    """A number as the kernels hold it: one past float32's range is an infinity."""
    try:
        return ctypes.c_float(x).value
    except OverflowError:                   # an int past float64's
        return math.inf


class _LayerNorm(_Stage):
    def __init__(self, eps: float, derivative: bool):
        super().__init__()
        self.eps, self.derivative = eps, derivative
        self.name = "layer_norm_vjp" if derivative else "layer_norm"
        if derivative:
            self.reads, self.may_read = ("x", "mean", "rstd", "bar_y"), ("weight",)
            self.writes = ("bar_x", "bar_weight", "bar_bias")
        else:
            self.reads, self.may_read, self.writes = ("x",), ("weight", "bias"), ("y", "mean", "rstd")
            self.vjp = _LayerNorm(eps, True)
            self.vjp.vjp_of = self

    def _make(self, t: dict) -> _Plan:
        job, x = _core.LayerNormJob(), t["x"]
        job.dtype = _element(self, x.dtype, (0, 2, 3))
        if x.dim() < 1:
            self._refuse("x has rows of at least one axis")
        job.cols = x.shape[-1]
        job.rows = x.shape[:-1].numel()
        for n in ("x", "y", "bar_y", "bar_x"):
            if n not in t:
                continue
            if t[n].shape != x.shape or t[n].dtype != x.dtype:
                self._refuse(f"{n!r} is {t[n].dtype} {tuple(t[n].shape)}, x is {x.dtype} {tuple(x.shape)}")
            stride = _row_stride(self, n, t[n])
            if n in self.writes and job.rows > 1 and stride < job.cols:
                self._refuse(f"the rows of {n!r} overlap (strides {tuple(t[n].stride())})")
            setattr(job, n + "_stride", stride)
        for n in ("mean", "rstd"):
            if n in t:
                _vector(self, n, t[n], x.shape[:-1].numel())
        weights = [n for n in ("weight", "bias", "bar_weight", "bar_bias") if n in t]
        kind = t[weights[0]].dtype if weights else x.dtype
        if kind not in (torch.float32, x.dtype):
            self._refuse(f"{weights[0]!r} is float32 or {x.dtype}, got {kind}")
        for n in weights:
            if t[n].dtype != kind or tuple(t[n].shape) != (job.cols,) or not t[n].is_contiguous():
                self._refuse(f"{n!r} is a contiguous {kind} tensor of {job.cols}, got {t[n].dtype} {tuple(t[n].shape)}")
        job.weight_dtype = _element(self, kind, (0, 2, 3))
        job.eps = self.eps
        slots = {}
        for n in t:
            slots[n] = _word(_core.LayerNormJob, n)
            setattr(job, n, 16)             # any address: which planes there are decides what a call works in
        L = _core.lib()
        fn = L.hk_layer_norm_vjp if self.derivative else L.hk_layer_norm
        if self.derivative:
            apart = (("bar_weight", "weight"), ("bar_weight", "bar_bias"), ("bar_bias", "weight"), ("bar_x", "weight"),
                     ("bar_x", "mean"), ("bar_x", "rstd"), ("bar_x", "bar_weight"), ("bar_x", "bar_bias"))
        else:
            apart = (*((out, n) for out in self.writes for n in self.may_read), ("mean", "x"), ("rstd", "x"), ("y", "mean"),
                     ("y", "rstd"), ("mean", "rstd"))
        return _Plan(job, slots, fn, int(L.hk_layer_norm_scratch_bytes(ctypes.byref(job), int(self.derivative))),
                     apart=apart)


def layer_norm(eps: float = 1e-5) -> Stage:
    """Layer norm over the last axis: ``y = (x - mean) rstd weight + bias`` with
    ``rstd = 1 / sqrt(var + eps)``.

    Planes: ``x``, ``y`` (written, it may be ``x``) of one shape and type (float32,
    bfloat16, float16), rows contiguous and evenly apart; ``weight`` and ``bias``
    (1 and 0 if not given) of one number a column, in float32 or the planes' type;
    ``mean`` and ``rstd`` float32, one a row, as a contiguous 1-D tensor, written
    where given (NaN where a row has no columns).  Each output is a tensor of its own.

    ``.vjp`` reads ``x``, ``weight``, ``mean``, ``rstd``, ``bar_y`` and writes those
    given of ``bar_x`` (it may be ``x`` or ``bar_y``), ``bar_weight`` and
    ``bar_bias`` (of the weight's type).  The sums over rows are taken in a fixed
    order, 0 where there are no rows."""
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not (eps >= 0 and _float32(eps) < math.inf):
        raise HawkError(f"layer_norm: eps= is a finite float32 from 0, got {eps!r}")
    return _LayerNorm(float(eps), False)


# -- linear attention ----------------------------------------------------------------------

class _LinearAttention(_Stage):
    def __init__(self, scale: float, derivative: bool):
        super().__init__()
        self.scale, self.derivative = scale, derivative
        self.name = "linear_attention_vjp" if derivative else "linear_attention"
        if derivative:
            self.reads, self.may_read = ("q", "k", "v", "decay", "bar_o"), ("h0", "bar_last", "offsets")
            self.writes = ("bar_q", "bar_k", "bar_v", "bar_h0")
        else:
            self.reads, self.may_read, self.writes = ("q", "k", "v", "decay"), ("h0", "offsets"), ("o", "last")
            self.vjp = _LinearAttention(scale, True)
            self.vjp.vjp_of = self

    def _make(self, t: dict) -> _Plan:
        job, q, packed = _core.LinearAttentionJob(), t["q"], t.get("offsets")
        job.dtype = _element(self, q.dtype, (0, 2, 3))
        if packed is None and q.dim() != 4:
            self._refuse(f"dense planes are (sequences, steps, heads, channels), got q {tuple(q.shape)}; packed ones "
                         "(rows, heads, channels) come with offsets")
        if packed is not None:
            if q.dim() != 3:
                self._refuse(f"packed planes are (rows, heads, channels), got q {tuple(q.shape)}")
            job.offsets64 = _integer(self, "offsets", packed)
            if packed.numel() < 1:
                self._refuse("offsets holds one number more than there are sequences")
            job.seqs = packed.numel() - 1
            job.steps, job.heads = q.shape[:2]
        else:
            job.seqs, job.steps, job.heads = q.shape[:3]
        job.keys, job.values = q.shape[-1], t["v"].shape[-1] if t["v"].dim() else 0
        for n, channels in (("q", job.keys), ("v", job.values)):
            if not 1 <= channels <= 256:
                self._refuse(f"a head of {n!r} has 1 to 256 channels, got {tuple(t[n].shape)}")
        slots = {}
        for n in ("q", "k", "v", "o", "bar_o", "bar_q", "bar_k", "bar_v"):
            x = t.get(n)
            if x is None:
                continue
            shape = (*q.shape[:-1], job.keys if n[-1] in "qk" else job.values)
            if tuple(x.shape) != shape or x.dtype != q.dtype:
                self._refuse(f"{n!r} is {x.dtype} {tuple(x.shape)}, where {q.dtype} {shape} goes with q "
                             f"{tuple(q.shape)} and v {tuple(t['v'].shape)}")
            if shape[-1] > 1 and x.stride(-1) != 1:
                self._refuse(f"a head of {n!r} is contiguous, got strides {tuple(x.stride())}")
            plane, strides = getattr(job, n), x.stride()
            plane.seq = 0 if packed is not None else strides[0]
            plane.step, plane.head = strides[-3], strides[-2]
            plane.data = 16                 # any address: which planes there are decides what a call works in
            slots[n] = _word(_core.LinearAttentionJob, n, "data")
        _vector(self, "decay", t["decay"], job.heads)
        for n in ("h0", "bar_last", "last", "bar_h0"):
            x = t.get(n)
            if x is None:
                continue
            shape = (job.seqs, job.heads, job.keys, job.values)
            if x.dtype != torch.float32 or tuple(x.shape) != shape or not x.is_contiguous():
                self._refuse(f"the state {n!r} is a contiguous float32 tensor {shape}, got {x.dtype} {tuple(x.shape)}")
        for n in ("decay", "h0", "bar_last", "last", "bar_h0", "offsets"):
            if n in t:
                slots[n] = _word(_core.LinearAttentionJob, n)
                setattr(job, n, 16)
        job.scale = self.scale
        L = _core.lib()
        fn = L.hk_linear_attention_vjp if self.derivative else L.hk_linear_attention
        scratch = int(L.hk_linear_attention_scratch_bytes(ctypes.byref(job), int(self.derivative)))
        given = [n for n in self.writes if n in t]
        read = [n for n in self.reads + self.may_read if n in t]
        apart = [(out, n) for out in given for n in read if (out, n) != ("last", "h0")]
        apart += [(a, b) for i, a in enumerate(given) for b in given[i + 1:]]
        return _Plan(job, slots, fn, scratch, apart=tuple(apart))


def linear_attention(scale: float = 1.0) -> Stage:
    """Linear attention with a decay for each head: ``S_t = decay S_(t-1) + k_t v_t^T``,
    ``o_t = scale q_t S_t``, from the state ``h0``.

    Planes: ``q``, ``k`` ``(sequences, steps, heads, keys)`` and ``v``, ``o``
    (written) ``(..., values)`` of one type (float32, bfloat16, float16), 1 to 256
    channels a head, those of a head contiguous, the other axes in any order; or
    packed ``(rows, heads, channels)`` with ``offsets``, the sequences' bounds as in
    :func:`recurrence`.  ``decay`` float32, one a head, in [0, 1] (another gives
    NaN); it is a constant and has no gradient.  ``h0`` (state that enters, 0 if not
    given) and ``last`` (state that leaves, written where given; it may be ``h0``)
    are ``(sequences, heads, keys, values)`` in float32.  One token of running
    sequences is the same call with one step, ``h0`` and ``last``.

    States and sums are held in 32 bits; products are taken to 2^-24 where states are made
    and read and for float32 planes; with 16-bit planes those of a token with the last 63
    before it are taken to 2^-16 of each.  A token
    with an infinity or a NaN makes what it reaches no number (an infinity may come
    out as a NaN) and leaves earlier tokens as they are.

    ``.vjp`` reads ``q``, ``k``, ``v``, ``decay``, ``bar_o``, ``h0``, ``bar_last``,
    ``offsets`` and writes those given of ``bar_q``, ``bar_k``, ``bar_v``,
    ``bar_h0``.  A plane that was expanded along an axis (heads that share keys and
    values) gets its full gradient; its own is the sum along that axis.  No output
    may be an input or another output."""
    if isinstance(scale, bool) or not isinstance(scale, (int, float)) or not math.isfinite(_float32(scale)):
        raise HawkError(f"linear_attention: scale= is a finite float32, got {scale!r}")
    return _LinearAttention(float(scale), False)


# -- sampling ------------------------------------------------------------------------------

class _Sample(_Stage):
    reads, writes = ("logits", "u"), ("token", "logp")
    may_read = ("temperature", "top_k", "top_p", "min_p")

    def __init__(self, **options):
        self.name = "sample"
        super().__init__()
        self.options = options

    def _make(self, t: dict) -> _Plan:
        job, logits = _core.SampleJob(), t["logits"]
        if logits.dim() != 2:
            self._refuse(f"logits are (rows, vocabulary), got {tuple(logits.shape)}")
        job.dtype = _element(self, logits.dtype, (0, 2, 3))
        job.rows, job.vocab = logits.shape
        if job.vocab > 1 << 22:
            self._refuse(f"a vocabulary has at most 2^22 tokens, got {job.vocab}")
        if job.vocab > 1 and logits.stride(1) != 1:
            self._refuse(f"a row of 'logits' is contiguous, got strides {tuple(logits.stride())}")
        job.row_stride = logits.stride(0)
        u = t["u"]
        if u.dtype not in (torch.float32, torch.float64) or tuple(u.shape) != (job.rows,) or not u.is_contiguous():
            self._refuse(f"'u' is a contiguous float32 or float64 tensor of {job.rows}, got {u.dtype} {tuple(u.shape)}")
        job.u64bits = int(u.dtype == torch.float64)
        for n in ("logp", "temperature", "top_p", "min_p"):
            if n in t:
                _vector(self, n, t[n], job.rows)
        for n in ("token", "top_k"):
            if n not in t:
                continue
            wide = _integer(self, n, t[n])
            if t[n].shape[0] != job.rows:
                self._refuse(f"{n!r} has {t[n].shape[0]} rows, logits {job.rows}")
            if n == "token":
                job.token64 = wide
            elif wide:
                self._refuse("'top_k' is a contiguous 1-D int32 tensor, got torch.int64")
        for n, v in self.options.items():
            setattr(job, n, v)
        slots = {n: _word(_core.SampleJob, "row_" + n if n in self.may_read else n) for n in t}
        L = _core.lib()
        return _Plan(job, slots, L.hk_sample, int(L.hk_sample_scratch_bytes(ctypes.byref(job))),
                     apart=tuple((out, n) for out in self.writes for n in self.reads + self.may_read) + (("token", "logp"),))


def sample(temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> Stage:
    """A token drawn from each row of logits by a given random number.

    With ``w = exp((logit - max) / temperature)`` and a row's tokens in descending
    order (equal ones by index), the tokens kept are those that every filter keeps:
    the first ``top_k`` (0: all); of these the ones before which less than ``top_p`` of
    their whole weight has passed (1: all); those with ``w >= min_p`` (0: all); the
    highest in any case.  The token is the first, by index, at which the kept
    tokens' running weight passes ``u`` times their whole weight.

    Planes: ``logits`` ``(rows, vocabulary)`` in float32, bfloat16 or float16, a row
    contiguous, rows any distance apart, 2^22 tokens at most; ``u`` float32 or
    float64, one a row in [0, 1) (below draws the first kept token, above the last);
    written where given: ``token`` (int32 or int64) and ``logp`` (float32), the
    token's log-probability among those kept.  ``temperature``, ``top_p``, ``min_p``
    (float32) and ``top_k`` (int32), one a row, stand for the stage's own where given.

    A temperature of 0 takes the highest logit, the first of equal ones, with a
    ``logp`` of 0.  A row that holds a NaN, or whose ``u`` is one or whose
    temperature is below 0 or one, gives token -1 and a NaN; a row of -inf alone
    (nothing is allowed) token -1 and -inf; logits of +inf share the whole.  Weights
    are whole numbers of 2^-40 of the highest (2^22 tokens; 2^-45 for 2^17) and summed
    exactly, so a call repeats bit for bit and a border is off by half of one for each
    token at most.  There is no derivative: the loss reads the token's
    ``token_logp``."""
    def number(x):
        return isinstance(x, (int, float)) and not isinstance(x, bool) and x == x
    if not number(temperature) or temperature < 0:
        raise HawkError(f"sample: temperature= is a number from 0, got {temperature!r}")
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k < 1 << 63:
        raise HawkError(f"sample: top_k= is an int from 0, got {top_k!r}")
    if not number(top_p) or top_p < 0:
        raise HawkError(f"sample: top_p= is a number from 0, got {top_p!r}")
    if not number(min_p):
        raise HawkError(f"sample: min_p= is a number, got {min_p!r}")
    return _Sample(temperature=float(temperature), top_k=top_k, top_p=float(top_p), min_p=float(min_p))
