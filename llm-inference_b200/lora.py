"""Low-rank adapters of many requests beside shared projections (q3_lora_plan, q3_lora_add, q3_lora_gate_up).

    plan = LoraPlan(rows, n_adapters)
    plan.update(index)                            # int32 [rows] on the device, -1: none; once per step
    stack = LoraStack([a_q, a_k, a_v], [b_q, b_k, b_v], scale)   # one projection, or several of one input
    lora_add([q, k, v], [q, k, v], x, stack, plan)               # q += scale * B (A x), and so on

a: bf16 [n_adapters, rank, k], b: bf16 [n_adapters, n, rank], contiguous. Launches go to torch's current stream unless one
is given; all tensors must be on the current device, and so must the plan.
"""
from __future__ import annotations

import ctypes
import struct

from ._lib import call, check, load
from .paged import _ARG, _ELSEWHERE, _NO_PLAN, _SHAPE, _refuse, _rows, _stream, _t, _vector
from . import paged


class Q3LoraSlice(ctypes.Structure):
    _fields_ = [("out", ctypes.c_void_p), ("base", ctypes.c_void_p), ("out_stride", ctypes.c_longlong),
                ("base_stride", ctypes.c_longlong), ("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("n", ctypes.c_int)]


class Q3Lora(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("x_stride", ctypes.c_longlong), ("k", ctypes.c_int), ("rank", ctypes.c_int),
                ("n_rows", ctypes.c_int), ("n_adapters", ctypes.c_int), ("ranks", ctypes.c_void_p),
                ("scale", ctypes.c_void_p), ("plan", ctypes.c_void_p)]


# the same two structs packed: these calls run four times a layer, and filling ctypes fields one by one took 1.5 us of 10.8
_SLICE, _LORA = "PPqqPPi4x", struct.Struct("PqiiiiPPP")
assert struct.calcsize(_SLICE) == ctypes.sizeof(Q3LoraSlice) and _LORA.size == ctypes.sizeof(Q3Lora)


class LoraPlan:
    """A step's rows sorted by adapter (q3_lora_plan): make one for the step's number of rows, `update` it once per step, use
    it in every layer. Calls that need it are refused before its first `update`. Calls only read a plan, so they may overlap;
    an `update` has to come after the calls that use the one before (as on one stream)."""

    def __init__(self, n_rows: int, n_adapters: int, device="cuda"):
        torch = _t()
        n = load().q3_lora_plan_bytes(n_rows, n_adapters)
        if n == 0:
            _refuse("q3_lora_plan", "the shape is not supported", _SHAPE)
        self.n_rows, self.n_adapters = n_rows, n_adapters
        # zeros are a plan without rows, for the time between a captured first update and its replay
        self.plan = torch.zeros(n, dtype=torch.uint8, device=device)
        self._ptr, self._on, self._updated, self._zeroed = self.plan.data_ptr(), self.plan.get_device(), False, None
        if self.plan.is_cuda and not torch.cuda.is_current_stream_capturing():
            made_on = torch.cuda.current_stream(self.plan.device)
            self._zeroed = made_on.cuda_stream, made_on.record_event()

    def update(self, index, stream=None):
        torch, name, dev = _t(), "q3_lora_plan", paged._device()
        if self._on != dev:
            _refuse(name, _ELSEWHERE)
        at, stream = _vector(name, index, "index", self.n_rows, torch.int32, dev), _stream(stream)
        if self._zeroed is not None and not torch.cuda.is_current_stream_capturing():  # a capture began after a wait for all
            made_on, zeroed = self._zeroed
            if stream != made_on:
                torch.cuda.ExternalStream(stream, self.plan.device).wait_event(zeroed)
            self._zeroed = None
        call(name, self._ptr, self.n_rows, self.n_adapters, at, stream)
        self._updated = True


class LoraStack:
    """The adapters of up to three projections of one input. scale: fp32 [n_adapters] or None (1); ranks: int32 [n_adapters] or
    None, each adapter's own rank where it is below that of a and b. Keeps the tensors, not copies of them."""

    def __init__(self, a, b, scale=None, ranks=None):
        torch, name = _t(), "q3_lora"
        a, b = list(a), list(b)
        dev = paged._device()
        if not 1 <= len(a) <= 3 or len(a) != len(b):
            _refuse(name, "one to three projections, each with an a and a b", _SHAPE)
        if a[0].dim() != 3 or any(t.shape != a[0].shape for t in a):
            _refuse(name, "a must be [n_adapters, rank, k], alike for all projections", _SHAPE)
        self.n_adapters, self.rank, self.k = a[0].shape
        self.n = []
        for t in b:
            if t.dim() != 3 or t.shape[0] != self.n_adapters or t.shape[2] != self.rank:
                _refuse(name, "b must be [n_adapters, n, rank]", _SHAPE)
            self.n.append(t.shape[1])
        if self.rank < 1 or self.rank > 128 or any(v < 1 or v % 8 for v in (self.rank, self.k, *self.n)):
            _refuse(name, "rank (up to 128), k and n must be multiples of 8", _SHAPE)
        self._a = [_vector(name, t, "a", None, torch.bfloat16, dev) for t in a]
        self._b = [_vector(name, t, "b", None, torch.bfloat16, dev) for t in b]
        self._ranks = _vector(name, ranks, "ranks", self.n_adapters, torch.int32, dev) or 0
        self._scale = _vector(name, scale, "scale", self.n_adapters, torch.float32, dev) or 0
        self._pack, self._kept, self._on = struct.Struct("".join([_SLICE] * len(a))).pack, (a, b, scale, ranks), dev

    def _bind(self, name, x, plan, dev):
        if not plan._updated:
            _refuse(name, _NO_PLAN)
        if plan._on != dev:
            _refuse(name, _ELSEWHERE)
        if self._on != dev:
            _refuse(name, "the adapters are on another device")
        if plan.n_adapters != self.n_adapters:
            _refuse(name, f"{self.n_adapters} adapters, the plan is for {plan.n_adapters}", _SHAPE)
        return _LORA.pack(x.data_ptr(), _rows(name, x, "x", plan.n_rows, self.k, _t().bfloat16, dev), self.k, self.rank, plan.n_rows,
                          self.n_adapters, self._ranks, self._scale, plan._ptr)


def lora_add(outs, bases, x, stack: LoraStack, plan: LoraPlan, stream=None):
    """out = base + scale * B (A x) of each row's adapter, for each projection of the stack (q3_lora_add). outs, bases: a bf16 tensor
    of [rows, n] for each, or one tensor where the stack has one; an out may be its base."""
    name, bf, dev = "q3_lora_add", _t().bfloat16, paged._device()
    if not isinstance(outs, (list, tuple)):
        outs, bases = [outs], [bases]
    lora, n = stack._bind(name, x, plan, dev), len(stack.n)
    if len(outs) != n or len(bases) != n:
        _refuse(name, f"{len(outs)} outputs and {len(bases)} bases for {n} projections", _SHAPE)
    rows, fields = plan.n_rows, []
    for out, base, width, a, b in zip(outs, bases, stack.n, stack._a, stack._b):
        fields += (out.data_ptr(), base.data_ptr(), _rows(name, out, "out", rows, width, bf, dev), _rows(name, base, "base", rows, width, bf, dev),
                   a, b, width)
    status = load().q3_lora_add(stack._pack(*fields), n, lora, _stream(stream))
    if status:
        check(name, status)


def lora_gate_up(act, gate, up, x, stack: LoraStack, plan: LoraPlan, stream=None):
    """act = silu(gate + its adapter's part) * (up + its adapter's part) for the rows with an adapter, the others stay
    (q3_lora_gate_up): gate and up are the shared projection's taps, bf16 [rows, n], act what it made of them. The stack has
    two projections, gate and up."""
    name, bf, dev = "q3_lora_gate_up", _t().bfloat16, paged._device()
    lora, rows = stack._bind(name, x, plan, dev), plan.n_rows
    if len(stack.n) != 2 or stack.n[0] != stack.n[1]:
        _refuse(name, "the stack must have two projections of the same width", _SHAPE)
    width, fields = stack.n[0], []
    for base, a, b in zip((gate, up), stack._a, stack._b):
        fields += (0, base.data_ptr(), 0, _rows(name, base, "gate and up", rows, width, bf, dev), a, b, width)
    status = load().q3_lora_gate_up(act.data_ptr(), _rows(name, act, "act", rows, width, bf, dev), stack._pack(*fields), lora, _stream(stream))
    if status:
        check(name, status)
