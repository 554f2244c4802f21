"""Paged serving: the step plan, rotary append, attention over pages and logits processing.

Page tensors are [n_pages, n_kv_heads, page_size, head_dim] torch views with a contiguous last
dimension; a pool laid out [n_pages, page_size, n_kv_heads, head_dim] is passed as
``pool.transpose(1, 2)``. Launches go to torch's current stream unless one is given; all tensors must be on
the current device, and so must the plan.
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._lib import Q3Error, call, check, load

_SHAPE, _ARG = 1, 5
_NO_DEVICE = -2  # no tensor's device: the CPU's is -1
_NO_PLAN = "the plan has not been updated"
_ELSEWHERE = "the plan is on another device"
_torch = _device = _raw_stream = None


def _t():
    """torch, imported when the first tensor arrives."""
    global _torch, _device, _raw_stream
    if _torch is None:
        import torch
        _torch = torch
        # the current device's index and its stream's handle without objects around them, where torch has these
        _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device) if torch.cuda.is_available() else lambda: _NO_DEVICE
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda _: torch.cuda.current_stream().cuda_stream)
    return _torch


class Q3PagedShape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("n_seqs", "n_tokens", "max_q_len", "n_heads", "n_kv_heads", "head_dim",
                                            "page_size", "n_pages", "max_pages")]


class Q3PagedCache(ctypes.Structure):
    _fields_ = [("key_pages", ctypes.c_void_p), ("value_pages", ctypes.c_void_p), ("page_stride", ctypes.c_longlong),
                ("head_stride", ctypes.c_longlong), ("pos_stride", ctypes.c_longlong)]


class Q3RopeScaling(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int), ("factor", ctypes.c_float), ("low_freq_factor", ctypes.c_float),
                ("high_freq_factor", ctypes.c_float), ("beta_fast", ctypes.c_float), ("beta_slow", ctypes.c_float),
                ("attention_factor", ctypes.c_float), ("original_max", ctypes.c_int)]


ROPE_KINDS = {"plain": 0, "linear": 1, "by_parts": 2, "yarn": 3}


def _stream(stream):
    return _raw_stream(_device()) if stream is None else stream


def _refuse(name, what, status=_ARG):
    raise Q3Error(name, status, what)


# These calls run once per layer of every step, so the checks read as few tensor attributes as they can.

def _rows(name, t, what, rows, width, dtype, dev):
    """Row stride of a [rows, ...] tensor whose rows are `width` contiguous elements."""
    if t.dtype is not dtype or t.get_device() != dev:
        _refuse(name, f"{what} must be a tensor of {dtype} on the current CUDA device")
    shape = t.shape
    if not shape or shape[0] != rows:
        _refuse(name, f"{what}: {tuple(shape)}, expected {rows} rows", _SHAPE)
    if t.is_contiguous() and t.numel() == rows * width:
        return width
    n = 1
    for size, step in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and step != n:
            _refuse(name, f"{what}: a row's elements must be contiguous")
        n *= size
    if n != width:
        _refuse(name, f"{what}: {n} elements a row, expected {width}", _SHAPE)
    return t.stride(0) if rows > 1 else width


def _vector(name, t, what, size, dtype, dev):
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
        _refuse(name, f"{what} must be a contiguous tensor of {dtype} on the current CUDA device")
    if size is not None and t.numel() != size:
        _refuse(name, f"{what}: {t.numel()} elements, expected {size}", _SHAPE)
    return t.data_ptr()


class PagedPlan:
    """Device work list of a step (q3_paged_plan): make one for the step's shape, `update` it once
    per step, use it in every layer. Owns the attention's scratch too, so calls that share a plan
    must follow each other on one stream (or be ordered by the caller). Calls that need the plan are
    refused before its first `update`."""

    def __init__(self, n_seqs: int, n_tokens: int, max_q_len: int, n_heads: int, n_kv_heads: int, head_dim: int,
                 page_size: int, n_pages: int, max_pages: int, device="cuda"):
        torch = _t()
        self.shape = Q3PagedShape(n_seqs, n_tokens, max_q_len, n_heads, n_kv_heads, head_dim, page_size, n_pages,
                                  max_pages)
        self._shape = ctypes.byref(self.shape)
        n = load().q3_paged_plan_bytes(self._shape)
        if n == 0:
            _refuse("q3_paged_plan", "the shape is not supported", _SHAPE)
        # zeros are a plan without any work, for the time between a captured first update and its replay
        self.plan = torch.zeros(n, dtype=torch.uint8, device=device)
        self._updated, self._zeroed, self._on = False, None, self.plan.get_device()
        if self.plan.is_cuda and not torch.cuda.is_current_stream_capturing():
            made_on = torch.cuda.current_stream(self.plan.device)
            self._zeroed = made_on.cuda_stream, made_on.record_event()
        self.scratch = torch.empty(load().q3_paged_attention_scratch_bytes(self._shape), dtype=torch.uint8,
                                   device=device)
        self.n_tokens, self.head_dim, self.scale = n_tokens, head_dim, head_dim ** -0.5
        self.q_width, self.kv_width = n_heads * head_dim, n_kv_heads * head_dim
        self._pages = (n_pages, n_kv_heads, page_size, head_dim)
        self._ptr, self._scratch_ptr = self.plan.data_ptr(), self.scratch.data_ptr()
        self._cache = Q3PagedCache()  # filled anew for every call, which reads it before it returns
        self._cache_ref = ctypes.byref(self._cache)
        self._strides = None  # of the pages that _cache describes

    def update(self, q_start, kv_len, page_table, stream=None):
        torch, s, name, stream = _t(), self.shape, "q3_paged_plan", _stream(stream)
        i32, dev = torch.int32, _device()
        if self._on != dev:
            _refuse(name, _ELSEWHERE)
        if self._zeroed is not None and not torch.cuda.is_current_stream_capturing():  # a capture began after a wait for all
            made_on, zeroed = self._zeroed
            if stream != made_on:
                torch.cuda.ExternalStream(stream, self.plan.device).wait_event(zeroed)
            self._zeroed = None
        call(name, self._ptr, self._shape, _vector(name, q_start, "q_start", s.n_seqs + 1, i32, dev),
             _vector(name, kv_len, "kv_len", s.n_seqs, i32, dev),
             _vector(name, page_table, "page_table", s.n_seqs * s.max_pages, i32, dev), stream)
        self._updated = True

    def _bind(self, name, key_pages, value_pages, dev):
        """The pages as the C struct."""
        bf16, c = _t().bfloat16, self._cache
        if key_pages.dtype is not bf16 or value_pages.dtype is not bf16 or not key_pages.get_device() == value_pages.get_device() == dev:
            _refuse(name, "pages must be tensors of torch.bfloat16 on the current CUDA device")
        if key_pages.shape != self._pages or value_pages.shape != self._pages:
            _refuse(name, f"pages {tuple(key_pages.shape)} and {tuple(value_pages.shape)}, expected {self._pages}", _SHAPE)
        strides = key_pages.stride()
        if strides != value_pages.stride():
            _refuse(name, "key and value pages must have the same strides", _SHAPE)
        if strides[3] != 1:
            _refuse(name, "pages: the last dimension must be contiguous")
        c.key_pages, c.value_pages = key_pages.data_ptr(), value_pages.data_ptr()
        if strides != self._strides:
            self._strides = strides
            c.page_stride, c.head_stride, c.pos_stride = strides[0], strides[1], strides[2]
        return self._cache_ref


def paged_rope_append(q_out, q, k, v, key_pages, value_pages, plan: PagedPlan, inv_freq=None, q_norm_w=None,
                      k_norm_w=None, eps: float = 1e-6, interleaved: bool = False, amplitude: float = 1.0, stream=None):
    """Norms, rotary positions and the write into the pages (q3_paged_rope_append). inv_freq holds
    rope_dim / 2 fp32 frequencies on the device (`rope_inv_freq`); None rotates nothing."""
    name, bf, n, qw, kw = "q3_paged_rope_append", _t().bfloat16, plan.n_tokens, plan.q_width, plan.kv_width
    if not plan._updated:
        _refuse(name, _NO_PLAN)
    dev = _device()
    if plan._on != dev:
        _refuse(name, _ELSEWHERE)
    status = load().q3_paged_rope_append(
        q_out.data_ptr(), _rows(name, q_out, "q_out", n, qw, bf, dev), q.data_ptr(), _rows(name, q, "q", n, qw, bf, dev),
        k.data_ptr(), _rows(name, k, "k", n, kw, bf, dev), v.data_ptr(), _rows(name, v, "v", n, kw, bf, dev),
        _vector(name, q_norm_w, "q_norm_w", plan.head_dim, bf, dev), _vector(name, k_norm_w, "k_norm_w", plan.head_dim, bf, dev),
        eps, _vector(name, inv_freq, "inv_freq", None, _torch.float32, dev), 0 if inv_freq is None else 2 * inv_freq.numel(),
        interleaved, amplitude, plan._bind(name, key_pages, value_pages, dev), plan._shape, plan._ptr, _stream(stream))
    if status:
        check(name, status)


def paged_attention(out, q, key_pages, value_pages, plan: PagedPlan, scale: float | None = None, stream=None):
    """Attention of the step's new tokens over the pages (q3_paged_attention); scale defaults to
    1 / sqrt(head_dim)."""
    name, bf, n, qw = "q3_paged_attention", _t().bfloat16, plan.n_tokens, plan.q_width
    if not plan._updated:
        _refuse(name, _NO_PLAN)
    dev = _device()
    if plan._on != dev:
        _refuse(name, _ELSEWHERE)
    status = load().q3_paged_attention(
        out.data_ptr(), _rows(name, out, "out", n, qw, bf, dev), q.data_ptr(), _rows(name, q, "q", n, qw, bf, dev),
        plan._bind(name, key_pages, value_pages, dev), plan.scale if scale is None else scale, plan._shape, plan._ptr,
        plan._scratch_ptr, _stream(stream))
    if status:
        check(name, status)


def rope_inv_freq(rope_dim: int, theta: float, kind: str = "plain", **scaling) -> tuple[np.ndarray, float]:
    """(fp32 frequencies, amplitude of cos and sin) on the host (q3_rope_inv_freq). kind is 'plain',
    'linear', 'by_parts' or 'yarn'; the other arguments are q3_rope_scaling's fields."""
    if kind not in ROPE_KINDS:
        _refuse("q3_rope_inv_freq", f"unknown kind {kind!r}")
    sc = Q3RopeScaling(kind=ROPE_KINDS[kind], **scaling)
    out = np.zeros(max(rope_dim // 2, 1), np.float32)
    amplitude = ctypes.c_float(0.0)
    call("q3_rope_inv_freq", out.ctypes.data, ctypes.byref(amplitude), rope_dim, theta, ctypes.byref(sc))
    return out, amplitude.value


def logits_process(out, logits, hist_start=None, hist_split=None, hist_ids=None, repetition=None, frequency=None,
                   presence=None, bias_start=None, bias_ids=None, bias=None, mask=None, stream=None):
    """Penalties, biases and grammar masks on [rows, vocab] logits, bf16 or fp32 (q3_logits_process_bounded);
    out may be logits. mask is int32 [rows, >= ceil(vocab / 32)], one bit per allowed token."""
    torch = _t()
    name, dtype, i32, f32 = "q3_logits_process", logits.dtype, torch.int32, torch.float32
    if dtype is not torch.bfloat16 and dtype is not f32:
        _refuse(name, "logits must be bfloat16 or float32")
    shape = logits.shape
    if len(shape) != 2 or out.shape != shape:
        _refuse(name, "logits and out must both be [rows, vocab]", _SHAPE)
    (rows, vocab), dev = shape, _device()
    mask_ptr, mask_stride = None, 0
    if mask is not None:
        if mask.dim() != 2 or mask.shape[1] * 32 < vocab:
            _refuse(name, "mask must be [rows, at least vocab / 32 words]", _SHAPE)
        mask_ptr, mask_stride = mask.data_ptr(), _rows(name, mask, "mask", rows, mask.shape[1], i32, dev)
    hist, history, n_hist = _vector(name, hist_start, "hist_start", rows + 1, i32, dev), None, 0
    if hist_ids is not None:  # an empty tensor has no address to pass; of none, nothing is read at another one
        n_hist = hist_ids.numel()
        history = _vector(name, hist_ids, "hist_ids", None, i32, dev) if n_hist else hist
    bias_at, biased, added, n_bias = _vector(name, bias_start, "bias_start", rows + 1, i32, dev), None, None, 0
    if bias_ids is not None:
        n_bias = bias_ids.numel()
        if bias is not None and bias.numel() != n_bias:
            _refuse(name, "bias and bias_ids differ in length", _SHAPE)
        biased = _vector(name, bias_ids, "bias_ids", None, i32, dev) if n_bias else bias_at
        added = _vector(name, bias, "bias", None, f32, dev) if n_bias else bias_at
    status = load().q3_logits_process_bounded(
        out.data_ptr(), logits.data_ptr(), dtype is f32, rows, vocab, _rows(name, out, "out", rows, vocab, dtype, dev),
        _rows(name, logits, "logits", rows, vocab, dtype, dev), hist, _vector(name, hist_split, "hist_split", rows, i32, dev), history,
        n_hist, _vector(name, repetition, "repetition", rows, f32, dev), _vector(name, frequency, "frequency", rows, f32, dev),
        _vector(name, presence, "presence", rows, f32, dev), bias_at, biased, added, n_bias, mask_ptr, mask_stride, _stream(stream))
    if status:
        check(name, status)


def sample_logits(out, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, draft=None, prob=None, stream=None):
    """The next token of each row of [rows, vocab] logits, bf16 or fp32, from random numbers u in [0, 1) (q3_sample_logits):
    int32 tokens to out and, if given, their fp32 probabilities to prob. temperature, top_p, min_p: fp32, top_k and draft:
    int32, one entry a row, or None. A row's draft token comes out with the probability that the row gives it."""
    torch = _t()
    name, dtype, i32, f32 = "q3_sample_logits", logits.dtype, torch.int32, torch.float32
    if dtype is not torch.bfloat16 and dtype is not f32:
        _refuse(name, "logits must be bfloat16 or float32")
    if logits.dim() != 2:
        _refuse(name, "logits must be [rows, vocab]", _SHAPE)
    (rows, vocab), dev = logits.shape, _device()
    status = load().q3_sample_logits(
        _vector(name, out, "out", rows, i32, dev), _vector(name, prob, "prob", rows, f32, dev), logits.data_ptr(), dtype is f32, rows,
        vocab, _rows(name, logits, "logits", rows, vocab, dtype, dev), _vector(name, u, "u", rows, f32, dev),
        _vector(name, temperature, "temperature", rows, f32, dev), _vector(name, top_k, "top_k", rows, i32, dev),
        _vector(name, top_p, "top_p", rows, f32, dev), _vector(name, min_p, "min_p", rows, f32, dev),
        _vector(name, draft, "draft", rows, i32, dev), _stream(stream))
    if status:
        check(name, status)
