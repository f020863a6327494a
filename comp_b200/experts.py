"""Layers of experts on MXFP4 weights (an extension beyond the reference): routing, the experts' products, and back.

    w_up, w_down = mx.pack(codes, scales), ...             # MXTensors [E][N][K]
    plan = experts.route(logits, 8)                        # logits [T][E] -> 8 experts for each token, sorted by expert
    h = act(experts.linear(x, w_up, plan))                 # x [T][K] -> sorted rows [T * 8][N]
    y = experts.linear(h, w_down, plan, gather=False)      # sorted rows in, sorted rows out
    out = experts.combine(y, plan, plan.weights)           # [T][K]: each token's rows, weighted and added

Nothing synchronizes: how many rows an expert has stays on the device, and all of it can be captured in a CUDA graph. The
kernels are this package's own, through the C-ABI (include/comp_b200.h, where layouts and formulas stand).
"""

import struct

import torch

from . import _lib
from .kv import DTYPE_ID, _dtype_id
from .mx import (FUSED_ROWS, MAX_EXPERTS, STAGE, STAGE_BYTES, TILE_ROWS, MXTensor, _check_out, _cuda, _enter, _few_size,
                 _out_dtype, _rows, _same, _scratch, _stride)

MAX_TOP = 32
_pack_route = struct.Struct(_lib.EXPERTS_ROUTE_ARGS).pack
_pack_linear = struct.Struct(_lib.EXPERTS_LINEAR_ARGS).pack
_pack_combine = struct.Struct(_lib.EXPERTS_COMBINE_ARGS).pack


class Plan:
    """Choices (token * top + j) sorted by expert. int32 tensors: ids [tokens][top] (each choice's expert, -1: none), offsets
    [experts + 1] (the sorted rows where each expert's begin), pos [tokens][top] (each choice's sorted row, -1: it goes nowhere),
    order [tokens * top] (each sorted row's choice, -1 past the last); weights f32 [tokens][top] (from route, else None). All lie in
    one allocation, whose parts are made tensors when they are asked for; ids of a plan from sort are worked out from its other
    parts then (the tensor that sort was given is the caller's, and may hold the next step's)."""

    def __init__(self, tokens, top, experts, like, routed):
        choices = tokens * top
        self.tokens, self.top, self.experts = tokens, top, experts
        words = 2 * (experts + 1) + 4 * choices if tokens <= 128 and choices <= 1024 else \
            _lib.load().b2q_experts_plan_words(tokens, top, experts)
        self._routed = words if routed else 0  # (ids and weights follow the plan's own words)
        self._words = like.new_empty(words + 2 * choices if routed else words, dtype=torch.int32)
        self._at, self._index = self._words.data_ptr(), self._words.get_device()

    def __getstate__(self):
        return {name: v for name, v in self.__dict__.items() if name not in ("_at", "_index")}

    def __setstate__(self, state):  # a copy's words lie elsewhere
        self.__dict__.update(state)
        self._index = _cuda("Plan", self._words)
        self._at = self._words.data_ptr()

    @property
    def device(self):
        return self._words.device

    def _part(self, at, rows=True):
        if rows:
            return self._words.as_strided((self.tokens, self.top), (self.top, 1), at)
        return self._words.as_strided((self.tokens * self.top,), (1,), at)

    @property
    def ids(self):
        if self._routed:
            return self._part(self._routed)
        pos = self.pos  # a choice's expert is the one among whose rows its own lies
        return torch.where(pos < 0, -1, torch.searchsorted(self.offsets[1:], pos, right=True, out_int32=True))

    @property
    def weights(self):
        return self._part(self._routed + self.tokens * self.top).view(torch.float32) if self._routed else None

    @property
    def offsets(self):
        return self._words.as_strided((self.experts + 1,), (1,))

    @property
    def pos(self):
        return self._part(2 * (self.experts + 1))

    @property
    def order(self):
        return self._part(2 * (self.experts + 1) + self.tokens * self.top, rows=False)


def _check_sizes(name, tokens, top, experts):
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"{name}: {experts} experts (1..{MAX_EXPERTS})")
    if not 1 <= top <= MAX_TOP:
        raise ValueError(f"{name}: {top} choices a token (1..{MAX_TOP})")
    if tokens * top > 1 << 26:
        raise ValueError(f"{name}: {tokens} tokens of {top} choices")


def route(logits, top, normalize=True):
    """logits [T][E] (f32, f16 or bf16) -> Plan of the `top` largest of each token: plan.ids (falling; the lowest index first
    among equals) and plan.weights, their softmax over the chosen, or (normalize=False) over all E. -inf and NaN are never
    chosen: a token with fewer others has ids -1, of weight 0, that go nowhere."""
    index = _cuda("route", logits)
    did = DTYPE_ID.get(logits.dtype)
    if did is None:
        _dtype_id("route: logits", logits)
    if logits.dim() != 2:
        raise ValueError(f"route: logits {tuple(logits.shape)}, expected [T][E]")
    if not isinstance(top, int):
        raise TypeError(f"route: top must be a whole number, got {type(top).__name__}")
    tokens, experts = logits.shape
    _check_sizes("route", tokens, top, experts)
    if top > experts:
        raise ValueError(f"route: {top} choices of {experts} experts")
    ld = experts
    if not logits.is_contiguous():
        s0, s1 = logits.stride()
        if (s1 != 1 and experts > 1) or (tokens > 1 and s0 < experts):
            logits = logits.clone(memory_format=torch.contiguous_format)
        ld = _stride(logits)
    plan = Plan(tokens, top, experts, logits, True)
    words = plan._at
    ids = words + 4 * plan._routed
    _enter(index, _lib.load().b2q_experts_route, _pack_route(logits.data_ptr(), ids, ids + 4 * tokens * top, words, ld, tokens,
                                                             experts, top, did, 1 if normalize else 0))
    return plan


def sort(ids, experts):
    """ids int32 [T][top], the experts of each token -> Plan. Negative ids go nowhere (experts held elsewhere, padding); so do
    ids beyond the experts, which set the device error word to 5."""
    index = _cuda("sort", ids)
    if ids.dtype != torch.int32:
        raise TypeError(f"sort: ids dtype {ids.dtype}, expected torch.int32")
    if ids.dim() != 2:
        raise ValueError(f"sort: ids {tuple(ids.shape)}, expected [T][top]")
    if not isinstance(experts, int):
        raise TypeError(f"sort: experts must be a whole number, got {type(experts).__name__}")
    tokens, top = ids.shape
    _check_sizes("sort", tokens, top, experts)
    ids = ids.contiguous()
    plan = Plan(tokens, top, experts, ids, False)
    _enter(index, _lib.load().b2q_experts_sort, ids.data_ptr(), tokens, top, experts, plan._at)
    return plan


def _check_pair(name, plan, w):
    if not isinstance(w, MXTensor):
        raise TypeError(f"{name}: w must be an MXTensor, got {type(w).__name__}")
    if not isinstance(plan, Plan):
        raise TypeError(f"{name}: plan must be a Plan (route, sort), got {type(plan).__name__}")
    if w.experts != plan.experts:
        raise ValueError(f"{name}: w {w.shape}, expected [{plan.experts}][N][K]")


def workspace_size(plan, w, gather=True):
    """Bytes of device workspace that linear(x, w, plan, gather) needs."""
    _check_pair("workspace_size", plan, w)
    return _workspace_size(plan, w, gather)


def _workspace_size(plan, w, gather):
    choices = plan.tokens * plan.top
    if (plan.tokens if gather else choices) <= FUSED_ROWS:
        return _few_size(w, (plan.tokens, plan.top, bool(gather)), "b2q_experts_linear_workspace_size", plan.tokens, plan.top,
                         plan.experts, 1 if gather else 0, w.rows, w.k)
    return (choices // TILE_ROWS + min(plan.experts, choices)) * -(-w.k // STAGE) * STAGE_BYTES


def linear(x, w, plan, gather=True, dtype=None, out=None, workspace=None):
    """Each sorted row, quantized to MXFP4, times its expert's weights w (MXTensor [E][N][K]) -> [T * top][N] of `dtype`
    (default: x's) in sorted order; rows past plan.offsets[E] stay unwritten. x: [T][K], a token's row for each of its choices,
    or with gather=False the sorted rows [T * top][K]. out: the tensor for the result (it shares no memory with x). workspace: a
    CUDA uint8 tensor of workspace_size(plan, w, gather) bytes, 128-byte aligned (allocated here when None)."""
    _check_pair("linear", plan, w)
    index, n, k, tokens, top = w._index, w.rows, w.k, plan.tokens, plan.top
    if plan._index != index:
        raise RuntimeError(f"comp_b200.linear: tensors on different devices ({w.device} and {plan.device})")
    _same("linear", index, x)
    given = x.dtype
    xid = DTYPE_ID.get(given)
    if xid is None:
        _dtype_id("linear: x", x)
    choices = tokens * top
    if x.shape != (tokens if gather else choices, k):
        raise ValueError(f"linear: x {tuple(x.shape)}, expected [{tokens if gather else choices}][{k}]")
    if dtype is None or dtype is given:
        dtype, did = given, xid
    else:
        did = _out_dtype("linear", dtype)
    x, x_at, ldx = _rows(x)
    if out is None:
        out = x.new_empty((choices, n)) if did == xid else x.new_empty((choices, n), dtype=dtype)
        at, ldy = out.data_ptr(), n
    else:
        at, ldy = _check_out("linear", out, dtype, (choices, n), index)
    if workspace is None:
        need = _workspace_size(plan, w, gather)
        workspace = _scratch(index, need, x) if need else None
    else:
        _same("linear", index, workspace)
        if not workspace.is_contiguous():
            raise ValueError("linear: workspace must be contiguous")
        need = workspace.numel() * workspace.element_size()
    _enter(index, _lib.load().b2q_experts_linear,
           _pack_linear(x_at, w._at, plan._at, at, 0 if workspace is None else workspace.data_ptr(), ldx, tokens, top, plan.experts, n,
                        k, ldy, need, xid, did, 1 if gather else 0))
    return out


def combine(y, plan, weights=None, out=None):
    """Sorted rows y [T * top][N] back to their tokens -> [T][N] of y's type: the sum of weights[t][j] (f32 [T][top]; None: 1) times
    y[pos[t][j]], in f32 and in order of j. A choice that goes nowhere adds nothing.
    out: the tensor for the result (it shares no memory with y)."""
    if not isinstance(plan, Plan):
        raise TypeError(f"combine: plan must be a Plan (route, sort), got {type(plan).__name__}")
    index, tokens, top = plan._index, plan.tokens, plan.top
    _same("combine", index, y)
    did = DTYPE_ID.get(y.dtype)
    if did is None:
        _dtype_id("combine: y", y)
    shape, choices = y.shape, tokens * top
    if len(shape) != 2 or shape[0] != choices:
        raise ValueError(f"combine: y {tuple(shape)}, expected [{choices}][N]")
    n = shape[1]
    w_at = 0
    if weights is not None:
        _same("combine", index, weights)
        if weights.dtype is not torch.float32:
            raise TypeError(f"combine: weights dtype {weights.dtype}, expected torch.float32")
        if weights.shape != (tokens, top):
            raise ValueError(f"combine: weights {tuple(weights.shape)}, expected ({tokens}, {top})")
        if not weights.is_contiguous():
            weights = weights.contiguous()
        w_at = weights.data_ptr()
    ldy = n
    if not y.is_contiguous():
        if (n > 1 and y.stride(1) != 1) or (choices > 1 and y.stride(0) < n):
            y = y.clone(memory_format=torch.contiguous_format)
        ldy = _stride(y)
    if out is None:
        out = y.new_empty((tokens, n))
        at, ldo = out.data_ptr(), n
    else:
        at, ldo = _check_out("combine", out, y.dtype, (tokens, n), index)
    _enter(index, _lib.load().b2q_experts_combine,
           _pack_combine(y.data_ptr(), plan._at, w_at, at, ldy, tokens, top, plan.experts, n, ldo, did))
    return out
