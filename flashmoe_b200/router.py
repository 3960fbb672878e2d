"""Router API: `initialize`, `RouterForwardArgs`, `forward`, `finalize`
(mirrors the reference's flashmoe/router.py:3-45)."""
from __future__ import annotations

import ctypes as C
from enum import IntEnum
from typing import Optional

from . import _native as N
from .jit import ContextHandle, DataType, InitArgs, _get_compiled


class _RouterModule:
    """Stands where the reference's JIT-built gate module stands (bindings.py:300-315)."""

    def __init__(self, lib, desc: N.ModelDesc, return_logits: bool):
        self._lib, self._desc, self._return_logits = lib, desc, return_logits

    def initialize(self, device_id: int, stream_ptr: int) -> int:
        ctx = C.c_void_p()
        N.check(self._lib.fmoe_router_create(C.byref(self._desc), device_id, int(self._return_logits),
                                             C.c_void_p(stream_ptr), C.byref(ctx)), "router.initialize")
        return ctx.value

    def forward(self, raw_ctx: int, tokens: int, weights: int, routing: int, expert_counts: int,
                token_indices: int, stream_ptr: int, *, moe_ctx: int, logit_bias: int = 0) -> None:
        args = N.RouterArgsC(tokens, weights, routing or None, expert_counts, logit_bias or None)
        N.check(self._lib.fmoe_router_forward(C.c_void_p(raw_ctx), C.c_void_p(moe_ctx), C.byref(args),
                                              C.c_void_p(stream_ptr)), "router.forward")

    def finalize(self, raw_ctx: int, stream_ptr: int) -> None:
        N.check(self._lib.fmoe_router_destroy(C.c_void_p(raw_ctx), C.c_void_p(stream_ptr)), "router.finalize")


def initialize(arg: InitArgs, return_logits: bool = False) -> ContextHandle:
    from . import _model_desc
    lib = _get_compiled(arg)
    mod = _RouterModule(lib, _model_desc(arg), return_logits)
    return ContextHandle(mod, mod.initialize(device_id=arg.device_id, stream_ptr=arg.stream_ptr))


class RouterForwardArgs:
    """Device addresses: tokens [S, H], weights stored [E, H], expert_counts [E] int32,
    routing [S, E] fp32 (only with return_logits).  `logit_bias` ([E] fp32, added to the logits
    before the softmax) is an addition of this package; 0 = none."""

    def __init__(self, tokens: int, weights: int, expert_counts: int, stream_ptr: int, *,
                 routing: int = 0, logit_bias: int = 0):
        self.tokens = tokens
        self.weights = weights
        self.routing = routing
        self.expert_counts = expert_counts
        self.stream_ptr = stream_ptr
        self.logit_bias = logit_bias


def forward(router_handle: ContextHandle, flash_handle: ContextHandle, arg: RouterForwardArgs) -> None:
    """Fills `expert_counts` and the routing table inside `flash_handle` (router.py:37-44)."""
    router_handle.mod.forward(router_handle.context,
                              tokens=arg.tokens, weights=arg.weights, routing=arg.routing,
                              expert_counts=arg.expert_counts, stream_ptr=arg.stream_ptr,
                              token_indices=flash_handle.mod.get_tIdx(flash_handle.context),
                              moe_ctx=flash_handle.context, logit_bias=arg.logit_bias)


def finalize(handle: ContextHandle, stream_ptr: int) -> None:
    handle.mod.finalize(handle.context, stream_ptr)


# ---- routing from logits (an addition of this package) ------------------------------------------

class Score(IntEnum):
    """What a logit becomes."""
    SOFTMAX = 0
    SIGMOID = 1


class GroupScore(IntEnum):
    """What a group of experts is ranked by: the sum of its two largest scores, or its largest."""
    TOP2 = 0
    MAX = 1


class SelectArgs:
    """Arguments of `select`.  Device addresses: logits [S, E] of `data_type` (BF16, FP16 or FP32);
    out: ids [S, k] int32 (descending by score, ties to the lower id), weights [S, k] fp32,
    expert_counts [E] int32, and, where not 0, offsets [E + 1] int32 (their exclusive sums) and
    positions [S, k] int32 (the row of every pair when the pairs are ordered by expert).

    `bias` ([E] fp32, 0 = none) is added to the scores for the choice only.  With `num_groups` > 1 the
    experts fall into that many equal runs, of which the `top_groups` best stay.  The weights are the
    chosen experts' scores, divided by their sum if `renormalize`, times `scale`.  A logit or bias of
    -infinity or NaN masks its expert.  Everything lives on `device_id`."""

    def __init__(self, logits: int, ids: int, weights: int, expert_counts: int, stream_ptr: int, *,
                 num_tokens: int, num_experts: int, top_k: int, data_type: DataType = DataType.FP32,
                 score: Score = Score.SOFTMAX, bias: int = 0, num_groups: int = 1,
                 top_groups: Optional[int] = None, group_score: GroupScore = GroupScore.TOP2,
                 renormalize: bool = True, scale: float = 1.0, offsets: int = 0, positions: int = 0,
                 device_id: int = 0):
        self.stream_ptr = stream_ptr
        self.c = N.SelectArgsC(logits or None, bias or None, ids or None, weights or None, expert_counts or None,
                               offsets or None, positions or None, num_tokens, num_experts, top_k, int(data_type),
                               int(score), num_groups, num_groups if top_groups is None else top_groups,
                               int(group_score), int(renormalize), scale, device_id)


def select(arg: SelectArgs, flash_handle: Optional[ContextHandle] = None) -> None:
    """Choose experts from logits on `arg.stream_ptr` (fmoe_router_select): softmax or sigmoid scores, a
    bias for the choice, groups, renormalised or scaled weights.  With `flash_handle` the context's
    routing table is filled as well, as `router.forward` does, so that `forward(flash_handle, ...)` on
    the same stream runs on this choice."""
    N.check(N.lib().fmoe_router_select(flash_handle.context if flash_handle is not None else None, arg.c,
                                       arg.stream_ptr), "router.select")
