"""router.select: routing from logits, against a plain 64-bit implementation.

Which experts are chosen is compared exactly, and so is the order of the pairs.  Weights: an expf (1 ulp), a
few roundings of 2^-24 each and a sum of at most 32 (renormalised) or 37 rounded additions in a row (softmax
over 1024 experts: 32 per lane, then 5); fewer than 64 roundings in all, so within 2^-18 of the value.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import flashmoe_b200 as flashmoe
from flashmoe_b200 import _native as N
from flashmoe_b200 import router
from flashmoe_b200.jit import DataType

gpu = pytest.mark.gpu
TYPES = {torch.bfloat16: DataType.BF16, torch.float16: DataType.FP16, torch.float32: DataType.FP32}
WEIGHT_TOL = 2.0 ** -18


def reference(logits, k, *, score="softmax", bias=None, groups=1, top_groups=None, group_max=False, renormalize=True,
              scale=1.0):
    """numpy, float64, one token at a time."""
    x = logits.double().cpu().numpy().copy()
    x[np.isnan(x)] = -np.inf
    x[x == np.inf] = np.finfo(np.float32).max
    S, E = x.shape
    top_groups = groups if top_groups is None else top_groups
    b = None
    if bias is not None:
        b = bias.double().cpu().numpy().copy()
        b[np.isnan(b)] = -np.inf
        b[b == np.inf] = np.finfo(np.float32).max
    ids = np.zeros((S, k), np.int64)
    w = np.zeros((S, k))
    for t in range(S):
        l = x[t]
        masked = l == -np.inf
        s = np.zeros(E)
        live = ~masked
        if score == "softmax":
            if live.any():
                s[live] = np.exp(l[live] - l[live].max())
                s = s / s.sum()
        else:
            with np.errstate(over="ignore"):
                s[live] = 1.0 / (1.0 + np.exp(-l[live]))
        c = s + (0.0 if b is None else b)
        c[masked] = -np.inf
        alive = np.ones(E, bool)
        if top_groups < groups:
            by = c.reshape(groups, -1)
            two = -np.sort(-by, axis=1)[:, :2]
            g = two[:, 0].copy()
            if not group_max and two.shape[1] == 2:
                g = np.where(two[:, 1] == -np.inf, g, g + two[:, 1])
            kept = sorted(range(groups), key=lambda i: (-g[i], i))[:top_groups]
            alive = np.repeat(np.isin(np.arange(groups), kept), E // groups)
        # without a bias the order is the logits' own (their scores may round to the same value)
        key = l if b is None else c
        ids[t] = sorted(np.nonzero(alive)[0], key=lambda e: (-key[e], e))[:k]
        w[t] = s[ids[t]]
        if renormalize:
            if score == "softmax":   # a share among the chosen: also where all their softmax values underflow
                ll = l[ids[t]]
                w[t] = 0.0 if ll.max() == -np.inf else np.where(ll == -np.inf, 0.0, np.exp(ll - ll.max()))
            total = w[t].sum()
            w[t] = w[t] / total if total > 0 else 0.0
    return ids, w * scale


def order(ids, E):
    flat = ids.reshape(-1)
    counts = np.bincount(flat, minlength=E)
    positions = np.empty(flat.size, np.int64)
    positions[np.argsort(flat, kind="stable")] = np.arange(flat.size)
    return counts, np.concatenate([[0], np.cumsum(counts)]), positions.reshape(ids.shape)


class Outputs:
    def __init__(self, S, E, k):
        new = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device="cuda")
        self.ids, self.counts, self.offsets, self.positions = new(S, k), new(E), new(E + 1), new(S, k)
        self.weights = torch.full((S, k), -7.0, device="cuda")


def args_for(logits, o, k, *, stream=None, score="softmax", bias=None, groups=1, top_groups=None, group_max=False,
             renormalize=True, scale=1.0):
    S, E = logits.shape
    return router.SelectArgs(
        logits.data_ptr(), o.ids.data_ptr(), o.weights.data_ptr(), o.counts.data_ptr(),
        (stream or torch.cuda.current_stream()).cuda_stream, num_tokens=S, num_experts=E, top_k=k,
        data_type=TYPES[logits.dtype], score=router.Score[score.upper()], bias=0 if bias is None else bias.data_ptr(),
        num_groups=groups, top_groups=top_groups,
        group_score=router.GroupScore.MAX if group_max else router.GroupScore.TOP2, renormalize=renormalize, scale=scale,
        offsets=o.offsets.data_ptr(), positions=o.positions.data_ptr())


def check(logits, o, k, **kw):
    ids, w = reference(logits, k, **kw)
    assert np.array_equal(o.ids.cpu().numpy(), ids), "ids"
    got = o.weights.double().cpu().numpy()
    assert np.all(np.abs(got - w) <= WEIGHT_TOL * np.abs(w) + 2.0 ** -140), np.abs(got - w).max()
    counts, offsets, positions = order(ids, logits.shape[1])
    assert np.array_equal(o.counts.cpu().numpy(), counts), "counts"
    assert np.array_equal(o.offsets.cpu().numpy(), offsets), "offsets"
    assert np.array_equal(o.positions.cpu().numpy(), positions), "positions"


def run(logits, k, **kw):
    logits = logits.cuda()
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].cuda()
    o = Outputs(*logits.shape, k)
    router.select(args_for(logits, o, k, **kw))
    torch.cuda.synchronize()
    check(logits, o, k, **kw)
    return o


def normal(S, E, dtype=torch.float32, seed=0, std=1.5):
    return (torch.randn(S, E, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def bias_of(E, seed=1, std=0.05):
    return torch.randn(E, generator=torch.Generator().manual_seed(seed)) * std


@gpu
@pytest.mark.parametrize("dtype", list(TYPES), ids=str)
@pytest.mark.parametrize("S,E,k", [(1, 8, 2), (1, 1, 1), (3, 37, 5), (33, 64, 8), (130, 128, 8), (257, 160, 6), (64, 300, 32),
                                   (40, 1024, 9)])
@pytest.mark.parametrize("score,renormalize,scale", [("softmax", True, 1.0), ("softmax", False, 2.5), ("sigmoid", True, 2.5),
                                                     ("sigmoid", False, 1.0)])
def test_plain_choice(S, E, k, dtype, score, renormalize, scale):
    run(normal(S, E, dtype, S + E), k, score=score, renormalize=renormalize, scale=scale)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("E,k,groups,top_groups", [(256, 8, 8, 4), (96, 5, 3, 2), (160, 6, 5, 1), (1024, 8, 32, 7), (64, 4, 32, 2),
                                                   (32, 8, 32, 8), (40, 3, 4, 4)])
@pytest.mark.parametrize("score,with_bias,group_max", [("sigmoid", True, False), ("softmax", False, True), ("softmax", True, False),
                                                       ("sigmoid", False, False)])
def test_groups_and_bias(E, k, groups, top_groups, dtype, score, with_bias, group_max):
    run(normal(77, E, dtype, E + k), k, score=score, bias=bias_of(E) if with_bias else None, groups=groups,
        top_groups=top_groups, group_max=group_max, scale=2.5)


@gpu
@pytest.mark.parametrize("S", [0, 1, 255, 256, 257, 5003, 16384])
def test_order_of_many_tokens(S):
    """Below and above the pair count from which several CTAs share the ordering; no tokens at all."""
    run(normal(S, 64, torch.bfloat16, S), 8)


@gpu
def test_every_token_chooses_the_same_experts():
    l = torch.zeros(3000, 24)
    l[:, 5], l[:, 17], l[:, 23] = 3.0, 2.0, 2.0
    run(l, 3)


@gpu
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_expert_and_group(score, with_bias):
    g = torch.Generator().manual_seed(5)
    l = torch.randint(-2, 3, (200, 64), generator=g).float()
    l[0] = 0.0
    l[1] = -0.0
    l[1, ::2] = 0.0
    b = torch.randint(-1, 2, (64,), generator=g).float() * 0.25 if with_bias else None
    run(l, 8, score=score, bias=b)
    run(l, 8, score=score, bias=b, groups=8, top_groups=3)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_that_fp32_cannot_tell_apart(score):
    """Biases that all but cancel the scores' differences: what is left is around 1e-9, in either
    direction.  Differences of the 64-bit implementations themselves are around 1e-16."""
    S, E = 64, 48
    l = normal(1, E, seed=3).repeat(S, 1)
    s = torch.softmax(l[0].double(), 0) if score == "softmax" else torch.sigmoid(l[0].double())
    b = (0.5 - s).float()                       # rounding of b leaves up to 2^-26 of difference
    run(l, 8, score=score, bias=b)
    run(l, 8, score=score, bias=b, groups=6, top_groups=3)
    assert len(set((s + b.double()).tolist())) == E


@gpu
def test_groups_whose_large_scores_cancel():
    """Two experts a group with biases of +-100: what their sums differ by, steps of 2^-17, is what fp32 loses when the
    scores are added to the biases (half a step of 2^-17 each)."""
    g = torch.Generator().manual_seed(3)
    bias = torch.empty(32, 2)
    bias[:, 0] = 100.0 + torch.randint(0, 64, (32,), generator=g) * 2.0 ** -17
    bias[:, 1] = -bias[:, 0] + torch.randperm(32, generator=g) * 2.0 ** -17
    run(normal(64, 64, seed=8, std=1e-4), 4, score="sigmoid", bias=bias.view(-1), groups=32, top_groups=5)
    run(torch.zeros(3, 64), 2, score="sigmoid", bias=bias.view(-1), groups=32, top_groups=1)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_masks_infinities_and_nan(score, with_bias, groups, top_groups):
    E, k = 32, 6
    l = normal(12, E, seed=9)
    l[0] = -math.inf                            # nothing left
    l[1, 3:] = -math.inf                        # fewer left than chosen
    l[2] = math.nan
    l[3, ::3] = math.nan
    l[4, 7] = math.inf
    l[5, [2, 30]] = math.inf
    l[6] = torch.finfo(torch.float32).min       # a mask by the type's lowest value, everywhere
    l[7, 1:] = torch.finfo(torch.float32).min
    l[8] = -200.0 + l[8]                        # sigmoids below fp32's range
    l[9, :16] = -math.inf
    l[10] = 80.0 + l[10]
    bias = bias_of(E, std=1.0) if with_bias else None
    if with_bias:
        bias[4], bias[9], bias[20] = -math.inf, math.nan, 5.0
        # sigmoids of one value that differ in 64 bits only behind fp32's smallest number: keep them apart
        l = torch.cat([l[:8], l[9:10]])
    elif score == "sigmoid":
        l = torch.cat([l[:8], l[9:10]])         # (at +-200 and 80 the scores' sums tie in 64 bits as well)
    run(l, k, score=score, bias=bias, groups=groups, top_groups=top_groups)


@gpu
def test_softmax_far_apart_is_renormalised_among_the_chosen():
    """The chosen groups lie 150 below the best expert: their softmax values underflow, their shares do not."""
    l = torch.full((4, 16), -150.0) + normal(4, 16, seed=2)
    l[:, 0] = 0.0                               # group 0's best, alone: 1 + tiny < the pairs of no group
    b = torch.zeros(16)
    b[0:4] = -2.0                               # ... and its group is not chosen
    run(l, 2, bias=b, groups=4, top_groups=1)


@gpu
def test_a_call_can_be_captured_and_replayed_on_another_stream():
    S, E, k = 700, 128, 8
    l = normal(S, E).cuda()
    o = Outputs(S, E, k)
    stream = torch.cuda.Stream()
    args = args_for(l, o, k, stream=stream)
    router.select(args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        router.select(args)
    for seed in (1, 2):
        l.copy_(normal(S, E, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        check(l, o, k)


@gpu
def test_outputs_that_are_not_asked_for_are_optional():
    l = normal(50, 16).cuda()
    o = Outputs(50, 16, 2)
    a = args_for(l, o, 2)
    a.c.offsets = a.c.positions = None
    router.select(a)
    torch.cuda.synchronize()
    ids, _ = reference(l, 2)
    assert np.array_equal(o.ids.cpu().numpy(), ids)
    assert np.array_equal(o.counts.cpu().numpy(), np.bincount(ids.reshape(-1), minlength=16))
    assert bool((o.offsets == -7).all()) and bool((o.positions == -7).all())


@gpu
@pytest.mark.parametrize("capacity", [None, 24])
def test_the_bf16_layer_runs_on_the_choice(capacity):
    """select with a context, then the fused forward: the layer's output for this choice (dropped pairs
    included), within the 2e-2 of the layer's own parity tests."""
    from flashmoe_b200.layer import MoELayer
    from flashmoe_b200.workloads import Workload, make_tokens, make_weights
    from helpers import assert_close, oracle_weights
    from oracle import moe_oracle as O
    w = Workload("select", 192, 256, 384, 16, 3, seed=21, capacity=capacity)
    lw, x = make_weights(w), make_tokens(w)
    logits = (x.float() @ lw.router.float().t()).cuda()
    bias = bias_of(16).cuda()
    kw = dict(score="sigmoid", bias=bias, groups=4, top_groups=2, scale=2.5)
    o = Outputs(192, 16, 3)
    layer = MoELayer(w, lw)
    try:
        layer.tokens.copy_(x)
        torch.cuda.synchronize()
        a = args_for(logits, o, 3, stream=layer.stream, **kw)
        a.c.expert_counts = layer.counts.data_ptr()
        router.select(a, layer.handle)
        layer.experts()
        layer.check()
        out = layer.out.clone()
        o.counts = layer.counts.clone()
    finally:
        layer.close()
    check(logits, o, 3, **kw)
    ids, weights = reference(logits, 3, **kw)
    counts, offsets, positions = order(ids, 16)
    ec = w.expert_peer_capacity
    slots = positions - offsets[ids]
    tok, wt = np.zeros((16, 192), np.int64), np.zeros((16, 192), np.float32)
    tok[ids, slots], wt[ids, slots] = np.arange(192)[:, None], weights
    fields = dict(counts=counts, table_tok=tok, table_w=wt, topk_idx=ids, topk_slot=slots, topk_w=weights.astype(np.float32))
    r = type("Choice", (), fields)()
    ref = O.moe_forward(x, r, oracle_weights(lw), 3, ec, int(w.mlp_type), int(w.act_type))
    assert_close(out.cpu(), ref, 0, "select + forward")


# ---- refusals (no GPU is touched) ------------------------------------------------------------------

def _args(**kw):
    a = dict(logits=64, ids=64, weights=64, expert_counts=64, num_tokens=4, num_experts=16, top_k=2)
    a.update(kw)
    pos = [a.pop(n) for n in ("logits", "ids", "weights", "expert_counts")]
    return router.SelectArgs(*pos, 0, **a)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(num_tokens=-1), 1, "num_tokens"), (dict(num_experts=0), 1, "num_experts"), (dict(num_experts=1025), 1, "1024"),
    (dict(top_k=0), 1, "top_k"), (dict(top_k=17), 1, "top_k"), (dict(num_experts=64, top_k=33), 1, "top_k"),
    (dict(num_groups=3), 1, "num_groups"), (dict(num_groups=0, top_groups=1), 1, "num_groups"),
    (dict(num_experts=64, num_groups=64), 1, "num_groups"), (dict(num_groups=4, top_groups=5), 1, "top_groups"),
    (dict(num_groups=4, top_groups=0), 1, "top_groups"), (dict(num_groups=8, top_groups=1, top_k=3), 1, "top_k"),
    (dict(data_type=DataType.FP64), 2, "logits"), (dict(score=2), 1, "score"), (dict(group_score=2), 1, "group_score"),
    (dict(logits=0), 1, "required"), (dict(ids=0), 1, "required"), (dict(expert_counts=0), 1, "required"),
    (dict(logits=66), 1, "aligned"), (dict(positions=2), 1, "aligned"), (dict(bias=1), 1, "aligned"),
    (dict(device_id=-1), 1, "device_id"), (dict(device_id=64), 1, "device_id"),
    (dict(num_tokens=1 << 30), 2, "32 bits"),
])
def test_refusals(kw, code, needle):
    with pytest.raises(flashmoe.FlashMoEError, match=needle) as e:
        router.select(_args(**kw))
    assert e.value.code == code


def test_null_arguments_are_refused():
    assert N.lib().fmoe_router_select(None, None, None) == 1
    assert C.sizeof(N.SelectArgsC) == 7 * 8 + 9 * 4 + 4 + 4 + 4   # the header's fields, and the padding behind them


@gpu
def test_a_context_of_another_shape_is_refused():
    from flashmoe_b200.layer import MoELayer
    from flashmoe_b200.workloads import Workload, make_weights
    w = Workload("select", 64, 64, 64, 8, 2, seed=2)
    layer = MoELayer(w, make_weights(w))
    try:
        l = normal(64, 16).cuda()
        o = Outputs(64, 16, 2)
        with pytest.raises(flashmoe.FlashMoEError, match="context"):
            router.select(args_for(l, o, 2, stream=layer.stream), layer.handle)
    finally:
        layer.close()
