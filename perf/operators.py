"""What the routing and 8-bit operators are measured on: their plain forms, and the calls a program makes.

Four operators of a mixture-of-experts layer:

* "select"   -- `flashmoe_b200.router.select`: from logits to the chosen experts, their weights, and the order of the
                (token, choice) pairs by expert;
* "quantize" -- `flashmoe_b200.fp8.quantize`: e4m3 codes with one fp32 scale per 128 values of a row (activations) or per
                128 x 128 block (weights);
* "matmul"   -- `flashmoe_b200.fp8.matmul`: the product of two such operands, dense or with one weight matrix per expert;
* "experts"  -- `flashmoe_b200.fp8.experts`: the gated expert layer on 8-bit weights, from tokens to combined rows.

A state holds the inputs and, where the framework's own calls are measured, its argument objects, output buffers and
workspace: what a program makes once per layer and batch shape.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
BLOCK = 128


def listed():
    return [
        # one token of a 128-expert model: the latency of a decode step's routing
        dict(name="select-1x128", op="select", tokens=1, experts=128, top_k=8, type="bf16", score="softmax", bias=False,
             groups=1, top_groups=1, renormalize=True, scale=1.0),
        # 256 experts in 8 groups of which 4 stay, sigmoid scores, a balance bias: one rank's prefill chunk
        dict(name="select-2048x256-groups", op="select", tokens=2048, experts=256, top_k=8, type="fp32", score="sigmoid",
             bias=True, groups=8, top_groups=4, renormalize=True, scale=2.5),
        # the largest step of the 128-expert sweep
        dict(name="select-8192x128", op="select", tokens=8192, experts=128, top_k=8, type="fp32", score="softmax",
             bias=False, groups=1, top_groups=1, renormalize=True, scale=1.0),
        # a decode batch of activations, one row more than a power of two
        dict(name="quantize-rows-33x2048", op="quantize", rows=33, cols=2048, type="bf16", block_rows=1, matrices=1),
        # a prefill chunk of activations
        dict(name="quantize-rows-8192x5120", op="quantize", rows=8192, cols=5120, type="bf16", block_rows=1, matrices=1),
        # eight experts' matrices as they are loaded, in blocks, with ragged edges
        dict(name="quantize-weights-8x1400x2064", op="quantize", rows=1400, cols=2064, type="bf16", block_rows=128,
             matrices=8),
        # one token through one projection: reading the weights is all there is
        dict(name="matmul-1x8192x5120", op="matmul", m=1, n=8192, k=5120, type="bf16", experts=1),
        # a ragged batch through an odd projection
        dict(name="matmul-777x2500x2064", op="matmul", m=777, n=2500, k=2064, type="fp16", experts=1),
        # a prefill chunk through a wide projection
        dict(name="matmul-4096x14336x4096", op="matmul", m=4096, n=14336, k=4096, type="bf16", experts=1),
        # one token of the 128-expert model through its eight experts
        dict(name="experts-1x128", op="experts", tokens=1, hidden=2048, ffn=768, experts=128, top_k=8, type="bf16"),
        # a prefill chunk of the same model: 64 rows an expert, bound by reading the weights
        dict(name="experts-1024x128", op="experts", tokens=1024, hidden=2048, ffn=768, experts=128, top_k=8, type="bf16"),
        # a prefill chunk of an 8-expert model: bound by the tensor cores
        dict(name="experts-4096x8", op="experts", tokens=4096, hidden=4096, ffn=14336, experts=8, top_k=2, type="bf16"),
    ]


def _log(rng, low, high, step=1):
    """A whole number between low and high, even over the logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["select", "quantize", "matmul", "experts"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op == "select":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        experts = groups * rng.randint(max(2, 8 // groups), max(4, 512 // groups // rng.choice([1, 2, 4])))
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, top_groups * (experts // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        return dict(op=op, tokens=_log(rng, 1, 8192), experts=experts, top_k=top_k, type=kind, score=score,
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, renormalize=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]))
    if op == "quantize":
        if rng.random() < 0.5:
            return dict(op=op, rows=_log(rng, 1, 8192), cols=_log(rng, 16, 8192, 16), type=kind, block_rows=1, matrices=1)
        return dict(op=op, rows=_log(rng, 16, 2048), cols=_log(rng, 16, 4096, 16), type=kind, block_rows=128,
                    matrices=rng.randint(1, 8))
    if op == "matmul":
        if rng.random() < 0.5:
            return dict(op=op, m=_log(rng, 1, 4096), n=_log(rng, 16, 8192), k=_log(rng, 16, 8192, 16), type=kind, experts=1)
        return dict(op=op, m=_log(rng, 1, 8192), n=_log(rng, 16, 4096), k=_log(rng, 16, 4096, 16), type=kind,
                    experts=rng.randint(2, 32))
    # (the layer is one of 16-bit models: its inner activations are rounded to 8 bits)
    hidden, ffn = _log(rng, 64, 4096, 16), _log(rng, 64, 4096, 16)
    experts = 8 * rng.randint(1, max(1, min(16, (8 * 4096 * 14336) // (8 * hidden * ffn))))
    return dict(op=op, tokens=_log(rng, 1, 2048), hidden=hidden, ffn=ffn, experts=experts, top_k=rng.randint(1, 8),
                type=rng.choice(["bf16", "fp16"]))


# ---- inputs ----------------------------------------------------------------------------------

def _normal(shape, gen, std=1.0, dtype=torch.float32):
    x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)
    return x.to(dtype)


def _activations(rows, cols, gen, dtype):
    """Rows as they come out of a norm: unit normal, a few channels ten times as large."""
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.005
    return (_normal((rows, cols), gen) * torch.where(loud, 10.0, 1.0)).to(dtype)


def _weights(matrices, rows, cols, gen, dtype=torch.float32):
    """Quantised weights [matrices, rows, cols] and their block scales; made one matrix at a time to keep the peak low."""
    q = torch.empty(matrices, rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(matrices, -(-rows // BLOCK), -(-cols // BLOCK), device="cuda")
    for i in range(matrices):
        q[i], s[i] = _quantize(_normal((rows, cols), gen, 0.02), BLOCK)
    return q, s


def _choice(tokens, experts, top_k, gen):
    """A routing decision with some experts more popular than others."""
    logits = _normal((tokens, experts), gen) + 0.5 * _normal((experts,), gen)
    ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top_k]
    w = torch.softmax(torch.gather(logits, 1, ids), dim=1)
    counts, offsets, positions = _order(ids, experts)
    return ids.int(), w.contiguous(), counts, offsets, positions


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dt = case["op"], TYPES[case["type"]]
    s = dict(case=case)
    if op == "select":
        s["logits"] = _normal((case["tokens"], case["experts"]), gen, 1.5, dt)
        s["bias"] = _normal((case["experts"],), gen, 0.05) if case["bias"] else None
    elif op == "quantize":
        shape = (case["matrices"], case["rows"], case["cols"])
        if case["block_rows"] == 1:
            s["x"] = _activations(shape[1], shape[2], gen, dt)[None]
        else:
            s["x"] = _normal(shape, gen, 0.02, dt)
    elif op == "matmul":
        s["a"], s["a_scale"] = _quantize(_activations(case["m"], case["k"], gen, torch.bfloat16), 1)
        s["w"], s["w_scale"] = _weights(case["experts"], case["n"], case["k"], gen)
        s["offsets"] = None
        if case["experts"] > 1:
            first = torch.randint(case["experts"], (case["m"], 1), generator=gen, device="cuda")
            s["offsets"] = _order(first, case["experts"])[1]
            s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())   # a plain batched product needs it on the host
    else:
        s["x"] = _activations(case["tokens"], case["hidden"], gen, dt)
        s["ids"], s["weights"], s["counts"], s["offsets"], s["positions"] = _choice(
            case["tokens"], case["experts"], case["top_k"], gen)
        s["most"] = int(s["counts"].max())
        s["up"], s["up_scale"] = _weights(case["experts"], case["ffn"], case["hidden"], gen)
        s["up_v"], s["up_v_scale"] = _weights(case["experts"], case["ffn"], case["hidden"], gen)
        s["down"], s["down_scale"] = _weights(case["experts"], case["hidden"], case["ffn"], gen)
    if own:
        _arguments(s)
    return s


# ---- the framework's calls ---------------------------------------------------------------------

def _arguments(s):
    """Output buffers, workspace and argument objects: made once, as a layer does."""
    import flashmoe_b200 as flashmoe
    case = s["case"]
    op, dt = case["op"], getattr(flashmoe.DataType, case["type"].upper())
    stream, dev = torch.cuda.current_stream().cuda_stream, torch.cuda.current_device()
    at = lambda t: 0 if t is None else t.data_ptr()
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="cuda")
    if op == "select":
        S, E, k = case["tokens"], case["experts"], case["top_k"]
        o = s["out"] = dict(ids=new(S, k, dtype=torch.int32), weights=new(S, k), counts=new(E, dtype=torch.int32),
                            offsets=new(E + 1, dtype=torch.int32), positions=new(S, k, dtype=torch.int32))
        s["args"] = flashmoe.router.SelectArgs(
            logits=at(s["logits"]), ids=at(o["ids"]), weights=at(o["weights"]), expert_counts=at(o["counts"]),
            stream_ptr=stream, num_tokens=S, num_experts=E, top_k=k, data_type=dt,
            score=getattr(flashmoe.router.Score, case["score"].upper()), bias=at(s["bias"]), num_groups=case["groups"],
            top_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"],
            offsets=at(o["offsets"]), positions=at(o["positions"]), device_id=dev)
    elif op == "quantize":
        B, R, C = s["x"].shape
        br = case["block_rows"]
        o = s["out"] = dict(q=new(B, R, C, dtype=torch.float8_e4m3fn), scale=new(B, -(-R // br), -(-C // BLOCK)))
        s["args"] = flashmoe.fp8.QuantizeArgs(
            x=at(s["x"]), q=at(o["q"]), scale=at(o["scale"]), stream_ptr=stream, rows=R, cols=C, data_type=dt,
            block_rows=br, num_matrices=B, device_id=dev)
    elif op == "matmul":
        o = s["out"] = dict(out=new(case["m"], case["n"], dtype=TYPES[case["type"]]))
        s["args"] = flashmoe.fp8.MatmulArgs(
            a=at(s["a"]), a_scale=at(s["a_scale"]), w=at(s["w"]), w_scale=at(s["w_scale"]), out=at(o["out"]),
            stream_ptr=stream, m=case["m"], n=case["n"], k=case["k"], data_type=dt, num_experts=case["experts"],
            offsets=at(s["offsets"]), device_id=dev)
    else:
        S, H, I, E, k = (case[n] for n in ("tokens", "hidden", "ffn", "experts", "top_k"))
        o = s["out"] = dict(out=new(S, H, dtype=TYPES[case["type"]]))
        size = flashmoe.fp8.get_workspace_bytes(num_tokens=S, token_dim=H, ffn_size=I, num_experts=E, top_k=k, data_type=dt)
        s["workspace"] = new(size, dtype=torch.uint8)
        s["args"] = flashmoe.fp8.ExpertsArgs(
            tokens=at(s["x"]), offsets=at(s["offsets"]), positions=at(s["positions"]), weights=at(s["weights"]),
            up=at(s["up"]), up_scale=at(s["up_scale"]), up_v=at(s["up_v"]), up_v_scale=at(s["up_v_scale"]),
            down=at(s["down"]), down_scale=at(s["down_scale"]), out=at(o["out"]), workspace=at(s["workspace"]),
            workspace_bytes=size, stream_ptr=stream, num_tokens=S, token_dim=H, ffn_size=I, num_experts=E, top_k=k,
            data_type=dt, device_id=dev)


def _run_own(s):
    from flashmoe_b200 import fp8, router
    call = dict(select=router.select, quantize=fp8.quantize, matmul=fp8.matmul, experts=fp8.experts)[s["case"]["op"]]
    call(s["args"])
    return s["out"]


# ---- the plain forms ---------------------------------------------------------------------------

def _order(ids, experts):
    """counts [E], offsets [E + 1], positions [S, k]: the pairs by expert, tokens ascending within one."""
    flat = ids.reshape(-1).long()
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0, dtype=torch.int32)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0, dtype=torch.int32)])
    by_expert = torch.sort(flat, stable=True)[1]
    positions = torch.empty_like(flat, dtype=torch.int32)
    positions[by_expert] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    return counts, offsets, positions.view(ids.shape)


def _select(s):
    """In 64 bits: which expert is chosen hangs on the last bits of scores that are close."""
    c = s["case"]
    l = s["logits"].double()
    if c["score"] == "softmax":
        e = torch.exp(l - l.max(dim=1, keepdim=True)[0])
        score = e / e.sum(dim=1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    key = score if s["bias"] is None else score + s["bias"].double()
    if c["groups"] > 1:
        by_group = key.view(c["tokens"], c["groups"], -1)
        group = torch.sort(by_group, dim=2, descending=True)[0][:, :, :2].sum(dim=2)
        kept = torch.sort(group, dim=1, descending=True, stable=True)[1][:, :c["top_groups"]]
        out = torch.ones_like(group, dtype=torch.bool)
        out[torch.arange(c["tokens"], device=l.device)[:, None], kept] = False
        key = by_group.masked_fill(out[:, :, None], -math.inf).view_as(key)
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :c["top_k"]]
    w = torch.gather(score, 1, ids)
    if c["renormalize"]:
        w = w / w.sum(dim=1, keepdim=True)
    counts, offsets, positions = _order(ids, c["experts"])
    return dict(ids=ids.int(), weights=(w * c["scale"]).float(), counts=counts, offsets=offsets, positions=positions)


def _blocks(x, block_rows):
    """[..., R, C] in fp32, padded with zeros to whole blocks: [..., R / block_rows, block_rows, C / 128, 128]."""
    R, C = x.shape[-2:]
    pad = torch.nn.functional.pad(x, (0, -C % BLOCK, 0, -R % block_rows))
    return pad.reshape(*x.shape[:-2], pad.shape[-2] // block_rows, block_rows, pad.shape[-1] // BLOCK, BLOCK)


def _quantize(x, block_rows):
    x = x.float()
    R, C = x.shape[-2:]
    b = _blocks(x, block_rows)
    amax = b.abs().amax(dim=(-3, -1), keepdim=True)
    q = torch.where(amax > 0, b * E4M3_MAX / amax, torch.zeros_like(b)).to(torch.float8_e4m3fn)
    q = q.view(torch.uint8).reshape(*x.shape[:-2], b.shape[-4] * block_rows, -1)[..., :R, :C].contiguous()
    scale = amax / torch.full_like(amax, E4M3_MAX)
    return q.view(torch.float8_e4m3fn), scale.squeeze(-1).squeeze(-2).contiguous()


def _values(q, scale, block_rows, dtype=torch.float32):
    """What codes and scales stand for."""
    R, C = q.shape[-2:]
    each = scale.to(dtype).repeat_interleave(block_rows, dim=-2)[..., :R, :].repeat_interleave(BLOCK, dim=-1)[..., :C]
    return q.to(dtype) * each


def _by_expert(rows, offsets, most, w):
    """rows [M, K] in expert order times w [E, N, K] transposed, as one padded batched product."""
    i = torch.arange(most, device=rows.device)
    at = offsets[:-1, None].long() + i
    here = i < (offsets[1:] - offsets[:-1])[:, None]
    padded = rows[at.clamp(max=rows.shape[0] - 1)]
    return torch.bmm(padded, w.transpose(1, 2))[here]


def _matmul(s):
    a, w = _values(s["a"], s["a_scale"], 1), _values(s["w"], s["w_scale"], BLOCK)
    out = a @ w[0].t() if s["offsets"] is None else _by_expert(a, s["offsets"], s["most"], w)
    return dict(out=out.to(TYPES[s["case"]["type"]]))


def _experts(s):
    c = s["case"]
    pairs = c["tokens"] * c["top_k"]
    q, scale = _quantize(s["x"], 1)
    token = torch.empty(pairs, dtype=torch.long, device="cuda")
    token[s["positions"].view(-1).long()] = torch.arange(pairs, device="cuda") // c["top_k"]
    rows = _values(q, scale, 1)[token]
    gate = _by_expert(rows, s["offsets"], s["most"], _values(s["up"], s["up_scale"], BLOCK))
    up = _by_expert(rows, s["offsets"], s["most"], _values(s["up_v"], s["up_v_scale"], BLOCK))
    h = _values(*_quantize(gate / (1.0 + torch.exp(-gate)) * up, 1), 1)
    y = _by_expert(h, s["offsets"], s["most"], _values(s["down"], s["down_scale"], BLOCK))
    y = y[s["positions"].long()]
    return dict(out=(y * s["weights"][:, :, None]).sum(dim=1).to(TYPES[c["type"]]))


def _run_plain(s):
    op = s["case"]["op"]
    if op == "quantize":
        return dict(zip(("q", "scale"), _quantize(s["x"], s["case"]["block_rows"])))
    return dict(select=_select, matmul=_matmul, experts=_experts)[op](s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op, eb = case["op"], 4 if case["type"] == "fp32" else 2
    up = lambda v: -(-v // BLOCK)
    if op == "select":
        S, E, k = case["tokens"], case["experts"], case["top_k"]
        return dict(bytes=S * E * eb + (4 * E if case["bias"] else 0) + 12 * S * k + 8 * E + 4, flops=10 * S * E)
    if op == "quantize":
        B, R, C, br = case["matrices"], case["rows"], case["cols"], case["block_rows"]
        return dict(bytes=B * (R * C * (eb + 1) + 4 * -(-R // br) * up(C)), flops=3 * B * R * C)
    if op == "matmul":
        m, n, k, E = case["m"], case["n"], case["k"], case["experts"]
        # of many experts only those that some row chose: m independent choices
        hit = E * (1 - (1 - 1 / E) ** m)
        return dict(bytes=m * k + 4 * m * up(k) + hit * (n * k + 4 * up(n) * up(k)) + m * n * eb, flops=2 * m * n * k)
    S, H, I, E, k = (case[n] for n in ("tokens", "hidden", "ffn", "experts", "top_k"))
    hit = E * (1 - (1 - k / E) ** S)
    return dict(bytes=2 * S * H * eb + 8 * S * k + hit * 3 * (H * I + 4 * up(H) * up(I)), flops=6 * S * k * H * I)


# ---- the definitions in 64 bits ------------------------------------------------------------------------

def _round_e4m3(v):
    """v in 64 bits to the nearest e4m3 value, ties to even: 3 mantissa bits, exponents from 2^-6, subnormals below."""
    exponent = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -30))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3.0)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _quantize64(x, block_rows):
    """Codes' values and scales of a matrix, from amax by index instead of by padded blocks."""
    x = x.double()
    R, C = x.shape
    row = torch.div(torch.arange(R, device=x.device), block_rows, rounding_mode="floor")
    col = torch.div(torch.arange(C, device=x.device), BLOCK, rounding_mode="floor")
    cols = int(col[-1]) + 1
    block = row[:, None] * cols + col
    amax = torch.zeros((int(row[-1]) + 1) * cols, dtype=x.dtype, device=x.device)
    amax.scatter_reduce_(0, block.reshape(-1), x.abs().reshape(-1), "amax")
    each = amax[block]
    # (times 448 first: it is exact, and the quotient then falls on a midpoint of two codes only where it truly does)
    return _round_e4m3(torch.where(each > 0, x * E4M3_MAX / each, 0.0)), (amax / E4M3_MAX).view(-1, cols)


def _values64(q, scale, block_rows):
    R, C = q.shape
    row = torch.div(torch.arange(R, device=q.device), block_rows, rounding_mode="floor")
    col = torch.div(torch.arange(C, device=q.device), BLOCK, rounding_mode="floor")
    return q.double() * scale.double()[row][:, col]


def _select64(s):
    """An expert's place is the number of experts that come before it; nothing is sorted."""
    c = s["case"]
    x = s["logits"].double()
    score = torch.softmax(x, dim=1) if c["score"] == "softmax" else torch.sigmoid(x)
    key = score + (0.0 if s["bias"] is None else s["bias"].double())
    size = c["experts"] // c["groups"]
    weights = torch.empty(c["tokens"], c["top_k"], dtype=torch.float64, device="cuda")

    def place(v):
        n = v.shape[1]
        lower = torch.ones(n, n, dtype=torch.bool, device=v.device).tril(-1)   # [j, i]: i < j
        a, b = v[:, :, None], v[:, None, :]
        return ((b > a) | ((b == a) & lower)).sum(dim=2)

    for t in range(0, c["tokens"], 64):
        k = key[t:t + 64]
        if c["groups"] > 1:
            group = k.unflatten(1, (c["groups"], size)).topk(min(2, size), dim=2)[0].sum(dim=2)
            k = torch.where((place(group) < c["top_groups"]).repeat_interleave(size, dim=1), k, -math.inf)
        r = place(k)
        chosen = (r[:, None, :] == torch.arange(c["top_k"], device=r.device)[:, None]).double()
        w = (chosen * score[t:t + 64, None, :]).sum(dim=2)
        weights[t:t + 64] = w / w.sum(dim=1, keepdim=True) if c["renormalize"] else w
    return dict(ids=None, weights=weights * c["scale"], counts=None, offsets=None, positions=None)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return _select64(s)
    if case["op"] == "quantize":
        parts = [_quantize64(x, case["block_rows"]) for x in s["x"]]
        return dict(q=torch.stack([p[0] for p in parts]), scale=torch.stack([p[1] for p in parts]))
    if case["op"] == "matmul":
        ends = [0, case["m"]] if s["offsets"] is None else s["offsets"].tolist()
        a = _values64(s["a"], s["a_scale"], 1)
        out = [a[i:j] @ _values64(s["w"][e], s["w_scale"][e], BLOCK).t() for e, (i, j) in enumerate(zip(ends, ends[1:]))]
        return dict(out=torch.cat(out))
    x = _values64(*_quantize64(s["x"], 1), 1)
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        token, choice = torch.where(s["ids"] == e)
        if token.numel():
            gate = x[token] @ _values64(s["up"][e], s["up_scale"][e], BLOCK).t()
            up = x[token] @ _values64(s["up_v"][e], s["up_v_scale"][e], BLOCK).t()
            h = _values64(*_quantize64(torch.nn.functional.silu(gate) * up, 1), 1)
            y = h @ _values64(s["down"][e], s["down_scale"][e], BLOCK).t()
            out.index_add_(0, token, y * s["weights"][token, choice, None].double())
    return dict(out=out)
