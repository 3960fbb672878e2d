"""Experts in 8 bits against plain 64-bit implementations.

Codes and scales of `quantize` are compared exactly with fp32 arithmetic that rounds as the definition says
(448 x, one division, e4m3 to nearest even).  Products: the tensor core sums the 128 exact products of a block in
fp32, a block is scaled (one rounding of the scales' product) and added (one fused rounding).  With T the sum of
the absolute values of all terms, every rounding is at most 2^-23 T (truncation counted), so the sum is within
(128 + 2 blocks + 2) 2^-23 T, and the result then half a step of its type.
"""
import ctypes as C

import pytest
import torch

import flashmoe_b200 as flashmoe
from flashmoe_b200 import _native as N
from flashmoe_b200 import fp8, router
from flashmoe_b200.jit import ActivationType, DataType

gpu = pytest.mark.gpu
TYPES = {torch.bfloat16: DataType.BF16, torch.float16: DataType.FP16, torch.float32: DataType.FP32}
E4M3 = torch.float8_e4m3fn


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stream():
    return torch.cuda.current_stream().cuda_stream


def blocks(n):
    return -(-n // 128)


# ---- plain forms -----------------------------------------------------------------------------------------

def plain_quantize(x, block_rows):
    """[B, R, C] -> codes and scales, in fp32 as the definition says."""
    B, R, K = x.shape
    f = x.float()
    pad = torch.nn.functional.pad(f, (0, -K % 128, 0, -R % block_rows))
    b = pad.view(B, pad.shape[1] // block_rows, block_rows, blocks(K), 128)
    amax = b.abs().amax(dim=(2, 4), keepdim=True)
    q = torch.where(amax > 0, (b * 448.0) / amax, torch.zeros_like(b))
    q = q.to(E4M3).view(torch.uint8).reshape(pad.shape)[:, :R, :K].contiguous().view(E4M3)
    return q, (amax / torch.full_like(amax, 448.0))[:, :, 0, :, 0].contiguous()


def values(q, scale, block_rows):
    """float64 values of [B, R, C] codes."""
    s = scale.double().repeat_interleave(block_rows, 1)[:, :q.shape[1]].repeat_interleave(128, 2)[:, :, :q.shape[2]]
    return q.double() * s


def normal(shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def rows8(m, k, seed):
    q, s = plain_quantize(normal((1, m, k), seed), 1)
    return q[0], s[0]


def weights8(e, n, k, seed):
    return plain_quantize(normal((e, n, k), seed, 0.05), 128)


# ---- quantize -------------------------------------------------------------------------------------------

def quantize(x, block_rows, positions=None):
    B, R, K = x.shape
    copies = 1 if positions is None else positions.shape[1]
    q = torch.full((B, R * copies, K), 1.0, device="cuda").to(E4M3)
    s = torch.full((B, -(-R // block_rows) * copies, blocks(K)), -7.0, device="cuda")
    fp8.quantize(fp8.QuantizeArgs(x.data_ptr(), q.data_ptr(), s.data_ptr(), stream(), rows=R, cols=K,
                                  data_type=TYPES[x.dtype], block_rows=block_rows, num_matrices=B,
                                  positions=0 if positions is None else positions.data_ptr(), copies=copies))
    torch.cuda.synchronize()
    return q, s


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@gpu
@pytest.mark.parametrize("dtype", list(TYPES), ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 16), (1, 1, 128), (1, 3, 2064), (2, 5, 144), (1, 513, 7168), (3, 200, 400)], ids=str)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_bits(shape, dtype, block_rows):
    x = normal(shape, sum(shape), dtype=dtype)
    x[0, 0, :8] *= 30
    q, s = quantize(x, block_rows)
    want_q, want_s = plain_quantize(x, block_rows)
    assert same(q, want_q) and torch.equal(s, want_s)


@gpu
def test_quantize_rounds_every_ratio_of_bf16_as_exact_arithmetic_does():
    """All 128 x 128 pairs of bf16 mantissas as (value, block maximum), over the codes' exponents: the code
    nearest to 448 x / amax, ties to even, decided in integers."""
    top = torch.arange(128, 256, device="cuda").float()                    # block maxima, one a row
    part = torch.arange(128, 256, device="cuda").float()
    for e in (0, 1, 2, 5, 8, 12, 16, 18, 19):                                 # x = part * 2^-e, at most amax
        x = (part / 2.0 ** e)[None, :].repeat(128, 1).clamp(max=top[:, None])
        both = torch.zeros(1, 128, 256, device="cuda")
        both[0, :, :128] = x
        both[0, :, 0] = top
        both[0, :, 128:] = x
        both[0, :, 128] = top
        q, s = quantize(both.bfloat16(), 1)
        a, m = both[0].cpu().double(), top.cpu().double()[:, None]
        n = (a * 448 * 2 ** 20).to(torch.int64)                              # 448 x, exact, in units of 2^-20
        d = (m * 2 ** 20).to(torch.int64)
        ratio = a * 448 / m
        exp = (torch.frexp(ratio)[1].to(torch.int64) - 1).clamp(min=-6)      # (a quotient of 8-bit numbers is no 2^-53 from a power of 2)
        step = exp - 3                                                       # a code's unit is 2^step
        num, den = n * 2 ** (-step).clamp(min=0), d * 2 ** step.clamp(min=0)
        whole, rest = num // den, num % den
        up = (2 * rest > den) | ((2 * rest == den) & (whole % 2 == 1))
        want = (whole + up.to(torch.int64)).double() * 2.0 ** step.double()
        assert torch.equal(q[0].double().cpu(), want), e
        assert torch.equal(s[0, :, 0].cpu(), (top.cpu() / 448.0))


@gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(block_rows):
    x = torch.zeros(1, 128 * 8, 256, device="cuda")
    r = 128
    x[0, r, 3] = 1e-44                          # a denormal block
    x[0, 2 * r, :4] = torch.tensor([3.4e38, -1.7e38, 1e30, 1e-30], device="cuda")
    x[0, 3 * r, 5] = float("inf")
    x[0, 3 * r, 6] = 1.0
    x[0, 4 * r, 130] = float("nan")
    x[0, 4 * r, 131] = 1.0
    x[0, 5 * r, :] = -448.0
    x[0, 6 * r, :2] = torch.tensor([-0.0, 2.0], device="cuda")
    q, s = quantize(x, block_rows)
    at = (lambda row: row) if block_rows == 1 else (lambda row: row // 128)
    v = values(q, s, block_rows)[0]
    assert not q[0, 0].float().any() and float(s[0, 0, 0]) == 0.0
    assert float(q[0, r, 3].float()) == 448.0
    assert [float(c) for c in q[0, 2 * r, :4].float()] == [448.0, -224.0, 0.0, 0.0]
    assert float(s[0, at(2 * r), 0]) == float(torch.tensor(3.4e38) / 448)
    assert bool(v[3 * r, :128].isnan().all()) and bool(v[4 * r, 128:].isnan().all())
    assert not v[3 * r, 128:].any() and not v[4 * r, :128].any()
    assert bool((v[5 * r] == -448.0).all())
    assert abs(float(v[6 * r, 1]) - 2.0) <= 2.0 ** -23     # the code is 448; the scale 2 / 448 is rounded by 2^-24 of itself


@gpu
@pytest.mark.parametrize("copies", [1, 3])
def test_quantize_into_expert_order(copies):
    R, K = 37, 272
    x = normal((1, R, K), 4, dtype=torch.bfloat16)
    p = torch.randperm(R * copies, generator=torch.Generator().manual_seed(1)).int().view(R, copies)
    p[5, 0], p[6, 0] = -1, R * copies            # outside: ignored
    q, s = quantize(x, 1, p.cuda())
    want_q, want_s = plain_quantize(x, 1)
    written = torch.zeros(R * copies, dtype=torch.bool)
    for r in range(R):
        for j in range(copies):
            to = int(p[r, j])
            if 0 <= to < R * copies:
                written[to] = True
                assert same(q[0, to], want_q[0, r]) and torch.equal(s[0, to], want_s[0, r])
    assert bool((q[0].float().cpu()[~written] == 1.0).all()) and bool((s[0].cpu()[~written] == -7.0).all())


# ---- products ---------------------------------------------------------------------------------------------

def spans_of(counts):
    ends = [0]
    for c in counts:
        ends.append(ends[-1] + c)
    return ends


def product64(a, sa, w, sw, spans):
    """The product and the sum of its terms' absolute values, float64."""
    av, wv = values(a[None], sa[None], 1)[0], values(w, sw, 128)
    out = torch.zeros(a.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    for e in range(w.shape[0]):
        i, j = spans[e], spans[e + 1]
        out[i:j] = av[i:j] @ wv[e].t()
        mag[i:j] = av[i:j].abs() @ wv[e].abs().t()
    return out, mag


def sum_tol(k):
    return (128 + 2 * blocks(k) + 2) * 2.0 ** -23


def run_matmul(a, sa, w, sw, dtype, offsets=None, m=None, out=None):
    e, n, k = w.shape
    m = a.shape[0] if m is None else m
    out = torch.full((a.shape[0], n), -7.0, dtype=dtype, device="cuda") if out is None else out
    fp8.matmul(fp8.MatmulArgs(a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(), out.data_ptr(), stream(), m=m, n=n,
                              k=k, data_type=TYPES[dtype], num_experts=e,
                              offsets=0 if offsets is None else offsets.data_ptr()))
    torch.cuda.synchronize()
    return out


def close(got, want, tol, dtype):
    """|got - want| within tol, then rounded to dtype (values near its smallest normal round absolutely)."""
    err = (got.double() - want).abs()
    room = tol + half_step(dtype) * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * half_step(dtype)
    worst = float((err / room).max()) if err.numel() else 0.0
    assert worst <= 1.0, worst


@gpu
@pytest.mark.parametrize("dtype", list(TYPES), ids=str)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 130, 144), (1, 4096, 2048), (2, 16, 128), (7, 129, 256), (16, 256, 1040),
                                   (17, 257, 512), (33, 1000, 400), (64, 640, 1024), (65, 384, 1536), (127, 255, 272),
                                   (128, 256, 128), (129, 512, 640), (300, 777, 2064), (520, 1032, 4096)])
def test_product(m, n, k, dtype):
    a, sa = rows8(m, k, m + n)
    w, sw = weights8(1, n, k, k)
    want, mag = product64(a, sa, w, sw, [0, m])
    close(run_matmul(a, sa, w, sw, dtype), want, sum_tol(k) * mag, dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("counts,n,k", [([1, 0, 3], 128, 256), ([0, 0, 5, 0], 144, 128), ([16, 17, 1, 40], 272, 384),
                                        ([130, 0, 1, 257], 300, 400), ([0] * 63 + [2], 64, 64), ([3] * 200, 96, 160),
                                        ([600, 20], 520, 1024), ([64, 65, 63, 100, 128], 384, 272)], ids=str)
def test_product_by_expert(counts, n, k, dtype):
    spans = spans_of(counts)
    m = spans[-1]
    a, sa = rows8(m + 9, k, m)                    # nine rows behind the last expert: not written
    w, sw = weights8(len(counts), n, k, n)
    off = torch.tensor(spans, dtype=torch.int32, device="cuda")
    got = run_matmul(a, sa, w, sw, dtype, off)
    want, mag = product64(a, sa, w, sw, spans)
    close(got[:m], want[:m], sum_tol(k) * mag[:m], dtype)
    assert bool((got[m:] == -7.0).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("counts,n,k", [([20], 512, 4096), ([3], 300, 8192), ([300], 777, 2064), ([520], 1032, 4096), ([900], 4112, 528),
                                        ([2304], 4864, 4112), ([2500], 9500, 2064), ([70] * 20, 1024, 1040), ([90] * 24, 1024, 1040),
                                        ([2000, 3000], 4864, 2064), ([0, 3000, 3500], 8192, 4112)],
                         ids=["16 rows, split", "16 rows, split more", "32 rows, split", "64 rows", "128 rows", "pairs", "pairs, odd rows",
                              "64 rows, experts", "128 rows, experts", "128 rows, few experts", "pairs, few experts"])
def test_every_tile_form(counts, n, k, dtype):
    """Sizes that take each of the kernels (what takes which is the library's choice: the results are what is held here)."""
    spans = spans_of(counts)
    m = spans[-1]
    a, sa = rows8(m, k, m)
    w, sw = weights8(len(counts), n, k, n)
    off = torch.tensor(spans, dtype=torch.int32, device="cuda") if len(counts) > 1 else None
    want, mag = product64(a, sa, w, sw, spans)
    close(run_matmul(a, sa, w, sw, dtype, off), want, sum_tol(k) * mag, dtype)
    assert fp8.last_status(0, stream()).code == 0


@gpu
def test_places_beyond_32_bits():
    """More than 2^31 values in and out: the last rows land where they belong."""
    rows, cols = 270_000, 8192
    x = torch.zeros(1, rows, cols, dtype=torch.bfloat16, device="cuda")
    x[0, -3:] = normal((3, cols), 1, dtype=torch.bfloat16)
    q = torch.zeros(1, rows, cols, dtype=E4M3, device="cuda")
    s = torch.full((1, rows, blocks(cols)), -7.0, device="cuda")
    fp8.quantize(fp8.QuantizeArgs(x.data_ptr(), q.data_ptr(), s.data_ptr(), stream(), rows=rows, cols=cols))
    torch.cuda.synchronize()
    want_q, want_s = plain_quantize(x[:, -3:], 1)
    assert same(q[0, -3:], want_q[0]) and torch.equal(s[0, -3:], want_s[0]) and not s[0, :-3].any()
    del x, q, s
    m, n, k = 66_000, 33_000, 16
    a, sa = rows8(m, k, 2)
    w, sw = weights8(1, n, k, 3)
    out = run_matmul(a, sa, w, sw, torch.bfloat16)
    for r in (slice(0, 2), slice(m // 2, m // 2 + 2), slice(m - 2, m)):
        want, mag = product64(a[r], sa[r], w, sw, [0, 2])
        close(out[r], want, sum_tol(k) * mag, torch.bfloat16)


@gpu
def test_no_rows_and_offsets_outside_the_rows():
    k, n = 256, 128
    a, sa = rows8(20, k, 1)
    w, sw = weights8(3, n, k, 2)
    assert bool((run_matmul(a, sa, w, sw, torch.float32, torch.zeros(4, dtype=torch.int32, device="cuda")) == -7.0).all())
    assert bool((run_matmul(a, sa, w[:1], sw[:1], torch.float32, m=0) == -7.0).all())
    # expert 0 has rows 0..7; expert 1 would begin before 0 and expert 2 end behind row 20: cut to the rows there are
    off = torch.tensor([0, 8, 8, 1000], dtype=torch.int32, device="cuda")
    got = run_matmul(a, sa, w, sw, torch.float32, off)
    want, mag = product64(a, sa, w, sw, [0, 8, 8, 20])
    close(got, want, sum_tol(k) * mag, torch.float32)
    off = torch.tensor([-5, 8, 4, 20], dtype=torch.int32, device="cuda")    # expert 1 runs backwards: no rows
    got = run_matmul(a, sa, w, sw, torch.float32, off)
    whole, mag = product64(a, sa, w, sw, [0, 8, 8, 20])
    assert bool((got[:4].double() - whole[:4]).abs().le(sum_tol(k) * mag[:4] + 2.0 ** -23 * whole[:4].abs()).all())


@gpu
def test_rows_of_nan_and_infinity_stay_among_themselves():
    m, n, k = 70, 200, 384
    a, sa = rows8(m, k, 3)
    w, sw = weights8(1, n, k, 4)
    sa[5, 1] = float("nan")
    sa[40, 0] = float("inf")
    clean = [r for r in range(m) if r not in (5, 40)]
    want, mag = product64(a, sa, w, sw, [0, m])
    got = run_matmul(a, sa, w, sw, torch.bfloat16)
    close(got[clean], want[clean], sum_tol(k) * mag[clean], torch.bfloat16)
    assert bool(got[5].isnan().all()) and not bool(got[40].isfinite().any())


@gpu
@pytest.mark.parametrize("dtype,offset", [(torch.bfloat16, 1), (torch.bfloat16, 8), (torch.float32, 1), (torch.float32, 4)], ids=str)
def test_output_alignments(dtype, offset):
    """Outputs that start off a 32-byte boundary, and what lies around them."""
    m, n, k = 40, 256, 256
    a, sa = rows8(m, k, 3)
    w, sw = weights8(1, n, k, 4)
    room = torch.full((offset + m * n + 8,), -7.0, dtype=dtype, device="cuda")
    got = run_matmul(a, sa, w, sw, dtype, out=room[offset:offset + m * n])
    want, mag = product64(a, sa, w, sw, [0, m])
    close(got.view(m, n), want, sum_tol(k) * mag, dtype)
    assert bool((room[:offset] == -7.0).all()) and bool((room[offset + m * n:] == -7.0).all())


@gpu
def test_two_calls_give_the_same_bits():
    a, sa = rows8(45, 2048, 3)
    w, sw = weights8(1, 520, 2048, 4)
    assert torch.equal(run_matmul(a, sa, w, sw, torch.float32), run_matmul(a, sa, w, sw, torch.float32))


# ---- gated product ------------------------------------------------------------------------------------------

def act64(x, act):
    return {ActivationType.IDENTITY: lambda: x, ActivationType.SILU: lambda: torch.nn.functional.silu(x),
            ActivationType.GELU: lambda: torch.nn.functional.gelu(x), ActivationType.RELU: lambda: torch.relu(x)}[act]()


def run_gated(a, sa, up, sup, v, sv, act, offsets=None):
    e, n, k = up.shape
    q = torch.full((a.shape[0], n), 1.0, device="cuda").to(E4M3)
    s = torch.full((a.shape[0], blocks(n)), -7.0, device="cuda")
    ptr = lambda t: 0 if t is None else t.data_ptr()
    fp8.gated_matmul(fp8.GatedArgs(a.data_ptr(), sa.data_ptr(), up.data_ptr(), sup.data_ptr(), ptr(v), ptr(sv), q.data_ptr(),
                                   s.data_ptr(), stream(), m=a.shape[0], ffn_size=n, k=k, num_experts=e,
                                   offsets=ptr(offsets), act_type=act))
    torch.cuda.synchronize()
    return q, s


def check_gated(q, s, m, g, tg, u, tu, k, act):
    """h = act(g) u from values g, u with error bounds tol * T: |act'| is below 1.13 for all four, the activation itself is
    within 2^-21 of its value (gelu: of |g|, erff's error is absolute); codes within half a step of 3 mantissa bits."""
    tol = sum_tol(k)
    h = act64(g, act)
    err = 1.13 * tol * tg + 2.0 ** -21 * g.abs()
    if u is not None:
        err = err * (u.abs() + tol * tu) + h.abs() * tol * tu
        h = h * u
    err = err + 2.0 ** -22 * h.abs()
    n = h.shape[1]
    pad = torch.nn.functional.pad
    amax = pad(h.abs(), (0, -n % 128)).view(m, -1, 128).amax(2)
    worst = pad(err, (0, -n % 128)).view(m, -1, 128).amax(2)
    got_s = s[:m].double()
    assert bool(((got_s * 448 - amax).abs() <= worst + 2.0 ** -22 * amax).all())
    got = q[:m].double() * got_s.repeat_interleave(128, 1)[:, :n]
    room = err + 2.0 ** -4 * (h.abs() + err) * (1 + 2.0 ** -20) + (2.0 ** -10 * got_s).repeat_interleave(128, 1)[:, :n]
    assert bool(((got - h).abs() <= room).all()), float(((got - h).abs() / room).max())
    assert float(q[:m].float().abs().amax()) == 448.0


@gpu
@pytest.mark.parametrize("act", list(ActivationType), ids=lambda a: a.name)
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("counts,n,k", [([1], 16, 16), ([5], 144, 256), ([64], 384, 272), ([200], 272, 1024), ([2, 0, 40, 1], 256, 384),
                                        ([130, 7, 0], 400, 512), ([1] * 40, 128, 144), ([5], 256, 4096), ([100], 1040, 2064),
                                        ([300], 2064, 2064), ([40] * 6, 2048, 1040)], ids=str)
def test_gated_product(counts, n, k, gated, act):
    spans = spans_of(counts)
    m, E = spans[-1], len(counts)
    a, sa = rows8(m + 3, k, m)
    up, sup = weights8(E, n, k, 1)
    v, sv = weights8(E, n, k, 2) if gated else (None, None)
    off = torch.tensor(spans, dtype=torch.int32, device="cuda") if E > 1 else None
    if E == 1:
        spans = [0, m + 3]
        m += 3
    q, s = run_gated(a, sa, up, sup, v, sv, act, off)
    g, tg = product64(a, sa, up, sup, spans)
    u, tu = product64(a, sa, v, sv, spans) if gated else (None, None)
    cut = lambda t: None if t is None else t[:m]
    check_gated(q, s, m, cut(g), cut(tg), cut(u), cut(tu), k, act)
    assert bool((q[m:].float() == 1.0).all()) and bool((s[m:] == -7.0).all())


@gpu
@pytest.mark.parametrize("gated", [True, False])
def test_gated_product_by_pairs(gated):
    counts, n, k = [2000, 3000], 4864, 2064
    spans, act = spans_of(counts), ActivationType.SILU
    a, sa = rows8(5000, k, 1)
    up, sup = weights8(2, n, k, 2)
    v, sv = weights8(2, n, k, 3) if gated else (None, None)
    q, s = run_gated(a, sa, up, sup, v, sv, act, torch.tensor(spans, dtype=torch.int32, device="cuda"))
    g, tg = product64(a, sa, up, sup, spans)
    u, tu = product64(a, sa, v, sv, spans) if gated else (None, None)
    check_gated(q, s, 5000, g, tg, u, tu, k, act)


# ---- the layer ---------------------------------------------------------------------------------------------

class Layer:
    def __init__(self, S, H, I, E, k, dtype=torch.bfloat16, gated=True, act=ActivationType.SILU, seed=0, stream_ptr=None):
        self.shape = S, H, I, E, k
        self.dtype, self.act, self.gated = dtype, act, gated
        self.x = normal((S, H), seed, dtype=dtype)
        self.logits = normal((S, E), seed + 1)
        self.up, self.sup = weights8(E, I, H, seed + 2)
        self.v, self.sv = weights8(E, I, H, seed + 3) if gated else (None, None)
        self.down, self.sdown = weights8(E, H, I, seed + 4)
        new = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.ids, self.counts, self.offsets, self.positions = new(S, k), new(E), new(E + 1), new(S, k)
        self.weights = torch.zeros(S, k, device="cuda")
        self.out = torch.full((S, H), -7.0, dtype=dtype, device="cuda")
        size = fp8.get_workspace_bytes(num_tokens=S, token_dim=H, ffn_size=I, num_experts=E, top_k=k, data_type=TYPES[dtype])
        self.ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        st = stream() if stream_ptr is None else stream_ptr
        ptr = lambda t: 0 if t is None else t.data_ptr()
        self.sargs = router.SelectArgs(self.logits.data_ptr(), self.ids.data_ptr(), self.weights.data_ptr(),
                                       self.counts.data_ptr(), st, num_tokens=S, num_experts=E, top_k=k,
                                       offsets=self.offsets.data_ptr(), positions=self.positions.data_ptr())
        self.eargs = fp8.ExpertsArgs(self.x.data_ptr(), self.offsets.data_ptr(), self.positions.data_ptr(),
                                     self.weights.data_ptr(), self.up.data_ptr(), self.sup.data_ptr(), self.down.data_ptr(),
                                     self.sdown.data_ptr(), self.out.data_ptr(), self.ws.data_ptr(), size, st, num_tokens=S,
                                     token_dim=H, ffn_size=I, num_experts=E, top_k=k, up_v=ptr(self.v),
                                     up_v_scale=ptr(self.sv), data_type=TYPES[dtype], act_type=act)

    def step(self):
        router.select(self.sargs)
        fp8.experts(self.eargs)

    def check(self):
        """Against the layer's parts: the quantised rows and the gated product's codes (tested above) as this
        step's kernels give them, the rest in 64 bits.  A down row is a product (sum_tol) in fp32; the sum of k
        weighted rows rounds k times in fp32 and once to 16 bits."""
        S, H, I, E, k = self.shape
        choice = torch.sort(self.logits, dim=1, descending=True, stable=True)[1][:, :k]
        assert torch.equal(self.ids.long(), choice)
        assert fp8.last_status(0, stream()).code == 0
        q, s = quantize(self.x[None], 1, self.positions)
        hq, hs = run_gated(q[0], s[0], self.up, self.sup, self.v, self.sv, self.act, self.offsets if E > 1 else None)
        y, mag = product64(hq, hs, self.down, self.sdown, self.offsets.tolist())
        p, w = self.positions.long(), self.weights.double()[:, :, None]
        want, terms = (y[p] * w).sum(1), (y[p] * w).abs().sum(1)
        row_err = sum_tol(I) * mag + 2.0 ** -24 * y.abs()
        tol = (row_err[p] * w).sum(1) + k * 2.0 ** -23 * terms
        close(self.out, want, tol, self.dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("S,H,I,E,k", [(1, 64, 64, 8, 2), (1, 512, 256, 16, 8), (5, 272, 144, 4, 1), (33, 256, 400, 8, 3),
                                       (64, 384, 272, 40, 8), (300, 512, 256, 4, 2), (70, 128, 128, 1, 1), (700, 256, 128, 64, 4)])
def test_layer(S, H, I, E, k, dtype):
    layer = Layer(S, H, I, E, k, dtype, seed=S)
    layer.step()
    torch.cuda.synchronize()
    layer.check()


@gpu
@pytest.mark.parametrize("gated,act", [(False, ActivationType.GELU), (False, ActivationType.RELU), (True, ActivationType.GELU)])
def test_layer_forms(gated, act):
    layer = Layer(50, 256, 272, 8, 2, gated=gated, act=act)
    layer.step()
    torch.cuda.synchronize()
    layer.check()


@gpu
def test_captured_layer_follows_its_inputs():
    """Routing and layer captured once on another stream; each replay's routing comes from that replay's logits."""
    side = torch.cuda.Stream()
    layer = Layer(40, 256, 256, 16, 4, stream_ptr=side.cuda_stream)
    torch.cuda.synchronize()
    layer.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer.step()
    for seed in (11, 12):
        layer.x.copy_(normal((40, 256), seed, dtype=torch.bfloat16))
        layer.logits.copy_(normal((40, 16), seed + 100, 3.0))
        graph.replay()
        torch.cuda.synchronize()
        layer.check()


@gpu
def test_two_layers_at_once_on_two_streams():
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    layers = [Layer(200, 512, 384, 8, 2, seed=i, stream_ptr=s.cuda_stream) for i, s in enumerate(streams)]
    torch.cuda.synchronize()
    for _ in range(5):
        for layer in layers:
            layer.step()
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()


@gpu
def test_two_graphs_and_eager_calls_of_one_layer():
    """Two captured steps and eager ones, ordered by one stream, share the layer's workspace and outputs."""
    side = torch.cuda.Stream()
    layer = Layer(24, 256, 272, 8, 2, stream_ptr=side.cuda_stream)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            layer.step()
        graphs.append(g)
    for seed, run in enumerate([graphs[0].replay, layer.step, graphs[1].replay, graphs[0].replay, layer.step]):
        layer.x.copy_(normal((24, 256), 50 + seed, dtype=torch.bfloat16))
        layer.logits.copy_(normal((24, 8), 80 + seed))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        layer.check()


FIRST_CALL = """
import sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
import test_fp8 as T
side = torch.cuda.Stream()
layer = T.Layer(24, 256, 272, 8, 2, stream_ptr=side.cuda_stream)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    layer.step()
graph.replay()
torch.cuda.synchronize()
layer.check()
"""


@gpu
def test_the_first_call_of_a_process_can_be_a_captured_one():
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=os.path.dirname(here), tests=here)], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@gpu
def test_large_layer_on_every_form():
    """4096 tokens on 4 experts (pairs) and 64 experts (128 rows)."""
    for E, k in ((4, 2), (64, 2)):
        layer = Layer(4096, 512, 640, E, k, seed=E)
        layer.step()
        torch.cuda.synchronize()
        layer.check()


@gpu
def test_no_tokens():
    layer = Layer(0, 64, 64, 8, 2)
    layer.step()
    torch.cuda.synchronize()
    assert not layer.offsets.any()


# ---- refusals (no GPU is touched) -----------------------------------------------------------------------------

def refused(call, args, code, needle):
    with pytest.raises(flashmoe.FlashMoEError, match=needle) as e:
        call(args)
    assert e.value.code == code


@pytest.mark.parametrize("kw,code,needle", [
    (dict(rows=-1), 1, "rows"), (dict(cols=0), 1, "cols"), (dict(cols=24), 1, "multiple of 16"), (dict(block_rows=64), 1, "block_rows"),
    (dict(data_type=DataType.FP64), 2, "BF16"), (dict(device_id=-1), 1, "device_id"), (dict(copies=2), 1, "copies"),
    (dict(positions=64, copies=0), 1, "copies"), (dict(positions=64, block_rows=128), 1, "positions"),
    (dict(positions=64, num_matrices=2), 1, "positions"), (dict(x=0), 1, "required"), (dict(scale=0), 1, "required"),
    (dict(x=72), 1, "16-byte"), (dict(q=8), 1, "16-byte"), (dict(scale=66), 1, "4-byte"),
    (dict(num_matrices=70000, block_rows=128), 2, "65535"), (dict(rows=1 << 30, positions=64, copies=4), 2, "32 bits"),
    (dict(rows=1 << 20, num_matrices=1 << 20), 2, "32 bits"),
])
def test_quantize_refusals(kw, code, needle):
    a = dict(x=64, q=64, scale=64, rows=4, cols=128)
    a.update(kw)
    refused(fp8.quantize, fp8.QuantizeArgs(a.pop("x"), a.pop("q"), a.pop("scale"), 0, **a), code, needle)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(m=-1), 1, "m must"), (dict(n=0), 1, "positive"), (dict(k=8), 1, "multiple of 16"), (dict(num_experts=0), 1, "num_experts"),
    (dict(num_experts=1025, offsets=64), 1, "1024"), (dict(num_experts=2), 1, "offsets"), (dict(data_type=DataType.FP64), 2, "BF16"),
    (dict(a=0), 1, "required"), (dict(out=0), 1, "out"), (dict(w=72), 1, "16-byte"), (dict(out=65), 1, "aligned"),
    (dict(w_scale=2), 1, "4-byte"), (dict(offsets=2), 1, "4-byte"), (dict(device_id=64), 1, "device_id"),
    (dict(num_experts=1024, n=1 << 22, offsets=64), 2, "32-bit"), (dict(m=0x7fffffff), 2, "32-bit"),
    (dict(m=1 << 24, n=1 << 24), 2, "32-bit"),
])
def test_matmul_refusals(kw, code, needle):
    a = dict(a=64, a_scale=64, w=64, w_scale=64, out=64, m=4, n=128, k=128)
    a.update(kw)
    pos = [a.pop(n) for n in ("a", "a_scale", "w", "w_scale", "out")]
    refused(fp8.matmul, fp8.MatmulArgs(*pos, 0, **a), code, needle)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(ffn_size=24), 1, "ffn_size"), (dict(act_type=4), 1, "act_type"), (dict(up_v_scale=0), 1, "up_v"), (dict(q=0), 1, "required"),
    (dict(up_v=72), 1, "16-byte"), (dict(scale=66), 1, "4-byte"), (dict(k=24), 1, "multiple of 16"), (dict(num_experts=2), 1, "offsets"),
])
def test_gated_refusals(kw, code, needle):
    a = dict(a=64, a_scale=64, up=64, up_scale=64, up_v=64, up_v_scale=64, q=64, scale=64, m=4, ffn_size=128, k=128)
    a.update(kw)
    pos = [a.pop(n) for n in ("a", "a_scale", "up", "up_scale", "up_v", "up_v_scale", "q", "scale")]
    refused(fp8.gated_matmul, fp8.GatedArgs(*pos, 0, **a), code, needle)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(num_tokens=-1), 1, "num_tokens"), (dict(token_dim=72), 1, "multiples of 16"), (dict(ffn_size=8), 1, "multiples of 16"),
    (dict(top_k=9), 1, "top_k"), (dict(num_experts=2000), 1, "num_experts"), (dict(data_type=DataType.FP32), 2, "BF16"),
    (dict(workspace_bytes=100), 1, "workspace"), (dict(workspace=0), 1, "workspace"), (dict(workspace=128), 1, "256-byte"),
    (dict(tokens=0), 1, "required"), (dict(tokens=8), 1, "16-byte"), (dict(positions=2), 1, "4-byte"),
    (dict(up=8), 1, "16-byte"), (dict(up_v=8, up_v_scale=64), 1, "16-byte"), (dict(up_v=64), 1, "up_v"), (dict(offsets=2), 1, "4-byte"),
    (dict(down_scale=2), 1, "4-byte"), (dict(num_tokens=1 << 30, workspace_bytes=1 << 60), 2, "32"), (dict(act_type=9), 1, "act_type"),
    (dict(device_id=99), 1, "device_id"),
])
def test_experts_refusals(kw, code, needle):
    names = ("tokens", "offsets", "positions", "weights", "up", "up_scale", "down", "down_scale", "out", "workspace")
    a = dict({n: 256 for n in names}, workspace_bytes=1 << 30, num_tokens=4, token_dim=64, ffn_size=64, num_experts=8, top_k=2)
    a.update(kw)
    pos = [a.pop(n) for n in names] + [a.pop("workspace_bytes")]
    refused(fp8.experts, fp8.ExpertsArgs(*pos, 0, **a), code, needle)


def test_last_status_refusals():
    assert N.lib().fmoe_fp8_last_status(0, None, None) == 1
    assert N.lib().fmoe_fp8_last_status(64, None, C.byref(N.Status())) == 1


def test_workspace_bytes():
    """Codes and scales of both operands and the fp32 rows of every pair, each part on a 256-byte boundary."""
    up = lambda v: -(-v // 256) * 256
    got = fp8.get_workspace_bytes(num_tokens=33, token_dim=272, ffn_size=400, num_experts=8, top_k=3)
    assert got == up(99 * 272) + up(99 * 3 * 4) + up(99 * 400) + up(99 * 4 * 4) + up(99 * 272 * 4)
    assert fp8.get_workspace_bytes(num_tokens=0, token_dim=64, ffn_size=64, num_experts=8, top_k=2) == 0
    with pytest.raises(flashmoe.FlashMoEError):
        fp8.get_workspace_bytes(num_tokens=1, token_dim=60, ffn_size=64, num_experts=8, top_k=2)


def test_argument_records_have_the_header_s_sizes():
    assert C.sizeof(N.Fp8QuantizeArgsC) == 4 * 8 + 7 * 4 + 4
    assert C.sizeof(N.Fp8MatmulArgsC) == 6 * 8 + 6 * 4
    assert C.sizeof(N.Fp8GatedArgsC) == 9 * 8 + 6 * 4
    assert C.sizeof(N.Fp8ExpertsArgsC) == 12 * 8 + 8 + 8 * 4
