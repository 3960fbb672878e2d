"""Experts in 8 bits: quantisation, products and the expert layer on e4m3 codes with block scales
(an addition of this package; the reference has no 8-bit path).

A matrix in 8 bits is two arrays: e4m3 codes, row-major, and one fp32 scale per block -- 1 x 128 values of a
row for activations (scale [rows, ceil(cols / 128)]), 128 x 128 values for weights (scale [matrices,
ceil(rows / 128), ceil(cols / 128)]).  A code stands for its value times its block's scale.

As everywhere in this package, arguments are device addresses and a stream; an args object holds no memory
and may be used again.  Every call only launches kernels: nothing is allocated, nothing waits, calls can be
captured in a CUDA graph, and the thread's current device stays as it is.  All memory and the stream belong
to `device_id`.  Arguments that a call cannot take raise `FlashMoEError` before anything is launched.

    q, scale  = weights once through `quantize` (block_rows=128)
    per step:   router.select(...)   -> weights, offsets, positions
                fp8.experts(...)     -> the layer's output rows
"""
from __future__ import annotations

import ctypes as C

from . import _native as N
from .jit import ActivationType, DataType

__all__ = ["QuantizeArgs", "quantize", "MatmulArgs", "matmul", "GatedArgs", "gated_matmul", "ExpertsArgs", "experts",
           "get_workspace_bytes", "last_status", "BLOCK"]

BLOCK = 128   # values per scale along a row; rows per scale of a weight block


class QuantizeArgs:
    """x [num_matrices, rows, cols] of `data_type` -> q (e4m3, same shape) and scale; cols a multiple of 16.
    `block_rows` 1: a scale per 128 values of a row; 128: a scale per 128 x 128 block.
    With `positions` [rows, copies] int32 (rows of one matrix) row r is written to the rows positions[r] of
    [rows * copies]: the layout in expert order that the products take."""

    def __init__(self, x: int, q: int, scale: int, stream_ptr: int, *, rows: int, cols: int,
                 data_type: DataType = DataType.BF16, block_rows: int = 1, num_matrices: int = 1, positions: int = 0,
                 copies: int = 1, device_id: int = 0):
        self.stream_ptr = stream_ptr
        self.c = N.Fp8QuantizeArgsC(x or None, q or None, scale or None, positions or None, copies, rows, cols,
                                    num_matrices, block_rows, int(data_type), device_id)


def quantize(arg: QuantizeArgs) -> None:
    """scale = amax / 448 of each block, code = e4m3(448 x / amax), to nearest even; a block of zeros has
    scale 0, a block with a NaN or an infinity reads back as NaN."""
    N.check(N.lib().fmoe_fp8_quantize(arg.c, arg.stream_ptr), "fp8.quantize")


class MatmulArgs:
    """out [m, n] of `data_type` (BF16, FP16, FP32) = a [m, k] times w [n, k] transposed; k a multiple of 16.
    With `num_experts` > 1: w [num_experts, n, k], the rows of a and out in expert order, expert e's at
    offsets[e] .. offsets[e + 1] (int32 on the device, as `router.select` writes it)."""

    def __init__(self, a: int, a_scale: int, w: int, w_scale: int, out: int, stream_ptr: int, *, m: int, n: int, k: int,
                 data_type: DataType = DataType.BF16, num_experts: int = 1, offsets: int = 0, device_id: int = 0):
        self.stream_ptr = stream_ptr
        self.c = N.Fp8MatmulArgsC(a or None, a_scale or None, w or None, w_scale or None, out or None, offsets or None,
                                  m, n, k, num_experts, int(data_type), device_id)


def matmul(arg: MatmulArgs) -> None:
    """The product, each block of 128 of k summed on the tensor cores and scaled in fp32; one rounding."""
    N.check(N.lib().fmoe_fp8_matmul(arg.c, arg.stream_ptr), "fp8.matmul")


class GatedArgs:
    """h = act(a up^T) * (a up_v^T), quantised: q [m, ffn_size] e4m3 and scale [m, ceil(ffn_size / 128)].
    up, up_v [num_experts, ffn_size, k] with their block scales; up_v 0: a plain MLP, h = act(a up^T).
    Experts and offsets as in `MatmulArgs`; ffn_size and k multiples of 16."""

    def __init__(self, a: int, a_scale: int, up: int, up_scale: int, up_v: int, up_v_scale: int, q: int, scale: int,
                 stream_ptr: int, *, m: int, ffn_size: int, k: int, num_experts: int = 1, offsets: int = 0,
                 act_type: ActivationType = ActivationType.SILU, device_id: int = 0):
        self.stream_ptr = stream_ptr
        self.c = N.Fp8GatedArgsC(a or None, a_scale or None, up or None, up_scale or None, up_v or None,
                                 up_v_scale or None, q or None, scale or None, offsets or None, m, ffn_size, k,
                                 num_experts, int(act_type), device_id)


def gated_matmul(arg: GatedArgs) -> None:
    """Both up products, the activation and the quantisation of the result in one kernel."""
    N.check(N.lib().fmoe_fp8_gated_matmul(arg.c, arg.stream_ptr), "fp8.gated_matmul")


class ExpertsArgs:
    """The expert layer: tokens [S, H] of `data_type` (BF16, FP16) -> out [S, H].  offsets [E + 1], positions
    [S, k] and weights [S, k] are what `router.select` wrote; up, up_v [E, I, H] and down [E, H, I] are
    quantised with block_rows=128 (up_v 0: a plain MLP); H and I multiples of 16.  `workspace`: 256-byte
    aligned, at least `get_workspace_bytes(...)`; two calls that share one must be ordered by their
    streams, and so must two graphs that captured such calls."""

    def __init__(self, tokens: int, offsets: int, positions: int, weights: int, up: int, up_scale: int, down: int,
                 down_scale: int, out: int, workspace: int, workspace_bytes: int, stream_ptr: int, *, num_tokens: int,
                 token_dim: int, ffn_size: int, num_experts: int, top_k: int, up_v: int = 0, up_v_scale: int = 0,
                 data_type: DataType = DataType.BF16, act_type: ActivationType = ActivationType.SILU,
                 device_id: int = 0):
        self.stream_ptr = stream_ptr
        self.c = N.Fp8ExpertsArgsC(tokens or None, offsets or None, positions or None, weights or None, up or None,
                                   up_scale or None, up_v or None, up_v_scale or None, down or None, down_scale or None,
                                   out or None, workspace or None, workspace_bytes, num_tokens, token_dim, ffn_size,
                                   num_experts, top_k, int(data_type), int(act_type), device_id)


def get_workspace_bytes(*, num_tokens: int, token_dim: int, ffn_size: int, num_experts: int, top_k: int,
                        data_type: DataType = DataType.BF16) -> int:
    """What `experts` needs for this shape (host arithmetic; no GPU is touched)."""
    args = N.Fp8ExpertsArgsC(num_tokens=num_tokens, token_dim=token_dim, ffn_size=ffn_size, num_experts=num_experts,
                             top_k=top_k, data_type=int(data_type))
    size = C.c_int64()
    N.check(N.lib().fmoe_fp8_workspace_bytes(args, size), "fp8.get_workspace_bytes")
    return size.value


def experts(arg: ExpertsArgs) -> None:
    """Quantise into expert order, gated up product, down product, weighted sum of each token's rows."""
    N.check(N.lib().fmoe_fp8_experts(arg.c, arg.stream_ptr), "fp8.experts")


def last_status(device_id: int, stream_ptr: int) -> N.Status:
    """Waits for the stream; the record of a device-side wait of an 8-bit product that ran out on this device
    since the last call (code 0: none)."""
    s = N.Status()
    N.check(N.lib().fmoe_fp8_last_status(device_id, stream_ptr, s), "fp8.last_status")
    return s
