// What the 8-bit kernels share: the block format, tensor-core and conversion wrappers, launch helpers.
//
// A matrix in 8 bits is a row-major array of e4m3 codes and one fp32 scale per block: 1 x 128 values
// of a row for activations (scale [rows, ceil(cols / 128)]), 128 x 128 values for weights (scale
// [matrices, ceil(rows / 128), ceil(cols / 128)]).  A code stands for (its value) * (its block's scale).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace fmoe::fp8 {

constexpr int kBlock = 128;          // values per scale along a row, rows per scale of a weight block
constexpr float kE4m3Max = 448.0f;   // largest finite e4m3 value

__host__ __device__ constexpr int blocks_of(int n) { return (n + kBlock - 1) / kBlock; }

// ---- pairs of fp32 ---------------------------------------------------------------------------
// Two independent operations an instruction, each rounded as a scalar one.
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}

// ---- quantisation arithmetic ----------------------------------------------------------------
// scale = amax / 448, code = e4m3(448 x / amax), all in IEEE fp32.  For 16-bit x the product 448 x
// is exact and the quotient correctly rounded, so the code is the one infinite precision would give:
// a quotient of two such numbers that is not a midpoint of two codes is at least 2^-11 of itself away
// from one, far more than half an fp32 step.
// The quotient is taken with the reciprocal and one correction, y = n r, y + r (n - y d): with r = 1 / d correctly
// rounded the result is the correctly rounded n / d (P. Markstein, Computation of elementary functions on the IBM
// RISC System/6000 processor, 1990), at four operations a value, two values to an instruction; a division
// instruction per value made the kernel wait for arithmetic at half the memory's rate.
// Very large and very small blocks are scaled by a power of two first, so that 448 x stays finite and 1 / d
// exists; values that underflow by it are below 2^-200 of amax and have the code 0 either way.
struct Quantizer {
  uint64_t num, neg_den, rcp;   // pairs
  __device__ __forceinline__ explicit Quantizer(float amax) {
    const float pre = amax > 0x1p+100f ? 0x1p-20f : (amax < 0x1p-100f ? 0x1p+100f : 1.0f);
    const float den = amax > 0.0f ? amax * pre : (amax == 0.0f ? 1.0f : amax);   // an empty block: codes 0; NaN stays
    const float n = kE4m3Max * pre, r = __frcp_rn(den);
    num = pack2(n, n);
    neg_den = pack2(-den, -den);
    rcp = pack2(r, r);
  }
  // 448 x / amax of two values
  __device__ __forceinline__ float2 scaled(float a, float b) const {
    const uint64_t n = mul2(pack2(a, b), num), y = mul2(n, rcp);
    return unpack2(fma2(fma2(y, neg_den, n), rcp, y));
  }
};
// The same for values that carry rounding errors of their own (a product's results): one division per
// block, then a product per value, at most 2^-23 from the quotient.
struct FastQuantizer {
  float pre, inv;   // code = e4m3((pre x) inv)
  __device__ __forceinline__ explicit FastQuantizer(float amax) {
    const bool tiny = amax < 0x1p-100f;                // 448 / amax must stay finite, and not underflow
    pre = tiny ? 0x1p+80f : 1.0f;
    inv = amax > 0.0f ? __fdiv_rn(kE4m3Max, amax * pre) : (amax == 0.0f ? 0.0f : amax);
  }
  __device__ __forceinline__ float scaled(float x) const { return (x * pre) * inv; }
};
// amax / 448 correctly rounded, in the same way; tiny ones, whose quotient loses bits, by a division.
__device__ __forceinline__ float block_scale(float amax) {
  if (!(amax >= 0x1p-90f && amax <= 0x1p+120f)) return __fdiv_rn(amax, kE4m3Max);
  constexpr float r = 1.0f / kE4m3Max;
  const float y = amax * r;
  return fmaf(fmaf(-kE4m3Max, y, amax), r, y);
}
// Two values to two codes (lo in the low byte), round to nearest even.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16);
}
// |x| as an integer that orders like the value, with NaN above infinity: a maximum over these keeps
// a NaN, which fmaxf would drop.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// ---- element types ----------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// 16 bytes as 16 / sizeof(T) floats
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&f)[16 / sizeof(T)]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(f[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// x sigmoid(x) within 2^-21 of its value: exp(-x) = 2^t (1 + d ln 2) with t = -x log2(e) rounded and d what the
// rounding and the second part of log2(e) left out, so that only the hardware's exponential (2^-22), the sum and
// the reciprocal (2^-23) round.  Two special-function operations; a range reduction would take two more.
__device__ __forceinline__ float silu(float x) {
  const float t = x * -1.44269502e+00f;
  const float d = fmaf(x, -1.92596303e-08f, fmaf(x, -1.44269502e+00f, -t));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fminf(t, 126.0f)));
  e = fmaf(e * 0.693147182f, d, e) + 1.0f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e));
  return x < -87.0f ? 0.0f : x * r;   // (below -87 the value is above -2^-118)
}
template <int kAct>
__device__ __forceinline__ float activate(float x) {
  if constexpr (kAct == FMOE_ACT_SILU) return silu(x);
  else if constexpr (kAct == FMOE_ACT_GELU) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
  else if constexpr (kAct == FMOE_ACT_RELU) return fmaxf(x, 0.0f);
  else return x;
}
// f(the activation as a compile-time constant): a choice per value, unrolled over a tile, is four times the code,
// and fetching it took a third of the tile's time
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  switch (act) {
    case FMOE_ACT_SILU: f(std::integral_constant<int, FMOE_ACT_SILU>{}); break;
    case FMOE_ACT_GELU: f(std::integral_constant<int, FMOE_ACT_GELU>{}); break;
    case FMOE_ACT_RELU: f(std::integral_constant<int, FMOE_ACT_RELU>{}); break;
    default: f(std::integral_constant<int, FMOE_ACT_IDENTITY>{});
  }
}

// ---- tensor core -------------------------------------------------------------------------------
// Instruction descriptor for kind::f8f6f4: fp32 accumulate (bit 4), A and B e4m3 (format 0), both
// K-major, N >> 3 at [17,23), M >> 4 at [24,29).
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// D[tmem, 256 rows over the pair] (+)= A[smem, 128 rows per CTA] * B[smem, N / 2 rows per CTA]^T over 32
// bytes of K, issued by one thread of the pair's leader.
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One CTA: D[tmem, 128 rows] (+)= A[smem, 128 rows] * B[smem, N rows]^T over 32 bytes of K.
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// ---- programmatic launches ------------------------------------------------------------------------
// Every kernel here is launched so that it may start while the stream's last kernel runs: it sets up, waits for that
// kernel to be complete before it touches global memory, and then lets the next one start likewise.  A kernel
// that waits is complete only after the one before it, so the stream's order holds throughout.  (Inside the expert
// layer a kernel may read before the wait what was complete before the layer began.)
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What another kernel wrote.  A plain load: __ldg promises that the memory never changes while the kernel runs, and could be
// moved in front of the wait.
template <typename T>
__device__ __forceinline__ T fetched(const T* p) { return *p; }

template <typename... Expected, typename... Given>
cudaError_t launch_behind(void (*kernel)(Expected...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                          Given&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  ++g_launches;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// ---- host side -----------------------------------------------------------------------------------
constexpr int kMaxDevices = 64;
// Makes `device` current for the scope and puts the caller's device back.
struct OnDevice {
  int prev = -1;
  cudaError_t err;
  explicit OnDevice(int device) {
    int cur = -1;
    err = cudaGetDevice(&cur);
    if (err == cudaSuccess && cur != device) {
      err = cudaSetDevice(device);
      if (err == cudaSuccess) prev = cur;
    }
  }
  ~OnDevice() { if (prev >= 0) cudaSetDevice(prev); }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};
inline bool misaligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }
// The products.  kInLayer: the stream's last kernel writes A, and everything else was complete before it let this one
// start; kCheckOnly: the arguments are looked at, nothing is launched.
enum class Launch { kPlain, kInLayer, kCheckOnly };
int matmul(const fmoe_fp8_matmul_args* a, Launch how, cudaStream_t stream);
int gated_matmul(const fmoe_fp8_gated_args* a, Launch how, cudaStream_t stream);
inline int element_bytes(int data_type) { return data_type == FMOE_DT_FP32 ? 4 : 2; }

}  // namespace fmoe::fp8
