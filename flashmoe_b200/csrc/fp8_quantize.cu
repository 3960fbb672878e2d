// Quantisation to e4m3 with a scale per block: rows in 1 x 128 blocks (optionally laid out by
// expert on the way), weights in 128 x 128 blocks.  Each value is read once and kept in registers
// between the maximum and the rounding.  Bound by HBM: 8192 x 5120 bf16 in 20.9 to 21.8 us (5.8 to 6.1 TB/s, 89 to
// 93 % of the copy rate), 8 x 1400 x 2064 weights in 13 us (5.3 TB/s).
#include "fp8.cuh"

namespace fmoe::fp8 {
namespace {

struct QuantizeParams {
  const void* x;
  unsigned char* q;
  float* scale;
  const int32_t* positions;   // rows: [rows, copies] or null
  int copies;
  int rows, cols;
  int row_blocks, col_blocks;
  unsigned long long per_row;   // rows: 2^64 / col_blocks + 1
};

// A thread's share of a block, kPieces pieces of 16 bytes: as loaded, their largest value, their codes.
template <typename T, int kPieces>
struct Raw {
  static constexpr int kPer = 16 / sizeof(T);   // values of a piece
  uint4 u[kPieces];
  // The largest |x|, as bits that order like the value (16-bit types: their own bits, two at a time).
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) m = max(m, w[j] & 0x7fffffffu);
        else m = __vmaxu2(m, w[j] & 0x7fff7fffu);
      }
    }
    if constexpr (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
    return m;
  }
  __device__ __forceinline__ static float amax_value(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(bits << 16);
    else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
  // four codes to a word
  __device__ __forceinline__ void codes(const Quantizer& z, uint32_t (&w)[kPieces * kPer / 4]) const {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      float f[kPer];
      unpack16<T>(u[i], f);
#pragma unroll
      for (int j = 0; j < kPer / 4; ++j) {
        const float2 a = z.scaled(f[4 * j], f[4 * j + 1]), b = z.scaled(f[4 * j + 2], f[4 * j + 3]);
        w[i * (kPer / 4) + j] = to_e4m3x4(a.x, a.y, b.x, b.y);
      }
    }
  }
};
template <typename T>
struct Raw16 : Raw<T, sizeof(T)> {   // 16 consecutive values
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) this->u[i] = fetched(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) this->u[i] = make_uint4(0, 0, 0, 0);
  }
};

// A block of 128 by kLanes threads, whose pieces of 16 bytes alternate, so that a load and a store of theirs lie side by
// side.  What a block costs besides its values (its place, the reciprocal, the scale) is shared by few lanes: with
// eight a block, 16 values each, that was half of the instructions.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantizeParams p) {
  wait_for_primary();
  launch_dependents();
  constexpr int kLanes = 4, kPer = 16 / sizeof(T), kPieces = kBlock / kPer / kLanes;
  const int sub = threadIdx.x & (kLanes - 1);
  const uint32_t block = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;   // (the host sees to it that it fits)
  // block / col_blocks: the high half of block * (2^64 / col_blocks + 1) (exact for 32-bit numbers)
  const uint32_t row = p.col_blocks == 1 ? block : static_cast<uint32_t>(__umul64hi(block, p.per_row));
  const int cb = static_cast<int>(block - row * p.col_blocks), col = cb * kBlock + sub * kPer;
  const bool live = row < static_cast<uint32_t>(p.rows);
  const T* x = static_cast<const T*>(p.x) + static_cast<size_t>(row) * p.cols + col;
  Raw<T, kPieces> raw;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    raw.u[i] = make_uint4(0, 0, 0, 0);
    if (live && col + i * kLanes * kPer < p.cols) raw.u[i] = fetched(reinterpret_cast<const uint4*>(x + i * kLanes * kPer));
  }
  uint32_t m = raw.amax_bits();
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (!live) return;
  const float amax = raw.amax_value(m);
  uint32_t codes[kPieces * kPer / 4];
  raw.codes(Quantizer(amax), codes);
  for (int j = 0; j < p.copies; ++j) {
    long long to = row;
    if (p.positions != nullptr) {
      to = fetched(p.positions + static_cast<size_t>(row) * p.copies + j);
      if (to < 0 || to >= static_cast<long long>(p.rows) * p.copies) continue;
    }
    unsigned char* q = p.q + to * p.cols + col;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (col + i * kLanes * kPer < p.cols) {
        if constexpr (kPer == 8) *reinterpret_cast<uint2*>(q + i * kLanes * kPer) = make_uint2(codes[2 * i], codes[2 * i + 1]);
        else *reinterpret_cast<uint32_t*>(q + i * kLanes * kPer) = codes[i];
      }
    }
    if (sub == 0) p.scale[to * p.col_blocks + cb] = block_scale(amax);
  }
}

// One CTA a block of 128 x 128: a pass takes 32 rows, eight threads each; four passes stay in registers.
template <typename T>
__global__ void __launch_bounds__(256) quantize_weights_kernel(const QuantizeParams p) {
  wait_for_primary();
  launch_dependents();
  __shared__ uint32_t s_max[8];
  const long long matrix = blockIdx.y;
  const int rb = blockIdx.x / p.col_blocks, cb = blockIdx.x - rb * p.col_blocks;
  const int row0 = rb * kBlock + (threadIdx.x >> 3), col = cb * kBlock + (threadIdx.x & 7) * 16;
  const size_t base = static_cast<size_t>(matrix) * p.rows * p.cols + col;
  Raw16<T> raw[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    raw[i].zero();
    if (row0 + 32 * i < p.rows && col < p.cols)
      raw[i].load(static_cast<const T*>(p.x) + base + static_cast<size_t>(row0 + 32 * i) * p.cols);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, raw[i].amax_bits());
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, s_max[i]);
  const float amax = Raw16<T>::amax_value(m);
  const Quantizer z(amax);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (row0 + 32 * i < p.rows && col < p.cols) {
      uint32_t w[4];
      raw[i].codes(z, w);
      *reinterpret_cast<uint4*>(p.q + base + static_cast<size_t>(row0 + 32 * i) * p.cols) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (threadIdx.x == 0) p.scale[(matrix * p.row_blocks + rb) * p.col_blocks + cb] = block_scale(amax);
}

template <typename T>
cudaError_t launch(const QuantizeParams& p, int block_rows, int matrices, cudaStream_t stream) {
  if (block_rows == 1) {
    const long long blocks = static_cast<long long>(p.rows) * p.col_blocks;
    return launch_behind(quantize_rows_kernel<T>, dim3(static_cast<unsigned>((blocks + 63) / 64)), 256, 0, 1, stream, p);
  }
  return launch_behind(quantize_weights_kernel<T>, dim3(static_cast<unsigned>(p.row_blocks * p.col_blocks), matrices), 256, 0,
                       1, stream, p);
}

}  // namespace
}  // namespace fmoe::fp8

extern "C" int fmoe_fp8_quantize(const fmoe_fp8_quantize_args* a, void* stream) {
  using namespace fmoe;
  using namespace fmoe::fp8;
  if (a == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "arguments are null");
  if (a->rows < 0 || a->num_matrices < 0 || a->cols < 1)
    return set_error(FMOE_ERR_INVALID_ARG, "rows and num_matrices must not be negative, cols must be positive");
  if (a->cols % 16 != 0) return set_error(FMOE_ERR_INVALID_ARG, "cols must be a multiple of 16");
  if (a->block_rows != 1 && a->block_rows != kBlock)
    return set_error(FMOE_ERR_INVALID_ARG, "block_rows must be 1 (rows) or 128 (weights)");
  if (a->data_type != FMOE_DT_BF16 && a->data_type != FMOE_DT_FP16 && a->data_type != FMOE_DT_FP32)
    return set_error(FMOE_ERR_UNSUPPORTED, "BF16, FP16 and FP32 can be quantised");
  if (a->device_id < 0 || a->device_id >= kMaxDevices) return set_error(FMOE_ERR_INVALID_ARG, "device_id out of range");
  if (a->positions != nullptr && (a->block_rows != 1 || a->num_matrices != 1))
    return set_error(FMOE_ERR_INVALID_ARG, "positions go with block_rows 1 and one matrix");
  if (a->copies < 1 || (a->positions == nullptr && a->copies != 1))
    return set_error(FMOE_ERR_INVALID_ARG, "copies must be positive, and 1 without positions");
  if (static_cast<long long>(a->rows) * a->copies > 0x7fffffffll)
    return set_error(FMOE_ERR_UNSUPPORTED, "rows * copies must fit 32 bits");
  if (a->rows == 0 || a->num_matrices == 0) return FMOE_OK;
  if (a->x == nullptr || a->q == nullptr || a->scale == nullptr)
    return set_error(FMOE_ERR_INVALID_ARG, "x, q and scale are required");
  if (misaligned(a->x, 16) || misaligned(a->q, 16)) return set_error(FMOE_ERR_INVALID_ARG, "x and q must be 16-byte aligned");
  if (misaligned(a->scale, 4) || misaligned(a->positions, 4))
    return set_error(FMOE_ERR_INVALID_ARG, "scale and positions must be 4-byte aligned");
  QuantizeParams p{a->x, static_cast<unsigned char*>(a->q), a->scale, a->positions, a->copies, a->rows, a->cols, 0, 0, 0};
  p.row_blocks = a->block_rows == 1 ? a->rows : blocks_of(a->rows);
  p.col_blocks = blocks_of(a->cols);
  p.per_row = ~0ull / p.col_blocks + 1;
  int matrices = a->num_matrices;
  if (a->block_rows == 1) {   // rows of several matrices are just more rows
    if (static_cast<long long>(a->rows) * matrices > 0x7fffffffll)
      return set_error(FMOE_ERR_UNSUPPORTED, "rows * num_matrices must fit 32 bits");
    p.rows *= matrices;
    p.row_blocks = p.rows;
    matrices = 1;
    if (static_cast<long long>(p.rows) * p.col_blocks > 0xffffff00ll)
      return set_error(FMOE_ERR_UNSUPPORTED, "more blocks than a grid holds");
  } else if (matrices > 65535 || static_cast<long long>(p.row_blocks) * p.col_blocks > 0x7fffffffll) {
    return set_error(FMOE_ERR_UNSUPPORTED, "at most 65535 matrices, and blocks of one must fit 32 bits");
  }
  OnDevice on(a->device_id);
  if (on.err != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(on.err));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->data_type == FMOE_DT_BF16) e = launch<__nv_bfloat16>(p, a->block_rows, matrices, st);
  else if (a->data_type == FMOE_DT_FP16) e = launch<__half>(p, a->block_rows, matrices, st);
  else e = launch<float>(p, a->block_rows, matrices, st);
  if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("quantize launch: ") + cudaGetErrorString(e));
  return FMOE_OK;
}
