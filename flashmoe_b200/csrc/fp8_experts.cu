// The expert layer on 8-bit weights as a chain of four launches: quantise the tokens into expert
// order, gated up product (activation and quantisation in its epilogue), down product, weighted sum.
// The first waits for whatever the layer reads from outside before it lets the second start; from there on each
// kernel sets up, and the few-row products fetch their first weights, before they wait for what the one before writes.
// Every CTA of every kernel waits before it ends, so the end of the last one is the end of all.
//
// The down product's rows stay in fp32 until they are summed: in 16 bits they would be half the bytes, a few per cent
// of a large layer's time, and their rounding would add as much error again as the one at the end.
#include "fp8.cuh"

namespace fmoe::fp8 {
namespace {

constexpr int kCombineThreads = 128;

struct CombineParams {
  const float* y;             // [tokens * top_k, dim], expert order
  const int32_t* positions;   // [tokens, top_k]
  const float* weights;       // [tokens, top_k]
  void* out;                  // [tokens, dim]
  int tokens, dim, top_k;
  int parts;                  // CTAs a token
};

// out[t] = sum over j of weights[t, j] * y[positions[t, j]], in fp32 in the order of j; eight values a thread.
template <typename T>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const CombineParams p) {
  wait_for_primary();   // the down product's rows
  const unsigned token = blockIdx.x / static_cast<unsigned>(p.parts);   // (the same for the whole CTA)
  const int col = 8 * static_cast<int>((blockIdx.x - token * p.parts) * kCombineThreads + threadIdx.x);
  if (col >= p.dim) return;
  const long long pairs = static_cast<long long>(p.tokens) * p.top_k;
  float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int j = 0; j < p.top_k; ++j) {
    const long long row = fetched(p.positions + static_cast<size_t>(token) * p.top_k + j);
    const float w = fetched(p.weights + static_cast<size_t>(token) * p.top_k + j);
    if (row < 0 || row >= pairs) continue;
    const float4* y = reinterpret_cast<const float4*>(p.y + row * p.dim + col);
    const float4 a = y[0], b = y[1];
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int x = 0; x < 8; ++x) sum[x] = fmaf(w, v[x], sum[x]);
  }
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + static_cast<size_t>(token) * p.dim + col) = pack16<T>(sum);
}

template <typename T>
cudaError_t launch_combine(CombineParams p, cudaStream_t stream) {
  p.parts = (p.dim / 8 + kCombineThreads - 1) / kCombineThreads;
  return launch_behind(combine_kernel<T>, dim3(static_cast<unsigned>(p.tokens) * static_cast<unsigned>(p.parts)), kCombineThreads,
                       0, 1, stream, p);
}

// Parts of the workspace, each 256-byte aligned.
struct Plan {
  size_t xq, xs, hq, hs, y, total;
};
Plan plan_of(const fmoe_fp8_experts_args& a) {
  const size_t pairs = static_cast<size_t>(a.num_tokens) * a.top_k;
  Plan pl{};
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t here = at; at = (at + bytes + 255) & ~size_t(255); return here; };
  pl.xq = take(pairs * a.token_dim);
  pl.xs = take(pairs * blocks_of(a.token_dim) * sizeof(float));
  pl.hq = take(pairs * a.ffn_size);
  pl.hs = take(pairs * blocks_of(a.ffn_size) * sizeof(float));
  pl.y = take(pairs * a.token_dim * sizeof(float));
  pl.total = at;
  return pl;
}

int check_shape(const fmoe_fp8_experts_args* a) {
  if (a == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "arguments are null");
  if (a->num_tokens < 0 || a->token_dim < 1 || a->ffn_size < 1)
    return set_error(FMOE_ERR_INVALID_ARG, "num_tokens must not be negative, token_dim and ffn_size must be positive");
  if (a->token_dim % 16 != 0 || a->ffn_size % 16 != 0)
    return set_error(FMOE_ERR_INVALID_ARG, "token_dim and ffn_size must be multiples of 16");
  if (a->num_experts < 1 || a->num_experts > 1024) return set_error(FMOE_ERR_INVALID_ARG, "num_experts must be between 1 and 1024");
  if (a->top_k < 1 || a->top_k > 32 || a->top_k > a->num_experts)
    return set_error(FMOE_ERR_INVALID_ARG, "top_k must not exceed num_experts (or 32)");
  if (a->data_type != FMOE_DT_BF16 && a->data_type != FMOE_DT_FP16)
    return set_error(FMOE_ERR_UNSUPPORTED, "the 8-bit expert layer handles BF16 and FP16 tokens");
  if (static_cast<long long>(a->num_tokens) * a->top_k > 0x7fff0000ll)
    return set_error(FMOE_ERR_UNSUPPORTED, "num_tokens * top_k must fit 32 bits");
  if (static_cast<long long>(a->num_tokens) * (a->token_dim / (8 * kCombineThreads) + 1) > 0x7fff0000ll)
    return set_error(FMOE_ERR_UNSUPPORTED, "num_tokens * token_dim is more than a grid holds (32 bits of CTAs)");
  return FMOE_OK;
}

}  // namespace
}  // namespace fmoe::fp8

using namespace fmoe;
using namespace fmoe::fp8;

extern "C" {

int fmoe_fp8_workspace_bytes(const fmoe_fp8_experts_args* a, int64_t* bytes_out) {
  const int rc = check_shape(a);
  if (rc != FMOE_OK) return rc;
  if (bytes_out == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "bytes_out is null");
  *bytes_out = static_cast<int64_t>(plan_of(*a).total);
  return FMOE_OK;
}

int fmoe_fp8_experts(const fmoe_fp8_experts_args* a, void* stream) {
  int rc = check_shape(a);
  if (rc != FMOE_OK) return rc;
  if (a->device_id < 0 || a->device_id >= kMaxDevices) return set_error(FMOE_ERR_INVALID_ARG, "device_id out of range");
  if (a->act_type < FMOE_ACT_IDENTITY || a->act_type > FMOE_ACT_RELU) return set_error(FMOE_ERR_INVALID_ARG, "unknown act_type");
  if (a->num_tokens == 0) return FMOE_OK;
  if (a->tokens == nullptr || a->offsets == nullptr || a->positions == nullptr || a->weights == nullptr || a->up == nullptr ||
      a->up_scale == nullptr || a->down == nullptr || a->down_scale == nullptr || a->out == nullptr)
    return set_error(FMOE_ERR_INVALID_ARG, "tokens, offsets, positions, weights, up, down, their scales and out are required");
  if (misaligned(a->tokens, 16) || misaligned(a->out, 16) || misaligned(a->down, 16))
    return set_error(FMOE_ERR_INVALID_ARG, "tokens, down and out must be 16-byte aligned");
  if (misaligned(a->positions, 4) || misaligned(a->weights, 4) || misaligned(a->down_scale, 4))
    return set_error(FMOE_ERR_INVALID_ARG, "positions, weights and scales must be 4-byte aligned");
  const Plan pl = plan_of(*a);
  if (a->workspace == nullptr || a->workspace_bytes < static_cast<int64_t>(pl.total))
    return set_error(FMOE_ERR_INVALID_ARG, "the workspace holds " + std::to_string(a->workspace ? a->workspace_bytes : 0) +
                                               " bytes; this layer needs " + std::to_string(pl.total));
  if (misaligned(a->workspace, 256)) return set_error(FMOE_ERR_INVALID_ARG, "workspace must be 256-byte aligned");
  unsigned char* ws = static_cast<unsigned char*>(a->workspace);
  const int pairs = a->num_tokens * a->top_k;
  const fmoe_fp8_quantize_args quantize{a->tokens, ws + pl.xq, reinterpret_cast<float*>(ws + pl.xs), a->positions, a->top_k,
                                        a->num_tokens, a->token_dim, 1, 1, a->data_type, a->device_id};
  const fmoe_fp8_gated_args gated{ws + pl.xq, reinterpret_cast<float*>(ws + pl.xs), a->up, a->up_scale, a->up_v, a->up_v_scale,
                                  ws + pl.hq, reinterpret_cast<float*>(ws + pl.hs), a->offsets, pairs, a->ffn_size,
                                  a->token_dim, a->num_experts, a->act_type, a->device_id};
  const fmoe_fp8_matmul_args down{ws + pl.hq, reinterpret_cast<float*>(ws + pl.hs), a->down, a->down_scale, ws + pl.y, a->offsets,
                                  pairs, a->token_dim, a->ffn_size, a->num_experts, FMOE_DT_FP32, a->device_id};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = gated_matmul(&gated, Launch::kCheckOnly, st);   // what any of the steps refuses is refused before the first
  if (rc == FMOE_OK) rc = matmul(&down, Launch::kCheckOnly, st);
  if (rc == FMOE_OK) rc = fmoe_fp8_quantize(&quantize, stream);
  if (rc == FMOE_OK) rc = gated_matmul(&gated, Launch::kInLayer, st);
  if (rc == FMOE_OK) rc = matmul(&down, Launch::kInLayer, st);
  if (rc != FMOE_OK) return rc;
  OnDevice on(a->device_id);
  if (on.err != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(on.err));
  const CombineParams c{reinterpret_cast<float*>(ws + pl.y), a->positions, a->weights, a->out, a->num_tokens, a->token_dim, a->top_k, 0};
  const cudaError_t e = a->data_type == FMOE_DT_BF16 ? launch_combine<__nv_bfloat16>(c, st)
                                                     : launch_combine<__half>(c, st);
  if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("combine launch: ") + cudaGetErrorString(e));
  return FMOE_OK;
}

}  // extern "C"
