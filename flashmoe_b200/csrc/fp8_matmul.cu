// Products of 8-bit matrices with block scales on the tensor cores, dense and by expert:
//
//   out[r, f] = sum over 128-blocks b of k:  sa[r, b] * sw[f / 128, b] * (sum over i in b of a[r, i] w[f, i])
//
// The inner sums are tcgen05 products of e4m3 (exact products, fp32 accumulation in TMEM), one
// TMEM accumulator per block of k; the outer sum is taken by the epilogue warps, which read each
// block's accumulator, scale it and add it to fp32 registers.  The tensor core never sees a scale, so
// any fp32 scales work, and no sum crosses a block boundary unscaled.
//
// CTA pairs (clusters of two SMs) work on tiles of 256 rows x 256 features (the gated form: 128 features of
// up and the same 128 of up_v) with cta_group::2 MMAs: each CTA fetches and accumulates its own 128
// rows, and half of the weight tile, which the pair's tensor cores share.  A CTA alone would move 48 KB
// through shared memory per 512 cycles of MMA, in and out again, which is more than shared memory passes;
// a pair's CTAs move 32 KB.  In a CTA, warp 0 loads tiles (TMA), warp 1 of the leader issues the MMAs,
// warps 2 and 3 fetch scales, warps 4..11 scale and add.  The two TMEM accumulators of 256 columns
// let the MMAs of one block run while the other block's sums are read.  The same kernel works 128 x 256 tiles by
// one CTA, for products too small, or experts with too few rows, to fill 256 x 256.
//
// Measured: 8192^3 575 to 593 us (1855 to 1910 TFLOP/s), 4096 x 14336 x 4096 266 us (1810).  A block of k takes a pair about 1050
// cycles: 512 of MMA, 440 to read and multiply-add 256 columns, 600 for the accumulator to change hands twice, over
// two accumulators.  The MMAs alone would run at 3300.
#include <atomic>
#include <cstdlib>
#include <mutex>
#include <type_traits>

#include "fp8.cuh"

namespace fmoe::fp8 {
namespace {

using namespace fmoe::ptx;

// TMA warp, MMA warp, two warps that fetch scales, then the epilogue warps: four per 128 rows and
// kColumnWarps of those side by side along the columns.
constexpr int kScaleWarp = 2, kScaleWarps = 2, kScaleSlots = 2, kScaleBlocks = 4, kEpilogueWarp = 4;
constexpr int kColumnWarps = 2, kEpilogueWarps = 4 * kColumnWarps, kThreads = 32 * (kEpilogueWarp + kEpilogueWarps);
constexpr int kRun = 128 / kColumnWarps;   // columns of one weight block that a warp adds up
// Registers a thread: 168 at launch (384 threads), then 88 and 208: 4 * 88 + 8 * 208 = 12 * 168.
constexpr int kLoadRegs = 88, kEpilogueRegs = 208;
constexpr int kMaxExperts = 1024;
constexpr uint32_t kBoxBytes = 128 * kBlock;   // 128 rows of one k block: 16 KB

struct Codes {};   // "output type" of the gated form

__device__ fmoe_status g_status;   // first wait that ran out (fmoe_fp8_last_status)

struct ProductParams {
  int m, n, k;
  int kblocks, nblocks;        // 128-blocks along k and n
  int experts, tiles_n;
  const int32_t* offsets;      // null: one product over all m rows
  const float* a_scale;
  const float* w_scale[2];     // the gated form: up, up_v
  void* out;                   // rows, or the codes of the gated form
  float* out_scale;            // gated form
  int act, has_v;              // gated form
  int wide;                    // output rows may be stored 32 bytes at a time
  int in_layer;                // weights and offsets may be read before the wait for the kernel that writes A
  long long spin_limit;
};

struct Tile {
  int expert, row0, row_end, n0;
};

// How many tiles come before each expert's; filled once per CTA.
struct TileTable {
  int first[kMaxExperts + 1];
};

// An expert's rows: whatever the array of offsets holds, they stay inside [0, m).
__device__ __forceinline__ void expert_rows(const ProductParams& p, int e, int& begin, int& end) {
  begin = 0;
  end = p.m;
  if (p.offsets != nullptr) {
    begin = min(max(fetched(p.offsets + e), 0), p.m);
    end = min(max(fetched(p.offsets + e + 1), begin), p.m);
  }
}

__device__ __forceinline__ bool find_tile(const TileTable& t, const ProductParams& p, int tile, int tile_m, int tile_n, Tile& out) {
  if (tile >= t.first[p.experts]) return false;
  int lo = 0, hi = p.experts - 1;
  while (lo < hi) {                      // the last expert that begins at or before this tile
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  int begin, end;
  expert_rows(p, lo, begin, end);
  const int m_tiles = (end - begin + tile_m - 1) / tile_m, i = tile - t.first[lo];
  out.expert = lo;                       // rows first: neighbouring CTAs share a weight tile
  out.row0 = begin + (i % m_tiles) * tile_m;
  out.row_end = end;
  out.n0 = (i / m_tiles) * tile_n;
  return true;
}

// Called by every thread; the tile counts are summed by warp 0.  With offsets that make sense the sums fit (the host
// checks); with others they stop at a number that a stride of the grid does not overflow.
constexpr long long kMostTiles = 0x7fff0000;
__device__ void fill_table(TileTable& t, const ProductParams& p, int tile_m) {
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int begin, end;
    expert_rows(p, e, begin, end);
    t.first[e] = ((end - begin + tile_m - 1) / tile_m) * p.tiles_n;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    long long before = 0;
    for (int e0 = 0; e0 < p.experts; e0 += 32) {
      const int e = e0 + threadIdx.x;
      const int own = e < p.experts ? t.first[e] : 0;
      long long sum = own;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, d);
        if (static_cast<int>(threadIdx.x) >= d) sum += v;
      }
      if (e < p.experts) t.first[e] = static_cast<int>(min(before + sum - own, kMostTiles));
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (threadIdx.x == 0) t.first[p.experts] = static_cast<int>(min(before, kMostTiles));
  }
  __syncthreads();
}

__device__ __noinline__ void wait_failed(volatile uint32_t* abort_word, int phase, int detail) {
  if (atomicCAS(&g_status.code, FMOE_OK, FMOE_ERR_DEVICE_TIMEOUT) == FMOE_OK) {
    g_status.phase = phase;
    g_status.rank = 0;
    g_status.cta = blockIdx.x;
    g_status.detail = detail;
  }
  *abort_word = 1;
}

__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Waits for this thread's TMEM loads; naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait_16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Arrives on a barrier of either CTA of the pair.  What it announces is that TMEM has been read, which tcgen05's
// own wait and fence order; no memory another CTA looks at, so it needs no release: a release at cluster scope
// waits for everything the warp has in flight, which halved the rate of the whole kernel.
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One lane of a converged warp.  What this predicate guards the compiler knows to be one thread's, so that TMA and
// tcgen05 operands go straight to uniform registers; behind `lane == 0` each such instruction becomes a loop
// over the active lanes (about 90 cycles an MMA).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// A bounded wait by a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const WaitCtx& wc) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, wc));
}

__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// kN features of each of a warp's 32 rows (a lane each), in order in acc (pairs), to dst (the first row's, rows
// `pitch` apart); `rows` and `valid` of them exist.  Rows that keep to 32 bytes are stored from the registers, whole
// sectors at a time; others pass through shared memory, 16 columns at a time, and leave with the lanes along the row.
template <typename Out, int kN>
__device__ __forceinline__ void store_features(Out* dst, size_t pitch, const uint64_t* acc, int rows, int valid, bool wide,
                                               float (*stage)[17], int lane) {
  constexpr int kPer = 32 / sizeof(Out);
  if (wide) {
    if (lane >= rows) return;
    dst += lane * pitch;
#pragma unroll
    for (int g = 0; g < kN / kPer; ++g) {
      if ((g + 1) * kPer > valid) break;   // (rows are a multiple of 32 bytes, so is what is left)
      uint32_t w[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float h[kPer / 2];
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) {
          const float2 v = unpack2(acc[g * (kPer / 2) + q * (kPer / 4) + i]);
          h[2 * i] = v.x;
          h[2 * i + 1] = v.y;
        }
        const uint4 u = pack16<Out>(h);
        w[4 * q] = u.x; w[4 * q + 1] = u.y; w[4 * q + 2] = u.z; w[4 * q + 3] = u.w;
      }
      st_global_32(dst + g * kPer, w);
    }
  } else {
#pragma unroll
    for (int g = 0; g < kN / 16; ++g) {
      if (g * 16 >= valid) break;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = unpack2(acc[g * 8 + i]);
        stage[lane][2 * i] = v.x;
        stage[lane][2 * i + 1] = v.y;
      }
      __syncwarp();
      const int col = g * 16 + (lane & 15);
      for (int r = lane >> 4; r < rows; r += 2)
        if (col < valid) dst[r * pitch + col] = from_float<Out>(stage[r][lane & 15]);
      __syncwarp();
    }
  }
}

// A place in the ring of stages, and the parity of the round it is in.
template <int kStages>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// A pair's CTA holds 128 rows of each operand, a CTA alone 128 rows and 256 features.
template <bool kPair>
struct Wide {
  static constexpr int kStages = kPair ? 6 : 4;
  static constexpr uint32_t kStageBytes = (kPair ? 2 : 3) * kBoxBytes;
  struct Tail;
  static constexpr size_t smem_bytes();
};
template <bool kPair>
struct Wide<kPair>::Tail {
  uint64_t full[kStages];         // the leader's: both CTAs' copies of the stage have landed
  uint64_t done[kStages];         // each CTA's: the MMAs of the stage are done: it is free, its sums are in TMEM
  uint64_t acc_empty[2];          // the leader's: both CTAs have read it
  uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];   // each CTA's
  uint64_t amax_full[4];          // all maxima of a quarter's rows are in
  uint32_t tmem_base;
  uint32_t abort_word;
  float scale[kScaleSlots][kScaleBlocks][2][128];   // [block of k][weight block][row]: a's scale times w's
  uint32_t amax[2][kColumnWarps][128];     // [tile parity]
  float stage[kEpilogueWarps][32][17];     // output rows on their way, 16 columns at a time
  TileTable table;
};
template <bool kPair>
constexpr size_t Wide<kPair>::smem_bytes() { return 1024 + kStages * kStageBytes + sizeof(Tail); }
static_assert(Wide<true>::smem_bytes() <= 227 * 1024 && Wide<false>::smem_bytes() <= 227 * 1024, "shared memory of one CTA");

// Rows on the TMEM lanes, features on its columns.
template <typename Out, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w0,
               const __grid_constant__ CUtensorMap map_w1, const ProductParams p) {
  constexpr bool kGated = std::is_same_v<Out, Codes>;
  constexpr int kCtas = kPair ? 2 : 1, kTileM = 128 * kCtas, kTileN = kGated ? 128 : 256;
  using W = Wide<kPair>;
  constexpr int kStages = W::kStages;
  constexpr uint32_t kStageBytes = W::kStageBytes;
  extern __shared__ __align__(16) unsigned char s_raw[];
  unsigned char* ring = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);   // swizzle atoms are 1024 bytes
  auto& sh = *reinterpret_cast<typename W::Tail*>(ring + kStages * kStageBytes);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // (uniform to the compiler)
  const uint32_t rank = kPair ? cluster_ctarank() : 0;
  const int pair = blockIdx.x / kCtas, pairs = gridDim.x / kCtas;
  const WaitCtx wc{&sh.abort_word, p.spin_limit};

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.done[i], 1); }
    for (int i = 0; i < 2; ++i) mbar_init(&sh.acc_empty[i], kCtas * kEpilogueWarps);
    for (int i = 0; i < 4; ++i) mbar_init(&sh.amax_full[i], kColumnWarps);
    for (int i = 0; i < kScaleSlots; ++i) {
      mbar_init(&sh.scale_full[i], kScaleWarps);
      mbar_init(&sh.scale_empty[i], kEpilogueWarps);
    }
    sh.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(&sh.tmem_base, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&sh.tmem_base, 512);
      tmem_relinquish();
    }
  }
  if (!p.in_layer) wait_for_primary();
  fill_table(sh.table, p, kTileM);
  if constexpr (kPair) cluster_sync_all();   // both CTAs' barriers exist before either is signalled from the other
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_base;
  const bool second = !kGated || p.has_v != 0;   // whether the second 128 weight rows exist
  launch_dependents();
  if (p.in_layer) wait_for_primary();

  if (warp < kEpilogueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLoadRegs));
    if (warp == 0) {
      // a plain MLP has no second weight tile: its follower loads the first one again, into columns nobody reads
      const CUtensorMap* map_w = rank == 0 ? &map_w0 : &map_w1;
      Ring<kStages> at;
      Tile t;
      bool ok = true;
      for (int i = pair; ok && find_tile(sh.table, p, i, kTileM, kTileN, t); i += pairs) {
        const int row = t.row0 + static_cast<int>(rank) * 128;
        const int w_row = t.expert * p.n + t.n0 + (kGated ? 0 : static_cast<int>(rank) * 128);   // (fits: checked by the host)
        for (int kb = 0; kb < p.kblocks; ++kb) {
          ok = warp_wait(&sh.done[at.stage], at.phase ^ 1, wc);
          if (!ok) break;
          if (elect_one()) {
            unsigned char* stage = ring + at.stage * kStageBytes;
            if constexpr (kPair) {
              if (rank == 0) mbar_expect_tx(&sh.full[at.stage], 2 * kStageBytes);
              tma_load_2d_pair(stage, &map_a, &sh.full[at.stage], kb * kBlock, row);
              tma_load_2d_pair(stage + kBoxBytes, map_w, &sh.full[at.stage], kb * kBlock, w_row);
            } else {
              mbar_expect_tx(&sh.full[at.stage], (second ? 3 : 2) * kBoxBytes);
              tma_load_2d(stage, &map_a, &sh.full[at.stage], kb * kBlock, row);
              tma_load_2d(stage + kBoxBytes, &map_w0, &sh.full[at.stage], kb * kBlock, w_row);
              if (second)
                tma_load_2d(stage + 2 * kBoxBytes, &map_w1, &sh.full[at.stage], kb * kBlock, kGated ? w_row : w_row + 128);
            }
          }
          __syncwarp();
          at.next();
        }
        if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_PIPE_EMPTY, i);
      }
      // no copy may be in flight when the CTA leaves: the MMAs that free a stage come after its copies
      const WaitCtx last{nullptr, p.spin_limit};
      for (int j = 0; j < kStages; ++j) {   // (a stage that was never filled passes at once)
        mbar_wait(&sh.done[at.stage], at.phase ^ 1, last);
        at.next();
      }
    } else if (warp == 1) {
      if (rank == 0) {
        const uint32_t idesc = kPair ? umma_idesc_e4m3(256, 256) : umma_idesc_e4m3(128, second ? 256 : 128);
        const uint64_t desc0 = umma_desc_sw128(smem_u32(ring));
        Ring<kStages> at;
        uint32_t b = 0, b_phase = 1, last_stage = 0, last_phase = 1;
        Tile t;
        bool ok = true;
        for (int i = pair; ok && find_tile(sh.table, p, i, kTileM, kTileN, t); i += pairs) {
          for (int kb = 0; kb < p.kblocks; ++kb) {
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[at.stage], at.phase, wc) && mbar_wait(&sh.acc_empty[b], b_phase, wc));
            if (!ok) break;
            tc_fence_after_sync();
            if (elect_one()) {
              const uint64_t da = desc0 + at.stage * (kStageBytes >> 4), dw = da + (kBoxBytes >> 4);
#pragma unroll
              for (int q = 0; q < 4; ++q) {   // 32 bytes of k each
                if constexpr (kPair) umma_f8_pair(tmem + b * 256, da + 2 * q, dw + 2 * q, idesc, q != 0);
                else umma_f8(tmem + b * 256, da + 2 * q, dw + 2 * q, idesc, q != 0);
              }
              if constexpr (kPair) umma_commit_pair(&sh.done[at.stage], 3);
              else umma_commit(&sh.done[at.stage]);
            }
            __syncwarp();
            last_stage = at.stage;
            last_phase = at.phase;
            at.next();
            b ^= 1;
            b_phase ^= b == 0;
          }
          if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_PIPE_FULL, i);
        }
        // no MMA may be running when TMEM is freed
        const WaitCtx last{nullptr, p.spin_limit};
        mbar_wait(&sh.done[last_stage], last_phase, last);
      }
    } else {
      // The scales of a block of k go with its accumulator: two rows a lane, loaded four blocks at a time
      // and four to eight blocks ahead, so that the epilogue never waits for global memory.
      const int r0 = (warp - kScaleWarp) * 64 + lane;
      int done = 0;
      Tile t;
      bool ok = true;
      for (int i = pair; ok && find_tile(sh.table, p, i, kTileM, kTileN, t); i += pairs) {
        const float* src[4] = {nullptr, nullptr, nullptr, nullptr};   // this lane's two rows, the two weight blocks
        for (int j = 0; j < 2; ++j) {
          const int row = t.row0 + static_cast<int>(rank) * 128 + r0 + 32 * j, nb = t.n0 / kBlock + (kGated ? 0 : j);
          if (row < t.row_end) src[j] = p.a_scale + static_cast<size_t>(row) * p.kblocks;
          const float* w = p.w_scale[kGated ? j : 0];
          if (nb < p.nblocks && w != nullptr) src[2 + j] = w + (static_cast<size_t>(t.expert) * p.nblocks + nb) * p.kblocks;
        }
        float now[4][4], next[4][4];   // [block][source]
        auto fetch = [&](int kb, float (&to)[4][4]) {
  #pragma unroll
          for (int x = 0; x < 4; ++x)
  #pragma unroll
            for (int j = 0; j < 4; ++j) to[x][j] = src[j] != nullptr && kb + x < p.kblocks ? fetched(src[j] + kb + x) : 0.0f;
        };
        fetch(0, next);
        for (int kb0 = 0; ok && kb0 < p.kblocks; kb0 += 4) {
  #pragma unroll
          for (int x = 0; x < 4; ++x)
  #pragma unroll
            for (int j = 0; j < 4; ++j) now[x][j] = next[x][j];
          fetch(kb0 + 4, next);
          const int slot = done % kScaleSlots;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.scale_empty[slot], ((done / kScaleSlots) & 1) ^ 1, wc));
          if (!ok) break;
  #pragma unroll
          for (int x = 0; x < 4; ++x)
  #pragma unroll
            for (int j = 0; j < 2; ++j)
  #pragma unroll
              for (int h = 0; h < 2; ++h) sh.scale[slot][x][h][r0 + 32 * j] = now[x][j] * now[x][2 + h];
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.scale_full[slot]);
          ++done;
        }
        if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TMEM_EMPTY, i);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpilogueRegs));
    // This warp's 32 rows and 256 / kColumnWarps columns, as two runs of kRun: of both weight blocks in the gated
    // form (the same features of up and up_v), one after the other in the plain form.
    const int quarter = warp & 3, column_warp = (warp - kEpilogueWarp) >> 2;
    constexpr int kSecond = kGated ? 128 : kRun;                        // where the second run begins
    const int column0 = column_warp * (kGated ? kRun : 2 * kRun);
    const int block0 = kGated ? 0 : column_warp * 2 / kColumnWarps, block1 = kGated ? 1 : block0;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + column0;
    const int r = quarter * 32 + lane;
    uint32_t acc_empty[2] = {0, 0};
    if constexpr (kPair) {
      acc_empty[0] = map_to_cta(&sh.acc_empty[0], 0);
      acc_empty[1] = map_to_cta(&sh.acc_empty[1], 0);
    }
    Ring<kStages> at;
    int b = 0, groups = 0, parity = 0;
    Tile t;
    bool ok = true;
    for (int i = pair; ok && find_tile(sh.table, p, i, kTileM, kTileN, t); i += pairs, parity ^= 1) {
      const int row = t.row0 + static_cast<int>(rank) * 128 + r;
      const bool live = row < t.row_end, any_live = row - lane < t.row_end;   // (any: the same for the whole warp)
      uint64_t acc[kRun];   // pairs of columns: the first run's, then the second's
#pragma unroll
      for (int j = 0; j < kRun; ++j) acc[j] = 0;
      constexpr int kChunks = kRun / 8;   // of 16 columns
      auto column = [&](int c) { return c < kChunks / 2 ? c * 16 : kSecond + (c - kChunks / 2) * 16; };
#pragma unroll 1
      for (int kb = 0; kb < p.kblocks; ++kb) {   // (a wait that fails goes on: nothing is stored then)
        const int slot = groups % kScaleSlots, x = kb % kScaleBlocks;
        if (x == 0) ok = mbar_wait(&sh.scale_full[slot], (groups / kScaleSlots) & 1, wc) && ok;
        const float f0 = sh.scale[slot][x][block0][r], f1 = kGated ? sh.scale[slot][x][block1][r] : f0;
        ok = mbar_wait(&sh.done[at.stage], at.phase, wc) && ok;
        __syncwarp();
        tc_fence_after_sync();
        const uint64_t s0 = pack2(f0, f0), s1 = kGated ? pack2(f1, f1) : s0;
        // chunk by chunk; the accumulator goes back as soon as the last one has been read (the branch over rows that do
        // not exist pays where tiles are half empty; in the pair kernel it costs 6 % of 8192^3)
        uint32_t d[16];
        auto add = [&](int c) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            acc[c * 8 + j] = fma2(pack2(d[2 * j], d[2 * j + 1]), c < kChunks / 2 ? s0 : s1, acc[c * 8 + j]);
        };
        if (kPair || any_live) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            tmem_ld_16(taddr + b * 256 + column(c), d);
            tmem_wait_16(d);
            if (c + 1 < kChunks) add(c);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) arrive_at(acc_empty[b]);
          else mbar_arrive(&sh.acc_empty[b]);
        }
        if (x == kScaleBlocks - 1 || kb + 1 == p.kblocks) {
          if (lane == 0) mbar_arrive(&sh.scale_empty[slot]);
          ++groups;
        }
        if (kPair || any_live) add(kChunks - 1);
        at.next();
        b ^= 1;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TMEM_FULL, i);
        break;
      }
      if constexpr (kGated) {
        // h = act(up) * up_v of this warp's features; the block's maximum with the row's other warps
        const int col = t.n0 + column0;
        uint32_t amax = 0;
        if (any_live) {
          if (t.n0 + kTileN > p.n) {   // features that do not exist: act(0) is 0
#pragma unroll
            for (int j = 0; j < kRun / 2; ++j)
              if (col + 2 * j >= p.n) acc[j] = acc[kRun / 2 + j] = 0;   // (n is even)
          }
          with_activation(p.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < kRun / 2; ++j) {
              const float2 g = unpack2(acc[j]), w = unpack2(acc[kRun / 2 + j]);
              float h0 = activate<decltype(act)::value>(g.x), h1 = activate<decltype(act)::value>(g.y);
              if (second) { h0 *= w.x; h1 *= w.y; }
              amax = max(amax, max(abs_bits(h0), abs_bits(h1)));
              acc[j] = pack2(h0, h1);
            }
          });
        }
        sh.amax[parity][column_warp][r] = amax;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.amax_full[quarter]);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.amax_full[quarter], parity, wc));
        if (!ok) {
          if (lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TASK, i);
          break;
        }
#pragma unroll
        for (int j = 0; j < kColumnWarps; ++j) amax = max(amax, sh.amax[parity][j][r]);
        const float top = __uint_as_float(amax);
        if (live) {
          const FastQuantizer z(top);
          unsigned char* q = static_cast<unsigned char*>(p.out) + static_cast<size_t>(row) * p.n + col;
#pragma unroll
          for (int g = 0; g < kRun / 16; ++g) {
            if (col + g * 16 < p.n) {   // (n is a multiple of 16)
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float2 lo = unpack2(acc[g * 8 + 2 * x]), hi = unpack2(acc[g * 8 + 2 * x + 1]);
                w[x] = to_e4m3x4(z.scaled(lo.x), z.scaled(lo.y), z.scaled(hi.x), z.scaled(hi.y));
              }
              *reinterpret_cast<uint4*>(q + g * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          if (column_warp == 0) p.out_scale[static_cast<size_t>(row) * p.nblocks + t.n0 / kBlock] = block_scale(top);
        }
      } else {
        const int col = t.n0 + column0, first_row = t.row0 + static_cast<int>(rank) * 128 + quarter * 32;
        if (col < p.n && first_row < t.row_end)   // (the same for the whole warp)
          store_features<Out, 2 * kRun>(static_cast<Out*>(p.out) + static_cast<size_t>(first_row) * p.n + col, p.n, acc,
                                        min(32, t.row_end - first_row), p.n - col, p.wide != 0,
                                        sh.stage[warp - kEpilogueWarp], lane);
      }
    }
  }
  __syncthreads();
  if constexpr (kPair) {
    cluster_sync_all();   // nothing of this CTA's is signalled from the other any more
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
  } else if (warp == 1) {
    tmem_dealloc(tmem, 512);
  }
}

// ---- few rows -----------------------------------------------------------------------------------------
//
// Where an expert (or the whole product) has few rows, reading the weights is what there is to do, and the
// roles turn round: 128 features on the TMEM lanes, kRows rows on its columns, one CTA a tile, and as many
// bytes of weights in flight as shared memory holds.  The gated form multiplies the tiles of up and up_v with
// the same rows, into accumulators side by side.  Where the tiles alone do not fill the GPU, the CTAs of a
// cluster share a tile: each takes a run of the blocks of k, leaves its sums in its shared memory, and adds
// up, in rank order, the sums of all for its share of the rows.
//
// Measured: one row of 8192 x 5120 12.7 us (42 MB of weights, 6.4 us at the copy rate; the rest is set-up, the first
// load and the cluster's sum), 16 rows of 128 experts of 2048 x 768, up and down, 61 us (389 MB, 59 us).

constexpr int kNarrowThreads = 384;   // TMA, MMA, scale warp, one idle; eight epilogue warps
constexpr int kMaxSplits = 8;
constexpr uint32_t kNarrowSmem = 208 * 1024;   // for the ring of stages

template <bool kGated, int kRows>
struct Narrow {
  static constexpr int kWeights = kGated ? 2 : 1;
  static constexpr uint32_t kRowBytes = kRows * kBlock;
  static constexpr uint32_t kStageBytes = kWeights * kBoxBytes + kRowBytes;
  static constexpr int kPart = kRows / 2;                       // columns of a weight that one warp adds up
  static constexpr uint32_t kReduceBytes = kRows <= 32 ? kWeights * kRows * 128 * sizeof(float) : 0;   // splits only
  static constexpr int kStages = (kNarrowSmem - kReduceBytes) / kStageBytes;
  static constexpr uint32_t kAccColumns = kWeights * kRows;
  static constexpr int kAccs = kAccColumns <= 128 ? 4 : 512 / kAccColumns;   // accumulators in flight
  static constexpr uint32_t kTmemColumns = kAccs * kAccColumns;
  struct Tail {
    uint64_t full[kStages], done[kStages];
    uint64_t acc_empty[kAccs];
    uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
    uint64_t amax_full[2];
    uint64_t sums_full, sums_empty;        // the cluster's sums of a tile are there; have been read by all
    uint32_t tmem_base;
    uint32_t abort_word;
    alignas(16) float scale[kScaleSlots][kScaleBlocks][kWeights][kRows];   // (read four at a time)
    uint32_t amax[2][8][kPart];
    TileTable table;
  };
  static constexpr size_t kSmem = 1024 + kStages * kStageBytes + kReduceBytes + sizeof(Tail);
};

template <int N>
__device__ __forceinline__ void tmem_ld_n(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    tmem_ld_16(taddr, r);
  } else {
    static_assert(N == 8);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
  }
}
template <int N>
__device__ __forceinline__ void tmem_wait_n(uint32_t (&r)[N]) {
  if constexpr (N == 16) {
    tmem_wait_16(r);
  } else {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :
                 : "memory");
  }
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <typename Out, int kRows>
__global__ void __launch_bounds__(kNarrowThreads, 1)
product_narrow_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w0,
                      const __grid_constant__ CUtensorMap map_w1, const ProductParams p) {
  constexpr bool kGated = std::is_same_v<Out, Codes>;
  using N = Narrow<kGated, kRows>;
  constexpr int kStages = N::kStages, kPart = N::kPart;
  extern __shared__ __align__(16) unsigned char s_raw[];
  unsigned char* ring = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
  float* sums = reinterpret_cast<float*>(ring + kStages * N::kStageBytes);   // [weight][row][feature], splits only
  auto& sh = *reinterpret_cast<typename N::Tail*>(ring + kStages * N::kStageBytes + N::kReduceBytes);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // (uniform to the compiler)
  const int splits = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_ctarank());
  const int first_tile = blockIdx.x / splits, tile_step = gridDim.x / splits;
  const int kb0 = p.kblocks * rank / splits, kb1 = p.kblocks * (rank + 1) / splits;   // this CTA's blocks of k
  const WaitCtx wc{&sh.abort_word, p.spin_limit};

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.done[i], 1); }
    for (int i = 0; i < N::kAccs; ++i) mbar_init(&sh.acc_empty[i], kEpilogueWarps);
    for (int i = 0; i < kScaleSlots; ++i) { mbar_init(&sh.scale_full[i], 1); mbar_init(&sh.scale_empty[i], kEpilogueWarps); }
    for (int i = 0; i < 2; ++i) mbar_init(&sh.amax_full[i], 4);
    mbar_init(&sh.sums_full, kEpilogueWarps * splits);
    mbar_init(&sh.sums_empty, kEpilogueWarps * splits);
    sh.abort_word = 0;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem_base, N::kTmemColumns);
    tmem_relinquish();
  }
  if (!p.in_layer) wait_for_primary();
  fill_table(sh.table, p, kRows);
  if (splits > 1) cluster_sync_all();   // the others' barriers exist before any is signalled
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_base;
  const bool second = kGated && p.has_v != 0;
  launch_dependents();
  if (p.in_layer && warp != 0) wait_for_primary();

  if (warp == 0) {
    const uint32_t bytes = N::kRowBytes + (second ? 2 : 1) * kBoxBytes;
    uint32_t stage = 0, phase = 1;
    Tile t;
    bool ok = true;
    int early = 0;   // blocks whose weights are on their way before the rows exist
    if (p.in_layer) {
      if (find_tile(sh.table, p, first_tile, kRows, kBlock, t)) {
        early = min(kStages, kb1 - kb0);
        if (elect_one()) {
          for (int j = 0; j < early; ++j) {
            unsigned char* to = ring + j * N::kStageBytes;
            mbar_expect_tx(&sh.full[j], bytes);
            tma_load_2d(to, &map_w0, &sh.full[j], (kb0 + j) * kBlock, t.expert * p.n + t.n0);
            if (second) tma_load_2d(to + kBoxBytes, &map_w1, &sh.full[j], (kb0 + j) * kBlock, t.expert * p.n + t.n0);
          }
        }
        __syncwarp();
      }
      wait_for_primary();
    }
    for (int i = first_tile; ok && find_tile(sh.table, p, i, kRows, kBlock, t); i += tile_step) {
      const int w_row = t.expert * p.n + t.n0;
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = warp_wait(&sh.done[stage], phase, wc);
        if (!ok) break;
        if (elect_one()) {
          unsigned char* to = ring + stage * N::kStageBytes;
          if (early <= 0) {
            mbar_expect_tx(&sh.full[stage], bytes);
            tma_load_2d(to, &map_w0, &sh.full[stage], kb * kBlock, w_row);
            if (second) tma_load_2d(to + kBoxBytes, &map_w1, &sh.full[stage], kb * kBlock, w_row);
          }
          tma_load_2d(to + N::kWeights * kBoxBytes, &map_a, &sh.full[stage], kb * kBlock, t.row0);
        }
        __syncwarp();
        --early;
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
      if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_PIPE_EMPTY, i);
    }
    // no copy may be in flight when the CTA leaves: the MMAs that free a stage come after its copies
    const WaitCtx last{nullptr, p.spin_limit};
    for (int j = 0; j < kStages; ++j) {   // (a stage that was never filled passes at once)
      mbar_wait(&sh.done[stage], phase, last);
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_e4m3(128, kRows);
    const uint64_t desc0 = umma_desc_sw128(smem_u32(ring));
    uint32_t stage = 0, phase = 0, b = 0, b_phase = 1, last_stage = 0, last_phase = 1;
    Tile t;
    bool ok = true;
    for (int i = first_tile; ok && find_tile(sh.table, p, i, kRows, kBlock, t); i += tile_step) {
      for (int kb = kb0; kb < kb1; ++kb) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[stage], phase, wc) && mbar_wait(&sh.acc_empty[b], b_phase, wc));
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t dw = desc0 + stage * (N::kStageBytes >> 4), da = dw + (N::kWeights * kBoxBytes >> 4);
          const uint32_t acc = tmem + b * N::kAccColumns;
#pragma unroll
          for (int q = 0; q < 4; ++q) {   // 32 bytes of k each
            umma_f8(acc, dw + 2 * q, da + 2 * q, idesc, q != 0);
            if (second) umma_f8(acc + kRows, dw + (kBoxBytes >> 4) + 2 * q, da + 2 * q, idesc, q != 0);
          }
          umma_commit(&sh.done[stage]);
        }
        __syncwarp();
        last_stage = stage;
        last_phase = phase;
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (++b == N::kAccs) { b = 0; b_phase ^= 1; }
      }
      if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_PIPE_FULL, i);
    }
    const WaitCtx last{nullptr, p.spin_limit};
    mbar_wait(&sh.done[last_stage], last_phase, last);   // no MMA may be running when TMEM is freed
  } else if (warp == kScaleWarp) {
    // each lane up to four rows, four blocks of k at a time, four to eight blocks ahead
    constexpr int kLaneRows = kRows < 32 ? 1 : kRows / 32;
    int groups = 0;
    Tile t;
    bool ok = true;
    for (int i = first_tile; ok && find_tile(sh.table, p, i, kRows, kBlock, t); i += tile_step) {
      const size_t w_at = (static_cast<size_t>(t.expert) * p.nblocks + t.n0 / kBlock) * p.kblocks;
      const float* w[2] = {p.w_scale[0] + w_at, second ? p.w_scale[1] + w_at : p.w_scale[0] + w_at};
      float a_next[kLaneRows][4], w_next[2][4];
      auto fetch = [&](int kb) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const bool in = kb + x < kb1;
#pragma unroll
          for (int j = 0; j < kLaneRows; ++j) {
            const int row = t.row0 + lane + 32 * j;
            a_next[j][x] = in && lane + 32 * j < kRows && row < t.row_end
                               ? fetched(p.a_scale + static_cast<size_t>(row) * p.kblocks + kb + x) : 0.0f;
          }
#pragma unroll
          for (int h = 0; h < N::kWeights; ++h) w_next[h][x] = in ? fetched(w[h] + kb + x) : 0.0f;
        }
      };
      fetch(kb0);
      for (int kb = kb0; kb < kb1; kb += 4, ++groups) {
        float v[N::kWeights][kLaneRows][4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int j = 0; j < kLaneRows; ++j)
#pragma unroll
            for (int h = 0; h < N::kWeights; ++h) v[h][j][x] = a_next[j][x] * w_next[h][x];
        if (kb + 4 < kb1) fetch(kb + 4);
        const int slot = groups % kScaleSlots;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.scale_empty[slot], ((groups / kScaleSlots) & 1) ^ 1, wc));
        if (!ok) break;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int j = 0; j < kLaneRows; ++j)
#pragma unroll
            for (int h = 0; h < N::kWeights; ++h)
              if (lane + 32 * j < kRows) sh.scale[slot][x][h][lane + 32 * j] = v[h][j][x];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.scale_full[slot]);
      }
      if (!ok && lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TMEM_EMPTY, i);
    }
  } else if (warp >= kEpilogueWarp) {
    // 32 features (a lane each) and half of the rows
    const int quarter = warp & 3, half = (warp - kEpilogueWarp) >> 2;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kPart;
    constexpr int kChunk = kPart < 16 ? kPart : 16;
    uint32_t stage = 0, phase = 0, b = 0;
    int groups = 0, parity = 0;
    Tile t;
    bool ok = true;
    for (int i = first_tile; ok && find_tile(sh.table, p, i, kRows, kBlock, t); i += tile_step, parity ^= 1) {
      const int feature = t.n0 + quarter * 32 + lane;
      uint64_t acc[N::kWeights][kPart / 2];   // pairs of rows
#pragma unroll
      for (int h = 0; h < N::kWeights; ++h)
#pragma unroll
        for (int j = 0; j < kPart / 2; ++j) acc[h][j] = 0;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; ++kb) {   // (a wait that fails goes on: nothing is stored then)
        const int slot = groups % kScaleSlots, x = (kb - kb0) % kScaleBlocks;
        if (x == 0) ok = mbar_wait(&sh.scale_full[slot], (groups / kScaleSlots) & 1, wc) && ok;
        ok = mbar_wait(&sh.done[stage], phase, wc) && ok;
        __syncwarp();
        tc_fence_after_sync();
#pragma unroll
        for (int h = 0; h < N::kWeights; ++h) {
#pragma unroll
          for (int c = 0; c < kPart / kChunk; ++c) {
            uint32_t d[kChunk];
            tmem_ld_n<kChunk>(taddr + b * N::kAccColumns + h * kRows + c * kChunk, d);
            const ulonglong2* s = reinterpret_cast<const ulonglong2*>(&sh.scale[slot][x][h][half * kPart + c * kChunk]);
            tmem_wait_n<kChunk>(d);
#pragma unroll
            for (int j = 0; j < kChunk / 4; ++j) {
              const ulonglong2 f = s[j];   // the scales of four rows
              uint64_t* to = &acc[h][c * (kChunk / 2) + 2 * j];
              to[0] = fma2(pack2(d[4 * j], d[4 * j + 1]), f.x, to[0]);
              to[1] = fma2(pack2(d[4 * j + 2], d[4 * j + 3]), f.y, to[1]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.acc_empty[b]);
        if (x == kScaleBlocks - 1 || kb + 1 == kb1) {
          if (lane == 0) mbar_arrive(&sh.scale_empty[slot]);
          ++groups;
        }
        if (++stage == kStages) { stage = 0; phase ^= 1; }
        if (++b == N::kAccs) b = 0;
      }
      // the rows this warp finishes: [from, from + count) of its half, sums in value(h, j)
      int from = 0, count = kPart;
      if (splits > 1) {
        // leave the sums where the cluster can read them, then add up this CTA's share of the rows
        ok = mbar_wait_cluster(&sh.sums_empty, parity ^ 1, wc) && ok;   // the last tile's have been read
        __syncwarp();
#pragma unroll
        for (int h = 0; h < N::kWeights; ++h)
#pragma unroll
          for (int j = 0; j < kPart / 2; ++j) {
            const float2 v = unpack2(acc[h][j]);
            float* to = sums + (h * kRows + half * kPart + 2 * j) * 128 + quarter * 32 + lane;
            to[0] = v.x;
            to[128] = v.y;
          }
        __syncwarp();
        if (lane < splits) mbar_arrive_cluster(map_to_cta(&sh.sums_full, lane));
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(&sh.sums_full, parity, wc) && ok);
        count = kPart / splits;              // (kPart is a multiple of splits)
        from = rank * count;
#pragma unroll
        for (int h = 0; h < N::kWeights; ++h)
#pragma unroll
          for (int j = 0; j < kPart / 2; ++j) acc[h][j] = 0;
        if (ok) {
          for (int q = 0; q < splits; ++q) {
#pragma unroll
            for (int h = 0; h < N::kWeights; ++h) {
              const uint32_t at = map_to_cta(sums + (h * kRows + half * kPart + from) * 128 + quarter * 32 + lane, q);
#pragma unroll
              for (int j = 0; j < kPart / 2; ++j) {
                if (2 * j < count) {
                  const float2 v = unpack2(acc[h][j]);
                  acc[h][j] = pack2(v.x + ld_cluster(at + 2 * j * 128 * sizeof(float)),
                                    2 * j + 1 < count ? v.y + ld_cluster(at + (2 * j + 1) * 128 * sizeof(float)) : 0.0f);
                }
              }
            }
          }
        }
        __syncwarp();
        if (lane < splits) mbar_arrive_cluster(map_to_cta(&sh.sums_empty, lane));
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TMEM_FULL, i);
        break;
      }
      const int row0 = t.row0 + half * kPart + from, live = min(count, t.row_end - row0);   // (may be none)
      if constexpr (kGated) {
        uint32_t* amax = sh.amax[parity][half * 4 + quarter];
        if (feature >= p.n) {   // act(0) is 0
#pragma unroll
          for (int j = 0; j < kPart / 2; ++j) acc[0][j] = acc[1][j] = 0;
        }
        with_activation(p.act, [&](auto act) {
#pragma unroll
          for (int j = 0; j < kPart; ++j) {
            if (j < live) {   // (the same for the whole warp)
              const float2 g = unpack2(acc[0][j / 2]), u = unpack2(acc[1][j / 2]);
              float h = activate<decltype(act)::value>(j & 1 ? g.y : g.x);
              if (second) h *= j & 1 ? u.y : u.x;
              acc[0][j / 2] = j & 1 ? pack2(g.x, h) : pack2(h, g.y);
              const uint32_t m = __reduce_max_sync(0xffffffffu, abs_bits(h));
              if (lane == 0) amax[j] = m;
            }
          }
        });
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.amax_full[half]);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.amax_full[half], parity, wc));
        if (!ok) {
          if (lane == 0) wait_failed(&sh.abort_word, FMOE_PHASE_TASK, i);
          break;
        }
        // each lane works out the scales of every 32nd row and hands them round
        float inv[(kPart + 31) / 32], pre[(kPart + 31) / 32];
#pragma unroll
        for (int c = 0; c < (kPart + 31) / 32; ++c) {
          const int j = c * 32 + lane;
          uint32_t m = 0;
          if (j < live) {
#pragma unroll
            for (int q = 0; q < 4; ++q) m = max(m, sh.amax[parity][half * 4 + q][j]);
            if (quarter == 0) p.out_scale[static_cast<size_t>(row0 + j) * p.nblocks + t.n0 / kBlock] = block_scale(__uint_as_float(m));
          }
          const FastQuantizer z(__uint_as_float(m));
          inv[c] = z.inv;
          pre[c] = z.pre;
        }
        unsigned char* to = static_cast<unsigned char*>(p.out) + static_cast<size_t>(row0) * p.n + feature;
#pragma unroll
        for (int j = 0; j < kPart; ++j) {
          if (j < live) {
            const float2 v = unpack2(acc[0][j / 2]);
            const float a = __shfl_sync(0xffffffffu, pre[j / 32], j & 31), f = __shfl_sync(0xffffffffu, inv[j / 32], j & 31);
            const uint32_t code = to_e4m3x2(((j & 1) ? v.y : v.x) * a * f, 0.0f);
            if (feature < p.n) *to = static_cast<unsigned char>(code);
            to += p.n;
          }
        }
      } else if (feature < p.n) {
        Out* to = static_cast<Out*>(p.out) + static_cast<size_t>(row0) * p.n + feature;
#pragma unroll
        for (int j = 0; j < kPart; ++j) {
          if (j < live) {
            const float2 v = unpack2(acc[0][j / 2]);
            *to = from_float<Out>(j & 1 ? v.y : v.x);
            to += p.n;
          }
        }
      }
    }
  }
  __syncthreads();
  if (splits > 1) cluster_sync_all();   // the others read this CTA's sums and signal its barriers
  if (warp == 1) tmem_dealloc(tmem, N::kTmemColumns);
}

// What a launch needs to know about a device, looked up once.
struct DeviceFacts {
  int sms = 0;
  long long spin_limit = 0;
};
const DeviceFacts& facts(int device) {
  static DeviceFacts all[kMaxDevices];
  static std::once_flag once[kMaxDevices];
  std::call_once(once[device], [&] {
    if (cudaDeviceGetAttribute(&all[device].sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) all[device].sms = 148;
    const char* ms = std::getenv("FMOE_SPIN_LIMIT_MS");
    all[device].spin_limit = spin_limit_cycles(ms ? std::atof(ms) : 2000.0, device);
  });
  return all[device];
}

// Launches a kernel in clusters of `cluster` CTAs; `registers`: what its warps will share out among themselves.
template <typename Kernel>
int launch_kernel(Kernel kernel, std::atomic<unsigned long long>& prepared, size_t smem, int threads, int registers, int grid,
                  int cluster, const CUtensorMap (&maps)[3], const ProductParams& p, int device, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (!(prepared.load(std::memory_order_acquire) >> device & 1)) {   // once a device
    cudaFuncAttributes made;
    e = cudaFuncGetAttributes(&made, kernel);
    if (e == cudaSuccess && made.numRegs * threads < registers)   // (a warp would wait for registers that do not exist)
      return set_error(FMOE_ERR_UNSUPPORTED, "the 8-bit product was compiled with fewer registers than its warps share out");
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("8-bit product: ") + cudaGetErrorString(e));
    prepared.fetch_or(1ull << device, std::memory_order_release);
  }
  e = launch_behind(kernel, dim3(grid), threads, smem, cluster, stream, maps[0], maps[1], maps[2], p);
  if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("8-bit product launch: ") + cudaGetErrorString(e));
  return FMOE_OK;
}

template <typename Out, bool kPair>
int launch_wide(const ProductParams& p, const CUtensorMap (&maps)[3], int grid, int device, cudaStream_t stream) {
  static std::atomic<unsigned long long> prepared{0};
  constexpr int kRegisters = 32 * (kEpilogueWarp * kLoadRegs + kEpilogueWarps * kEpilogueRegs);
  return launch_kernel(product_kernel<Out, kPair>, prepared, Wide<kPair>::smem_bytes(), kThreads, kRegisters, grid,
                       kPair ? 2 : 1, maps, p, device, stream);
}
template <typename Out, int kRows>
int launch_narrow(const ProductParams& p, const CUtensorMap (&maps)[3], int grid, int splits, int device, cudaStream_t stream) {
  using N = Narrow<std::is_same_v<Out, Codes>, kRows>;
  static_assert(N::kSmem <= 227 * 1024, "shared memory of one CTA");
  static std::atomic<unsigned long long> prepared{0};
  return launch_kernel(product_narrow_kernel<Out, kRows>, prepared, N::kSmem, kNarrowThreads, 0, grid, splits, maps, p, device, stream);
}

// Which kernel a product takes, and its launch shape.
struct Shape {
  int rows;     // rows a tile has: 256 (pairs), 128 (a CTA alone), or 16, 32, 64 (few rows)
  int splits;   // CTAs that share a tile (few rows only)
  int grid;
};

// The kernels differ in how much of a tile they can keep busy, so the choice goes by waves of tiles times what a block
// of k of one tile takes, measured (k = 4096, 8192 features, 24 to 2560 rows; and 8 and 128 experts of 12 to 1024
// rows): about 0.24 us for 16 and 32 rows x 128 features, 0.32 for 64 x 128, 0.62 for 128 x 256, 0.58 for the
// pair's 256 x 256, whose launch takes some 3 us more; outputs whose rows are no multiple of 32 bytes cost the last
// two another 5 us.  (640 rows: 51, 36.9 and 39.4 us by 64, 128 and 256 rows; 8 experts of 1024: 952, 645, 607 us.)
Shape shape_for(int m, int features, int kblocks, int experts, bool gated, bool wide_rows, int sms) {
  struct Kind { int rows; double block, fixed; };
  const int features_wide = gated ? 128 : 256;
  const double odd = wide_rows ? 0.0 : 5.0, twice = gated ? 2.0 : 1.0;   // (128 features of two weights)
  const Kind kinds[] = {{16, 0.24 * twice, 0.0}, {32, 0.24 * twice, 0.0}, {64, 0.32 * twice, 0.0}, {128, 0.62, odd},
                        {256, 0.58, odd + 3.0}};
  const int hit = experts > 1 ? (m < experts ? m : experts) : 1;   // experts that can have rows
  Shape best{0, 1, 0};
  double least = 0.0;
  for (const Kind& kind : kinds) {
    const int tile_n = kind.rows >= 128 ? features_wide : kBlock;
    const int slots = kind.rows == 256 ? sms / 2 : sms;            // tiles at work at a time
    const long long tiles_n = (features + tile_n - 1) / tile_n;
    // How the rows spread over the experts is known on the device only: at most `most` tiles, and with rows spread
    // at random around the mean half a tile more than the mean fills.
    const long long most = (experts > 1 ? m / kind.rows + hit : (m + kind.rows - 1) / kind.rows) * tiles_n;
    double tiles = static_cast<double>(most);
    if (experts > 1) {
      const double each = static_cast<double>(m) / hit / kind.rows + 0.5;
      tiles = (each < 1.0 ? 1.0 : each) * hit * tiles_n;
    }
    Shape s{kind.rows, 1, 0};
    while (s.rows <= 32 && s.splits < kMaxSplits && 2 * s.splits <= s.rows / 2 && 2 * s.splits * most <= sms &&
           kblocks >= 8 * s.splits)
      s.splits *= 2;
    double waves = tiles * s.splits / slots;
    if (experts == 1) waves = static_cast<double>((most * s.splits + slots - 1) / slots);
    if (waves < 1.0) waves = 1.0;
    const double cost = waves * kblocks / s.splits * kind.block + kind.fixed;
    const long long ctas = kind.rows == 256 ? 2 * (most < slots ? most : slots)
                                            : s.splits * (most < slots / s.splits ? most : slots / s.splits);
    s.grid = static_cast<int>(ctas);
    if (best.rows == 0 || cost < least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

template <typename Out>
int launch_product(ProductParams p, const void* a, const void* w0, const void* w1, int device, cudaStream_t stream) {
  constexpr int kWideN = std::is_same_v<Out, Codes> ? 128 : 256;
  const Shape s = shape_for(p.m, p.n, p.kblocks, p.experts, std::is_same_v<Out, Codes>, std::is_same_v<Out, Codes> || p.wide != 0, facts(device).sms);
  const int tile_n = s.rows >= 128 ? kWideN : kBlock;
  p.tiles_n = (p.n + tile_n - 1) / tile_n;
  CUtensorMap maps[3];
  const uint64_t w_rows = static_cast<uint64_t>(p.experts) * p.n;
  int rc = make_byte_map(&maps[0], a, p.m, p.k, s.rows >= 128 ? 128 : s.rows);
  if (rc == FMOE_OK) rc = make_byte_map(&maps[1], w0, w_rows, p.k, 128);
  if (rc == FMOE_OK && w1 != w0) rc = make_byte_map(&maps[2], w1, w_rows, p.k, 128);
  if (rc != FMOE_OK) return rc;
  if (w1 == w0) maps[2] = maps[1];
  switch (s.rows) {
    case 16: return launch_narrow<Out, 16>(p, maps, s.grid, s.splits, device, stream);
    case 32: return launch_narrow<Out, 32>(p, maps, s.grid, s.splits, device, stream);
    case 64: return launch_narrow<Out, 64>(p, maps, s.grid, s.splits, device, stream);
    case 128: return launch_wide<Out, false>(p, maps, s.grid, device, stream);
    default: return launch_wide<Out, true>(p, maps, s.grid, device, stream);
  }
}

// The checks that both products share.
int check_product(const void* a, const float* a_scale, const void* w, const float* w_scale, const int32_t* offsets, int m,
                  int n, int k, int experts, int device) {
  if (m < 0 || n < 1 || k < 1) return set_error(FMOE_ERR_INVALID_ARG, "m must not be negative, n and k must be positive");
  if (experts < 1 || experts > kMaxExperts)
    return set_error(FMOE_ERR_INVALID_ARG, "num_experts must be between 1 and " + std::to_string(kMaxExperts));
  if (device < 0 || device >= kMaxDevices) return set_error(FMOE_ERR_INVALID_ARG, "device_id out of range");
  if (k % 16 != 0) return set_error(FMOE_ERR_INVALID_ARG, "k must be a multiple of 16");
  if (experts > 1 && offsets == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "several experts need offsets");
  const long long tiles = (static_cast<long long>(m) / 16 + experts) * (n / 128 + 1);
  if (m > kMostTiles || static_cast<long long>(experts) * n > kMostTiles || tiles > kMostTiles)
    return set_error(FMOE_ERR_UNSUPPORTED, "more rows, features or tiles than 32-bit tile numbers hold");
  if (m > 0 && (a == nullptr || a_scale == nullptr || w == nullptr || w_scale == nullptr))
    return set_error(FMOE_ERR_INVALID_ARG, "both operands and their scales are required");
  if (misaligned(a, 16) || misaligned(w, 16)) return set_error(FMOE_ERR_INVALID_ARG, "operands must be 16-byte aligned");
  if (misaligned(a_scale, 4) || misaligned(w_scale, 4) || misaligned(offsets, 4))
    return set_error(FMOE_ERR_INVALID_ARG, "scales and offsets must be 4-byte aligned");
  return FMOE_OK;
}

ProductParams product_params(int m, int n, int k, int experts, const int32_t* offsets, int device) {
  ProductParams p{};
  p.m = m; p.n = n; p.k = k;
  p.kblocks = blocks_of(k); p.nblocks = blocks_of(n);
  p.experts = experts;
  p.offsets = offsets;
  p.spin_limit = facts(device).spin_limit;
  return p;
}

}  // namespace

int matmul(const fmoe_fp8_matmul_args* a, Launch how, cudaStream_t st) {
  if (a == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "arguments are null");
  int rc = check_product(a->a, a->a_scale, a->w, a->w_scale, a->offsets, a->m, a->n, a->k, a->num_experts, a->device_id);
  if (rc != FMOE_OK) return rc;
  if (a->data_type != FMOE_DT_BF16 && a->data_type != FMOE_DT_FP16 && a->data_type != FMOE_DT_FP32)
    return set_error(FMOE_ERR_UNSUPPORTED, "the 8-bit product is written as BF16, FP16 or FP32");
  const int eb = element_bytes(a->data_type);
  if (a->m == 0) return FMOE_OK;
  if (a->out == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "out is required");
  if (misaligned(a->out, eb)) return set_error(FMOE_ERR_INVALID_ARG, "out must be aligned to its type");
  if (how == Launch::kCheckOnly) return FMOE_OK;
  OnDevice on(a->device_id);
  if (on.err != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(on.err));
  ProductParams p = product_params(a->m, a->n, a->k, a->num_experts, a->offsets, a->device_id);
  p.a_scale = a->a_scale;
  p.w_scale[0] = a->w_scale;
  p.out = a->out;
  p.wide = !misaligned(a->out, 32) && (static_cast<size_t>(a->n) * eb) % 32 == 0;
  p.in_layer = how == Launch::kInLayer;
  if (a->data_type == FMOE_DT_BF16) return launch_product<__nv_bfloat16>(p, a->a, a->w, a->w, a->device_id, st);
  if (a->data_type == FMOE_DT_FP16) return launch_product<__half>(p, a->a, a->w, a->w, a->device_id, st);
  return launch_product<float>(p, a->a, a->w, a->w, a->device_id, st);
}

int gated_matmul(const fmoe_fp8_gated_args* a, Launch how, cudaStream_t st) {
  if (a == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "arguments are null");
  int rc = check_product(a->a, a->a_scale, a->up, a->up_scale, a->offsets, a->m, a->ffn_size, a->k, a->num_experts,
                         a->device_id);
  if (rc != FMOE_OK) return rc;
  if (a->ffn_size % 16 != 0) return set_error(FMOE_ERR_INVALID_ARG, "ffn_size must be a multiple of 16");
  if (a->act_type < FMOE_ACT_IDENTITY || a->act_type > FMOE_ACT_RELU)
    return set_error(FMOE_ERR_INVALID_ARG, "unknown act_type");
  if (a->m == 0) return FMOE_OK;
  if (a->q == nullptr || a->scale == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "q and scale are required");
  if (misaligned(a->q, 16) || misaligned(a->up_v, 16)) return set_error(FMOE_ERR_INVALID_ARG, "q and up_v must be 16-byte aligned");
  if (misaligned(a->scale, 4) || misaligned(a->up_v_scale, 4))
    return set_error(FMOE_ERR_INVALID_ARG, "scales must be 4-byte aligned");
  if (a->up_v != nullptr && a->up_v_scale == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "up_v needs its scales");
  if (how == Launch::kCheckOnly) return FMOE_OK;
  OnDevice on(a->device_id);
  if (on.err != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(on.err));
  ProductParams p = product_params(a->m, a->ffn_size, a->k, a->num_experts, a->offsets, a->device_id);
  p.a_scale = a->a_scale;
  p.w_scale[0] = a->up_scale;
  p.w_scale[1] = a->up_v_scale;
  p.out = a->q;
  p.out_scale = a->scale;
  p.act = a->act_type;
  p.has_v = a->up_v != nullptr;
  p.in_layer = how == Launch::kInLayer;
  return launch_product<Codes>(p, a->a, a->up, a->up_v != nullptr ? a->up_v : a->up, a->device_id, st);
}

}  // namespace fmoe::fp8

using namespace fmoe;
using namespace fmoe::fp8;

extern "C" {

int fmoe_fp8_matmul(const fmoe_fp8_matmul_args* a, void* stream) { return matmul(a, Launch::kPlain, static_cast<cudaStream_t>(stream)); }

int fmoe_fp8_gated_matmul(const fmoe_fp8_gated_args* a, void* stream) {
  return gated_matmul(a, Launch::kPlain, static_cast<cudaStream_t>(stream));
}

int fmoe_fp8_last_status(int32_t device_id, void* stream, fmoe_status* out) {
  if (out == nullptr) return set_error(FMOE_ERR_INVALID_ARG, "out is null");
  if (device_id < 0 || device_id >= kMaxDevices) return set_error(FMOE_ERR_INVALID_ARG, "device_id out of range");
  OnDevice on(device_id);
  cudaError_t e = on.err;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const fmoe_status none{};
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(out, g_status, sizeof(fmoe_status), 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && out->code != FMOE_OK) {
    e = cudaMemcpyToSymbolAsync(g_status, &none, sizeof(none), 0, cudaMemcpyHostToDevice, st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) return set_error(FMOE_ERR_CUDA, std::string("fmoe_fp8_last_status: ") + cudaGetErrorString(e));
  return FMOE_OK;
}

}  // extern "C"
