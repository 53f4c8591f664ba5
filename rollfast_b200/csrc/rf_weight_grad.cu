// Weight gradient X^T G from an activation saved in 8 bits.
//
//   out[i][o] = initial[i][o] + sum_t X[t][i] G[t][o]    (or its transpose)
//
// X [T][K] is the saved activation (rf_act8.cuh), G [T][N] the gradient of
// the product's output.  Bound by the tensor cores (2 T K N operations).
//
// Operands.  The steps of X differ along the sum, so they cannot be applied
// to the accumulator; X is expanded to bfloat16 once, in the workspace, which
// is exact because the steps are powers of two.  Converting in the product
// kernel instead, on the way to shared memory, was built and measured: every
// column block converts X again, and the 2.5 instructions per element do not
// fit beside the products (8192 x 4096 x 4096: 321 us against 210).  The
// copy costs 346 / N of the product's time.  Float16 and float32 gradients
// become two or three bfloat16 terms that add up to them.
//
// 8192 x 4096 x 14336, bfloat16 gradient, float32 result, with the expansion:
// 681 to 689 us in bursts of five calls (1.40 PFLOP/s), 686 to 699 in 200 back
// to back; added to an earlier gradient 715 to 724 and 761 to 768.  cuBLAS on
// ready bfloat16 operands, in turn with these, 669 to 673 and 699 to 708.
//
// Products.  One persistent CTA pair (cluster of 2, tcgen05 cta_group::2) per
// 256 x 256 output tile; each CTA brings 128 rows of one operand and 128
// columns of the other, 128 tokens a step.  The sum runs over rows of both
// arrays, so both operands are MN-major:
//   warps 0, 2   TMA: boxes of 128 tokens x 64 columns (128-byte swizzle) into a
//                ring of kStages
//   warp 1       the leader's lane 0 issues tcgen05.mma (M = N = 256, K = 16)
//   warps 4..11  accumulators -> registers -> memory
// Accuracy.  The tensor cores truncate when they add to the accumulator: over
// 8192 tokens that left a relative error of 2.8e-6, five times that of float32
// additions.  So the accumulator is closed every kSegment steps (1024 tokens:
// 3.7e-7), and the epilogue warps add the segments in float32 registers (128
// per thread) while the next segment runs into the other half of TMEM.
//
// Few tiles: the tokens are split over several units whose float32 partial
// tiles a second kernel adds in a fixed order.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "rf_act8.cuh"
#include "rf_kernels.cuh"
#include "rf_tc.cuh"

namespace rf {
namespace wg {

using namespace rf::tc;

constexpr int kTile = 256;          // output tile of a CTA pair, both ways
constexpr int kHalf = 128;          // operand rows per CTA
// Tokens per step.  A step costs the issuing thread a wait and a commit beside
// its products; with 64 tokens that thread, not the tensor cores, was the
// bound (8192 x 4096 x 14336: 771 us against 650).
constexpr int kTokens = 128;
constexpr int kSegment = 8;         // steps per accumulator
constexpr int kStages = 3;
constexpr int kOperandBytes = kTokens * kHalf * 2;
constexpr int kBlockBytes = kTokens * 128;  // 64 columns of an operand
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kFirstEpilogue = 4, kEpilogueWarps = 8;  // a multiple of 4: a warp reads TMEM lanes 32 (warp % 4) ..
constexpr int kThreads = (kFirstEpilogue + kEpilogueWarps) * 32;
constexpr int kColumns = kTile / (kEpilogueWarps / 4);  // accumulator columns per epilogue warp
static_assert(kColumns == 128, "the epilogue names its eight blocks of 16");
constexpr int kStagingFloats = 32 * 16;                 // a warp's 32 x 16 block on its way out
constexpr int kStagingOff = kStages * kStageBytes;
constexpr int kBarOff = kStagingOff + kEpilogueWarps * kStagingFloats * 4;
constexpr int kSmemBytes = kBarOff + 256 + 1024;
static_assert(kSmemBytes <= 232448, "dynamic shared memory per CTA is at most 227 KB");
constexpr uint32_t kTmemCols = 512;

struct Params {
  int64_t m, n;            // output rows and columns
  int64_t units;           // whole tiles, then the splits of the tail's tiles
  int64_t whole;           // tiles computed by one unit
  int tiles_i, tiles_j;    // 256-row and 256-column blocks
  int splits;              // units per tile of the tail
  int steps;               // 128-token steps of all tokens
  int terms;               // bfloat16 terms of G (1, 2 or 3)
  int x_first;             // X is the row operand (out is [K][N]), else the column operand
  const void* initial;     // added when there is one unit per tile
  void* out;
  int64_t ld_out;
  int out_dt;
  int vec;                 // 4 columns of out and initial can be read and written at once
  float* partial;          // [tail tile][split][256][256]
  uint32_t idesc;
  int* error;              // the device's error word, may be null
};

// Tile -> (row block, column block): down the row blocks in groups of 8, so
// that the ~74 tiles in flight share their operands' panels in L2.
__host__ __device__ __forceinline__ void tile_at(int64_t tile, int tiles_i, int tiles_j, int& I, int& J) {
  const int t = int(tile), G = 8;
  const int grp = t / (G * tiles_j);
  const int first = grp * G;
  const int gm = tiles_i - first < G ? tiles_i - first : G;
  const int r = t - grp * G * tiles_j;
  I = first + r % gm;
  J = r / gm;
}
// A unit's tile, its steps [k0, k1) of the tokens, each taken once per term
// of G, and its partial tile (-1: it writes the output itself).
__device__ __forceinline__ void decode_unit(const Params& P, int64_t u, int& I, int& J, int& k0, int& k1,
                                            int64_t& part) {
  int64_t tile = u;
  part = -1;
  k0 = 0;
  k1 = P.steps;
  if (u >= P.whole) {
    const int64_t v = u - P.whole;
    const int s = int(v % P.splits);
    tile = P.whole + v / P.splits;
    if (P.splits > 1) part = v;
    k0 = int(int64_t(P.steps) * s / P.splits);
    k1 = int(int64_t(P.steps) * (s + 1) / P.splits);
  }
  tile_at(tile, P.tiles_i, P.tiles_j, I, J);
}

__device__ __forceinline__ void record_error(const Params& P, int code, volatile int* abort_flag) {
  *abort_flag = 1;
  if (P.error) atomicCAS(P.error, 0, code);
}

// 4 consecutive columns at element i of the output's array `initial`.
__device__ __forceinline__ float4 initial4(const Params& P, int64_t i) {
  if (P.out_dt == RF_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(P.initial) + i);
  const uint2 a = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(P.initial) + i);
  if (P.out_dt == RF_BF16)
    return make_float4(__uint_as_float(a.x << 16), __uint_as_float(a.x & 0xFFFF0000u), __uint_as_float(a.y << 16),
                       __uint_as_float(a.y & 0xFFFF0000u));
  const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
  const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ void put4(const Params& P, int64_t i, float4 v) {
  if (P.out_dt == RF_F32)
    *reinterpret_cast<float4*>(static_cast<float*>(P.out) + i) = v;
  else
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out) + i) =
        P.out_dt == RF_BF16 ? make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w))
                            : make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
}
// The same without vectors, `live` of the columns.
__device__ __forceinline__ void add_put_each(const Params& P, int64_t i, int64_t live, float4 v) {
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= live) break;
    float x = f[k];
    if (P.initial) x += ld_as_float(P.initial, P.out_dt, i + k);
    st_from_float(P.out, P.out_dt, i + k, x);
  }
}
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

// A warp's 32 x 16 block of sums, lane = row, goes through its staging buffer,
// so that a store instruction covers 8 rows of 64 bytes.  16-byte chunk c of
// row r lies at c ^ (r / 2 % 4): both the row writes and the reads of 8 rows
// by 4 chunks touch every bank once.
__device__ __forceinline__ void stage_block(int lane, const float* v, float* stg) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<float4*>(stg + lane * 16 + ((c ^ ((lane >> 1) & 3)) << 2)) =
        make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}
// The initial values of a block, loaded together and ahead of the staging: one
// at a time, their latency outlasted the next tile's products.
struct BlockAt {
  int64_t i, ld, live;
  int rows;  // this lane's row r + 8 it is inside while 8 it < rows
  bool vec;
  float4 initial[4];
};
__device__ __forceinline__ BlockAt block_at(const Params& P, const float* part, int64_t row0, int64_t col0, int lane) {
  BlockAt b;
  const int r = lane >> 2;
  const int64_t col = col0 + 4 * (lane & 3);
  b.live = P.n - col;
  b.vec = P.vec && b.live >= 4;
  b.ld = part ? kTile : P.ld_out;
  b.i = part ? (row0 + r) % kTile * kTile + col % kTile : (row0 + r) * P.ld_out + col;
  b.rows = b.live > 0 ? int(min(P.m - row0 - r, int64_t(32))) : 0;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    b.initial[it] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!part && P.initial && b.vec && 8 * it < b.rows) b.initial[it] = initial4(P, b.i + 8 * it * b.ld);
  }
  return b;
}
__device__ __forceinline__ void store_block(const Params& P, float* part, const BlockAt& b, int lane, const float* stg) {
  const int r = lane >> 2;  // row r + 8 it: its / 2 % 4 is that of r
  const float* src = stg + r * 16 + (((lane & 3) ^ ((r >> 1) & 3)) << 2);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    if (8 * it >= b.rows) break;
    const float4 x = *reinterpret_cast<const float4*>(src + 128 * it);
    const int64_t i = b.i + 8 * it * b.ld;
    if (part) *reinterpret_cast<float4*>(part + i) = x;
    else if (b.vec) put4(P, i, add4(x, b.initial[it]));
    else add_put_each(P, i, b.live, x);
  }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_weight_grad(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_g,
                  const __grid_constant__ Params P) {
  // The join's CTAs may take the SMs that this grid leaves.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOff);
  const uint32_t full0 = smem_u32(bars);              // loads landed (the leader's: both CTAs')
  const uint32_t empty0 = full0 + 8 * kStages;        // loads consumed (commit, both CTAs)
  const uint32_t accf0 = empty0 + 8 * kStages;        // accumulator complete (commit, both CTAs)
  const uint32_t acce0 = accf0 + 16;                  // accumulator read (leader: both CTAs' warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int64_t pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 2);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(accf0 + 8 * s, 1);
      mbar_init(acce0 + 8 * s, 2 * kEpilogueWarps);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < kFirstEpilogue) {
  // Registers move to the epilogue's sums: 72 + 2 x 216 of the launch's 3 x 168.
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 0 || warp == 2) {
    if (lane == 0) {
      // ---------------- loads (both CTAs, each its own halves) ----------------
      // A warp for each operand: a wait and four copies take one thread about
      // as long as the products of a step.
      prior_kernel_done();  // X and the terms of G are complete
      const bool x = warp == 0;
      const CUtensorMap* map = x ? &tm_x : &tm_g;
      int stage = 0;
      uint32_t phase = 0;
      int64_t fills = 0;
      bool ok = true;
      for (int64_t u = pair; ok && u < P.units; u += npairs) {
        int I, J, k0, k1;
        int64_t part;
        decode_unit(P, u, I, J, k0, k1, part);
        const int col = ((P.x_first != 0) == x ? I : J) * kTile + int(rank) * kHalf;
        // The smallest term first: what the accumulator's truncation costs
        // goes with its magnitude, which only the last pass brings up.
        for (int term = P.terms - 1; ok && term >= 0; --term) {
          for (int k = k0; k < k1; ++k) {
            if (!mbar_wait_short(empty0 + 8 * stage, phase ^ 1, abort_flag)) {
              record_error(P, kDevTimeoutProducer, abort_flag);
              ok = false;
              break;
            }
            // Both CTAs' copies complete on the leader's barrier.
            if (leader) mbar_arrive_expect_tx(full0 + 8 * stage, 2 * kOperandBytes);
            const uint32_t fb = map_to_rank(full0 + 8 * stage, 0);
            const uint32_t dst = smem_u32(smem + stage * kStageBytes) + (x ? 0 : kOperandBytes);
            tma_load_3d_pair(dst, map, fb, col, k * kTokens, x ? 0 : term);
            tma_load_3d_pair(dst + kBlockBytes, map, fb, col + 64, k * kTokens, x ? 0 : term);
            ++fills;
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
      }
      // The last fills have been consumed: no copy into this CTA and no
      // commit's arrival on these barriers is pending.
      for (int64_t f = fills > kStages ? fills - kStages : 0; f < fills; ++f)
        mbar_drain(empty0 + 8 * uint32_t(f % kStages), uint32_t((f / kStages) & 1));
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ---------------- products ----------------
      const uint32_t ring = smem_u32(smem);
      const uint64_t xd = sdesc(ring, kBlockBytes, 1024), gd = sdesc(ring + kOperandBytes, kBlockBytes, 1024);
      const uint64_t ad = P.x_first ? xd : gd, bd = P.x_first ? gd : xd;
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      int64_t segments = 0;
      uint32_t loaded = 0;  // the current stage's loads were seen complete
      for (int64_t u = pair; ok && u < P.units; u += npairs) {
        int I, J, k0, k1;
        int64_t part;
        decode_unit(P, u, I, J, k0, k1, part);
        const int n_steps = (k1 - k0) * P.terms;
        for (int b = 0; ok && b < n_steps; b += kSegment) {
          if (!mbar_wait_short(acce0 + 8 * acc, acc_phase ^ 1, abort_flag)) {
            record_error(P, kDevTimeoutMma, abort_flag);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + uint32_t(acc * kTile);
          const int e = min(b + kSegment, n_steps);
          for (int k = b; k < e; ++k) {
            if (!loaded && !mbar_wait_short(full0 + 8 * stage, phase, abort_flag)) {
              record_error(P, kDevTimeoutMma, abort_flag);
              ok = false;
              break;
            }
            const uint32_t now = uint32_t(stage);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1;
            }
            loaded = mbar_test(full0 + 8 * stage, phase);
            tc_fence_after();
            // Descriptors count 16-byte units: a stage further, 16 tokens further.
            const uint64_t off = uint64_t(now * (kStageBytes >> 4));
#pragma unroll
            for (int q = 0; q < kTokens / 16; ++q)
              mma_f16_pair(d_tmem, ad + off + q * (2048 >> 4), bd + off + q * (2048 >> 4), P.idesc,
                           (k > b || q > 0) ? 1u : 0u);
            mma_commit_pair(empty0 + 8 * now);
          }
          if (!ok) break;
          mma_commit_pair(accf0 + 8 * acc);
          ++segments;
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      // Both CTAs' epilogues have released the last two accumulators.
      for (int64_t k = segments > 2 ? segments - 2 : 0; k < segments; ++k)
        mbar_drain(acce0 + 8 * uint32_t(k & 1), uint32_t((k >> 1) & 1));
    }
  }
  } else {
    // ---------------- segments -> registers -> memory (both CTAs) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int quarter = warp & 3;                         // TMEM lanes 32 * quarter .. + 31
    const int first_col = ((warp - kFirstEpilogue) >> 2) * kColumns;
    int acc = 0;
    uint32_t acc_phase = 0;
    float* stg = reinterpret_cast<float*>(smem + kStagingOff) + (warp - kFirstEpilogue) * kStagingFloats;
    bool ok = true;
    for (int64_t u = pair; ok && u < P.units; u += npairs) {
      int I, J, k0, k1;
      int64_t part;
      decode_unit(P, u, I, J, k0, k1, part);
      const int n_steps = (k1 - k0) * P.terms;
      float sum[kColumns];
#pragma unroll
      for (int i = 0; i < kColumns; ++i) sum[i] = 0.f;
      for (int b = 0; b < n_steps; b += kSegment) {
        // One lane polls, for the other waits' sake.
        if (lane == 0) ok = mbar_wait_short(accf0 + 8 * acc, acc_phase, abort_flag);
        ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
        if (!ok) {
          record_error(P, kDevTimeoutEpilogue, abort_flag);
          break;
        }
        tc_fence_after();
        const uint32_t t = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc * kTile + first_col);
#pragma unroll
        for (int c = 0; c < kColumns; c += 32) {
          uint32_t v[2][16];
          tmem_ld16_async(t + c, v[0]);
          tmem_ld16_async(t + c + 16, v[1]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[c + i] += __uint_as_float(v[i >> 4][i & 15]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(map_to_rank(acce0 + 8 * acc, 0));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (!ok) break;
      const int64_t row0 = int64_t(I) * kTile + int64_t(rank) * kHalf + quarter * 32;
      const int64_t col0 = int64_t(J) * kTile + first_col;
      float* dst = part < 0 ? nullptr : P.partial + part * (kTile * kTile);
      // Whole float32 blocks to a partial tile or an output without initial
      // values: four reads, four stores.
      float* plain = dst ? dst + (row0 % kTile + (lane >> 2)) * kTile + first_col + 4 * (lane & 3)
                         : static_cast<float*>(P.out) + (row0 + (lane >> 2)) * P.ld_out + col0 + 4 * (lane & 3);
      const int64_t plain_ld = 8 * (dst ? kTile : P.ld_out);
      const bool fast = (dst || (P.vec && P.out_dt == RF_F32 && !P.initial)) && row0 + 32 <= P.m;
      // One copy of the store's code for all blocks (unrolled, it did not fit
      // the instruction cache: 17 us a tile); only the registers that a block
      // comes from are spelled out.
#pragma unroll 1
      for (int c = 0; c < kColumns / 16; ++c) {
        if (row0 >= P.m || col0 + 16 * c >= P.n) break;
        const bool simple = fast && col0 + 16 * c + 16 <= P.n;
        BlockAt at;
        if (!simple) at = block_at(P, dst, row0, col0 + 16 * c, lane);
        switch (c) {
          case 0: stage_block(lane, sum, stg); break;
          case 1: stage_block(lane, sum + 16, stg); break;
          case 2: stage_block(lane, sum + 32, stg); break;
          case 3: stage_block(lane, sum + 48, stg); break;
          case 4: stage_block(lane, sum + 64, stg); break;
          case 5: stage_block(lane, sum + 80, stg); break;
          case 6: stage_block(lane, sum + 96, stg); break;
          default: stage_block(lane, sum + 112, stg); break;
        }
        __syncwarp();
        if (simple) {
          const float* src = stg + (lane >> 2) * 16 + (((lane & 3) ^ ((lane >> 3) & 3)) << 2);
          float4 x[4];
#pragma unroll
          for (int it = 0; it < 4; ++it) x[it] = *reinterpret_cast<const float4*>(src + 128 * it);
#pragma unroll
          for (int it = 0; it < 4; ++it) *reinterpret_cast<float4*>(plain + it * plain_ld + 16 * c) = x[it];
        } else {
          store_block(P, dst, at, lane, stg);
        }
        __syncwarp();
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  cluster_sync();  // no CTA leaves while its peer may still touch its TMEM / shared memory
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
  }
}

// G as bfloat16 terms [terms][rows][ld] (ld a multiple of 8, zeros behind the
// last column): truncating to 8 significant bits leaves an exactly
// representable remainder, so 2 terms hold a float16 and 3 a float32.  A term
// cut from an infinity or a NaN stays alone (the others are 0).
__global__ void __launch_bounds__(256) k_grad_terms(RowView g, uint16_t* out, int64_t rows, int64_t n, int64_t ld,
                                                    int terms) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  if (col >= ld) return;
  for (int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; row < rows; row += int64_t(gridDim.x) * blockDim.y) {
    float f[8];
    load8(g, row, col, n, f);
    for (int t = 0; t < terms; ++t) {
      uint32_t h[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t b = __float_as_uint(f[k]);
        const bool special = (b & 0x7F800000u) == 0x7F800000u;
        h[k] = (special && (b & 0x7FFFFFu)) ? 0x7FC0u : b >> 16;
        f[k] = special ? 0.f : f[k] - __uint_as_float(b & 0xFFFF0000u);
      }
      *reinterpret_cast<uint4*>(out + (int64_t(t) * rows + row) * ld + col) =
          make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
  }
}

// The tail's tiles: out = initial + partial[0] + partial[1] + ... in this
// order.  A CTA takes 4 rows of a tile; without splits (no tokens) the sum is
// 0 everywhere.
__global__ void __launch_bounds__(256) k_weight_grad_join(const __grid_constant__ Params P) {
  const int64_t tail = blockIdx.x / (kTile / 4);
  const int r = int(blockIdx.x % (kTile / 4)) * 4 + int(threadIdx.x >> 6), c = int(threadIdx.x & 63) * 4;
  int I, J;
  tile_at(P.whole + tail, P.tiles_i, P.tiles_j, I, J);
  const int64_t row = int64_t(I) * kTile + r, col = int64_t(J) * kTile + c;
  if (row >= P.m || col >= P.n) return;
  prior_kernel_done();
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* p = P.partial + tail * P.splits * (kTile * kTile) + r * kTile + c;
#pragma unroll 4
  for (int s = 0; s < P.splits; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(p + int64_t(s) * (kTile * kTile));
    a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
  }
  const int64_t i = row * P.ld_out + col;
  if (!P.vec || P.n - col < 4) add_put_each(P, i, P.n - col, a);
  else put4(P, i, P.initial ? add4(a, initial4(P, i)) : a);
}

// Boxes of kTokens tokens x 64 columns over [terms][rows][cols] bfloat16, rows ld
// elements apart (a multiple of 8); columns and tokens behind the last read 0.
rf_status make_map(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t terms, int64_t ld) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(RF_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(terms)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * 2, cuuint64_t(ld) * 2 * cuuint64_t(rows)};
  const cuuint32_t box[3] = {64, kTokens, 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RF_ECUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(int(r)));
  return RF_OK;
}

// Which tiles are split over the tokens, and into how many units.  All tiles
// that fill a wave of pairs stay whole; the rest (all, when there are fewer
// than pairs) would leave pairs idle and are split into the number that
// minimises a model of the remaining time, in steps of one pair: waves of
// units, each its steps plus about 4 of prologue and epilogue, and for a split
// the partial tiles' way through L2 (about 6 steps, and 1.5 for every tile a
// pair has to write and read).
struct Tail {
  int64_t whole;
  int splits;
};
Tail choose_tail(int64_t tiles, int64_t steps, int64_t pairs) {
  Tail t{tiles - tiles % pairs, 1};
  const int64_t rest = tiles - t.whole;
  if (rest == 0) return t;
  double best = double(steps) + 4;
  for (int s = 2; s <= 64 && s * 2 <= steps; ++s) {
    const double waves = double(ceil_div(rest * s, pairs));
    const double cost = waves * (double(ceil_div(steps, s)) + 4) + 6 + 1.5 * double(rest * s) / double(pairs);
    if (cost < best) {
      best = cost;
      t.splits = s;
    }
  }
  if (t.splits == 1) t.whole = tiles;
  return t;
}

// A kernel that starts while the one before it drains (rf_tc.cuh).
template <typename... Args>
rf_status launch_dependent(void (*kernel)(Args...), unsigned grid, int threads, int smem, cudaStream_t st,
                           const std::decay_t<Args>&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return fail(RF_ECUDA, std::string("rf_weight_gradient launch: ") + cudaGetErrorString(e));
  return check_launch("rf_weight_gradient");
}

struct Plan {
  int64_t ld_x;         // row stride of the expanded X
  int64_t ld_terms;     // 0: G is read in place
  size_t x_bytes, terms_bytes, partial_bytes;
  int terms;
  Tail tail;
  int64_t steps;
  size_t total() const { return x_bytes + terms_bytes + partial_bytes; }
};

// `in_place`: the gradient is bfloat16 and its rows start on 16-byte boundaries.
Plan make_plan(int64_t rows, int64_t features, int64_t n_out, int32_t dt, bool in_place, int64_t pairs) {
  Plan p{};
  p.terms = dt == RF_BF16 ? 1 : dt == RF_F16 ? 2 : 3;
  p.steps = ceil_div(rows, kTokens);
  p.ld_x = round_up(features, 8);
  p.x_bytes = align_up(size_t(rows) * size_t(p.ld_x) * 2, 256);
  if (!(dt == RF_BF16 && in_place)) {
    p.ld_terms = round_up(n_out, 8);
    p.terms_bytes = align_up(size_t(p.terms) * size_t(rows) * size_t(p.ld_terms) * 2, 256);
  }
  const int64_t tiles = ceil_div(features, kTile) * ceil_div(n_out, kTile);
  if (rows > 0) p.tail = choose_tail(tiles, p.steps, pairs);
  else p.tail = Tail{0, 0};
  p.partial_bytes = size_t(tiles - p.tail.whole) * size_t(p.tail.splits) * kTile * kTile * 4;
  return p;
}

int64_t max_pairs() {
  static std::mutex mu;
  static int64_t cache[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  int64_t& c = cache[dev & 63];
  if (c == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(num_sms() & ~1), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kSmemBytes;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, k_weight_grad, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = num_sms() / 2;
    }
    c = n;
  }
  return c;
}

rf_status allow_smem() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev & 63]) return RF_OK;
  const cudaError_t e = cudaFuncSetAttribute(k_weight_grad, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return fail(RF_ECUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  done[dev & 63] = true;
  return RF_OK;
}

// Half the SMs: the split rule must not depend on a query that fails without
// a GPU, and a workspace planned on one B200 serves another.
int64_t plan_pairs() { return 74; }

rf_status check_sizes(int64_t rows, int64_t features, int64_t n_out, int32_t dt, int64_t ld) {
  if (!valid_dtype(dt)) return fail(RF_EINVAL, "rf_weight_gradient: grad dtype must be RF_F32, RF_BF16 or RF_F16");
  if (rows < 0 || rows > 0x7FFFFFFF - kTokens || features <= 0 || features > kMaxFeatures || n_out <= 0 ||
      n_out > kMaxFeatures || ceil_div(features, kTile) * ceil_div(n_out, kTile) > (int64_t(1) << 24))
    return fail(RF_EINVAL, "rf_weight_gradient: rows in [0, 2^31 - 128), features and n_out in [1, 2^26], at most "
                           "2^24 tiles of 256 x 256");
  if (ld < n_out) return fail(RF_EINVAL, "rf_weight_gradient: ld_grad below n_out");
  return RF_OK;
}

}  // namespace wg
}  // namespace rf

using namespace rf;

extern "C" rf_status rf_weight_gradient_workspace_size(int64_t rows, int64_t features, int64_t n_out,
                                                       const void* grad_out, int64_t ld_grad, int32_t grad_dtype,
                                                       size_t* bytes) {
  if (!bytes) return fail(RF_EINVAL, "rf_weight_gradient_workspace_size: null output");
  RF_TRY(wg::check_sizes(rows, features, n_out, grad_dtype, ld_grad));
  const bool in_place = grad_dtype == RF_BF16 && rows_vectorised(grad_out, ld_grad, RF_BF16);
  const wg::Plan p = wg::make_plan(rows, features, n_out, grad_dtype, in_place, wg::plan_pairs());
  *bytes = p.total();
  return RF_OK;
}

extern "C" rf_status rf_weight_gradient(const rf_saved_activation* saved, const void* grad_out, int64_t ld_grad,
                                        int32_t grad_dtype, int64_t n_out, int32_t layout, const void* initial,
                                        void* out, int64_t ld_out, int32_t out_dtype, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  using namespace rf::wg;
  RF_TRY(check_saved(saved, "rf_weight_gradient"));
  const int64_t rows = saved->rows, features = saved->features;
  RF_TRY(check_sizes(rows, features, n_out, grad_dtype, ld_grad));
  if (layout != RF_IN_OUT && layout != RF_OUT_IN)
    return fail(RF_EINVAL, "rf_weight_gradient: layout must be RF_IN_OUT or RF_OUT_IN");
  if (!valid_dtype(out_dtype)) return fail(RF_EINVAL, "rf_weight_gradient: out dtype must be RF_F32, RF_BF16 or RF_F16");
  const int64_t m = layout == RF_IN_OUT ? features : n_out, n = layout == RF_IN_OUT ? n_out : features;
  if (!out || ld_out < n) return fail(RF_EINVAL, "rf_weight_gradient: null out, or ld_out below its columns");
  if (rows > 0 && !grad_out) return fail(RF_EINVAL, "rf_weight_gradient: null gradient");
  const size_t oes = dtype_size(out_dtype), ges = dtype_size(grad_dtype);
  if (reinterpret_cast<uintptr_t>(out) % oes || reinterpret_cast<uintptr_t>(initial) % oes ||
      reinterpret_cast<uintptr_t>(grad_out) % ges)
    return fail(RF_EINVAL, "rf_weight_gradient: misaligned pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool in_place = grad_dtype == RF_BF16 && rows_vectorised(grad_out, ld_grad, RF_BF16);
  const Plan p = make_plan(rows, features, n_out, grad_dtype, in_place, plan_pairs());
  if (p.total() > workspace_bytes)
    return fail(RF_EINVAL, "rf_weight_gradient: workspace too small: " + std::to_string(p.total()) + " bytes needed");
  if (p.total() > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256))
    return fail(RF_EINVAL, "rf_weight_gradient: the workspace must be 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  Params P{};
  P.m = m;
  P.n = n;
  P.tiles_i = int(ceil_div(m, kTile));
  P.tiles_j = int(ceil_div(n, kTile));
  const int64_t tiles = int64_t(P.tiles_i) * P.tiles_j;
  P.whole = p.tail.whole;
  P.splits = p.tail.splits;
  P.units = P.whole + (tiles - P.whole) * P.splits;
  P.steps = int(p.steps);
  P.terms = p.terms;
  P.x_first = layout == RF_IN_OUT;
  P.initial = initial;
  P.out = out;
  P.ld_out = ld_out;
  P.out_dt = out_dtype;
  P.vec = ld_out % 4 == 0 && (reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(initial)) % (4 * oes) == 0;
  P.partial = reinterpret_cast<float*>(ws + p.x_bytes + p.terms_bytes);
  P.error = device_error_word();
  // bfloat16 operands, float32 accumulator, both operands MN-major.
  P.idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(kTile >> 3) << 17) |
            (uint32_t(kTile >> 4) << 24);

  if (rows > 0) {
    RF_TRY(rf_load_activation(saved, ws, p.ld_x, RF_BF16, stream));
    const void* g = grad_out;
    int64_t ldg = ld_grad;
    if (p.ld_terms) {
      const int64_t nv = p.ld_terms / 8;
      const int tx = int(nv < 256 ? nv : 256), ty = 256 / tx;
      const int64_t gx = std::min<int64_t>(ceil_div(rows, ty), 65535);
      k_grad_terms<<<dim3(unsigned(gx), unsigned(ceil_div(nv, tx))), dim3(unsigned(tx), unsigned(ty)), 0, st>>>(
          row_view(grad_out, ld_grad, grad_dtype, rows, n_out), reinterpret_cast<uint16_t*>(ws + p.x_bytes), rows, n_out,
          p.ld_terms, p.terms);
      RF_TRY(check_launch("k_grad_terms"));
      g = ws + p.x_bytes;
      ldg = p.ld_terms;
    }
    CUtensorMap mx, mg;
    RF_TRY(make_map(&mx, ws, features, rows, 1, p.ld_x));
    RF_TRY(make_map(&mg, g, n_out, rows, p.terms, ldg));
    RF_TRY(allow_smem());
    const int64_t pairs = std::min(P.units, max_pairs());
    RF_TRY(launch_dependent(k_weight_grad, unsigned(2 * pairs), kThreads, kSmemBytes, st, mx, mg, P));
  }
  if (P.whole == tiles) return RF_OK;
  return launch_dependent(k_weight_grad_join, unsigned((tiles - P.whole) * (kTile / 4)), 256, 0, st, P);
}
