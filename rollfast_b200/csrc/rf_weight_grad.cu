// Weight gradient X^T G read straight from an activation saved in 8 bits.
//
//   out[i][o] = initial[i][o] + sum_t X[t][i] G[t][o]    (or its transpose)
//
// X [T][K] is the saved activation (rf_act8.cuh), G [T][N] the gradient of
// the product's output.  The sum runs over tokens, along which both operands
// are strided, so both are MN-major tensor-core operands, and the block steps
// of X differ along the sum, so they cannot be applied to the accumulator: X
// is turned into bfloat16 on its way to shared memory, which is exact because
// the steps are powers of two.  The 16-bit copy of X never exists in memory.
//
// One persistent CTA pair (cluster of 2, tcgen05 cta_group::2) per 256 x 256
// output tile; each CTA brings 128 rows of one operand and 128 columns of the
// other, 64 tokens at a time:
//   warp 0      TMA: 64 x 128 codes, their 256 bytes of steps, and 64 x 128
//               of G (two 128-byte swizzled boxes) into a ring of kLoads
//   warp 1      the leader's lane 0 issues tcgen05.mma (M = N = 256, K = 16)
//   warps 2..5  epilogue: accumulator -> memory, while the next tile's
//               products run into the other half of TMEM
//   warps 6..9  codes -> bfloat16, into a ring of kOperands swizzled buffers
// Few tiles: the tokens are split over several units whose float32 partial
// tiles a second kernel adds in a fixed order.
#include <algorithm>
#include <mutex>

#include "rf_act8.cuh"
#include "rf_kernels.cuh"
#include "rf_tc.cuh"

namespace rf {
namespace wg {

using namespace rf::tc;

constexpr int kTile = 256;          // output tile of a CTA pair, both ways
constexpr int kHalf = 128;          // operand rows per CTA
constexpr int kTokens = 64;         // tokens per step
constexpr int kLoads = 6;           // ring of loaded tiles
constexpr int kOperands = 3;        // ring of converted tiles
constexpr int kGradBytes = kTokens * kHalf * 2;
constexpr int kCodeBytes = kTokens * kHalf;
constexpr int kStepBytes = kTokens * 4;
constexpr int kLoadBytes = kGradBytes + kCodeBytes + kStepBytes;
constexpr int kOperandBytes = kTokens * kHalf * 2;
constexpr int kConvertWarps = 4;
constexpr int kThreads = (6 + kConvertWarps) * 32;
constexpr int kStagingBytes = 4 * 32 * 33 * 4;
constexpr int kGradOff = 0;
constexpr int kOperandOff = kGradOff + kLoads * kGradBytes;
constexpr int kCodeOff = kOperandOff + kOperands * kOperandBytes;
constexpr int kStepOff = kCodeOff + kLoads * kCodeBytes;
constexpr int kStagingOff = kStepOff + kLoads * kStepBytes;
constexpr int kBarOff = kStagingOff + kStagingBytes;
constexpr int kSmemBytes = kBarOff + 256 + 1024;
static_assert(kSmemBytes <= 232448, "dynamic shared memory per CTA is at most 227 KB");
constexpr uint32_t kTmemCols = 512;

struct Params {
  const uint8_t* scales;   // steps of X
  int64_t scale_rows;
  int64_t m, n;            // output rows and columns
  int64_t rows;            // tokens
  int64_t units;           // tiles x splits
  int tiles_i, tiles_j;    // 256-row and 256-column blocks
  int splits;              // units per tile
  int steps;               // 64-token steps of all tokens
  int terms;               // bfloat16 terms of G (1, 2 or 3)
  int x_first;             // X is the row operand (out is [K][N]), else the column operand
  int panels;              // panels of steps
  int format;
  const void* initial;     // added when there is one unit per tile
  void* out;
  int64_t ld_out;
  int out_dt;
  float* partial;          // [splits][m][ld_partial] when splits > 1
  int64_t ld_partial;
  uint32_t idesc;
  int* error;              // the device's error word, may be null
};

// Unit -> (row block, column block, split).  All splits of a tile are
// neighbours; tiles go down the row blocks in groups of 8 so that the ~74 in
// flight share their operands' panels in L2.
__device__ __forceinline__ void decode_unit(const Params& P, int64_t u, int& I, int& J, int& s) {
  s = int(u % P.splits);
  const int t = int(u / P.splits);
  const int G = 8;
  const int grp = t / (G * P.tiles_j);
  const int first = grp * G;
  const int gm = min(P.tiles_i - first, G);
  const int r = t - grp * G * P.tiles_j;
  I = first + r % gm;
  J = r / gm;
}
__device__ __forceinline__ void split_range(const Params& P, int s, int& k0, int& k1) {
  k0 = int(int64_t(P.steps) * s / P.splits);
  k1 = int(int64_t(P.steps) * (s + 1) / P.splits);
}

__device__ __forceinline__ void record_error(const Params& P, int code, volatile int* abort_flag) {
  *abort_flag = 1;
  if (P.error) atomicCAS(P.error, 0, code);
}

__device__ __forceinline__ uint32_t bf2_mul(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf2_sub(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Four codes -> four bfloat16 (two words), times the step; every operation is
// exact.  int8: with b the byte, 0x4300 | (b & 0x7F) is 128 + (b & 0x7F) and
// 0x4300 | (b & 0x80) is 128 or 256, so their difference is the code.  e4m3:
// its exponent and significand in bfloat16's places stand for 2^-120 of the
// value (subnormals too).
template <int kFormat>
__device__ __forceinline__ void convert4(uint32_t w, uint32_t step2, uint32_t& lo, uint32_t& hi) {
  if (kFormat == RF_INT8) {
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    lo = bf2_mul(bf2_sub(a & 0xFF7FFF7Fu, a & 0xFF80FF80u), step2);
    hi = bf2_mul(bf2_sub(b & 0xFF7FFF7Fu, b & 0xFF80FF80u), step2);
  } else {
    const uint32_t a = __byte_perm(w, 0u, 0x1404), b = __byte_perm(w, 0u, 0x3424);
    const uint32_t k2p120 = 0x7B807B80u;
    lo = bf2_mul(bf2_mul((a & 0x80008000u) | ((a >> 4) & 0x07F007F0u), k2p120), step2);
    hi = bf2_mul(bf2_mul((b & 0x80008000u) | ((b >> 4) & 0x07F007F0u), k2p120), step2);
  }
}

// One 32 x 32 block of the output, lane = row in v[], through the warp's
// staging buffer so that a store covers a row's 32 columns.
__device__ __forceinline__ void store_block(const Params& P, int split, int64_t row0, int64_t col0, int lane,
                                            const float* v, float* stg) {
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 32; ++k) stg[lane * 33 + k] = v[k];
  __syncwarp();
  const int64_t col = col0 + lane;
  if (col >= P.n) return;
  const int rows = int(P.m - row0 < 32 ? P.m - row0 : 32);
  if (P.splits > 1) {
    float* o = P.partial + (int64_t(split) * P.m + row0) * P.ld_partial + col;
    for (int r = 0; r < rows; ++r) o[int64_t(r) * P.ld_partial] = stg[r * 33 + lane];
  } else {
    const int64_t base = row0 * P.ld_out + col;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) {
      float x = stg[r * 33 + lane];
      const int64_t i = base + int64_t(r) * P.ld_out;
      if (P.initial) x += ld_as_float(P.initial, P.out_dt, i);
      st_from_float(P.out, P.out_dt, i, x);
    }
  }
}

template <int kFormat>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    k_weight_grad(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_grad,
                  const __grid_constant__ Params P) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBarOff);
  const uint32_t full0 = smem_u32(bars);                       // loads landed (own CTA)
  const uint32_t empty0 = full0 + 8 * kLoads;                  // loads consumed (commit, both CTAs)
  const uint32_t ready0 = empty0 + 8 * kLoads;                 // operand converted (leader: both CTAs' warps)
  const uint32_t free0 = ready0 + 8 * kOperands;               // operand consumed (commit, both CTAs)
  const uint32_t accf0 = free0 + 8 * kOperands;                // accumulator complete
  const uint32_t acce0 = accf0 + 16;                           // accumulator read (leader: both CTAs' warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kLoads + 2 * kOperands + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int64_t pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kLoads; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int s = 0; s < kOperands; ++s) {
      mbar_init(ready0 + 8 * s, 2 * kConvertWarps);
      mbar_init(free0 + 8 * s, 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(accf0 + 8 * s, 1);
      mbar_init(acce0 + 8 * s, 8);
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

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- loads (both CTAs, each its own halves) ----------------
      int stage = 0;
      uint32_t phase = 0;
      int64_t fills = 0;
      bool ok = true;
      for (int64_t u = pair; ok && u < P.units; u += npairs) {
        int I, J, s, k0, k1;
        decode_unit(P, u, I, J, s);
        split_range(P, s, k0, k1);
        const int xcol = (P.x_first ? I : J) * kTile + int(rank) * kHalf;
        const int gcol = (P.x_first ? J : I) * kTile + int(rank) * kHalf;
        const int panel = min(xcol / kPanel8, P.panels - 1);  // columns behind the last read zeros under any step
        for (int k = k0; ok && k < k1; ++k) {
          for (int term = 0; term < P.terms; ++term) {
            if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, abort_flag)) {
              record_error(P, kDevTimeoutProducer, abort_flag);
              ok = false;
              break;
            }
            const uint32_t fb = full0 + 8 * stage;
            mbar_arrive_expect_tx(fb, kLoadBytes);
            const uint32_t g = smem_u32(smem + kGradOff + stage * kGradBytes);
            tma_load_2d(smem_u32(smem + kCodeOff + stage * kCodeBytes), &tm_codes, fb, xcol, k * kTokens);
            bulk_load(smem_u32(smem + kStepOff + stage * kStepBytes),
                      P.scales + (int64_t(panel) * P.scale_rows + int64_t(k) * kTokens) * 4, fb, kStepBytes);
            tma_load_3d(g, &tm_grad, fb, gcol, k * kTokens, term);
            tma_load_3d(g + 8192, &tm_grad, fb, gcol + 64, k * kTokens, term);
            ++fills;
            if (++stage == kLoads) {
              stage = 0;
              phase ^= 1;
            }
          }
        }
      }
      // The last fills have been consumed: no copy into this CTA and no
      // commit's arrival on these barriers is pending.
      for (int64_t f = fills > kLoads ? fills - kLoads : 0; f < fills; ++f)
        mbar_drain(empty0 + 8 * uint32_t(f % kLoads), uint32_t((f / kLoads) & 1));
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ---------------- products ----------------
      int stage = 0, buf = 0;
      uint32_t bphase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      int tiles_done = 0;
      for (int64_t u = pair; ok && u < P.units; u += npairs) {
        int I, J, s, k0, k1;
        decode_unit(P, u, I, J, s);
        split_range(P, s, k0, k1);
        if (!mbar_wait_cluster(acce0 + 8 * acc, acc_phase ^ 1, abort_flag)) {
          record_error(P, kDevTimeoutMma, abort_flag);
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + uint32_t(acc * kTile);
        const int n_steps = (k1 - k0) * P.terms;
        for (int k = 0; k < n_steps; ++k) {
          if (!mbar_wait_cluster(ready0 + 8 * buf, bphase, abort_flag)) {
            record_error(P, kDevTimeoutMma, abort_flag);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t g = smem_u32(smem + kGradOff + stage * kGradBytes);
          const uint32_t x = smem_u32(smem + kOperandOff + buf * kOperandBytes);
          const uint32_t sa = P.x_first ? x : g, sb = P.x_first ? g : x;
#pragma unroll
          for (int q = 0; q < kTokens / 16; ++q)
            mma_f16_pair(d_tmem, sdesc(sa + q * 2048, 8192, 1024), sdesc(sb + q * 2048, 8192, 1024), P.idesc,
                         (k | q) != 0);
          mma_commit_pair(empty0 + 8 * stage);
          mma_commit_pair(free0 + 8 * buf);
          if (++stage == kLoads) stage = 0;
          if (++buf == kOperands) {
            buf = 0;
            bphase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair(accf0 + 8 * acc);
        ++tiles_done;
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // Both CTAs' epilogues have released the last two tiles.
      for (int k = tiles_done > 2 ? tiles_done - 2 : 0; k < tiles_done; ++k)
        mbar_drain(acce0 + 8 * uint32_t(k & 1), uint32_t((k >> 1) & 1));
    }
  } else if (warp < 6) {
    // ---------------- epilogue (both CTAs) ----------------
    const int quarter = warp & 3;  // TMEM lanes 32 * quarter .. + 31
    int acc = 0;
    uint32_t acc_phase = 0;
    float* stg = reinterpret_cast<float*>(smem + kStagingOff) + (warp - 2) * (32 * 33);
    for (int64_t u = pair; u < P.units; u += npairs) {
      int I, J, s;
      decode_unit(P, u, I, J, s);
      if (!mbar_wait(accf0 + 8 * acc, acc_phase, abort_flag)) {
        record_error(P, kDevTimeoutEpilogue, abort_flag);
        break;
      }
      tc_fence_after();
      const int64_t row0 = int64_t(I) * kTile + int64_t(rank) * kHalf + quarter * 32;
      const int64_t col0 = int64_t(J) * kTile;
      for (int ch = 0; ch < kTile / 32; ++ch) {
        if (row0 >= P.m || col0 + ch * 32 >= P.n) break;
        float v[32];
        __syncwarp();
        tmem_ld32(tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc * kTile + ch * 32), v);
        store_block(P, s, row0, col0 + ch * 32, lane, v, stg);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_rank(acce0 + 8 * acc, 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  } else {
    // ---------------- codes -> bfloat16 (both CTAs) ----------------
    const int tid = int(threadIdx.x) - 6 * 32;
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    int64_t fills = 0;
    bool ok = true;
    for (int64_t u = pair; ok && u < P.units; u += npairs) {
      int I, J, s, k0, k1;
      decode_unit(P, u, I, J, s);
      split_range(P, s, k0, k1);
      for (int k = k0; ok && k < k1; ++k) {
        for (int term = 0; term < P.terms; ++term) {
          ok = mbar_wait(full0 + 8 * stage, phase, abort_flag) && mbar_wait(free0 + 8 * buf, bphase ^ 1, abort_flag);
          if (!ok) {
            record_error(P, kDevTimeoutProducer, abort_flag);
            break;
          }
          const uint8_t* codes = smem + kCodeOff + stage * kCodeBytes;
          const uint8_t* steps = smem + kStepOff + stage * kStepBytes;
          uint8_t* dst = smem + kOperandOff + buf * kOperandBytes;
          const int live = int(P.rows - int64_t(k) * kTokens < kTokens ? P.rows - int64_t(k) * kTokens : kTokens);
#pragma unroll
          for (int it = 0; it < kTokens * 8 / (kConvertWarps * 32); ++it) {
            const int idx = it * (kConvertWarps * 32) + tid;
            const int t = idx >> 3, j = idx & 7;  // token, group of 16 features
            const uint4 c = *reinterpret_cast<const uint4*>(codes + t * kHalf + j * 16);
            uint32_t st = steps[t * 4 + (j >> 1)];
            // Tokens behind the last have zero codes and unwritten steps.
            if (t >= live) st = 127u;
            uint32_t st2 = st == kNanStep ? 0x7FC0u : st << 7;
            st2 |= st2 << 16;
            uint4 lo, hi;
            convert4<kFormat>(c.x, st2, lo.x, lo.y);
            convert4<kFormat>(c.y, st2, lo.z, lo.w);
            convert4<kFormat>(c.z, st2, hi.x, hi.y);
            convert4<kFormat>(c.w, st2, hi.z, hi.w);
            // MN-major, 128-byte swizzle: 64-feature blocks of [token][128
            // bytes], 16-byte chunk c of token t at c ^ (t & 7).  The two
            // blocks' threads store their chunks in opposite order, so that a
            // row's 8 stores fall on 8 different chunks.
            uint8_t* row = dst + (j >> 2) * 8192 + t * 128;
            const int c0 = (j & 3) * 2, sw = t & 7, odd = j >> 2;
            *reinterpret_cast<uint4*>(row + (((c0 + odd) ^ sw) << 4)) = odd ? hi : lo;
            *reinterpret_cast<uint4*>(row + (((c0 + 1 - odd) ^ sw) << 4)) = odd ? lo : hi;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_to_rank(ready0 + 8 * buf, 0));
          ++fills;
          if (++stage == kLoads) {
            stage = 0;
            phase ^= 1;
          }
          if (++buf == kOperands) {
            buf = 0;
            bphase ^= 1;
          }
        }
      }
    }
    if (tid == 0)
      for (int64_t f = fills > kOperands ? fills - kOperands : 0; f < fills; ++f)
        mbar_drain(free0 + 8 * uint32_t(f % kOperands), uint32_t((f / kOperands) & 1));
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

// out = initial + partial[0] + partial[1] + ... in this order.
__global__ void __launch_bounds__(256) k_weight_grad_join(const float* partial, int splits, int64_t m, int64_t n,
                                                          int64_t ld_partial, const void* initial, void* out,
                                                          int64_t ld_out, int out_dt) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 4;
  if (col >= n) return;
  const int live = int(n - col < 4 ? n - col : 4);
  for (int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y; row < m; row += int64_t(gridDim.x) * blockDim.y) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(partial + (int64_t(s) * m + row) * ld_partial + col);
      a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
    }
    const float f[4] = {a.x, a.y, a.z, a.w};
    const int64_t base = row * ld_out + col;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= live) break;
      float x = f[k];
      if (initial) x += ld_as_float(initial, out_dt, base + k);
      st_from_float(out, out_dt, base + k, x);
    }
  }
}

rf_status make_map(CUtensorMap* map, CUtensorMapDataType dt, const void* base, int rank, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  auto fn = tensor_map_encoder();
  if (!fn) return fail(RF_ECUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = fn(map, dt, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RF_ECUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(int(r)));
  return RF_OK;
}

// Units per tile.  With at least a wave of tiles the tokens stay whole.
// Otherwise the number that minimises a model of the time, in 64-token steps
// of one pair: waves of units, each its steps plus about 8 steps of prologue
// and epilogue, and the partial tiles' way through L2 (a pair moves a 256 x
// 256 float32 tile in about 3 steps; each split adds one tile written and read).
int choose_splits(int64_t tiles, int64_t steps, int64_t pairs) {
  if (tiles >= pairs || steps <= 1) return 1;
  double best = 0;
  int split = 1;
  for (int s = 1; s <= 64 && s * 2 <= steps; ++s) {
    const double waves = double(ceil_div(tiles * s, pairs));
    const double t = waves * (double(ceil_div(steps, s)) + 8) + (s > 1 ? 12 + 3.0 * double(tiles) * s / pairs : 0);
    if (s == 1 || t < best) {
      best = t;
      split = s;
    }
  }
  return split;
}

struct Plan {
  int64_t ld_terms;     // 0: G is read in place
  size_t terms_bytes, partial_bytes;
  int terms, splits;
  int64_t ld_partial, steps;
};

// `in_place`: the gradient is bfloat16 and its rows start on 16-byte boundaries.
Plan make_plan(int64_t rows, int64_t features, int64_t n_out, int32_t dt, bool in_place, int64_t pairs) {
  Plan p{};
  p.terms = dt == RF_BF16 ? 1 : dt == RF_F16 ? 2 : 3;
  p.steps = ceil_div(rows, kTokens);
  if (!(dt == RF_BF16 && in_place)) {
    p.ld_terms = round_up(n_out, 8);
    p.terms_bytes = align_up(size_t(p.terms) * size_t(rows) * size_t(p.ld_terms) * 2, 256);
  }
  const int64_t tiles = ceil_div(features, kTile) * ceil_div(n_out, kTile);
  p.splits = rows > 0 ? choose_splits(tiles, p.steps * p.terms, pairs) : 0;
  if (p.splits > p.steps) p.splits = int(p.steps);
  // Rows of the partial tiles are output rows, so either layout may be the
  // longer one; both are counted with the larger padding.
  p.ld_partial = 0;
  if (p.splits > 1)
    p.partial_bytes = size_t(p.splits) * 4 *
                      size_t(std::max(features * round_up(n_out, 4), n_out * round_up(features, 4)));
  return p;
}

template <int kFormat>
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
    if (cudaOccupancyMaxActiveClusters(&n, k_weight_grad<kFormat>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = num_sms() / 2;
    }
    c = n;
  }
  return c;
}

template <int kFormat>
rf_status allow_smem() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev & 63]) return RF_OK;
  const cudaError_t e =
      cudaFuncSetAttribute(k_weight_grad<kFormat>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (e != cudaSuccess) return fail(RF_ECUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  done[dev & 63] = true;
  return RF_OK;
}

template <int kFormat>
rf_status launch(const CUtensorMap& mc, const CUtensorMap& mg, const Params& P, cudaStream_t st) {
  RF_TRY(allow_smem<kFormat>());
  const int64_t cap = max_pairs<kFormat>();
  const int64_t pairs = P.units < cap ? P.units : cap;
  k_weight_grad<kFormat><<<unsigned(2 * pairs), kThreads, kSmemBytes, st>>>(mc, mg, P);
  return check_launch("k_weight_grad");
}

// Half the SMs: the split rule must not depend on a query that fails without
// a GPU, and a workspace planned on one B200 serves another.
int64_t plan_pairs() { return 74; }

rf_status check_sizes(int64_t rows, int64_t features, int64_t n_out, int32_t dt, int64_t ld) {
  if (!valid_dtype(dt)) return fail(RF_EINVAL, "rf_weight_gradient: grad dtype must be RF_F32, RF_BF16 or RF_F16");
  if (rows < 0 || rows > 0x7FFFFFFF - kTokens || features <= 0 || features > kMaxFeatures || n_out <= 0 ||
      n_out > kMaxFeatures)
    return fail(RF_EINVAL, "rf_weight_gradient: rows in [0, 2^31 - 64), features and n_out in [1, 2^26]");
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
  *bytes = p.terms_bytes + p.partial_bytes;
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
  Plan p = make_plan(rows, features, n_out, grad_dtype, in_place, plan_pairs());
  p.ld_partial = round_up(n, 4);
  if (p.terms_bytes + p.partial_bytes > workspace_bytes)
    return fail(RF_EINVAL, "rf_weight_gradient: workspace too small: " +
                               std::to_string(p.terms_bytes + p.partial_bytes) + " bytes needed");
  if (p.terms_bytes + p.partial_bytes > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256))
    return fail(RF_EINVAL, "rf_weight_gradient: the workspace must be 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* partial = reinterpret_cast<float*>(ws + p.terms_bytes);

  if (rows > 0) {
    const void* g = grad_out;
    int64_t ldg = ld_grad;
    if (p.ld_terms) {
      const int64_t nv = p.ld_terms / 8;
      const int tx = int(nv < 256 ? nv : 256), ty = 256 / tx;
      const int64_t gx = std::min<int64_t>(ceil_div(rows, ty), 65535);
      k_grad_terms<<<dim3(unsigned(gx), unsigned(ceil_div(nv, tx))), dim3(unsigned(tx), unsigned(ty)), 0, st>>>(
          row_view(grad_out, ld_grad, grad_dtype), reinterpret_cast<uint16_t*>(ws), rows, n_out, p.ld_terms, p.terms);
      RF_TRY(check_launch("k_grad_terms"));
      g = ws;
      ldg = p.ld_terms;
    }
    CUtensorMap mc, mg;
    const cuuint64_t cdims[2] = {cuuint64_t(saved->ld), cuuint64_t(rows)}, cstr[1] = {cuuint64_t(saved->ld)};
    const cuuint32_t cbox[2] = {kHalf, kTokens};
    RF_TRY(make_map(&mc, CU_TENSOR_MAP_DATA_TYPE_UINT8, saved->codes, 2, cdims, cstr, cbox, CU_TENSOR_MAP_SWIZZLE_NONE));
    const cuuint64_t gdims[3] = {cuuint64_t(n_out), cuuint64_t(rows), cuuint64_t(p.terms)};
    const cuuint64_t gstr[2] = {cuuint64_t(ldg) * 2, cuuint64_t(ldg) * 2 * cuuint64_t(rows)};
    const cuuint32_t gbox[3] = {64, kTokens, 1};
    RF_TRY(make_map(&mg, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, g, 3, gdims, gstr, gbox, CU_TENSOR_MAP_SWIZZLE_128B));
    Params P{};
    P.scales = saved->scales;
    P.scale_rows = saved->scale_rows;
    P.m = m;
    P.n = n;
    P.rows = rows;
    P.tiles_i = int(ceil_div(m, kTile));
    P.tiles_j = int(ceil_div(n, kTile));
    P.splits = p.splits;
    P.units = int64_t(P.tiles_i) * P.tiles_j * p.splits;
    P.steps = int(p.steps);
    P.terms = p.terms;
    P.x_first = layout == RF_IN_OUT;
    P.panels = int(ceil_div(features, kPanel8));
    P.format = saved->format;
    P.initial = initial;
    P.out = out;
    P.ld_out = ld_out;
    P.out_dt = out_dtype;
    P.partial = partial;
    P.ld_partial = p.ld_partial;
    P.error = device_error_word();
    // bfloat16 operands, float32 accumulator, both operands MN-major.
    P.idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(kTile >> 3) << 17) |
              (uint32_t(kTile >> 4) << 24);
    RF_TRY(saved->format == RF_INT8 ? launch<RF_INT8>(mc, mg, P, st) : launch<RF_E4M3>(mc, mg, P, st));
    if (p.splits == 1) return RF_OK;
  }
  const int64_t nv = ceil_div(n, 4);
  const int tx = int(nv < 256 ? nv : 256), ty = 256 / tx;
  const int64_t gx = std::min<int64_t>(ceil_div(m, ty), 65535);
  k_weight_grad_join<<<dim3(unsigned(gx), unsigned(ceil_div(nv, tx))), dim3(unsigned(tx), unsigned(ty)), 0, st>>>(
      partial, p.splits, m, n, p.ld_partial, initial, out, ld_out, out_dtype);
  return check_launch("k_weight_grad_join");
}
