// Block norms for the usual element types: x and branch both bfloat16, both
// float16, both float32, or a float32 stream with a bfloat16 branch; up to
// 8192 features, RMS without biases or LayerNorm.  Everything else goes
// through rf_block_norm.cu's kernels.
//
// Bound by HBM.  A row belongs to a team of whole warps, 8 V features to a
// thread, and a CTA holds several teams when rows are short.  CTAs stay and
// walk down the rows with the next row's loads in flight, and a thread keeps
// the parameters of its columns in registers, scale, gate and weight folded
// into one factor.  Rows on 16-byte boundaries move in 16-byte pieces, others
// element by element.
// Measured on a B200, 16384 x 4096 bfloat16 RMS norms (a copy: 6549 GB/s):
// Measured at 16384 x 4096 bfloat16 (RMSNorm): forward 100 us (5.4 TB/s), with
// the 8-bit copies 172; backward 170 us (4.7 TB/s), from saved activations 186.
// With copies and backward, the issue slots are the bound, not HBM.
#include <type_traits>

#include "rf_block_norm.cuh"

namespace rf {
namespace bn {

namespace {

constexpr int kTypedThreads = 512;
constexpr int kMaxTeams = 8;
constexpr int64_t kMaxTyped = 2 * kTypedThreads * 8;
constexpr int kFwdVectors = 2;  // vectors per thread, forward

// -- vectors of 8, whole or in part --------------------------------------------
// The first n of 8 elements at i; zeros behind.  kVec: rows of whole vectors
// on 16-byte boundaries, n is 0 or 8.
template <int DT, bool kVec>
__device__ __forceinline__ Raw8<DT> load_part(const RowView& t, int64_t i, int n) {
  if (kVec) return n ? load_raw<DT>(t.p, i) : zero_raw<DT>();
  if (n == 8 && t.vec) return load_raw<DT>(t.p, i);
  Raw8<DT> r = zero_raw<DT>();
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w[k] = 0u;
    if (k < n) {
      if (DT == RF_F32) w[k] = __ldg(static_cast<const uint32_t*>(t.p) + i + k);
      else w[k] = __ldg(static_cast<const uint16_t*>(t.p) + i + k);
    }
  }
  if (DT == RF_F32) {
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.u[DT == RF_F32 ? 1 : 0] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    r.u[0] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
  }
  return r;
}
template <int DT>
__device__ __forceinline__ Raw8<DT> pack(const float (&f)[8]) {
  Raw8<DT> r;
  if (DT == RF_F32) {
    r.u[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    r.u[DT == RF_F32 ? 1 : 0] =
        make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
  } else if (DT == RF_BF16) {
    r.u[0] = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  } else {
    r.u[0] = make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
  }
  return r;
}
template <int DT, bool kVec>
__device__ __forceinline__ void store_part(const RowOut& t, int64_t i, int n, const Raw8<DT>& r) {
  if (kVec || (n == 8 && t.vec)) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<uint8_t*>(t.p) + i * (DT == RF_F32 ? 4 : 2));
    p[0] = r.u[0];
    if (DT == RF_F32) p[1] = r.u[DT == RF_F32 ? 1 : 0];
    if (kVec) return;
  }
  if (n == 8 && t.vec) return;
  const uint4 b = r.u[DT == RF_F32 ? 1 : 0];
  const uint32_t w[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (k >= n) break;
    if (DT == RF_F32) static_cast<uint32_t*>(t.p)[i + k] = w[k];
    else static_cast<uint16_t*>(t.p)[i + k] = uint16_t(w[k >> 1] >> (16 * (k & 1)));
  }
}

// -- teams ---------------------------------------------------------------------
// Sums over a row cost more instructions than the row's own arithmetic when
// every value takes its own five shuffles and every thread adds every warp's
// part (99 instructions an element, backward).  So values share shuffles: of
// N = 2 or 4, a lane hands on one half and keeps the other until a half or a
// quarter of the warp carries each; the warps' parts are added the same way.
struct TeamSums {
  float v[2][kMaxTeams][4 * 16];  // per buffer and team: N x 16 warps, zeros for warps that are not there
};
struct TeamCtx {
  int lane, threads, id;
  bool alone;  // one warp
};
__device__ __forceinline__ TeamCtx team_ctx(int threads, TeamSums& s) {
  TeamCtx t;
  t.threads = threads;
  t.id = int(threadIdx.x) / threads;
  t.lane = int(threadIdx.x) - t.id * threads;
  t.alone = threads == 32;
  for (int i = int(threadIdx.x); i < int(sizeof(s.v) / 4); i += int(blockDim.x)) (&s.v[0][0][0])[i] = 0.f;
  __syncthreads();
  return t;
}
__device__ __forceinline__ float other(float x, int bit) { return __shfl_xor_sync(0xFFFFFFFFu, x, bit); }
// Two values into one: lanes with `bit` go on with b, the others with a.
__device__ __forceinline__ float fold(float a, float b, int lane, int bit) {
  const bool hi = lane & bit;
  return (hi ? b : a) + other(hi ? a : b, bit);
}
// Sums of N values over a team, through one of two buffers in turn, so that
// one barrier per sum is enough: the team's own (0 is the CTA's).  All threads
// get the same bits.
template <int N>
__device__ __forceinline__ void sum_over(float (&v)[N], const TeamCtx& t, TeamSums& s, int& turn) {
  static_assert(N == 1 || N == 2 || N == 4, "");
  constexpr int kSpan = 32 / N;  // lanes that carry one value
  const int lane = t.lane & 31;
  float x;
  if (N == 1) x = v[0] + other(v[0], 16);
  else if (N == 2) x = fold(v[0], v[N - 1], lane, 16);
  else x = fold(fold(v[0], v[N == 4 ? 2 : 0], lane, 16), fold(v[N == 4 ? 1 : 0], v[N - 1], lane, 16), lane, 8);
#pragma unroll
  for (int o = N == 1 ? 8 : kSpan / 2; o; o >>= 1) x += other(x, o);
  if (!t.alone) {
    float* part = s.v[turn][t.id];
    if ((lane & (kSpan - 1)) == 0) part[(lane / kSpan) * 16 + (t.lane >> 5)] = x;
    asm volatile("bar.sync %0, %1;" ::"r"(t.id + 1), "r"(t.threads) : "memory");
    if (N == 4) {
      const float2 p = *reinterpret_cast<const float2*>(part + (lane >> 3) * 16 + (lane & 7) * 2);
      x = p.x + p.y;
    } else {
      x = part[N == 2 ? lane : lane & 15];
    }
#pragma unroll
    for (int o = N == 4 ? 4 : 8; o; o >>= 1) x += other(x, o);
    turn ^= 1;
  }
  if (N == 1) v[0] = x;
  else
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xFFFFFFFFu, x, i * kSpan);
}

template <int V>
__device__ __forceinline__ float sum8(const float (&f)[V][8]) {
  float2 s = both(0.f);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 4; ++k) s = __fadd2_rn(s, pair(f[v], k));
  return s.x + s.y;
}
template <int V>
__device__ __forceinline__ float dot8(const float (&f)[V][8], const float (&g)[V][8]) {
  float2 s = both(0.f);
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 4; ++k) s = __ffma2_rn(pair(f[v], k), pair(g[v], k), s);
  return s.x + s.y;
}
// Zeros at and behind element n of a vector (kVec: n is 0 or 8).
template <bool kVec>
__device__ __forceinline__ void clear_behind(float (&f)[8], int n) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (kVec ? n > 0 : k < n) ? f[k] : 0.f;
}
// Takes a mean off; places behind the last feature stay 0.
template <int V, bool kVec>
__device__ __forceinline__ void centre(float (&f)[V][8], float mean, const int (&n)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) put_pair(f[v], k, __fadd2_rn(pair(f[v], k), both(-mean)));
    clear_behind<kVec>(f[v], n[v]);
  }
}
template <int V>
__device__ __forceinline__ void times(float (&f)[V][8], float r) {
#pragma unroll
  for (int v = 0; v < V; ++v) mul8(f[v], both(r));
}
__device__ __forceinline__ float factor(float sum_sq, const Common& c) { return rsqrtf(fmaf(sum_sq, c.inv_d, c.eps)); }
// Normalises a row in place.  The variance is taken around the mean, a second
// pass over the registers, so a large mean costs no digits.
template <int V, bool kLayer, bool kVec>
__device__ __forceinline__ void normalise_row(float (&f)[V][8], const int (&n)[V], const Common& c, const TeamCtx& t,
                                              TeamSums& s, int& turn) {
  if (kLayer) {
    float m[1] = {sum8<V>(f)};
    sum_over(m, t, s, turn);
    centre<V, kVec>(f, m[0] * c.inv_d, n);
  }
  float q[1] = {dot8<V>(f, f)};
  sum_over(q, t, s, turn);
  times<V>(f, factor(q[0], c));
}
// Element offset of a row's column; strides here are below 2^31.
__device__ __forceinline__ int64_t at(int row, int64_t ld, int col) {
  return int64_t(uint64_t(uint32_t(row)) * uint32_t(ld) + uint32_t(col));
}
template <int V>
__device__ __forceinline__ void own_columns(const TeamCtx& t, const Common& c, int (&col)[V], int (&n)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    col[v] = (v * t.threads + t.lane) * 8;
    n[v] = min(max(int(c.d) - col[v], 0), 8);
  }
}
// A gate that is the same for all rows is part of a column's factor.
__device__ __forceinline__ bool gate_is_fixed(const Common& c) { return !c.gate.p || c.gate_rows >= c.rows; }
// Offset of a column's step byte in row 0 of any activation saved with these
// rows, and whether the column lies in its panels.
__device__ __forceinline__ int64_t first_step(const Common& c, int col) {
  const int64_t scale_rows = (c.rows + 63) / 64 * 64;
  return ((int64_t(col) / kPanel8) * scale_rows) * 4 + (col % kPanel8) / kBlock8;
}
// A vector as it lies in memory (raw, f its values) into a saved row.
template <int DT>
__device__ __forceinline__ void save_raw(const Saved8& s, const Common& c, int64_t step0, int row, int col,
                                         const Raw8<DT>& raw, const float (&f)[8]) {
  const uint32_t st = step_byte(raw_max_bits<DT>(raw), s.format);
  const uint2 code = encode8(f, st, s.format);
  if (col < int(s.ld)) *reinterpret_cast<uint2*>(s.codes + at(row, s.ld, col)) = code;
  if ((col & (kBlock8 - 1)) == 0 && col < (int(c.d) + kPanel8 - 1) / kPanel8 * kPanel8)
    s.scales[step0 + 4 * int64_t(row)] = uint8_t(st);
}

template <int XT, int BT, bool kLayer, bool kSave, bool kVec>
__global__ void __launch_bounds__(kTypedThreads, 1)
    k_norm_fwd_typed(const __grid_constant__ FwdArgs A, int team_threads) {
  constexpr int V = kFwdVectors;
  __shared__ TeamSums sums;
  int turn = 0;
  const Common& c = A.c;
  const TeamCtx t = team_ctx(team_threads, sums);
  const int teams = int(blockDim.x) / team_threads;
  const int64_t step = int64_t(gridDim.x) * teams;
  const bool has_b = A.b.p != nullptr, has_y = A.y.p != nullptr, fixed = gate_is_fixed(c);
  // x' = x + normalised * mul + add;  y = normalised * pw + pb
  float mul[V][8], pw[V][8], add[kLayer ? V : 1][8], pb[kLayer ? V : 1][8];
  int col[V], n[V];
  int64_t step0[V];
  own_columns<V>(t, c, col, n);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    step0[v] = kSave ? first_step(c, col[v]) : 0;
    float w[8], g[8];
    param8(c.pre_w, col[v], c.d, 1.f, pw[v]);
    scale8(c, col[v], w);
    if (fixed) {
      gate8(c, 0, col[v], g);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] *= g[k];
    }
    param8(c.post_w, col[v], c.d, 1.f, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) mul[v][k] = k < n[v] ? g[k] * w[k] : 0.f;
    if (kLayer) {
      param8(c.pre_b, col[v], c.d, 0.f, pb[v]);
      param8(c.post_b, col[v], c.d, 0.f, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) add[v][k] = k < n[v] ? g[k] * w[k] : 0.f;
    }
  }
  const int rows = int(c.rows);
  int64_t next = int64_t(blockIdx.x) * teams + t.id;  // up to 2^31 and a step beyond
  Raw8<XT> nx[V];
  Raw8<BT> nb[V];
  auto fetch = [&]() {
    const bool live = next < rows;
    const int r = live ? int(next) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      nx[v] = load_part<XT, kVec>(A.x, at(r, A.x.ld, col[v]), live ? n[v] : 0);
      nb[v] = load_part<BT, kVec>(A.b, at(r, A.b.ld, col[v]), live && has_b ? n[v] : 0);
    }
  };
  // Float32 branches, and LayerNorm that saves, have no registers for the next
  // row: with it, 65536 x 768 saved took 281 instead of 240 us, and LayerNorm
  // 16384 x 4096 in float32 took 279 instead of 238 us.
  constexpr bool kAhead = BT != RF_F32 && !(kLayer && kSave);
  if (kAhead) fetch();
  while (next < rows) {
    const int row = int(next);
    if (!kAhead) fetch();
    Raw8<XT> rx[V];
    Raw8<BT> rb[V];
    float x[V][8], b[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rx[v] = nx[v];
      rb[v] = nb[v];
      unpack<XT>(rx[v], x[v]);
      unpack<BT>(rb[v], b[v]);
    }
    next += step;
    if (kAhead) fetch();
    if (has_b) {
      if (kSave && A.sb.codes) {
#pragma unroll
        for (int v = 0; v < V; ++v) save_raw<BT>(A.sb, c, step0[v], row, col[v], rb[v], b[v]);
      }
      if (c.post_norm) normalise_row<V, kLayer, kVec>(b, n, c, t, sums, turn);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (fixed) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = kLayer ? __fadd2_rn(pair(x[v], k), pair(add[kLayer ? v : 0], k)) : pair(x[v], k);
            put_pair(x[v], k, __ffma2_rn(pair(b[v], k), pair(mul[v], k), y));
          }
        } else {
          float g[8];
          gate8(c, row, col[v], g);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = kLayer ? __ffma2_rn(pair(b[v], k), pair(mul[v], k), pair(add[kLayer ? v : 0], k))
                                    : __fmul2_rn(pair(b[v], k), pair(mul[v], k));
            put_pair(x[v], k, __ffma2_rn(y, pair(g, k), pair(x[v], k)));
          }
        }
        rx[v] = pack<XT>(x[v]);
        if (n[v]) store_part<XT, kVec>(A.x_out, at(row, A.x_out.ld, col[v]), n[v], rx[v]);
      }
    }
    if (kSave && A.sx.codes) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f[8];
        unpack<XT>(rx[v], f);
        save_raw<XT>(A.sx, c, step0[v], row, col[v], rx[v], f);
      }
    }
    if (!has_y) continue;
    normalise_row<V, kLayer, kVec>(x, n, c, t, sums, turn);
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        put_pair(x[v], k, kLayer ? __ffma2_rn(pair(x[v], k), pair(pw[v], k), pair(pb[kLayer ? v : 0], k))
                                 : __fmul2_rn(pair(x[v], k), pair(pw[v], k)));
      const Raw8<BT> raw = pack<BT>(x[v]);
      if (n[v]) store_part<BT, kVec>(A.y, at(row, A.y.ld, col[v]), n[v], raw);
      if (kSave && A.sy.codes) {
        unpack<BT>(raw, x[v]);
        save_raw<BT>(A.sy, c, step0[v], row, col[v], raw, x[v]);
      }
    }
  }
}

// One vector of x or b as it lies in memory: 8 elements, or 8 codes and a step.
template <int DT, bool kSaved, bool kVec>
struct Held {
  Raw8<DT> raw;
  __device__ __forceinline__ void fetch(const RowView& t, const Saved8&, int64_t, int row, int col, int n) {
    raw = load_part<DT, kVec>(t, at(row, t.ld, col), n);
  }
  __device__ __forceinline__ void values(const Saved8&, float (&f)[8]) const { unpack<DT>(raw, f); }
};
template <int DT, bool kVec>
struct Held<DT, true, kVec> {
  uint2 codes;
  uint32_t step;
  __device__ __forceinline__ void fetch(const RowView&, const Saved8& s, int64_t step0, int row, int col, int n) {
    codes = n ? __ldg(reinterpret_cast<const uint2*>(s.codes + at(row, s.ld, col))) : make_uint2(0, 0);
    step = n ? __ldg(s.scales + step0 + 4 * int64_t(row)) : 1u;
  }
  __device__ __forceinline__ void values(const Saved8& s, float (&f)[8]) const {
    decode4(codes.x, s.format, f);
    decode4(codes.y, s.format, f + 4);
    mul8(f, both(step_value(step)));
  }
};

template <int XT, int BT, int V, bool kLayer, bool kSaved, bool kVec>
__global__ void __launch_bounds__(kTypedThreads, 1) k_norm_bwd_typed(const __grid_constant__ BwdArgs A, int team_threads) {
  constexpr int kSums = kLayer ? 4 : 2;  // P, R, then Q, U
  // Wider rows and float32 branches have no registers for the next row: with it,
  // LayerNorm 16384 x 4096 in float32 took 486 instead of 394 us.
  constexpr bool kAhead = V == 1 && BT != RF_F32;
  __shared__ TeamSums sums;
  extern __shared__ float join[];        // [kSums][team_threads * 8 V] when a CTA has several teams
  int turn = 0;
  const Common& c = A.c;
  const TeamCtx t = team_ctx(team_threads, sums);
  const int teams = int(blockDim.x) / team_threads;
  const bool has_y = A.gy.p != nullptr, has_gx = A.gx.p != nullptr;
  const bool has_b = A.b.p != nullptr || A.sb.codes != nullptr;
  const bool token_gate = A.row_gate && A.dgate && !c.gate_per_channel;
  float pw[V][8];
  int col[V], n[V];
  int64_t step0[V];  // x and b are saved alike, so their steps lie at the same offsets
  own_columns<V>(t, c, col, n);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    param8(c.pre_w, col[v], c.d, 1.f, pw[v]);
    step0[v] = kSaved ? first_step(c, col[v]) : 0;
  }

  for (int64_t item = blockIdx.x; item < A.items; item += gridDim.x) {
    const int64_t group = item / A.chunks;
    const int64_t first64 = group * A.group_rows + (item - group * A.chunks) * A.rows_per_chunk;
    const int first = int(first64), last = int(min(first64 + A.rows_per_chunk, (group + 1) * A.group_rows));
    // h = e mul: the scale, w_post, and the group's gate unless it varies by row.
    float mul[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float w[8], g[8];
      scale8(c, col[v], w);
      param8(c.post_w, col[v], c.d, 1.f, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) mul[v][k] = w[k] * g[k];
      if (!A.row_gate && c.gate.p) {
        gate8(c, first, col[v], g);
#pragma unroll
        for (int k = 0; k < 8; ++k) mul[v][k] *= g[k];
      }
    }
    float acc[kSums][V][8];
#pragma unroll
    for (int i = 0; i < kSums; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[i][v][k] = 0.f;

    Raw8<XT> ngx[V];
    Raw8<BT> ngy[V];
    Held<XT, kSaved, kVec> nx[V];
    Held<BT, kSaved, kVec> nb[V];
    auto fetch = [&](int r) {
      const bool in = r < last && r >= 0;  // r may pass 2^31 behind the last row
      const int row = in ? r : first;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int live = in ? n[v] : 0;
        ngx[v] = load_part<XT, kVec>(A.gx, at(row, A.gx.ld, col[v]), has_gx ? live : 0);
        ngy[v] = load_part<BT, kVec>(A.gy, at(row, A.gy.ld, col[v]), has_y ? live : 0);
        nx[v].fetch(A.x, A.sx, step0[v], row, col[v], has_y ? live : 0);
        nb[v].fetch(A.b, A.sb, step0[v], row, col[v], has_b ? live : 0);
      }
    };
    if (kAhead) fetch(first + t.id);
    for (int64_t row64 = first + t.id; row64 < last; row64 += teams) {
      const int row = int(row64);
      if (!kAhead) fetch(row);
      float e[V][8], b[V][8], x[V][8], g[V][8];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        unpack<XT>(ngx[v], e[v]);
        unpack<BT>(ngy[v], g[v]);
        nx[v].values(A.sx, x[v]);
        nb[v].values(A.sb, b[v]);
      }
      if (kAhead) fetch(int(uint32_t(row) + uint32_t(teams)));

      // Row sums.  RMS in one round, of the raw x: with n = r x, sum g n is
      // r sum g x.  LayerNorm takes the means off first.
      float sxx, sgx, sg = 0.f, sbb;
      if (kLayer) {
        float m[2] = {sum8<V>(x), sum8<V>(b)};
        sum_over(m, t, sums, turn);
        centre<V, kVec>(x, m[0] * c.inv_d, n);
        if (c.post_norm) centre<V, kVec>(b, m[1] * c.inv_d, n);
      }
      {
        float gw[V][8];
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 4; ++k) put_pair(gw[v], k, __fmul2_rn(pair(g[v], k), pair(pw[v], k)));
        float s[4] = {dot8<V>(x, x), dot8<V>(gw, x), dot8<V>(b, b), kLayer ? sum8<V>(gw) : 0.f};
        sum_over(s, t, sums, turn);
        sxx = s[0];
        sgx = s[1];
        sbb = s[2];
        sg = s[3];
        if (has_y) {
          const float r = factor(sxx, c);
          const float mgn = sgx * r * c.inv_d, mg = kLayer ? sg * c.inv_d : 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 nk = __fmul2_rn(pair(x[v], k), both(r));
              put_pair(acc[1][v], k, __ffma2_rn(pair(g[v], k), nk, pair(acc[1][v], k)));
              if (kLayer) put_pair(acc[kSums - 1][v], k, __fadd2_rn(pair(acc[kSums - 1][v], k), pair(g[v], k)));
              const float2 t0 = kLayer ? __fadd2_rn(pair(gw[v], k), both(-mg)) : pair(gw[v], k);
              put_pair(e[v], k, __ffma2_rn(both(r), __ffma2_rn(nk, both(-mgn), t0), pair(e[v], k)));
            }
            if (kLayer) clear_behind<kVec>(e[v], n[v]);
          }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (n[v]) store_part<XT, kVec>(A.dx, at(row, A.dx.ld, col[v]), n[v], pack<XT>(e[v]));
      if (!has_b) continue;

      const float rb = c.post_norm ? factor(sbb, c) : 1.f;
      times<V>(b, rb);
      float token = 0.f;  // sum e s n, the gradient of a gate per row
      if (A.row_gate) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a[8], sc[8], w[8], f[8];
          gate8(c, row, col[v], a);
          scale8(c, col[v], sc);
          param8(c.post_w, col[v], c.d, 1.f, w);
          param8(c.post_b, col[v], c.d, 0.f, f);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = e[v][k] * sc[k] * fmaf(b[v][k], w[k], f[k]);
          if (A.dgate && c.gate_per_channel && n[v]) {
            float dg[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) dg[k] = f[k] * gate_slope(a[k], c.gate_act);
            store8(row_out_dev(A.dgate, c.d, c.gate.dt), row, col[v], c.d, dg);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            token += f[k];
            e[v][k] *= a[k];
          }
        }
        if (token_gate) {
          float s[1] = {token};
          sum_over(s, t, sums, turn);
          if (t.lane == 0) {
            const float a = gate_value(ld_as_float(c.gate.p, c.gate.dt, row), c.gate_act);
            st_from_float(A.dgate, c.gate.dt, row, s[0] * gate_slope(a, c.gate_act));
          }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          put_pair(acc[0][v], k, __ffma2_rn(pair(e[v], k), pair(b[v], k), pair(acc[0][v], k)));
          if (kLayer) put_pair(acc[kLayer ? 2 : 0][v], k, __fadd2_rn(pair(acc[kLayer ? 2 : 0][v], k), pair(e[v], k)));
          put_pair(e[v], k, __fmul2_rn(pair(e[v], k), pair(mul[v], k)));
        }
      if (c.post_norm) {
        float mhm, mh = 0.f;
        if (kLayer) {
          float s[2] = {dot8<V>(e, b), sum8<V>(e)};
          sum_over(s, t, sums, turn);
          mhm = s[0] * c.inv_d;
          mh = s[1] * c.inv_d;
        } else {
          float s[1] = {dot8<V>(e, b)};
          sum_over(s, t, sums, turn);
          mhm = s[0] * c.inv_d;
        }
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 t0 = kLayer ? __fadd2_rn(pair(e[v], k), both(-mh)) : pair(e[v], k);
            put_pair(e[v], k, __fmul2_rn(both(rb), __ffma2_rn(pair(b[v], k), both(-mhm), t0)));
          }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (n[v]) store_part<BT, kVec>(A.db, at(row, A.db.ld, col[v]), n[v], pack<BT>(e[v]));
    }

    if (!A.partial) continue;
    const int width = t.threads * 8 * V;
    if (teams > 1) {
      // The teams' sums, added in the order of the teams.
      for (int w = 0; w < teams; ++w) {
        __syncthreads();
        if (t.id == w) {
#pragma unroll
          for (int i = 0; i < kSums; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                float& o = join[i * width + (v * 8 + k) * t.threads + t.lane];
                o = w ? o + acc[i][v][k] : acc[i][v][k];
              }
        }
      }
      __syncthreads();
      if (t.id == 0) {
#pragma unroll
        for (int i = 0; i < kSums; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[i][v][k] = join[i * width + (v * 8 + k) * t.threads + t.lane];
      }
    }
    if (t.id == 0) {
      float* out = A.partial + item * A.sums * A.ldp;  // ldp is a multiple of 8
#pragma unroll
      for (int i = 0; i < kSums; ++i) {
        if (i >= A.sums) break;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (!n[v]) continue;
          float4* o = reinterpret_cast<float4*>(out + i * A.ldp + col[v]);
          o[0] = make_float4(acc[i][v][0], acc[i][v][1], acc[i][v][2], acc[i][v][3]);
          o[1] = make_float4(acc[i][v][4], acc[i][v][5], acc[i][v][6], acc[i][v][7]);
        }
      }
    }
  }
}

// An absent array, or one of this type with a stride that fits 32 bits.
template <typename View>
bool type_is(const View& t, int dt) {
  return !t.p || (t.dt == dt && t.ld <= 0x7FFFFFFF);
}
template <typename View>
bool whole_vectors(const View& t) {
  return !t.p || t.vec;
}

// Calls f with the pair of types and whether rows are whole vectors as
// constants; false for a combination that has no kernel.
template <typename F>
bool with_types(int xt, int bt, bool vec, F&& f) {
  using F32 = std::integral_constant<int, RF_F32>;
  using B16 = std::integral_constant<int, RF_BF16>;
  using F16 = std::integral_constant<int, RF_F16>;
  if (xt == RF_BF16 && bt == RF_BF16) vec ? f(B16{}, B16{}, std::true_type{}) : f(B16{}, B16{}, std::false_type{});
  else if (xt == RF_F32 && bt == RF_F32) vec ? f(F32{}, F32{}, std::true_type{}) : f(F32{}, F32{}, std::false_type{});
  else if (xt == RF_F32 && bt == RF_BF16 && vec) f(F32{}, B16{}, std::true_type{});
  else if (xt == RF_F16 && bt == RF_F16 && vec) f(F16{}, F16{}, std::true_type{});
  else return false;
  return true;
}

TypedTeam team_for(int64_t d, int vectors) {
  const int64_t nv = ceil_div(d, kPanel8) * (kPanel8 / 8);  // whole panels, for a saved row's last one
  const int t = int(std::min<int64_t>(round_up(ceil_div(nv, vectors), 32), kTypedThreads));
  return {t, vectors, std::min(kTypedThreads / t, kMaxTeams)};
}

}  // namespace

TypedTeam typed_team(int64_t d) { return team_for(d, d <= kMaxTyped / 2 ? 1 : 2); }

bool try_typed_fwd(const rf_block_norm& p, const FwdArgs& A, cudaStream_t st) {
  const bool layer = p.kind == RF_LAYER_NORM;
  const int xt = A.x.dt, bt = A.b.p ? A.b.dt : A.y.p ? A.y.dt : xt;
  if (p.features > kMaxTyped || !type_is(A.x, xt) || !type_is(A.b, bt) || !type_is(A.x_out, xt) || !type_is(A.y, bt) ||
      (!layer && (p.pre_bias.value || p.post_bias.value)))
    return false;
  const bool vec = p.features % 8 == 0 && whole_vectors(A.x) && whole_vectors(A.b) && whole_vectors(A.x_out) &&
                   whole_vectors(A.y);
  const bool save = A.sx.codes || A.sb.codes || A.sy.codes;
  const TypedTeam t = team_for(p.features, kFwdVectors);
  const unsigned g = unsigned(std::min(ceil_div(p.rows, t.teams), int64_t(num_sms()))), b = unsigned(t.threads * t.teams);
  return with_types(xt, bt, vec, [&](auto x, auto y, auto w) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value;
    constexpr bool W = decltype(w)::value;
    auto go = [&](auto kernel) { kernel<<<g, b, 0, st>>>(A, t.threads); };
    if (layer) save ? go(k_norm_fwd_typed<X, B, true, true, W>) : go(k_norm_fwd_typed<X, B, true, false, W>);
    else save ? go(k_norm_fwd_typed<X, B, false, true, W>) : go(k_norm_fwd_typed<X, B, false, false, W>);
  });
}

bool try_typed_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st) {
  const bool layer = p.kind == RF_LAYER_NORM;
  const bool saved = A.sx.codes || A.sb.codes;
  const int xt = A.dx.dt, bt = A.db.p ? A.db.dt : A.gy.p ? A.gy.dt : xt;
  if (p.features > kMaxTyped || (!layer && bias) || !type_is(A.gx, xt) || !type_is(A.gy, bt) || !type_is(A.x, xt) ||
      !type_is(A.b, bt) || (saved && (A.x.p || A.b.p)) || !type_is(A.dx, xt) || !type_is(A.db, bt))
    return false;
  const bool vec = p.features % 8 == 0 && whole_vectors(A.gx) && whole_vectors(A.gy) && whole_vectors(A.x) &&
                   whole_vectors(A.b) && whole_vectors(A.dx) && whole_vectors(A.db);
  const TypedTeam t = typed_team(p.features);
  const unsigned g = unsigned(std::min<int64_t>(A.items, 148 * 32)), b = unsigned(t.threads * t.teams);
  const size_t smem = t.teams > 1 ? size_t(layer ? 4 : 2) * t.threads * 8 * t.vectors * 4 : 0;  // at most 32 KB
  return with_types(xt, bt, vec, [&](auto x, auto y, auto w) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value;
    constexpr bool W = decltype(w)::value;
    auto go = [&](auto kernel) { kernel<<<g, b, smem, st>>>(A, t.threads); };
    auto by_v = [&](auto v) {
      constexpr int V = decltype(v)::value;
      if (layer) saved ? go(k_norm_bwd_typed<X, B, V, true, true, W>) : go(k_norm_bwd_typed<X, B, V, true, false, W>);
      else saved ? go(k_norm_bwd_typed<X, B, V, false, true, W>) : go(k_norm_bwd_typed<X, B, V, false, false, W>);
    };
    t.vectors == 1 ? by_v(std::integral_constant<int, 1>{}) : by_v(std::integral_constant<int, 2>{});
  });
}

}  // namespace bn
}  // namespace rf
