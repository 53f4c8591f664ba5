// Block norms for the usual element types: x and branch both bfloat16, both
// float16, both float32, or a float32 stream with a bfloat16 branch; up to
// 8192 features, RMS without biases or LayerNorm.  Everything else goes
// through rf_block_norm.cu's kernels.
//
// Bound by HBM.  A row belongs to a team of whole warps, 8 V features to a
// thread, and a CTA holds several teams when rows are short.  CTAs stay and
// walk down the rows, where registers allow with the next row's loads in
// flight; scale, gate and weight of a column are folded into one factor.  Rows
// that start off 16-byte boundaries, or are no whole number of vectors wide,
// are shifted into place (rf_act8.cuh).
//
// Measured on a B200 (a copy: 6549 GB/s), 16384 x 4096 bfloat16 RMS: forward
// 98 us (5.5 TB/s), with the 8-bit copies 174; backward 168 us (4.8 TB/s), from
// saved activations 186.  With copies and backward neither HBM (DRAM 44 to
// 47 % busy) nor the issue slots (55 %) are the bound, but the latency of a
// row's chain of sums with 16 warps an SM.  Backward beyond 4096 features a
// thread holds two vectors, which do not fit its 128 registers (700 to 1400
// bytes spilled): 8192 x 5120 in 194 us, 2.1 TB/s.
#pragma once

#include <type_traits>

#include "rf_block_norm.cuh"

namespace rf {
namespace bn {

namespace {

constexpr int kTypedThreads = 512;
constexpr int kFwdThreads = 768;  // forward, where registers suffice for more warps
constexpr int kMaxTeams = 12;
constexpr int64_t kMaxTyped = 2 * kTypedThreads * 8;
constexpr int kFwdVectors = 2;  // vectors per thread, forward

// -- vectors of 8, whole or in part --------------------------------------------
// A vector on its way from memory: with kVec rows are whole vectors on 16-byte
// boundaries, else they start and end anywhere (rf_act8.cuh).
template <int DT, bool kVec>
struct Vec {
  Raw8<DT> raw;
  __device__ __forceinline__ void fetch(const RowView& t, int64_t i, int left) {
    raw = left > 0 ? load_raw<DT>(t.p, i) : zero_raw<DT>();
  }
  __device__ __forceinline__ Raw8<DT> get(const RowView&) const { return raw; }
};
template <int DT>
struct Vec<DT, false> {
  Span8<DT> span;
  int64_t i;
  int left;
  __device__ __forceinline__ void fetch(const RowView& t, int64_t at, int l) {
    i = at, left = l;
    span = fetch_span<DT>(t, i, left);
  }
  __device__ __forceinline__ Raw8<DT> get(const RowView& t) const { return align_span<DT>(span, t, i, left); }
};
// Called by all lanes of a warp, `left` of the row's elements from the first on.
template <int DT, bool kVec>
__device__ __forceinline__ void store_part(const RowOut& t, int64_t i, int left, const Raw8<DT>& r) {
  if (!kVec) {
    store_span<DT>(t.p, i, left, r);
  } else if (left > 0) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<uint8_t*>(t.p) + i * (DT == RF_F32 ? 4 : 2));
    p[0] = r.u[0];
    if (DT == RF_F32) p[1] = r.u[DT == RF_F32 ? 1 : 0];
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
    n[v] = int(c.d) - col[v];  // elements of the row from there on, 0 or less behind it
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
// Step 1 for the blocks behind the last feature of every row's last panel,
// once for all rows: there a row that is not finite has NaNs for its zeros.
__device__ __forceinline__ void steps_behind(const Saved8& s, const Common& c) {
  const int first = (int(c.d) + kBlock8 - 1) / kBlock8;
  if (!s.codes || first % 4 == 0) return;
  uint8_t* p = s.scales + int64_t(first / 4) * s.scale_rows * 4;
  for (int64_t row = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; row < c.rows; row += int64_t(gridDim.x) * blockDim.x)
    for (int k = first % 4; k < 4; ++k) p[4 * row + k] = 1;
}
// A vector as it lies in memory (raw, f its values) into a saved row.
template <int DT>
__device__ __forceinline__ void save_raw(const Saved8& s, const Common& c, int64_t step0, int row, int col,
                                         const Raw8<DT>& raw, const float (&f)[8]) {
  const uint32_t st = step_byte(raw_max_bits<DT>(raw), s.format);
  const uint2 code = encode8(f, st, s.format);
  if (col < int(s.ld)) *reinterpret_cast<uint2*>(s.codes + at(row, s.ld, col)) = code;
  if ((col & (kBlock8 - 1)) == 0 && col < int(c.d)) s.scales[step0 + 4 * int64_t(row)] = uint8_t(st);
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
  auto go = [&](auto x, auto b) { vec ? f(x, b, std::true_type{}) : f(x, b, std::false_type{}); };
  if (xt == RF_BF16 && bt == RF_BF16) go(B16{}, B16{});
  else if (xt == RF_F32 && bt == RF_F32) go(F32{}, F32{});
  else if (xt == RF_F32 && bt == RF_BF16) go(F32{}, B16{});
  else if (xt == RF_F16 && bt == RF_F16) go(F16{}, F16{});
  else return false;
  return true;
}

TypedTeam team_for(int64_t d, int vectors, int threads = kTypedThreads) {
  const int64_t nv = ceil_div(d, kPanel8) * (kPanel8 / 8);  // whole panels, for a saved row's last one
  const int t = int(std::min<int64_t>(round_up(ceil_div(nv, vectors), 32), kTypedThreads));
  return {t, vectors, std::min(threads / t, kMaxTeams)};
}

}  // namespace
}  // namespace bn
}  // namespace rf
