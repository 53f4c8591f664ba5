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
// MEASURED.
#include <type_traits>

#include "rf_block_norm.cuh"

namespace rf {
namespace bn {

namespace {

constexpr int kTypedThreads = 512;
constexpr int kMaxTeams = 8;
constexpr int64_t kMaxTyped = 2 * kTypedThreads * 8;

// -- vectors of 8, whole or in part --------------------------------------------
// The first n of 8 elements at i; zeros behind.
template <int DT>
__device__ __forceinline__ Raw8<DT> load_part(const RowView& t, int64_t i, int n) {
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
template <int DT>
__device__ __forceinline__ void store_part(const RowOut& t, int64_t i, int n, const Raw8<DT>& r) {
  if (n == 8 && t.vec) {
    uint4* p = reinterpret_cast<uint4*>(static_cast<uint8_t*>(t.p) + i * (DT == RF_F32 ? 4 : 2));
    p[0] = r.u[0];
    if (DT == RF_F32) p[1] = r.u[DT == RF_F32 ? 1 : 0];
    return;
  }
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
struct TeamSums {
  float v[2][3][kMaxTeams][kTypedThreads / 32];
};
struct TeamCtx {
  int lane, threads, warps, id;
};
__device__ __forceinline__ TeamCtx team_ctx(int threads) {
  TeamCtx t;
  t.threads = threads;
  t.id = int(threadIdx.x) / threads;
  t.lane = int(threadIdx.x) - t.id * threads;
  t.warps = threads >> 5;
  return t;
}
// Sums of N values over a team, through one of two buffers in turn, so that
// one barrier per sum is enough: the team's own (0 is the CTA's).  Every
// thread adds the warps' values in the same order.
template <int N>
__device__ __forceinline__ void sum_over(float (&v)[N], const TeamCtx& t, TeamSums& s, int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
  if (t.warps == 1) return;
  if ((t.lane & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s.v[turn][i][t.id][t.lane >> 5] = v[i];
  asm volatile("bar.sync %0, %1;" ::"r"(t.id + 1), "r"(t.threads) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float x = 0.f;
    for (int w = 0; w < t.warps; ++w) x += s.v[turn][i][t.id][w];
    v[i] = x;
  }
  turn ^= 1;
}
// Normalises a row in place and returns its factor; places behind the last
// feature (n[v] of a vector are before it) hold 0 and stay 0.  The variance is
// taken around the mean, a second pass over the registers, so a large mean
// costs no digits.
template <int V, bool kLayer>
__device__ __forceinline__ float normalise_row(float (&f)[V][8], const int (&n)[V], const Common& c, const TeamCtx& t,
                                               TeamSums& s, int& turn) {
  if (kLayer) {
    float m[1] = {0.f};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) m[0] += f[v][k];
    sum_over(m, t, s, turn);
    const float mean = m[0] * c.inv_d;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] = k < n[v] ? f[v][k] - mean : 0.f;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) q[0] = fmaf(f[v][k], f[v][k], q[0]);
  sum_over(q, t, s, turn);
  const float r = rsqrtf(fmaf(q[0], c.inv_d, c.eps));
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) f[v][k] *= r;
  return r;
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

template <int XT, int BT, int V, bool kLayer>
__global__ void __launch_bounds__(kTypedThreads, V == 1 ? 2 : 1)
    k_norm_fwd_typed(const __grid_constant__ FwdArgs A, int team_threads) {
  __shared__ TeamSums sums;
  int turn = 0;
  const Common& c = A.c;
  const TeamCtx t = team_ctx(team_threads);
  const int teams = int(blockDim.x) / team_threads;
  const int64_t step = int64_t(gridDim.x) * teams;
  const bool has_b = A.b.p != nullptr, has_y = A.y.p != nullptr, fixed = gate_is_fixed(c);
  // x' = x + normalised * mul + add;  y = normalised * pw + pb
  float mul[V][8], pw[V][8], add[kLayer ? V : 1][8], pb[kLayer ? V : 1][8];
  int col[V], n[V];
  own_columns<V>(t, c, col, n);
#pragma unroll
  for (int v = 0; v < V; ++v) {
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
  int64_t row = int64_t(blockIdx.x) * teams + t.id;
  Raw8<XT> nx[V];
  Raw8<BT> nb[V];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      nx[v] = load_part<XT>(A.x, at * A.x.ld + col[v], at < c.rows ? n[v] : 0);
      nb[v] = load_part<BT>(A.b, at * A.b.ld + col[v], at < c.rows && has_b ? n[v] : 0);
    }
  };
  fetch(row);
  for (; row < c.rows; row += step) {
    float x[V][8], b[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      unpack<XT>(nx[v], x[v]);
      unpack<BT>(nb[v], b[v]);
    }
    fetch(row + step);
    if (has_b) {
      if (A.sb.codes) {
#pragma unroll
        for (int v = 0; v < V; ++v) save_row8(A.sb, row, col[v], c.d, b[v]);
      }
      if (c.post_norm) normalise_row<V, kLayer>(b, n, c, t, sums, turn);
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < 8; ++k) b[v][k] = kLayer ? fmaf(b[v][k], mul[v][k], add[kLayer ? v : 0][k]) : b[v][k] * mul[v][k];
        if (!fixed) {
          float g[8];
          gate8(c, row, col[v], g);
#pragma unroll
          for (int k = 0; k < 8; ++k) b[v][k] *= g[k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) x[v][k] += b[v][k];
        const Raw8<XT> raw = pack<XT>(x[v]);
        if (n[v]) store_part<XT>(A.x_out, row * A.x_out.ld + col[v], n[v], raw);
        if (A.sx.codes) {
          float r[8];
          unpack<XT>(raw, r);
          save_row8(A.sx, row, col[v], c.d, r);
        }
      }
    } else if (A.sx.codes) {
#pragma unroll
      for (int v = 0; v < V; ++v) save_row8(A.sx, row, col[v], c.d, x[v]);
    }
    if (!has_y) continue;
    normalise_row<V, kLayer>(x, n, c, t, sums, turn);
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[v][k] = kLayer ? fmaf(x[v][k], pw[v][k], pb[kLayer ? v : 0][k]) : x[v][k] * pw[v][k];
      const Raw8<BT> raw = pack<BT>(x[v]);
      if (n[v]) store_part<BT>(A.y, row * A.y.ld + col[v], n[v], raw);
      if (A.sy.codes) {
        unpack<BT>(raw, x[v]);
        save_row8(A.sy, row, col[v], c.d, x[v]);
      }
    }
  }
}

// One vector of x or b as it lies in memory: 8 elements, or 8 codes and a step.
template <int DT, bool kSaved>
struct Held {
  Raw8<DT> raw;
  __device__ __forceinline__ void fetch(const RowView& t, const Saved8&, int64_t row, int64_t col, int n) {
    raw = load_part<DT>(t, row * t.ld + col, n);
  }
  __device__ __forceinline__ void values(const Saved8&, float (&f)[8]) const { unpack<DT>(raw, f); }
};
template <int DT>
struct Held<DT, true> {
  uint2 codes;
  uint32_t step;
  __device__ __forceinline__ void fetch(const RowView&, const Saved8& s, int64_t row, int64_t col, int n) {
    codes = n ? __ldg(reinterpret_cast<const uint2*>(s.codes + row * s.ld + col)) : make_uint2(0, 0);
    step = n ? __ldg(s.scales + scale_index(s, row, col)) : 1u;
  }
  // Codes behind the last feature are 0; a NaN step must not reach them.
  __device__ __forceinline__ void values(const Saved8& s, float (&f)[8]) const {
    decode4(codes.x, s.format, f);
    decode4(codes.y, s.format, f + 4);
    const float st = step_value(step);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] *= st;
  }
};

template <int XT, int BT, int V, bool kLayer, bool kSaved>
__global__ void __launch_bounds__(kTypedThreads, 1) k_norm_bwd_typed(const __grid_constant__ BwdArgs A, int team_threads) {
  constexpr int kSums = kLayer ? 4 : 2;  // P, R, then Q, U
  constexpr bool kAhead = V == 1;        // wider rows have no registers for the next one
  __shared__ TeamSums sums;
  extern __shared__ float join[];        // [kSums][team_threads * 8 V] when a CTA has several teams
  int turn = 0;
  const Common& c = A.c;
  const TeamCtx t = team_ctx(team_threads);
  const int teams = int(blockDim.x) / team_threads;
  const bool has_y = A.gy.p != nullptr, has_gx = A.gx.p != nullptr;
  const bool has_b = A.b.p != nullptr || A.sb.codes != nullptr;
  float pw[V][8];
  int col[V], n[V];
  own_columns<V>(t, c, col, n);
#pragma unroll
  for (int v = 0; v < V; ++v) param8(c.pre_w, col[v], c.d, 1.f, pw[v]);

  for (int64_t item = blockIdx.x; item < A.items; item += gridDim.x) {
    const int64_t group = item / A.chunks;
    const int64_t first = group * A.group_rows + (item - group * A.chunks) * A.rows_per_chunk;
    const int64_t last = min(first + A.rows_per_chunk, (group + 1) * A.group_rows);
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
    Held<XT, kSaved> nx[V];
    Held<BT, kSaved> nb[V];
    auto fetch = [&](int64_t at) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int live = at < last ? n[v] : 0;
        ngx[v] = load_part<XT>(A.gx, at * A.gx.ld + col[v], has_gx ? live : 0);
        ngy[v] = load_part<BT>(A.gy, at * A.gy.ld + col[v], has_y ? live : 0);
        nx[v].fetch(A.x, A.sx, at, col[v], has_y ? live : 0);
        nb[v].fetch(A.b, A.sb, at, col[v], has_b ? live : 0);
      }
    };
    if (kAhead) fetch(first + t.id);
    for (int64_t row = first + t.id; row < last; row += teams) {
      if (!kAhead) fetch(row);
      float e[V][8], b[V][8];
      {
        float x[V][8], g[V][8];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          unpack<XT>(ngx[v], e[v]);
          unpack<BT>(ngy[v], g[v]);
          nx[v].values(A.sx, x[v]);
          nb[v].values(A.sb, b[v]);
        }
        if (kAhead) fetch(row + teams);
        if (has_y) {
          const float r = normalise_row<V, kLayer>(x, n, c, t, sums, turn);
          float s[2] = {0.f, 0.f};
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              acc[1][v][k] = fmaf(g[v][k], x[v][k], acc[1][v][k]);
              if (kLayer) acc[kSums - 1][v][k] += g[v][k];
              g[v][k] *= pw[v][k];
              s[0] = fmaf(g[v][k], x[v][k], s[0]);
              if (kLayer) s[1] += g[v][k];
            }
          sum_over(s, t, sums, turn);
          const float mgn = s[0] * c.inv_d, mg = kLayer ? s[1] * c.inv_d : 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              e[v][k] = fmaf(r, fmaf(-x[v][k], mgn, kLayer ? g[v][k] - mg : g[v][k]), e[v][k]);
              if (kLayer && k >= n[v]) e[v][k] = 0.f;
            }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (n[v]) store_part<XT>(A.dx, row * A.dx.ld + col[v], n[v], pack<XT>(e[v]));
      if (!has_b) continue;

      const float rb = c.post_norm ? normalise_row<V, kLayer>(b, n, c, t, sums, turn) : 1.f;
      float s[3] = {0.f, 0.f, 0.f};  // sum h m, sum h, sum e s n (a gate per row)
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
            s[2] += f[k];
            e[v][k] *= a[k];
          }
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          acc[0][v][k] = fmaf(e[v][k], b[v][k], acc[0][v][k]);
          if (kLayer) acc[kLayer ? 2 : 0][v][k] += e[v][k];
          e[v][k] *= mul[v][k];
          s[0] = fmaf(e[v][k], b[v][k], s[0]);
          if (kLayer) s[1] += e[v][k];
        }
      const bool token_gate = A.row_gate && A.dgate && !c.gate_per_channel;
      if (c.post_norm || token_gate) {
        sum_over(s, t, sums, turn);
        if (token_gate && t.lane == 0) {
          const float a = gate_value(ld_as_float(c.gate.p, c.gate.dt, row), c.gate_act);
          st_from_float(A.dgate, c.gate.dt, row, s[2] * gate_slope(a, c.gate_act));
        }
      }
      if (c.post_norm) {
        const float mhm = s[0] * c.inv_d, mh = kLayer ? s[1] * c.inv_d : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) e[v][k] = rb * fmaf(-b[v][k], mhm, kLayer ? e[v][k] - mh : e[v][k]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (n[v]) store_part<BT>(A.db, row * A.db.ld + col[v], n[v], pack<BT>(e[v]));
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

bool type_is(const RowView& t, int dt) { return !t.p || t.dt == dt; }
bool type_is(const RowOut& t, int dt) { return !t.p || t.dt == dt; }

// Calls f with the pair of types and V as constants; false for another pair.
template <typename F>
bool with_types(int xt, int bt, int vectors, F&& f) {
  auto by_v = [&](auto x, auto b) {
    if (vectors == 1) f(x, b, std::integral_constant<int, 1>{});
    else f(x, b, std::integral_constant<int, 2>{});
    return true;
  };
  using F32 = std::integral_constant<int, RF_F32>;
  using B16 = std::integral_constant<int, RF_BF16>;
  using F16 = std::integral_constant<int, RF_F16>;
  if (xt == RF_BF16 && bt == RF_BF16) return by_v(B16{}, B16{});
  if (xt == RF_F32 && bt == RF_BF16) return by_v(F32{}, B16{});
  if (xt == RF_F32 && bt == RF_F32) return by_v(F32{}, F32{});
  if (xt == RF_F16 && bt == RF_F16) return by_v(F16{}, F16{});
  return false;
}

}  // namespace

TypedTeam typed_team(int64_t d) {
  const int64_t nv = ceil_div(d, kPanel8) * (kPanel8 / 8);  // whole panels, for a saved row's last one
  const int v = nv <= kTypedThreads ? 1 : 2;
  const int t = int(std::min<int64_t>(round_up(ceil_div(nv, v), 32), kTypedThreads));
  return {t, v, std::min(kTypedThreads / t, kMaxTeams)};
}

bool try_typed_fwd(const rf_block_norm& p, const FwdArgs& A, cudaStream_t st) {
  const bool layer = p.kind == RF_LAYER_NORM;
  const int xt = A.x.dt, bt = A.b.p ? A.b.dt : A.y.p ? A.y.dt : xt;
  if (p.features > kMaxTyped || !type_is(A.x_out, xt) || !type_is(A.y, bt) ||
      (!layer && (p.pre_bias.value || p.post_bias.value)))
    return false;
  const TypedTeam t = typed_team(p.features);
  const int64_t ctas = ceil_div(p.rows, t.teams);
  const unsigned g = unsigned(std::min(ctas, int64_t(num_sms()) * (t.vectors == 1 ? 2 : 1)));
  const unsigned b = unsigned(t.threads * t.teams);
  return with_types(xt, bt, t.vectors, [&](auto x, auto y, auto v) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value, V = decltype(v)::value;
    if (layer) k_norm_fwd_typed<X, B, V, true><<<g, b, 0, st>>>(A, t.threads);
    else k_norm_fwd_typed<X, B, V, false><<<g, b, 0, st>>>(A, t.threads);
  });
}

bool try_typed_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st) {
  const bool layer = p.kind == RF_LAYER_NORM;
  const bool saved = A.sx.codes || A.sb.codes;
  const int xt = A.dx.dt, bt = A.db.p ? A.db.dt : A.gy.p ? A.gy.dt : xt;
  if (p.features > kMaxTyped || (!layer && bias) || !type_is(A.gx, xt) || !type_is(A.gy, bt) || !type_is(A.x, xt) ||
      !type_is(A.b, bt) || (saved && (A.x.p || A.b.p)))
    return false;
  const TypedTeam t = typed_team(p.features);
  const unsigned g = unsigned(std::min<int64_t>(A.items, 148 * 32)), b = unsigned(t.threads * t.teams);
  const size_t smem = t.teams > 1 ? size_t(layer ? 4 : 2) * t.threads * 8 * t.vectors * 4 : 0;  // at most 32 KB
  return with_types(xt, bt, t.vectors, [&](auto x, auto y, auto v) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value, V = decltype(v)::value;
    if (layer) saved ? k_norm_bwd_typed<X, B, V, true, true><<<g, b, smem, st>>>(A, t.threads)
                     : k_norm_bwd_typed<X, B, V, true, false><<<g, b, smem, st>>>(A, t.threads);
    else saved ? k_norm_bwd_typed<X, B, V, false, true><<<g, b, smem, st>>>(A, t.threads)
               : k_norm_bwd_typed<X, B, V, false, false><<<g, b, smem, st>>>(A, t.threads);
  });
}

}  // namespace bn
}  // namespace rf
