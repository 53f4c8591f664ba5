// The norms before and after a block, with its gate, residual scale and the
// residual addition, forward and backward.
//
//   x' = x + s a(gamma) N_post(b),   y = N_pre(x')
//
// The C entry points and the kernels for every type and width; the usual
// types up to 8192 features go through rf_block_norm_typed.cuh's kernels, which
// hold their rows the same way and are several times as fast (these: 8192 x
// 12288 bfloat16 RMS forward 944 us, 0.85 TB/s, backward 1737; they read the
// parameters again for every row and tell the types apart at run time).
//
// Both directions cannot do without reading a row once, so it is held in registers
// while its statistics are formed, and each output is written once.  A row
// belongs to a team: one warp up to 1024 features (no barrier), else the
// whole CTA; a thread holds V vectors of 8 features, strided by the team, so
// loads are 16 bytes wide and the 4 lanes of an 8-bit block are neighbours.
//
// Backward, with n = N_pre's normalised x', g = dy w and mean over a row:
//   e  = dx' + r (g - mean(g) [layer] - n mean(g n))
//   h  = e s a w_post,  db = r_b (h - mean(h) [layer] - m mean(h m)),  m = normalised b
// Parameter gradients are sums over rows of four products only:
//   P = sum e a m, Q = sum e a, R = sum dy n, U = sum dy      (per feature)
// (a inside the sums when the gate varies by row, else outside):
//   dw_post = s P, dbias_post = s Q, ds = w P + bias Q, da = s (w P + bias Q),
//   dw_pre = R, dbias_pre = U.
// A CTA keeps them in registers over a chunk of rows of one gate group and
// writes one partial row; a second kernel adds the partials in order.
#include <algorithm>

#include "rf_block_norm.cuh"

namespace rf {
namespace bn {

// Sums of N values over a team.  A CTA's sum goes through one of two buffers
// in turn, so that one barrier per sum is enough; every thread adds the
// warps' values in the same order.
template <bool kWarp, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (&buf)[2][4][32], int& turn) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
  if (kWarp) return;
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) buf[turn][i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < nw; ++w) s += buf[turn][i][w];
    v[i] = s;
  }
  turn ^= 1;
}

// Normalises a row in place and returns its factor r.  Places behind the last
// feature hold 0 and stay 0.  The variance is taken around the mean, a second
// pass over the registers, so a large mean costs no digits.
template <int V, bool kWarp, bool kLayer>
__device__ __forceinline__ float normalise(float (&f)[V][8], int team, int lane, const Common& c,
                                           float (&buf)[2][4][32], int& turn) {
  if (kLayer) {
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[0] += f[v][k];
    team_sum<kWarp>(s, buf, turn);
    const float mean = s[0] * c.inv_d;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t col = int64_t(v * team + lane) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[v][k] = col + k < c.d ? f[v][k] - mean : 0.f;
    }
  }
  float q[1] = {0.f};
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) q[0] = fmaf(f[v][k], f[v][k], q[0]);
  team_sum<kWarp>(q, buf, turn);
  const float r = rsqrtf(fmaf(q[0], c.inv_d, c.eps));
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) f[v][k] *= r;
  return r;
}

template <int V, bool kWarp, bool kLayer>
__global__ void __launch_bounds__(kWarp ? 32 * kWarpsPerCta : 512) k_norm_fwd(const __grid_constant__ FwdArgs A) {
  __shared__ float buf[2][4][32];
  int turn = 0;
  const Common& c = A.c;
  const int team = kWarp ? 32 : int(blockDim.x);
  const int lane = kWarp ? int(threadIdx.x & 31) : int(threadIdx.x);
  const int64_t row = kWarp ? int64_t(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5) : int64_t(blockIdx.x);
  if (row >= c.rows) return;  // a whole team
  float x[V][8], b[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t col = int64_t(v * team + lane) * 8;
    load8(A.x, row, col, c.d, x[v]);
    if (A.b.p) load8(A.b, row, col, c.d, b[v]);
  }
  if (A.b.p) {
    if (A.sb.codes) {
#pragma unroll
      for (int v = 0; v < V; ++v) save_row8(A.sb, row, int64_t(v * team + lane) * 8, c.d, b[v]);
    }
    if (c.post_norm) normalise<V, kWarp, kLayer>(b, team, lane, c, buf, turn);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t col = int64_t(v * team + lane) * 8;
      float w[8];
      if (c.post_w.p) {
        param8(c.post_w, col, c.d, 1.f, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) b[v][k] *= w[k];
      }
      if (c.post_b.p) {
        param8(c.post_b, col, c.d, 0.f, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) b[v][k] += w[k];
      }
      gate8(c, row, col, w);
      float s[8];
      scale8(c, col, s);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[v][k] = fmaf(b[v][k] * w[k], s[k], x[v][k]);
      if (A.x_out.p) store8(A.x_out, row, col, c.d, x[v]);
      if (A.sx.codes) {
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = x[v][k];
        round8(A.x_out.dt, t);
        save_row8(A.sx, row, col, c.d, t);
      }
    }
  } else if (A.sx.codes) {
#pragma unroll
    for (int v = 0; v < V; ++v) save_row8(A.sx, row, int64_t(v * team + lane) * 8, c.d, x[v]);
  }
  if (!A.y.p) return;
  normalise<V, kWarp, kLayer>(x, team, lane, c, buf, turn);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int64_t col = int64_t(v * team + lane) * 8;
    float w[8];
    if (c.pre_w.p) {
      param8(c.pre_w, col, c.d, 1.f, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[v][k] *= w[k];
    }
    if (c.pre_b.p) {
      param8(c.pre_b, col, c.d, 0.f, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[v][k] += w[k];
    }
    store8(A.y, row, col, c.d, x[v]);
    if (A.sy.codes) {
      round8(A.y.dt, x[v]);
      save_row8(A.sy, row, col, c.d, x[v]);
    }
  }
}

template <int V, bool kWarp, bool kLayer, bool kBias>
__global__ void __launch_bounds__(kWarp ? 32 * kWarpsPerCta : 512) k_norm_bwd(const __grid_constant__ BwdArgs A) {
  constexpr int kSums = kBias ? 4 : 2;  // P, R, then Q, U
  __shared__ float buf[2][4][32];
  __shared__ float join[kWarp ? kSums : 1][kWarp ? V * 256 : 1];
  int turn = 0;
  const Common& c = A.c;
  const int team = kWarp ? 32 : int(blockDim.x);
  const int lane = kWarp ? int(threadIdx.x & 31) : int(threadIdx.x);
  const int warp = int(threadIdx.x >> 5);
  const bool has_y = A.gy.p != nullptr;
  const bool has_b = A.b.p != nullptr || A.sb.codes != nullptr;

  for (int64_t item = blockIdx.x; item < A.items; item += gridDim.x) {
    const int64_t group = item / A.chunks;
    const int64_t first = group * A.group_rows + (item - group * A.chunks) * A.rows_per_chunk;
    const int64_t last = min(first + A.rows_per_chunk, (group + 1) * A.group_rows);
    float acc[kSums][V][8];
#pragma unroll
    for (int i = 0; i < kSums; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[i][v][k] = 0.f;

    for (int64_t row = first + (kWarp ? warp : 0); row < last; row += kWarp ? kWarpsPerCta : 1) {
      float e[V][8], x[V][8], g[V][8];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int64_t col = int64_t(v * team + lane) * 8;
        if (A.gx.p) {
          load8(A.gx, row, col, c.d, e[v]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) e[v][k] = 0.f;
        }
        if (has_y) {
          load8(A.gy, row, col, c.d, g[v]);
          if (A.sx.codes) load8(A.sx, row, col, x[v]);
          else load8(A.x, row, col, c.d, x[v]);
        }
      }
      if (has_y) {
        const float r = normalise<V, kWarp, kLayer>(x, team, lane, c, buf, turn);
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float w[8];
          param8(c.pre_w, int64_t(v * team + lane) * 8, c.d, 1.f, w);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            acc[1][v][k] = fmaf(g[v][k], x[v][k], acc[1][v][k]);
            if (kBias) acc[kSums - 1][v][k] += g[v][k];
            g[v][k] *= w[k];
            s[0] = fmaf(g[v][k], x[v][k], s[0]);
            s[1] += g[v][k];
          }
        }
        team_sum<kWarp>(s, buf, turn);
        const float mgn = s[0] * c.inv_d, mg = kLayer ? s[1] * c.inv_d : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) e[v][k] = fmaf(r, g[v][k] - mg - x[v][k] * mgn, e[v][k]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) store8(A.dx, row, int64_t(v * team + lane) * 8, c.d, e[v]);
      if (!has_b) continue;

#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int64_t col = int64_t(v * team + lane) * 8;
        if (A.sb.codes) load8(A.sb, row, col, x[v]);
        else load8(A.b, row, col, c.d, x[v]);
      }
      const float rb = c.post_norm ? normalise<V, kWarp, kLayer>(x, team, lane, c, buf, turn) : 1.f;
      float s[3] = {0.f, 0.f, 0.f};  // sum h m, sum h, sum e s n (a gate per row)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int64_t col = int64_t(v * team + lane) * 8;
        float a[8], w[8], sc[8];
        gate8(c, row, col, a);
        scale8(c, col, sc);
        param8(c.post_w, col, c.d, 1.f, w);
        float n[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) n[k] = x[v][k] * w[k];
        if (kBias && c.post_b.p) {
          float bias[8];
          param8(c.post_b, col, c.d, 0.f, bias);
#pragma unroll
          for (int k = 0; k < 8; ++k) n[k] += bias[k];
        }
        if (A.row_gate && A.dgate) {
          if (c.gate_per_channel) {
            float dg[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) dg[k] = e[v][k] * sc[k] * n[k] * gate_slope(a[k], c.gate_act);
            store8(row_out_dev(A.dgate, c.d, c.gate.dt), row, col, c.d, dg);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) s[2] += col + k < c.d ? e[v][k] * sc[k] * n[k] : 0.f;
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float ea = A.row_gate ? e[v][k] * a[k] : e[v][k];
          acc[0][v][k] = fmaf(ea, x[v][k], acc[0][v][k]);
          if (kBias) acc[2][v][k] += ea;
          const float h = col + k < c.d ? e[v][k] * a[k] * sc[k] * w[k] : 0.f;
          e[v][k] = h;
          s[0] = fmaf(h, x[v][k], s[0]);
          s[1] += h;
        }
      }
      const bool token_gate = A.row_gate && A.dgate && !c.gate_per_channel;
      if (c.post_norm || token_gate) {
        team_sum<kWarp>(s, buf, turn);
        if (token_gate && lane == 0) {
          const float a = gate_value(ld_as_float(c.gate.p, c.gate.dt, row), c.gate_act);
          st_from_float(A.dgate, c.gate.dt, row, s[2] * gate_slope(a, c.gate_act));
        }
      }
      if (c.post_norm) {
        const float mhm = s[0] * c.inv_d, mh = kLayer ? s[1] * c.inv_d : 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
          for (int k = 0; k < 8; ++k) e[v][k] = rb * (e[v][k] - mh - x[v][k] * mhm);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) store8(A.db, row, int64_t(v * team + lane) * 8, c.d, e[v]);
    }

    if (!A.partial) continue;
    float* out = A.partial + item * kSums * A.ldp;
    if (kWarp) {
      // The warps' sums, added in the order of the warps.
      for (int w = 0; w < kWarpsPerCta; ++w) {
        __syncthreads();
        if (warp == w) {
#pragma unroll
          for (int i = 0; i < kSums; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                float& t = join[i][(k * V + v) * 32 + lane];
                t = w ? t + acc[i][v][k] : acc[i][v][k];
              }
        }
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int i = 0; i < kSums; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v)
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[i][v][k] = join[i][(k * V + v) * 32 + lane];
      }
      __syncthreads();
      if (warp != 0) continue;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t col = int64_t(v * team + lane) * 8;
      if (col >= A.ldp) continue;
#pragma unroll
      for (int i = 0; i < kSums; ++i) {
        float4* o = reinterpret_cast<float4*>(out + i * A.ldp + col);
        o[0] = make_float4(acc[i][v][0], acc[i][v][1], acc[i][v][2], acc[i][v][3]);
        o[1] = make_float4(acc[i][v][4], acc[i][v][5], acc[i][v][6], acc[i][v][7]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Partial rows -> parameter gradients.
// ---------------------------------------------------------------------------
struct ColArgs {
  Common c;
  const float* partial;
  int64_t ldp, groups, chunks;
  int32_t sums;              // 2 or 4 rows per item
  int32_t group_gate;        // the gate is constant within a group
  void *pre_w, *pre_b, *post_w, *post_b, *scale, *gate;  // gradients, null: not wanted
  float* gate_cols;          // [groups][ldp]: summands of a scalar gate's gradient
  float* scale_cols;         // [ldp]: summands of a scalar scale's gradient
};
constexpr int kColLanes = 32;

__global__ void __launch_bounds__(32 * kColLanes) k_norm_cols(const __grid_constant__ ColArgs A) {
  __shared__ float sm[4][kColLanes][33];
  const Common& c = A.c;
  const int tx = int(threadIdx.x) & 31, ty = int(threadIdx.x) >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + tx;
  const bool in = col < c.d;
  const int64_t cc = in ? col : 0;
  const float w = c.post_w.p ? ld_as_float(c.post_w.p, c.post_w.dt, cc) : 1.f;
  const float bias = c.post_b.p ? ld_as_float(c.post_b.p, c.post_b.dt, cc) : 0.f;
  const float s = c.scale.p ? ld_as_float(c.scale.p, c.scale.dt, c.scale_per_channel ? cc : 0) : c.scale_value;
  float P = 0.f, Q = 0.f, R = 0.f, U = 0.f;  // over all groups, P and Q times the group's gate

  // One group's sums -> its gate's gradient and the totals.
  auto close_group = [&](int64_t g, float p, float q) {
    float a = 1.f;
    if (A.group_gate) {
      const int64_t i = c.gate_per_channel ? g * c.d + cc : g;
      a = gate_value(ld_as_float(c.gate.p, c.gate.dt, i), c.gate_act);
      const float da = s * fmaf(w, p, bias * q) * gate_slope(a, c.gate_act);
      if (in && A.gate) {
        if (c.gate_per_channel) st_from_float(A.gate, c.gate.dt, i, da);
        else A.gate_cols[g * A.ldp + col] = da;
      }
    }
    P = fmaf(a, p, P);
    Q = fmaf(a, q, Q);
  };
  auto add_items = [&](int64_t i0, int64_t i1, int64_t step, float& p, float& q) {
    if (!in) return;
#pragma unroll 4
    for (int64_t i = i0; i < i1; i += step) {
      const float* o = A.partial + i * A.sums * A.ldp + col;
      p += o[0];
      R += o[A.ldp];
      if (A.sums == 4) {
        q += o[2 * A.ldp];
        U += o[3 * A.ldp];
      }
    }
  };
  if (A.groups >= kColLanes) {
    for (int64_t g = ty; g < A.groups; g += kColLanes) {
      float p = 0.f, q = 0.f;
      add_items(g * A.chunks, (g + 1) * A.chunks, 1, p, q);
      close_group(g, p, q);
    }
  } else if (A.groups > 0) {
    // Few groups: each gets a share of the lanes, whose parts its first lane adds.
    const int share = kColLanes / int(A.groups);
    const int g = ty / share, j = ty - g * share;
    float p = 0.f, q = 0.f;
    if (g < A.groups) add_items(g * A.chunks + j, (int64_t(g) + 1) * A.chunks, share, p, q);
    sm[0][ty][tx] = p;
    sm[1][ty][tx] = q;
    __syncthreads();
    if (j == 0 && g < A.groups) {
      for (int k = 1; k < share; ++k) {
        p += sm[0][ty + k][tx];
        q += sm[1][ty + k][tx];
      }
      close_group(g, p, q);
    }
    __syncthreads();
  }
  sm[0][ty][tx] = P;
  sm[1][ty][tx] = Q;
  sm[2][ty][tx] = R;
  sm[3][ty][tx] = U;
  __syncthreads();
  if (ty != 0 || !in) return;
  for (int k = 1; k < kColLanes; ++k) {
    P += sm[0][k][tx];
    Q += sm[1][k][tx];
    R += sm[2][k][tx];
    U += sm[3][k][tx];
  }
  if (A.pre_w) st_from_float(A.pre_w, c.pre_w.dt, col, R);
  if (A.pre_b) st_from_float(A.pre_b, c.pre_b.dt, col, U);
  if (A.post_w) st_from_float(A.post_w, c.post_w.dt, col, s * P);
  if (A.post_b) st_from_float(A.post_b, c.post_b.dt, col, s * Q);
  if (A.scale) {
    const float ds = fmaf(w, P, bias * Q);
    if (c.scale_per_channel) st_from_float(A.scale, c.scale.dt, col, ds);
    else A.scale_cols[col] = ds;
  }
}

// out[r] = sum over d columns of cols[r][...], in a fixed order.
__global__ void __launch_bounds__(256) k_norm_rowsum(const float* cols, int64_t ld, int64_t d, void* out, int dt) {
  __shared__ float buf[2][4][32];
  int turn = 0;
  float s[1] = {0.f};
  const float* r = cols + int64_t(blockIdx.x) * ld;
  for (int64_t i = threadIdx.x; i < d; i += blockDim.x) s[0] += r[i];
  team_sum<false>(s, buf, turn);
  if (threadIdx.x == 0) st_from_float(out, dt, blockIdx.x, s[0]);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Threads of a row's team and vectors per thread: whole panels of 16 vectors,
// so that a saved row's last panel is complete.
struct Team {
  int threads, vectors;
  bool warp;
};
Team team_of(int64_t d) {
  const int64_t nv = ceil_div(d, kPanel8) * (kPanel8 / 8);
  if (nv <= 32) return {32, 1, true};
  if (nv <= 64) return {32, 2, true};
  if (nv <= 128) return {32, 4, true};
  const int v = nv <= 1024 ? 2 : 4;
  return {int(round_up(ceil_div(nv, v), 32)), v, false};
}

// Rows of an item, and how many items; never a row of partial sums for fewer
// than 2 rows of a team unless the group is that short.
struct Split {
  int64_t groups, group_rows, chunks, rows_per_chunk, items;
};
Split split_rows(const rf_block_norm& p) {
  Split s{};
  const bool grouped = p.gate.value && p.gate_rows > 1;
  s.group_rows = grouped ? p.gate_rows : p.rows;
  s.groups = p.rows == 0 ? 0 : p.rows / s.group_rows;
  // An item for each SM, which holds one CTA of the typed kernels.
  const int64_t target = 148;
  const int64_t per = 2 * typed_team(p.features).teams;
  if (s.groups > 0) {
    const int64_t want = std::max<int64_t>(1, target / s.groups);
    s.chunks = std::max<int64_t>(1, std::min(want, s.group_rows / per));
    s.rows_per_chunk = ceil_div(s.group_rows, s.chunks);
    s.chunks = ceil_div(s.group_rows, s.rows_per_chunk);
  }
  s.items = s.groups * s.chunks;
  return s;
}

struct Needs {
  bool cols, bias, gate_cols, scale_cols;
};
Needs needs_of(const rf_block_norm& p) {
  Needs n{};
  const bool group_gate = p.gate.value && p.gate.grad && p.gate_rows != 1;
  n.cols = p.pre_weight.grad || p.pre_bias.grad || p.post_weight.grad || p.post_bias.grad || p.residual_scale.grad ||
           group_gate;
  n.bias = p.pre_bias.value || p.post_bias.value;
  n.gate_cols = group_gate && !p.gate_per_channel;
  n.scale_cols = p.residual_scale.grad && !p.scale_per_channel;
  return n;
}

rf_status check_param(const rf_norm_param& w, const char* what) {
  if (!w.value) {
    if (w.grad) return fail(RF_EINVAL, std::string(what) + ": a gradient without its value");
    return RF_OK;
  }
  if (!valid_dtype(w.dtype)) return fail(RF_EINVAL, std::string(what) + ": dtype must be RF_F32, RF_BF16 or RF_F16");
  if ((reinterpret_cast<uintptr_t>(w.value) | reinterpret_cast<uintptr_t>(w.grad)) % dtype_size(w.dtype))
    return fail(RF_EINVAL, std::string(what) + ": misaligned pointer");
  return RF_OK;
}
rf_status check_norm(const rf_block_norm* p) {
  if (!p) return fail(RF_EINVAL, "rf_block_norm: null parameters");
  if (p->rows < 0 || p->rows > 0x7FFFFFFF || p->features <= 0 || p->features > kMaxNorm)
    return fail(RF_EINVAL, "rf_block_norm: rows in [0, 2^31) and features in [1, 16384]");
  if (p->kind != RF_RMS_NORM && p->kind != RF_LAYER_NORM)
    return fail(RF_EINVAL, "rf_block_norm: kind must be RF_RMS_NORM or RF_LAYER_NORM");
  if (!(p->eps >= 0.f)) return fail(RF_EINVAL, "rf_block_norm: eps must be >= 0");
  RF_TRY(check_param(p->pre_weight, "rf_block_norm: pre_weight"));
  RF_TRY(check_param(p->pre_bias, "rf_block_norm: pre_bias"));
  RF_TRY(check_param(p->post_weight, "rf_block_norm: post_weight"));
  RF_TRY(check_param(p->post_bias, "rf_block_norm: post_bias"));
  RF_TRY(check_param(p->residual_scale, "rf_block_norm: residual_scale"));
  RF_TRY(check_param(p->gate, "rf_block_norm: gate"));
  if (!p->post_norm && (p->post_weight.value || p->post_bias.value))
    return fail(RF_EINVAL, "rf_block_norm: post_weight and post_bias need post_norm");
  if (p->gate.value) {
    if (p->gate_act != RF_GATE_IDENTITY && p->gate_act != RF_GATE_SIGMOID && p->gate_act != RF_GATE_TANH)
      return fail(RF_EINVAL, "rf_block_norm: unknown gate activation");
    if (p->gate_rows <= 0 || p->rows % p->gate_rows)
      return fail(RF_EINVAL, "rf_block_norm: gate_rows must divide rows");
  }
  return RF_OK;
}
rf_status check_array(const rf_rows* t, int64_t rows, int64_t d, const char* what, bool saved_ok) {
  if (!t) return fail(RF_EINVAL, std::string(what) + ": null description");
  if (t->saved) {
    if (!saved_ok) return fail(RF_EINVAL, std::string(what) + ": cannot be a saved activation");
    RF_TRY(check_saved(t->saved, what));
    if (t->saved->rows != rows || t->saved->features != d)
      return fail(RF_EINVAL, std::string(what) + ": the saved activation has another shape");
    return RF_OK;
  }
  if (!valid_dtype(t->dtype)) return fail(RF_EINVAL, std::string(what) + ": dtype must be RF_F32, RF_BF16 or RF_F16");
  if (t->ld < d) return fail(RF_EINVAL, std::string(what) + ": row stride below the number of features");
  if (rows > 0 && !t->data) return fail(RF_EINVAL, std::string(what) + ": null pointer");
  if (reinterpret_cast<uintptr_t>(t->data) % dtype_size(t->dtype))
    return fail(RF_EINVAL, std::string(what) + ": misaligned pointer");
  return RF_OK;
}
bool present(const rf_rows* t) { return t && (t->data || t->saved); }

Common common_of(const rf_block_norm& p) {
  auto par = [](const rf_norm_param& w) { return Param{w.value, w.dtype}; };
  Common c{};
  c.rows = p.rows;
  c.d = p.features;
  c.gate_rows = p.gate.value ? p.gate_rows : 1;
  c.pre_w = par(p.pre_weight);
  c.pre_b = par(p.pre_bias);
  c.post_w = par(p.post_weight);
  c.post_b = par(p.post_bias);
  c.scale = par(p.residual_scale);
  c.gate = par(p.gate);
  c.eps = p.eps;
  c.scale_value = p.scale;
  c.inv_d = float(1.0 / double(p.features));
  c.post_norm = p.post_norm;
  c.scale_per_channel = p.scale_per_channel;
  c.gate_per_channel = p.gate_per_channel;
  c.gate_act = p.gate_act;
  return c;
}
RowView view(const rf_rows* t, const rf_block_norm& p) {
  return present(t) && t->data ? row_view(t->data, t->ld, t->dtype, p.rows, p.features) : RowView{};
}
RowOut out(const rf_rows* t) {
  return present(t) ? row_out(const_cast<void*>(t->data), t->ld, t->dtype) : RowOut{};
}

template <bool kLayer>
void launch_fwd(const Team& t, const FwdArgs& A, cudaStream_t st) {
  if (t.warp) {
    const unsigned g = unsigned(ceil_div(A.c.rows, kWarpsPerCta)), b = 32 * kWarpsPerCta;
    if (t.vectors == 1) k_norm_fwd<1, true, kLayer><<<g, b, 0, st>>>(A);
    else if (t.vectors == 2) k_norm_fwd<2, true, kLayer><<<g, b, 0, st>>>(A);
    else k_norm_fwd<4, true, kLayer><<<g, b, 0, st>>>(A);
  } else {
    const unsigned g = unsigned(A.c.rows), b = unsigned(t.threads);
    if (t.vectors == 2) k_norm_fwd<2, false, kLayer><<<g, b, 0, st>>>(A);
    else k_norm_fwd<4, false, kLayer><<<g, b, 0, st>>>(A);
  }
}
template <bool kLayer, bool kBias>
void launch_bwd(const Team& t, const BwdArgs& A, cudaStream_t st) {
  const unsigned g = unsigned(std::min<int64_t>(A.items, 148 * 32)), b = unsigned(t.warp ? 32 * kWarpsPerCta : t.threads);
  if (t.warp) {
    if (t.vectors == 1) k_norm_bwd<1, true, kLayer, kBias><<<g, b, 0, st>>>(A);
    else if (t.vectors == 2) k_norm_bwd<2, true, kLayer, kBias><<<g, b, 0, st>>>(A);
    else k_norm_bwd<4, true, kLayer, kBias><<<g, b, 0, st>>>(A);
  } else {
    if (t.vectors == 2) k_norm_bwd<2, false, kLayer, kBias><<<g, b, 0, st>>>(A);
    else k_norm_bwd<4, false, kLayer, kBias><<<g, b, 0, st>>>(A);
  }
}

size_t workspace_bytes(const rf_block_norm& p) {
  const Needs n = needs_of(p);
  if (!n.cols) return 0;
  const Split s = split_rows(p);
  const size_t ldp = size_t(round_up(p.features, 8));
  size_t floats = size_t(s.items) * (n.bias ? 4 : 2) * ldp;
  if (n.gate_cols) floats += size_t(s.groups) * ldp;
  if (n.scale_cols) floats += ldp;
  return floats * 4;
}

}  // namespace bn
}  // namespace rf

using namespace rf;

extern "C" rf_status rf_block_norm_forward(const rf_block_norm* p, const rf_rows* x, const rf_rows* branch,
                                           const rf_rows* x_out, const rf_rows* y, const rf_saved_activation* saved_x,
                                           const rf_saved_activation* saved_branch, const rf_saved_activation* saved_y,
                                           void* stream) {
  using namespace rf::bn;
  RF_TRY(check_norm(p));
  const int64_t rows = p->rows, d = p->features;
  RF_TRY(check_array(x, rows, d, "rf_block_norm_forward: x", false));
  if (rows == 0) return RF_OK;  // arrays without elements have no address
  const bool has_b = present(branch), has_y = present(y);
  if (has_b) {
    RF_TRY(check_array(branch, rows, d, "rf_block_norm_forward: branch", false));
    RF_TRY(check_array(x_out, rows, d, "rf_block_norm_forward: x_out", false));
  } else if (saved_branch) {
    return fail(RF_EINVAL, "rf_block_norm_forward: saved_branch without a branch");
  } else if (p->post_weight.value || p->post_bias.value || p->gate.value || p->residual_scale.value) {
    return fail(RF_EINVAL, "rf_block_norm_forward: the branch's parameters without a branch");
  }
  if (has_y) RF_TRY(check_array(y, rows, d, "rf_block_norm_forward: y", false));
  else if (saved_y) return fail(RF_EINVAL, "rf_block_norm_forward: saved_y without y");
  else if (p->pre_weight.value || p->pre_bias.value)
    return fail(RF_EINVAL, "rf_block_norm_forward: pre_weight and pre_bias without y");
  const rf_saved_activation* saved[3] = {saved_x, saved_branch, saved_y};
  for (const rf_saved_activation* s : saved) {
    if (!s) continue;
    RF_TRY(check_saved(s, "rf_block_norm_forward"));
    if (s->rows != rows || s->features != d)
      return fail(RF_EINVAL, "rf_block_norm_forward: a saved activation has another shape");
  }
  if (!has_b && !has_y && !saved_x) return RF_OK;
  FwdArgs A{};
  A.c = common_of(*p);
  A.x = view(x, *p);
  if (has_b) {
    A.b = view(branch, *p);
    A.x_out = out(x_out);
  }
  if (has_y) A.y = out(y);
  if (saved_x) A.sx = saved8(*saved_x);
  if (saved_branch) A.sb = saved8(*saved_branch);
  if (saved_y) A.sy = saved8(*saved_y);
  const Team t = team_of(d);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (try_typed_fwd(*p, A, st)) return check_launch("k_norm_fwd_typed");
  if (p->kind == RF_LAYER_NORM) launch_fwd<true>(t, A, st);
  else launch_fwd<false>(t, A, st);
  return check_launch("k_norm_fwd");
}

extern "C" rf_status rf_block_norm_workspace_size(const rf_block_norm* p, size_t* bytes) {
  if (!bytes) return fail(RF_EINVAL, "rf_block_norm_workspace_size: null output");
  RF_TRY(rf::bn::check_norm(p));
  *bytes = rf::bn::workspace_bytes(*p);
  return RF_OK;
}

extern "C" rf_status rf_block_norm_backward(const rf_block_norm* p, const rf_rows* grad_x, const rf_rows* grad_y,
                                            const rf_rows* x, const rf_rows* branch, const rf_rows* out_x,
                                            const rf_rows* out_branch, void* workspace, size_t ws_bytes,
                                            void* stream) {
  using namespace rf::bn;
  RF_TRY(check_norm(p));
  const int64_t rows = p->rows, d = p->features;
  const bool has_gx = present(grad_x), has_gy = present(grad_y), has_b = present(branch);
  if (has_gx) RF_TRY(check_array(grad_x, rows, d, "rf_block_norm_backward: grad_x", false));
  if (has_gy) {
    RF_TRY(check_array(grad_y, rows, d, "rf_block_norm_backward: grad_y", false));
    RF_TRY(check_array(x, rows, d, "rf_block_norm_backward: x", true));
  }
  if (has_b) {
    RF_TRY(check_array(branch, rows, d, "rf_block_norm_backward: branch", true));
    RF_TRY(check_array(out_branch, rows, d, "rf_block_norm_backward: out_branch", false));
  } else if (rows > 0 && (p->post_weight.grad || p->post_bias.grad || p->residual_scale.grad || p->gate.grad)) {
    return fail(RF_EINVAL, "rf_block_norm_backward: gradients of the branch's parameters without a branch");
  }
  RF_TRY(check_array(out_x, rows, d, "rf_block_norm_backward: out_x", false));
  const size_t need = workspace_bytes(*p);
  if (need > ws_bytes || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)))
    return fail(RF_EINVAL, "rf_block_norm_backward: needs " + std::to_string(need) +
                               " bytes of 16-byte aligned workspace");
  const Needs n = needs_of(*p);
  const Split s = split_rows(*p);
  const int64_t ldp = round_up(d, 8);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  float* partial = static_cast<float*>(workspace);
  if (rows > 0) {
    BwdArgs A{};
    A.c = common_of(*p);
    if (has_gx) A.gx = view(grad_x, *p);
    if (has_gy) {
      A.gy = view(grad_y, *p);
      if (x->saved) A.sx = saved8(*x->saved);
      else A.x = view(x, *p);
    }
    if (has_b) {
      if (branch->saved) A.sb = saved8(*branch->saved);
      else A.b = view(branch, *p);
      A.db = out(out_branch);
    }
    A.dx = out(out_x);
    A.row_gate = p->gate.value && p->gate_rows == 1;
    A.dgate = A.row_gate ? p->gate.grad : nullptr;
    A.partial = n.cols ? partial : nullptr;
    A.ldp = ldp;
    A.sums = n.bias ? 4 : 2;
    A.items = s.items;
    A.chunks = s.chunks;
    A.rows_per_chunk = s.rows_per_chunk;
    A.group_rows = s.group_rows;
    const Team t = team_of(d);
    if (try_typed_bwd(*p, A, n.bias, st)) {
    } else if (p->kind == RF_LAYER_NORM) n.bias ? launch_bwd<true, true>(t, A, st) : launch_bwd<true, false>(t, A, st);
    else n.bias ? launch_bwd<false, true>(t, A, st) : launch_bwd<false, false>(t, A, st);
    RF_TRY(check_launch("k_norm_bwd"));
  }
  if (!n.cols) return RF_OK;
  ColArgs C{};
  C.c = common_of(*p);
  C.partial = partial;
  C.ldp = ldp;
  C.groups = s.groups;
  C.chunks = s.chunks;
  C.sums = n.bias ? 4 : 2;
  C.group_gate = p->gate.value && p->gate_rows != 1;
  C.pre_w = p->pre_weight.grad;
  C.pre_b = p->pre_bias.grad;
  C.post_w = p->post_weight.grad;
  C.post_b = p->post_bias.grad;
  C.scale = p->residual_scale.grad;
  C.gate = C.group_gate ? p->gate.grad : nullptr;
  float* next = partial + s.items * C.sums * ldp;
  if (n.gate_cols) {
    C.gate_cols = next;
    next += s.groups * ldp;
  }
  if (n.scale_cols) C.scale_cols = next;
  k_norm_cols<<<unsigned(ceil_div(d, 32)), 32 * kColLanes, 0, st>>>(C);
  RF_TRY(check_launch("k_norm_cols"));
  if (n.gate_cols && s.groups > 0) {
    k_norm_rowsum<<<unsigned(s.groups), 256, 0, st>>>(C.gate_cols, ldp, d, p->gate.grad, p->gate.dtype);
    RF_TRY(check_launch("k_norm_rowsum"));
  }
  if (n.scale_cols) {
    k_norm_rowsum<<<1, 256, 0, st>>>(C.scale_cols, ldp, d, p->residual_scale.grad, p->residual_scale.dtype);
    RF_TRY(check_launch("k_norm_rowsum"));
  }
  return RF_OK;
}
