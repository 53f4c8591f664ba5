// Backward pass of the typed block norms (rf_block_norm_typed.cuh), one source
// file for each kind of norm, since they take minutes to compile.
#pragma once

#include "rf_block_norm_typed.cuh"

namespace rf {
namespace bn {

namespace {

// One vector of x or b as it lies in memory: 8 elements, or 8 codes and a step.
template <int DT, bool kSaved, bool kVec>
struct Held {
  Vec<DT, kVec> vec;
  __device__ __forceinline__ void fetch(const RowView& t, const Saved8&, int64_t, int row, int col, int n) {
    vec.fetch(t, at(row, t.ld, col), n);
  }
  __device__ __forceinline__ void values(const RowView& t, const Saved8&, float (&f)[8]) const {
    unpack<DT>(vec.get(t), f);
  }
};
template <int DT, bool kVec>
struct Held<DT, true, kVec> {
  uint2 codes;
  uint32_t step;
  __device__ __forceinline__ void fetch(const RowView&, const Saved8& s, int64_t step0, int row, int col, int n) {
    codes = n > 0 ? __ldg(reinterpret_cast<const uint2*>(s.codes + at(row, s.ld, col))) : make_uint2(0, 0);
    step = n > 0 ? __ldg(s.scales + step0 + 4 * int64_t(row)) : 1u;
  }
  __device__ __forceinline__ void values(const RowView&, const Saved8& s, float (&f)[8]) const {
    decode4(codes.x, s.format, f);
    decode4(codes.y, s.format, f + 4);
    mul8(f, both(step_value(step)));
  }
};

template <int XT, int BT, int V, bool kLayer, bool kSaved, bool kVec>
__global__ void __launch_bounds__(kTypedThreads, 1) k_norm_bwd_typed(const __grid_constant__ BwdArgs A, int team_threads) {
  constexpr int kSums = kLayer ? 4 : 2;  // P, R, then Q, U
  // Wider rows, float32 branches and rows off the 16-byte boundaries (whose vectors
  // take twice the registers on their way) have none for the next row: with it,
  // LayerNorm 16384 x 4096 in float32 took 486 instead of 394 us.
  constexpr bool kAhead = kVec && V == 1 && BT != RF_F32;
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

    Vec<XT, kVec> ngx[V];
    Vec<BT, kVec> ngy[V];
    Held<XT, kSaved, kVec> nx[V];
    Held<BT, kSaved, kVec> nb[V];
    auto fetch = [&](int r) {
      const bool in = r < last && r >= 0;  // r may pass 2^31 behind the last row
      const int row = in ? r : first;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int live = in ? n[v] : 0;
        ngx[v].fetch(A.gx, at(row, A.gx.ld, col[v]), has_gx ? live : 0);
        ngy[v].fetch(A.gy, at(row, A.gy.ld, col[v]), has_y ? live : 0);
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
        unpack<XT>(ngx[v].get(A.gx), e[v]);
        unpack<BT>(ngy[v].get(A.gy), g[v]);
        nx[v].values(A.x, A.sx, x[v]);
        nb[v].values(A.b, A.sb, b[v]);
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
      for (int v = 0; v < V; ++v) store_part<XT, kVec>(A.dx, at(row, A.dx.ld, col[v]), n[v], pack<XT>(e[v]));
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
          if (A.dgate && c.gate_per_channel && n[v] > 0) {
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
      for (int v = 0; v < V; ++v) store_part<BT, kVec>(A.db, at(row, A.db.ld, col[v]), n[v], pack<BT>(e[v]));
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
          if (n[v] <= 0) continue;
          float4* o = reinterpret_cast<float4*>(out + i * A.ldp + col[v]);
          o[0] = make_float4(acc[i][v][0], acc[i][v][1], acc[i][v][2], acc[i][v][3]);
          o[1] = make_float4(acc[i][v][4], acc[i][v][5], acc[i][v][6], acc[i][v][7]);
        }
      }
    }
  }
}

template <bool kLayer>
bool typed_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st) {
  const bool saved = A.sx.codes || A.sb.codes;
  const int xt = A.dx.dt, bt = A.db.p ? A.db.dt : A.gy.p ? A.gy.dt : xt;
  if (p.features > kMaxTyped || (!kLayer && bias) || !type_is(A.gx, xt) || !type_is(A.gy, bt) || !type_is(A.x, xt) ||
      !type_is(A.b, bt) || (saved && (A.x.p || A.b.p)) || !type_is(A.dx, xt) || !type_is(A.db, bt))
    return false;
  const bool vec = p.features % 8 == 0 && whole_vectors(A.gx) && whole_vectors(A.gy) && whole_vectors(A.x) &&
                   whole_vectors(A.b) && whole_vectors(A.dx) && whole_vectors(A.db);
  const TypedTeam t = typed_team(p.features);
  const unsigned g = unsigned(std::min<int64_t>(A.items, 148 * 32)), b = unsigned(t.threads * t.teams);
  const size_t smem = t.teams > 1 ? size_t(kLayer ? 4 : 2) * t.threads * 8 * t.vectors * 4 : 0;  // at most 32 KB
  return with_types(xt, bt, vec, [&](auto x, auto y, auto w) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value;
    constexpr bool W = decltype(w)::value;
    auto go = [&](auto kernel) { kernel<<<g, b, smem, st>>>(A, t.threads); };
    auto by_v = [&](auto v) {
      constexpr int V = decltype(v)::value;
      saved ? go(k_norm_bwd_typed<X, B, V, kLayer, true, W>) : go(k_norm_bwd_typed<X, B, V, kLayer, false, W>);
    };
    t.vectors == 1 ? by_v(std::integral_constant<int, 1>{}) : by_v(std::integral_constant<int, 2>{});
  });
}

}  // namespace
}  // namespace bn
}  // namespace rf
