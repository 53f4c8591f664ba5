// Forward pass of the typed block norms (rf_block_norm_typed.cuh).
#include "rf_block_norm_typed.cuh"

namespace rf {
namespace bn {

namespace {

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
  Vec<XT, kVec> nx[V];
  Vec<BT, kVec> nb[V];
  auto fetch = [&]() {
    const bool live = next < rows;
    const int r = live ? int(next) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      nx[v].fetch(A.x, at(r, A.x.ld, col[v]), live ? n[v] : 0);
      nb[v].fetch(A.b, at(r, A.b.ld, col[v]), live && has_b ? n[v] : 0);
    }
  };
  // Float32 branches, LayerNorm that saves, and rows off the 16-byte boundaries
  // (whose vectors take twice the registers on their way) have none for the next
  // row: with it, 65536 x 768 saved took 281 instead of 240 us, and LayerNorm
  // 16384 x 4096 in float32 took 279 instead of 238 us.
  constexpr bool kAhead = kVec && BT != RF_F32 && !(kLayer && kSave);
  if (kAhead) fetch();
  while (next < rows) {
    const int row = int(next);
    if (!kAhead) fetch();
    Raw8<XT> rx[V];
    Raw8<BT> rb[V];
    float x[V][8], b[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rx[v] = nx[v].get(A.x);
      rb[v] = nb[v].get(A.b);
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
        store_part<XT, kVec>(A.x_out, at(row, A.x_out.ld, col[v]), n[v], rx[v]);
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
      store_part<BT, kVec>(A.y, at(row, A.y.ld, col[v]), n[v], raw);
      if (kSave && A.sy.codes) {
        unpack<BT>(raw, x[v]);
        save_raw<BT>(A.sy, c, step0[v], row, col[v], raw, x[v]);
      }
    }
  }
}

}  // namespace

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

}  // namespace bn
}  // namespace rf
