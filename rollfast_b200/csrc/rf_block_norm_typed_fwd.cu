// Forward pass of the typed block norms (rf_block_norm_typed.cuh).
#include "rf_block_norm_typed.cuh"

namespace rf {
namespace bn {

namespace {

constexpr int kMaxFactorBytes = 4 * int(kMaxTyped) * 4;

// Threads of a CTA, one to an SM.  Whole vectors of 16 bits: 512, whose 128
// registers each hold the next row's loads too.  Others: 768 without the next
// row, since float32 takes twice the registers on its way, and so do rows off
// the 16-byte boundaries (512 and the next row took 197 instead of 180 us for
// 16384 x 4096 float32, 278 instead of 225 with copies; 444 instead of 290
// for 16384 x 4097 bfloat16; bfloat16 LayerNorm with copies, the other way
// round, 264 instead of 209 with 768).
__host__ __device__ constexpr int fwd_threads(int bt, bool vec) {
  return vec && bt != RF_F32 ? kTypedThreads : kFwdThreads;
}

template <int XT, int BT, bool kLayer, bool kSave, bool kVec>
__global__ void __launch_bounds__(fwd_threads(BT, kVec), 1)
    k_norm_fwd_typed(const __grid_constant__ FwdArgs A, int team_threads) {
  constexpr int V = kFwdVectors;
  __shared__ TeamSums sums;
  int turn = 0;
  const Common& c = A.c;
  const TeamCtx t = team_ctx(team_threads, sums);
  const int teams = int(blockDim.x) / team_threads;
  const int64_t step = int64_t(gridDim.x) * teams;
  const bool has_b = A.b.p != nullptr, has_y = A.y.p != nullptr, fixed = gate_is_fixed(c);
  // x' = x + normalised * mul + add;  y = normalised * pw + pb.  The columns'
  // factors lie in shared memory, one copy for the CTA's teams: in registers
  // they left none for the next row or more warps (65536 x 768 bfloat16
  // LayerNorm 131 us, now 115; with copies 240, now 193).
  extern __shared__ float4 factors[];  // [mul, pw, add, pb][vector][half][thread of a team]
  int col[V], n[V];
  int64_t step0[V];
  own_columns<V>(t, c, col, n);
  auto slot = [&](int which, int v, int half) -> float4& {
    return factors[((which * V + v) * 2 + half) * team_threads + t.lane];
  };
  auto put = [&](int which, int v, const float (&f)[8]) {
    slot(which, v, 0) = make_float4(f[0], f[1], f[2], f[3]);
    slot(which, v, 1) = make_float4(f[4], f[5], f[6], f[7]);
  };
  auto get = [&](int which, int v, float (&f)[8]) {
    const float4 p = slot(which, v, 0), q = slot(which, v, 1);
    f[0] = p.x, f[1] = p.y, f[2] = p.z, f[3] = p.w, f[4] = q.x, f[5] = q.y, f[6] = q.z, f[7] = q.w;
  };
#pragma unroll
  for (int v = 0; v < V; ++v) step0[v] = kSave ? first_step(c, col[v]) : 0;
  if (t.id == 0) {
#pragma unroll 1
    for (int v = 0; v < V; ++v) {
      float w[8], g[8];
      const int cv = (v * t.threads + t.lane) * 8, nv = int(c.d) - cv;
      param8(c.pre_w, cv, c.d, 1.f, w);
      put(1, v, w);
      scale8(c, cv, w);
      if (fixed) {
        gate8(c, 0, cv, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] *= g[k];
      }
      param8(c.post_w, cv, c.d, 1.f, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = k < nv ? g[k] * w[k] : 0.f;
      put(0, v, g);
      if (kLayer) {
        param8(c.post_b, cv, c.d, 0.f, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = k < nv ? g[k] * w[k] : 0.f;
        put(2, v, g);
        param8(c.pre_b, cv, c.d, 0.f, g);
        put(3, v, g);
      }
    }
  }
  if (kSave) {
    steps_behind(A.sx, c);
    steps_behind(A.sb, c);
    steps_behind(A.sy, c);
  }
  __syncthreads();
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
  constexpr bool kAhead = fwd_threads(BT, kVec) == kTypedThreads;
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
        float mul[8], add[8];
        get(0, v, mul);
        if (kLayer) get(2, v, add);
        if (fixed) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = kLayer ? __fadd2_rn(pair(x[v], k), pair(add, k)) : pair(x[v], k);
            put_pair(x[v], k, __ffma2_rn(pair(b[v], k), pair(mul, k), y));
          }
        } else {
          float g[8];
          gate8(c, row, col[v], g);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = kLayer ? __ffma2_rn(pair(b[v], k), pair(mul, k), pair(add, k))
                                    : __fmul2_rn(pair(b[v], k), pair(mul, k));
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
      float pw[8], pb[8];
      get(1, v, pw);
      if (kLayer) get(3, v, pb);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        put_pair(x[v], k, kLayer ? __ffma2_rn(pair(x[v], k), pair(pw, k), pair(pb, k))
                                 : __fmul2_rn(pair(x[v], k), pair(pw, k)));
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
  const TypedTeam t = team_for(p.features, kFwdVectors, fwd_threads(bt, vec));
  const size_t smem = size_t(layer ? 4 : 2) * kFwdVectors * 8 * t.threads * sizeof(float);
  const unsigned g = unsigned(std::min(ceil_div(p.rows, t.teams), int64_t(num_sms()))), b = unsigned(t.threads * t.teams);
  return with_types(xt, bt, vec, [&](auto x, auto y, auto w) {
    constexpr int X = decltype(x)::value, B = decltype(y)::value;
    constexpr bool W = decltype(w)::value;
    auto go = [&](auto kernel) {
      // Beside the sums, above what a launch may take without asking.
      if (smem > 32768) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxFactorBytes);
      kernel<<<g, b, smem, st>>>(A, t.threads);
    };
    if (layer) save ? go(k_norm_fwd_typed<X, B, true, true, W>) : go(k_norm_fwd_typed<X, B, true, false, W>);
    else save ? go(k_norm_fwd_typed<X, B, false, true, W>) : go(k_norm_fwd_typed<X, B, false, false, W>);
  });
}

}  // namespace bn
}  // namespace rf
