// Launch descriptors and device helpers shared by the block-norm kernels.
#pragma once

#include <algorithm>

#include "rf_act8.cuh"
#include "rf_kernels.cuh"

namespace rf {
namespace bn {

constexpr int64_t kMaxNorm = 16384;
constexpr int kWarpsPerCta = 4;  // warp-per-row CTAs

struct Param {
  const void* p;
  int32_t dt;
};
struct Common {
  int64_t rows, d;
  int64_t gate_rows;
  Param pre_w, pre_b, post_w, post_b, scale, gate;
  float eps, scale_value, inv_d;
  int32_t post_norm, scale_per_channel, gate_per_channel, gate_act;
};

struct FwdArgs {
  Common c;
  RowView x, b;
  RowOut x_out, y;
  Saved8 sx, sb, sy;  // codes null: not saved
};

struct BwdArgs {
  Common c;
  RowView gx, gy;      // gradients of x' and y; p null: absent
  RowView x, b;
  Saved8 sx, sb;       // codes set: read instead of x, b
  RowOut dx, db;
  void* dgate;         // gate varying by row: written here
  int32_t row_gate;    // gate varies by row
  float* partial;      // [items][sums][ldp]
  int64_t ldp;
  int32_t sums;        // rows of sums per item: 2, or 4 with biases
  int64_t items, chunks, rows_per_chunk, group_rows;
};

// A parameter's 8 values at a column, `absent` where there is none.
__device__ __forceinline__ void param8(const Param& w, int64_t col, int64_t d, float absent, float (&f)[8]) {
  if (!w.p) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = absent;
    return;
  }
  load8_param(w.p, w.dt, col, d, f);
}
__device__ __forceinline__ float gate_value(float g, int act) {
  return act == RF_GATE_SIGMOID ? 1.f / (1.f + expf(-g)) : act == RF_GATE_TANH ? tanhf(g) : g;
}
// Derivative from the value.
__device__ __forceinline__ float gate_slope(float a, int act) {
  return act == RF_GATE_SIGMOID ? a * (1.f - a) : act == RF_GATE_TANH ? 1.f - a * a : 1.f;
}
// a(gamma) at 8 columns of a row, 1 without a gate.
__device__ __forceinline__ void gate8(const Common& c, int64_t row, int64_t col, float (&f)[8]) {
  if (!c.gate.p) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 1.f;
    return;
  }
  const int64_t g = row / c.gate_rows;
  if (c.gate_per_channel) {
    const int es = c.gate.dt == RF_F32 ? 4 : 2;
    load8_param(static_cast<const uint8_t*>(c.gate.p) + g * c.d * es, c.gate.dt, col, c.d, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = gate_value(f[k], c.gate_act);
  } else {
    const float a = gate_value(ld_as_float(c.gate.p, c.gate.dt, g), c.gate_act);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = a;
  }
}
__device__ __forceinline__ void scale8(const Common& c, int64_t col, float (&f)[8]) {
  if (c.scale.p && c.scale_per_channel) {
    param8(c.scale, col, c.d, 1.f, f);
    return;
  }
  const float s = c.scale.p ? ld_as_float(c.scale.p, c.scale.dt, 0) : c.scale_value;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = s;
}

// The typed kernels (rf_block_norm_typed.cuh): arrays of one of four pairs of
// element types.  Each returns true when it took the call.
struct TypedTeam {
  int threads, vectors, teams;  // threads of a row's team, 8-feature vectors per thread, teams per CTA
};
TypedTeam typed_team(int64_t d);
bool try_typed_fwd(const rf_block_norm& p, const FwdArgs& A, cudaStream_t st);
bool try_typed_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st);
bool try_typed_layer_bwd(const rf_block_norm& p, const BwdArgs& A, bool bias, cudaStream_t st);  // LayerNorm only

}  // namespace bn
}  // namespace rf
