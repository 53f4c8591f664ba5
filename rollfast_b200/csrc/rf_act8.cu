// Activations saved in 8 bits (rf_act8.cuh has the form): save, load, and a
// SwiGLU whose two inputs are saved in the forward pass and read in the
// backward pass.
//
// All four kernels are bound by HBM: one pass, each element read and written
// once.  A thread takes 8 consecutive features (16 bytes of a 16-bit type, 8
// codes), so the 4 lanes that share a block find its largest magnitude with
// two shuffles, and kRows rows, so that its loads are in flight together.
#include "rf_act8.cuh"

#include "rf_kernels.cuh"

namespace rf {

rf_status check_saved(const rf_saved_activation* s, const char* what) {
  const std::string w(what);
  if (!s) return fail(RF_EINVAL, w + ": null saved activation");
  if (s->format != RF_INT8 && s->format != RF_E4M3) return fail(RF_EINVAL, w + ": format must be RF_INT8 or RF_E4M3");
  if (s->rows < 0 || s->features <= 0) return fail(RF_EINVAL, w + ": rows must be >= 0 and features > 0");
  if (s->rows > 0x7FFFFFFF || s->features > kMaxFeatures)
    return fail(RF_EINVAL, w + ": at most 2^31 - 1 rows and 2^26 features");
  if (s->ld != round_up(s->features, 16) || s->scale_rows != round_up(s->rows, 64))
    return fail(RF_EINVAL, w + ": codes are [rows][features rounded up to 16], steps [panels][rows rounded up to 64][4]");
  if (s->rows > 0) {
    if (!s->codes || !s->scales) return fail(RF_EINVAL, w + ": null codes or steps");
    if ((reinterpret_cast<uintptr_t>(s->codes) | reinterpret_cast<uintptr_t>(s->scales)) & 15)
      return fail(RF_EINVAL, w + ": codes and steps must be 16-byte aligned");
  }
  return RF_OK;
}

namespace {

constexpr int kThreads = 256;

// Block shape and grid of a kernel over rows x 8-feature vectors: threads
// along x cover a row (whole panels of 16 vectors), rows along y.
struct Tiling {
  dim3 block, grid;
};
Tiling tiling(int64_t rows, int64_t features, int rows_per_thread) {
  const int64_t nv = ceil_div(features, kPanel8) * (kPanel8 / 8);
  // A multiple of 16 threads holds whole panels; whole warps for the shuffles.
  const int tx = int(nv >= kThreads ? kThreads : nv == 16 ? 16 : round_up(nv, 32));
  const int ty = kThreads / tx;
  const int64_t gy = ceil_div(rows, int64_t(ty) * rows_per_thread);
  Tiling t;
  t.block = dim3(unsigned(tx), unsigned(ty));
  // Row tiles along x (up to 2^31 - 1 of them), columns along y.
  t.grid = dim3(unsigned(gy), unsigned(ceil_div(nv, tx)));
  return t;
}

// The 16-bit noise of 8 consecutive elements from element i of a SplitMix64
// stream: output c serves elements 4c .. 4c+3 (rf_common.cuh).
__device__ __forceinline__ void noise8(uint64_t seed, uint64_t i, float (&u)[8]) {
  const uint64_t c = i >> 2;
  uint64_t a = splitmix64_at(seed, c), b = splitmix64_at(seed, c + 1);
  const int sh = int(i & 3) * 16;
  if (sh) {  // rows whose length is no multiple of 4 start inside an output
    const uint64_t d = splitmix64_at(seed, c + 2);
    a = (a >> sh) | (b << (64 - sh));
    b = (b >> sh) | (d << (64 - sh));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    u[k] = float(uint32_t(a >> (16 * k)) & 0xFFFFu) * (1.f / 65536.f);
    u[4 + k] = float(uint32_t(b >> (16 * k)) & 0xFFFFu) * (1.f / 65536.f);
  }
}

// Stochastic rounding: with u uniform on [0, 1), the grid point below plus
// one step when the fraction and u pass 1, so the mean is the value.  int8
// takes floor(v + u); e4m3 does it on the magnitude, in steps of
// 2^(exponent - 3) (2^-9 below 2^-6).  No result leaves the range: |v| is at
// most 127 (448 = 14 steps), and floor(127 + u) = 127.
__device__ __forceinline__ uint2 encode8_stochastic(const float (&f)[8], const float (&u)[8], uint32_t s, int format) {
  if (s == kNanStep) return make_uint2(0u, 0u);
  const float inv = __uint_as_float((254u - s) << 23);
  float g[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float v = f[k] * inv;
    if (format == RF_INT8) {
      g[k] = floorf(v + u[k]);
    } else {
      const float m = fminf(fabsf(v), 448.f);
      const uint32_t e = max(int(__float_as_uint(m) >> 23) - 3, 127 - 9);
      const float step = __uint_as_float(e << 23), rstep = __uint_as_float((254u - e) << 23);
      g[k] = copysignf(floorf(m * rstep + u[k]) * step, v);
    }
  }
  return encode8(g, 127u, format);  // step 1: the values are on the grid
}

template <int kRows, bool kStochastic>
__global__ void __launch_bounds__(kThreads) k_save(RowView x, Saved8 out, int64_t rows, int64_t features,
                                                   uint64_t seed) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  float f[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    load8(x, row, col, row < rows ? features : 0, f[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const uint32_t s = step_byte(block_max_bits(f[r]), out.format);
    if (!in || row >= rows) continue;
    uint2 c;
    if (kStochastic) {
      float u[8];
      noise8(seed, uint64_t(row) * uint64_t(features) + uint64_t(col), u);
      c = encode8_stochastic(f[r], u, s, out.format);
    } else {
      c = encode8(f[r], s, out.format);
    }
    store_saved(out, row, col, c, s);
  }
}

template <int kRows>
__global__ void __launch_bounds__(kThreads) k_load(Saved8 in, RowOut out, int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  if (col >= features) return;
  float f[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    if (row < rows) load8(in, row, col, f[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    if (row >= rows) continue;
    saturate8(out.dt, f[r]);
    store8(out, row, col, features, f[r]);
  }
}

// sigma(g) from one exponential that cannot overflow, so that very negative
// g fade out through the subnormals.
__device__ __forceinline__ float sigmoid(float g) {
  const float e = __expf(-fabsf(g));
  return (g < 0.f ? e : 1.f) / (1.f + e);
}

template <int kRows, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_fwd(RowView gate, RowView up, RowOut h, Saved8 sg, Saved8 su,
                                                         int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  float g[kRows][8], u[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const int64_t n = row < rows ? features : 0;
    load8(gate, row, col, n, g[r]);
    load8(up, row, col, n, u[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const bool live = in && row < rows;
    if (kSave) {
      const uint32_t a = step_byte(block_max_bits(g[r]), sg.format);
      const uint32_t b = step_byte(block_max_bits(u[r]), su.format);
      if (live) {
        store_saved(sg, row, col, encode8(g[r], a, sg.format), a);
        store_saved(su, row, col, encode8(u[r], b, su.format), b);
      }
    }
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < 8; ++k) g[r][k] = g[r][k] * sigmoid(g[r][k]) * u[r][k];
    store8(h, row, col, features, g[r]);
  }
}

template <int kRows, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_bwd(RowView dh, Saved8 gate, Saved8 up, RowOut dgate, RowOut dup,
                                                         Saved8 sh, int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  float d[kRows][8], g[kRows][8], u[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const bool live = in && row < rows;
    load8(dh, row, col, live ? features : 0, d[r]);
    load8(gate, live ? row : 0, live ? col : gate.ld, g[r]);
    load8(up, live ? row : 0, live ? col : up.ld, u[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const bool live = in && row < rows;
    float h[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // h = silu(g) u; dh/du = silu(g); dh/dg = u s (1 + g (1 - s)).
      const float s = sigmoid(g[r][k]);
      const float a = g[r][k] * s;
      h[k] = a * u[r][k];
      const float slope = s + a * (1.f - s);
      g[r][k] = d[r][k] * u[r][k] * slope;
      u[r][k] = d[r][k] * a;
    }
    if (kSave) {
      const uint32_t b = step_byte(block_max_bits(h), sh.format);
      if (live) store_saved(sh, row, col, encode8(h, b, sh.format), b);
    }
    if (!live) continue;
    store8(dgate, row, col, features, g[r]);
    store8(dup, row, col, features, u[r]);
  }
}

rf_status check_rows(const void* p, int64_t ld, int32_t dt, int64_t rows, int64_t features, const char* what) {
  const std::string w(what);
  if (!valid_dtype(dt)) return fail(RF_EINVAL, w + ": dtype must be RF_F32, RF_BF16 or RF_F16");
  if (ld < features) return fail(RF_EINVAL, w + ": row stride below the number of features");
  if (rows > 0 && !p) return fail(RF_EINVAL, w + ": null pointer");
  if (reinterpret_cast<uintptr_t>(p) % dtype_size(dt)) return fail(RF_EINVAL, w + ": misaligned pointer");
  return RF_OK;
}

bool same_shape(const rf_saved_activation& a, const rf_saved_activation& b) {
  return a.rows == b.rows && a.features == b.features;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" rf_status rf_save_activation(const void* x, int64_t ldx, int32_t dtype, const rf_saved_activation* out,
                                        int32_t stochastic, uint64_t seed, void* stream) {
  RF_TRY(check_saved(out, "rf_save_activation"));
  RF_TRY(check_rows(x, ldx, dtype, out->rows, out->features, "rf_save_activation: x"));
  if (out->rows == 0) return RF_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Tiling t = tiling(out->rows, out->features, 4);
  if (stochastic)
    k_save<4, true><<<t.grid, t.block, 0, st>>>(row_view(x, ldx, dtype), saved8(*out), out->rows, out->features, seed);
  else
    k_save<4, false><<<t.grid, t.block, 0, st>>>(row_view(x, ldx, dtype), saved8(*out), out->rows, out->features, 0);
  return check_launch("k_save");
}

extern "C" rf_status rf_load_activation(const rf_saved_activation* saved, void* out, int64_t ldo, int32_t dtype,
                                        void* stream) {
  RF_TRY(check_saved(saved, "rf_load_activation"));
  RF_TRY(check_rows(out, ldo, dtype, saved->rows, saved->features, "rf_load_activation: out"));
  if (saved->rows == 0) return RF_OK;
  const Tiling t = tiling(saved->rows, saved->features, 4);
  k_load<4><<<t.grid, t.block, 0, static_cast<cudaStream_t>(stream)>>>(saved8(*saved), row_out(out, ldo, dtype),
                                                                       saved->rows, saved->features);
  return check_launch("k_load");
}

extern "C" rf_status rf_swiglu_forward(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, void* h,
                                       int64_t ld_h, int32_t dtype, int64_t rows, int64_t features,
                                       const rf_saved_activation* saved_gate, const rf_saved_activation* saved_up,
                                       void* stream) {
  if (rows < 0 || features <= 0 || rows > 0x7FFFFFFF || features > kMaxFeatures)
    return fail(RF_EINVAL, "rf_swiglu_forward: rows in [0, 2^31) and features in [1, 2^26]");
  RF_TRY(check_rows(gate, ld_gate, dtype, rows, features, "rf_swiglu_forward: gate"));
  RF_TRY(check_rows(up, ld_up, dtype, rows, features, "rf_swiglu_forward: up"));
  RF_TRY(check_rows(h, ld_h, dtype, rows, features, "rf_swiglu_forward: h"));
  if (!saved_gate != !saved_up) return fail(RF_EINVAL, "rf_swiglu_forward: save both inputs or neither");
  Saved8 sg{}, su{};
  if (saved_gate) {
    RF_TRY(check_saved(saved_gate, "rf_swiglu_forward: saved_gate"));
    RF_TRY(check_saved(saved_up, "rf_swiglu_forward: saved_up"));
    if (!same_shape(*saved_gate, *saved_up) || saved_gate->rows != rows || saved_gate->features != features)
      return fail(RF_EINVAL, "rf_swiglu_forward: the saved activations have another shape");
    sg = saved8(*saved_gate);
    su = saved8(*saved_up);
  }
  if (rows == 0) return RF_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Tiling t = tiling(rows, features, 2);
  const RowView g = row_view(gate, ld_gate, dtype), u = row_view(up, ld_up, dtype);
  const RowOut o = row_out(h, ld_h, dtype);
  if (saved_gate) k_swiglu_fwd<2, true><<<t.grid, t.block, 0, st>>>(g, u, o, sg, su, rows, features);
  else k_swiglu_fwd<2, false><<<t.grid, t.block, 0, st>>>(g, u, o, sg, su, rows, features);
  return check_launch("k_swiglu_fwd");
}

extern "C" rf_status rf_swiglu_backward(const void* grad_h, int64_t ld_grad, const rf_saved_activation* saved_gate,
                                        const rf_saved_activation* saved_up, void* grad_gate, int64_t ld_gate,
                                        void* grad_up, int64_t ld_up, int32_t dtype,
                                        const rf_saved_activation* saved_h, void* stream) {
  RF_TRY(check_saved(saved_gate, "rf_swiglu_backward: saved_gate"));
  RF_TRY(check_saved(saved_up, "rf_swiglu_backward: saved_up"));
  if (!same_shape(*saved_gate, *saved_up))
    return fail(RF_EINVAL, "rf_swiglu_backward: the saved activations differ in shape");
  const int64_t rows = saved_gate->rows, features = saved_gate->features;
  RF_TRY(check_rows(grad_h, ld_grad, dtype, rows, features, "rf_swiglu_backward: grad_h"));
  RF_TRY(check_rows(grad_gate, ld_gate, dtype, rows, features, "rf_swiglu_backward: grad_gate"));
  RF_TRY(check_rows(grad_up, ld_up, dtype, rows, features, "rf_swiglu_backward: grad_up"));
  Saved8 sh{};
  if (saved_h) {
    RF_TRY(check_saved(saved_h, "rf_swiglu_backward: saved_h"));
    if (!same_shape(*saved_gate, *saved_h))
      return fail(RF_EINVAL, "rf_swiglu_backward: saved_h has another shape");
    sh = saved8(*saved_h);
  }
  if (rows == 0) return RF_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Tiling t = tiling(rows, features, 2);
  const RowView d = row_view(grad_h, ld_grad, dtype);
  const RowOut dg = row_out(grad_gate, ld_gate, dtype), du = row_out(grad_up, ld_up, dtype);
  if (saved_h)
    k_swiglu_bwd<2, true><<<t.grid, t.block, 0, st>>>(d, saved8(*saved_gate), saved8(*saved_up), dg, du, sh, rows,
                                                      features);
  else
    k_swiglu_bwd<2, false><<<t.grid, t.block, 0, st>>>(d, saved8(*saved_gate), saved8(*saved_up), dg, du, sh, rows,
                                                       features);
  return check_launch("k_swiglu_bwd");
}
