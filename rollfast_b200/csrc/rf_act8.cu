// Activations saved in 8 bits (rf_act8.cuh has the form): save, load, and a
// SwiGLU whose two inputs are saved in the forward pass and read in the
// backward pass.
//
// All are bound by HBM: one pass, each element read and written once.  A
// thread takes 8 consecutive features (16 bytes of a 16-bit type, 8 codes), so
// the 4 lanes that share a block find its largest magnitude with two
// shuffles.  Rows on 16-byte boundaries go through kernels typed by element
// and format, whose CTAs stay and walk down the rows with the next tile's
// loads in flight; others (odd widths, shifted views) through one of the
// simple kernels below them.
// Measured on a B200, bfloat16, int8 (a copy: 6549 GB/s): 16384 x 14336 saved
// in 115 us (6.2 TB/s), loaded in 117, saved stochastically in 219 in either
// format (28 instructions an element, most of them the generator's; issue
// slots are busy 71 % of the time, with 14 warps an SM at 106 registers, so
// latency takes the rest; e4m3 took 238 while values below its normal range
// were looked for element by element after the scaling, not two at a time
// before it); SwiGLU 8192 x 14336 forward 164 us (5.8 TB/s), backward 170, with
// h saved 190; float32 310, 313 and 342.
// 16384 x 4097, off the boundaries: saved in 76 us (4096: 39), loaded in 92
// (39), SwiGLU forward 206 (94), backward 239 (100); there a vector takes two
// or three loads and 13 to 17 selects, and the kernels hold 16 to 24 warps an SM.
#include "rf_act8.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

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

// Threads along a row of nv vectors: a multiple of 16 holds whole panels; whole
// warps for the shuffles.  Wide rows are cut into equal column tiles, so that
// few threads of the last one idle (4097 columns: 3 x 192 threads for 528
// vectors, not 3 x 256: SwiGLU forward 16384 x 4097 in 211 us, not 262).
int row_threads(int64_t nv) {
  return int(nv == 16 ? 16 : round_up(ceil_div(nv, ceil_div(nv, int64_t(kThreads))), 32));
}

// Whole tiles of a typed kernel: CTAs of tx x ty threads over 8-feature
// vectors x rows, rows_per_thread rows per thread and tile; grid.y column tiles, and
// along x as many CTAs as the GPU holds, each walking down the rows.
struct Walk {
  dim3 block, grid;
};
template <auto kernel>
Walk walk(int64_t rows, int64_t features, int rows_per_thread, int elements = 8) {
  const int64_t nv = ceil_div(features, kPanel8) * (kPanel8 / elements);
  const int tx = row_threads(nv), ty = kThreads / tx;
  const int64_t gy = ceil_div(nv, tx), tiles = ceil_div(rows, int64_t(ty) * rows_per_thread);
  // Asked once per kernel (and block size: whole warps up to 256 threads): the
  // answer is the same on every GPU of the kind, and asking takes microseconds.
  static std::atomic<int> asked[kThreads / 32 + 1];
  std::atomic<int>& known = asked[tx * ty / 32];
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, tx * ty, 0) != cudaSuccess || per_sm < 1) {
      cudaGetLastError();
      per_sm = 2;
    }
    known.store(per_sm, std::memory_order_relaxed);
  }
  // Three CTAs per SM: 16384 x 14336 saved in 117 us; with two or four 131.
  const int64_t held = std::max<int64_t>(1, int64_t(num_sms()) * std::min(per_sm, 3) / gy);
  Walk w;
  w.block = dim3(unsigned(tx), unsigned(ty));
  w.grid = dim3(unsigned(std::min(tiles, held)), unsigned(gy));
  return w;
}

// Block shape and grid of a simple kernel over rows x 8-feature vectors: threads
// along x cover a row (whole panels of 16 vectors), rows along y.
struct Tiling {
  dim3 block, grid;
};
Tiling tiling(int64_t rows, int64_t features, int rows_per_thread) {
  const int64_t nv = ceil_div(features, kPanel8) * (kPanel8 / 8);
  const int tx = row_threads(nv), ty = kThreads / tx;
  const int64_t gy = ceil_div(rows, int64_t(ty) * rows_per_thread);
  Tiling t;
  t.block = dim3(unsigned(tx), unsigned(ty));
  // Row tiles along x (up to 2^31 - 1 of them), columns along y.
  t.grid = dim3(unsigned(gy), unsigned(ceil_div(nv, tx)));
  return t;
}

// The 16-bit noise of 8 consecutive elements from element i of a SplitMix64
// stream, as two words, the first element lowest: output c serves elements
// 4c .. 4c+3 (rf_common.cuh).
__device__ __forceinline__ void noise8(uint64_t seed, uint64_t i, uint64_t& a, uint64_t& b) {
  const uint64_t c = i >> 2;
  a = splitmix64_at(seed, c);
  b = splitmix64_at(seed, c + 1);
  const int sh = int(i & 3) * 16;
  if (sh) {  // rows whose length is no multiple of 4 start inside an output
    const uint64_t d = splitmix64_at(seed, c + 2);
    a = (a >> sh) | (b << (64 - sh));
    b = (b >> sh) | (d << (64 - sh));
  }
}
__device__ __forceinline__ uint32_t noise_word(uint64_t a, uint64_t b, int k) {  // the two elements 2k, 2k + 1
  return k == 0 ? uint32_t(a) : k == 1 ? uint32_t(a >> 32) : k == 2 ? uint32_t(b) : uint32_t(b >> 32);
}

// Stochastic rounding: with u = noise / 2^16, uniform on [0, 1), the grid point
// below plus one step when the fraction and u pass 1, so the mean is the value.
// No result leaves the range below the largest step: |v| is at most 127 (448
// = 14 steps of 32), and floor(127 + u) = 127.
// int8: floor(v + u), the sum rounded to float32; adding 1.5 * 2^23 towards
// minus infinity takes the floor and leaves it in the low byte.
__device__ __forceinline__ uint2 encode8_stochastic_int8(const float (&f)[8], uint64_t na, uint64_t nb, uint32_t s) {
  const float inv = __uint_as_float((254u - s) << 23);
  uint32_t b[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t w = noise_word(na, nb, k >> 1);
    // u + 1 has the noise in the top 16 bits of its significand.
    const float u = __uint_as_float(0x3F800000u | ((k & 1) ? (w >> 16) << 7 : (w << 7) & 0x7FFF80u)) - 1.f;
    b[k] = __float_as_uint(__fadd_rd(fmaf(f[k], inv, u), 12582912.f));  // f * inv is exact
  }
  if (s == 248u) {  // the largest step: larger magnitudes saturate
#pragma unroll
    for (int k = 0; k < 8; ++k) b[k] = __float_as_uint(fminf(fmaxf(__uint_as_float(b[k]), 12582785.f), 12583039.f));
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = __byte_perm(__byte_perm(b[4 * h], b[4 * h + 1], 0x0040), __byte_perm(b[4 * h + 2], b[4 * h + 3], 0x0040),
                       0x5410);
  return make_uint2(w[0], w[1]);
}
// e4m3, on the magnitude in steps of 2^(exponent - 3), 2^-9 below 2^-6.  From
// 2^-6 up the noise goes in below the 3 significand bits that stay, and the
// rest is cut off: the same, since magnitude / step + u has at most 24
// significant bits below 16, and above 16 only its floor counts.
// `low`: some magnitude may lie below 2^-6 (and above 0).
__device__ __forceinline__ uint2 encode8_stochastic_e4m3(const float (&f)[8], uint64_t na, uint64_t nb, uint32_t s,
                                                         bool low) {
  const float inv = __uint_as_float((254u - s) << 23);
  float g[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t w = noise_word(na, nb, k);
    const float2 v = __fmul2_rn(pair(f, k), both(inv));
    // The halves by byte permutation, so that shift and addition are one instruction.
    g[2 * k] = __uint_as_float((__float_as_uint(v.x) + (__byte_perm(w, 0u, 0x4410) << 4)) & 0xFFF00000u);
    g[2 * k + 1] = __uint_as_float((__float_as_uint(v.y) + (__byte_perm(w, 0u, 0x4432) << 4)) & 0xFFF00000u);
  }
  if (low) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float v = f[k] * inv, m = fabsf(v);
      const uint32_t w = noise_word(na, nb, k >> 1);
      const float u = float((k & 1) ? w >> 16 : w & 0xFFFFu) * (1.f / 65536.f);
      if (m < 0.015625f) g[k] = copysignf(floorf(__fadd_rn(m * 512.f, u)) * (1.f / 512.f), v);
    }
  }
  return encode8(g, 127u, RF_E4M3);  // step 1: the values are on the grid, or above 448 and saturate
}
// Whether a vector holds a magnitude in (0, 2^-6) steps, for the e4m3 code.
__device__ __forceinline__ bool any_low(const float (&f)[8], uint32_t s) {
  uint32_t least = 0xFFFFFFFFu;
#pragma unroll
  for (int k = 0; k < 8; ++k) least = min(least, (__float_as_uint(f[k]) & 0x7FFFFFFFu) - 1u);  // 0 wraps around
  return s <= 6u || least < ((s - 6u) << 23) - 1u;
}
// The same of bfloat16 as it lies in memory, two at a time.  Where the low
// half is 0, the subtraction takes one more from the high half: a magnitude of
// 2^-133 may go unseen, which every draw rounds to 0 from steps of 2^-107 up
// (smaller steps count as low), and one more may be seen, which only takes the
// longer path.
template <int DT>
__device__ __forceinline__ bool any_low(const Raw8<DT>& r, const float (&f)[8], uint32_t s) {
  if (DT != RF_BF16) return any_low(f, s);
  const uint32_t a = __vminu2((r.u[0].x & 0x7FFF7FFFu) - 0x00010001u, (r.u[0].y & 0x7FFF7FFFu) - 0x00010001u);
  const uint32_t b = __vminu2((r.u[0].z & 0x7FFF7FFFu) - 0x00010001u, (r.u[0].w & 0x7FFF7FFFu) - 0x00010001u);
  const uint32_t m = __vminu2(a, b);
  return s <= 20u || min(m & 0xFFFFu, m >> 16) < ((s - 6u) << 7) - 1u;
}
__device__ __forceinline__ uint2 encode8_stochastic(const float (&f)[8], uint64_t a, uint64_t b, uint32_t s,
                                                    int format, bool low) {
  if (s == kNanStep) return make_uint2(0u, 0u);
  return format == RF_INT8 ? encode8_stochastic_int8(f, a, b, s) : encode8_stochastic_e4m3(f, a, b, s, low);
}

// One thread's column of an array, walked down by rows.  Addresses move by
// constant strides: as products of 64-bit row numbers they were a third of
// the save kernel's instructions.
template <int DT>
struct Column {
  const uint8_t* p;
  int64_t stride, turn;  // bytes from row to row, and from tile to tile
  __device__ __forceinline__ Column(const void* base, int64_t ld, int64_t row, int64_t col, int64_t step) {
    constexpr int es = DT == RF_F32 ? 4 : 2;
    p = static_cast<const uint8_t*>(base) + (row * ld + col) * es;
    stride = ld * es;
    turn = step * stride;
  }
  template <int R>
  __device__ __forceinline__ void fetch(Raw8<DT> (&to)[R], int n) const {  // the first n rows of the tile, others 0
#pragma unroll
    for (int r = 0; r < R; ++r) to[r] = r < n ? load_raw<DT>(p + r * stride, 0) : zero_raw<DT>();
  }
  __device__ __forceinline__ void store(int r, const float (&f)[8]) const {
    store_vec<DT>(const_cast<uint8_t*>(p) + r * stride, 0, f);
  }
};
struct SavedColumn {
  uint8_t *codes, *steps;
  int64_t stride, turn, steps_turn;
  bool has_codes, has_step;  // the last vectors of a row may lie behind the codes; one lane of four has the step
  __device__ __forceinline__ SavedColumn(const Saved8& s, int64_t row, int64_t col, int64_t step, bool in) {
    has_codes = in && col < s.ld;
    has_step = in && col % kBlock8 == 0;
    codes = s.codes + (has_codes ? row * s.ld + col : 0);
    steps = s.scales + (in ? scale_index(s, row, col) : 0);
    stride = s.ld;
    turn = step * s.ld;
    steps_turn = step * 4;
  }
  __device__ __forceinline__ void next() {
    codes += turn;
    steps += steps_turn;
  }
  __device__ __forceinline__ void store(int r, uint2 c, uint32_t s) const {
    if (has_codes) *reinterpret_cast<uint2*>(codes + r * stride) = c;
    if (has_step) steps[4 * r] = uint8_t(s);
  }
};
// Rows of a tile of R that start at `row`.
template <int R>
__device__ __forceinline__ int rows_here(int64_t row, int64_t rows) {
  return int(min(max(rows - row, int64_t(0)), int64_t(R)));
}

template <int DT, int kFormat, bool kStochastic>
__global__ void __launch_bounds__(kThreads) k_save_typed(const void* x, int64_t ldx, Saved8 out, int64_t rows,
                                                         int64_t features, uint64_t seed) {
  constexpr int R = DT == RF_F32 ? 2 : 4;
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const bool data = col + 8 <= features;  // widths here are multiples of 8
  const int64_t step = int64_t(gridDim.x) * blockDim.y * R;
  int64_t row = (int64_t(blockIdx.x) * blockDim.y + threadIdx.y) * R;
  // The noise generator's state moves by a constant from row to row (rows
  // start on a multiple of 8 elements), which leaves its two multiplications.
  const uint64_t row_state = uint64_t(features / 4) * kSplitmixGamma, turn_state = uint64_t(step) * row_state;
  uint64_t state = seed + (uint64_t(row) * uint64_t(features / 4) + uint64_t(col / 4) + 1) * kSplitmixGamma;
  Column<DT> in(x, ldx, row, col, step);
  SavedColumn to(out, row, col, step, col < round_up_dev(features, kPanel8));
  Raw8<DT> next[R];
  in.fetch(next, data ? rows_here<R>(row, rows) : 0);
  // All threads of the CTA take the same number of turns, for the shuffles.
  for (int64_t base = int64_t(blockIdx.x) * blockDim.y * R; base < rows; base += step) {
    const int n = rows_here<R>(row, rows);
    row += step;
    in.p += in.turn;
    Raw8<DT> cur[R];
#pragma unroll
    for (int r = 0; r < R; ++r) cur[r] = next[r];
    in.fetch(next, data ? rows_here<R>(row, rows) : 0);
    uint64_t z = state;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t s = step_byte(raw_max_bits<DT>(cur[r]), kFormat);
      float f[8];
      unpack<DT>(cur[r], f);
      uint2 c;
      if (kStochastic) {
        c = encode8_stochastic(f, splitmix64_mix(z), splitmix64_mix(z + kSplitmixGamma), s, kFormat,
                               kFormat == RF_E4M3 && any_low<DT>(cur[r], f, s));
        z += row_state;
      } else {
        c = encode8(f, s, kFormat);
      }
      if (r < n) to.store(r, c, s);
    }
    state += turn_state;
    to.next();
  }
}

// A thread writes 16 bytes of a row: 8 values of a 16-bit type, 4 of float32
// (with 8, in two stores 32 bytes apart, the half-filled sectors took 288
// instead of 209 us for 16384 x 14336).
template <int DT, int kFormat>
__global__ void __launch_bounds__(kThreads) k_load_typed(Saved8 in, void* out, int64_t ldo, int64_t rows,
                                                         int64_t features) {
  // The weight gradient's products may set up while this drains.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int R = 4, E = DT == RF_F32 ? 4 : 8;
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * E;
  if (col >= features) return;  // widths here are multiples of 8
  const int64_t step = int64_t(gridDim.x) * blockDim.y * R;
  int64_t row = (int64_t(blockIdx.x) * blockDim.y + threadIdx.y) * R;
  const uint8_t* codes = in.codes + row * in.ld + col;
  const uint8_t* steps = in.scales + scale_index(in, row, col);
  const int64_t stride = in.ld, turn = step * in.ld;
  Column<DT> to(out, ldo, row, col, step);
  uint2 c[R];
  uint32_t s[R];
  auto fetch = [&](int n) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      c[r] = make_uint2(0, 0);
      s[r] = 1u;
      if (r >= n) continue;
      if (E == 8) c[r] = __ldg(reinterpret_cast<const uint2*>(codes + r * stride));
      else c[r].x = __ldg(reinterpret_cast<const uint32_t*>(codes + r * stride));
      s[r] = __ldg(steps + 4 * r);
    }
  };
  fetch(rows_here<R>(row, rows));
  while (row < rows) {
    const int n = rows_here<R>(row, rows);
    uint2 w[R];
    float st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      w[r] = c[r];
      st[r] = step_value(s[r]);
    }
    row += step;
    codes += turn;
    steps += 4 * step;
    fetch(rows_here<R>(row, rows));
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= n) break;
      float f[8];
      decode4(w[r].x, kFormat, f);
      if (E == 8) decode4(w[r].y, kFormat, f + 4);
#pragma unroll
      for (int k = 0; k < E / 2; ++k) put_pair(f, k, __fmul2_rn(pair(f, k), both(st[r])));
      if (E == 8) {
        saturate8(DT, f);
        to.store(r, f);
      } else {
        *reinterpret_cast<float4*>(const_cast<uint8_t*>(to.p) + r * to.stride) = make_float4(f[0], f[1], f[2], f[3]);
      }
    }
    to.p += to.turn;
  }
}

// Neighbouring lanes that hold one row's vectors (tiling).
__device__ __forceinline__ int row_lanes() { return blockDim.x < 32 ? 16 : 32; }

template <int DT, int kRows, bool kStochastic>
__global__ void __launch_bounds__(kThreads) k_save(RowView x, Saved8 out, int64_t rows, int64_t features,
                                                   uint64_t seed) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  Span8<DT> span[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    span[r] = fetch_span<DT>(x, row * x.ld + col, row < rows ? features - col : 0);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const Raw8<DT> raw = align_span<DT>(span[r], x, row * x.ld + col, row < rows ? features - col : 0);
    float f[8];
    unpack<DT>(raw, f);
    const uint32_t s = step_byte(raw_max_bits<DT>(raw), out.format);
    if (!in || row >= rows) continue;
    uint2 c;
    if (kStochastic) {
      uint64_t na, nb;
      noise8(seed, uint64_t(row) * uint64_t(features) + uint64_t(col), na, nb);
      c = encode8_stochastic(f, na, nb, s, out.format, out.format == RF_E4M3 && any_low<DT>(raw, f, s));
    } else {
      c = encode8(f, s, out.format);
    }
    store_saved(out, row, col, c, s);
  }
}

template <int DT, int kRows>
__global__ void __launch_bounds__(kThreads) k_load(Saved8 in, RowOut out, int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  float f[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    load8(in, row < rows ? row : 0, row < rows ? col : in.ld, f[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    saturate8(DT, f[r]);
    store_span<DT>(out.p, row * out.ld + col, row < rows ? features - col : 0, pack<DT>(f[r]), row_lanes());
  }
}

// sigma(g) from one exponential that cannot overflow, so that very negative
// g fade out through the subnormals; 1 + e lies in [1, 2].
// Float32 arrays: expf and a rounded division, at most 4 units off throughout.
// 16-bit arrays: the fast exponential, off by up to 2 + 1.2 |g| units of
// float32, and the approximate reciprocal, off by one: at |g| = 80 that is
// 2^-16 of the value, where bfloat16 rounds by 2^-9 and float16 by 2^-12.
template <int DT>
__device__ __forceinline__ float sigmoid(float g) {
  if (DT == RF_F32) {
    const float e = expf(-fabsf(g));
    return (g < 0.f ? e : 1.f) / (1.f + e);
  }
  const float e = __expf(-fabsf(g));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return (g < 0.f ? e : 1.f) * r;
}

template <int DT, int kFormat, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_fwd_typed(const void* gate, int64_t ldg, const void* up,
                                                               int64_t ldu, void* h, int64_t ldh, Saved8 sg, Saved8 su,
                                                               int64_t rows, int64_t features) {
  constexpr int R = DT == RF_F32 ? 1 : 2;
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const bool data = col + 8 <= features;  // widths here are multiples of 8
  const bool in = kSave && col < round_up_dev(features, kPanel8);
  const int64_t step = int64_t(gridDim.x) * blockDim.y * R;
  int64_t row = (int64_t(blockIdx.x) * blockDim.y + threadIdx.y) * R;
  Column<DT> cg(gate, ldg, row, col, step), cu(up, ldu, row, col, step), ch(h, ldh, row, col, step);
  SavedColumn kg(sg, row, col, step, in), ku(su, row, col, step, in);
  Raw8<DT> ng[R], nu[R];
  int n = rows_here<R>(row, rows);
  cg.fetch(ng, data ? n : 0);
  cu.fetch(nu, data ? n : 0);
  for (int64_t base = int64_t(blockIdx.x) * blockDim.y * R; base < rows; base += step) {
    Raw8<DT> rg[R], ru[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rg[r] = ng[r];
      ru[r] = nu[r];
    }
    row += step;
    cg.p += cg.turn;
    cu.p += cu.turn;
    const int after = rows_here<R>(row, rows);
    cg.fetch(ng, data ? after : 0);
    cu.fetch(nu, data ? after : 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float g[8], u[8];
      unpack<DT>(rg[r], g);
      unpack<DT>(ru[r], u);
      if (kSave) {
        const uint32_t a = step_byte(raw_max_bits<DT>(rg[r]), kFormat);
        const uint32_t b = step_byte(raw_max_bits<DT>(ru[r]), kFormat);
        const uint2 x = encode8(g, a, kFormat), y = encode8(u, b, kFormat);
        if (r < n) {
          kg.store(r, x, a);
          ku.store(r, y, b);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        put_pair(g, k, __fmul2_rn(__fmul2_rn(pair(g, k), make_float2(sigmoid<DT>(g[2 * k]), sigmoid<DT>(g[2 * k + 1]))),
                                  pair(u, k)));
      if (data && r < n) ch.store(r, g);
    }
    n = after;
    ch.p += ch.turn;
    kg.next();
    ku.next();
  }
}

// h = silu(g) u; dh/du = silu(g); dh/dg = u s (1 + g (1 - s)).  g and u become
// the gradients.
template <int DT>
__device__ __forceinline__ void swiglu_back8(const float (&d)[8], float (&g)[8], float (&u)[8], float (&h)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 s = make_float2(sigmoid<DT>(g[2 * k]), sigmoid<DT>(g[2 * k + 1]));
    const float2 x = pair(u, k), y = pair(d, k);
    const float2 a = __fmul2_rn(pair(g, k), s);
    put_pair(h, k, __fmul2_rn(a, x));
    const float2 slope = __ffma2_rn(a, __ffma2_rn(s, both(-1.f), both(1.f)), s);
    put_pair(g, k, __fmul2_rn(__fmul2_rn(y, x), slope));
    put_pair(u, k, __fmul2_rn(y, a));
  }
}

template <int DT, int kFormat, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_bwd_typed(const void* dh, int64_t ldd, Saved8 gate, Saved8 up,
                                                               void* dgate, int64_t ldg, void* dup, int64_t ldu,
                                                               Saved8 sh, int64_t rows, int64_t features) {
  constexpr int R = 1;  // two rows a turn took 3 % longer
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const bool data = col + 8 <= features;  // widths here are multiples of 8
  const int64_t step = int64_t(gridDim.x) * blockDim.y * R;
  int64_t row = (int64_t(blockIdx.x) * blockDim.y + threadIdx.y) * R;
  Column<DT> cd(dh, ldd, row, col, step), cg(dgate, ldg, row, col, step), cu(dup, ldu, row, col, step);
  SavedColumn kg(gate, row, col, step, data), ku(up, row, col, step, data);
  SavedColumn kh(sh, row, col, step, kSave && col < round_up_dev(features, kPanel8));
  Raw8<DT> nd[R];
  uint2 wg[R], wu[R];
  uint32_t sg[R], su[R];
  auto fetch = [&](int n) {
    cd.fetch(nd, n);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      wg[r] = wu[r] = make_uint2(0, 0);
      sg[r] = su[r] = 1u;
      if (r >= n) continue;
      wg[r] = __ldg(reinterpret_cast<const uint2*>(kg.codes + r * kg.stride));
      wu[r] = __ldg(reinterpret_cast<const uint2*>(ku.codes + r * ku.stride));
      sg[r] = __ldg(kg.steps + 4 * r);
      su[r] = __ldg(ku.steps + 4 * r);
    }
  };
  int n = rows_here<R>(row, rows);
  fetch(data ? n : 0);
  for (int64_t base = int64_t(blockIdx.x) * blockDim.y * R; base < rows; base += step) {
    Raw8<DT> rd[R];
    uint2 rg[R], ru[R];
    float fg[R], fu[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rd[r] = nd[r];
      rg[r] = wg[r];
      ru[r] = wu[r];
      fg[r] = step_value(sg[r]);
      fu[r] = step_value(su[r]);
    }
    row += step;
    cd.p += cd.turn;
    kg.next();
    ku.next();
    const int after = rows_here<R>(row, rows);
    fetch(data ? after : 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float d[8], g[8], u[8], h[8];
      unpack<DT>(rd[r], d);
      decode4(rg[r].x, gate.format, g);
      decode4(rg[r].y, gate.format, g + 4);
      decode4(ru[r].x, up.format, u);
      decode4(ru[r].y, up.format, u + 4);
      mul8(g, both(fg[r]));
      mul8(u, both(fu[r]));
      swiglu_back8<DT>(d, g, u, h);
      if (kSave) {
        const uint32_t b = step_byte(block_max_bits(h), kFormat);
        const uint2 c = encode8(h, b, kFormat);
        if (r < n) kh.store(r, c, b);
      }
      if (data && r < n) {
        cg.store(r, g);
        cu.store(r, u);
      }
    }
    n = after;
    cg.p += cg.turn;
    cu.p += cu.turn;
    kh.next();
  }
}

template <int DT, int kRows, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_fwd(RowView gate, RowView up, RowOut h, Saved8 sg, Saved8 su,
                                                         int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  Span8<DT> ng[kRows], nu[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y, left = row < rows ? features - col : 0;
    ng[r] = fetch_span<DT>(gate, row * gate.ld + col, left);
    nu[r] = fetch_span<DT>(up, row * up.ld + col, left);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y, left = row < rows ? features - col : 0;
    const Raw8<DT> rg = align_span<DT>(ng[r], gate, row * gate.ld + col, left);
    const Raw8<DT> ru = align_span<DT>(nu[r], up, row * up.ld + col, left);
    float g[8], u[8];
    unpack<DT>(rg, g);
    unpack<DT>(ru, u);
    if (kSave) {
      const uint32_t a = step_byte(raw_max_bits<DT>(rg), sg.format);
      const uint32_t b = step_byte(raw_max_bits<DT>(ru), su.format);
      if (in && row < rows) {
        store_saved(sg, row, col, encode8(g, a, sg.format), a);
        store_saved(su, row, col, encode8(u, b, su.format), b);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = g[k] * sigmoid<DT>(g[k]) * u[k];
    store_span<DT>(h.p, row * h.ld + col, left, pack<DT>(g), row_lanes());
  }
}

template <int DT, int kRows, bool kSave>
__global__ void __launch_bounds__(kThreads) k_swiglu_bwd(RowView dh, Saved8 gate, Saved8 up, RowOut dgate, RowOut dup,
                                                         Saved8 sh, int64_t rows, int64_t features) {
  const int64_t col = (int64_t(blockIdx.y) * blockDim.x + threadIdx.x) * 8;
  const int64_t row0 = int64_t(blockIdx.x) * blockDim.y * kRows + threadIdx.y;
  const bool in = col < round_up_dev(features, kPanel8);
  Span8<DT> nd[kRows];
  float g[kRows][8], u[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const bool live = in && row < rows;
    nd[r] = fetch_span<DT>(dh, row * dh.ld + col, live ? features - col : 0);
    load8(gate, live ? row : 0, live ? col : gate.ld, g[r]);
    load8(up, live ? row : 0, live ? col : up.ld, u[r]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + int64_t(r) * blockDim.y;
    const bool live = in && row < rows;
    const int64_t left = live ? features - col : 0;
    float d[8], h[8];
    unpack<DT>(align_span<DT>(nd[r], dh, row * dh.ld + col, left), d);
    swiglu_back8<DT>(d, g[r], u[r], h);
    if (kSave) {
      const uint32_t b = step_byte(block_max_bits(h), sh.format);
      if (live) store_saved(sh, row, col, encode8(h, b, sh.format), b);
    }
    store_span<DT>(dgate.p, row * dgate.ld + col, left, pack<DT>(g[r]), row_lanes());
    store_span<DT>(dup.p, row * dup.ld + col, left, pack<DT>(u[r]), row_lanes());
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

// Calls f with the element type, or with it and the format, as constants.
template <typename F>
void with_type(int32_t dt, F&& f) {
  if (dt == RF_F32) f(std::integral_constant<int, RF_F32>{});
  else if (dt == RF_BF16) f(std::integral_constant<int, RF_BF16>{});
  else f(std::integral_constant<int, RF_F16>{});
}
template <typename F>
void with_types(int32_t dt, int32_t format, F&& f) {
  with_type(dt, [&](auto t) {
    if (format == RF_INT8) f(t, std::integral_constant<int, RF_INT8>{});
    else f(t, std::integral_constant<int, RF_E4M3>{});
  });
}
// Rows of 8-element vectors on 16-byte boundaries.
bool typed(int64_t features, const void* p, int64_t ld, int32_t dt) {
  return features % 8 == 0 && rows_vectorised(p, ld, dt);
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
  if (typed(out->features, x, ldx, dtype)) {
    with_types(dtype, out->format, [&](auto dt, auto fmt) {
      constexpr int DT = decltype(dt)::value, F = decltype(fmt)::value, R = DT == RF_F32 ? 2 : 4;
      auto go = [&](auto sr) {
        constexpr auto kernel = k_save_typed<DT, F, decltype(sr)::value>;
        const Walk w = walk<kernel>(out->rows, out->features, R);
        kernel<<<w.grid, w.block, 0, st>>>(x, ldx, saved8(*out), out->rows, out->features, seed);
      };
      stochastic ? go(std::true_type{}) : go(std::false_type{});
    });
    return check_launch("k_save");
  }
  const Tiling t = tiling(out->rows, out->features, 2);
  with_type(dtype, [&](auto dt) {
    auto go = [&](auto kernel) {
      kernel<<<t.grid, t.block, 0, st>>>(row_view(x, ldx, dtype, out->rows, out->features), saved8(*out), out->rows, out->features, seed);
    };
    stochastic ? go(k_save<decltype(dt)::value, 2, true>) : go(k_save<decltype(dt)::value, 2, false>);
  });
  return check_launch("k_save");
}

extern "C" rf_status rf_load_activation(const rf_saved_activation* saved, void* out, int64_t ldo, int32_t dtype,
                                        void* stream) {
  RF_TRY(check_saved(saved, "rf_load_activation"));
  RF_TRY(check_rows(out, ldo, dtype, saved->rows, saved->features, "rf_load_activation: out"));
  if (saved->rows == 0) return RF_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Typed float32 column tiles are 1024 features, not 2048: beyond 65535 of
  // them (grid.y) the simple kernel takes the row.
  const bool fits = dtype != RF_F32 || saved->features <= int64_t(65535) * kThreads * 4;
  if (fits && typed(saved->features, out, ldo, dtype)) {
    with_types(dtype, saved->format, [&](auto dt, auto fmt) {
      constexpr int DT = decltype(dt)::value;
      constexpr auto kernel = k_load_typed<DT, decltype(fmt)::value>;
      const Walk w = walk<kernel>(saved->rows, saved->features, 4, DT == RF_F32 ? 4 : 8);
      kernel<<<w.grid, w.block, 0, st>>>(saved8(*saved), out, ldo, saved->rows, saved->features);
    });
    return check_launch("k_load");
  }
  const Tiling t = tiling(saved->rows, saved->features, 2);
  with_type(dtype, [&](auto dt) {
    k_load<decltype(dt)::value, 2>
        <<<t.grid, t.block, 0, st>>>(saved8(*saved), row_out(out, ldo, dtype), saved->rows, saved->features);
  });
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
  if (typed(features, gate, ld_gate, dtype) && typed(features, up, ld_up, dtype) && typed(features, h, ld_h, dtype) &&
      (!saved_gate || saved_gate->format == saved_up->format)) {
    with_types(dtype, saved_gate ? saved_gate->format : int32_t(RF_INT8), [&](auto dt, auto fmt) {
      constexpr int DT = decltype(dt)::value, F = decltype(fmt)::value, R = DT == RF_F32 ? 1 : 2;
      auto go = [&](auto save) {
        constexpr auto kernel = k_swiglu_fwd_typed<DT, F, decltype(save)::value>;
        const Walk w = walk<kernel>(rows, features, R);
        kernel<<<w.grid, w.block, 0, st>>>(gate, ld_gate, up, ld_up, h, ld_h, sg, su, rows, features);
      };
      saved_gate ? go(std::true_type{}) : go(std::false_type{});
    });
    return check_launch("k_swiglu_fwd");
  }
  const Tiling t = tiling(rows, features, 1);
  const RowView g = row_view(gate, ld_gate, dtype, rows, features), u = row_view(up, ld_up, dtype, rows, features);
  const RowOut o = row_out(h, ld_h, dtype);
  with_type(dtype, [&](auto dt) {
    auto go = [&](auto kernel) { kernel<<<t.grid, t.block, 0, st>>>(g, u, o, sg, su, rows, features); };
    saved_gate ? go(k_swiglu_fwd<decltype(dt)::value, 1, true>) : go(k_swiglu_fwd<decltype(dt)::value, 1, false>);
  });
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
  if (typed(features, grad_h, ld_grad, dtype) && typed(features, grad_gate, ld_gate, dtype) &&
      typed(features, grad_up, ld_up, dtype)) {
    with_types(dtype, saved_h ? saved_h->format : int32_t(RF_INT8), [&](auto dt, auto fmt) {
      constexpr int DT = decltype(dt)::value, F = decltype(fmt)::value, R = 1;
      auto go = [&](auto save) {
        constexpr auto kernel = k_swiglu_bwd_typed<DT, F, decltype(save)::value>;
        const Walk w = walk<kernel>(rows, features, R);
        kernel<<<w.grid, w.block, 0, st>>>(grad_h, ld_grad, saved8(*saved_gate), saved8(*saved_up), grad_gate, ld_gate,
                                           grad_up, ld_up, sh, rows, features);
      };
      saved_h ? go(std::true_type{}) : go(std::false_type{});
    });
    return check_launch("k_swiglu_bwd");
  }
  const Tiling t = tiling(rows, features, 1);
  const RowView d = row_view(grad_h, ld_grad, dtype, rows, features);
  const RowOut dg = row_out(grad_gate, ld_gate, dtype), du = row_out(grad_up, ld_up, dtype);
  with_type(dtype, [&](auto dt) {
    auto go = [&](auto kernel) {
      kernel<<<t.grid, t.block, 0, st>>>(d, saved8(*saved_gate), saved8(*saved_up), dg, du, sh, rows, features);
    };
    saved_h ? go(k_swiglu_bwd<decltype(dt)::value, 1, true>) : go(k_swiglu_bwd<decltype(dt)::value, 1, false>);
  });
  return check_launch("k_swiglu_bwd");
}
