// The 8-bit form of a saved activation, and 8-element row access for the
// kernels that read or write one.
//
// A row of features is cut into blocks of 32.  A block holds 32 codes (int8
// in two's complement, or e4m3) and one byte s: value = code * 2^(s - 127).
// s is the smallest in [1, top] with max|x| <= 127 * 2^(s - 127) (448 for
// e4m3), so nothing saturates below the largest step; top (248, 246) is the
// largest at which every code is finite in float32 and bfloat16, and larger
// magnitudes saturate there.  s = 255: the block held an infinity or a NaN,
// and every value of it reads as NaN.  Powers of two make each value exact in
// bfloat16 (8 significant bits at most), so a tensor-core product over these
// values has no rounding of its operand.
//
// Codes: [rows][ld] bytes, ld = features rounded up to 16, zeros behind the
// last feature.  Steps: [panels of 128 features][scale_rows][4], scale_rows =
// rows rounded up to 64: a warp that reads 128 features of consecutive rows
// reads consecutive words, and panels start on 256-byte boundaries; blocks
// behind the last feature hold 1.
#pragma once

#include <cuda_fp8.h>

#include "rf_common.cuh"

namespace rf {

constexpr int kBlock8 = 32;       // features that share a step
constexpr int kPanel8 = 128;      // features per panel of steps
constexpr uint32_t kNanStep = 255u;
constexpr int64_t kMaxFeatures = int64_t(1) << 26;  // keeps column tiles of 2048 features inside a grid's 65535 in y

// A device view of a row-strided array of one of the float types.
struct RowView {
  const void* p;
  int64_t ld;     // elements between rows
  int32_t dt;     // rf_dtype
  int32_t vec;    // rows start on 16-byte boundaries
  int64_t size;   // elements from p to the last row's end
};
struct RowOut {
  void* p;
  int64_t ld;
  int32_t dt;
  int32_t vec;
};
struct Saved8 {
  uint8_t* codes;
  uint8_t* scales;
  int64_t ld;
  int64_t scale_rows;
  int32_t format;
};

inline bool rows_vectorised(const void* p, int64_t ld, int dt) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * int64_t(dtype_size(dt))) % 16 == 0;
}
inline RowView row_view(const void* p, int64_t ld, int dt, int64_t rows, int64_t features) {
  return RowView{p, ld, dt, rows_vectorised(p, ld, dt), rows > 0 ? (rows - 1) * ld + features : 0};
}
inline RowOut row_out(void* p, int64_t ld, int dt) { return RowOut{p, ld, dt, rows_vectorised(p, ld, dt)}; }
inline Saved8 saved8(const rf_saved_activation& s) {
  return Saved8{s.codes, s.scales, s.ld, s.scale_rows, s.format};
}
__device__ __forceinline__ RowOut row_out_dev(void* p, int64_t ld, int dt) {
  return RowOut{p, ld, dt, (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * (dt == RF_F32 ? 4 : 2)) % 16 == 0};
}
// Checks of a caller's saved activation; `what` names it in the message.
rf_status check_saved(const rf_saved_activation* s, const char* what);

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// -- typed rows on 16-byte boundaries ------------------------------------------
// 8 elements as they lie in memory, so that the next tile's loads can be in
// flight in few registers while this one is worked on.
template <int DT>
struct Raw8 {
  uint4 u[DT == RF_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw(const void* p, int64_t i) {
  Raw8<DT> r;
  if (DT == RF_F32) {
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
    r.u[0] = __ldg(q);
    r.u[DT == RF_F32 ? 1 : 0] = __ldg(q + 1);
  } else {
    r.u[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ Raw8<DT> zero_raw() {
  Raw8<DT> r;
  r.u[0] = make_uint4(0, 0, 0, 0);
  r.u[DT == RF_F32 ? 1 : 0] = make_uint4(0, 0, 0, 0);
  return r;
}
template <int DT>
__device__ __forceinline__ void unpack(const Raw8<DT>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
  if (DT == RF_F32) {
    const uint4 v = r.u[DT == RF_F32 ? 1 : 0];
    const uint32_t z[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[k] = __uint_as_float(w[k]);
      f[4 + k] = __uint_as_float(z[k]);
    }
  } else if (DT == RF_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      f[2 * k] = x.x;
      f[2 * k + 1] = x.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ void store_vec(void* p, int64_t i, const float (&f)[8]) {
  if (DT == RF_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(f[0], f[1], f[2], f[3]);
    q[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else if (DT == RF_BF16) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
  }
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

// -- typed rows that start and end anywhere --------------------------------------
// One by one, 8 elements are 8 accesses that each touch every line of a warp's
// span: 16384 x 4097 bfloat16 loaded in 187 us (now 92), 1527 x 1001 float32
// LayerNorm backward 40 us (now 33).
// So whole 16-byte pieces on their boundaries move, and registers shift them
// into place.  A load may take in neighbouring elements of the array, never any
// outside it: at its two ends, elements go one by one.  Stores write a row's
// own elements only, the pieces that hang over its ends one by one.
//
// `i`: the first element's index behind p; `left`: how many of the row's
// elements start there (0 or less: none).
template <int DT>
struct Span8 {
  uint4 c[DT == RF_F32 ? 3 : 2];
};
// Elements between a 16-byte boundary and element i.
template <int DT>
__device__ __forceinline__ int lead(const void* p, int64_t i) {
  constexpr int es = DT == RF_F32 ? 4 : 2;
  return int(uint32_t(reinterpret_cast<uintptr_t>(p) / es + uint64_t(i)) & uint32_t(16 / es - 1));
}
// Whether the pieces that hold n elements lie within the array.
template <int DT>
__device__ __forceinline__ bool span_inside(int a, int64_t i, int n, int64_t size) {
  constexpr int per = DT == RF_F32 ? 4 : 8;
  return i >= a && i - a + (a + n + per - 1) / per * per <= size;
}
template <int DT>
__device__ __forceinline__ Span8<DT> fetch_span(const RowView& t, int64_t i, int64_t left) {
  constexpr int es = DT == RF_F32 ? 4 : 2, per = 16 / es, C = DT == RF_F32 ? 3 : 2;
  const int a = lead<DT>(t.p, i), n = int(min(left, int64_t(8)));
  const bool inside = span_inside<DT>(a, i, n, t.size);
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(t.p) + (i - a) * es);
  Span8<DT> s;
#pragma unroll
  for (int k = 0; k < C; ++k) s.c[k] = inside && n > 0 && k * per < a + n ? __ldg(q + k) : make_uint4(0, 0, 0, 0);
  return s;
}
// The vector out of its pieces; zeros behind the row.
template <int DT>
__device__ __forceinline__ Raw8<DT> align_span(const Span8<DT>& s, const RowView& t, int64_t i, int64_t left) {
  const int a = lead<DT>(t.p, i);
  Raw8<DT> r;
  if (DT == RF_F32) {
    const uint4 z = s.c[DT == RF_F32 ? 2 : 0];
    uint32_t w[11] = {s.c[0].x, s.c[0].y, s.c[0].z, s.c[0].w, s.c[1].x, s.c[1].y, s.c[1].z, s.c[1].w, z.x, z.y, z.z};
#pragma unroll
    for (int k = 0; k < 9; ++k) w[k] = a & 2 ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = a & 1 ? w[k + 1] : w[k];
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
    r.u[DT == RF_F32 ? 1 : 0] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    uint32_t w[8] = {s.c[0].x, s.c[0].y, s.c[0].z, s.c[0].w, s.c[1].x, s.c[1].y, s.c[1].z, s.c[1].w};
#pragma unroll
    for (int k = 0; k < 6; ++k) w[k] = a & 4 ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = a & 2 ? w[k + 1] : w[k];
    const uint32_t halves = a & 1 ? 0x5432u : 0x3210u;
    r.u[0] = make_uint4(__byte_perm(w[0], w[1], halves), __byte_perm(w[1], w[2], halves),
                        __byte_perm(w[2], w[3], halves), __byte_perm(w[3], w[4], halves));
  }
  const int n = int(min(left, int64_t(8)));
  if (n > 0 && !span_inside<DT>(a, i, n, t.size)) {
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
  } else if (n < 8) {
    uint4& u = r.u[0];
    if (DT == RF_F32) {
      uint4& v = r.u[DT == RF_F32 ? 1 : 0];
      u.x = n > 0 ? u.x : 0u, u.y = n > 1 ? u.y : 0u, u.z = n > 2 ? u.z : 0u, u.w = n > 3 ? u.w : 0u;
      v.x = n > 4 ? v.x : 0u, v.y = n > 5 ? v.y : 0u, v.z = n > 6 ? v.z : 0u, v.w = 0u;
    } else {
      auto keep = [&](uint32_t x, int k) { return n >= k + 2 ? x : n == k + 1 ? x & 0xFFFFu : 0u; };
      u = make_uint4(keep(u.x, 0), keep(u.y, 2), keep(u.z, 4), keep(u.w, 6));
    }
  }
  return r;
}
// Writes a vector.  Called by all lanes of a warp; `width` neighbouring lanes
// hold consecutive vectors of one row, and each writes the pieces that end
// within its own, with the first elements from the lane before.
template <int DT>
__device__ __forceinline__ void store_span(void* p, int64_t i, int64_t left, const Raw8<DT>& r, int width = 32) {
  constexpr int es = DT == RF_F32 ? 4 : 2;
  const int a = lead<DT>(p, i), lane = int(threadIdx.x + blockDim.x * threadIdx.y) & (width - 1);
  uint8_t* q = static_cast<uint8_t*>(p) + (i - a) * es;
  bool head, next;  // the piece that starts at q, and the one that holds this vector's last elements
  if (DT == RF_F32) {
    const uint4 u = r.u[DT == RF_F32 ? 1 : 0];
    uint32_t w[11] = {0, 0, 0, r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k] = __shfl_up_sync(0xFFFFFFFFu, w[k + 8], 1);
#pragma unroll
    for (int k = 10; k >= 2; --k) w[k] = a & 2 ? w[k - 2] : w[k];
#pragma unroll
    for (int k = 10; k >= 3; --k) w[k] = a & 1 ? w[k - 1] : w[k];
    head = left >= 4 - a && (a == 0 || lane != 0);
    const bool mid = left >= 8 - a;
    next = a == 0 || (lane != width - 1 && left - 8 >= 4 - a);
    if (head) *reinterpret_cast<uint4*>(q) = make_uint4(w[3], w[4], w[5], w[6]);
    if (mid) *reinterpret_cast<uint4*>(q + 16) = make_uint4(w[7], w[8], w[9], w[10]);
    if (head && mid && next) return;
    const uint32_t f[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left && !(k < 4 - a ? head : k < 8 - a ? mid : next)) static_cast<uint32_t*>(p)[i + k] = f[k];
  } else {
    const uint32_t f[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = __shfl_up_sync(0xFFFFFFFFu, f[k], 1);
      w[4 + k] = f[k];
    }
#pragma unroll
    for (int k = 7; k >= 2; --k) w[k] = a & 4 ? w[k - 2] : w[k];
#pragma unroll
    for (int k = 7; k >= 3; --k) w[k] = a & 2 ? w[k - 1] : w[k];
    const uint32_t halves = a & 1 ? 0x5432u : 0x7654u;
    head = left >= 8 - a && (a == 0 || lane != 0);
    next = a == 0 || (lane != width - 1 && left - 8 >= 8 - a);
    if (head)
      *reinterpret_cast<uint4*>(q) = make_uint4(__byte_perm(w[3], w[4], halves), __byte_perm(w[4], w[5], halves),
                                                __byte_perm(w[5], w[6], halves), __byte_perm(w[6], w[7], halves));
    if (head && next) return;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left && !(k < 8 - a ? head : next))
        static_cast<uint16_t*>(p)[i + k] = uint16_t(f[k >> 1] >> (16 * (k & 1)));
  }
}

// -- 8 elements with the type known at run time -----------------------------------
// Short code, for kernels of any combination of types and for parameters:
// shifted pieces of three types took no less time there.  Those at or behind
// `n` read as 0.
__device__ __forceinline__ void load8(const RowView& t, int64_t row, int64_t col, int64_t n, float (&f)[8]) {
  const int64_t i = row * t.ld + col;
  if (t.vec && col + 8 <= n) {
    if (t.dt == RF_F32) unpack<RF_F32>(load_raw<RF_F32>(t.p, i), f);
    else if (t.dt == RF_BF16) unpack<RF_BF16>(load_raw<RF_BF16>(t.p, i), f);
    else unpack<RF_F16>(load_raw<RF_F16>(t.p, i), f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = col + k < n ? ld_as_float(t.p, t.dt, i + k) : 0.f;
  }
}
// 8 values of a parameter or a gate with d elements.
__device__ __forceinline__ void load8_param(const void* p, int dt, int64_t col, int64_t d, float (&f)[8]) {
  load8(RowView{p, 0, dt, (reinterpret_cast<uintptr_t>(p) & 15) == 0, d}, 0, col, d, f);
}
// Writes 8 elements but those at or behind `n`.
__device__ __forceinline__ void store8(const RowOut& t, int64_t row, int64_t col, int64_t n, const float (&f)[8]) {
  const int64_t i = row * t.ld + col;
  if (t.vec && col + 8 <= n) {
    if (t.dt == RF_F32) store_vec<RF_F32>(t.p, i, f);
    else if (t.dt == RF_BF16) store_vec<RF_BF16>(t.p, i, f);
    else store_vec<RF_F16>(t.p, i, f);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col + k < n) st_from_float(t.p, t.dt, i + k, f[k]);
  }
}
// -- pairs ------------------------------------------------------------------
// sm_100 multiplies and adds two float32 in one instruction; these kernels are
// short of issue slots, not of arithmetic.  Same roundings as one by one.
__device__ __forceinline__ float2 pair(const float* f, int k) { return make_float2(f[2 * k], f[2 * k + 1]); }
__device__ __forceinline__ void put_pair(float* f, int k, float2 v) {
  f[2 * k] = v.x;
  f[2 * k + 1] = v.y;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ void mul8(float (&f)[8], float2 s) {
#pragma unroll
  for (int k = 0; k < 4; ++k) put_pair(f, k, __fmul2_rn(pair(f, k), s));
}
__device__ __forceinline__ void mul8(float (&f)[8], const float (&g)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) put_pair(f, k, __fmul2_rn(pair(f, k), pair(g, k)));
}

// -- codes ------------------------------------------------------------------
__device__ __forceinline__ float step_value(uint32_t s) {
  return __uint_as_float(s == kNanStep ? 0x7FC00000u : s << 23);
}

// Four codes of a word -> floats (before the step).
__device__ __forceinline__ void decode4(uint32_t w, int format, float* f) {
  if (format == RF_INT8) {
    // q + 128 in the low byte of 2^23's significand, then an exact subtraction.
    const uint32_t o = w ^ 0x80808080u;
    const float2 off = both(-8388736.f);
    put_pair(f, 0, __fadd2_rn(make_float2(__uint_as_float(__byte_perm(o, 0x4B000000u, 0x7650)),
                                          __uint_as_float(__byte_perm(o, 0x4B000000u, 0x7651))), off));
    put_pair(f, 1, __fadd2_rn(make_float2(__uint_as_float(__byte_perm(o, 0x4B000000u, 0x7652)),
                                          __uint_as_float(__byte_perm(o, 0x4B000000u, 0x7653))), off));
  } else {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w & 0xFFFFu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w >> 16), __NV_E4M3);
    const float2 x = __half22float2(__half2(a)), y = __half22float2(__half2(b));
    f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
  }
}

__device__ __forceinline__ int64_t scale_index(const Saved8& s, int64_t row, int64_t col) {
  return ((col / kPanel8) * s.scale_rows + row) * 4 + (col % kPanel8) / kBlock8;
}

// 8 values of a saved row; zeros at and behind column s.ld (col % 8 == 0).
__device__ __forceinline__ void load8(const Saved8& s, int64_t row, int64_t col, float (&f)[8]) {
  if (col >= s.ld) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
    return;
  }
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(s.codes + row * s.ld + col));
  const float st = step_value(__ldg(s.scales + scale_index(s, row, col)));
  decode4(w.x, s.format, f);
  decode4(w.y, s.format, f + 4);
  mul8(f, both(st));
}

// The step byte for a block whose largest magnitude has the float bits `a`
// (0x7F800000 and above: not finite).
__device__ __forceinline__ uint32_t step_byte(uint32_t a, int format) {
  if (a >= 0x7F800000u) return kNanStep;
  const int sh = format == RF_INT8 ? 6 : 8;
  const uint32_t border = format == RF_INT8 ? 0x7E0000u : 0x600000u;  // significands of 127 / 64 and 448 / 256
  const int top = format == RF_INT8 ? 248 : 246;
  const int s = int(a >> 23) - sh + ((a & 0x7FFFFFu) > border ? 1 : 0);
  return uint32_t(min(max(s, 1), top));
}

// Largest magnitude over a block: 8 values here, 4 neighbouring lanes in all.
// As unsigned integers the magnitudes' bits order like the magnitudes, and an
// infinity or a NaN is above every finite value.
__device__ __forceinline__ uint32_t block_max_bits(const float (&f)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) a = max(a, __float_as_uint(f[k]) & 0x7FFFFFFFu);
  a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
  return max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 2));
}

// The same straight from memory's form: the magnitudes' bits of 16-bit types
// order like the magnitudes too, two at a time.
template <int DT>
__device__ __forceinline__ uint32_t raw_max_bits(const Raw8<DT>& r) {
  if (DT == RF_F32) {
    float f[8];
    unpack<DT>(r, f);
    return block_max_bits(f);
  }
  uint32_t m = __vmaxu2(__vmaxu2(r.u[0].x & 0x7FFF7FFFu, r.u[0].y & 0x7FFF7FFFu),
                        __vmaxu2(r.u[0].z & 0x7FFF7FFFu, r.u[0].w & 0x7FFF7FFFu));
  m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  m = max(m & 0xFFFFu, m >> 16);
  return DT == RF_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half(uint16_t(m))));
}

// 8 values -> 8 codes under step byte s, to nearest even.
__device__ __forceinline__ uint2 encode8(const float (&f)[8], uint32_t s, int format) {
  if (s == kNanStep) return make_uint2(0u, 0u);
  const float inv = __uint_as_float((254u - s) << 23);
  uint32_t w[2];
  if (format == RF_INT8) {
    uint32_t b[8];
    if (s == 248u) {  // the largest step: larger magnitudes saturate
#pragma unroll
      for (int k = 0; k < 8; ++k) b[k] = __float_as_uint(fminf(fmaxf(f[k] * inv, -127.f), 127.f) + 12582912.f);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // adding 1.5 * 2^23 rounds to an integer, whose low byte is the code
        const float2 r = __ffma2_rn(pair(f, k), both(inv), both(12582912.f));
        b[2 * k] = __float_as_uint(r.x);
        b[2 * k + 1] = __float_as_uint(r.y);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __byte_perm(__byte_perm(b[4 * h], b[4 * h + 1], 0x0040), __byte_perm(b[4 * h + 2], b[4 * h + 3], 0x0040),
                         0x5410);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo =
          __nv_cvt_float2_to_fp8x2(__fmul2_rn(pair(f, 2 * h), both(inv)), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi =
          __nv_cvt_float2_to_fp8x2(__fmul2_rn(pair(f, 2 * h + 1), both(inv)), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | (hi << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}

// Writes a block quarter: the codes, and by the quad's first lane the step.
// All 4 lanes of a quad call with consecutive columns; col < panels * 128.
__device__ __forceinline__ void store_saved(const Saved8& s, int64_t row, int64_t col, uint2 codes, uint32_t step) {
  if (col < s.ld) *reinterpret_cast<uint2*>(s.codes + row * s.ld + col) = codes;
  if ((col & (kBlock8 - 1)) == 0) s.scales[scale_index(s, row, col)] = uint8_t(step);
}

// One vector of a row held by a team of whole warps, to nearest even; columns
// behind the last panel only take part in the shuffles.
__device__ __forceinline__ void save_row8(const Saved8& s, int64_t row, int64_t col, int64_t n, const float (&f)[8]) {
  // A block behind the last feature has step 1, also where the row's
  // normalisation has made NaNs of its zeros.
  const uint32_t a = block_max_bits(f), st = col / kBlock8 * kBlock8 < n ? step_byte(a, s.format) : 1u;
  if (col < (n + kPanel8 - 1) / kPanel8 * kPanel8) store_saved(s, row, col, encode8(f, st, s.format), st);
}

// A float16 array has no value above 65504; a step of the 8-bit form may.
__device__ __forceinline__ void saturate8(int dt, float (&f)[8]) {
  if (dt != RF_F16) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = f[k] != f[k] ? f[k] : fminf(fmaxf(f[k], -65504.f), 65504.f);
}

__device__ __forceinline__ int64_t round_up_dev(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// The value that a float holds once stored as `dt`.
__device__ __forceinline__ void round8(int dt, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = round_to(dt, f[k]);
}

}  // namespace rf
