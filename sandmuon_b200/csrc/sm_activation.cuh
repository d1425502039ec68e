// sm_activation.cuh -- 8-bit activation checkpoints: pack, unpack and GELU.
//
// A checkpoint holds an activation x [rows, cols] for the backward pass as
// int8 values in groups of kGroup = 32 consecutive columns of one row, each
// group with the scale 2^e, e the smallest integer with max|x| <= 127 * 2^e
// (clamped to the range below), q = rint(x * 2^-e), x^ = q * 2^e, so
// |x - x^| <= 2^(e-1) < max|x| / 127.  A power of two keeps x^ exact in BF16
// (7 significant bits) and makes the scaling itself free of rounding: the
// products the backward pass takes of x^ lose nothing beyond this one
// quantisation.  A group with a non-finite member has code 255 and stands for
// NaN, so an overflow reaches the gradient as it would without a checkpoint.
//
// Memory: values [rows, ld] int8, ld = cols rounded up to 16 (a TMA row
// stride), padding 0; codes e + 127 [rows, lde] uint8, lde = groups rounded up
// to 4, padding 127 (scale 1).
//
// All kernels here read and write each element once and are bound by HBM.
// Two mappings of a warp onto a row:
//   VEC   a lane owns 8 consecutive columns (16- or 32-byte accesses, 4 lanes
//         share a group's maximum by two shuffles); needs cols % 8 == 0 and
//         16-byte-aligned contiguous rows
//   else  a lane owns columns base + 32 i + lane (element accesses that are
//         contiguous across the warp, one redux per group); any stride
#pragma once

#include <cuda_fp16.h>

#include "sm_common.cuh"

namespace smb {

constexpr int kGroup = SM_ACTIVATION_GROUP;
constexpr int kActThreads = 256;
constexpr uint32_t kCodeNan = 255;
constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the rounded integer

// Exponent codes e + 127 a type's checkpoint may use.  The lower ends keep
// every non-zero x^ a normal number of BF16 (e >= -126), and an FP16 number
// where x was one (e >= -24).  The upper ends keep x^ finite: 127 * 2^e is the
// largest such value below the type's maximum, and the few numbers above it
// (over 65024 in FP16, over 127 * 2^121 else) are held as it, less than a step
// away.
template <typename T>
struct CodeRange {
  static constexpr int kLow = 1, kHigh = 127 + 121;
};
template <>
struct CodeRange<__half> {
  static constexpr int kLow = 127 - 24, kHigh = 127 + 9;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Eight consecutive elements as 16-byte words, and their FP32 values.
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ void vec8_load(const T* p, Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
}

template <typename T>
__device__ __forceinline__ void vec8_store(T* p, const Vec8<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

__device__ __forceinline__ void vec8_unpack(const Vec8<float>& r, float (&v)[8]) {
  const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void vec8_unpack(const Vec8<__nv_bfloat16>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo_to_f(w[i]);
    v[2 * i + 1] = bf16_hi_to_f(w[i]);
  }
}
__device__ __forceinline__ void vec8_unpack(const Vec8<__half>& r, float (&v)[8]) {
  const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void vec8_pack(const float (&v)[8], Vec8<float>& r) {
  r.w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  r.w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
}
__device__ __forceinline__ void vec8_pack(const float (&v)[8], Vec8<__nv_bfloat16>& r) {
  r.w[0] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                      pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void vec8_pack(const float (&v)[8], Vec8<__half>& r) {
  r.w[0] =
      make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}

// ------------------------------------------------------------- quantisation

// The exponent code of a group from the bits of its largest magnitude (as an
// integer NaN > inf > every finite number).  With max = 1.f * 2^k:
// 127 * 2^(k-6) = 1.984375 * 2^k, so e = k - 6, or k - 5 for a fraction above
// 0x7e0000; the sum below carries into the exponent in exactly that case.
template <typename T>
__device__ __forceinline__ uint32_t group_code(uint32_t max_bits) {
  if (max_bits >= 0x7f800000u) return kCodeNan;
  const int code = static_cast<int>((max_bits + 0x01ffffu) >> 23) - 6;
  return static_cast<uint32_t>(min(max(code, CodeRange<T>::kLow), CodeRange<T>::kHigh));
}

// 2^-e, and 0 for a group that stands for NaN.
__device__ __forceinline__ float code_inverse(uint32_t code) {
  return code == kCodeNan ? 0.0f : __uint_as_float((254u - code) << 23);
}

// 2^e, and NaN for a group that stands for NaN.
__device__ __forceinline__ float code_scale(uint32_t code) {
  return __uint_as_float(code == kCodeNan ? 0x7fffffffu : code << 23);
}

// Bits whose low byte is rint(v * inv) in two's complement, |v * inv| <= 127.
__device__ __forceinline__ uint32_t quantise_bits(float v, float inv) {
  return __float_as_uint(fmaf(v, inv, kRoundMagic));
}

// v, or in a group at the upper end of its type's exponents v cut to what the
// group can hold.
template <typename T>
__device__ __forceinline__ float cut_to_group(float v, uint32_t code) {
  if (code != CodeRange<T>::kHigh) return v;
  constexpr float kTop = CodeRange<T>::kHigh == 127 + 9 ? 65024.0f : 127.0f * 0x1p121f;
  return fminf(fmaxf(v, -kTop), kTop);
}

__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Where a checkpoint lives.
struct Checkpoint {
  int8_t* values;
  uint8_t* codes;
  int64_t ld, lde;
};

// Quantises and stores this lane's 8 elements of row r.  Every lane of the
// warp takes part; `ok` says whether the lane's row exists.  Columns past the
// input hold v = 0 (their group's padding).
template <typename T, bool VEC>
__device__ __forceinline__ void store_packed(const Checkpoint& c, int64_t r, bool ok, int64_t col0, int lane,
                                             const float (&v)[8]) {
  if (VEC) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t code = group_code<T>(m);
    const float inv = code_inverse(code);
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = quantise_bits(cut_to_group<T>(v[i], code), inv);
    uint2 w = make_uint2(bytes4(b[0], b[1], b[2], b[3]), bytes4(b[4], b[5], b[6], b[7]));
    if (code == kCodeNan) w = make_uint2(0u, 0u);
    if (ok && col0 < c.ld) *reinterpret_cast<uint2*>(c.values + r * c.ld + col0) = w;
    const int64_t g = col0 / kGroup;
    if (ok && (lane & 3) == 0 && g < c.lde)
      c.codes[r * c.lde + g] = static_cast<uint8_t>(col0 < c.ld ? code : 127u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t col = col0 + 32 * i;
      const uint32_t m = __reduce_max_sync(0xffffffffu, ok ? __float_as_uint(v[i]) & 0x7fffffffu : 0u);
      const uint32_t code = group_code<T>(m);
      uint32_t b = quantise_bits(cut_to_group<T>(v[i], code), code_inverse(code));
      if (code == kCodeNan) b = 0;
      if (ok && col < c.ld) c.values[r * c.ld + col] = static_cast<int8_t>(b & 0xffu);
      const int64_t g = col / kGroup;
      if (ok && lane == 0 && g < c.lde) c.codes[r * c.lde + g] = static_cast<uint8_t>(col < c.ld ? code : 127u);
    }
  }
}

// Loads this lane's 8 elements of a strided row; columns past `cols` read 0.
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* x, int64_t r, int64_t rs, int64_t cs, int64_t col0, int64_t cols,
                                          bool ok, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  if (VEC) {
    if (ok && col0 < cols) {
      Vec8<T> w;
      vec8_load(x + r * rs + col0, w);
      vec8_unpack(w, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (ok && col0 + 32 * i < cols) v[i] = to_f32(x[r * rs + (col0 + 32 * i) * cs]);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_row8(T* y, int64_t r, int64_t col0, int64_t cols, bool ok, const float (&v)[8]) {
  if (VEC) {
    if (ok && col0 < cols) {
      Vec8<T> w;
      vec8_pack(v, w);
      vec8_store(y + r * cols + col0, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (ok && col0 + 32 * i < cols) y[r * cols + col0 + 32 * i] = from_f32<T>(v[i]);
  }
}

// The 8 checkpointed values of this lane, x^ in FP32.
template <bool VEC>
__device__ __forceinline__ void load_packed(const Checkpoint& c, int64_t r, bool ok, int64_t col0, int64_t cols,
                                            float (&v)[8]) {
  // u = q + 128 in the low mantissa bits of 2^23: (2^23 + u) - (2^23 + 128) = q exactly
  constexpr float kBias = 8388608.0f + 128.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  if (VEC) {
    if (ok && col0 < cols) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(c.values + r * c.ld + col0));
      const float s = code_scale(c.codes[r * c.lde + col0 / kGroup]);
      const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t f = __byte_perm(u[i / 4], 0x4b000000u, 0x7650u | (i & 3));
        v[i] = (__uint_as_float(f) - kBias) * s;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t col = col0 + 32 * i;
      if (ok && col < cols) {
        const uint32_t u = static_cast<uint8_t>(c.values[r * c.ld + col]) ^ 0x80u;
        v[i] = (__uint_as_float(0x4b000000u | u) - kBias) * code_scale(c.codes[r * c.lde + col / kGroup]);
      }
    }
  }
}

// ------------------------------------------------------ rows, columns, sums

// How a launch covers [rows, cols]: a CTA takes a strip of columns and a
// range of rows; 2^log_lanes lanes of a warp share a row (VEC), so that narrow
// inputs still fill a warp.
struct ActGeometry {
  int64_t rows, cols;
  int64_t rows_per_cta;
  int log_lanes;
};

struct ActLane {
  int lane, row_lane, row_lanes;
  int64_t col0, r_begin, r_end;
};

template <bool VEC>
__device__ __forceinline__ ActLane act_lane(const ActGeometry& g) {
  ActLane a;
  const int lanes = VEC ? 1 << g.log_lanes : 32;
  a.lane = threadIdx.x & (lanes - 1);
  a.row_lane = VEC ? threadIdx.x >> g.log_lanes : threadIdx.x >> 5;
  a.row_lanes = VEC ? kActThreads >> g.log_lanes : kActThreads / 32;
  a.col0 = VEC ? (static_cast<int64_t>(blockIdx.x) * lanes + a.lane) * 8
               : static_cast<int64_t>(blockIdx.x) * 256 + a.lane;
  a.r_begin = static_cast<int64_t>(blockIdx.y) * g.rows_per_cta;
  a.r_end = min(a.r_begin + g.rows_per_cta, g.rows);
  return a;
}

// Column sums of one CTA: per-lane FP32 sums over its rows, joined across the
// CTA's row lanes in a fixed order (FP64) and written to slot blockIdx.y of
// partials [splits, 2, cols] -- or, with one split, to the result [2, cols].
template <bool VEC>
__device__ __forceinline__ void write_column_sums(const ActGeometry& g, const ActLane& a, const float (&sq)[8],
                                                  const float (&su)[8], float* out) {
  __shared__ float sh[2][kActThreads * 8];
  const int width = VEC ? 8 << g.log_lanes : 256;  // columns of this CTA's strip
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = VEC ? a.lane * 8 + i : a.lane + 32 * i;
    sh[0][a.row_lane * width + c] = sq[i];
    sh[1][a.row_lane * width + c] = su[i];
  }
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * width;
  for (int t = threadIdx.x; t < 2 * width; t += kActThreads) {
    const int which = t >= width;
    const int c = t - which * width;
    if (base + c >= g.cols) continue;
    double s = 0.0;
    for (int l = 0; l < a.row_lanes; ++l) s += static_cast<double>(sh[which][l * width + c]);
    out[(static_cast<int64_t>(blockIdx.y) * 2 + which) * g.cols + base + c] = static_cast<float>(s);
  }
}

// sums[j] = sum over splits of partials[s][j], j < n = 2 * cols, in a fixed
// order: 32 columns x 8 split lanes per CTA, FP64.
__global__ void __launch_bounds__(256) k_column_sums_finish(const float* __restrict__ partials, int64_t n, int splits,
                                                            float* __restrict__ sums) {
  __shared__ double sh[8][33];
  const int c = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + c;
  grid_dep_wait();
  double s = 0.0;
  if (j < n) {
#pragma unroll 8
    for (int k = l; k < splits; k += 8) s += static_cast<double>(partials[static_cast<int64_t>(k) * n + j]);
  }
  sh[l][c] = s;
  __syncthreads();
  if (l == 0 && j < n) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][c];
    sums[j] = static_cast<float>(s);
  }
}

// --------------------------------------------------------------- the kernels

// Rows in flight per lane: enough loads to cover HBM latency at 8 warps a CTA.
constexpr int kActUnroll = 4;

template <typename T, bool VEC, bool STATS>
__global__ void __launch_bounds__(kActThreads)
    k_activation_pack(const T* __restrict__ x, int64_t rs, int64_t cs, ActGeometry g, Checkpoint c,
                      float* __restrict__ sums) {
  const ActLane a = act_lane<VEC>(g);
  float sq[8], su[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sq[i] = su[i] = 0.0f;
  for (int64_t r0 = a.r_begin; r0 < a.r_end; r0 += static_cast<int64_t>(a.row_lanes) * kActUnroll) {
    float v[kActUnroll][8];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      load_row8<T, VEC>(x, r, rs, cs, a.col0, g.cols, r < a.r_end, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      store_packed<T, VEC>(c, r, r < a.r_end, a.col0, a.lane, v[u]);
      if (STATS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sq[i] += v[u][i] * v[u][i];
          su[i] += v[u][i];
        }
      }
    }
  }
  if (STATS) write_column_sums<VEC>(g, a, sq, su, sums);
  grid_dep_launch();
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kActThreads)
    k_activation_unpack(ActGeometry g, Checkpoint c, T* __restrict__ out) {
  const ActLane a = act_lane<VEC>(g);
  for (int64_t r0 = a.r_begin; r0 < a.r_end; r0 += static_cast<int64_t>(a.row_lanes) * kActUnroll) {
    float v[kActUnroll][8];
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      load_packed<VEC>(c, r, r < a.r_end, a.col0, g.cols, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kActUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      store_row8<T, VEC>(out, r, a.col0, g.cols, r < a.r_end, v[u]);
    }
  }
}

// ---------------------------------------------------------------------- GELU

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kGeluCubic = 0.044715f;

template <bool TANH>
__device__ __forceinline__ float gelu_value(float x) {
  if (TANH) return 0.5f * x * (1.0f + tanhf(kSqrt2OverPi * (x + kGeluCubic * x * x * x)));
  // erfc keeps the relative accuracy of the negative tail
  return 0.5f * x * erfcf(-x * kSqrtHalf);
}

// Beyond |x| = 30 the slope is 0 or 1 in FP32; the clamp (which lets NaN
// through) keeps the tanh form's x^2 and x^3 finite.
template <bool TANH>
__device__ __forceinline__ float gelu_slope(float x) {
  x = x > 30.0f ? 30.0f : x < -30.0f ? -30.0f : x;
  if (TANH) {
    const float t = tanhf(kSqrt2OverPi * (x + kGeluCubic * x * x * x));
    return 0.5f * (1.0f + t) + 0.5f * x * (1.0f - t * t) * kSqrt2OverPi * (1.0f + 3.0f * kGeluCubic * x * x);
  }
  return 0.5f * erfcf(-x * kSqrtHalf) + x * expf(-0.5f * x * x) * kInvSqrt2Pi;
}

// y = gelu(x); packs x into `in` (PACK_IN) and the rounded y into `out` with
// y's column sums (PACK_OUT; sums may be null).
template <typename T, bool VEC, bool TANH, bool PACK_IN, bool PACK_OUT>
__global__ void __launch_bounds__(kActThreads)
    k_gelu_forward(const T* __restrict__ x, int64_t rs, int64_t cs, ActGeometry g, T* __restrict__ y, Checkpoint in,
                   Checkpoint out, float* __restrict__ sums) {
  constexpr int kUnroll = 2;
  const ActLane a = act_lane<VEC>(g);
  float sq[8], su[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sq[i] = su[i] = 0.0f;
  for (int64_t r0 = a.r_begin; r0 < a.r_end; r0 += static_cast<int64_t>(a.row_lanes) * kUnroll) {
    float v[kUnroll][8];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      load_row8<T, VEC>(x, r, rs, cs, a.col0, g.cols, r < a.r_end, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      const bool ok = r < a.r_end;
      if (PACK_IN) store_packed<T, VEC>(in, r, ok, a.col0, a.lane, v[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = to_f32(from_f32<T>(gelu_value<TANH>(v[u][i])));
      store_row8<T, VEC>(y, r, a.col0, g.cols, ok, v[u]);
      if (PACK_OUT) {
        store_packed<T, VEC>(out, r, ok, a.col0, a.lane, v[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sq[i] += v[u][i] * v[u][i];
          su[i] += v[u][i];
        }
      }
    }
  }
  if (PACK_OUT && sums != nullptr) write_column_sums<VEC>(g, a, sq, su, sums);
  grid_dep_launch();
}

// dx = delta * gelu'(x^)
template <typename T, bool VEC, bool TANH>
__global__ void __launch_bounds__(kActThreads)
    k_gelu_backward(const T* __restrict__ delta, int64_t rs, int64_t cs, ActGeometry g, Checkpoint c,
                    T* __restrict__ dx) {
  constexpr int kUnroll = 2;
  const ActLane a = act_lane<VEC>(g);
  for (int64_t r0 = a.r_begin; r0 < a.r_end; r0 += static_cast<int64_t>(a.row_lanes) * kUnroll) {
    float v[kUnroll][8], d[kUnroll][8];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
      load_packed<VEC>(c, r, r < a.r_end, a.col0, g.cols, v[u]);
      load_row8<T, VEC>(delta, r, rs, cs, a.col0, g.cols, r < a.r_end, d[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t r = r0 + u * a.row_lanes + a.row_lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = d[u][i] * gelu_slope<TANH>(v[u][i]);
      store_row8<T, VEC>(dx, r, a.col0, g.cols, r < a.r_end, v[u]);
    }
  }
}

}  // namespace smb
