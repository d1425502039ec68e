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
// All kernels here read and write each element once.  Packing and unpacking of
// aligned rows are bound by HBM, the strided mapping by its element accesses and
// GELU by load latency and instruction issue together (see there).
// Two mappings of a warp onto a row:
//   VEC   a lane owns 8 consecutive columns (16- or 32-byte accesses, 4 lanes
//         share a group's maximum by two shuffles); needs cols % 8 == 0 and
//         16-byte-aligned contiguous rows
//   else  a lane owns columns base + 32 i + lane (element accesses that are
//         contiguous across the warp, one redux per group); any stride
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

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

// Two FP32 values in one 64-bit register pair, for the packed instructions of
// sm_100: one packed instruction takes one issue slot for two elements' work,
// with the same roundings (GELU of 16384 x 4096 BF16: forward 107 -> 99 us,
// backward 76 -> 60 us).
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float a, float b) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  }
  __device__ __forceinline__ explicit Pair(float both) : Pair(both, both) {}
  __device__ __forceinline__ void get(float& a, float& b) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
  }
};
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

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
// Results from CodeRange<T>::kHigh up need `rare_group`.
template <typename T>
__device__ __forceinline__ uint32_t group_code(uint32_t max_bits) {
  return static_cast<uint32_t>(max(static_cast<int>((max_bits + 0x01ffffu) >> 23) - 6, CodeRange<T>::kLow));
}

// 2^-e
__device__ __forceinline__ float code_inverse(uint32_t code) { return __uint_as_float((254u - code) << 23); }

// 2^e, and NaN for a group that stands for NaN.
__device__ __forceinline__ float code_scale(uint32_t code) {
  return __uint_as_float(code == kCodeNan ? 0x7fffffffu : code << 23);
}

// A group at the upper end of its type's exponents, where v is cut to what the
// group can hold, or with a non-finite member (values 0, code 255).
template <typename T, int N>
__device__ __forceinline__ void rare_group(uint32_t max_bits, uint32_t& code, float& inv, float (&v)[N]) {
  constexpr float kTop = CodeRange<T>::kHigh == 127 + 9 ? 65024.0f : 127.0f * 0x1p121f;
  const bool finite = max_bits < 0x7f800000u;
  code = finite ? CodeRange<T>::kHigh : kCodeNan;
  inv = code_inverse(CodeRange<T>::kHigh);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = finite ? fminf(fmaxf(v[i], -kTop), kTop) : 0.0f;
}

// Bits whose low byte is rint(v * inv) in two's complement, |v * inv| <= 127.
__device__ __forceinline__ uint32_t quantise_bits(float v, float inv) {
  return __float_as_uint(fmaf(v, inv, kRoundMagic));
}

// Bits of the largest magnitude in the 4 lanes that share a group, NaN above
// inf above the rest: 16-bit types compare their own bits, two at a time.
__device__ __forceinline__ uint32_t group_max4(uint32_t m) {
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t max_s16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.s16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t group_max4_x2(const uint4& w) {
  constexpr uint32_t kAbs = 0x7fff7fffu;
  uint32_t m = max_s16x2(__vimax3_s16x2(w.x & kAbs, w.y & kAbs, w.z & kAbs), w.w & kAbs);
  m = max_s16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max_s16x2(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t group_max_bits(const Vec8<float>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m = max(m, max(r.w[i].x & 0x7fffffffu, r.w[i].y & 0x7fffffffu));
    m = max(m, max(r.w[i].z & 0x7fffffffu, r.w[i].w & 0x7fffffffu));
  }
  return group_max4(m);
}
__device__ __forceinline__ uint32_t group_max_bits(const Vec8<__nv_bfloat16>& r) {
  const uint32_t m = group_max4_x2(r.w[0]);
  return max(m << 16, m & 0xffff0000u);
}
__device__ __forceinline__ uint32_t group_max_bits(const Vec8<__half>& r) {
  const uint32_t m = group_max4_x2(r.w[0]);
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(max(m & 0xffffu, m >> 16)))));
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

// The two mappings' accesses.  `ok`: the lane's row exists.  FULL: every row
// and column of the access does, and nothing is checked.

// VEC: quantises 8 consecutive elements, given as words and as FP32 values
// (which a rare group changes), to `values` and, from a group's first lane,
// their code to `codes`.  All lanes of the warp take part.
template <typename T, bool FULL>
__device__ __forceinline__ void pack8(int8_t* values, uint8_t* codes, const Vec8<T>& words, const float (&in)[8],
                                      bool ok, bool in_values, bool in_codes) {
  const uint32_t max_bits = group_max_bits(words);
  uint32_t code = group_code<T>(max_bits);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = in[i];
  float inv = code_inverse(code);
  if (code >= CodeRange<T>::kHigh) rare_group<T>(max_bits, code, inv, v);
  uint32_t b[8];
  const Pair inv2(inv), magic(kRoundMagic);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float lo, hi;
    fma2(Pair(v[i], v[i + 1]), inv2, magic).get(lo, hi);
    b[i] = __float_as_uint(lo);
    b[i + 1] = __float_as_uint(hi);
  }
  if (FULL || (ok && in_values))
    *reinterpret_cast<uint2*>(values) = make_uint2(bytes4(b[0], b[1], b[2], b[3]), bytes4(b[4], b[5], b[6], b[7]));
  if ((threadIdx.x & 3) == 0 && (FULL || (ok && in_codes)))
    *codes = static_cast<uint8_t>(FULL || in_values ? code : 127u);
}

// Not VEC: elements 32 columns apart, a group across the warp's lanes.
template <typename T>
__device__ __forceinline__ void pack_strided(const Checkpoint& c, int64_t r, bool ok, int64_t col0, int lane,
                                             const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t col = col0 + 32 * i;
    const uint32_t m = __reduce_max_sync(0xffffffffu, ok ? __float_as_uint(v[i]) & 0x7fffffffu : 0u);
    uint32_t code = group_code<T>(m);
    float one[1] = {v[i]}, inv = code_inverse(code);
    if (code >= CodeRange<T>::kHigh) rare_group<T>(m, code, inv, one);
    const uint32_t b = quantise_bits(one[0], inv);
    if (ok && col < c.ld) c.values[r * c.ld + col] = static_cast<int8_t>(b & 0xffu);
    const int64_t g = col / kGroup;
    if (ok && lane == 0 && g < c.lde) c.codes[r * c.lde + g] = static_cast<uint8_t>(col < c.ld ? code : 127u);
  }
}

template <typename T>
__device__ __forceinline__ void load_strided(const T* x, int64_t r, int64_t rs, int64_t cs, int64_t col0, int64_t cols,
                                             bool ok, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = ok && col0 + 32 * i < cols ? to_f32(x[r * rs + (col0 + 32 * i) * cs]) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store_strided(T* y, int64_t r, int64_t col0, int64_t cols, bool ok,
                                              const float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (ok && col0 + 32 * i < cols) y[r * cols + col0 + 32 * i] = from_f32<T>(v[i]);
}

// x^ of 8 consecutive values, exactly: u = q + 128 in the low mantissa bits of
// 2^23, ((2^23 + u) - (2^23 + 128)) * 2^e = q * 2^e, in one fused step while
// 2^23 * 2^e is finite.
constexpr float kByteBias = 8388608.0f + 128.0f;
constexpr uint32_t kFusedCodes = 127 + 100;

__device__ __forceinline__ void unpack8(uint2 w, uint32_t code, float (&v)[8]) {
  const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(__byte_perm(u[i / 4], 0x4b000000u, 0x7650u | (i & 3)));
  if (code <= kFusedCodes) {
    const float s = __uint_as_float(code << 23);
    const Pair scale(s), bias(-kByteBias * s);
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma2(Pair(v[i], v[i + 1]), scale, bias).get(v[i], v[i + 1]);
  } else {
    const float s = code_scale(code);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (v[i] - kByteBias) * s;
  }
}

__device__ __forceinline__ void unpack_strided(const Checkpoint& c, int64_t r, bool ok, int64_t col0, int64_t cols,
                                               float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t col = col0 + 32 * i;
    v[i] = 0.0f;
    if (ok && col < cols) {
      const uint32_t u = static_cast<uint8_t>(c.values[r * c.ld + col]) ^ 0x80u;
      v[i] = (__uint_as_float(0x4b000000u | u) - kByteBias) * code_scale(c.codes[r * c.lde + col / kGroup]);
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

// A lane's running sums of its 8 columns' squares and values.
struct ColumnSums {
  Pair sq[4], su[4];
  __device__ __forceinline__ ColumnSums() {
#pragma unroll
    for (int i = 0; i < 4; ++i) sq[i] = su[i] = Pair(0.0f);
  }
  __device__ __forceinline__ void add(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Pair x(v[2 * i], v[2 * i + 1]);
      sq[i] = fma2(x, x, sq[i]);
      su[i] = add2(su[i], x);
    }
  }
};

// Column sums of one CTA: per-lane FP32 sums over its rows, joined across the
// CTA's row lanes in a fixed order (FP64) and written to slot blockIdx.y of
// partials [splits, 2, cols] -- or, with one split, to the result [2, cols].
template <bool VEC>
__device__ __forceinline__ void write_column_sums(const ActGeometry& g, const ActLane& a, const ColumnSums& s,
                                                  float* out) {
  float sq[8], su[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s.sq[i].get(sq[2 * i], sq[2 * i + 1]);
    s.su[i].get(su[2 * i], su[2 * i + 1]);
  }
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
// order: 32 columns x 32 split lanes per CTA (all loads of a few hundred splits
// in flight at once), FP64.
constexpr int kFinishLanes = 32;

__global__ void __launch_bounds__(32 * kFinishLanes)
    k_column_sums_finish(const float* __restrict__ partials, int64_t n, int splits, float* __restrict__ sums) {
  __shared__ double sh[kFinishLanes][33];
  const int c = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + c;
  grid_dep_wait();
  double s = 0.0;
  if (j < n) {
#pragma unroll 8
    for (int k = l; k < splits; k += kFinishLanes) s += static_cast<double>(partials[static_cast<int64_t>(k) * n + j]);
  }
  sh[l][c] = s;
  __syncthreads();
  // warp l joins column l of the block, its lanes the split lanes
  const int64_t out = static_cast<int64_t>(blockIdx.x) * 32 + l;
  s = warp_sum_d(sh[c][l]);
  if (c == 0 && out < n) sums[out] = static_cast<float>(s);
}

// --------------------------------------------------------------- the kernels

// Rows in flight per lane, and CTAs per SM of a launch: one wave of them (VEC).
constexpr int kActUnroll = 4;
constexpr int kPackCtas = 4, kUnpackCtas = 4, kGeluForwardCtas = 4, kGeluBackwardCtas = 4;
// The residency asked of the compiler; the strided mapping, bound by its
// element accesses, is left its registers and runs in two waves.
__host__ __device__ constexpr int resident(bool vec, int ctas) { return vec ? ctas : 2; }

// A VEC lane's walk down its rows: where its next row's 8 elements of each
// tensor are (null where there is none), and how far apart rows it visits are.
template <typename T>
struct RowPointer {
  T* p;
  int64_t step;
  __device__ __forceinline__ RowPointer(T* base, int64_t row, int64_t stride, int64_t offset, int rows)
      : p(base == nullptr ? nullptr : base + row * stride + offset), step(stride * rows) {}
  __device__ __forceinline__ T* take() {
    T* at = p;
    p += step;
    return at;
  }
};

struct PackPointer {
  RowPointer<int8_t> values;
  RowPointer<uint8_t> codes;
  __device__ __forceinline__ PackPointer(const Checkpoint& c, const ActLane& a)
      : values(c.values, a.r_begin + a.row_lane, c.ld, a.col0, a.row_lanes),
        codes(c.codes, a.r_begin + a.row_lane, c.lde, a.col0 / kGroup, a.row_lanes) {}
};

// Runs body<FULL>(rows in flight, first row) over the CTA's rows, U at a time.
// FULL needs the whole strip inside the columns and U rows for every lane.
template <int U, typename Body>
__device__ __forceinline__ void act_rows(const ActGeometry& g, const ActLane& a, Body&& body) {
  const bool full = (static_cast<int64_t>(blockIdx.x) + 1) * (int64_t{8} << g.log_lanes) <= g.cols;
  int64_t r0 = a.r_begin;
  if (full)
    for (; r0 + U * a.row_lanes <= a.r_end; r0 += U * a.row_lanes) body(std::true_type(), r0);
  for (; r0 < a.r_end; r0 += U * a.row_lanes) body(std::false_type(), r0);
}

template <typename T, bool VEC, bool STATS>
__global__ void __launch_bounds__(kActThreads, resident(VEC, kPackCtas))
    k_activation_pack(const T* __restrict__ x, int64_t rs, int64_t cs, ActGeometry g, Checkpoint c,
                      float* __restrict__ sums) {
  const ActLane a = act_lane<VEC>(g);
  ColumnSums column;
  if constexpr (VEC) {
    constexpr int kUnroll = sizeof(T) == 2 ? kActUnroll : 2;
    const bool in_x = a.col0 < g.cols, in_values = a.col0 < c.ld, in_codes = a.col0 / kGroup < c.lde;
    RowPointer<const T> xp(x, a.r_begin + a.row_lane, rs, a.col0, a.row_lanes);
    PackPointer pp(c, a);
    act_rows<kUnroll>(g, a, [&](auto full, int64_t r0) {
      constexpr bool kFull = decltype(full)::value;
      Vec8<T> w[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        memset(&w[u], 0, sizeof(w[u]));
        const T* at = xp.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) vec8_load(at, w[u]);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float v[8];
        vec8_unpack(w[u], v);
        pack8<T, kFull>(pp.values.take(), pp.codes.take(), w[u], v, r0 + u * a.row_lanes + a.row_lane < a.r_end,
                        in_values, in_codes);
        if (STATS) column.add(v);
      }
    });
  } else {
    for (int64_t r = a.r_begin + a.row_lane; r - a.row_lane < a.r_end; r += a.row_lanes) {
      float v[8];
      load_strided(x, r, rs, cs, a.col0, g.cols, r < a.r_end, v);
      pack_strided<T>(c, r, r < a.r_end, a.col0, a.lane, v);
      if (STATS) column.add(v);
    }
  }
  if (STATS) write_column_sums<VEC>(g, a, column, sums);
  grid_dep_launch();
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kActThreads, resident(VEC, kUnpackCtas))
    k_activation_unpack(ActGeometry g, Checkpoint c, T* __restrict__ out) {
  const ActLane a = act_lane<VEC>(g);
  if constexpr (VEC) {
    const bool in_x = a.col0 < g.cols;
    PackPointer pp(c, a);
    RowPointer<T> op(out, a.r_begin + a.row_lane, g.cols, a.col0, a.row_lanes);
    act_rows<kActUnroll>(g, a, [&](auto full, int64_t r0) {
      constexpr bool kFull = decltype(full)::value;
      uint2 w[kActUnroll];
      uint32_t code[kActUnroll];
#pragma unroll
      for (int u = 0; u < kActUnroll; ++u) {
        const int8_t* v = pp.values.take();
        const uint8_t* k = pp.codes.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) {
          w[u] = __ldg(reinterpret_cast<const uint2*>(v));
          code[u] = __ldg(k);
        }
      }
#pragma unroll
      for (int u = 0; u < kActUnroll; ++u) {
        T* at = op.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) {
          float v[8];
          unpack8(w[u], code[u], v);
          Vec8<T> o;
          vec8_pack(v, o);
          vec8_store(at, o);
        }
      }
    });
  } else {
    for (int64_t r = a.r_begin + a.row_lane; r < a.r_end; r += a.row_lanes) {
      float v[8];
      unpack_strided(c, r, true, a.col0, g.cols, v);
      store_strided(out, r, a.col0, g.cols, true, v);
    }
  }
}

// ---------------------------------------------------------------------- GELU
//
// gelu(x) = x Phi(x).  With h = Phi(-|x|):  gelu = max(x, 0) - |x| h, in which
// the negative tail does not cancel.  h = exp(-x^2/2) u G(u),
// u = 1 / (1 + p |x|): exp(x^2/2) Phi(-|x|) is smooth in u down to u = 0, and a
// polynomial of degree 8 holds it within 3e-8 relative over |x| < 14.5 (3.2e-7
// with FP32 coefficients and roundings).  The exponential adds the rounding of
// its argument, x^2 / 2: measured against FP64, gelu is within 4e-7 relative
// for -1 < x, 1.3e-6 to -5, 4.9e-6 to -10 and 8.8e-6 to -13.2; below, the
// exponential underflows and gelu is 0 (true values under 5e-39).  The
// coefficients are a minimax fit (iteratively reweighted least squares on
// Chebyshev nodes) to exp(x^2/2) erfc(|x|/sqrt 2) / (2 u).  The same
// exponential gives the density phi(x) of the derivative Phi(x) + x phi(x).
// CUDA's erfcf instead of this: 241 us forward, 187 us backward for
// 16384 x 4096 BF16, where this takes 98 and 60 (floors 62 and 51.5).  The
// forward pass issues in 63% of its cycles and stalls first for its loads, two
// rows of which are in flight per lane; the backward pass issues in 70%.

__device__ __forceinline__ float ex2_approx(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kGeluCubic = 0.044715f;

// For two elements: t = Phi(-|x|) / exp(-x^2 / 2) and d = exp(-x^2 / 2).
__device__ __forceinline__ void normal_tail(float x0, float x1, Pair& t, Pair& d) {
  const Pair x(x0, x1);
  const Pair u(rcp_approx(fmaf(fabsf(x0), 0.35f, 1.0f)), rcp_approx(fmaf(fabsf(x1), 0.35f, 1.0f)));
  float a0, a1;
  mul2(x, mul2(x, Pair(-0.5f * kLog2E))).get(a0, a1);
  d = Pair(ex2_approx(a0), ex2_approx(a1));
  Pair g = fma2(Pair(-0.029157886f), u, Pair(0.14403091f));
  g = fma2(g, u, Pair(-0.25583899f));
  g = fma2(g, u, Pair(0.15931970f));
  g = fma2(g, u, Pair(-0.023212353f));
  g = fma2(g, u, Pair(0.10555250f));
  g = fma2(g, u, Pair(0.11982129f));
  g = fma2(g, u, Pair(0.13986352f));
  g = fma2(g, u, Pair(0.13962130f));
  t = mul2(g, u);
}

// The logistic function of 2 sqrt(2/pi) (x + 0.044715 x^3): the tanh form is
// 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z)).
__device__ __forceinline__ Pair tanh_gate(Pair x, Pair x2) {
  constexpr float kScale = -2.0f * kLog2E * kSqrt2OverPi;
  float z0, z1;
  mul2(x, fma2(x2, Pair(kScale * kGeluCubic), Pair(kScale))).get(z0, z1);
  return Pair(rcp_approx(1.0f + ex2_approx(z0)), rcp_approx(1.0f + ex2_approx(z1)));
}

// v <- gelu(v).  +inf gives inf and -inf gives NaN, as x * Phi(x) does in
// floating point.
template <bool TANH>
__device__ __forceinline__ void gelu_values(float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if (TANH) {
      const Pair x(v[i], v[i + 1]);
      mul2(x, tanh_gate(x, mul2(x, x))).get(v[i], v[i + 1]);
    } else {
      Pair t, d;
      normal_tail(v[i], v[i + 1], t, d);
      float h0, h1;
      mul2(d, t).get(h0, h1);
      v[i] = fmaf(-fabsf(fminf(v[i], 40.0f)), h0, fmaxf(v[i], 0.0f));
      v[i + 1] = fmaf(-fabsf(fminf(v[i + 1], 40.0f)), h1, fmaxf(v[i + 1], 0.0f));
    }
  }
}

// v <- d * gelu'(v)
template <bool TANH>
__device__ __forceinline__ void gelu_gradients(float (&v)[8], const float (&d)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    Pair slope;
    if (TANH) {
      // beyond |x| = 30 the slope is 0 or 1; the clamp (which lets NaN through)
      // keeps x^2 finite
      const float x0 = v[i] > 30.0f ? 30.0f : v[i] < -30.0f ? -30.0f : v[i];
      const float x1 = v[i + 1] > 30.0f ? 30.0f : v[i + 1] < -30.0f ? -30.0f : v[i + 1];
      const Pair x(x0, x1), x2 = mul2(x, x), s = tanh_gate(x, x2);
      const Pair inner = mul2(x, fma2(x2, Pair(6.0f * kSqrt2OverPi * kGeluCubic), Pair(2.0f * kSqrt2OverPi)));
      slope = fma2(mul2(s, fma2(s, Pair(-1.0f), Pair(1.0f))), inner, s);
    } else {
      // Phi(x) + x phi(x) = [x >= 0] + exp(-x^2 / 2) (x / sqrt(2 pi) - sign(x) t),
      // both by x's sign bit
      Pair t, density;
      normal_tail(v[i], v[i + 1], t, density);
      float t0, t1;
      t.get(t0, t1);
      const Pair minus(-copysignf(t0, v[i]), -copysignf(t1, v[i + 1]));
      const Pair step(__float_as_int(v[i]) >= 0 ? 1.0f : 0.0f, __float_as_int(v[i + 1]) >= 0 ? 1.0f : 0.0f);
      slope = fma2(density, fma2(Pair(v[i], v[i + 1]), Pair(kInvSqrt2Pi), minus), step);
    }
    mul2(Pair(d[i], d[i + 1]), slope).get(v[i], v[i + 1]);
  }
}

// y = gelu(x); packs x into `in` (PACK_IN) and the rounded y into `out` with
// y's column sums (PACK_OUT; sums may be null).
template <typename T, bool VEC, bool TANH, bool PACK_IN, bool PACK_OUT>
__global__ void __launch_bounds__(kActThreads, resident(VEC, kGeluForwardCtas))
    k_gelu_forward(const T* __restrict__ x, int64_t rs, int64_t cs, ActGeometry g, T* __restrict__ y, Checkpoint in,
                   Checkpoint out, float* __restrict__ sums) {
  const ActLane a = act_lane<VEC>(g);
  ColumnSums column;
  if constexpr (VEC) {
    constexpr int kUnroll = 2;
    const bool in_x = a.col0 < g.cols, in_values = a.col0 < in.ld, in_codes = a.col0 / kGroup < in.lde;
    RowPointer<const T> xp(x, a.r_begin + a.row_lane, rs, a.col0, a.row_lanes);
    RowPointer<T> yp(y, a.r_begin + a.row_lane, g.cols, a.col0, a.row_lanes);
    PackPointer ip(in, a), op(out, a);
    act_rows<kUnroll>(g, a, [&](auto full, int64_t r0) {
      constexpr bool kFull = decltype(full)::value;
      Vec8<T> w[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        memset(&w[u], 0, sizeof(w[u]));
        const T* at = xp.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) vec8_load(at, w[u]);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const bool ok = r0 + u * a.row_lanes + a.row_lane < a.r_end;
        float v[8];
        vec8_unpack(w[u], v);
        if (PACK_IN) pack8<T, kFull>(ip.values.take(), ip.codes.take(), w[u], v, ok, in_values, in_codes);
        gelu_values<TANH>(v);
        vec8_pack(v, w[u]);
        T* at = yp.take();
        if (kFull || (in_x && ok)) vec8_store(at, w[u]);
        if (PACK_OUT) {
          vec8_unpack(w[u], v);
          pack8<T, kFull>(op.values.take(), op.codes.take(), w[u], v, ok, in_values, in_codes);
          column.add(v);
        }
      }
    });
  } else {
    for (int64_t r = a.r_begin + a.row_lane; r - a.row_lane < a.r_end; r += a.row_lanes) {
      const bool ok = r < a.r_end;
      float v[8];
      load_strided(x, r, rs, cs, a.col0, g.cols, ok, v);
      if (PACK_IN) pack_strided<T>(in, r, ok, a.col0, a.lane, v);
      gelu_values<TANH>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(from_f32<T>(v[i]));
      store_strided(y, r, a.col0, g.cols, ok, v);
      if (PACK_OUT) {
        pack_strided<T>(out, r, ok, a.col0, a.lane, v);
        column.add(v);
      }
    }
  }
  if (PACK_OUT && sums != nullptr) write_column_sums<VEC>(g, a, column, sums);
  grid_dep_launch();
}

// dx = delta * gelu'(x^)
template <typename T, bool VEC, bool TANH>
__global__ void __launch_bounds__(kActThreads, resident(VEC, kGeluBackwardCtas))
    k_gelu_backward(const T* __restrict__ delta, int64_t rs, int64_t cs, ActGeometry g, Checkpoint c,
                    T* __restrict__ dx) {
  const ActLane a = act_lane<VEC>(g);
  if constexpr (VEC) {
    constexpr int kUnroll = sizeof(T) == 2 ? kActUnroll : 2;
    const bool in_x = a.col0 < g.cols;
    RowPointer<const T> dp(delta, a.r_begin + a.row_lane, rs, a.col0, a.row_lanes);
    RowPointer<T> op(dx, a.r_begin + a.row_lane, g.cols, a.col0, a.row_lanes);
    PackPointer pp(c, a);
    act_rows<kUnroll>(g, a, [&](auto full, int64_t r0) {
      constexpr bool kFull = decltype(full)::value;
      Vec8<T> d[kUnroll];
      uint2 w[kUnroll];
      uint32_t code[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const T* at = dp.take();
        const int8_t* v = pp.values.take();
        const uint8_t* k = pp.codes.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) {
          vec8_load(at, d[u]);
          w[u] = __ldg(reinterpret_cast<const uint2*>(v));
          code[u] = __ldg(k);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        T* at = op.take();
        if (kFull || (in_x && r0 + u * a.row_lanes + a.row_lane < a.r_end)) {
          float v[8], dv[8];
          unpack8(w[u], code[u], v);
          vec8_unpack(d[u], dv);
          gelu_gradients<TANH>(v, dv);
          vec8_pack(v, d[u]);
          vec8_store(at, d[u]);
        }
      }
    });
  } else {
    for (int64_t r = a.r_begin + a.row_lane; r < a.r_end; r += a.row_lanes) {
      float v[8], d[8];
      unpack_strided(c, r, true, a.col0, g.cols, v);
      load_strided(delta, r, rs, cs, a.col0, g.cols, true, d);
      gelu_gradients<TANH>(v, d);
      store_strided(dx, r, a.col0, g.cols, true, v);
    }
  }
}

}  // namespace smb
