// sm_activation_host.cuh -- launches and C-ABI of the 8-bit activation
// checkpoint operators (sm_activation.cuh, sm_wgrad.cuh).  Part of the single
// translation unit libsandmuon_b200.cu, which includes it last.
#pragma once

#include <atomic>

namespace smb {

static int64_t act_ld(int64_t cols) { return SM_ACTIVATION_LD(cols); }
static int64_t act_lde(int64_t cols) { return SM_ACTIVATION_LDE(cols); }

static int elem_size(int dtype) {
  return dtype == SM_DTYPE_F32 ? 4 : dtype == SM_DTYPE_BF16 || dtype == SM_DTYPE_F16 ? 2 : 0;
}

static bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Contiguous rows every 16-byte access of which is whole and aligned.
static bool vec8_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t rs, int64_t cs) {
  return cs == 1 && cols % 8 == 0 && aligned(x, 16) && (rows <= 1 || (rs * elem_size(dtype)) % 16 == 0);
}

struct ActLaunch {
  ActGeometry g;
  dim3 grid;
  int splits;
};

// Rows that a lane adds to its column sums in FP32 before the FP64 join: about the
// length of the chains of the statistics kernels, whose place these sums take.
constexpr int kSumChain = 128;

// CTAs of 256 threads: strips of up to 256 columns times enough row ranges for
// `ctas` CTAs per SM, each range of whole passes (32 rows by 256 columns).  VEC:
// one wave.  The strided mapping is resident twice per SM and runs two waves:
// 16384 x 1023 BF16 in one wave instead packs in 65 us, not 74, but its GELU of
// 16384 x 1111 FP32 takes 57 us, not 39.
// `sums`: the launch takes column sums.  Two passes then stay in one range, for
// which no second launch has to join them (64 x 768: pack 3.6 us against 4.5,
// GELU 5.9 against 5.7; from three passes on the split is faster: 7.7 against
// 5.7 for GELU), and tall inputs get more ranges.
static ActLaunch act_launch(int64_t rows, int64_t cols, bool vec, int sms, int ctas, bool sums) {
  ActLaunch l;
  const int64_t padded = act_lde(cols) * kGroup;
  int log_lanes = 2;
  while (log_lanes < 5 && (int64_t{8} << log_lanes) < padded) ++log_lanes;
  if (!vec) log_lanes = 5;
  const int64_t strips = cdiv(padded, int64_t{8} << log_lanes);
  const int64_t per_pass = (kActThreads >> log_lanes) * kActUnroll;
  const int64_t want = std::max<int64_t>(1, static_cast<int64_t>(ctas) * sms / strips);
  const int64_t most = sums && rows <= 2 * per_pass ? 1 : cdiv(rows, per_pass);
  int64_t splits = std::min<int64_t>(std::min(want, most), 65535);
  int64_t rows_per_cta = round_up(cdiv(rows, splits), per_pass);
  if (sums)
    rows_per_cta = std::min(rows_per_cta, std::max<int64_t>(kSumChain * (kActThreads >> log_lanes),
                                                            round_up(cdiv(rows, 65535), per_pass)));
  splits = std::max<int64_t>(1, cdiv(rows, rows_per_cta));
  l.g.rows = rows;
  l.g.cols = cols;
  l.g.rows_per_cta = rows_per_cta;
  l.g.log_lanes = log_lanes;
  l.grid = dim3(static_cast<unsigned>(strips), static_cast<unsigned>(splits));
  l.splits = static_cast<int>(splits);
  return l;
}

static int act_shape_check(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return fail(SM_ERR_ARG, "negative shape");
  // strips ride on gridDim.x and TMA coordinates are 32-bit
  if (rows > INT32_MAX || cols > INT32_MAX - 512)
    return fail(SM_ERR_ARG, "an activation checkpoint has fewer than 2^31 rows and columns");
  return SM_OK;
}

static int act_checkpoint_check(const int8_t* values, const uint8_t* exponents) {
  if (values == nullptr || exponents == nullptr) return fail(SM_ERR_ARG, "null checkpoint");
  if (!aligned(values, 16) || !aligned(exponents, 4))
    return fail(SM_ERR_ARG, "checkpoint values must be 16-byte and exponents 4-byte aligned");
  return SM_OK;
}

static Checkpoint act_checkpoint(const int8_t* values, const uint8_t* exponents, int64_t cols) {
  Checkpoint c;
  c.values = const_cast<int8_t*>(values);
  c.codes = const_cast<uint8_t*>(exponents);
  c.ld = act_ld(cols);
  c.lde = act_lde(cols);
  return c;
}

// Where a launch of `l.splits` row ranges writes its column sums.
static int act_sums_target(const ActLaunch& l, float* sums, void* ws, size_t ws_bytes, float** out) {
  *out = sums;
  if (sums == nullptr || l.splits == 1) return SM_OK;
  if (ws == nullptr || ws_bytes < static_cast<size_t>(l.splits) * 2 * l.g.cols * sizeof(float))
    return fail(SM_ERR_WORKSPACE, "column-sum workspace too small");
  *out = static_cast<float*>(ws);
  return SM_OK;
}

static int act_sums_finish(const ActLaunch& l, const float* partials, float* sums, cudaStream_t st) {
  if (sums == nullptr || l.splits == 1) return SM_OK;
  PdlScope pdl(true);
  const int64_t n = 2 * l.g.cols;
  return launch_kernel(k_column_sums_finish, dim3(static_cast<unsigned>(cdiv(n, 32))), dim3(32 * kFinishLanes), 0, st,
                       partials, n, l.splits, sums);
}

template <typename T>
static int pack_run(const T* x, int64_t rs, int64_t cs, bool vec, const ActLaunch& l, const Checkpoint& c,
                    float* sums, float* target, cudaStream_t st) {
  auto kern = sums != nullptr ? (vec ? k_activation_pack<T, true, true> : k_activation_pack<T, false, true>)
                              : (vec ? k_activation_pack<T, true, false> : k_activation_pack<T, false, false>);
  SM_TRY(launch_kernel(kern, l.grid, dim3(kActThreads), 0, st, x, rs, cs, l.g, c, target));
  return act_sums_finish(l, target, sums, st);
}

template <typename T>
static int unpack_run(const ActLaunch& l, const Checkpoint& c, T* out, bool vec, cudaStream_t st) {
  auto kern = vec ? k_activation_unpack<T, true> : k_activation_unpack<T, false>;
  return launch_kernel(kern, l.grid, dim3(kActThreads), 0, st, l.g, c, out);
}

template <typename T, bool VEC, bool TANH>
static int gelu_forward_t(const T* x, int64_t rs, int64_t cs, const ActLaunch& l, T* y, const Checkpoint& in,
                          const Checkpoint& out, float* target, cudaStream_t st) {
  const bool pi = in.values != nullptr, po = out.values != nullptr;
  auto kern = pi ? (po ? k_gelu_forward<T, VEC, TANH, true, true> : k_gelu_forward<T, VEC, TANH, true, false>)
                 : (po ? k_gelu_forward<T, VEC, TANH, false, true> : k_gelu_forward<T, VEC, TANH, false, false>);
  return launch_kernel(kern, l.grid, dim3(kActThreads), 0, st, x, rs, cs, l.g, y, in, out, target);
}

template <typename T>
static int gelu_forward_run(const T* x, int64_t rs, int64_t cs, bool vec, bool tanh_form, const ActLaunch& l, T* y,
                            const Checkpoint& in, const Checkpoint& out, float* sums, float* target,
                            cudaStream_t st) {
  if (tanh_form)
    SM_TRY((vec ? gelu_forward_t<T, true, true>(x, rs, cs, l, y, in, out, target, st)
                : gelu_forward_t<T, false, true>(x, rs, cs, l, y, in, out, target, st)));
  else
    SM_TRY((vec ? gelu_forward_t<T, true, false>(x, rs, cs, l, y, in, out, target, st)
                : gelu_forward_t<T, false, false>(x, rs, cs, l, y, in, out, target, st)));
  return act_sums_finish(l, target, sums, st);
}

template <typename T>
static int gelu_backward_run(const T* d, int64_t rs, int64_t cs, bool vec, bool tanh_form, const ActLaunch& l,
                             const Checkpoint& c, T* dx, cudaStream_t st) {
  auto kern = tanh_form ? (vec ? k_gelu_backward<T, true, true> : k_gelu_backward<T, false, true>)
                        : (vec ? k_gelu_backward<T, true, false> : k_gelu_backward<T, false, false>);
  return launch_kernel(kern, l.grid, dim3(kActThreads), 0, st, d, rs, cs, l.g, c, dx);
}

// ---------------------------------------------------------- weight gradient

// WgradArgs::expired of the launches to come (sm_inject_expired_wait).
static std::atomic<int> g_expired_worker{-1};

// 2-D tensor map over rows of `stride` bytes.
static int make_map_rows(CUtensorMap* m, CUtensorMapDataType type, const void* base, int64_t inner, int64_t outer,
                         int64_t stride, uint32_t box_inner, uint32_t box_outer, bool swizzle) {
  PFN_cuTensorMapEncodeTiled_v12000 enc;
  SM_TRY(get_encode(&enc));
  if (!aligned(base, 16) || stride % 16 != 0) return fail(SM_ERR_ARG, "TMA rows not 16-byte aligned");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SM_ERR_CUDA, "cuTensorMapEncodeTiled failed: " + std::to_string(r));
  return SM_OK;
}

struct WgradGeometry {
  bool direct;         // the cotangent is read in place (16-bit, TMA-aligned rows)
  int planes, bk;
  int64_t plane_ld;    // elements
  int64_t tiles_m, tiles_n, kblocks;
  int workers, shared, parts;  // see WgradArgs
  bool partial;        // some tile is held by several workers
  size_t plane_bytes, partial_bytes;
};

static void wgrad_shares(const WgradGeometry& g, WgradArgs* p) {
  p->tiles = static_cast<int>(g.tiles_m * g.tiles_n);
  p->tiles_n = static_cast<int>(g.tiles_n);
  p->kblocks = static_cast<int>(g.kblocks);
  p->workers = g.workers;
  p->shared = g.shared;
  p->parts = g.parts;
  p->each = g.parts > 0 ? 0 : p->shared * p->kblocks / g.workers;
  p->more = g.parts > 0 ? 0 : p->shared * p->kblocks % g.workers;
}

static int wgrad_geometry(const void* delta, int dtype, int64_t rows, int64_t d_out, int64_t rs, int64_t cs,
                          int64_t d_in, WgradGeometry* g) {
  DeviceInfo* di;
  SM_TRY(current_device_info(&di));
  int pairs = 0;
  SM_TRY(pair_workers(di, &pairs));
  if (pairs <= 0) return fail(SM_ERR_UNSUPPORTED, "no CTA pair of the GEMM fits on this device");
  g->planes = dtype == SM_DTYPE_F32 ? 3 : 1;
  g->bk = g->planes == 3 ? 32 : 64;
  g->direct = dtype != SM_DTYPE_F32 && cs == 1 && aligned(delta, 16) && (rows <= 1 || (rs % 8 == 0 && rs >= d_out));
  g->plane_ld = round_up(d_out, 8);
  g->tiles_m = cdiv(d_out, kWgTileM);
  g->tiles_n = cdiv(d_in, kWgTileN);
  g->kblocks = cdiv(rows, g->bk);
  const int64_t tiles = g->tiles_m * g->tiles_n;
  if (tiles > INT32_MAX / 2) return fail(SM_ERR_ARG, "too many output tiles");
  g->shared = static_cast<int>(tiles % pairs);
  g->parts = 0;
  const int64_t least = kWgMinTokens / g->bk;  // k-blocks of a share
  g->workers = tiles >= pairs ? pairs : static_cast<int>(std::min<int64_t>(pairs, cdiv(tiles * g->kblocks, least)));
  if (g->shared > 0 && tiles < pairs) {
    // Equal parts of each tile leave workers idle but give each worker one
    // tile; stretches across tiles keep all busy but cost most workers a
    // second epilogue, about kWgEpilogueBlocks k-blocks of time.
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(g->workers / tiles, g->kblocks / least));
    const int64_t even = cdiv(g->kblocks, parts);
    const int64_t across = cdiv(tiles * g->kblocks, g->workers) + kWgEpilogueBlocks;
    if (even <= across) g->parts = static_cast<int>(parts), g->workers = static_cast<int>(tiles * parts);
  }
  // WgradArgs counts k-blocks in 32 bits
  if (g->kblocks * std::max(pairs, g->workers) > INT32_MAX)
    return fail(SM_ERR_ARG, "too many rows for a weight gradient");
  WgradArgs p;
  wgrad_shares(*g, &p);
  g->partial = false;
  for (int w = 1; w < g->workers && !g->partial; ++w) g->partial = wgrad_begin(p, w) % p.kblocks != 0;
  g->plane_bytes = g->direct ? 0 : round_up(static_cast<int64_t>(g->planes) * rows * g->plane_ld * 2, 256);
  g->partial_bytes = g->partial ? static_cast<size_t>(2 * g->workers) * kWgPartialFloats * sizeof(float) : 0;
  return SM_OK;
}

template <int PLANES, bool F16, int BK, typename OUT>
static int wgrad_launch(const WgradArgs& p, bool planes, bool partial, cudaStream_t st) {
  using S = WgSmem<PLANES, BK>;
  auto kern = k_wgrad<PLANES, F16, BK, OUT>;
  static bool attr_done[64] = {};
  int dev = 0;
  SM_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(SM_ERR_UNSUPPORTED, "device ordinal out of range");
  if (!attr_done[dev]) {
    SM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal));
    attr_done[dev] = true;
  }
  {
    // after k_wgrad_planes the prologue may overlap its end
    PdlScope pdl(planes);
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    pair_launch_config(&cfg, attr, 2 * p.workers, S::kTotal, st);
    cfg.blockDim = dim3(kWgThreads);
    SM_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  }
  if (!partial) return SM_OK;
  PdlScope pdl(true);
  return launch_kernel(k_wgrad_join<OUT>, dim3(static_cast<unsigned>(p.shared), 64), dim3(256), 0, st, p);
}

template <int PLANES, bool F16, int BK>
static int wgrad_dispatch(int out_dtype, const WgradArgs& p, bool planes, bool partial, cudaStream_t st) {
  if (out_dtype == SM_DTYPE_F32) return wgrad_launch<PLANES, F16, BK, float>(p, planes, partial, st);
  if (out_dtype == SM_DTYPE_BF16) return wgrad_launch<PLANES, F16, BK, __nv_bfloat16>(p, planes, partial, st);
  return wgrad_launch<PLANES, F16, BK, __half>(p, planes, partial, st);
}

}  // namespace smb

using namespace smb;

extern "C" {

size_t sm_activation_sums_workspace_bytes(int64_t n_rows, int64_t n_cols) {
  if (n_rows <= 0 || n_cols <= 0) return 0;
  int sms = 148;
  DeviceInfo* di;
  if (current_device_info(&di) == SM_OK) sms = di->sms;
  constexpr int kCtas = std::max(kPackCtas, kGeluForwardCtas);
  const int splits = std::max(act_launch(n_rows, n_cols, true, sms, kCtas, true).splits,
                              act_launch(n_rows, n_cols, false, sms, kCtas, true).splits);
  return splits == 1 ? 0 : static_cast<size_t>(splits) * 2 * static_cast<size_t>(n_cols) * sizeof(float);
}

int sm_activation_pack(const void* x, int dtype, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                       int64_t col_stride, int8_t* values, uint8_t* exponents, float* sums, void* workspace,
                       size_t workspace_bytes, void* stream) {
  SM_TRY(act_shape_check(n_rows, n_cols));
  if (elem_size(dtype) == 0) return fail(SM_ERR_ARG, "activations are packed from F32, BF16 or F16");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_rows == 0 || n_cols == 0) {
    if (sums != nullptr && n_cols > 0) SM_CUDA(cudaMemsetAsync(sums, 0, sizeof(float) * 2 * n_cols, st));
    return SM_OK;
  }
  if (x == nullptr) return fail(SM_ERR_ARG, "null input");
  SM_TRY(act_checkpoint_check(values, exponents));
  DeviceInfo* di;
  SM_TRY(current_device_info(&di));
  const bool vec = vec8_rows(x, dtype, n_rows, n_cols, row_stride, col_stride);
  const ActLaunch l = act_launch(n_rows, n_cols, vec, di->sms, kPackCtas, sums != nullptr);
  const Checkpoint c = act_checkpoint(values, exponents, n_cols);
  float* target = nullptr;
  SM_TRY(act_sums_target(l, sums, workspace, workspace_bytes, &target));
  if (dtype == SM_DTYPE_F32)
    return pack_run(static_cast<const float*>(x), row_stride, col_stride, vec, l, c, sums, target, st);
  if (dtype == SM_DTYPE_BF16)
    return pack_run(static_cast<const __nv_bfloat16*>(x), row_stride, col_stride, vec, l, c, sums, target, st);
  return pack_run(static_cast<const __half*>(x), row_stride, col_stride, vec, l, c, sums, target, st);
}

int sm_activation_unpack(const int8_t* values, const uint8_t* exponents, int64_t n_rows, int64_t n_cols, void* out,
                         int dtype, void* stream) {
  SM_TRY(act_shape_check(n_rows, n_cols));
  if (elem_size(dtype) == 0) return fail(SM_ERR_ARG, "activations are unpacked to F32, BF16 or F16");
  if (n_rows == 0 || n_cols == 0) return SM_OK;
  if (out == nullptr) return fail(SM_ERR_ARG, "null output");
  SM_TRY(act_checkpoint_check(values, exponents));
  DeviceInfo* di;
  SM_TRY(current_device_info(&di));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vec = vec8_rows(out, dtype, n_rows, n_cols, n_cols, 1);
  const ActLaunch l = act_launch(n_rows, n_cols, vec, di->sms, kUnpackCtas, false);
  const Checkpoint c = act_checkpoint(values, exponents, n_cols);
  if (dtype == SM_DTYPE_F32) return unpack_run(l, c, static_cast<float*>(out), vec, st);
  if (dtype == SM_DTYPE_BF16) return unpack_run(l, c, static_cast<__nv_bfloat16*>(out), vec, st);
  return unpack_run(l, c, static_cast<__half*>(out), vec, st);
}

int sm_gelu_forward(const void* x, int dtype, int64_t n_rows, int64_t n_cols, int64_t row_stride, int64_t col_stride,
                    int form, void* y, int8_t* in_values, uint8_t* in_exponents, int8_t* out_values,
                    uint8_t* out_exponents, float* sums, void* workspace, size_t workspace_bytes, void* stream) {
  SM_TRY(act_shape_check(n_rows, n_cols));
  if (elem_size(dtype) == 0) return fail(SM_ERR_ARG, "GELU takes F32, BF16 or F16");
  if (form != SM_GELU_ERF && form != SM_GELU_TANH) return fail(SM_ERR_ARG, "unknown GELU form");
  if (sums != nullptr && out_values == nullptr) return fail(SM_ERR_ARG, "column sums go with a packed output");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_rows == 0 || n_cols == 0) {
    if (sums != nullptr && n_cols > 0) SM_CUDA(cudaMemsetAsync(sums, 0, sizeof(float) * 2 * n_cols, st));
    return SM_OK;
  }
  if (x == nullptr || y == nullptr) return fail(SM_ERR_ARG, "null input or output");
  if (in_values != nullptr || in_exponents != nullptr) SM_TRY(act_checkpoint_check(in_values, in_exponents));
  if (out_values != nullptr || out_exponents != nullptr) SM_TRY(act_checkpoint_check(out_values, out_exponents));
  DeviceInfo* di;
  SM_TRY(current_device_info(&di));
  const bool vec = vec8_rows(x, dtype, n_rows, n_cols, row_stride, col_stride) &&
                   vec8_rows(y, dtype, n_rows, n_cols, n_cols, 1);
  const ActLaunch l = act_launch(n_rows, n_cols, vec, di->sms, kGeluForwardCtas, sums != nullptr);
  const Checkpoint in = act_checkpoint(in_values, in_exponents, n_cols);
  const Checkpoint out = act_checkpoint(out_values, out_exponents, n_cols);
  float* target = nullptr;
  SM_TRY(act_sums_target(l, sums, workspace, workspace_bytes, &target));
  const bool th = form == SM_GELU_TANH;
  if (dtype == SM_DTYPE_F32)
    return gelu_forward_run(static_cast<const float*>(x), row_stride, col_stride, vec, th, l, static_cast<float*>(y),
                            in, out, sums, target, st);
  if (dtype == SM_DTYPE_BF16)
    return gelu_forward_run(static_cast<const __nv_bfloat16*>(x), row_stride, col_stride, vec, th, l,
                            static_cast<__nv_bfloat16*>(y), in, out, sums, target, st);
  return gelu_forward_run(static_cast<const __half*>(x), row_stride, col_stride, vec, th, l, static_cast<__half*>(y),
                          in, out, sums, target, st);
}

int sm_gelu_backward(const void* delta, int dtype, int64_t n_rows, int64_t n_cols, int64_t row_stride,
                     int64_t col_stride, const int8_t* values, const uint8_t* exponents, int form, void* dx,
                     void* stream) {
  SM_TRY(act_shape_check(n_rows, n_cols));
  if (elem_size(dtype) == 0) return fail(SM_ERR_ARG, "GELU takes F32, BF16 or F16");
  if (form != SM_GELU_ERF && form != SM_GELU_TANH) return fail(SM_ERR_ARG, "unknown GELU form");
  if (n_rows == 0 || n_cols == 0) return SM_OK;
  if (delta == nullptr || dx == nullptr) return fail(SM_ERR_ARG, "null input or output");
  SM_TRY(act_checkpoint_check(values, exponents));
  DeviceInfo* di;
  SM_TRY(current_device_info(&di));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vec = vec8_rows(delta, dtype, n_rows, n_cols, row_stride, col_stride) &&
                   vec8_rows(dx, dtype, n_rows, n_cols, n_cols, 1);
  const ActLaunch l = act_launch(n_rows, n_cols, vec, di->sms, kGeluBackwardCtas, false);
  const Checkpoint c = act_checkpoint(values, exponents, n_cols);
  const bool th = form == SM_GELU_TANH;
  if (dtype == SM_DTYPE_F32)
    return gelu_backward_run(static_cast<const float*>(delta), row_stride, col_stride, vec, th, l, c,
                             static_cast<float*>(dx), st);
  if (dtype == SM_DTYPE_BF16)
    return gelu_backward_run(static_cast<const __nv_bfloat16*>(delta), row_stride, col_stride, vec, th, l, c,
                             static_cast<__nv_bfloat16*>(dx), st);
  return gelu_backward_run(static_cast<const __half*>(delta), row_stride, col_stride, vec, th, l, c,
                           static_cast<__half*>(dx), st);
}

size_t sm_weight_gradient_workspace_bytes(const void* delta, int dtype, int64_t n_rows, int64_t d_out,
                                          int64_t row_stride, int64_t col_stride, int64_t d_in) {
  if (n_rows <= 0 || d_out <= 0 || d_in <= 0 || elem_size(dtype) == 0) return 0;
  if (act_shape_check(n_rows, d_in) != SM_OK || act_shape_check(n_rows, d_out) != SM_OK) return 0;
  WgradGeometry g;
  if (wgrad_geometry(delta, dtype, n_rows, d_out, row_stride, col_stride, d_in, &g) != SM_OK) return 0;
  return g.plane_bytes + g.partial_bytes;
}

int sm_weight_gradient(const void* delta, int dtype, int64_t n_rows, int64_t d_out, int64_t row_stride,
                       int64_t col_stride, const int8_t* values, const uint8_t* exponents, int64_t d_in, void* out,
                       int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  SM_TRY(act_shape_check(n_rows, d_in));
  SM_TRY(act_shape_check(n_rows, d_out));
  if (elem_size(dtype) == 0 || elem_size(out_dtype) == 0)
    return fail(SM_ERR_ARG, "weight gradients take and give F32, BF16 or F16");
  if (d_out == 0 || d_in == 0) return SM_OK;
  if (out == nullptr) return fail(SM_ERR_ARG, "null output");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (n_rows == 0) {
    SM_CUDA(cudaMemsetAsync(out, 0, static_cast<size_t>(elem_size(out_dtype)) * d_out * d_in, st));
    return SM_OK;
  }
  if (delta == nullptr) return fail(SM_ERR_ARG, "null cotangent");
  SM_TRY(act_checkpoint_check(values, exponents));
  WgradGeometry g;
  SM_TRY(wgrad_geometry(delta, dtype, n_rows, d_out, row_stride, col_stride, d_in, &g));
  if (g.plane_bytes + g.partial_bytes > 0 &&
      (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < g.plane_bytes + g.partial_bytes))
    return fail(SM_ERR_WORKSPACE, "weight gradient workspace too small or not 256-byte aligned");
  WgradArgs p;
  memset(&p, 0, sizeof(p));
  const int64_t plane_elems = n_rows * g.plane_ld;
  const uint8_t* base = static_cast<const uint8_t*>(delta);
  // a single row has no stride of its own
  int64_t stride = 2 * (n_rows == 1 ? g.plane_ld : row_stride);
  if (!g.direct) {
    uint16_t* planes = static_cast<uint16_t*>(workspace);
    const dim3 block(32, 8);
    const int64_t strips = cdiv(g.plane_ld, 32 * 8);
    const dim3 grid(static_cast<unsigned>(strips),
                    static_cast<unsigned>(std::min<int64_t>(cdiv(n_rows, 8), std::max<int64_t>(1, 16 * 148 / strips))));
    if (dtype == SM_DTYPE_F32) {
      auto kern = vec8_rows(delta, dtype, n_rows, d_out, row_stride, col_stride) ? k_wgrad_planes<float, 3, true>
                                                                                : k_wgrad_planes<float, 3, false>;
      SM_TRY(launch_kernel(kern, grid, block, 0, st, static_cast<const float*>(delta), row_stride, col_stride, n_rows,
                           d_out, g.plane_ld, planes));
    } else {
      SM_TRY(launch_kernel(k_wgrad_planes<__half, 1, false>, grid, block, 0, st, static_cast<const __half*>(delta),
                           row_stride, col_stride, n_rows, d_out, g.plane_ld, planes));
    }
    base = static_cast<const uint8_t*>(workspace);
    stride = g.plane_ld * 2;
  }
  for (int j = 0; j < g.planes; ++j)
    SM_TRY(make_map_rows(&p.a[j], CU_TENSOR_MAP_DATA_TYPE_UINT16, base + 2 * j * plane_elems, d_out, n_rows, stride, 64,
                         static_cast<uint32_t>(g.bk), true));
  SM_TRY(make_map_rows(&p.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, values, act_ld(d_in), n_rows, act_ld(d_in), 128,
                       static_cast<uint32_t>(g.bk), false));
  p.codes = exponents;
  p.lde = act_lde(d_in);
  p.rows = static_cast<int>(n_rows);
  p.d_out = static_cast<int>(d_out);
  p.d_in = static_cast<int>(d_in);
  wgrad_shares(g, &p);
  p.out = out;
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + g.plane_bytes);
  p.expired = g_expired_worker.load();
  p.vec_out = aligned(out, 16) && (d_in * elem_size(out_dtype)) % 16 == 0;
  if (dtype == SM_DTYPE_F32) return wgrad_dispatch<3, false, 32>(out_dtype, p, !g.direct, g.partial, st);
  if (dtype == SM_DTYPE_BF16) return wgrad_dispatch<1, false, 64>(out_dtype, p, !g.direct, g.partial, st);
  return wgrad_dispatch<1, true, 64>(out_dtype, p, !g.direct, g.partial, st);
}

int sm_inject_expired_wait(int worker) {
  g_expired_worker.store(worker < 0 ? -1 : worker);
  return SM_OK;
}

}  // extern "C"
