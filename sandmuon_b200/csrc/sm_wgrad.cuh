// sm_wgrad.cuh -- weight gradient from an 8-bit activation checkpoint:
//
//   dW[o, i] = sum_t delta[t, o] * x^[t, i],   x^[t, i] = q[t, i] * 2^e[t, i / 32]
//
// on sm_100a tensor cores (tcgen05 + TMEM + TMA), the checkpoint dequantised
// on its way into the product.  x^ has 7 significant bits and a power-of-two
// scale, so its 16-bit form is exact; a 16-bit cotangent enters as it is and
// an FP32 one as three BF16 planes of 8 significant bits each (exact: 24 bits
// in all).  Every product is therefore exact and the only rounding is that of
// the FP32 sum.
//
// Both operands have the sum's axis t as their slow dimension, so both are
// MN-major tiles (see Swz).  A CTA pair computes a 256 x 256 tile
// (cta_group::2): each CTA stages 128 delta columns and 128 x^ columns.
//   warp 0       TMA producer: delta tiles (128-byte swizzle, counted on the
//                leader's full barrier) and raw int8 tiles (this CTA's barrier)
//   warp 1       MMA issuer (the leader's thread, for both CTAs)
//   warps 2..5   epilogue: TMEM -> registers -> global
//   warps 6..13  converters: raw int8 tile -> 16-bit x^ in the swizzled layout
//                the MMA reads, then an arrival on the leader's full barrier
// The weight gradients of a transformer layer have few output tiles and a
// long sum (768 x 768 over 16384 tokens: 9 tiles of 256 k-blocks), so the work
// is split along t: worker w of W takes the k-blocks [w N / W, (w + 1) N / W)
// of the N = tiles * k-blocks total.  A tile that one worker covers is stored
// at once; the others leave FP32 partial tiles that k_wgrad_join adds in
// worker order (no atomics: results do not depend on timing).
#pragma once

#include <cuda_fp16.h>

#include "sm_activation.cuh"
#include "sm_common.cuh"

namespace smb {

constexpr int kWgTileM = 256, kWgTileN = 256;  // of a CTA pair
constexpr int kWgConvWarps = 8;
constexpr int kWgEpiWarps = 4;
constexpr int kWgThreads = 64 + 32 * (kWgEpiWarps + kWgConvWarps);
constexpr int kWgPartialFloats = kWgTileM * kWgTileN;
// k-blocks of one worker's share are at least this many (256 tokens), so that
// a short sum is not cut into partial tiles that cost more than they save
constexpr int kWgMinTokens = 256;

constexpr int kStatusTimeoutWgradProducer = 0x131;
constexpr int kStatusTimeoutWgradMma = 0x132;
constexpr int kStatusTimeoutWgradEpilogue = 0x133;
constexpr int kStatusTimeoutWgradConvert = 0x134;

struct WgradArgs {
  CUtensorMap a[3];         // delta planes [t, o]: box 64 x BK, 128-byte swizzle
  CUtensorMap q;            // values [t, ld] int8: box 128 x BK
  const uint8_t* codes;     // [t, lde]
  int64_t lde;
  int rows, d_out, d_in;    // t, o, i
  int tiles_n, kblocks;     // tiles along i; k-blocks of one tile
  int64_t total;            // tiles * kblocks
  int workers;
  void* out;                // [d_out, d_in]
  float* partials;          // [2 * workers, kWgPartialFloats]
  int vec_out;              // rows of `out` take 16-byte stores
};

__host__ __device__ inline int64_t wgrad_begin(int64_t total, int workers, int w) { return total * w / workers; }

// A worker's stretch of k-blocks inside one tile.
struct WgSegment {
  int tile, kb0, kb1;
};

struct WgIter {
  int64_t pos, end;
  int kblocks, index;
  __device__ __forceinline__ WgIter(const WgradArgs& p, int worker)
      : pos(wgrad_begin(p.total, p.workers, worker)),
        end(wgrad_begin(p.total, p.workers, worker + 1)),
        kblocks(p.kblocks),
        index(0) {}
  __device__ __forceinline__ bool valid() const { return pos < end; }
  __device__ __forceinline__ WgSegment get() const {
    WgSegment s;
    s.tile = static_cast<int>(pos / kblocks);
    s.kb0 = static_cast<int>(pos - static_cast<int64_t>(s.tile) * kblocks);
    s.kb1 = static_cast<int>(min(static_cast<int64_t>(kblocks), s.kb0 + (end - pos)));
    return s;
  }
  __device__ __forceinline__ void next(const WgSegment& s) {
    pos += s.kb1 - s.kb0;
    ++index;
  }
};

template <int PLANES, int BK>
struct WgSmem {
  static constexpr int kABytes = 128 * BK * 2;    // one plane of this CTA's delta columns
  static constexpr int kBBytes = 128 * BK * 2;    // this CTA's x^ columns
  static constexpr int kRawBytes = 128 * BK;
  static constexpr int kStageBytes = PLANES * kABytes + kBBytes + kRawBytes;
  static constexpr int kStagingBytes = kWgEpiWarps * 32 * 33 * 4;
  static constexpr int kFit = (232448 - 1024 - 256 - kStagingBytes) / kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBarrierBytes = (3 * kStages + 4) * 8 + 16;
  static constexpr int kTotal = kStages * kStageBytes + kBarrierBytes + kStagingBytes + 1024;
  static_assert(kTotal <= 232448 && kStages >= 2, "shared memory budget");
};

// mbar_wait whose success also acquires the cluster peer's generic writes
// (the converters' tiles).
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  const uint64_t start = globaltimer_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i) {
      uint32_t ok;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}\n"
          : "=r"(ok)
          : "r"(bar), "r"(parity)
          : "memory");
      if (ok) return true;
    }
    if (abort_flag != nullptr && *abort_flag != 0) return false;
    if (globaltimer_ns() - start > kWaitTimeoutNs) {
      atomicExch(&g_status, code);
      if (abort_flag != nullptr) *abort_flag = code;
      return false;
    }
  }
}

// Instruction descriptor with both operands MN-major; F16 or BF16.
__host__ __device__ constexpr uint32_t wgrad_idesc(bool f16) {
  return f16 ? umma_idesc_bf16(kWgTileM, kWgTileN, true, true) & ~((1u << 7) | (1u << 10))
             : umma_idesc_bf16(kWgTileM, kWgTileN, true, true);
}

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 2^e (NaN for code 255) twice in 16-bit halves.  A BF16's exponent field is
// FP32's.
template <bool F16>
__device__ __forceinline__ uint32_t scale_pair(uint32_t code) {
  if (F16) {
    const uint32_t h = __half_as_ushort(__float2half_rn(code_scale(code)));
    return h | (h << 16);
  }
  const uint32_t h = code == kCodeNan ? 0x7fffu : code << 7;
  return h | (h << 16);
}

// Four int8 values -> four 16-bit x^ (two words), exactly.
//   F16:  the byte q + 128 in the mantissa of 1024 gives 1152 + q.
//   BF16: 7 mantissa bits hold only q's low 7 bits: 128 + (q & 127), from
//         which 128 or, for a negative q, 256 is taken.  Both constants come
//         from 0x4300 by setting the sign bit of q as the exponent's lowest bit.
template <bool F16>
__device__ __forceinline__ uint2 dequant4(uint32_t w, uint32_t scale) {
  if (F16) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t k = 0x64806480u;  // 1152
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    return make_uint2(mul_f16x2(sub_f16x2(a, k), scale), mul_f16x2(sub_f16x2(b, k), scale));
  }
  const uint32_t a = __byte_perm(w, 0u, 0x4140), b = __byte_perm(w, 0u, 0x4342);
  const uint32_t m = 0x43004300u;
  return make_uint2(mul_bf16x2(sub_bf16x2((a & 0x007f007fu) | m, (a & 0x00800080u) | m), scale),
                    mul_bf16x2(sub_bf16x2((b & 0x007f007fu) | m, (b & 0x00800080u) | m), scale));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// 2-D load into this CTA's shared memory counted on a shared::cluster barrier
// (the leader's).  Plain (non-multicast) form.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* map, uint32_t bar_cluster, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}

// A row of up to 32 columns of the result, from a staging tile padded to 33.
template <typename OUT>
__device__ __forceinline__ void store_tile32(OUT* out, int64_t ld, int row0, int col0, int rows, int cols,
                                             const float* stg, int lane, bool vec) {
  constexpr int kVec = 16 / sizeof(OUT);
  constexpr int kLanes = 32 / kVec;  // lanes per row
  if (vec && col0 + 32 <= cols) {
#pragma unroll
    for (int it = 0; it < kLanes; ++it) {
      const int rr = it * (32 / kLanes) + lane / kLanes;
      const int c = (lane % kLanes) * kVec;
      if (row0 + rr >= rows) continue;
      OUT v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = from_f32<OUT>(stg[rr * 33 + c + e]);
      uint4 w;
      memcpy(&w, v, 16);
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + rr) * ld + col0 + c) = w;
    }
  } else if (col0 + lane < cols) {
#pragma unroll 4
    for (int rr = 0; rr < 32; ++rr)
      if (row0 + rr < rows) out[static_cast<int64_t>(row0 + rr) * ld + col0 + lane] = from_f32<OUT>(stg[rr * 33 + lane]);
  }
}

// Partial tiles are laid out as the epilogue holds them: [cta][lane quarter]
// [32-column chunk][4-column step][lane][4], so that a warp's accesses are
// 512 contiguous bytes.
__device__ __forceinline__ int64_t partial_offset(int cta, int quarter, int chunk, int step, int lane) {
  return ((((static_cast<int64_t>(cta) * 4 + quarter) * (kWgTileN / 32) + chunk) * 8 + step) * 32 + lane) * 4;
}

template <int PLANES, bool F16, int BK, typename OUT>
__global__ void __launch_bounds__(kWgThreads, 1) k_wgrad(const __grid_constant__ WgradArgs p) {
  using S = WgSmem<PLANES, BK>;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kChunkBytes = Swz::chunk_bytes(BK);
  constexpr uint32_t kIdesc = wgrad_idesc(F16);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kStages + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* staging = reinterpret_cast<float*>(smem + kStages * S::kStageBytes + S::kBarrierBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int worker = static_cast<int>(blockIdx.x) / 2;
  const uint32_t bar_base = smem_u32(bars);
  // full: delta bytes of both CTAs + the converters of both (leader's only);
  // raw: this CTA's int8 tile; empty: the MMAs that read the slot are done
  auto bar_full = [&](int s) { return bar_base + 8u * s; };
  auto bar_raw = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto bar_empty = [&](int s) { return bar_base + 8u * (2 * kStages + s); };
  auto bar_tfull = [&](int a) { return bar_base + 8u * (3 * kStages + a); };
  auto bar_tempty = [&](int a) { return bar_base + 8u * (3 * kStages + 2 + a); };
  auto slot_a = [&](int s) { return smem_u32(smem + s * S::kStageBytes); };
  auto slot_b = [&](int s) { return smem_u32(smem + s * S::kStageBytes + PLANES * S::kABytes); };
  auto slot_raw = [&](int s) { return smem_u32(smem + s * S::kStageBytes + PLANES * S::kABytes + S::kBBytes); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1 + 2 * kWgConvWarps);
      mbar_init(bar_raw(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull(a), 1);
      mbar_init(bar_tempty(a), 2 * kWgEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tmem_alloc_pair(smem_u32(tmem_slot), 2 * kWgTileN);
  }
  if (warp == 0 && lane == 0) {
#pragma unroll
    for (int j = 0; j < PLANES; ++j) tma_prefetch_desc(&p.a[j]);
    tma_prefetch_desc(&p.q);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  grid_dep_wait();
  grid_dep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (WgIter it(p, worker); it.valid() && ok;) {
        const WgSegment s = it.get();
        const int mc = s.tile / p.tiles_n * kWgTileM + static_cast<int>(rank) * 128;
        const int nc = s.tile % p.tiles_n * kWgTileN + static_cast<int>(rank) * 128;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!mbar_wait(bar_empty(stage), phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(bar_raw(stage), S::kRawBytes);
          tma_load_2d(slot_raw(stage), &p.q, bar_raw(stage), nc, kb * BK);
          const uint32_t fb = mapa_shared(bar_full(stage), 0);
          if (rank == 0) mbar_arrive_expect_tx(bar_full(stage), 2 * PLANES * S::kABytes);
#pragma unroll
          for (int j = 0; j < PLANES; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tma_load_2d_pair(slot_a(stage) + j * S::kABytes + h * kChunkBytes, &p.a[j], fb, mc + 64 * h, kb * BK);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        it.next(s);
      }
      // every slot's last release (a commit of the leader) has arrived before
      // this CTA may leave
      for (int i = 0; i < kStages && ok; ++i) {
        ok = mbar_wait(bar_empty(stage), phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (WgIter it(p, worker); it.valid() && ok; ++local) {
        const WgSegment s = it.get();
        const int acc = local & 1;
        if (!mbar_wait(bar_tempty(acc), ((local >> 1) & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kWgTileN);
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!mbar_wait_cluster(bar_full(stage), phase, abort_flag, kStatusTimeoutWgradMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < BK / 16; ++ks) {
            const uint64_t b = umma_desc(slot_b(stage) + ks * Swz::kMnStepBytes, kChunkBytes, Swz::kSbo, Swz::kLayout);
#pragma unroll
            for (int j = PLANES - 1; j >= 0; --j) {  // smallest plane first
              const uint64_t a = umma_desc(slot_a(stage) + j * S::kABytes + ks * Swz::kMnStepBytes, kChunkBytes,
                                           Swz::kSbo, Swz::kLayout);
              umma_bf16_pair(d_tmem, a, b, kIdesc, (kb > s.kb0 || ks > 0 || j < PLANES - 1) ? 1u : 0u);
            }
          }
          umma_commit_pair(bar_empty(stage), 0x3);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(bar_tfull(acc), 0x3);
        it.next(s);
      }
      for (int i = 0; i < 2 && ok; ++i, ++local)
        ok = mbar_wait(bar_tempty(local & 1), ((local >> 1) & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
    }
  } else if (warp < 2 + kWgEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;
    const uint32_t tempty0 = mapa_shared(bar_tempty(0), 0);
    float* stg = staging + (warp - 2) * 32 * 33;
    int local = 0;
    for (WgIter it(p, worker); it.valid(); ++local) {
      const WgSegment s = it.get();
      const int acc = local & 1;
      const bool ready = mbar_wait(bar_tfull(acc), (local >> 1) & 1, abort_flag, kStatusTimeoutWgradEpilogue);
      if (!__all_sync(0xffffffffu, ready)) break;
      tc_fence_after();
      const bool whole = s.kb0 == 0 && s.kb1 == p.kblocks;
      const int row0 = s.tile / p.tiles_n * kWgTileM + static_cast<int>(rank) * 128 + quarter * 32;
      const int colt = s.tile % p.tiles_n * kWgTileN;
      float* part = p.partials + static_cast<int64_t>(2 * worker + (it.index > 0 ? 1 : 0)) * kWgPartialFloats;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * kWgTileN);
#pragma unroll 1
      for (int j = 0; j < kWgTileN / 32; ++j) {
        uint32_t r[32];
        tmem_ld_32x32(t_row + j * 32, r);
        tmem_wait_ld();
        if (j == kWgTileN / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * acc);
        }
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(part + partial_offset(rank, quarter, j, c, lane)) =
                make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) stg[lane * 33 + c] = __uint_as_float(r[c]);
          __syncwarp();
          store_tile32(static_cast<OUT*>(p.out), p.d_in, row0, colt + 32 * j, p.d_out, p.d_in, stg, lane,
                       p.vec_out != 0);
          __syncwarp();
        }
      }
      it.next(s);
    }
  } else {
    // ---------------------------------------------------------- converters
    // A task is 16 columns of one token: 8 lanes cover a token's 128 columns.
    constexpr int kTasks = BK * 8 / (32 * kWgConvWarps);
    static_assert(kTasks * 32 * kWgConvWarps == BK * 8, "whole tasks per thread");
    const int tid = threadIdx.x - 32 * (2 + kWgEpiWarps);
    const int seg = tid & 7;
    const uint32_t full0 = mapa_shared(bar_base, 0);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (WgIter it(p, worker); it.valid() && ok;) {
      const WgSegment s = it.get();
      const int64_t g = (s.tile % p.tiles_n * kWgTileN + static_cast<int>(rank) * 128 + seg * 16) / kGroup;
      const bool g_ok = g < p.lde;
      auto code_of = [&](int kb, int t) -> uint32_t {
        const int r = kb * BK + t * (BK / kTasks) + (tid >> 3);
        return g_ok && r < p.rows ? p.codes[static_cast<int64_t>(r) * p.lde + g] : 127u;
      };
      uint32_t code[kTasks];
#pragma unroll
      for (int t = 0; t < kTasks; ++t) code[t] = code_of(s.kb0, t);
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        uint32_t next[kTasks];
#pragma unroll
        for (int t = 0; t < kTasks; ++t) next[t] = kb + 1 < s.kb1 ? code_of(kb + 1, t) : 127u;
        ok = mbar_wait(bar_raw(stage), phase, abort_flag, kStatusTimeoutWgradConvert);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int t = 0; t < kTasks; ++t) {
          const int k = t * (BK / kTasks) + (tid >> 3);
          const uint4 w = lds128(slot_raw(stage) + k * 128 + seg * 16);
          const uint32_t sc = scale_pair<F16>(code[t]);
          const uint2 v0 = dequant4<F16>(w.x, sc), v1 = dequant4<F16>(w.y, sc);
          const uint2 v2 = dequant4<F16>(w.z, sc), v3 = dequant4<F16>(w.w, sc);
          const uint32_t row = slot_b(stage) + (seg >> 2) * kChunkBytes + k * 128;
          const uint32_t u = (seg & 3) * 2;
          const uint32_t at0 = row + ((u ^ (k & 7)) << 4), at1 = row + (((u + 1) ^ (k & 7)) << 4);
          // lanes of the two chunks store their halves in opposite order: no bank is hit twice
          const bool flip = (seg & 4) != 0;
          sts128(flip ? at1 : at0, flip ? v2.x : v0.x, flip ? v2.y : v0.y, flip ? v3.x : v1.x, flip ? v3.y : v1.y);
          sts128(flip ? at0 : at1, flip ? v0.x : v2.x, flip ? v0.y : v2.y, flip ? v1.x : v3.x, flip ? v1.y : v3.y);
          code[t] = next[t];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(full0 + 8u * stage);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      it.next(s);
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * kWgTileN);
  }
}

// Adds the partial tiles of every tile that no single worker covers, in worker
// order.  One warp per 32 x 32 block; grid (tile, 64 blocks / 4 warps).
template <typename OUT>
__global__ void __launch_bounds__(128) k_wgrad_join(const __grid_constant__ WgradArgs p) {
  __shared__ float sh[4][32 * 33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x;
  const int64_t k_begin = static_cast<int64_t>(tile) * p.kblocks, k_end = k_begin + p.kblocks;
  // the worker that holds a k-block b: the largest w with begin(w) <= b
  auto worker_of = [&](int64_t b) {
    int w = static_cast<int>((b * p.workers) / p.total);
    while (w + 1 < p.workers && wgrad_begin(p.total, p.workers, w + 1) <= b) ++w;
    while (w > 0 && wgrad_begin(p.total, p.workers, w) > b) --w;
    return w;
  };
  const int w0 = worker_of(k_begin), w1 = worker_of(k_end - 1);
  grid_dep_wait();
  if (w0 == w1) return;
  const int block = blockIdx.y * 4 + warp;  // [cta][quarter][chunk]
  const int cta = block >> 5, quarter = (block >> 3) & 3, chunk = block & 7;
  const int row0 = tile / p.tiles_n * kWgTileM + cta * 128 + quarter * 32;
  const int col0 = tile % p.tiles_n * kWgTileN + chunk * 32;
  if (row0 >= p.d_out || col0 >= p.d_in) return;
  float4 acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int w = w0; w <= w1; ++w) {
    // a worker's first segment is in its slot 0, a later one (its last) in slot 1
    const bool first = wgrad_begin(p.total, p.workers, w) >= k_begin;
    const float* part = p.partials + static_cast<int64_t>(2 * w + (first ? 0 : 1)) * kWgPartialFloats;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float4 v = *reinterpret_cast<const float4*>(part + partial_offset(cta, quarter, chunk, c, lane));
      acc[c].x += v.x;
      acc[c].y += v.y;
      acc[c].z += v.z;
      acc[c].w += v.w;
    }
  }
  float* stg = sh[warp];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    stg[lane * 33 + 4 * c] = acc[c].x;
    stg[lane * 33 + 4 * c + 1] = acc[c].y;
    stg[lane * 33 + 4 * c + 2] = acc[c].z;
    stg[lane * 33 + 4 * c + 3] = acc[c].w;
  }
  __syncwarp();
  store_tile32(static_cast<OUT*>(p.out), p.d_in, row0, col0, p.d_out, p.d_in, stg, lane, p.vec_out != 0);
}

// delta [t, o] of any strides -> PLANES dense planes [t, ld] (ld a multiple of
// 8 elements, padding 0).  One plane keeps the type; three split an FP32 value
// by truncation into BF16 parts of 8 significant bits: h + m + l == v exactly
// (short of BF16's underflow).  inf and NaN live in the first plane alone.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256)
    k_wgrad_planes(const T* __restrict__ delta, int64_t rs, int64_t cs, int64_t rows, int64_t cols, int64_t ld,
                   uint16_t* __restrict__ planes) {
  const int64_t n = rows * ld;
  const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t r = i / ld, c = i - r * ld;
    if (PLANES == 1) {
      uint16_t bits = 0;
      if (c < cols) memcpy(&bits, &delta[r * rs + c * cs], 2);
      planes[i] = bits;
    } else {
      float v = c < cols ? to_f32(delta[r * rs + c * cs]) : 0.0f;
#pragma unroll
      for (int j = 0; j < PLANES; ++j) {
        uint32_t top = __float_as_uint(v) & 0xffff0000u;
        const bool special = (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u;
        if (special && v != v) top |= 0x00400000u;  // NaN whatever its payload
        planes[j * n + i] = static_cast<uint16_t>(top >> 16);
        v = special ? 0.0f : v - __uint_as_float(top);
      }
    }
  }
}

}  // namespace smb
