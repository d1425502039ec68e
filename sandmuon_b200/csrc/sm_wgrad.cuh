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
//   warp 0        producer: TMA loads of the delta tiles (128-byte swizzle,
//                 counted on the leader's full barrier) and of the raw int8
//                 tiles, and 4-byte asynchronous copies of their exponent codes
//                 (both counted on this CTA's raw barrier)
//   warp 1        MMA issuer (the leader's thread, for both CTAs)
//   warps 2..9    epilogue: TMEM -> registers -> global
//   warps 10..17  converters: raw int8 tile -> 16-bit x^ in the swizzled layout
//                 the MMA reads, then an arrival on the leader's full barrier
//
// The tensor core's FP32 accumulation truncates, so its error grows with the
// length of a chain of MMAs (7e-6 relative after 1024 steps of 16 tokens).  A
// chain is cut at kWgChain steps: TMEM holds two accumulators, a tile's first
// chain stays in its "home", each later one runs in the other and is added to
// the home by the epilogue warps with a correctly rounded FP32 addition.  A
// tile of a single chain leaves the other accumulator to the next tile, so
// that its epilogue runs beside that tile's MMAs.
// The weight gradients of a transformer layer have few output tiles and a
// long sum (768 x 768 over 16384 tokens: 9 tiles of 256 k-blocks), so work is
// split along t.  Of the output's tiles as many as fill whole waves of the W
// workers (CTA pairs) are computed one per worker, all at the same t, so that
// the waves read each operand from HBM about once; the remaining tiles are
// shared out by k-blocks (WgradArgs::parts).  A worker that holds only a part
// of a tile leaves an FP32 partial tile, and k_wgrad_join adds those in worker
// order (no atomics: results do not depend on timing).
#pragma once

#include <cuda_fp16.h>

#include "sm_activation.cuh"
#include "sm_common.cuh"

namespace smb {

constexpr int kWgTileM = 256, kWgTileN = 256;  // of a CTA pair
constexpr int kWgConvWarps = 8;
constexpr int kWgEpiWarps = 8;
constexpr int kWgChain = 128;  // MMA steps summed by the tensor core alone
constexpr int kWgThreads = 64 + 32 * (kWgEpiWarps + kWgConvWarps);
constexpr int kWgPartialFloats = kWgTileM * kWgTileN;
// k-blocks of one worker's share are at least this many (256 tokens), so that
// a short sum is not cut into partial tiles that cost more than they save
constexpr int kWgMinTokens = 256;
// time of one more epilogue (a 256 KB partial tile) in k-blocks of 64 tokens
constexpr int kWgEpilogueBlocks = 8;

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
  int tiles, tiles_n;       // output tiles; tiles along i
  int kblocks;              // k-blocks of one tile
  int workers;
  int shared;               // tiles 0 .. shared - 1 are shared out by k-blocks
  int parts;                // > 0: into this many equal parts, one per worker; 0: into
                            // equal stretches of all workers, across tile borders
  void* out;                // [d_out, d_in]
  float* partials;          // [2 * workers, kWgPartialFloats]
  int vec_out;              // rows of `out` take 16-byte stores
};

// First k-block (of the shared tiles, end to end) of worker w; w = workers
// gives the end of the last worker's.
__host__ __device__ inline int64_t wgrad_begin(int shared, int parts, int kblocks, int workers, int w) {
  const int64_t total = static_cast<int64_t>(shared) * kblocks;
  if (parts == 0) return total * w / workers;
  return w >= shared * parts ? total
                             : static_cast<int64_t>(w / parts) * kblocks + static_cast<int64_t>(kblocks) * (w % parts) / parts;
}
__device__ __forceinline__ int64_t wgrad_begin(const WgradArgs& p, int w) {
  return wgrad_begin(p.shared, p.parts, p.kblocks, p.workers, w);
}

// A worker's stretch of k-blocks inside one tile.
struct WgSegment {
  int tile, kb0, kb1;
};

// The segments of a worker: its share of the shared tiles, then whole tiles.
struct WgIter {
  int64_t pos, end;
  int kblocks, index, tile, tiles, workers;
  __device__ __forceinline__ WgIter(const WgradArgs& p, int worker)
      : pos(wgrad_begin(p, worker)),
        end(wgrad_begin(p, worker + 1)),
        kblocks(p.kblocks),
        index(0),
        tile(p.shared + worker),
        tiles(p.tiles),
        workers(p.workers) {}
  __device__ __forceinline__ bool valid() const { return pos < end || tile < tiles; }
  __device__ __forceinline__ WgSegment get() const {
    WgSegment s;
    if (pos < end) {
      s.tile = static_cast<int>(pos / kblocks);
      s.kb0 = static_cast<int>(pos - static_cast<int64_t>(s.tile) * kblocks);
      s.kb1 = static_cast<int>(min(static_cast<int64_t>(kblocks), s.kb0 + (end - pos)));
    } else {
      s.tile = tile;
      s.kb0 = 0;
      s.kb1 = kblocks;
    }
    return s;
  }
  __device__ __forceinline__ void next(const WgSegment& s) {
    if (pos < end) {
      pos += s.kb1 - s.kb0;
      ++index;
    } else {
      tile += workers;
    }
  }
};

template <int PLANES, int BK>
struct WgSmem {
  static constexpr int kABytes = 128 * BK * 2;    // one plane of this CTA's delta columns
  static constexpr int kBBytes = 128 * BK * 2;    // this CTA's x^ columns
  static constexpr int kRawBytes = 128 * BK;
  static constexpr int kStageBytes = PLANES * kABytes + kBBytes + kRawBytes;
  static constexpr int kCodeBytes = 4 * BK;       // exponent codes of a raw tile
  static constexpr int kStagingBytes = kWgEpiWarps * 32 * 17 * 4;
  static constexpr int kFit = (232448 - 1024 - 256 - kStagingBytes) / (kStageBytes + kCodeBytes);
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kBarrierBytes = (3 * kStages + 4) * 8 + 16;
  static constexpr int kTotal = kStages * (kStageBytes + kCodeBytes) + kBarrierBytes + kStagingBytes + 1024;
  static constexpr int kChainBlocks = kWgChain / (PLANES * BK / 16);  // k-blocks of one chain
  static_assert(kTotal <= 232448 && kStages >= 2, "shared memory budget");
};

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

// Arrival on a cluster CTA's barrier in the default (CTA) scope.
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// 4 bytes global -> shared (zeros where !ok), completing with the arrival below.
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
// One of the barrier's expected arrivals, once this thread's copies so far are done.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2-D load into this CTA's shared memory counted on a shared::cluster barrier
// (the leader's).  Plain (non-multicast) form.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* map, uint32_t bar_cluster, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(c0), "r"(c1)
      : "memory");
}

// Stores a 32-row, W-column block of the result from a staging tile whose rows
// are padded to W + 1 floats.
template <int W, typename OUT>
__device__ __forceinline__ void store_block(OUT* out, int64_t ld, int row0, int col0, int rows, int cols,
                                            const float* stg, int lane, bool vec) {
  constexpr int kVec = 16 / sizeof(OUT);
  constexpr int kLanes = W / kVec;       // lanes per row
  constexpr int kRows = 32 / kLanes;     // rows per pass
  if (vec && col0 + W <= cols) {
#pragma unroll
    for (int it = 0; it < 32 / kRows; ++it) {
      const int rr = it * kRows + lane / kLanes;
      const int c = (lane % kLanes) * kVec;
      if (row0 + rr >= rows) continue;
      OUT v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = from_f32<OUT>(stg[rr * (W + 1) + c + e]);
      uint4 w;
      memcpy(&w, v, 16);
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row0 + rr) * ld + col0 + c) = w;
    }
  } else {
    constexpr int kPer = 32 / W;  // rows per pass
    const int c = lane % W;
#pragma unroll 4
    for (int rr = lane / W; rr < 32; rr += kPer)
      if (row0 + rr < rows && col0 + c < cols)
        out[static_cast<int64_t>(row0 + rr) * ld + col0 + c] = from_f32<OUT>(stg[rr * (W + 1) + c]);
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
  uint8_t* code_slots = reinterpret_cast<uint8_t*>(staging) + S::kStagingBytes;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int worker = static_cast<int>(blockIdx.x) / 2;
  const uint32_t bar_base = smem_u32(bars);
  // full: delta bytes of both CTAs + the converters of both (leader's only);
  // raw: this CTA's int8 tile and its codes; empty: the MMAs that read the slot are done
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
      mbar_init(bar_raw(s), 1 + 32);
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
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (WgIter it(p, worker); it.valid() && ok;) {
      const WgSegment s = it.get();
      const int mc = s.tile / p.tiles_n * kWgTileM + static_cast<int>(rank) * 128;
      const int nc = s.tile % p.tiles_n * kWgTileN + static_cast<int>(rank) * 128;
      const bool c_ok = nc / kGroup < p.lde;
      for (int kb = s.kb0; kb < s.kb1; ++kb) {
        ok = mbar_wait(bar_empty(stage), phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (lane == 0) {
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
        }
        // codes outside the checkpoint become 0: their values are 0 as well
#pragma unroll
        for (int t = 0; t < BK / 32; ++t) {
          const int k = t * 32 + lane, r = kb * BK + k;
          const bool r_ok = c_ok && r < p.rows;
          cp_async4(smem_u32(code_slots + stage * S::kCodeBytes) + 4 * k,
                    p.codes + (r_ok ? static_cast<int64_t>(r) * p.lde + nc / kGroup : 0), r_ok);
        }
        cp_async_arrive(bar_raw(stage));
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
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    if (lane == 0 && rank == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int home = 0;
      uint32_t uses0 = 0, uses1 = 0;  // chains that ran in each accumulator
      bool ok = true;
      for (WgIter it(p, worker); it.valid() && ok; home ^= 1) {
        const WgSegment s = it.get();
        for (int begin = s.kb0; begin < s.kb1 && ok; begin += S::kChainBlocks) {
          const int end = min(begin + S::kChainBlocks, s.kb1);
          const int acc = begin == s.kb0 ? home : home ^ 1;
          const uint32_t uses = acc ? uses1++ : uses0++;
          if (!mbar_wait(bar_tempty(acc), (uses & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kWgTileN);
          for (int kb = begin; kb < end; ++kb) {
            if (!mbar_wait(bar_full(stage), phase, abort_flag, kStatusTimeoutWgradMma)) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks) {
              const uint64_t b =
                  umma_desc(slot_b(stage) + ks * Swz::kMnStepBytes, kChunkBytes, Swz::kSbo, Swz::kLayout);
#pragma unroll
              for (int j = PLANES - 1; j >= 0; --j) {  // smallest plane first
                const uint64_t a = umma_desc(slot_a(stage) + j * S::kABytes + ks * Swz::kMnStepBytes, kChunkBytes,
                                             Swz::kSbo, Swz::kLayout);
                umma_bf16_pair(d_tmem, a, b, kIdesc, (kb > begin || ks > 0 || j < PLANES - 1) ? 1u : 0u);
              }
            }
            umma_commit_pair(bar_empty(stage), 0x3);
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) umma_commit_pair(bar_tfull(acc), 0x3);
        }
        it.next(s);
      }
      // both accumulators' last chains have been read by both CTAs
      if (ok) ok = mbar_wait(bar_tempty(0), (uses0 & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
      if (ok) mbar_wait(bar_tempty(1), (uses1 & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
    }
  } else if (warp < 2 + kWgEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;           // TMEM lanes this warp may access
    const int half = (warp - 2) >> 2;       // its 128 of the tile's 256 columns
    const uint32_t tempty0 = mapa_shared(bar_tempty(0), 0);
    float* stg = staging + (warp - 2) * 32 * 17;
    auto release = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0 + 8u * acc);
    };
    int home = 0;
    uint32_t uses0 = 0, uses1 = 0;
    bool ok = true;
    for (WgIter it(p, worker); it.valid() && ok; home ^= 1) {
      const WgSegment s = it.get();
      const bool whole = s.kb0 == 0 && s.kb1 == p.kblocks;
      const int row0 = s.tile / p.tiles_n * kWgTileM + static_cast<int>(rank) * 128 + quarter * 32;
      const int colt = s.tile % p.tiles_n * kWgTileN;
      float* part = p.partials + static_cast<int64_t>(2 * worker + (it.index > 0 ? 1 : 0)) * kWgPartialFloats;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t t_home = t_row + static_cast<uint32_t>(home * kWgTileN);
      const uint32_t t_other = t_row + static_cast<uint32_t>((home ^ 1) * kWgTileN);
      for (int begin = s.kb0; begin < s.kb1; begin += S::kChainBlocks) {
        const bool first = begin == s.kb0, last = begin + S::kChainBlocks >= s.kb1;
        const int acc = first ? home : home ^ 1;
        const uint32_t uses = acc ? uses1++ : uses0++;
        ok = mbar_wait(bar_tfull(acc), uses & 1, abort_flag, kStatusTimeoutWgradEpilogue);
        // the vote keeps the warp converged for the .sync.aligned TMEM accesses
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (first && !last) continue;  // stays in the home accumulator
#pragma unroll 1
        for (int j = 4 * half; j < 4 * half + 4; ++j) {
          uint32_t r[32];
          tmem_ld_32x32(t_home + j * 32, r);
          if (!first) {
            uint32_t x[32];
            tmem_ld_32x32(t_other + j * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) + __uint_as_float(x[c]));
            if (j == 4 * half + 3) release(home ^ 1);
          } else {
            tmem_wait_ld();
          }
          if (!last) {
            tmem_st_32x32(t_home + j * 32, r);
            continue;
          }
          if (j == 4 * half + 3) release(home);
          if (!whole) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(part + partial_offset(rank, quarter, j, c, lane)) =
                  make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int c = 0; c < 16; ++c) stg[lane * 17 + c] = __uint_as_float(r[16 * h + c]);
              __syncwarp();
              store_block<16>(static_cast<OUT*>(p.out), p.d_in, row0, colt + 32 * j + 16 * h, p.d_out, p.d_in, stg,
                              lane, p.vec_out != 0);
              __syncwarp();
            }
          }
        }
        if (!last) tmem_wait_st();
      }
      it.next(s);
    }
  } else {
    // ---------------------------------------------------------- converters
    // A task is 16 columns of one token: 8 lanes cover a token's 128 columns.
    constexpr int kTasks = BK * 8 / (32 * kWgConvWarps);
    static_assert(kTasks * 32 * kWgConvWarps == BK * 8, "whole tasks per thread");
    const int tid = threadIdx.x - 32 * (2 + kWgEpiWarps);
    const int seg = tid & 7, k0 = tid >> 3;  // k0 < 32; a thread's tokens are 32 apart
    const uint32_t full0 = mapa_shared(bar_base, 0);
    // Offsets inside a slot.  Tokens 32 apart have the same swizzle; lanes of
    // the two 64-column chunks store their halves in opposite order, so that
    // no bank is hit twice.
    const bool flip = (seg & 4) != 0;
    const uint32_t u = (seg & 3) * 2;
    const uint32_t in_off = k0 * 128 + seg * 16;
    const uint32_t row_off = (seg >> 2) * kChunkBytes + k0 * 128;
    const uint32_t off0 = row_off + (((u + flip) ^ (k0 & 7)) << 4);
    const uint32_t off1 = row_off + (((u + !flip) ^ (k0 & 7)) << 4);
    const uint32_t code_off = 4 * k0 + (seg >> 1);
    int stage = 0;
    uint32_t phase = 0;
    int64_t left = 0;
    for (WgIter it(p, worker); it.valid();) {
      const WgSegment s = it.get();
      left += s.kb1 - s.kb0;
      it.next(s);
    }
    for (; left > 0; --left) {
      const bool ok = mbar_wait(bar_raw(stage), phase, abort_flag, kStatusTimeoutWgradConvert);
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint32_t raw = slot_raw(stage) + in_off, out = slot_b(stage);
      const uint8_t* codes = code_slots + stage * S::kCodeBytes + code_off;
      uint4 w[kTasks];
      uint32_t code[kTasks];
#pragma unroll
      for (int t = 0; t < kTasks; ++t) {
        w[t] = lds128(raw + t * 32 * 128);
        code[t] = codes[t * 128];
      }
#pragma unroll
      for (int t = 0; t < kTasks; ++t) {
        const uint32_t sc = scale_pair<F16>(code[t]);
        const uint2 a0 = dequant4<F16>(flip ? w[t].z : w[t].x, sc), a1 = dequant4<F16>(flip ? w[t].w : w[t].y, sc);
        const uint2 b0 = dequant4<F16>(flip ? w[t].x : w[t].z, sc), b1 = dequant4<F16>(flip ? w[t].y : w[t].w, sc);
        sts128(out + off0 + t * 32 * 128, a0.x, a0.y, a1.x, a1.y);
        sts128(out + off1 + t * 32 * 128, b0.x, b0.y, b1.x, b1.y);
      }
      // The MMA that these arrivals admit reads this tile through this CTA's
      // own async proxy, to which the fence has made it visible; no data is
      // handed to the peer, so the arrival carries no cluster-scope release
      // (which waits for all of the thread's memory traffic: 1270 us instead
      // of 614 for 16384 x 2048 x 8192).
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(full0 + 8u * stage);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
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

// Adds the partial tiles of the shared tiles, in worker order.  A CTA takes a
// 32 x 32 block of one tile (grid: tiles x 64 blocks), each of its 8 warps 4
// columns of it, so that every access of a partial tile is 512 bytes.
template <typename OUT>
__global__ void __launch_bounds__(256) k_wgrad_join(const __grid_constant__ WgradArgs p) {
  __shared__ float stg[32 * 33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x;
  const int block = blockIdx.y;  // [cta][quarter][chunk]
  const int cta = block >> 5, quarter = (block >> 3) & 3, chunk = block & 7;
  const int row0 = tile / p.tiles_n * kWgTileM + cta * 128 + quarter * 32;
  const int col0 = tile % p.tiles_n * kWgTileN + chunk * 32;
  const int64_t k_begin = static_cast<int64_t>(tile) * p.kblocks;
  // the worker that holds k-block b: the largest w with begin(w) <= b
  auto worker_of = [&](int64_t b) {
    int w = p.parts > 0 ? static_cast<int>(b / p.kblocks * p.parts + b % p.kblocks * p.parts / p.kblocks)
                        : static_cast<int>(b * p.workers / (static_cast<int64_t>(p.shared) * p.kblocks));
    while (w + 1 < p.workers && wgrad_begin(p, w + 1) <= b) ++w;
    while (w > 0 && wgrad_begin(p, w) > b) --w;
    return w;
  };
  const int w0 = worker_of(k_begin), w1 = worker_of(k_begin + p.kblocks - 1);
  // a worker's first segment is in its slot 0, a later one (its last) in slot 1
  const bool late = wgrad_begin(p, w0) < k_begin;
  grid_dep_wait();
  if (w0 == w1 || row0 >= p.d_out || col0 >= p.d_in) return;
  const float* part = p.partials + partial_offset(cta, quarter, chunk, warp, lane);
  float4 acc = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(2 * w0 + (late ? 1 : 0)) * kWgPartialFloats);
#pragma unroll 4
  for (int w = w0 + 1; w <= w1; ++w) {
    const float4 v = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(2 * w) * kWgPartialFloats);
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  stg[lane * 33 + 4 * warp] = acc.x;
  stg[lane * 33 + 4 * warp + 1] = acc.y;
  stg[lane * 33 + 4 * warp + 2] = acc.z;
  stg[lane * 33 + 4 * warp + 3] = acc.w;
  __syncthreads();
  // 4 rows per warp
  OUT* out = static_cast<OUT*>(p.out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = warp * 4 + i;
    if (row0 + r < p.d_out && col0 + lane < p.d_in)
      out[static_cast<int64_t>(row0 + r) * p.d_in + col0 + lane] = from_f32<OUT>(stg[r * 33 + lane]);
  }
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
