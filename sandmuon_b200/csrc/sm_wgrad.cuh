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
//   warp 0        delta producer: TMA loads (128-byte swizzle), counted on the
//                 leader's barrier
//   warp 1        MMA issuer (the leader's warp, for both CTAs)
//   warp 2        raw producer: TMA loads of the int8 tiles
//   warp 3        code producer: 4-byte asynchronous copies of their exponents
//   warps 4..11   epilogue: TMEM -> registers -> global
//   warps 12..27  converters: raw int8 tile -> 16-bit x^ in the swizzled layout
//                 the MMA reads, then an arrival on the leader's barrier
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
//
// Every wait is bounded (kWaitTimeoutNs).  One that runs out sets the status
// word, and whatever it kept from its result becomes NaN: `out` never shows
// memory that was not written.
#pragma once

#include <cuda_fp16.h>

#include "sm_activation.cuh"
#include "sm_common.cuh"

namespace smb {

constexpr int kWgTileM = 256, kWgTileN = 256;  // of a CTA pair
constexpr int kWgConvWarps = 16;
constexpr int kWgConvGroups = 4;
constexpr int kWgEpiWarps = 8;
constexpr int kWgChain = 128;  // MMA steps summed by the tensor core alone
// Warps 0..3 issue loads and MMAs; then come the epilogue and the converters,
// each whole groups of four warps that trade registers (setmaxnreg): the
// launch's 28 warps of 72 registers cover 4 of 40, 8 of 104 and 16 of 64.
constexpr int kWgEpiWarp0 = 4, kWgConvWarp0 = kWgEpiWarp0 + kWgEpiWarps;
constexpr int kWgThreads = 32 * (kWgConvWarp0 + kWgConvWarps);
constexpr int kWgLaunchRegs = 72, kWgIssueRegs = 40, kWgEpiRegs = 104, kWgConvRegs = 64;
static_assert(kWgThreads * kWgLaunchRegs <= 65536 &&
                  32 * (kWgEpiWarp0 * kWgIssueRegs + kWgEpiWarps * kWgEpiRegs + kWgConvWarps * kWgConvRegs) <=
                      kWgThreads * kWgLaunchRegs,
              "the register split fits what the block is launched with");
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
                            // stretches of `each` k-blocks (`more` workers take one
                            // more), across tile borders
  int each, more;
  void* out;                // [d_out, d_in]
  float* partials;          // [2 * workers, kWgPartialFloats]
  int vec_out;              // rows of `out` take 16-byte stores
  int expired;              // a worker whose first wait counts as run out, for tests; -1: none
};

// First k-block (counting through the shared tiles, end to end) of worker w,
// w <= workers.  32 bits: the host keeps workers * kblocks below 2^31.
__host__ __device__ inline int wgrad_begin(const WgradArgs& p, int w) {
  if (p.parts == 0) return w * p.each + (w < p.more ? w : p.more);
  if (w >= p.shared * p.parts) return p.shared * p.kblocks;
  const int tile = w / p.parts;
  return tile * p.kblocks + p.kblocks * (w - tile * p.parts) / p.parts;
}

// The worker that holds k-block b: the largest w with wgrad_begin(w) <= b.
// b is the first or the last k-block of a tile.
__host__ __device__ inline int wgrad_worker(const WgradArgs& p, int b) {
  if (p.parts > 0) {
    const int tile = b / p.kblocks;
    return tile * p.parts + (b == tile * p.kblocks ? 0 : p.parts - 1);
  }
  const int big = p.more * (p.each + 1);
  return b < big ? b / (p.each + 1) : p.more + (b - big) / p.each;
}

// A worker's stretch of k-blocks inside one tile, at tile row mi, column ni.
struct WgSegment {
  int mi, ni, kb0, kb1;
};

// The segments of a worker: its share of the shared tiles, then whole tiles.
struct WgIter {
  int left, kb, tile, next_tile, index;
  const WgradArgs& p;
  __device__ __forceinline__ WgIter(const WgradArgs& args, int worker)
      : next_tile(args.shared + worker), index(0), p(args) {
    const int pos = wgrad_begin(p, worker);
    left = wgrad_begin(p, worker + 1) - pos;
    tile = pos / p.kblocks;
    kb = pos - tile * p.kblocks;
    skip();
  }
  __device__ __forceinline__ void skip() {
    if (left == 0 && next_tile < p.tiles) {
      tile = next_tile;
      next_tile += p.workers;
      kb = 0;
      left = p.kblocks;
    }
  }
  __device__ __forceinline__ bool valid() const { return left > 0; }
  __device__ __forceinline__ WgSegment get() const {
    WgSegment s;
    s.mi = tile / p.tiles_n;
    s.ni = tile - s.mi * p.tiles_n;
    s.kb0 = kb;
    s.kb1 = min(p.kblocks, kb + left);
    return s;
  }
  __device__ __forceinline__ void next(const WgSegment& s) {
    left -= s.kb1 - s.kb0;
    ++tile;
    kb = 0;
    ++index;
    skip();
  }
};

// Three rings, each as deep as its slots live long (measured in k-blocks of
// about 0.3 us): delta tiles from their TMA load to the end of their MMAs
// (about 2 us), raw tiles from their load to their conversion, converted tiles
// from there to the end of the MMAs.  One ring of five whole stages instead
// was bound by its depth: 512 us for 16384 x 2048 x 8192.
template <int PLANES, int BK>
struct WgSmem {
  static constexpr int kABytes = 128 * BK * 2;    // one plane of this CTA's delta columns
  static constexpr int kBBytes = 128 * BK * 2;    // this CTA's x^ columns
  static constexpr int kRawBytes = 128 * BK;
  static constexpr int kCodeBytes = 4 * BK;       // exponent codes of a raw tile
  static constexpr int kAStages = 5;
  static constexpr int kBStages = 4;
  static constexpr int kRawStages = 8;
  // A converter group sees every kWgConvGroups-th k-block.  It must see every
  // use of a slot that it waits on: were uses skipped, a wait for one phase
  // parity could not tell the use before the awaited one from the awaited one.
  static_assert(kRawStages % kWgConvGroups == 0, "a raw slot belongs to one group");
  static constexpr int kStagingBytes = kWgEpiWarps * 32 * 9 * 4;
  // Barriers per k-block, not per slot: "full" (both operands are there) and
  // "done" (its MMAs are), in rings whose length both slot rings divide.  One
  // wait and one commit a k-block are what the issuing warp has time for.
  static constexpr int kRing = 20;
  static_assert(kRing % kAStages == 0 && kRing % kBStages == 0, "a slot's barriers repeat with it");
  static_assert(kRing % kWgConvGroups == 0, "a done barrier belongs to one group");
  static constexpr int kBars = 2 * kRing + 2 * kRawStages + 4;
  static constexpr int kOffB = kAStages * PLANES * kABytes;
  static constexpr int kOffRaw = kOffB + kBStages * kBBytes;
  static constexpr int kOffCodes = kOffRaw + kRawStages * kRawBytes;
  static constexpr int kOffStaging = kOffCodes + kRawStages * kCodeBytes;
  static constexpr int kOffBars = kOffStaging + kStagingBytes;
  static constexpr int kTotal = kOffBars + kBars * 8 + 16 + 1024;
  static constexpr int kChainBlocks = kWgChain / (PLANES * BK / 16);  // k-blocks of one chain
  static_assert(kTotal <= 232448, "shared memory budget");
};

// Position in a ring of N slots: the slot, and the parity of its use.
template <int N>
struct WgRing {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() { skip<1>(); }
  // by n uses, where n <= N
  template <int n>
  __device__ __forceinline__ void skip() {
    slot += n;
    if (slot >= N) {
      slot -= N;
      phase ^= 1u;
    }
  }
};

// Instruction descriptor with both operands MN-major; F16 or BF16.
__host__ __device__ constexpr uint32_t wgrad_idesc(bool f16) {
  return f16 ? umma_idesc_bf16(kWgTileM, kWgTileN, true, true) & ~((1u << 7) | (1u << 10))
             : umma_idesc_bf16(kWgTileM, kWgTileN, true, true);
}

__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four int8 values -> four 16-bit x^ = q * 2^e, exactly, as the pairs (0, 2)
// and (1, 3): what masks give without a byte permutation.  The tile's columns
// stay in that order and the epilogue swaps the two in the middle of every
// four back.  The 16-bit float pipe is the converters' limit (32 lanes a clock
// and SM), so the scale enters through exponent bits and one addition a pair
// is all it does:
//   BF16: q's low 7 bits as the mantissa of 128 * 2^e, minus 128 * 2^e or, for
//         a negative q, 256 * 2^e (the sign bit added to the exponent field)
//   F16:  q + 128 in the mantissa of 1024 * 2^e, minus 1152 * 2^e
// That needs these powers of two to be normal numbers of the type.
// `dequant4_any` works for every code, NaN's included.
template <bool F16>
struct Dequant {
  // codes of the short form: e in [-24, 5], or up to 119
  static constexpr uint32_t kFirst = F16 ? 127 - 24 : 0, kLast = F16 ? 127 + 5 : 127 + 119;
  uint32_t base, minus;
  __device__ __forceinline__ static bool fits(uint32_t code) { return code - kFirst <= kLast - kFirst; }
  __device__ __forceinline__ explicit Dequant(uint32_t code) {
    if (F16) {
      const uint32_t h = (code - 127 + 25) << 10;  // 1024 * 2^e
      base = h | (h << 16);
      minus = base | 0x80808080u;  // 1152 = 1024 + 128: mantissa bit 7, and the sign (bit 15)
    } else {
      const uint32_t h = (code + 7) << 7;  // 128 * 2^e
      base = h | (h << 16);
      minus = base | 0x80008000u;
    }
  }
  __device__ __forceinline__ uint2 operator()(uint32_t w) const {
    if (F16) {
      const uint32_t u = w ^ 0x80808080u;
      return make_uint2(add_f16x2((u & 0x00ff00ffu) | base, minus), add_f16x2(((u >> 8) & 0x00ff00ffu) | base, minus));
    }
    const uint32_t v = w >> 8;
    return make_uint2(add_bf16x2((w & 0x007f007fu) | base, (w & 0x00800080u) + minus),
                      add_bf16x2((v & 0x007f007fu) | base, (v & 0x00800080u) + minus));
  }
};

template <bool F16>
__device__ __noinline__ uint2 dequant4_any(uint32_t w, uint32_t code) {
  const float scale = code_scale(code);
  if (F16) {
    const uint32_t h = __half_as_ushort(__float2half_rn(scale)), s = h | (h << 16);
    const uint32_t u = w ^ 0x80808080u, m = 0x64006400u, k = 0xe480e480u;  // 1024, -1152
    return make_uint2(mul_f16x2(add_f16x2((u & 0x00ff00ffu) | m, k), s),
                      mul_f16x2(add_f16x2(((u >> 8) & 0x00ff00ffu) | m, k), s));
  }
  const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rn(scale)), s = h | (h << 16);
  const uint32_t v = w >> 8, m = 0x43004300u, n = 0xc300c300u;  // 128, -128
  return make_uint2(mul_bf16x2(add_bf16x2((w & 0x007f007fu) | m, (w & 0x00800080u) | n), s),
                    mul_bf16x2(add_bf16x2((v & 0x007f007fu) | m, (v & 0x00800080u) | n), s));
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}

// Whether the phase is complete, without waiting (try_wait may suspend the
// thread for a while).
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
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

// 32 lanes x 16 consecutive 32-bit columns.
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
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
  constexpr uint32_t kChunkBytes = Swz::chunk_bytes(BK);
  constexpr uint32_t kIdesc = wgrad_idesc(F16);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kOffBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int worker = static_cast<int>(blockIdx.x) / 2;
  const bool live = worker != p.expired;
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_u32(bars);
  // full (the leader's): delta bytes and converters of both CTAs.  done: the
  // MMAs of a k-block are done, in both CTAs.  raw_full: this CTA's int8 tile
  // and its codes.  raw_empty: its converters have read it.
  auto bar_full = [&](int i) { return bar_base + 8u * i; };
  auto bar_done = [&](int i) { return bar_base + 8u * (S::kRing + i); };
  auto bar_rfull = [&](int i) { return bar_base + 8u * (2 * S::kRing + i); };
  auto bar_rempty = [&](int i) { return bar_base + 8u * (2 * S::kRing + S::kRawStages + i); };
  auto bar_tfull = [&](int i) { return bar_base + 8u * (S::kBars - 4 + i); };
  auto bar_tempty = [&](int i) { return bar_base + 8u * (S::kBars - 2 + i); };
  auto slot_a = [&](int i) { return smem_base + i * (PLANES * S::kABytes); };
  auto slot_b = [&](int i) { return smem_base + S::kOffB + i * S::kBBytes; };
  auto slot_raw = [&](int i) { return smem_base + S::kOffRaw + i * S::kRawBytes; };
  auto slot_codes = [&](int i) { return smem_base + S::kOffCodes + i * S::kCodeBytes; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kRing; ++i) {
      mbar_init(bar_full(i), 1 + 2 * kWgConvWarps / kWgConvGroups);
      mbar_init(bar_done(i), 1);
    }
    for (int i = 0; i < S::kRawStages; ++i) {
      mbar_init(bar_rfull(i), 1 + 32);
      mbar_init(bar_rempty(i), kWgConvWarps / kWgConvGroups);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_tfull(i), 1);
      mbar_init(bar_tempty(i), 2 * kWgEpiWarps);
    }
    *abort_flag = live ? 0 : kStatusTimeoutWgradProducer;
    if (!live) atomicExch(&g_status, kStatusTimeoutWgradProducer);
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

  if (warp < kWgEpiWarp0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWgIssueRegs));
  if (warp == 0) {
    // ------------------------------------------------------ delta producer
    if (lane == 0) {
      WgRing<S::kAStages> ra;
      WgRing<S::kRing> rf, rd;  // this k-block, and the one kAStages back
      int64_t i = 0;
      bool ok = live;
      for (WgIter it(p, worker); it.valid() && ok;) {
        const WgSegment s = it.get();
        const int mc = s.mi * kWgTileM + static_cast<int>(rank) * 128;
        for (int kb = s.kb0; kb < s.kb1; ++kb, ++i, ra.next(), rf.next()) {
          if (i >= S::kAStages) {
            if (!mbar_wait(bar_done(rd.slot), rd.phase, abort_flag, kStatusTimeoutWgradProducer)) {
              ok = false;
              break;
            }
            rd.next();
          }
          const uint32_t fb = mapa_shared(bar_full(rf.slot), 0);
          if (rank == 0) mbar_arrive_expect_tx(bar_full(rf.slot), 2 * PLANES * S::kABytes);
#pragma unroll
          for (int j = 0; j < PLANES; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tma_load_2d_pair(slot_a(ra.slot) + j * S::kABytes + h * kChunkBytes, &p.a[j], fb, mc + 64 * h, kb * BK);
          }
        }
        it.next(s);
      }
      // the leader's last commits have arrived before this CTA may leave
      for (int64_t left = i < S::kAStages ? i : S::kAStages; left > 0 && ok; --left, rd.next())
        ok = mbar_wait(bar_done(rd.slot), rd.phase, abort_flag, kStatusTimeoutWgradProducer);
    }
  } else if (warp == 2) {
    // -------------------------------------------------------- raw producer
    // (apart from delta's, whose waits for the MMAs would hold it back)
    if (lane == 0) {
      WgRing<S::kRawStages> rr;
      bool ok = live;
      for (WgIter it(p, worker); it.valid() && ok;) {
        const WgSegment s = it.get();
        const int nc = s.ni * kWgTileN + static_cast<int>(rank) * 128;
        for (int kb = s.kb0; kb < s.kb1; ++kb, rr.next()) {
          if (!mbar_wait(bar_rempty(rr.slot), rr.phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(bar_rfull(rr.slot), S::kRawBytes);
          tma_load_2d(slot_raw(rr.slot), &p.q, bar_rfull(rr.slot), nc, kb * BK);
        }
        it.next(s);
      }
      // the converters have read every slot
      for (int i = 0; i < S::kRawStages && ok; ++i, rr.next())
        ok = mbar_wait(bar_rempty(rr.slot), rr.phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer);
    }
  } else if (warp == 3) {
    // ------------------------------------------------------- code producer
    // A lane copies the 4 codes of a token's 128 columns.  Codes outside the
    // checkpoint become 0: their values are 0 as well.
    WgRing<S::kRawStages> rr;
    bool ok = live;
    for (WgIter it(p, worker); it.valid() && ok;) {
      const WgSegment s = it.get();
      const int g = (s.ni * kWgTileN + static_cast<int>(rank) * 128) / kGroup;
      const int rows = g < p.lde ? p.rows : 0;
      const uint8_t* src = p.codes + (static_cast<int64_t>(s.kb0) * BK + lane) * p.lde + g;
      int r = s.kb0 * BK + lane;
      for (int kb = s.kb0; kb < s.kb1; ++kb, rr.next()) {
        ok = mbar_wait(bar_rempty(rr.slot), rr.phase ^ 1u, abort_flag, kStatusTimeoutWgradProducer);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int t = 0; t < BK; t += 32, r += 32, src += 32 * p.lde)
          cp_async4(slot_codes(rr.slot) + 4 * (t + lane), r < rows ? src : p.codes, r < rows);
        cp_async_arrive(bar_rfull(rr.slot));
      }
      it.next(s);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- MMA issuer
    // The whole warp walks the loop, so that descriptors and barriers stay in
    // uniform registers; one elected lane issues.  (One lane alone in a
    // divergent branch took 95 clocks to issue an MMA that runs for 128.)
    if (rank == 0) {
      const bool elected = elect_one();
      WgRing<S::kAStages> ra;
      WgRing<S::kBStages> rb;
      WgRing<S::kRing> rf;
      int home = 0;
      uint32_t uses0 = 0, uses1 = 0;  // chains that ran in each accumulator
      bool ok = live, ready = false;
      const uint64_t a_desc = umma_desc(slot_a(0), kChunkBytes, Swz::kSbo, Swz::kLayout);
      const uint64_t b_desc = umma_desc(slot_b(0), kChunkBytes, Swz::kSbo, Swz::kLayout);
      for (WgIter it(p, worker); it.valid() && ok; home ^= 1) {
        const WgSegment s = it.get();
        for (int begin = s.kb0; begin < s.kb1 && ok; begin += S::kChainBlocks) {
          const int end = min(begin + S::kChainBlocks, s.kb1);
          const int acc = begin == s.kb0 ? home : home ^ 1;
          const uint32_t uses = acc ? uses1++ : uses0++;
          ok = mbar_wait(bar_tempty(acc), (uses & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kWgTileN);
          uint32_t accumulate = 0;
          for (int kb = begin; kb < end; ++kb) {
            if (!ready) {
              ok = mbar_wait(bar_full(rf.slot), rf.phase, abort_flag, kStatusTimeoutWgradMma);
              if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
              }
            }
            tc_fence_after();
            // the start address is in units of 16 bytes in the lowest bits
            const uint64_t a0 = a_desc + static_cast<uint32_t>(ra.slot) * (PLANES * S::kABytes / 16);
            const uint64_t b0 = b_desc + static_cast<uint32_t>(rb.slot) * (S::kBBytes / 16);
            const uint32_t done = bar_done(rf.slot);
            ra.next();
            rb.next();
            rf.next();
            // asked before the MMAs are issued: the answer arrives meanwhile
            ready = mbar_test_wait(bar_full(rf.slot), rf.phase);
            if (elected) {
#pragma unroll
              for (int ks = 0; ks < BK / 16; ++ks) {
#pragma unroll
                for (int j = PLANES - 1; j >= 0; --j)  // smallest plane first
                  umma_bf16_pair(d_tmem, a0 + (j * S::kABytes + ks * Swz::kMnStepBytes) / 16,
                                 b0 + ks * Swz::kMnStepBytes / 16, kIdesc,
                                 ks > 0 || j < PLANES - 1 ? 1u : accumulate);
              }
              umma_commit_pair(done, 0x3);
            }
            accumulate = 1;
            ready = __all_sync(0xffffffffu, ready);
          }
          if (ok && elected) umma_commit_pair(bar_tfull(acc), 0x3);
          __syncwarp();
        }
        it.next(s);
      }
      // both accumulators' last chains have been read by both CTAs
      if (ok) ok = mbar_wait(bar_tempty(0), (uses0 & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
      if (ok) mbar_wait(bar_tempty(1), (uses1 & 1) ^ 1u, abort_flag, kStatusTimeoutWgradMma);
      __syncwarp();
    }
  } else if (warp >= kWgEpiWarp0 && warp < kWgConvWarp0) {
    // ------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWgEpiRegs));
    const int quarter = warp & 3;                // TMEM lanes this warp may access
    const int half = (warp - kWgEpiWarp0) >> 2;  // its 128 of the tile's 256 columns
    const uint32_t tempty0 = mapa_shared(bar_tempty(0), 0);
    float* stg = reinterpret_cast<float*>(smem + S::kOffStaging) + (warp - kWgEpiWarp0) * 32 * 9;
    auto release = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(tempty0 + 8u * acc);
    };
    int home = 0;
    uint32_t uses0 = 0, uses1 = 0;
    bool ok = live;
    for (WgIter it(p, worker); it.valid(); home ^= 1) {
      const WgSegment s = it.get();
      const bool whole = s.kb0 == 0 && s.kb1 == p.kblocks;
      const int row0 = s.mi * kWgTileM + static_cast<int>(rank) * 128 + quarter * 32;
      const int colt = s.ni * kWgTileN;
      float* part = p.partials + static_cast<int64_t>(2 * worker + (it.index > 0 ? 1 : 0)) * kWgPartialFloats;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t t_home = t_row + static_cast<uint32_t>(home * kWgTileN);
      const uint32_t t_other = t_row + static_cast<uint32_t>((home ^ 1) * kWgTileN);
      for (int begin = s.kb0; begin < s.kb1 && ok; begin += S::kChainBlocks) {
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
        if (!last) {
          // home += other, 32 columns at a time
#pragma unroll 1
          for (int col = kWgTileN / 2 * half; col < kWgTileN / 2 * (half + 1); col += 32) {
            uint32_t r[32], x[32];
            tmem_ld_32x32(t_other + col, x);
            tmem_ld_32x32(t_home + col, r);
            tmem_wait_ld();
            if (col == kWgTileN / 2 * (half + 1) - 32) release(home ^ 1);
#pragma unroll
            for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) + __uint_as_float(x[c]));
            tmem_st_32x32(t_home + col, r);
          }
          tmem_wait_st();
          continue;
        }
        constexpr int kSteps = kWgTileN / 2 / 16;  // 16 columns each
#pragma unroll 1
        for (int i = 0; i < kSteps; ++i) {
          const int col = kWgTileN / 2 * half + 16 * i;
          uint32_t r[16];
          tmem_ld_32x16(t_home + col, r);
          if (!first) {
            uint32_t x[16];
            tmem_ld_32x16(t_other + col, x);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) + __uint_as_float(x[c]));
            if (i == kSteps - 1) release(home ^ 1);
          } else {
            tmem_wait_ld();
          }
          if (i == kSteps - 1) release(home);
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // the converters' column order back to the result's
            const uint32_t swap = r[4 * c + 1];
            r[4 * c + 1] = r[4 * c + 2];
            r[4 * c + 2] = swap;
          }
          if (!whole) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              *reinterpret_cast<uint4*>(part + partial_offset(rank, quarter, col / 32, col / 4 % 8 + c, lane)) =
                  make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int c = 0; c < 8; ++c) stg[lane * 9 + c] = __uint_as_float(r[8 * h + c]);
              __syncwarp();
              store_block<8>(static_cast<OUT*>(p.out), p.d_in, row0, colt + col + 8 * h, p.d_out, p.d_in, stg, lane,
                             p.vec_out != 0);
              __syncwarp();
            }
          }
        }
      }
      if (!ok) {
        // A wait ran out, here or (then this warp's own does too) before an MMA
        // of the segment: its part of the result or partial tile becomes NaN,
        // as do those of the segments that follow.
        const float nan = __uint_as_float(0x7fffffffu);
        if (!whole) {
#pragma unroll 1
          for (int col = kWgTileN / 2 * half; col < kWgTileN / 2 * (half + 1); col += 4)
            *reinterpret_cast<float4*>(part + partial_offset(rank, quarter, col / 32, col / 4 % 8, lane)) =
                make_float4(nan, nan, nan, nan);
        } else {
#pragma unroll 1
          for (int i = 0; i < 32 * (kWgTileN / 2 / 32); ++i) {
            const int row = row0 + i / (kWgTileN / 2 / 32);
            const int col = colt + kWgTileN / 2 * half + 32 * (i % (kWgTileN / 2 / 32)) + lane;
            if (row < p.d_out && col < p.d_in)
              static_cast<OUT*>(p.out)[static_cast<int64_t>(row) * p.d_in + col] = from_f32<OUT>(nan);
          }
        }
      }
      it.next(s);
    }
  } else if (warp >= kWgConvWarp0) {
    // ---------------------------------------------------------- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWgConvRegs));
    // Groups of warps take k-blocks in turn, so that one group's latency hides
    // behind the other's.  A task is 16 columns of one token.  8 neighbouring
    // lanes hold 4 tasks of token k in one 64-column chunk and 4 of token k ^ 1
    // in the other: their 16-byte loads and swizzled stores each cover all 32
    // banks once.
    constexpr int kGroupWarps = kWgConvWarps / kWgConvGroups;
    constexpr int kTasks = BK * 8 / (32 * kGroupWarps);
    constexpr int kTaskRows = 4 * kGroupWarps;  // tokens of one task round, a multiple of the swizzle's 8
    static_assert(kTaskRows % 8 == 0 && kTasks * kTaskRows == BK, "whole task rounds");
    const int group = (warp - kWgConvWarp0) / kGroupWarps;
    const int k0 = ((warp - kWgConvWarp0) % kGroupWarps) * 4 + (lane >> 4) * 2 + ((lane >> 2) & 1);
    const int chunk = ((lane >> 3) ^ k0) & 1, seg = lane & 3;
    const uint32_t in_off = k0 * 128 + chunk * 64 + seg * 16;
    const uint32_t out_off = chunk * kChunkBytes + k0 * 128;
    const uint32_t off0 = out_off + (((2 * seg) ^ (k0 & 7)) << 4), off1 = out_off + (((2 * seg + 1) ^ (k0 & 7)) << 4);
    const uint32_t code_off = 4 * k0 + 2 * chunk + (seg >> 1);
    const uint32_t full0 = mapa_shared(bar_full(0), 0);
    WgRing<S::kRawStages> rr;
    WgRing<S::kBStages> rb;
    WgRing<S::kRing> rf, rd;  // this k-block, and the one kBStages back (from there on)
    // k-blocks of this worker: its share and its whole tiles
    const int64_t whole = p.shared + worker < p.tiles ? (p.tiles - 1 - p.shared - worker) / p.workers + 1 : 0;
    const int64_t blocks = live ? wgrad_begin(p, worker + 1) - wgrad_begin(p, worker) + whole * p.kblocks : 0;
    rr.slot = rb.slot = rf.slot = rd.slot = group;
    constexpr int kSkip = kWgConvGroups;
    static_assert(kSkip <= S::kBStages, "a group's first k-block finds its slot empty");
    for (int64_t i = group; i < blocks; i += kSkip, rr.template skip<kSkip>(), rb.template skip<kSkip>(),
                 rf.template skip<kSkip>()) {
      bool ok = mbar_wait(bar_rfull(rr.slot), rr.phase, abort_flag, kStatusTimeoutWgradConvert);
      if (!__all_sync(0xffffffffu, ok)) break;
      uint4 w[kTasks];
      uint32_t code[kTasks];
#pragma unroll
      for (int t = 0; t < kTasks; ++t) {
        w[t] = lds128(slot_raw(rr.slot) + in_off + t * (kTaskRows * 128));
        code[t] = lds8(slot_codes(rr.slot) + code_off + t * (kTaskRows * 4));
      }
      if (i >= S::kBStages) {
        ok = mbar_wait(bar_done(rd.slot), rd.phase, abort_flag, kStatusTimeoutWgradConvert);
        if (!__all_sync(0xffffffffu, ok)) break;
        rd.template skip<kSkip>();
      }
#pragma unroll
      for (int t = 0; t < kTasks; ++t) {
        uint2 a0, a1, b0, b1;
        if (Dequant<F16>::fits(code[t])) {
          const Dequant<F16> d(code[t]);
          a0 = d(w[t].x), a1 = d(w[t].y), b0 = d(w[t].z), b1 = d(w[t].w);
        } else {
          a0 = dequant4_any<F16>(w[t].x, code[t]), a1 = dequant4_any<F16>(w[t].y, code[t]);
          b0 = dequant4_any<F16>(w[t].z, code[t]), b1 = dequant4_any<F16>(w[t].w, code[t]);
        }
        sts128(slot_b(rb.slot) + off0 + t * (kTaskRows * 128), a0.x, a0.y, a1.x, a1.y);
        sts128(slot_b(rb.slot) + off1 + t * (kTaskRows * 128), b0.x, b0.y, b1.x, b1.y);
      }
      // Every value read from the raw slot has been used, so the loads are done
      // and the slot is free.  (Released right after the loads were issued, the
      // slot's next codes could overtake a delayed load: about one k-block in a
      // million came out with some tokens at a wrong scale.)
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_rempty(rr.slot));
      // The MMA that these arrivals admit reads this tile through this CTA's
      // own async proxy, to which the fence has made it visible before the
      // arrival is issued.  The arrival has CTA scope, also where the leader's
      // barrier is the peer's: the memory model promises an order across CTAs
      // for cluster scope only, which waits for all of the thread's memory
      // traffic (16384 tokens, 768 -> 768: 36.9 us instead of 28.0; 2048 ->
      // 8192: 625 instead of 470; one forwarding warp per CTA: 45.6 and 839).
      // Every k-block's result is held to its bits by the repetition test.
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(full0 + 8u * rf.slot);
    }
  }

  // After a wait that ran out, copies may still be in flight into this CTA's
  // shared memory, which has to outlive them: leave 100 us later.
  if (*abort_flag != 0)
    for (int i = 0; i < 100; ++i) __nanosleep(1000);
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
  const int mi = tile / p.tiles_n;
  const int row0 = mi * kWgTileM + cta * 128 + quarter * 32;
  const int col0 = (tile - mi * p.tiles_n) * kWgTileN + chunk * 32;
  const int k_begin = tile * p.kblocks;
  const int w0 = wgrad_worker(p, k_begin), w1 = wgrad_worker(p, k_begin + p.kblocks - 1);
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
// A thread makes 8 columns of a plane row (16-byte stores; 16-byte loads where
// VEC says that delta's rows allow them).
template <typename T, int PLANES, bool VEC>
__global__ void __launch_bounds__(256)
    k_wgrad_planes(const T* __restrict__ delta, int64_t rs, int64_t cs, int64_t rows, int64_t cols, int64_t ld,
                   uint16_t* __restrict__ planes) {
  const int64_t c0 = (static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x) * 8;
  if (c0 < ld) {
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; r < rows;
         r += static_cast<int64_t>(gridDim.y) * blockDim.y) {
      const T* src = delta + r * rs + c0 * cs;
      uint16_t* dst = planes + r * ld + c0;
      if constexpr (PLANES == 1) {
        uint16_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          b[i] = 0;
          if (c0 + i < cols) memcpy(&b[i], src + i * cs, 2);
        }
        uint4 w;
        memcpy(&w, b, 16);
        *reinterpret_cast<uint4*>(dst) = w;
      } else {
        float v[8];
        if constexpr (VEC) {
          Vec8<float> w;
          vec8_load(src, w);
          vec8_unpack(w, v);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = c0 + i < cols ? src[i * cs] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PLANES; ++j) {
          uint32_t top[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t bits = __float_as_uint(v[i]);
            const bool special = (bits & 0x7f800000u) == 0x7f800000u;
            top[i] = bits & 0xffff0000u;
            if (special && (bits & 0x007fffffu) != 0) top[i] |= 0x00400000u;  // NaN whatever its payload
            v[i] = special ? 0.0f : v[i] - __uint_as_float(top[i]);
          }
          *reinterpret_cast<uint4*>(dst + j * rows * ld) =
              make_uint4(__byte_perm(top[0], top[1], 0x7632), __byte_perm(top[2], top[3], 0x7632),
                         __byte_perm(top[4], top[5], 0x7632), __byte_perm(top[6], top[7], 0x7632));
        }
      }
    }
  }
  grid_dep_launch();
}

}  // namespace smb
