// mx_gemm.cuh — block-scaled tcgen05 products of microscaled matrices (sm_100a).
//
//   C[m][n] = ts_a * ts_b * sum_k (a[m][k] * sa[m][k / block]) * (b[n][k] * sb[n][k / block])
//
// The tensor core applies the block scales itself (tcgen05.mma ... block_scale): it reads
// them from TMEM, where tcgen05.cp puts the 128-row x 4-block scale tiles as they lie in
// memory (32 lanes x 16 bytes, repeated for the four lane quarters). Elements go through
// shared memory as in the plain GEMM: TMA boxes of one 128-byte K atom per row with
// 128-byte swizzle, 32 bytes of K per MMA. An atom is 128 elements of MX_FP8 (one scale
// tile per 128 rows) or 256 elements of a 4-bit format (two tiles for MX_FP4, four for
// NV_FP4).
#pragma once

#include "gemm_sm100.cuh"
#include "mx_common.cuh"

namespace b200 {

// ---------------------------------------------------------------------------------
// PTX
// ---------------------------------------------------------------------------------
// Shared-memory descriptor of one 512-byte scale tile: no swizzle, 32 rows of 16 bytes
// as four 8-row core matrices 128 bytes apart.
__device__ __forceinline__ uint64_t sdesc_scale_tile(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(128u >> 4) << 32) | (uint64_t(1u) << 46);
}
// One scale tile into four TMEM columns, repeated in the four lane quarters. Copies and
// MMAs issued by one thread execute in order, so no wait is needed in either direction.
template <int CG>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t sdesc) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

// Instruction descriptor of a block-scaled MMA, both operands K-major, fp32 accumulator:
//   bits  4-5  B scale byte id      bits 29-30  A scale byte id
//   bits  7-9 / 10-12  A / B format (mxf8f6f4: 0 e4m3; mxf4, mxf4nvf4: 1 e2m1)
//   bits 17-22 N >> 3               bits 24-28  M >> 4
//   bit  23    scale format (0 e4m3, 1 e8m0)
template <int FMT>
__host__ __device__ constexpr uint32_t idesc_mx(uint32_t M, uint32_t N, uint32_t sf_id) {
  const uint32_t f = FMT == MX_FP8 ? 0u : 1u;
  return (sf_id << 4) | (f << 7) | (f << 10) | ((N >> 3) << 17) | ((FMT == NV_FP4 ? 0u : 1u) << 23) |
         ((M >> 4) << 24) | (sf_id << 29);
}

#define B200_UMMA_MX(GROUP, KIND)                                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                               \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d_tmem), \
               "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate))
template <int CG, int FMT>
__device__ __forceinline__ void umma_mx(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 1) {
    if constexpr (FMT == MX_FP8) B200_UMMA_MX("1", "mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (FMT == MX_FP4) B200_UMMA_MX("1", "mxf4.block_scale.scale_vec::2X");
    else B200_UMMA_MX("1", "mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    if constexpr (FMT == MX_FP8) B200_UMMA_MX("2", "mxf8f6f4.block_scale.scale_vec::1X");
    else if constexpr (FMT == MX_FP4) B200_UMMA_MX("2", "mxf4.block_scale.scale_vec::2X");
    else B200_UMMA_MX("2", "mxf4nvf4.block_scale.scale_vec::4X");
  }
}
#undef B200_UMMA_MX

__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ float4 ld_shared_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// True in one lane of the (converged) warp. The compiler knows a branch on elect.sync to
// be taken by one thread, so descriptors and addresses inside it go straight to uniform
// registers; under `lane == 0` every MMA or scale copy pays a per-lane loop instead:
// 119 clocks per MMA and 14 per copy measured, against 96 (N = 192, copies hidden).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ---------------------------------------------------------------------------------
// format facts of one 128-byte K atom
// ---------------------------------------------------------------------------------
template <int FMT>
struct MxAtom {
  static constexpr uint32_t GROUPS = FMT == MX_FP8 ? 1 : FMT == MX_FP4 ? 2 : 4;  // scale tiles per 128 rows
  // MMA step s (32 bytes of K): its scale tile within the atom, and the byte id of its
  // first scale in the tile's 4-byte words
  static constexpr uint32_t group(uint32_t s) { return FMT == MX_FP8 ? 0 : FMT == MX_FP4 ? s / 2 : s; }
  static constexpr uint32_t sf_id(uint32_t s) { return FMT == MX_FP8 ? s : FMT == MX_FP4 ? 2 * (s % 2) : 0; }
};

// Scale copies and MMAs of one stage, issued by one thread: `g_n` scale tiles per band,
// `steps` MMA steps, both at their maximum when FULL. The issue itself is what a stage can
// wait for (16 copies and 8 MMAs against 768 clocks of MMA time), so a full stage has no
// run-time conditions, and every descriptor is a base plus a constant: with a condition per
// step a 192-wide pair stage took 511 clocks, without 386 (its MMAs alone: 384).
//   sa / sb     TMEM columns of the two operands' scales; BANDS tiles of 4 columns per group
//   a / b       shared-memory descriptors of the first step
//   d           first accumulator column
template <int CG, int FMT, uint32_t N, uint32_t BANDS, bool FULL>
struct MxStage {
  using Atom = MxAtom<FMT>;
  static __device__ __forceinline__ void copy_scales(uint32_t sa, uint32_t sb, uint64_t tile_a, uint64_t tile_b,
                                                     uint32_t g_n) {
#pragma unroll
    for (uint32_t g = 0; g < Atom::GROUPS; ++g) {
      if (FULL || g < g_n) {
        tmem_cp_scales<CG>(sa + 4 * g, tile_a + g * 32u);
#pragma unroll
        for (uint32_t b = 0; b < BANDS; ++b)
          tmem_cp_scales<CG>(sb + 4 * (BANDS * g + b), tile_b + (b * Atom::GROUPS + g) * 32u);
      }
    }
  }
  static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t sa, uint32_t sb,
                                             uint32_t steps, uint32_t accumulate) {
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s)
      if (FULL || s < steps)
        umma_mx<CG, FMT>(d, a + 2 * s, b + 2 * s, idesc_mx<FMT>(128 * CG, N, Atom::sf_id(s)), sa + 4 * Atom::group(s),
                         sb + 4 * BANDS * Atom::group(s), s ? 1u : accumulate);
  }
};

struct MxParams {
  uint32_t np, nq;     // rows of the 128-row operand (P) and of the other one (Q)
  uint32_t row_bytes;  // K in bytes
  uint32_t k_atoms, groups;
  uint32_t p_tiles, q_tiles, splits;
  uint32_t stages;
  const uint8_t* sf_p;
  const uint8_t* sf_q;
  const float* ts_p;  // tensor scales, may be null
  const float* ts_q;
  uint8_t* c;
  uint64_t ldc;   // elements
  uint32_t vec;   // C rows take 4-element stores
  uint32_t* status;
  uint64_t wait_ns;
  uint32_t fault_inject;  // test hook: 1 = the producer issues no loads, 2 = the MMA warp gives up
};

// ---------------------------------------------------------------------------------
// mx_gemm_rows_kernel: 128 rows of B (P) x NT rows of A (Q) per CTA, K split over the
// CTAs of a cluster
// ---------------------------------------------------------------------------------
// The accumulator is C transposed: TMEM lane = row of B (column of C), column = row of A.
// With few rows of A the weights B are the long operand and take the MMA's 128-row side;
// the other side is only as wide as the tokens need (NT = 16 ... 128), so one token does
// not pay for 128. K is split over a cluster of up to 8 CTAs when the tiles alone leave
// SMs idle; the partial sums meet in distributed shared memory, added in rank order, so
// results do not depend on timing and no workspace or second launch is needed.
template <int FMT, int NT>
struct MxRowsCfg {
  static constexpr uint32_t GROUPS = MxAtom<FMT>::GROUPS;
  static constexpr uint32_t P_BYTES = 128 * 128;
  static constexpr uint32_t Q_BYTES = NT * 128;
  static constexpr uint32_t SFP_BYTES = GROUPS * 512;
  static constexpr uint32_t SFQ_BYTES = GROUPS * 512;
  static constexpr uint32_t STAGE = P_BYTES + Q_BYTES + SFP_BYTES + SFQ_BYTES;
  static constexpr uint32_t BAR_BYTES = 256;
  static constexpr uint32_t MAX_SMEM = 232448;
  static constexpr uint32_t FIT = (MAX_SMEM - 1024 - BAR_BYTES) / STAGE;
  static constexpr uint32_t MAX_STAGES = FIT > 8 ? 8 : FIT;
  // ring of a CTA that shares its SM with a second one (113 KB each)
  static constexpr uint32_t HALF_STAGES = (113 * 1024 - 1024 - BAR_BYTES) / STAGE;
  static constexpr uint32_t PARTIAL = NT * 128 * 4;  // overlays the ring after the main loop
  static constexpr uint32_t ACC_COLS = NT < 32 ? 32 : NT;
  static constexpr uint32_t SFP_COL = ACC_COLS;
  static constexpr uint32_t SFQ_COL = SFP_COL + 4 * GROUPS;
  static constexpr uint32_t COLS = SFQ_COL + 4 * GROUPS;
  static constexpr uint32_t TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : 256;
  static_assert(NT <= 128 && COLS <= 256, "a tile's rows lie in one scale band, two CTAs share an SM's TMEM");
  static uint32_t smem_bytes(uint32_t stages) {
    const uint32_t ring = stages * STAGE;
    return (ring > PARTIAL ? ring : PARTIAL) + BAR_BYTES + 1024;
  }
};

// ts_a * ts_b as two factors that a sum is multiplied by one after the other. The product of
// two tensor scales (positive and normal) may leave fp32 where C does not: A near 1e-30 and B
// near 1e-8 have scales of 4e-34 and 4e-12, and two large ones overflow, which would make a
// sum of zero NaN. Inside fp32's normal numbers it is one factor (the other is 1). Sums are
// multiples of 2^-20 below 2^54, so the first product is normal wherever C is not 0, and
// infinite only where C is. A negative or NaN scale comes through too.
struct SumScale {
  float first, second = 1.0f;
  __device__ __forceinline__ SumScale(const float* ts_a, const float* ts_b) {
    const float a = ts_a ? *ts_a : 1.0f, b = ts_b ? *ts_b : 1.0f;
    first = a * b;
    if (fabsf(first) < 0x1p-126f && a != 0.0f && b != 0.0f) {  // neither is above 2^23
      first = (a * 0x1p64f) * (b * 0x1p64f);
      second = 0x1p-128f;
    } else if (fabsf(first) > 0x1.fffffep127f) {  // neither is below 1
      first = (a * 0x1p-63f) * (b * 0x1p-64f);
      first = fminf(fmaxf(first, -0x1.fffffep127f), 0x1.fffffep127f);
      second = 0x1p127f;
    }
  }
  template <int FMT>
  __device__ __forceinline__ float apply(float sum) const {
    return FMT == NV_FP4 ? sum * first * second : sum;  // the other formats have no tensor scale
  }
};

template <int CD>
struct OutElem;
template <>
struct OutElem<DT_F16> { using E = Elem<0>; };
template <>
struct OutElem<DT_BF16> { using E = Elem<1>; };
template <>
struct OutElem<DT_F32> { using E = Elem<3>; };

// Four consecutive elements of a C row; `n` of them exist.
template <int CD>
__device__ __forceinline__ void store_c4(uint8_t* c, uint64_t index, const float4& v, uint32_t n, bool vec) {
  using E = typename OutElem<CD>::E;
  typename E::T* d = reinterpret_cast<typename E::T*>(c) + index;
  if (vec && n >= 4) {
    if constexpr (CD == DT_F32) *reinterpret_cast<float4*>(d) = v;
    else *reinterpret_cast<uint2*>(d) = make_uint2(E::pack(v.x, v.y), E::pack(v.z, v.w));
  } else {
    if (n > 0) d[0] = E::store(v.x);
    if (n > 1) d[1] = E::store(v.y);
    if (n > 2) d[2] = E::store(v.z);
    if (n > 3) d[3] = E::store(v.w);
  }
}

template <int FMT, int CD, int NT>
__global__ void __launch_bounds__(256, 1)
    mx_gemm_rows_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                        const MxParams p) {
  using Cfg = MxRowsCfg<FMT, NT>;
  using Atom = MxAtom<FMT>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* base_ptr = smem_raw + (base - raw);
  const uint32_t S = p.stages;
  const uint32_t sP = base, sQ = sP + S * Cfg::P_BYTES;
  const uint32_t sSP = sQ + S * Cfg::Q_BYTES, sSQ = sSP + S * Cfg::SFP_BYTES;
  const uint32_t ring = S * Cfg::STAGE;
  const uint32_t bar_off = ring > Cfg::PARTIAL ? ring : Cfg::PARTIAL;
  const uint32_t sBar = base + bar_off;
  // full[8], empty[8], tfull, done; the TMEM address, the abort flag, the issued stages
  const uint32_t bar_full = sBar, bar_empty = sBar + 64, bar_tfull = sBar + 128, bar_done = sBar + 136;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + bar_off + 144);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + bar_off + 148);
  volatile uint32_t* issued_word = reinterpret_cast<volatile uint32_t*>(base_ptr + bar_off + 152);

  const uint32_t warp = __shfl_sync(0xffffffffu, warp_id(), 0), lane = lane_id();
  if (warp == 0 && lane == 0) {
    for (uint32_t s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    mbar_init(bar_done, 1);
    *abort_flag = 0u;
    fence_mbar_init();
    tma_prefetch_desc(&tmP);
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  auto fail = [&](uint32_t code) {
    *abort_flag = 1u;
    if (p.status) atomicOr(p.status, code | ST_ABORTED);
  };

  const uint32_t tile = blockIdx.x / p.splits, rank = blockIdx.x % p.splits;
  const uint32_t tq = tile % p.q_tiles, tp = tile / p.q_tiles;
  const uint32_t q0 = tq * NT, p0 = tp * 128;
  // this CTA's atoms of K (at least one: splits <= k_atoms)
  const uint32_t k0 = uint32_t(uint64_t(p.k_atoms) * rank / p.splits);
  const uint32_t k1 = uint32_t(uint64_t(p.k_atoms) * (rank + 1) / p.splits);

  if (warp == 0) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0, issued = 0;
      const uint64_t hint_p = policy_evict_first(), hint_q = policy_evict_last();
      for (uint32_t kb = p.fault_inject == 1 ? k1 : k0; kb < k1; ++kb) {
        if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1u, p.wait_ns, abort_flag)) {
          fail(ST_PRODUCER_EMPTY);
          break;
        }
        const uint32_t g0 = kb * Cfg::GROUPS;
        const uint32_t ng = min(Cfg::GROUPS, p.groups - g0);
        const uint32_t bar = bar_full + 8 * stage;
        mbar_arrive_expect_tx(bar, Cfg::P_BYTES + Cfg::Q_BYTES + ng * 1024u);
        tma_load_2d(sP + stage * Cfg::P_BYTES, &tmP, int32_t(kb * 128u), int32_t(p0), bar, hint_p);
        tma_load_2d(sQ + stage * Cfg::Q_BYTES, &tmQ, int32_t(kb * 128u), int32_t(q0), bar, hint_q);
        bulk_load(sSP + stage * Cfg::SFP_BYTES, p.sf_p + (uint64_t(tp) * p.groups + g0) * 512u, ng * 512u, bar);
        bulk_load(sSQ + stage * Cfg::SFQ_BYTES, p.sf_q + (uint64_t(q0 / 128) * p.groups + g0) * 512u, ng * 512u, bar);
        ++issued;
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      *issued_word = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      bool ok = p.fault_inject != 2;
      if (!ok) fail(ST_MMA_FULL);
      for (uint32_t kb = k0; kb < k1 && ok; ++kb) {
        if (!mbar_wait(bar_full + 8 * stage, phase, p.wait_ns, abort_flag)) {
          fail(ST_MMA_FULL);
          ok = false;
          break;
        }
        const uint32_t ng = min(Cfg::GROUPS, p.groups - kb * Cfg::GROUPS);
        const uint32_t steps = min(4u, (p.row_bytes - kb * 128u + 31u) / 32u);
        const uint32_t sfp = tmem_base + Cfg::SFP_COL, sfq = tmem_base + Cfg::SFQ_COL;
        const uint64_t tile_p = sdesc_scale_tile(sSP + stage * Cfg::SFP_BYTES);
        const uint64_t tile_q = sdesc_scale_tile(sSQ + stage * Cfg::SFQ_BYTES);
        const uint64_t dp = sdesc_k_sw128(sP + stage * Cfg::P_BYTES), dq = sdesc_k_sw128(sQ + stage * Cfg::Q_BYTES);
        const uint32_t acc = kb != k0 ? 1u : 0u;
        if (steps == 4) {
          using Stage = MxStage<1, FMT, NT, 1, true>;
          Stage::copy_scales(sfp, sfq, tile_p, tile_q, 0);
          Stage::mma(tmem_base, dp, dq, sfp, sfq, 4, acc);
        } else {
          using Stage = MxStage<1, FMT, NT, 1, false>;
          Stage::copy_scales(sfp, sfq, tile_p, tile_q, ng);
          Stage::mma(tmem_base, dp, dq, sfp, sfq, steps, acc);
        }
        umma_commit<1>(bar_empty + 8 * stage);
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      if (ok) umma_commit<1>(bar_tfull);
      umma_commit<1>(bar_done);
      if (!mbar_wait_bounded(bar_done, 0, p.wait_ns)) fail(ST_DRAIN);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // TMEM -> fp32 partial sums in shared memory, [row of A][row of B]: consecutive lanes
    // write consecutive words. The ring is idle: the accumulator is complete, so every
    // load has landed and every MMA has read its stage.
    uint32_t okw = 0;
    if (lane == 0) {
      okw = mbar_wait(bar_tfull, 0, p.wait_ns, abort_flag) ? 1u : 0u;
      if (!okw) fail(ST_EPI_TMEM_FULL);
    }
    okw = __shfl_sync(0xffffffffu, okw, 0);
    tc_fence_after();
    if (okw) {
      const uint32_t quarter = warp & 3u;
      const uint32_t t_row = tmem_base + ((32u * quarter) << 16);
      float* part = reinterpret_cast<float*>(base_ptr) + 32u * quarter + lane;
#pragma unroll 2
      for (uint32_t c = 0; c < NT; c += 16) {
        uint32_t r[16];
        tmem_ld_x16(t_row + c, r);
        tmem_wait_ld();
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) part[(c + i) * 128u] = __uint_as_float(r[i]);
      }
    }
    tc_fence_before();
  }

  // ---- join the cluster's partial sums and store C ----
  // TMEM is released before the cluster barrier: a CTA never waits for another one while
  // it holds columns that a third one on its SM may be waiting to allocate.
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, Cfg::TMEM_COLS);
  }
  if (p.splits > 1) cluster_sync();
  if (*abort_flag) {
    // No copy may land after this CTA's shared memory is released. Looked at behind every
    // role's end: a role may give up long after the producer issued its last copy.
    if (warp == 0 && lane == 0) {
      const uint32_t issued = *issued_word;
      for (uint32_t i = issued > S ? issued - S : 0u; i < issued; ++i) {
        if (!mbar_wait_bounded(bar_full + 8 * (i % S), (i / S) & 1u, p.wait_ns)) {
          fail(ST_DRAIN);
          break;
        }
      }
    }
  } else {
    const SumScale scale(p.ts_p, p.ts_q);
    const uint32_t rows = min(uint32_t(NT), p.nq - q0);
    const uint32_t col = p0 + 4 * lane;
    const uint32_t ncol = col < p.np ? min(4u, p.np - col) : 0u;
    // warp w of cluster rank r takes rows w * splits + r, w * splits + r + 8 * splits, ...
    for (uint32_t r = warp * p.splits + rank; r < rows; r += 8 * p.splits) {
      const uint32_t off = base + (r * 128u + 4 * lane) * 4u;
      float4 v;
      if (p.splits == 1) {
        v = *reinterpret_cast<const float4*>(base_ptr + (r * 128u + 4 * lane) * 4u);
      } else {
        v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t s = 0; s < p.splits; ++s) {
          const float4 w = ld_shared_cluster_f4(mapa_shared(off, s));
          v.x += w.x;
          v.y += w.y;
          v.z += w.z;
          v.w += w.w;
        }
      }
      v.x = scale.apply<FMT>(v.x);
      v.y = scale.apply<FMT>(v.y);
      v.z = scale.apply<FMT>(v.z);
      v.w = scale.apply<FMT>(v.w);
      store_c4<CD>(p.c, uint64_t(q0 + r) * p.ldc + col, v, ncol, p.vec);
    }
  }
  // no CTA leaves while another one may still read its partial sums
  if (p.splits > 1) cluster_sync();
}

// ---------------------------------------------------------------------------------
// mx_gemm_pair_kernel: 256 x TN tiles of C per CTA pair (cta_group::2), persistent
// ---------------------------------------------------------------------------------
// Each CTA of the pair loads its 128 rows of A, half of the tile's rows of B and, since
// both SMs multiply by every column's scale, its own A scale band and all of B's. The
// leader issues the scale copies (cta_group::2: each CTA's TMEM from its own shared
// memory) and the MMAs. TMEM: two accumulator slots of MMA_N columns, then two buffers of
// scale columns, used by alternate stages. A tile of one MMA width uses the slots in turn
// (the epilogue of tile t overlaps the main loop of t + 1); TN = 384 uses both.
struct MxPairParams {
  uint32_t M, N, row_bytes;
  uint32_t m_tiles, n_tiles, num_tiles, k_atoms, group_m;
  const float* ts_a;
  const float* ts_b;
  uint8_t* c;
  uint64_t ldc;   // elements
  uint32_t align;  // of C's rows: 32, 16, 8, 4 or 2 bytes
  uint32_t* status;
  uint64_t wait_ns;
  uint32_t fault_inject;  // test hook: 1 = the producer issues no loads, 2 = the MMA warp gives up
};

template <int FMT, int TN>
struct MxPairCfg {
  static constexpr uint32_t MMA_N = TN == 384 ? 192 : TN;
  static constexpr uint32_t NH = TN / MMA_N;
  static constexpr uint32_t GROUPS = MxAtom<FMT>::GROUPS;
  // 128-row scale bands that a tile's TN columns touch (a 192-wide tile starts at a band
  // or in the middle of one)
  static constexpr uint32_t BANDS = TN == 128 ? 1 : TN == 384 ? 3 : 2;
  static constexpr uint32_t A_BYTES = 128 * 128;
  static constexpr uint32_t B_HALF = MMA_N / 2 * 128;  // one MMA's B rows of this CTA
  static constexpr uint32_t B_BYTES = NH * B_HALF;
  static constexpr uint32_t SFA_BYTES = GROUPS * 512;
  static constexpr uint32_t SFB_BYTES = BANDS * GROUPS * 512;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr uint32_t BAR_BYTES = 256;
  static constexpr uint32_t MAX_SMEM = 232448;
  static constexpr uint32_t EPI_GROUPS = MMA_N / 64;      // 64 columns per epilogue warp
  static constexpr uint32_t EPI_WARPS = 4 * EPI_GROUPS;
  static constexpr uint32_t EPI_BYTES = EPI_WARPS * 2048; // staging of C rows at odd pitches
  static constexpr uint32_t FIT = (MAX_SMEM - 1024 - BAR_BYTES - EPI_BYTES) / STAGE;
  static constexpr uint32_t STAGES = FIT > 8 ? 8 : FIT;
  static constexpr uint32_t SMEM = STAGES * STAGE + EPI_BYTES + BAR_BYTES + 1024;
  static constexpr uint32_t SF_COLS = 4 * GROUPS * (1 + BANDS);
  static constexpr uint32_t SF_COL = 2 * MMA_N;
  static constexpr uint32_t THREADS = 128 + 32 * EPI_WARPS;
  static_assert(SF_COL + 2 * SF_COLS <= 512, "accumulators and scales fit TMEM");
  static_assert(SMEM > MAX_SMEM / 2, "one CTA per SM: a second one could wait for its TMEM");
};

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* m, int32_t x, int32_t y, int32_t z,
                                                 uint32_t cluster_bar, uint64_t hint) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(cluster_bar), "l"(hint)
      : "memory");
}

// One lane's 64 accumulators of a C row, scaled and rounded: 32 words of a 16-bit type (then
// both halves of a TN = 384 tile fit the registers at once) or 64 of fp32.
template <int CD>
struct CRow {
  using E = typename OutElem<CD>::E;
  using T = typename E::T;
  static constexpr uint32_t PER = 4 / sizeof(T);  // columns per word
  uint32_t w[64 / PER];

  // from 32 accumulators, columns 32 * half on
  template <int FMT>
  __device__ __forceinline__ void set(uint32_t (&r)[32], uint32_t half, const SumScale& scale) {
    if constexpr (FMT == NV_FP4) {  // the other formats have no tensor scale
#pragma unroll
      for (uint32_t i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * scale.first);
      if (scale.second != 1.0f) {  // rare: a branch, not a multiplication each
#pragma unroll
        for (uint32_t i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * scale.second);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 32 / PER; ++i) {
      if constexpr (PER == 1) w[32 * half + i] = r[i];
      else w[16 * half + i] = E::pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    }
  }

  // Columns [32 * half, 32 * half + 32) as whole 32-byte sectors (a 32-byte aligned address).
  __device__ __forceinline__ void store(uint32_t half, uint8_t* c, uint64_t index) const {
    T* d = reinterpret_cast<T*>(c) + index;
#pragma unroll
    for (uint32_t j = 0; j < 4 / PER; ++j) {
      uint32_t v[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) v[i] = w[32 / PER * half + 8 * j + i];
      st_global_v8(d + 8 * PER * j, v);
    }
  }

  // The same for a warp's 32 rows at any pitch and column count: 64 bytes of each row go
  // through the warp's shared buffer (16-byte chunk j of row l at chunk j ^ (l / 2 % 4)) and
  // leave along the rows, VB bytes per lane: 8, 4, or one 16-bit element, as C is aligned.
  // One lane per row storing its own elements one by one touched 32 sectors per store (777 x
  // 5001 x 2200: 73 us, 12.5 this way). 4000 x N x 500 MXFP4 with N = 4000, 4004, 4002, 4001:
  // 10.9, 13.4, 15.3, 16.0 us; rows at odd addresses leave sectors in parts.
  template <uint32_t VB>
  __device__ __forceinline__ void store_any(uint32_t half, uint8_t* c, uint64_t ldc, uint32_t row0, uint32_t rows,
                                            uint32_t col0, uint32_t cols, uint32_t buf) const {
    const uint32_t lane = lane_id();
    constexpr uint32_t ES = sizeof(T), W = 64 / ES;  // columns per pass
    constexpr uint32_t LPR = 64 / VB;                // lanes per row
#pragma unroll
    for (uint32_t x = 0; x < 32; x += W) {
      const uint32_t* v = w + 32 / PER * half + x;  // x is 0 for 16-bit types
      __syncwarp();
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j)
        st_shared_v4(buf + lane * 64u + ((j ^ (lane / 2 & 3u)) << 4), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      __syncwarp();
      const uint32_t byte = lane % LPR * VB, col = x + byte / ES;
      T* d = reinterpret_cast<T*>(c) + uint64_t(row0) * ldc + col0 + col;
      const bool whole = col + VB / ES <= cols;
#pragma unroll 8
      for (uint32_t l0 = 0; l0 < 32; l0 += 32 / LPR) {
        const uint32_t l = l0 + lane / LPR;
        const uint32_t a = buf + l * 64u + (((byte / 16) ^ (l / 2 & 3u)) << 4) + byte % 16;
        T* at = d + uint64_t(l) * ldc;
        if constexpr (VB == 2) {
          uint16_t u;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(u) : "r"(a) : "memory");
          if (whole && l < rows) *reinterpret_cast<uint16_t*>(at) = u;
        } else {
          uint32_t u[VB / 4];
          if constexpr (VB == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u[0]) : "r"(a) : "memory");
          else asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u[0]), "=r"(u[VB / 4 - 1]) : "r"(a) : "memory");
          if (whole && l < rows) {
            if constexpr (VB == 4) *reinterpret_cast<uint32_t*>(at) = u[0];
            else *reinterpret_cast<uint2*>(at) = make_uint2(u[0], u[VB / 4 - 1]);
          } else if (col < cols && l < rows) {  // the last column falls inside
            const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
            for (uint32_t i = 0; i < VB / ES; ++i)
              if (col + i < cols) at[i] = e[i];
          }
        }
      }
    }
  }
};

template <int FMT, int CD, int TN>
__global__ void __launch_bounds__(MxPairCfg<FMT, TN>::THREADS, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                        const MxPairParams p) {
  using Cfg = MxPairCfg<FMT, TN>;
  using Atom = MxAtom<FMT>;
  constexpr uint32_t S = Cfg::STAGES, NH = Cfg::NH;
  extern __shared__ uint8_t smem_raw[];
  // Same offsets in both CTAs: the MMA and the scale copies read the peer's shared memory
  // at the leader's addresses, commits land on the peer's barriers.
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t sA = base, sB = sA + S * Cfg::A_BYTES;
  const uint32_t sSA = sB + S * Cfg::B_BYTES, sSB = sSA + S * Cfg::SFA_BYTES;
  const uint32_t sEpi = base + S * Cfg::STAGE, sBar = sEpi + Cfg::EPI_BYTES;
  uint8_t* bar_ptr = smem_raw + (sBar - raw);
  // full[8], empty[8], tfull[2], tempty[2], done, the TMEM address, the abort flag, the two
  // producers' issued-stage counts
  const uint32_t bar_full = sBar, bar_empty = sBar + 64, bar_tfull = sBar + 128, bar_tempty = sBar + 144;
  const uint32_t bar_done = sBar + 160;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_ptr + 168);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(bar_ptr + 172);
  const uint32_t abort_addr = sBar + 172;
  volatile uint32_t* issued_words = reinterpret_cast<volatile uint32_t*>(bar_ptr + 176);
  const uint32_t issued_addr = sBar + 176;

  const uint32_t warp = __shfl_sync(0xffffffffu, warp_id(), 0), lane = lane_id();
  // the cluster's rank in a form that the compiler knows to be uniform
  const uint32_t rank = blockIdx.x & 1u, peer = rank ^ 1u;
  if (warp == 0 && lane == 0) {
    for (uint32_t s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (uint32_t a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, Cfg::EPI_WARPS * 2);
    }
    mbar_init(bar_done, 1);
    *abort_flag = 0u;
    issued_words[0] = 0u;
    issued_words[1] = 0u;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(tmem_slot), 512);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  // Raises both CTAs' abort flags (the peer is alive: see the teardown).
  auto fail = [&](uint32_t code) {
    *abort_flag = 1u;
    st_shared_cluster_u32(mapa_shared(abort_addr, peer), 1u);
    if (p.status) atomicOr(p.status, code | ST_ABORTED);
  };
  auto acc_slot = [](uint32_t it, uint32_t h) -> uint32_t { return NH == 1 ? (it & 1u) : h; };
  auto acc_use = [](uint32_t it) -> uint32_t { return NH == 1 ? (it >> 1) : it; };
  const uint32_t first_tile = blockIdx.x / 2, tile_stride = gridDim.x / 2;

  if (warp == 0) {
    // =============================== TMA producer ===============================
    if (elect_one()) {
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = p.fault_inject != 1;
      const uint64_t hint_a = policy_evict_last(), hint_b = policy_evict_first();
      const uint32_t leader_full0 = mapa_shared(bar_full, 0);
      for (uint32_t tile = first_tile; tile < p.num_tiles && ok; tile += tile_stride) {
        uint32_t bm, bn;
        tile_to_bmn(tile, p.m_tiles, p.n_tiles, p.group_m, bm, bn);
        const int32_t a_row = int32_t((2 * bm + rank) * 128);
        const int32_t b_row = int32_t(bn * TN + rank * (Cfg::MMA_N / 2));
        const int32_t b_band = int32_t(bn * TN / 128);
        for (uint32_t kb = 0; kb < p.k_atoms; ++kb) {
          if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1u, p.wait_ns, abort_flag)) {
            fail(ST_PRODUCER_EMPTY);
            ok = false;
            break;
          }
          // both CTAs' bytes are credited to the leader's barrier, which the leader arms
          if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * stage, 2 * Cfg::STAGE);
          const uint32_t lf = leader_full0 + 8 * stage;
          const int32_t x = int32_t(kb * 128u), g = int32_t(kb * Cfg::GROUPS);
          tma_load_3d_pair(sSA + stage * Cfg::SFA_BYTES, &tmSA, 0, g, int32_t(2 * bm + rank), lf, hint_a);
          tma_load_3d_pair(sSB + stage * Cfg::SFB_BYTES, &tmSB, 0, g, b_band, lf, hint_b);
          tma_load_2d_pair(sA + stage * Cfg::A_BYTES, &tmA, x, a_row, lf, hint_a);
#pragma unroll
          for (uint32_t h = 0; h < NH; ++h)
            tma_load_2d_pair(sB + stage * Cfg::B_BYTES + h * Cfg::B_HALF, &tmB, x, b_row + int32_t(h * Cfg::MMA_N), lf,
                             hint_b);
          ++issued;
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      if (rank == 0) issued_words[0] = issued;
      else st_shared_cluster_u32(mapa_shared(issued_addr + 4, 0), issued);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ============================ MMA issuer (leader) ============================
    if (rank != 0) {
    } else if (elect_one()) {
      uint32_t stage = 0, phase = 0, it = 0, sf_buf = 0;
      bool ok = p.fault_inject != 2;
      if (!ok) fail(ST_MMA_FULL);
      for (uint32_t tile = first_tile; tile < p.num_tiles && ok; tile += tile_stride, ++it) {
        uint32_t bm, bn;
        tile_to_bmn(tile, p.m_tiles, p.n_tiles, p.group_m, bm, bn);
        const uint32_t band_shift = bn * TN % 128 / 32;  // scale columns before the tile's first
        for (uint32_t kb = 0; kb < p.k_atoms; ++kb) {
          if (!mbar_wait(bar_full + 8 * stage, phase, p.wait_ns, abort_flag)) {
            fail(ST_MMA_FULL);
            ok = false;
            break;
          }
          const uint32_t sfa = tmem_base + Cfg::SF_COL + sf_buf * Cfg::SF_COLS, sfb = sfa + 4 * Cfg::GROUPS;
          sf_buf ^= 1u;
          const uint64_t tile_a = sdesc_scale_tile(sSA + stage * Cfg::SFA_BYTES);
          const uint64_t tile_b = sdesc_scale_tile(sSB + stage * Cfg::SFB_BYTES);
          const uint64_t da = sdesc_k_sw128(sA + stage * Cfg::A_BYTES), db = sdesc_k_sw128(sB + stage * Cfg::B_BYTES);
          const uint32_t steps = min(4u, (p.row_bytes - kb * 128u + 31u) / 32u);
          const uint32_t acc = kb ? 1u : 0u;
          // boxes past the last scale tile read as zero, so every copy has its source
          MxStage<2, FMT, Cfg::MMA_N, Cfg::BANDS, true>::copy_scales(sfa, sfb, tile_a, tile_b, 0);
#pragma unroll
          for (uint32_t h = 0; h < NH; ++h) {
            const uint32_t slot = acc_slot(it, h);
            if (kb == 0) {
              if (!mbar_wait(bar_tempty + 8 * slot, (acc_use(it) & 1u) ^ 1u, p.wait_ns, abort_flag)) {
                fail(ST_MMA_TMEM_EMPTY);
                ok = false;
                break;
              }
              tc_fence_after();
            }
            const uint32_t sfb_h = sfb + (NH == 1 ? band_shift : h * Cfg::MMA_N / 32);
            const uint32_t d = tmem_base + slot * Cfg::MMA_N;
            const uint64_t db_h = db + h * (Cfg::B_HALF >> 4);
            if (steps == 4) MxStage<2, FMT, Cfg::MMA_N, Cfg::BANDS, true>::mma(d, da, db_h, sfa, sfb_h, 4, acc);
            else MxStage<2, FMT, Cfg::MMA_N, Cfg::BANDS, false>::mma(d, da, db_h, sfa, sfb_h, steps, acc);
            if (kb + 1 == p.k_atoms) umma_commit_pair(bar_tfull + 8 * slot, uint16_t(3u));
          }
          if (!ok) break;
          umma_commit_pair(bar_empty + 8 * stage, uint16_t(3u));
          if (++stage == S) { stage = 0; phase ^= 1u; }
        }
      }
      umma_commit<2>(bar_done);
      if (!mbar_wait_bounded(bar_done, 0, p.wait_ns)) fail(ST_DRAIN);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ================================ epilogue ================================
    // Warp 4 + 4e + q drains lanes 32q ... 32q + 31, columns 64e ... 64e + 63 of each slot
    // and hands the slot back before it stores. A lane owns one C row: its 64 columns are
    // whole 32-byte sectors, stored straight from registers.
    const uint32_t q = warp & 3u, e = (warp - 4) >> 2;
    const SumScale scale(p.ts_a, p.ts_b);
    const uint32_t leader_tempty0 = mapa_shared(bar_tempty, 0);
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t tile = first_tile; tile < p.num_tiles && ok; tile += tile_stride, ++it) {
      uint32_t bm, bn;
      tile_to_bmn(tile, p.m_tiles, p.n_tiles, p.group_m, bm, bn);
      const uint32_t row0 = (2 * bm + rank) * 128 + 32 * q;
      // Both halves of a 16-bit TN = 384 tile are drained before either is stored: the next
      // tile's MMAs wait for the drain, and behind half the stores of a tile it would come
      // a microsecond late.
      constexpr uint32_t HELD = CD == DT_F32 ? 1 : NH;
      CRow<CD> out[HELD];
#pragma unroll 1
      for (uint32_t h0 = 0; h0 < NH && ok; h0 += HELD) {
#pragma unroll
        for (uint32_t x = 0; x < HELD; ++x) {
          const uint32_t slot = acc_slot(it, h0 + x);
          uint32_t okw = 0;
          if (lane == 0) okw = mbar_wait(bar_tfull + 8 * slot, acc_use(it) & 1u, p.wait_ns, abort_flag) ? 1u : 0u;
          okw = __shfl_sync(0xffffffffu, okw, 0);
          if (!okw) {
            if (lane == 0) fail(ST_EPI_TMEM_FULL);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t t0 = tmem_base + ((32u * q) << 16) + slot * Cfg::MMA_N + 64u * e;
          uint32_t r[2][32];
          tmem_ld_x32(t0, r[0]);
          tmem_ld_x32(t0 + 32, r[1]);
          tmem_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty0 + 8 * slot);
          out[x].template set<FMT>(r[0], 0, scale);
          out[x].template set<FMT>(r[1], 1, scale);
        }
        if (!ok) break;
        if (row0 < p.M) {
#pragma unroll
          for (uint32_t x = 0; x < HELD; ++x) {
            const uint32_t col = bn * TN + (h0 + x) * Cfg::MMA_N + 64u * e;
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
              const uint32_t cx = col + 32u * half;
              const uint64_t at = uint64_t(row0 + lane) * p.ldc + cx;
              const uint32_t rows = min(32u, p.M - row0), cols = p.N - cx, buf = sEpi + (warp - 4) * 2048u;
              if (p.align == 32 && cx + 32 <= p.N) {
                if (lane < rows) out[x].store(half, p.c, at);
              } else if (cx < p.N) {
                if (p.align >= 8) out[x].template store_any<8>(half, p.c, p.ldc, row0, rows, cx, cols, buf);
                else if (CD == DT_F32 || p.align == 4)
                  out[x].template store_any<4>(half, p.c, p.ldc, row0, rows, cx, cols, buf);
                else if constexpr (CD != DT_F32)
                  out[x].template store_any<2>(half, p.c, p.ldc, row0, rows, cx, cols, buf);
              }
            }
          }
        }
        __syncwarp();
      }
    }
  }

  // ---- teardown: as the plain pair kernel's (gemm_sm100.cuh): after an abort the leader
  // waits for every stage still in flight before either CTA leaves ----
  tc_fence_before();
  cluster_sync();
  if (*abort_flag) {
    if (warp == 0 && lane == 0 && rank == 0) {
      const uint32_t il = issued_words[0], ip = issued_words[1];
      const uint32_t hi = il > ip ? il : ip;
      for (uint32_t i = hi > S ? hi - S : 0u; i < hi; ++i) {
        const uint32_t bar = bar_full + 8 * (i % S);
        if (i >= il) mbar_arrive_expect_tx(bar, Cfg::STAGE);
        else if (i >= ip) mbar_complete_tx(bar, Cfg::STAGE);
        if (!mbar_wait_bounded(bar, (i / S) & 1u, p.wait_ns)) {
          fail(ST_DRAIN);
          break;
        }
      }
    }
    cluster_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

}  // namespace b200
