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
// Untiled bulk copy into this CTA's shared memory; both addresses and the size are
// multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

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
};

// ---------------------------------------------------------------------------------
// mx_gemm_rows_kernel: 128 rows of B (P) x NT rows of A (Q) per CTA, K split over the
// CTAs of a cluster
// ---------------------------------------------------------------------------------
// The accumulator is C transposed: TMEM lane = row of B (column of C), column = row of A.
// With few rows of A the weights B are the long operand and take the MMA's 128-row side;
// the other side is only as wide as the tokens need (NT = 16 ... 256), so one token does
// not pay for 128. K is split over a cluster of up to 8 CTAs when the tiles alone leave
// SMs idle; the partial sums meet in distributed shared memory, added in rank order, so
// results do not depend on timing and no workspace or second launch is needed.
template <int FMT, int NT>
struct MxRowsCfg {
  static constexpr uint32_t GROUPS = MxAtom<FMT>::GROUPS;
  static constexpr uint32_t QB = NT > 128 ? NT / 128 : 1;  // scale bands of Q
  static constexpr uint32_t P_BYTES = 128 * 128;
  static constexpr uint32_t Q_BYTES = NT * 128;
  static constexpr uint32_t SFP_BYTES = GROUPS * 512;
  static constexpr uint32_t SFQ_BYTES = QB * GROUPS * 512;
  static constexpr uint32_t STAGE = P_BYTES + Q_BYTES + SFP_BYTES + SFQ_BYTES;
  static constexpr uint32_t BAR_BYTES = 256;
  static constexpr uint32_t MAX_SMEM = 232448;
  static constexpr uint32_t FIT = (MAX_SMEM - 1024 - BAR_BYTES) / STAGE;
  static constexpr uint32_t MAX_STAGES = FIT > 8 ? 8 : FIT;
  static constexpr uint32_t PARTIAL = NT * 128 * 4;  // overlays the ring after the main loop
  static constexpr uint32_t ACC_COLS = NT < 32 ? 32 : NT;
  static constexpr uint32_t SFP_COL = ACC_COLS;
  static constexpr uint32_t SFQ_COL = SFP_COL + 4 * GROUPS;
  static constexpr uint32_t COLS = SFQ_COL + 4 * GROUPS * QB;
  static constexpr uint32_t TMEM_COLS = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static uint32_t smem_bytes(uint32_t stages) {
    const uint32_t ring = stages * STAGE;
    return (ring > PARTIAL ? ring : PARTIAL) + BAR_BYTES + 1024;
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
  // full[8], empty[8], tfull, done; the TMEM address and the abort flag
  const uint32_t bar_full = sBar, bar_empty = sBar + 64, bar_tfull = sBar + 128, bar_done = sBar + 136;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + bar_off + 144);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_ptr + bar_off + 148);

  const uint32_t warp = warp_id(), lane = lane_id();
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
  const uint32_t q_bands = (p.nq + 127) / 128 - q0 / 128;  // scale bands left from this tile on
  const uint32_t qb = q_bands < Cfg::QB ? q_bands : Cfg::QB;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = true;
      const uint64_t hint_p = policy_evict_first(), hint_q = policy_evict_last();
      for (uint32_t kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(bar_empty + 8 * stage, phase ^ 1u, p.wait_ns, abort_flag)) {
          fail(ST_PRODUCER_EMPTY);
          ok = false;
          break;
        }
        const uint32_t g0 = kb * Cfg::GROUPS;
        const uint32_t ng = min(Cfg::GROUPS, p.groups - g0);
        const uint32_t bar = bar_full + 8 * stage;
        mbar_arrive_expect_tx(bar, Cfg::P_BYTES + Cfg::Q_BYTES + ng * 512u * (1u + qb));
        tma_load_2d(sP + stage * Cfg::P_BYTES, &tmP, int32_t(kb * 128u), int32_t(p0), bar, hint_p);
        tma_load_2d(sQ + stage * Cfg::Q_BYTES, &tmQ, int32_t(kb * 128u), int32_t(q0), bar, hint_q);
        bulk_load(sSP + stage * Cfg::SFP_BYTES, p.sf_p + (uint64_t(tp) * p.groups + g0) * 512u, ng * 512u, bar);
        for (uint32_t b = 0; b < qb; ++b)
          bulk_load(sSQ + stage * Cfg::SFQ_BYTES + b * Cfg::SFP_BYTES,
                    p.sf_q + (uint64_t(q0 / 128 + b) * p.groups + g0) * 512u, ng * 512u, bar);
        ++issued;
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      if (!ok || *abort_flag) {
        // no copy may land after this CTA's shared memory is released
        for (uint32_t i = issued > S ? issued - S : 0u; i < issued; ++i) {
          if (!mbar_wait_bounded(bar_full + 8 * (i % S), (i / S) & 1u, p.wait_ns)) {
            fail(ST_DRAIN);
            break;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (uint32_t kb = k0; kb < k1; ++kb) {
        if (!mbar_wait(bar_full + 8 * stage, phase, p.wait_ns, abort_flag)) {
          fail(ST_MMA_FULL);
          ok = false;
          break;
        }
        const uint32_t ng = min(Cfg::GROUPS, p.groups - kb * Cfg::GROUPS);
        const uint32_t steps = min(4u, (p.row_bytes - kb * 128u + 31u) / 32u);
#pragma unroll
        for (uint32_t g = 0; g < Cfg::GROUPS; ++g) {
          if (g < ng) {
            tmem_cp_scales<1>(tmem_base + Cfg::SFP_COL + 4 * g,
                              sdesc_scale_tile(sSP + stage * Cfg::SFP_BYTES + g * 512u));
#pragma unroll
            for (uint32_t b = 0; b < Cfg::QB; ++b)
              if (b < qb)
                tmem_cp_scales<1>(tmem_base + Cfg::SFQ_COL + 4 * (Cfg::QB * g + b),
                                  sdesc_scale_tile(sSQ + stage * Cfg::SFQ_BYTES + b * Cfg::SFP_BYTES + g * 512u));
          }
        }
        const uint32_t a0 = sP + stage * Cfg::P_BYTES, b0 = sQ + stage * Cfg::Q_BYTES;
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
          if (s < steps)
            umma_mx<1, FMT>(tmem_base, sdesc_k_sw128(a0 + 32u * s), sdesc_k_sw128(b0 + 32u * s),
                            idesc_mx<FMT>(128, NT, Atom::sf_id(s)), tmem_base + Cfg::SFP_COL + 4 * Atom::group(s),
                            tmem_base + Cfg::SFQ_COL + 4 * Cfg::QB * Atom::group(s), (kb != k0 || s != 0) ? 1u : 0u);
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
  if (!*abort_flag) {
    float scale = 1.0f;
    if (p.ts_p) scale *= __ldg(p.ts_p);
    if (p.ts_q) scale *= __ldg(p.ts_q);
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
      v.x *= scale;
      v.y *= scale;
      v.z *= scale;
      v.w *= scale;
      store_c4<CD>(p.c, uint64_t(q0 + r) * p.ldc + col, v, ncol, p.vec);
    }
  }
  // no CTA leaves while another one may still read its partial sums
  if (p.splits > 1) cluster_sync();
}

}  // namespace b200
