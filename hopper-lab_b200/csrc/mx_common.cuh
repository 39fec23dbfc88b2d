// mx_common.cuh — the microscaled formats: constants, scale-tile addressing and the
// device conversions shared by the quantiser, the RMS norm and the dequantiser.
//
// A microscaled matrix stores, for each row, elements of 8 or 4 bits and one scale per
// block of consecutive elements:
//   MX_FP8  e4m3 elements, blocks of 32, scale 2^(byte - 127)   (e8m0, 0xFF = NaN)
//   MX_FP4  e2m1 elements, blocks of 32, scale 2^(byte - 127)
//   NV_FP4  e2m1 elements, blocks of 16, scale e4m3 (0x7F = NaN), fp32 scale per tensor
// Rows are padded with zero elements to a multiple of 32. Scale bytes are stored as the
// tensor core's scale operand reads them: tiles of 128 rows x 4 blocks, 512 bytes each,
// row r and block c of a tile at byte (r % 32) * 16 + (r / 32) * 4 + c; the tiles of a
// 128-row band follow one another along the row, padding bytes are zero.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace b200 {

enum : int { MX_FP8 = 0, MX_FP4 = 1, NV_FP4 = 2 };

template <int FMT>
struct MxFmt {
  static constexpr int BITS = (FMT == MX_FP8) ? 8 : 4;
  static constexpr int BLOCK = (FMT == NV_FP4) ? 16 : 32;
};

__host__ __device__ constexpr int mx_block(int fmt) { return fmt == NV_FP4 ? 16 : 32; }
__host__ __device__ constexpr int64_t mx_padded_cols(int64_t cols) { return (cols + 31) / 32 * 32; }
__host__ __device__ constexpr int64_t mx_row_bytes(int fmt, int64_t cols) {
  return fmt == MX_FP8 ? mx_padded_cols(cols) : mx_padded_cols(cols) / 2;
}
// scale tiles along one row band: groups of four blocks
__host__ __device__ constexpr int64_t mx_groups(int fmt, int64_t cols) {
  return (mx_padded_cols(cols) / mx_block(fmt) + 3) / 4;
}
__host__ __device__ constexpr int64_t mx_scale_bytes(int fmt, int64_t rows, int64_t cols) {
  return (rows + 127) / 128 * mx_groups(fmt, cols) * 512;
}
// byte offset of the four scales of (row, group)
__host__ __device__ constexpr int64_t mx_scale_word(int64_t row, int64_t group, int64_t groups) {
  return ((row / 128) * groups + group) * 512 + (row % 32) * 16 + (row % 128) / 32 * 4;
}

// ---------------------------------------------------------------------------------
// input / output element types (the B200_DT_* codes)
// ---------------------------------------------------------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<0> {
  using T = __half;
  static __device__ __forceinline__ float load(T v) { return __half2float(v); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ T store(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<1> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float load(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ T store(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<3> {
  using T = float;
  static __device__ __forceinline__ float load(T v) { return v; }
  static __device__ __forceinline__ T store(float v) { return v; }
};

// Untiled bulk copy into this CTA's shared memory; both addresses and the size are
// multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// 32 bytes in one access (sm_100's widest), for a 32-byte aligned address.
__device__ __forceinline__ void ld_global_v8(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
// The same, kept in L1: for data that a CTA reads again.
__device__ __forceinline__ void ld_global_v8_l1(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// W words of a row of `len` elements that starts at any element-aligned address, from element
// c on: the whole 16-byte chunks around them, shifted into place (word selects and one funnel
// shift, the same code for every offset). Elements read one by one touch 16 times as many
// sectors. A chunk that reaches outside the row is put together from its elements inside, so
// nothing beside the row is read (a strided matrix's gaps may hold what another stream writes)
// and what lies behind its end is zero. Host code too, for the test of its addresses.
template <int DT, int W>
__host__ __device__ __forceinline__ void load_words_any(const typename Elem<DT>::T* row, int64_t len, int64_t c0,
                                                        uint32_t (&r)[W]) {
  constexpr int ES = sizeof(typename Elem<DT>::T);
  const uintptr_t a = reinterpret_cast<uintptr_t>(row + c0);
  const int o = int(a & 15);
  // bytes of the row ahead of c0 and from it on, as far as they matter here
  const int lead = int(c0 < 16 ? c0 : 16) * ES, rest = int(len - c0 < 64 ? len - c0 : 64) * ES;
  const char* base = reinterpret_cast<const char*>(a - o);
  uint32_t w[W + 4];
#pragma unroll
  for (int c = 0; c <= W / 4; ++c) {
    const int at = 16 * c - o;  // the chunk's place relative to c0
    uint4 v = make_uint4(0, 0, 0, 0);
    if (c < W / 4 || o != 0) {
      if (at >= -lead && at + 16 <= rest) {
        v = *reinterpret_cast<const uint4*>(base + 16 * c);
      } else {
        uint32_t e[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16 / ES; ++i) {
          const char* q = base + 16 * c + ES * i;
          if (at + ES * i >= -lead && at + ES * (i + 1) <= rest) {
            if constexpr (ES == 2) e[i / 2] |= uint32_t(*reinterpret_cast<const uint16_t*>(q)) << (16 * (i & 1));
            else e[i] = *reinterpret_cast<const uint32_t*>(q);
          }
        }
        v = make_uint4(e[0], e[1], e[2], e[3]);
      }
    }
    w[4 * c] = v.x;
    w[4 * c + 1] = v.y;
    w[4 * c + 2] = v.z;
    w[4 * c + 3] = v.w;
  }
  uint32_t t[W + 3], u[W + 1];
#pragma unroll
  for (int i = 0; i < W + 3; ++i) t[i] = (o & 4) ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < W + 1; ++i) u[i] = (o & 8) ? t[i + 2] : t[i];
#pragma unroll
  for (int i = 0; i < W; ++i)
    r[i] = ES == 2 ? uint32_t((uint64_t(u[i + 1]) << 32 | u[i]) >> ((o & 2) * 8)) : u[i];
}

// 16 consecutive elements as they lie in memory (two to a register for 16-bit types).
template <int DT>
struct Raw16 {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr bool PACKED = sizeof(T) == 2;
  uint32_t r[PACKED ? 8 : 16];

  // `wide`: the address is 32-byte aligned and all 16 exist; otherwise the `n` existing
  // ones are read one by one and the rest are zero.
  template <bool KEEP = false>
  __device__ __forceinline__ void load(const T* p, bool wide, int n) {
    if (wide) {
      uint32_t(&lo)[8] = *reinterpret_cast<uint32_t(*)[8]>(r);
      if constexpr (KEEP) ld_global_v8_l1(p, lo);
      else ld_global_v8(p, lo);
      if constexpr (!PACKED) {
        uint32_t(&hi)[8] = *reinterpret_cast<uint32_t(*)[8]>(r + 8);
        if constexpr (KEEP) ld_global_v8_l1(p + 8, hi);
        else ld_global_v8(p + 8, hi);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        uint32_t e = 0;
        if (i < n) {
          if constexpr (PACKED) e = *reinterpret_cast<const uint16_t*>(p + i);
          else e = __float_as_uint(p[i]);
        }
        if constexpr (!PACKED) r[i] = e;
        else if (i & 1) r[i / 2] |= e << 16;
        else r[i / 2] = e;
      }
    }
  }
  // Elements c to c + 15 of a row of `len` at any element-aligned address: the existing ones,
  // the rest zero.
  __host__ __device__ __forceinline__ void load_any(const T* row, int64_t len, int64_t c) {
    constexpr int W = PACKED ? 8 : 16;
    if (c < len) {
      load_words_any<DT, W>(row, len, c, r);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) r[i] = 0;
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[16]) const {
    if constexpr (PACKED) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f = E::unpack(r[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
    }
  }
};

// 16 consecutive elements as fp32; `wide` and `n` as above, KEEP: through L1.
template <int DT, bool KEEP = false>
__device__ __forceinline__ void load16(const typename Elem<DT>::T* p, bool wide, int n, float (&v)[16]) {
  Raw16<DT> w;
  w.template load<KEEP>(p, wide, n);
  w.unpack(v);
}

// Store 16 fp32 values rounded to the element type; `wide` and `n` as above.
template <int DT>
__device__ __forceinline__ void store16(typename Elem<DT>::T* p, bool wide, int n, const float (&v)[16]) {
  using E = Elem<DT>;
  if (wide) {
    uint32_t r[8];
    if constexpr (sizeof(typename E::T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = E::pack(v[2 * i], v[2 * i + 1]);
      st_global_v8(p, r);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[i]);
      st_global_v8(p, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[8 + i]);
      st_global_v8(p + 8, r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = E::store(v[i]);
  }
}

template <int DT>
__device__ __forceinline__ void load16_any(const typename Elem<DT>::T* row, int64_t len, int64_t c, float (&v)[16]) {
  Raw16<DT> w;
  w.load_any(row, len, c);
  w.unpack(v);
}

// Store 16 fp32 values per lane, rounded, to a row that starts at any element-aligned
// address: they change hands in shared memory (256 at a time, kStageFloats of it per warp)
// and leave lanes side by side. A lane storing its own 16 one by one touches 32 sectors per
// store (1001 x 5003 to bf16: the dequantiser took 34 us that way, 5.3 this way; 7.7 with
// whole 16-byte chunks shifted together across lanes, whose ragged ends cost more than they
// save). All lanes take part; `p` is the warp's first element, of which `n` exist (n may be
// negative).
constexpr int kStageFloats = 272;  // 256 and one of padding per 16
template <int DT>
__device__ __forceinline__ void warp_store16(typename Elem<DT>::T* p, int64_t n, float* stage, const float (&v)[16]) {
  const uint32_t lane = lane_id();
#pragma unroll
  for (uint32_t half = 0; half < 2; ++half) {
    __syncwarp();
    if (lane / 16 == half) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) stage[lane % 16 * 17 + i] = v[i];
    }
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t k = 32 * i + lane;
      if (int64_t(256 * half + k) < n) p[256 * half + k] = Elem<DT>::store(stage[k + k / 16]);
    }
  }
}

// ---------------------------------------------------------------------------------
// element and scale conversions
// ---------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}
// eight fp32 -> eight e2m1 (nearest, ties to even, saturating at 6), first in the low bits
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t byte) {
  uint32_t h2;
  const uint16_t b = uint16_t(byte);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(b));
  return __half22float2(*reinterpret_cast<const __half2*>(&h2)).x;
}

// Largest magnitude of n values (n even) as a bit pattern, with "holds a NaN or an
// infinity" folded in: a NaN survives max.NaN, non-negative patterns order as integers, and
// every non-finite one is at or above 0x7F800000.
template <int N>
__device__ __forceinline__ uint32_t amax_bits(const float* v) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(v[i]), "f"(v[i + 1]));
  return __float_as_uint(m) & 0x7FFFFFFFu;
}

// The same of packed 16-bit values, two patterns at a time (their order is that of unsigned
// integers too): the maximum of the low halves and of the high ones.
template <int N>
__device__ __forceinline__ uint32_t amax_packed(const uint32_t* r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; i += 2) m = __vimax3_u16x2(m, r[i] & 0x7FFF7FFFu, r[i + 1] & 0x7FFF7FFFu);
  return m;
}
// fp32 pattern of a 16-bit magnitude pattern in the low half; non-finite stays non-finite.
template <int DT>
__device__ __forceinline__ uint32_t widen_bits(uint32_t h) {
  return __float_as_uint(Elem<DT>::unpack(h & 0xFFFFu).x);
}
template <int DT>
__device__ __forceinline__ uint32_t amax_raw(const Raw16<DT>& w) {
  if constexpr (Raw16<DT>::PACKED) {
    const uint32_t m = amax_packed<8>(w.r);
    return widen_bits<DT>(max(m & 0xFFFFu, m >> 16));
  } else {
    return amax_bits<16>(reinterpret_cast<const float*>(w.r));
  }
}

// Scale byte of an MX block with largest magnitude `amax` (bits as above): the smallest
// e >= -127 with amax <= QMAX * 2^e, so no element saturates (a floor of the exponent
// alone would clip blocks whose largest element's significand exceeds QMAX's). With
// amax = m * 2^k, 1 <= m < 2, and QMAX = q * 2^EMAX: e = k - EMAX, one more when m > q.
// Significands compare as the pattern's low 23 bits. Subnormal amax gives e below -127,
// clamped. Non-finite: 0xFF (NaN).
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  constexpr int EMAX = (FMT == MX_FP8) ? 8 : 2;
  constexpr uint32_t Q = (FMT == MX_FP8) ? 0x600000u : 0x400000u;  // 448 = 1.75 * 2^8, 6 = 1.5 * 2^2
  if (amax >= 0x7F800000u) return 0xFFu;
  const int byte = int(amax >> 23) - EMAX + ((amax & 0x7FFFFFu) > Q ? 1 : 0);
  return uint32_t(byte < 0 ? 0 : byte);
}
// 2^(127 - byte), the multiplier that brings the block into the element's range. Exact:
// byte is at most 253 for a finite block, so the result is a normal number; the product
// with an element rounds only where it is subnormal, far below the smallest element.
__device__ __forceinline__ float mx_inverse_scale(uint32_t byte) {
  return byte == 0xFFu ? __uint_as_float(0x7FC00000u) : __uint_as_float((254u - byte) << 23);
}

// NV_FP4 block scale: nearest e4m3 to min(fl(amax * fl(1/6)), 448). The product with the
// rounded reciprocal is the definition (one multiplication, the same everywhere); it is
// within 2^-23 of amax / 6, so a scale differs from the exact quotient's only next to a
// border between two e4m3 values.
__device__ __forceinline__ uint32_t nv_scale_byte(uint32_t amax) {
  if (amax >= 0x7F800000u) return 0x7Fu;
  const float s = fminf(__uint_as_float(amax) * (1.0f / 6.0f), 448.0f);
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(s));
  return r & 0xFFu;
}

// u / s for one NV_FP4 block: one Newton residual step on u * (1/s) with fused
// multiply-adds (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990) gives the correctly rounded quotient for the 4-bit
// significand of s. A border t between two e2m1 values has 3 significant bits, so t * s has 7
// and is an fp32 number: a u that differs from it does so by at least a unit of its last
// place, which is more than half a unit of the quotient's, and no such quotient rounds onto
// t. Ties between e2m1 values therefore fall as those of the exact quotient. Nothing
// overflows: u / s is below 10 unless s = 448, the largest scale, and then it is below u.
struct NvInverse {
  float s, r;
  __device__ __forceinline__ explicit NvInverse(uint32_t byte) {
    s = e4m3_to_f32(byte);
    r = s > 0.0f ? __frcp_rn(s) : (byte == 0x7Fu ? s : 0.0f);  // s = 0: every element 0; NaN stays NaN
  }
  __device__ __forceinline__ float quotient(float u) const {
    const float y = u * r;
    return fmaf(fmaf(-y, s, u), r, y);
  }
};

// 16 scaled values to their element bytes.
template <int FMT>
__device__ __forceinline__ void mx_pack16(const float (&v)[16], uint32_t (&out)[4]) {
  if constexpr (FMT == MX_FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = cvt_e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    out[0] = cvt_e2m1x8(v);
    out[1] = cvt_e2m1x8(v + 8);
  }
}

// Quantise 16 consecutive fp32 values of one row, `amax` their largest magnitude's bits, and
// return their bytes and scale byte. Blocks of 32 are shared by lanes 2i and 2i + 1 (all
// lanes of the warp take part).
template <int FMT>
__device__ __forceinline__ uint32_t mx_quantize16(float (&v)[16], uint32_t amax, uint32_t (&out)[4]) {
  if constexpr (MxFmt<FMT>::BLOCK == 32) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  uint32_t byte;
  if constexpr (FMT == NV_FP4) {
    byte = nv_scale_byte(amax);
    const NvInverse inv(byte);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = inv.quotient(v[i]);
  } else {
    byte = mx_scale_byte<FMT>(amax);
    const float m = mx_inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] *= m;
  }
  mx_pack16<FMT>(v, out);
  return byte;
}

// Four consecutive blocks' scale bytes of this lane's group as one word, valid in the
// group's first lane (8 lanes for blocks of 32, 4 lanes for blocks of 16).
template <int FMT>
__device__ __forceinline__ uint32_t mx_gather_scales(uint32_t byte) {
  if constexpr (MxFmt<FMT>::BLOCK == 32) {
    uint32_t w = byte | (__shfl_down_sync(0xffffffffu, byte, 2) << 8);
    return w | (__shfl_down_sync(0xffffffffu, w, 4) << 16);
  } else {
    uint32_t w = byte | (__shfl_down_sync(0xffffffffu, byte, 1) << 8);
    return w | (__shfl_down_sync(0xffffffffu, w, 2) << 16);
  }
}
template <int FMT>
constexpr int kLanesPerGroup = MxFmt<FMT>::BLOCK == 32 ? 8 : 4;

}  // namespace b200
