// mx_quant.cu — microscaled quantiser, dequantiser and RMS norm (formats: mx_common.cuh).
//
//   quantise     rows of x, or of x transposed, to elements + block scales
//   dequantise   element * block scale (exact) * tensor scale in fp32, to f16 / bf16 / f32
//   RMS norm     h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight; y quantised
//
// All are streaming passes bound by HBM: per element they read and write what the
// tensors hold once (bf16 to MX_FP8: 2 + 1.03 bytes). One thread owns 16 consecutive
// elements of a row: one 32-byte load for 16-bit types, one NV_FP4 block or half a block
// of 32 (a shuffle joins the halves), 16 or 8 bytes out.
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

#include "b200gemm.h"
#include "gemm_internal.h"
#include "mx_common.cuh"

namespace {

using namespace b200;

// ---------------------------------------------------------------------------------
// per-tensor scale of NV_FP4: amax * fl(1 / (6 * 448))
// ---------------------------------------------------------------------------------
// The first kernel leaves one maximum of finite magnitudes per cluster of CTAs behind the
// scale, at most kPartials; every warp of the quantiser reduces them again (the maximum does
// not depend on the order) and the first CTA writes the scale. No counter or flag has to
// start at zero, so there is no memset, and the quantiser's launch overlaps the first
// kernel's end.
constexpr int kPartials = 64;
constexpr int kAmaxCluster = 8;
static_assert(16 + kPartials * 4 <= B200_MX_SCALE_BYTES, "scratch behind the tensor scale");

__global__ void mx_unit_scale_kernel(float* ts) {
  griddep_wait();
  *ts = 1.0f;
}

struct AmaxParams {
  const void* x;
  int64_t rows, cols, ld, segs;  // segs: 512-element segments per row
  int32_t wide;
  float* partials;
};

// WIDE: every row starts on 32 bytes. One 512-element segment per warp and step, four (two
// of fp32) in flight.
template <int DT, bool WIDE>
__global__ void __launch_bounds__(256, 4) mx_amax_kernel(const AmaxParams p) {
  cluster_arrive_started();
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  constexpr int FLY = sizeof(T) == 2 ? (WIDE ? 4 : 2) : (WIDE ? 2 : 1);
  __shared__ uint32_t red[8];
  __shared__ uint32_t part[kAmaxCluster];
  const T* x = static_cast<const T*>(p.x);
  const int64_t tasks = p.rows * p.segs;
  const uint32_t lane = lane_id(), warp = warp_id();
  const int64_t step = int64_t(gridDim.x) * 8;
  const auto segment = [&](int64_t t, Raw16<DT>& w) {
    const int64_t row = p.rows == 1 ? 0 : t >> 32 ? t / p.segs : uint32_t(t) / uint32_t(p.segs);
    const int64_t c0 = (t - row * p.segs) * 512, left = p.cols - c0;
    const T* src = x + row * p.ld + c0;
    const int64_t rest = left - 16 * int64_t(lane);
    const int n = rest < 16 ? int(rest) : 16;
    if constexpr (WIDE) w.load(src + 16 * lane, n == 16, n);
    else w.load_any(x + row * p.ld, p.cols, c0 + 16 * int64_t(lane));
  };
  uint32_t m = 0;
  const auto fold = [&](const Raw16<DT>& w) {
    const uint32_t a = amax_raw<DT>(w);
    if (a < 0x7F800000u) {
      m = max(m, a);
    } else {  // rare: something in it does not count
      float v[16];
      w.unpack(v);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        if (b < 0x7F800000u) m = max(m, b);
      }
    }
  };
  int64_t t = int64_t(blockIdx.x) * 8 + warp;
  for (; t + (FLY - 1) * step < tasks; t += FLY * step) {
    Raw16<DT> w[FLY];
#pragma unroll
    for (int i = 0; i < FLY; ++i) segment(t + i * step, w[i]);
#pragma unroll
    for (int i = 0; i < FLY; ++i) fold(w[i]);
  }
  for (; t < tasks; t += step) {
    Raw16<DT> w;
    segment(t, w);
    fold(w);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  cluster_wait();  // the first CTA of the cluster has started: its shared memory is there
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, red[i]);
    st_shared_cluster_u32(mapa_shared(smem_u32(part + cluster_ctarank()), 0), m);
  }
  cluster_sync();
  if (cluster_ctarank() == 0 && threadIdx.x == 0) {
    const uint32_t n = cluster_nctarank();
    for (uint32_t i = 0; i < n; ++i) m = max(m, part[i]);
    p.partials[blockIdx.x / n] = __uint_as_float(m);
  }
}

// The tensor scale from `n` <= 64 partial maxima, in every lane of the warp; kept normal so
// that its reciprocal is finite. Ordinary loads, here and of given tensor scales: an earlier
// kernel of the stream may have written them after this one was launched, which the
// read-only path does not allow for, and reading past L1 (every warp the same line of L2)
// took 10 us of a 17 us launch at 2048 x 4096.
__device__ __forceinline__ float tensor_scale_from(const float* partials, uint32_t n) {
  const uint32_t lane = lane_id();
  uint32_t m = lane < n ? __float_as_uint(partials[lane]) : 0u;
  if (lane + 32 < n) m = max(m, __float_as_uint(partials[lane + 32]));
  m = __reduce_max_sync(0xffffffffu, m);
  return m ? fmaxf(__uint_as_float(m) * (1.0f / 2688.0f), 1.17549435e-38f) : 1.0f;
}

// ---------------------------------------------------------------------------------
// quantise along the rows
// ---------------------------------------------------------------------------------
struct QuantParams {
  const void* x;
  int64_t rows, cols, ldx;  // of the quantised matrix (after the transposition, if any)
  uint8_t* data;
  uint8_t* scales;
  float* tensor_scale;    // may be null
  const float* partials;  // not null: find the tensor scale from these and store it
  uint32_t n_partials;
  int64_t ld;             // bytes
  int64_t groups;
  int32_t wide;
};

// Reciprocal of the tensor scale that an NV_FP4 quantiser works with (1 without one).
__device__ __forceinline__ float scale_reciprocal(const QuantParams& p) {
  if (p.partials) {
    const float ts = tensor_scale_from(p.partials, p.n_partials);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.tensor_scale = ts;
    return __frcp_rn(ts);
  }
  return p.tensor_scale ? __frcp_rn(*p.tensor_scale) : 1.0f;
}

// One warp per CH segments of 512 consecutive elements of a row; rows run on to a multiple
// of 128 so that the padding bytes of the last scale tiles are written (as zero). WIDE:
// every row starts on 32 bytes.
template <int FMT, int DT, int CH, bool WIDE>
__global__ void __launch_bounds__(256) mx_quant_rows_kernel(const QuantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  const uint32_t lane = lane_id(), warp = warp_id();
  const uint32_t warps_per_row = uint32_t((p.groups * 4 * MxFmt<FMT>::BLOCK + 512 * CH - 1) / (512 * CH));
  const int64_t t = int64_t(blockIdx.x) * 8 + warp;
  const int64_t row = t >> 32 ? t / warps_per_row : uint32_t(t) / warps_per_row;
  if (row >= (p.rows + 127) / 128 * 128) return;  // whole warps
  const int64_t c0 = (t - row * warps_per_row) * (512 * CH);
  const T* x = static_cast<const T*>(p.x);
  const T* src = x + row * p.ldx + c0;
  Raw16<DT> w[CH];
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int64_t left = row < p.rows ? p.cols - c0 - 512 * ch : 0;
    const int64_t rest = left - 16 * int64_t(lane);
    const int n = rest < 16 ? int(rest) : 16;
    if constexpr (WIDE) w[ch].load(src + 512 * ch + 16 * lane, n == 16, n);
    else w[ch].load_any(x + row * p.ldx, row < p.rows ? p.cols : 0, c0 + 512 * ch + 16 * int64_t(lane));
  }
  float r = 1.0f;
  if constexpr (FMT == NV_FP4) r = scale_reciprocal(p);
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int64_t c = c0 + 512 * ch + 16 * lane;
    uint32_t amax = amax_raw<DT>(w[ch]);
    float v[16];
    w[ch].unpack(v);
    if constexpr (FMT == NV_FP4) {  // r > 0 and rounding are monotone: the largest stays the largest
      amax = __float_as_uint(__uint_as_float(amax) * r);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= r;
    }
    uint32_t q[4];
    const uint32_t word = mx_gather_scales<FMT>(mx_quantize16<FMT>(v, amax, q));
    const int64_t g = c / (4 * MxFmt<FMT>::BLOCK);
    if (lane % kLanesPerGroup<FMT> == 0 && g < p.groups)
      *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, g, p.groups)) = word;
    if (row < p.rows && c < mx_padded_cols(p.cols)) {
      uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
      if constexpr (FMT == MX_FP8) *reinterpret_cast<uint4*>(d) = make_uint4(q[0], q[1], q[2], q[3]);
      else *reinterpret_cast<uint2*>(d) = make_uint2(q[0], q[1]);
    }
  }
}

// ---------------------------------------------------------------------------------
// quantise along the columns of x: q = quantise(x^T)
// ---------------------------------------------------------------------------------
// A CTA takes 128 rows (k) x 64 columns of x through shared memory. A thread then owns two
// output rows (columns of x) and a 32-long piece of k: lane = 8 columns or column pairs x 4
// pieces, so four lanes write 128 (64) consecutive bytes of one output row. 16-bit types are
// read as pairs of neighbouring columns, fp32 as single ones 32 apart; both sit flipped by
// 8 * piece (in pairs or columns), so the four pieces' reads fall into different banks.
template <int DT>
struct ColsTile {
  using E = Elem<DT>;
  using T = typename E::T;
  static constexpr bool PAIRS = sizeof(T) == 2;
  static constexpr int VEC = 16 / sizeof(T);  // elements per 16-byte access
  // place of column c in a tile row of piece s (a 16-byte vector never straddles a flip)
  static __device__ __forceinline__ int place(int c, int s) { return c ^ (PAIRS ? 16 * s : 8 * s); }
};

template <int FMT, int DT>
__global__ void __launch_bounds__(128) mx_quant_cols_kernel(const QuantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using Tile = ColsTile<DT>;
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int kVec = Tile::VEC;
  __shared__ alignas(16) T tile[128][64];
  float r = 1.0f;
  if constexpr (FMT == NV_FP4) r = scale_reciprocal(p);
  const uint32_t strips = uint32_t((p.rows + 127) / 128 * 2);
  const int64_t k0 = int64_t(blockIdx.x / strips) * 128;  // x row
  const int64_t c0 = int64_t(blockIdx.x % strips) * 64;   // x column = output row
  const T* x = static_cast<const T*>(p.x);
  const int64_t kleft = p.cols - k0, cleft = p.rows - c0;
  if (p.wide) {
    // asynchronous copies: the whole tile is in flight and takes no registers (8192 x 8192
    // fp32 72 us through registers, eight at a time); what lies outside x reads as zero
    constexpr int kPerRow = 64 / kVec;
#pragma unroll
    for (int j = 0; j < kPerRow; ++j) {
      const int i = j * 128 + threadIdx.x, k = i / kPerRow, c = i % kPerRow * kVec;
      const int64_t left = k < kleft ? cleft - c : 0;
      const uint32_t bytes = left >= kVec ? 16u : left > 0 ? uint32_t(left) * sizeof(T) : 0u;
      const T* src = bytes ? x + (k0 + k) * p.ldx + c0 + c : x;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&tile[k][Tile::place(c, k / 32)])),
                   "l"(src), "r"(bytes)
                   : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    constexpr int kPerRow = 64 / kVec;
#pragma unroll 4
    for (int i = threadIdx.x; i < 128 * kPerRow; i += 128) {
      const int k = i / kPerRow, c = i % kPerRow * kVec;
      uint32_t w[4] = {0, 0, 0, 0};
      if (k < kleft && c < cleft) load_words_any<DT, 4>(x + (k0 + k) * p.ldx, p.rows, c0 + c, w);
      *reinterpret_cast<uint4*>(&tile[k][Tile::place(c, k / 32)]) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncthreads();
  const uint32_t lane = lane_id();
  const int piece = lane & 3, slot = warp_id() * 8 + (lane >> 2);
  constexpr int NB = 32 / MxFmt<FMT>::BLOCK;
  uint32_t pairs[Tile::PAIRS ? 32 : 1], two[NB];  // two: both columns' block maxima
  if constexpr (Tile::PAIRS) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      pairs[i] = *reinterpret_cast<const uint32_t*>(&tile[32 * piece + i][Tile::place(2 * slot, piece)]);
#pragma unroll
    for (int b = 0; b < NB; ++b) two[b] = amax_packed<32 / NB>(pairs + b * (32 / NB));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int col = Tile::PAIRS ? 2 * slot + h : slot + 32 * h;
    const int64_t row = c0 + col;  // output row
    uint32_t byte[2];
    uint32_t q[8];
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if constexpr (Tile::PAIRS) {
        const float2 f = E::unpack(pairs[i]);
        v[i] = h ? f.y : f.x;
      } else {
        v[i] = tile[32 * piece + i][Tile::place(col, piece)];
      }
      if constexpr (FMT == NV_FP4) v[i] *= r;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      uint32_t amax;
      if constexpr (Tile::PAIRS) {
        amax = widen_bits<DT>(h ? two[b] >> 16 : two[b]);
        if constexpr (FMT == NV_FP4) amax = __float_as_uint(__uint_as_float(amax) * r);
      } else {
        amax = amax_bits<32 / NB>(v + b * (32 / NB));
      }
      if constexpr (FMT == NV_FP4) {
        byte[b] = nv_scale_byte(amax);
        const NvInverse inv(byte[b]);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[16 * b + i] = inv.quotient(v[16 * b + i]);
      } else {
        byte[b] = mx_scale_byte<FMT>(amax);
        const float m = mx_inverse_scale(byte[b]);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= m;
      }
    }
    const int64_t k = k0 + 32 * piece;
    if (row < p.rows && k < mx_padded_cols(p.cols)) {
      uint8_t* d = p.data + row * p.ld + k * MxFmt<FMT>::BITS / 8;
      if constexpr (FMT == MX_FP8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = cvt_e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        reinterpret_cast<uint4*>(d)[0] = make_uint4(q[0], q[1], q[2], q[3]);
        reinterpret_cast<uint4*>(d)[1] = make_uint4(q[4], q[5], q[6], q[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = cvt_e2m1x8(v + 8 * i);
        *reinterpret_cast<uint4*>(d) = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
    // scale words of the k range: one group of 128 (MX) or two of 64 (NV_FP4)
    if constexpr (FMT == NV_FP4) {
      uint32_t w = byte[0] | (byte[1] << 8);
      w |= __shfl_down_sync(0xffffffffu, w, 1) << 16;
      const int64_t g = k / 64;
      if ((piece & 1) == 0 && g < p.groups)
        *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, g, p.groups)) = w;
    } else {
      uint32_t w = byte[0] | (__shfl_down_sync(0xffffffffu, byte[0], 1) << 8);
      w |= __shfl_down_sync(0xffffffffu, w, 2) << 16;
      if (piece == 0) *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, k0 / 128, p.groups)) = w;
    }
  }
}

// ---------------------------------------------------------------------------------
// dequantise
// ---------------------------------------------------------------------------------
struct DequantParams {
  const uint8_t* data;
  const uint8_t* scales;
  const float* tensor_scale;
  void* y;
  int64_t rows, cols, ld, ldy, groups;
  int32_t wide;
};

template <int FMT>
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  if constexpr (FMT == NV_FP4) return e4m3_to_f32(byte);
  if (byte == 0xFFu) return __uint_as_float(0x7FC00000u);
  return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);  // 2^-127 is subnormal
}

template <int FMT, int DT, bool WIDE>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const DequantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  const uint32_t warps_per_row = uint32_t((p.cols + 511) / 512);
  const int64_t t = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t row = t >> 32 ? t / warps_per_row : uint32_t(t) / warps_per_row;
  if (row >= p.rows) return;  // whole warps
  const int64_t c0 = (t - row * warps_per_row) * 512;
  const bool mine = c0 + 16 * int64_t(lane_id()) < p.cols;
  const int64_t c = mine ? c0 + 16 * lane_id() : c0;  // lanes behind the row repeat its first chunk
  const uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
  const int64_t b = c / MxFmt<FMT>::BLOCK;
  float s = mx_scale_value<FMT>(p.scales[mx_scale_word(row, b / 4, p.groups) + (b & 3)]);
  const float ts = (FMT == NV_FP4 && p.tensor_scale) ? *p.tensor_scale : 1.0f;
  float v[16];
  if constexpr (FMT == MX_FP8) {
    const uint4 w = *reinterpret_cast<const uint4*>(d);
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t h;
      const uint16_t e = uint16_t(q[i / 2] >> (16 * (i & 1)));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(e));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(d);
    const uint32_t q[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t h;
      asm("{\n\t.reg .b8 b, x1, x2, x3;\n\t"
          "mov.b32 {b, x1, x2, x3}, %1;\n\t"
          "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
          : "=r"(h)
          : "r"(q[i / 4] >> (8 * (i & 3))));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      // element * block scale is exact (at most 6 significant bits)
      v[2 * i] = f.x * s * ts;
      v[2 * i + 1] = f.y * s * ts;
    }
  }
  if constexpr (WIDE) {
    const int64_t left = mine ? p.cols - c : 0;
    store16<DT>(static_cast<T*>(p.y) + row * p.ldy + c, left >= 16, left < 16 ? int(left) : 16, v);
  } else {
    __shared__ float stage[8][kStageFloats];
    warp_store16<DT>(static_cast<T*>(p.y) + row * p.ldy + c0, p.cols - c0, stage[warp_id()], v);
  }
}

// ---------------------------------------------------------------------------------
// RMS norm with the residual's addition
// ---------------------------------------------------------------------------------
struct NormParams {
  const void* x;
  const void* weight;
  const void* residual;  // may be null
  void* h;               // x + residual, rounded; null when there is no residual
  int64_t rows, cols, ldx, ldr, ldh;
  float eps, inv_cols;
  uint8_t* data;
  uint8_t* scales;
  const float* tensor_scale;
  int64_t ld, groups;
  int32_t wide, wide_weight, weight_f32, stream;
  uint32_t* status;
  uint64_t wait_ns;
  uint32_t fault_inject;  // test hook: 1 = no loads are issued, 2 = their readers give up
};

// x + residual is kept unrounded in fp32 for the norm; h is its one rounding. The whole row
// stays in registers between the sum of squares and the quantisation, so every tensor is
// read or written once.
//
// 16 consecutive elements of a row in shared memory (16-byte aligned), n of which exist; a
// row's length is a multiple of 16 bytes.
template <int DT>
__device__ __forceinline__ void norm_read16(const uint8_t* a, int n, float (&v)[16]) {
  using E = Elem<DT>;
  constexpr int PER = 16 / sizeof(typename E::T);
#pragma unroll
  for (int j = 0; j < 16 / PER; ++j) {
    const uint4 w = j * PER < n ? reinterpret_cast<const uint4*>(a)[j] : make_uint4(0, 0, 0, 0);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (PER == 8) {
        const float2 f = E::unpack(u[i]);
        v[8 * j + 2 * i] = f.x;
        v[8 * j + 2 * i + 1] = f.y;
      } else {
        v[4 * j + i] = __uint_as_float(u[i]);
      }
    }
  }
}

// 16 weights at column c, of which n exist, through L1 (every row reads them). ANY: rows at
// odd addresses, whose ends are ragged too.
template <int DT, bool ANY>
__device__ __forceinline__ void load_weight(const NormParams& p, int c, int n, float (&w)[16]) {
  const auto load = [&](auto dt, const auto* g) {
    constexpr int D = decltype(dt)::value;
    if constexpr (ANY) {
      if (!p.wide_weight || n < 16) return load16_any<D>(g, p.cols, c, w);
    }
    load16<D, true>(g + c, p.wide_weight && n == 16, n, w);
  };
  if (p.weight_f32) load(std::integral_constant<int, 3>{}, static_cast<const float*>(p.weight));
  else load(std::integral_constant<int, DT>{}, static_cast<const typename Elem<DT>::T*>(p.weight));
}

// Pairwise: an error of the row's sum moves every element of the row against its rounding
// borders, so the sum is worth a few more bits than one running total of 16 keeps.
__device__ __forceinline__ float sum_squares(const float (&v)[16]) {
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s[i] = v[i] * v[i];
#pragma unroll
    for (int j = 4; j < 16; j += 4) s[i] = fmaf(v[i + j], v[i + j], s[i]);
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// n values (a power of two) added pairwise.
template <int N>
__device__ __forceinline__ float sum_of(const float* v) {
  if constexpr (N == 1) return v[0];
  else return sum_of<N / 2>(v) + sum_of<N / 2>(v + N / 2);
}

// 1 / sqrt(m) by one Newton step from rsqrtf: every thread of a row computes it, so it has to
// be short (a correctly rounded division and root cost 10 % of an 8192-wide row). 0 and
// infinity keep their rsqrtf.
__device__ __forceinline__ float reciprocal_root(float m) {
  const float r = rsqrtf(m);
  const float e = fmaf(-(m * r), r, 1.0f);
  return e == e ? fmaf(0.5f * r, e, r) : r;
}

// A row whose factor is far from 1 (or NaN) takes a detour, so that what fp32 can hold at the
// ends does not limit what lies between:
//   * its squares may have left fp32: the sum overflowed, or it and eps are so small that
//     squares round away. h is then multiplied by a power of two (2^-80 brings the largest
//     fp32 to 2^48, 2^100 the smallest to 2^-49), summed again (`join` adds the warps' sums)
//     and normalised as that row with eps times its square, which is the same y;
//   * h * w below could leave fp32 though y does not (h = 2^60, w = 2^80): h is multiplied by
//     the factor first. Without this only |y| from 2^120 on overflows.
// NaN rows stay as they are, rows with an infinity come back with the same sum. Returns the
// row's factor, 1 where h was multiplied by it, then by `lift` too.
template <int CH, typename Join>
__device__ __forceinline__ float rescale_row(float (&v)[CH][16], float ss, float rstd, float inv_cols, float eps,
                                             float lift, Join&& join) {
  if (ss > 0x1p120f || (ss < 0x1p-90f && eps < 0x1p-90f)) {
    const float f = ss > 1.0f ? 0x1p-80f : 0x1p100f;
    ss = 0.0f;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[ch][i] *= f;
      ss += sum_squares(v[ch]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    rstd = reciprocal_root(fmaf(join(ss), inv_cols, eps * f * f));
  }
  if (!(rstd > 0.0f && rstd < __int_as_float(0x7F800000))) return rstd;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[ch][i] *= rstd * lift;
  return 1.0f;
}

// A row's factor from its sum of squares: 1 / rms and, for NV_FP4, the reciprocal tensor scale
// `pre`, which may be any number that fp32 holds. Their product has room on both sides (in
// norm_store it meets a block's reciprocal scale, 2^-9 to 2^9); where it has not, h is
// multiplied by the row's own part first and by 2^64 or 2^-64 of a far `pre`, so that h * w and
// what is left of `pre` are ordinary numbers wherever the quantised value is one. h * w that
// leaves fp32 by it leaves it behind `pre` too.
template <int FMT, int CH, typename Join>
__device__ __forceinline__ float row_factor(float (&v)[CH][16], float ss, float inv_cols, float eps, float pre,
                                            Join&& join) {
  const float rstd = reciprocal_root(fmaf(ss, inv_cols, eps));
  const float both = FMT == NV_FP4 ? rstd * pre : rstd;
  const bool near = rstd > 0x1p-8f && rstd < 0x1p10f && (FMT != NV_FP4 || (both > 0x1p-100f && both < 0x1p100f));
  if (near) return both;  // the same for all threads of the row
  if constexpr (FMT != NV_FP4) return rescale_row(v, ss, rstd, inv_cols, eps, 1.0f, join);
  const float lift = pre >= 0x1p64f ? 0x1p64f : pre <= 0x1p-64f ? 0x1p-64f : 1.0f;
  return rescale_row(v, ss, rstd, inv_cols, eps, lift, join) * (pre / lift);
}

// The last part of both kernels: one 16-element chunk at column c of row `row`, of which n
// elements exist, from h in fp32 to elements and scales. Elements behind the last column and
// rows behind the last are zero even where the row's norm is NaN. Whole warps, 512 columns.
//
// y = h * rstd * w is held in 32 bits as z = h * w and the row's factor: the block's largest
// |y| is rstd * max|z|, and the element is z times one factor, rstd over the block scale.
// That is two multiplications per element where y, its scaling and (NV_FP4) a correctly
// rounded quotient took up to seven; y is rounded arithmetic either way, so nothing hangs on
// a tie. `rstd` includes the reciprocal tensor scale.
template <int FMT>
__device__ __forceinline__ void norm_store(const NormParams& p, int64_t row, bool live, int c, int n, float rstd,
                                           const float (&w)[16], float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] *= w[i];
  if (n < 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i >= n) v[i] = 0.0f;
  }
  uint32_t amax = amax_bits<16>(v);
  if constexpr (MxFmt<FMT>::BLOCK == 32) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  // an all-zero block stays zero whatever the factor is (rstd may be infinite or NaN only
  // where the row itself is not finite)
  const uint32_t ymax = amax ? __float_as_uint(__uint_as_float(amax) * rstd) & 0x7FFFFFFFu : 0u;
  uint32_t byte;
  float f;
  if constexpr (FMT == NV_FP4) {
    byte = nv_scale_byte(ymax);
    f = rstd * NvInverse(byte).r;
  } else {
    byte = mx_scale_byte<FMT>(ymax);
    f = rstd * mx_inverse_scale(byte);
    if (byte < 32) {  // |y| below 2^-90: the factor alone could overflow
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= rstd;
      f = mx_inverse_scale(byte);
    }
  }
  if (amax == 0) f = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] *= f;
  uint32_t q[4];
  mx_pack16<FMT>(v, q);
  const uint32_t word = mx_gather_scales<FMT>(byte);
  const int g = c / (4 * MxFmt<FMT>::BLOCK);
  if (lane_id() % kLanesPerGroup<FMT> == 0 && g < p.groups && row < (p.rows + 127) / 128 * 128)
    *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, g, p.groups)) = word;
  if (live && c < mx_padded_cols(p.cols)) {
    uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
    if constexpr (FMT == MX_FP8) *reinterpret_cast<uint4*>(d) = make_uint4(q[0], q[1], q[2], q[3]);
    else *reinterpret_cast<uint2*>(d) = make_uint2(q[0], q[1]);
  }
}

// mx_rms_norm_kernel: TR threads per row, CH chunks of 16 elements per thread. A thread has
// read its chunk of x and residual before it writes that chunk of h, and no other thread
// reads it (rows at odd addresses: the row is read before h is written), so h may be x or
// residual itself.
template <int FMT, int DT, int TR, int CH, bool WIDE>
__global__ void __launch_bounds__(TR < 256 ? 256 : TR) mx_rms_norm_kernel(const NormParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  constexpr int NT = TR < 256 ? 256 : TR;
  constexpr int ROWS = NT / TR;       // rows per CTA
  constexpr int WARPS = TR / 32;      // warps per row
  const int r_in = threadIdx.x / TR, t = threadIdx.x % TR;
  const uint32_t warp = warp_id(), lane = lane_id();
  const int64_t row = int64_t(blockIdx.x) * ROWS + r_in;
  const bool live = row < p.rows;     // rows behind the last only write zero scales
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const int64_t len = live ? p.cols : 0;
  float v[CH][16];
  float ss = 0.0f;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (ch * TR + t) * 16;
    const int n = min(16, max(0, live ? int(p.cols) - c : 0));
    if constexpr (WIDE) load16<DT>(x + c, n == 16, n, v[ch]);
    else load16_any<DT>(x, len, c, v[ch]);
    if (p.residual) {
      const T* res = static_cast<const T*>(p.residual) + row * p.ldr;
      float r[16];
      if constexpr (WIDE) load16<DT>(res + c, n == 16, n, r);
      else load16_any<DT>(res, len, c, r);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[ch][i] += r[i];
      if constexpr (WIDE) store16<DT>(static_cast<T*>(p.h) + row * p.ldh + c, n == 16, n, v[ch]);
    }
    ss += sum_squares(v[ch]);
  }
  if constexpr (!WIDE) {
    if (p.residual) {
      // a thread's whole chunks reach into its neighbours' elements: in place, h waits for them
      if (p.h == p.x || p.h == p.residual) __syncthreads();
      T* h = static_cast<T*>(p.h) + row * p.ldh;
      __shared__ float stage[NT / 32][kStageFloats];
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const int wc = (ch * TR + t) * 16 - 16 * int(lane);  // the warp's first column
        warp_store16<DT>(h + wc, live ? int(p.cols) - wc : 0, stage[warp], v[ch]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  __shared__ float red[NT / 32];
  if constexpr (WARPS > 1) {
    if (lane == 0) red[warp] = ss;
    __syncthreads();
    ss = sum_of<WARPS>(red + r_in * WARPS);
  }
  float pre = 1.0f;
  if constexpr (FMT == NV_FP4)
    if (p.tensor_scale) pre = __frcp_rn(*p.tensor_scale);
  const float rstd = row_factor<FMT>(v, ss, p.inv_cols, p.eps, pre, [&](float sum) {
    if constexpr (WARPS > 1) {
      const auto row_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + r_in), "n"(TR) : "memory"); };
      row_sync();
      if (lane == 0) red[warp] = sum;
      row_sync();
      sum = sum_of<WARPS>(red + r_in * WARPS);
    }
    return sum;
  });
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int c = (ch * TR + t) * 16;
    if (c - 16 * int(lane) >= p.groups * (4 * MxFmt<FMT>::BLOCK)) continue;  // the whole warp is behind the row
    const int n = min(16, max(0, live ? int(p.cols) - c : 0));
    float w[16];
    load_weight<DT, !WIDE>(p, c, n, w);
    norm_store<FMT>(p, row, live, c, n, rstd, w, v[ch]);
  }
}

// mx_rms_norm_stream_kernel: many rows. The kernel above keeps as many bytes in flight as
// its threads hold in registers, 32 or 64 each, and stops loading while a row is reduced and
// stored (8192 x 8192 bf16 with a residual: 95 us, streamed 76; the bytes alone: 73).
// Here a CTA takes rows r, r + grid, ... and one thread copies whole rows of x and residual
// into a ring in shared memory with cp.async.bulk, kNormStages rows ahead, so the loads of
// the next rows run under everything else. NT threads, CH chunks each. Rows start on 16
// bytes and are a multiple of 16 bytes long. A row of h is written after its row of x and
// residual was read whole, so h may again be either of them.
constexpr int kNormStages = 3;

template <int FMT, int DT, int NT, int CH>
__global__ void __launch_bounds__(NT, CH == 1 ? 1024 / NT : 1) mx_rms_norm_stream_kernel(const NormParams p) {
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][NT / 32];
  __shared__ __align__(8) uint64_t full[kNormStages];
  const uint32_t warp = warp_id(), lane = lane_id();
  const uint32_t row_bytes = uint32_t(p.cols * sizeof(T));
  const uint32_t stage_bytes = row_bytes * (p.residual ? 2 : 1);
  if (threadIdx.x == 0) {
#pragma unroll
    for (int s = 0; s < kNormStages; ++s) mbar_init(smem_u32(full + s), 1);
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();
  const T* x = static_cast<const T*>(p.x);
  const T* res = static_cast<const T*>(p.residual);
  const auto load_row = [&](int64_t row, int s) {
    const uint32_t bar = smem_u32(full + s), dst = smem_u32(smem) + s * stage_bytes;
    mbar_arrive_expect_tx(bar, stage_bytes);
    bulk_load(dst, x + row * p.ldx, row_bytes, bar);
    if (res) bulk_load(dst + row_bytes, res + row * p.ldr, row_bytes, bar);
  };
  // behind the ring, only there when h is at an odd pitch
  float* stage = reinterpret_cast<float*>(smem + kNormStages * stage_bytes) + warp * kStageFloats;
  const int64_t first = blockIdx.x, step = gridDim.x;
  if (threadIdx.x == 0 && p.fault_inject != 1)
    for (int s = 0; s < kNormStages; ++s)
      if (first + s * step < p.rows) load_row(first + s * step, s);
  float pre = 1.0f;
  if constexpr (FMT == NV_FP4)
    if (p.tensor_scale) pre = __frcp_rn(*p.tensor_scale);

  int s = 0;
  uint32_t phase = 0, parity = 0;
  bool ok = p.fault_inject != 2;
  int64_t row = first;
  for (; row < p.rows && ok; row += step) {
    // all threads wait; a wait that runs out ends this CTA's work (status word)
    ok = mbar_wait_bounded(smem_u32(full + s), phase, p.wait_ns);
    const uint8_t* sx = smem + s * stage_bytes;
    float v[CH][16];
    float ss = 0.0f;
    T* h = static_cast<T*>(p.h) + row * p.ldh;
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + threadIdx.x) * 16;
      const int n = min(16, max(0, int(p.cols) - c));
      if (c - 16 * int(lane) >= int(p.cols)) {  // the whole warp is behind the row
#pragma unroll
        for (int i = 0; i < 16; ++i) v[ch][i] = 0.0f;
        continue;
      }
      norm_read16<DT>(sx + c * sizeof(T), n, v[ch]);
      if (res) {
        float r[16];
        norm_read16<DT>(sx + row_bytes + c * sizeof(T), n, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[ch][i] += r[i];
        if (p.wide) store16<DT>(h + c, n == 16, n, v[ch]);
        else warp_store16<DT>(h + c - 16 * int(lane), int(p.cols) - c + 16 * int(lane), stage, v[ch]);
      }
      ss += sum_squares(v[ch]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) red[parity][warp] = ss;
    ok = __syncthreads_and(ok);
    if (!ok) break;
    // every thread has read the stage: refill it
    if (threadIdx.x == 0 && row + kNormStages * step < p.rows) load_row(row + kNormStages * step, s);
    ss = sum_of<NT / 32>(red[parity]);
    const float rstd = row_factor<FMT>(v, ss, p.inv_cols, p.eps, pre, [&](float sum) {
      __syncthreads();
      if (lane == 0) red[parity][warp] = sum;
      __syncthreads();
      return sum_of<NT / 32>(red[parity]);
    });
    parity ^= 1u;  // the other buffer: a fast warp's next sum must not overtake a slow one's read
#pragma unroll
    for (int ch = 0; ch < CH; ++ch) {
      const int c = (ch * NT + threadIdx.x) * 16;
      const int n = min(16, max(0, int(p.cols) - c));
      if (c - 16 * int(lane) >= p.groups * (4 * MxFmt<FMT>::BLOCK)) continue;
      float w[16];
      load_weight<DT, false>(p, c, n, w);
      norm_store<FMT>(p, row, true, c, n, rstd, w, v[ch]);
    }
    if (++s == kNormStages) {
      s = 0;
      phase ^= 1u;
    }
  }
  if (!ok) {
    // a copy never landed: report it, and wait once more for those in flight (this row's and the
    // ones behind it) before the shared memory goes away
    if (threadIdx.x == 0) {
      uint32_t code = ST_PRODUCER_EMPTY | ST_ABORTED;
      for (int i = 0; i < kNormStages && row + i * step < p.rows; ++i) {
        const int at = s + i < kNormStages ? s + i : s + i - kNormStages;
        if (!mbar_wait_bounded(smem_u32(full + at), at < s ? phase ^ 1u : phase, p.wait_ns)) code |= ST_DRAIN;
      }
      if (p.status) atomicOr(p.status, code);
    }
    __syncthreads();
  }
  // zero scales of the rows behind the last one
  const int64_t end = (p.rows + 127) / 128 * 128;
  for (int64_t i = int64_t(blockIdx.x) * NT + threadIdx.x; i < (end - p.rows) * p.groups; i += step * NT)
    *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(p.rows + i / p.groups, i % p.groups, p.groups)) = 0u;
}

// ---------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------
// Programmatic dependent launch, as the GEMM's: every kernel here waits
// (griddepcontrol.wait) before its first global access.
template <typename P>
int launch(void (*kern)(P), dim3 grid, unsigned threads, unsigned cluster, const P& p, cudaStream_t stream,
           size_t smem = 0) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_ERR_LAUNCH;
  }
  return B200_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int elem_size(int dt) { return dt == B200_DT_F32 ? 4 : (dt == B200_DT_F16 || dt == B200_DT_BF16) ? 2 : 0; }

constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr int kNormSmem = 224 * 1024;  // most of a streaming CTA's shared memory

template <int FMT, int DT>
int quantize_t(const QuantParams& p, bool transpose, int sms, cudaStream_t s) {
  if (!transpose) {
    // Two segments per warp for 16-bit types, 64 bytes in flight per thread (8192 x 8192
    // bf16: MX_FP8 34.6 -> 33.2 us, NV_FP4 44.4 -> 38.4; fp32 has 64 with one), unless that
    // leaves SMs without their 64 warps.
    const int64_t rows = (p.rows + 127) / 128 * 128, segs = (p.groups * 4 * MxFmt<FMT>::BLOCK + 511) / 512;
    const bool two = DT != B200_DT_F32 && segs > 1 && rows * segs >= int64_t(sms) * 64;
    const int64_t grid = (rows * (two ? (segs + 1) / 2 : segs) + 7) / 8;
    if (grid > kMaxGrid) return B200_ERR_SHAPE;
    const dim3 g{unsigned(grid)};
    if constexpr (DT != B200_DT_F32)
      if (two)
        return launch(p.wide ? mx_quant_rows_kernel<FMT, DT, 2, true> : mx_quant_rows_kernel<FMT, DT, 2, false>, g, 256,
                      1, p, s);
    return launch(p.wide ? mx_quant_rows_kernel<FMT, DT, 1, true> : mx_quant_rows_kernel<FMT, DT, 1, false>, g, 256, 1,
                  p, s);
  }
  const int64_t grid = ((p.rows + 127) / 128 * 2) * ((p.cols + 127) / 128);
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  return launch(mx_quant_cols_kernel<FMT, DT>, dim3(unsigned(grid)), 128, 1, p, s);
}

template <int FMT>
int quantize_f(int dt, const QuantParams& p, bool transpose, int sms, cudaStream_t s) {
  switch (dt) {
    case B200_DT_F16: return quantize_t<FMT, 0>(p, transpose, sms, s);
    case B200_DT_BF16: return quantize_t<FMT, 1>(p, transpose, sms, s);
    default: return quantize_t<FMT, 3>(p, transpose, sms, s);
  }
}

template <int DT>
int amax_t(AmaxParams p, uint32_t* n_partials, cudaStream_t s) {
  if (p.ld == p.cols && p.rows < (int64_t(1) << 62) / p.cols) {
    p.cols *= p.rows;  // no gaps between the rows: one long row
    p.rows = 1;
    p.wide = aligned(p.x, 32);
  }
  p.segs = (p.cols + 511) / 512;
  // clusters of 8 CTAs, about two segments to a warp and at most kPartials clusters; a
  // matrix of one CTA's size stays with one
  const int64_t ctas = (p.rows * p.segs + 15) / 16;
  const unsigned cluster = ctas < kAmaxCluster ? 1 : kAmaxCluster;
  int64_t n = ctas < kAmaxCluster ? ctas : (ctas + kAmaxCluster - 1) / kAmaxCluster;
  if (n > kPartials) n = kPartials;
  *n_partials = uint32_t(n);
  return launch(p.wide ? mx_amax_kernel<DT, true> : mx_amax_kernel<DT, false>, dim3(unsigned(n) * cluster), 256,
                cluster, p, s);
}

template <int FMT>
int dequantize_f(int dt, const DequantParams& p, cudaStream_t s) {
  const int64_t grid = (p.rows * ((p.cols + 511) / 512) + 7) / 8;
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  const dim3 g{unsigned(grid)};
  const auto go = [&](auto wide, auto any) { return p.wide ? launch(wide, g, 256, 1, p, s) : launch(any, g, 256, 1, p, s); };
  switch (dt) {
    case B200_DT_F16: return go(mx_dequant_kernel<FMT, 0, true>, mx_dequant_kernel<FMT, 0, false>);
    case B200_DT_BF16: return go(mx_dequant_kernel<FMT, 1, true>, mx_dequant_kernel<FMT, 1, false>);
    default: return go(mx_dequant_kernel<FMT, 3, true>, mx_dequant_kernel<FMT, 3, false>);
  }
}

template <int FMT, int DT, int TR, int CH>
int norm_launch(const NormParams& p, cudaStream_t s) {
  constexpr int NT = TR < 256 ? 256 : TR;
  const int64_t rows = (p.rows + 127) / 128 * 128;
  const int64_t grid = rows / (NT / TR);
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  return launch(p.wide ? mx_rms_norm_kernel<FMT, DT, TR, CH, true> : mx_rms_norm_kernel<FMT, DT, TR, CH, false>,
                dim3(unsigned(grid)), NT, 1, p, s);
}

template <int FMT, int DT, int NT, int CH>
int norm_stream(const NormParams& p, int sms, int dev, cudaStream_t s) {
  auto kern = mx_rms_norm_stream_kernel<FMT, DT, NT, CH>;
  const size_t smem = size_t(kNormStages) * p.cols * 2 * (p.residual ? 2 : 1) +
                      (p.residual && !p.wide ? NT / 32 * kStageFloats * sizeof(float) : 0);
  static std::atomic<int> configured[64];
  if (!configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kNormSmem) != cudaSuccess) {
      (void)cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev].store(1, std::memory_order_release);
  }
  // as many CTAs as the device holds at once: one more would run its rows after the others
  static std::atomic<uint64_t> known[64];  // the last answer: shared memory and CTAs per SM
  uint64_t last = known[dev].load(std::memory_order_relaxed);
  if (last >> 8 != smem) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, NT, smem) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    last = uint64_t(smem) << 8 | uint64_t(n);
    known[dev].store(last, std::memory_order_relaxed);
  }
  const int per_sm = int(last & 0xFF);
  return launch(kern, dim3(unsigned(sms * per_sm)), NT, 1, p, s, smem);
}

// Many aligned rows of a 16-bit type stream through shared memory, otherwise a row gets as
// many threads as its 16-element chunks and scale groups. Streaming wins from 4096 columns
// on (8192 x 8192 with a residual, MX_FP8: 76 us against 95; 8192 x 12288: 138 against 187)
// and where a power of two of threads would leave many idle (8192 x 2560: 28.9 against 33);
// it loses at 2048 x 4096 (14.9 against 12.9). fp32 rows bring twice the bytes per thread
// and run at the copy rate as they are (8192 x 8192: 134 us, 164 streamed).
template <int FMT, int DT>
int norm_t(const NormParams& p, int sms, int dev, cudaStream_t s) {
  const int64_t chunks = p.groups * 4 * MxFmt<FMT>::BLOCK / 16;
  constexpr int es = DT == B200_DT_F32 ? 4 : 2;
  const int64_t row = p.cols * es * (p.residual ? 2 : 1);
  const bool idle = chunks > 128 && chunks <= 256 && chunks * 8 < 256 * 7;
  const bool stream = es == 2 && p.stream && p.rows >= 4 * int64_t(sms) && (idle || chunks > 256) && chunks <= 1024 &&
                      row * kNormStages <= kNormSmem - 18 * 1024;
  if constexpr (es == 2) {
    if (stream && chunks <= 256) return norm_stream<FMT, DT, 256, 1>(p, sms, dev, s);
    if (stream && chunks <= 512) return norm_stream<FMT, DT, 512, 1>(p, sms, dev, s);
    if (stream) return norm_stream<FMT, DT, 512, 2>(p, sms, dev, s);
  }
  if (chunks <= 32) return norm_launch<FMT, DT, 32, 1>(p, s);
  if (chunks <= 64) return norm_launch<FMT, DT, 64, 1>(p, s);
  if (chunks <= 128) return norm_launch<FMT, DT, 128, 1>(p, s);
  if (chunks <= 256) return norm_launch<FMT, DT, 256, 1>(p, s);
  if (chunks <= 512) return norm_launch<FMT, DT, 512, 1>(p, s);
  if (chunks <= 1024) return norm_launch<FMT, DT, 1024, 1>(p, s);
  return norm_launch<FMT, DT, 1024, 2>(p, s);
}

template <int FMT>
int norm_f(int dt, const NormParams& p, int sms, int dev, cudaStream_t s) {
  switch (dt) {
    case B200_DT_F16: return norm_t<FMT, 0>(p, sms, dev, s);
    case B200_DT_BF16: return norm_t<FMT, 1>(p, sms, dev, s);
    default: return norm_t<FMT, 3>(p, sms, dev, s);
  }
}

}  // namespace

namespace b200 {

constexpr uint64_t kDefaultWaitNs = 1000000000ull;  // 1 s per device wait
static thread_local MxWaits t_waits = {kDefaultWaitNs, 0};
const MxWaits& mx_waits() { return t_waits; }

// Checks of one microscaled operand that need no GPU.
int mx_validate(const B200MxTensor* t) {
  if (!t || t->format < B200_MX_FP8 || t->format > B200_NV_FP4 || t->reserved != 0) return B200_ERR_INVALID_ARG;
  if (t->rows < 0 || t->cols < 0) return B200_ERR_SHAPE;
  const int64_t lim = (int64_t(1) << 31) - 128;  // rows and padded columns stay int32
  if (t->rows > lim || t->cols > lim) return B200_ERR_SHAPE;
  if (t->format != B200_NV_FP4 && t->tensor_scale) return B200_ERR_INVALID_ARG;
  if (t->tensor_scale && !aligned(t->tensor_scale, 4)) return B200_ERR_ALIGN;
  if (t->rows == 0 || t->cols == 0) return B200_OK;
  if (!t->data || !t->scales) return B200_ERR_INVALID_ARG;
  if (t->ld < mx_row_bytes(t->format, t->cols) || t->ld >= (int64_t(1) << 40)) return B200_ERR_SHAPE;
  if (!aligned(t->data, 16) || !aligned(t->scales, 16) || t->ld % 16) return B200_ERR_ALIGN;
  return B200_OK;
}

}  // namespace b200

extern "C" {

int b200_mx_layout(int32_t format, int64_t rows, int64_t cols, int64_t* row_bytes, int64_t* scale_bytes) {
  if (format < B200_MX_FP8 || format > B200_NV_FP4) return B200_ERR_INVALID_ARG;
  const int64_t lim = (int64_t(1) << 31) - 128;
  if (rows < 0 || cols < 0 || rows > lim || cols > lim) return B200_ERR_SHAPE;
  if (row_bytes) *row_bytes = mx_row_bytes(format, cols);
  if (scale_bytes) *scale_bytes = mx_scale_bytes(format, rows, cols);
  return B200_OK;
}

int b200_mx_wait_limit(uint64_t wait_limit_ns, int32_t fault_inject) {
  if (fault_inject < 0 || fault_inject > 2) return B200_ERR_INVALID_ARG;
  b200::t_waits = {wait_limit_ns ? wait_limit_ns : b200::kDefaultWaitNs, uint32_t(fault_inject)};
  return B200_OK;
}

int b200_mx_quantize(const void* x, int32_t x_dtype, int64_t ldx, int32_t transpose, int32_t find_scale,
                     const B200MxTensor* q, void* stream_v) {
  int rc = b200::mx_validate(q);
  if (rc != B200_OK) return rc;
  const int es = elem_size(x_dtype);
  if (!es) return B200_ERR_INVALID_ARG;
  if (find_scale && (q->format != B200_NV_FP4 || !q->tensor_scale)) return B200_ERR_INVALID_ARG;
  if (find_scale && !aligned(q->tensor_scale, 16)) return B200_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream_v);
  if (q->rows > 0 && q->cols > 0) {
    if (!x) return B200_ERR_INVALID_ARG;
    if (ldx < (transpose ? q->rows : q->cols) || ldx >= (int64_t(1) << 40)) return B200_ERR_SHAPE;
    if (!aligned(x, es)) return B200_ERR_ALIGN;
  } else if (!find_scale) {
    return B200_OK;
  }
  int sms = 0;
  rc = b200::gemm_device(nullptr, &sms, nullptr);
  if (rc != B200_OK) return rc;
  const int64_t xrows = transpose ? q->cols : q->rows, xcols = transpose ? q->rows : q->cols;
  const bool wide32 = aligned(x, 32) && (ldx * es) % 32 == 0;
  const bool wide16 = aligned(x, 16) && (ldx * es) % 16 == 0;
  uint32_t n_partials = 0;
  if (find_scale) {
    if (q->rows == 0 || q->cols == 0) {  // nothing to look at: 1
      return launch(mx_unit_scale_kernel, dim3(1), 1, 1, q->tensor_scale, s);
    }
    const AmaxParams ap{x, xrows, xcols, ldx, 0, wide32, q->tensor_scale + 4};
    switch (x_dtype) {
      case B200_DT_F16: rc = amax_t<0>(ap, &n_partials, s); break;
      case B200_DT_BF16: rc = amax_t<1>(ap, &n_partials, s); break;
      default: rc = amax_t<3>(ap, &n_partials, s); break;
    }
    if (rc != B200_OK) return rc;
  }
  QuantParams p{x, q->rows, q->cols, ldx, static_cast<uint8_t*>(q->data), static_cast<uint8_t*>(q->scales),
                q->tensor_scale, find_scale ? q->tensor_scale + 4 : nullptr, n_partials, q->ld, mx_groups(q->format, q->cols),
                transpose ? wide16 : wide32};
  switch (q->format) {
    case B200_MX_FP8: return quantize_f<MX_FP8>(x_dtype, p, transpose != 0, sms, s);
    case B200_MX_FP4: return quantize_f<MX_FP4>(x_dtype, p, transpose != 0, sms, s);
    default: return quantize_f<NV_FP4>(x_dtype, p, transpose != 0, sms, s);
  }
}

int b200_mx_dequantize(const B200MxTensor* q, void* y, int32_t y_dtype, int64_t ldy, void* stream_v) {
  int rc = b200::mx_validate(q);
  if (rc != B200_OK) return rc;
  const int es = elem_size(y_dtype);
  if (!es) return B200_ERR_INVALID_ARG;
  if (q->rows == 0 || q->cols == 0) return B200_OK;
  if (!y) return B200_ERR_INVALID_ARG;
  if (ldy < q->cols || ldy >= (int64_t(1) << 40)) return B200_ERR_SHAPE;
  if (!aligned(y, es)) return B200_ERR_ALIGN;
  rc = b200::gemm_device(nullptr, nullptr, nullptr);
  if (rc != B200_OK) return rc;
  DequantParams p{static_cast<const uint8_t*>(q->data), static_cast<const uint8_t*>(q->scales), q->tensor_scale, y,
                  q->rows, q->cols, q->ld, ldy, mx_groups(q->format, q->cols),
                  aligned(y, 32) && (ldy * es) % 32 == 0};
  cudaStream_t s = static_cast<cudaStream_t>(stream_v);
  switch (q->format) {
    case B200_MX_FP8: return dequantize_f<MX_FP8>(y_dtype, p, s);
    case B200_MX_FP4: return dequantize_f<MX_FP4>(y_dtype, p, s);
    default: return dequantize_f<NV_FP4>(y_dtype, p, s);
  }
}

int b200_mx_rms_norm(const B200MxNormArgs* a, const B200MxTensor* q, void* stream_v) {
  int rc = b200::mx_validate(q);
  if (rc != B200_OK) return rc;
  if (!a || a->reserved != 0) return B200_ERR_INVALID_ARG;
  const int es = elem_size(a->dtype);
  if (!es || (a->weight_dtype != a->dtype && a->weight_dtype != B200_DT_F32)) return B200_ERR_INVALID_ARG;
  if (!(a->eps >= 0.0f) || !(a->eps <= 3.4e38f)) return B200_ERR_INVALID_ARG;
  if (q->cols > B200_MX_NORM_MAX_COLS) return B200_ERR_SHAPE;
  if (q->rows == 0 || q->cols == 0) return B200_OK;
  if (!a->x || !a->weight || (a->residual && !a->h)) return B200_ERR_INVALID_ARG;
  const int64_t lim = int64_t(1) << 40;
  if (a->ldx < q->cols || a->ldx >= lim) return B200_ERR_SHAPE;
  if (a->residual && (a->ldr < q->cols || a->ldh < q->cols || a->ldr >= lim || a->ldh >= lim)) return B200_ERR_SHAPE;
  const int ws = elem_size(a->weight_dtype);
  if (!aligned(a->x, es) || !aligned(a->weight, ws) || !aligned(a->residual, es) || !aligned(a->h, es))
    return B200_ERR_ALIGN;
  int dev = 0, sms = 0;
  NormParams p{};
  rc = b200::gemm_device(&dev, &sms, &p.status);
  if (rc != B200_OK) return rc;
  p.wait_ns = mx_waits().wait_ns;
  p.fault_inject = mx_waits().fault_inject;
  p.x = a->x;
  p.weight = a->weight;
  p.residual = a->residual;
  p.h = a->residual ? a->h : nullptr;
  p.rows = q->rows;
  p.cols = q->cols;
  p.ldx = a->ldx;
  p.ldr = a->ldr;
  p.ldh = a->ldh;
  p.eps = a->eps;
  p.inv_cols = 1.0f / float(q->cols);
  p.data = static_cast<uint8_t*>(q->data);
  p.scales = static_cast<uint8_t*>(q->scales);
  p.tensor_scale = q->tensor_scale;
  p.ld = q->ld;
  p.groups = mx_groups(q->format, q->cols);
  p.wide_weight = aligned(a->weight, 32);
  p.wide = aligned(a->x, 32) && (a->ldx * es) % 32 == 0 &&
           (!a->residual || (aligned(a->residual, 32) && aligned(a->h, 32) && (a->ldr * es) % 32 == 0 &&
                             (a->ldh * es) % 32 == 0));
  p.weight_f32 = a->weight_dtype == B200_DT_F32;
  p.stream = (q->cols * es) % 16 == 0 && aligned(a->x, 16) && (a->ldx * es) % 16 == 0 &&
             (!a->residual || (aligned(a->residual, 16) && (a->ldr * es) % 16 == 0));
  cudaStream_t s = static_cast<cudaStream_t>(stream_v);
  switch (q->format) {
    case B200_MX_FP8: return norm_f<MX_FP8>(a->dtype, p, sms, dev, s);
    case B200_MX_FP4: return norm_f<MX_FP4>(a->dtype, p, sms, dev, s);
    default: return norm_f<NV_FP4>(a->dtype, p, sms, dev, s);
  }
}

}  // extern "C"
