// mx_quant.cu — microscaled quantiser, dequantiser and RMS norm (formats: mx_common.cuh).
//
//   quantise     rows of x, or of x transposed, to elements + block scales
//   dequantise   element * block scale * tensor scale, rounded once to f16 / bf16 / f32
//   RMS norm     h = x + residual; y = h * rsqrt(mean(h^2) + eps) * weight; y quantised
//
// All are streaming passes bound by HBM: per element they read and write what the
// tensors hold once (bf16 to MX_FP8: 2 + 1.03 bytes). One thread owns 16 consecutive
// elements of a row: one 32-byte load for 16-bit types, one NV_FP4 block or half a block
// of 32 (a shuffle joins the halves), 16 or 8 bytes out.
#include <cuda_runtime.h>

#include <cstdint>

#include "b200gemm.h"
#include "gemm_internal.h"
#include "mx_common.cuh"

namespace {

using namespace b200;

// ---------------------------------------------------------------------------------
// per-tensor scale of NV_FP4: amax / (6 * 448)
// ---------------------------------------------------------------------------------
// ts[0] the scale, ts[1] the running maximum's bits, ts[2] the count of finished blocks;
// ts[1] and ts[2] start at zero. The maximum of the finite magnitudes does not depend on
// the order of the atomics; the last block turns it into the scale.
template <int DT>
__global__ void __launch_bounds__(256) mx_amax_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t rows,
                                                      int64_t cols, int64_t ld, int wide, uint32_t* ts) {
  griddep_wait();
  griddep_launch_dependents();
  const int64_t per_row = (cols + 15) / 16;
  const int64_t warps_per_row = (per_row + 31) / 32;
  const int64_t tasks = rows * warps_per_row;
  const uint32_t lane = lane_id();
  uint32_t m = 0;
  for (int64_t t = int64_t(blockIdx.x) * 8 + warp_id(); t < tasks; t += int64_t(gridDim.x) * 8) {
    const int64_t row = t / warps_per_row;
    const int64_t c = ((t - row * warps_per_row) * 32 + lane) * 16;
    float v[16];
    const int64_t left = cols - c;
    load16<DT>(x + row * ld + c, wide && left >= 16, left < 16 ? int(left) : 16, v);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t b = abs_bits(v[i]);
      m = max(m, b < 0x7F800000u ? b : 0u);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t red[8];
  if (lane == 0) red[warp_id()] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, red[i]);
    atomicMax(ts + 1, m);
    __threadfence();
    if (atomicAdd(ts + 2, 1u) == gridDim.x - 1) {
      __threadfence();
      const float amax = __uint_as_float(atomicMax(ts + 1, 0u));
      // kept normal so that its reciprocal is finite
      *reinterpret_cast<float*>(ts) = amax > 0.0f ? fmaxf(__fdiv_rn(amax, 2688.0f), 1.17549435e-38f) : 1.0f;
    }
  }
}

// ---------------------------------------------------------------------------------
// quantise along the rows
// ---------------------------------------------------------------------------------
struct QuantParams {
  const void* x;
  int64_t rows, cols, ldx;  // of the quantised matrix (after the transposition, if any)
  uint8_t* data;
  uint8_t* scales;
  const float* tensor_scale;  // may be null
  int64_t ld;                 // bytes
  int64_t groups;
  int32_t wide;
};

// One warp per 512 consecutive elements of a row; rows run on to a multiple of 128 so
// that the padding bytes of the last scale tiles are written (as zero).
template <int FMT, int DT>
__global__ void __launch_bounds__(256) mx_quant_rows_kernel(const QuantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  const int64_t warps_per_row = (p.groups * 4 * MxFmt<FMT>::BLOCK + 511) / 512;
  const int64_t t = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t row = t / warps_per_row;
  if (row >= (p.rows + 127) / 128 * 128) return;  // whole warps
  const uint32_t lane = lane_id();
  const int64_t c = ((t - row * warps_per_row) * 32 + lane) * 16;
  float v[16];
  const int64_t left = row < p.rows ? p.cols - c : 0;
  load16<DT>(static_cast<const T*>(p.x) + row * p.ldx + c, p.wide && left >= 16, left < 16 ? int(left) : 16, v);
  if constexpr (FMT == NV_FP4) {
    if (p.tensor_scale) {
      const float r = __frcp_rn(__ldg(p.tensor_scale));
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= r;
    }
  }
  uint32_t q[4];
  const uint32_t word = mx_gather_scales<FMT>(mx_quantize16<FMT>(v, q));
  const int64_t g = c / (4 * MxFmt<FMT>::BLOCK);
  if (lane % kLanesPerGroup<FMT> == 0 && g < p.groups)
    *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, g, p.groups)) = word;
  if (row < p.rows && c < mx_padded_cols(p.cols)) {
    uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
    if constexpr (FMT == MX_FP8) *reinterpret_cast<uint4*>(d) = make_uint4(q[0], q[1], q[2], q[3]);
    else *reinterpret_cast<uint2*>(d) = make_uint2(q[0], q[1]);
  }
}

// ---------------------------------------------------------------------------------
// quantise along the columns of x: q = quantise(x^T)
// ---------------------------------------------------------------------------------
// A CTA takes 128 rows (k) x 64 columns of x through shared memory. Thread t then owns
// output rows (columns of x) 2p, 2p + 1 and a 32-long piece s of k: lane = 8 pairs x 4
// pieces, so four lanes write 128 (64) consecutive bytes of one output row. Column pairs
// are stored at p ^ (8 * piece), so the four pieces' reads of one step fall into
// different banks.
template <int FMT, int DT>
__global__ void __launch_bounds__(128) mx_quant_cols_kernel(const QuantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int kVec = 16 / sizeof(T);  // elements per 16-byte load
  __shared__ alignas(16) T tile[128][64];
  const uint32_t strips = uint32_t((p.rows + 127) / 128 * 2);
  const int64_t k0 = int64_t(blockIdx.x / strips) * 128;  // x row
  const int64_t c0 = int64_t(blockIdx.x % strips) * 64;   // x column = output row
  const T* x = static_cast<const T*>(p.x);
  const int64_t kleft = p.cols - k0, cleft = p.rows - c0;
  // element (k, c) sits at [k][((c / 2) ^ (8 * (k / 32))) * 2 + c % 2]
  if (p.wide) {
    constexpr int kPerRow = 64 / kVec;
#pragma unroll 4
    for (int i = threadIdx.x; i < 128 * kPerRow; i += 128) {
      const int k = i / kPerRow, c = i % kPerRow * kVec;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (k < kleft) {
        const T* src = x + (k0 + k) * p.ldx + c0 + c;
        if (c + kVec <= cleft) {
          w = *reinterpret_cast<const uint4*>(src);
        } else if (c < cleft) {
          alignas(16) T e[kVec];
#pragma unroll
          for (int j = 0; j < kVec; ++j) e[j] = c + j < cleft ? src[j] : E::store(0.0f);
          w = *reinterpret_cast<const uint4*>(e);
        }
      }
      // a 16-byte vector holds 4 or 2 pairs and the flip moves groups of 8 pairs
      *reinterpret_cast<uint4*>(&tile[k][((c / 2) ^ (8 * (k / 32))) * 2]) = w;
    }
  } else {
    for (int i = threadIdx.x; i < 128 * 64; i += 128) {
      const int k = i / 64, c = i % 64;
      tile[k][((c / 2) ^ (8 * (k / 32))) * 2 + c % 2] =
          k < kleft && c < cleft ? x[(k0 + k) * p.ldx + c0 + c] : E::store(0.0f);
    }
  }
  __syncthreads();
  const uint32_t lane = lane_id();
  const int piece = lane & 3, pair = warp_id() * 8 + (lane >> 2);
  const int col = (pair ^ (8 * piece)) * 2;
  float r = 1.0f;
  if constexpr (FMT == NV_FP4)
    if (p.tensor_scale) r = __frcp_rn(__ldg(p.tensor_scale));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t row = c0 + 2 * pair + h;  // output row
    uint32_t amax = 0, byte[2];
    uint32_t q[8];
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = E::load(tile[32 * piece + i][col + h]) * r;
    constexpr int NB = 32 / MxFmt<FMT>::BLOCK;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      amax = 0;
#pragma unroll
      for (int i = 0; i < 32 / NB; ++i) amax = max(amax, abs_bits(v[b * (32 / NB) + i]));
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

template <int FMT, int DT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const DequantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  const int64_t warps_per_row = (p.cols + 511) / 512;
  const int64_t t = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t row = t / warps_per_row;
  if (row >= p.rows) return;
  const int64_t c = ((t - row * warps_per_row) * 32 + lane_id()) * 16;
  if (c >= p.cols) return;
  const uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
  const int64_t b = c / MxFmt<FMT>::BLOCK;
  float s = mx_scale_value<FMT>(__ldg(p.scales + mx_scale_word(row, b / 4, p.groups) + (b & 3)));
  const float ts = (FMT == NV_FP4 && p.tensor_scale) ? __ldg(p.tensor_scale) : 1.0f;
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
  const int64_t left = p.cols - c;
  store16<DT>(static_cast<T*>(p.y) + row * p.ldy + c, p.wide && left >= 16, left < 16 ? int(left) : 16, v);
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
  int32_t wide, weight_f32;
};

// TR threads per row, CH chunks of 16 elements per thread: the whole row stays in
// registers between the sum of squares and the quantisation, so every tensor is read or
// written once. x + residual is kept unrounded in fp32 for the norm; h is its one
// rounding. A row's h is written before its thread has anything to read again, so h may
// be x or residual itself.
template <int FMT, int DT, int TR, int CH>
__global__ void __launch_bounds__(TR < 256 ? 256 : TR) mx_rms_norm_kernel(const NormParams p) {
  griddep_wait();
  griddep_launch_dependents();
  using T = typename Elem<DT>::T;
  constexpr int NT = TR < 256 ? 256 : TR;
  constexpr int ROWS = NT / TR;       // rows per CTA
  constexpr int WARPS = TR / 32;      // warps per row
  const int r_in = threadIdx.x / TR, t = threadIdx.x % TR;
  const int64_t row = int64_t(blockIdx.x) * ROWS + r_in;
  const bool live = row < p.rows;     // rows behind the last only write zero scales
  float v[CH][16];
  float ss = 0.0f;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int64_t c = int64_t(ch * TR + t) * 16;
    const int64_t left = live ? p.cols - c : 0;
    const int n = left < 16 ? (left < 0 ? 0 : int(left)) : 16;
    const bool wide = p.wide && n == 16;
    load16<DT>(static_cast<const T*>(p.x) + row * p.ldx + c, wide, n, v[ch]);
    if (p.residual) {
      float r[16];
      load16<DT>(static_cast<const T*>(p.residual) + row * p.ldr + c, wide, n, r);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[ch][i] += r[i];
      store16<DT>(static_cast<T*>(p.h) + row * p.ldh + c, wide, n, v[ch]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(v[ch][i], v[ch][i], ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if constexpr (WARPS > 1) {
    __shared__ float red[NT / 32];
    if (lane_id() == 0) red[warp_id()] = ss;
    __syncthreads();
    const float* mine = red + r_in * WARPS;
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) ss += mine[i];
  }
  const float rstd = rsqrtf(fmaf(ss, p.inv_cols, p.eps));
  float pre = 1.0f;
  if constexpr (FMT == NV_FP4)
    if (p.tensor_scale) pre = __frcp_rn(__ldg(p.tensor_scale));
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    const int64_t c = int64_t(ch * TR + t) * 16;
    const int64_t left = live ? p.cols - c : 0;
    const int n = left < 16 ? (left < 0 ? 0 : int(left)) : 16;
    float w[16];
    if (p.weight_f32) load16<3>(static_cast<const float*>(p.weight) + c, p.wide && n == 16, n, w);
    else load16<DT>(static_cast<const T*>(p.weight) + c, p.wide && n == 16, n, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = v[ch][i] * rstd * w[i];
      if constexpr (FMT == NV_FP4) y *= pre;
      v[ch][i] = y;
    }
    if (live) {
      // elements behind the last column: zero even where the row's norm is NaN
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i >= n) v[ch][i] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[ch][i] = 0.0f;
    }
    uint32_t q[4];
    const uint32_t word = mx_gather_scales<FMT>(mx_quantize16<FMT>(v[ch], q));
    const int64_t g = c / (4 * MxFmt<FMT>::BLOCK);
    if (t % kLanesPerGroup<FMT> == 0 && g < p.groups && row < (p.rows + 127) / 128 * 128)
      *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, g, p.groups)) = word;
    if (live && c < mx_padded_cols(p.cols)) {
      uint8_t* d = p.data + row * p.ld + c * MxFmt<FMT>::BITS / 8;
      if constexpr (FMT == MX_FP8) *reinterpret_cast<uint4*>(d) = make_uint4(q[0], q[1], q[2], q[3]);
      else *reinterpret_cast<uint2*>(d) = make_uint2(q[0], q[1]);
    }
  }
}

// ---------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------
// Programmatic dependent launch, as the GEMM's: every kernel here waits
// (griddepcontrol.wait) before its first global access.
template <typename P>
int launch(void (*kern)(P), dim3 grid, unsigned threads, const P& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_ERR_LAUNCH;
  }
  return B200_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int elem_size(int dt) { return dt == B200_DT_F32 ? 4 : (dt == B200_DT_F16 || dt == B200_DT_BF16) ? 2 : 0; }

constexpr int64_t kMaxGrid = 0x7fffffff;

template <int FMT, int DT>
int quantize_t(QuantParams p, bool transpose, cudaStream_t s) {
  if (!transpose) {
    const int64_t warps = (p.rows + 127) / 128 * 128 * ((p.groups * 4 * MxFmt<FMT>::BLOCK + 511) / 512);
    const int64_t grid = (warps + 7) / 8;
    if (grid > kMaxGrid) return B200_ERR_SHAPE;
    return launch(mx_quant_rows_kernel<FMT, DT>, dim3(unsigned(grid)), 256, p, s);
  }
  const int64_t grid = ((p.rows + 127) / 128 * 2) * ((p.cols + 127) / 128);
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  return launch(mx_quant_cols_kernel<FMT, DT>, dim3(unsigned(grid)), 128, p, s);
}

template <int FMT>
int quantize_f(int dt, const QuantParams& p, bool transpose, cudaStream_t s) {
  switch (dt) {
    case B200_DT_F16: return quantize_t<FMT, 0>(p, transpose, s);
    case B200_DT_BF16: return quantize_t<FMT, 1>(p, transpose, s);
    default: return quantize_t<FMT, 3>(p, transpose, s);
  }
}

template <int DT>
int amax_t(const void* x, int64_t rows, int64_t cols, int64_t ld, int wide, float* ts, int sms, cudaStream_t s) {
  if (cudaMemsetAsync(ts, 0, 16, s) != cudaSuccess) return B200_ERR_CUDA;
  const int64_t warps = rows * (((cols + 15) / 16 + 31) / 32);
  int64_t grid = (warps + 7) / 8;
  if (grid > int64_t(sms) * 8) grid = int64_t(sms) * 8;
  if (grid < 1) grid = 1;
  // a memset precedes, so an ordinary launch
  mx_amax_kernel<DT><<<unsigned(grid), 256, 0, s>>>(static_cast<const typename Elem<DT>::T*>(x), rows, cols, ld, wide,
                                                    reinterpret_cast<uint32_t*>(ts));
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_LAUNCH;
}

template <int FMT>
int dequantize_f(int dt, const DequantParams& p, cudaStream_t s) {
  const int64_t grid = (p.rows * ((p.cols + 511) / 512) + 7) / 8;
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  const dim3 g{unsigned(grid)};
  switch (dt) {
    case B200_DT_F16: return launch(mx_dequant_kernel<FMT, 0>, g, 256, p, s);
    case B200_DT_BF16: return launch(mx_dequant_kernel<FMT, 1>, g, 256, p, s);
    default: return launch(mx_dequant_kernel<FMT, 3>, g, 256, p, s);
  }
}

template <int FMT, int DT, int TR, int CH>
int norm_launch(const NormParams& p, cudaStream_t s) {
  constexpr int NT = TR < 256 ? 256 : TR;
  const int64_t rows = (p.rows + 127) / 128 * 128;
  const int64_t grid = rows / (NT / TR);
  if (grid > kMaxGrid) return B200_ERR_SHAPE;
  return launch(mx_rms_norm_kernel<FMT, DT, TR, CH>, dim3(unsigned(grid)), NT, p, s);
}

// Threads per row: the fewest whose 16-element chunks cover the row and its scale groups.
template <int FMT, int DT>
int norm_t(const NormParams& p, cudaStream_t s) {
  const int64_t chunks = p.groups * 4 * MxFmt<FMT>::BLOCK / 16;
  if (chunks <= 32) return norm_launch<FMT, DT, 32, 1>(p, s);
  if (chunks <= 64) return norm_launch<FMT, DT, 64, 1>(p, s);
  if (chunks <= 128) return norm_launch<FMT, DT, 128, 1>(p, s);
  if (chunks <= 256) return norm_launch<FMT, DT, 256, 1>(p, s);
  if (chunks <= 512) return norm_launch<FMT, DT, 512, 1>(p, s);
  if (chunks <= 1024) return norm_launch<FMT, DT, 1024, 1>(p, s);
  return norm_launch<FMT, DT, 1024, 2>(p, s);
}

template <int FMT>
int norm_f(int dt, const NormParams& p, cudaStream_t s) {
  switch (dt) {
    case B200_DT_F16: return norm_t<FMT, 0>(p, s);
    case B200_DT_BF16: return norm_t<FMT, 1>(p, s);
    default: return norm_t<FMT, 3>(p, s);
  }
}

}  // namespace

namespace b200 {

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
  int dev = 0, sms = 0;
  rc = b200::gemm_device(&dev, &sms, nullptr);
  if (rc != B200_OK) return rc;
  const int64_t xrows = transpose ? q->cols : q->rows, xcols = transpose ? q->rows : q->cols;
  const bool wide32 = aligned(x, 32) && (ldx * es) % 32 == 0;
  const bool wide16 = aligned(x, 16) && (ldx * es) % 16 == 0;
  if (find_scale) {
    switch (x_dtype) {
      case B200_DT_F16: rc = amax_t<0>(x, xrows, xcols, ldx, wide32, q->tensor_scale, sms, s); break;
      case B200_DT_BF16: rc = amax_t<1>(x, xrows, xcols, ldx, wide32, q->tensor_scale, sms, s); break;
      default: rc = amax_t<3>(x, xrows, xcols, ldx, wide32, q->tensor_scale, sms, s); break;
    }
    if (rc != B200_OK) return rc;
    if (q->rows == 0 || q->cols == 0) return B200_OK;
  }
  QuantParams p{x, q->rows, q->cols, ldx, static_cast<uint8_t*>(q->data), static_cast<uint8_t*>(q->scales),
                q->tensor_scale, q->ld, mx_groups(q->format, q->cols), transpose ? wide16 : wide32};
  switch (q->format) {
    case B200_MX_FP8: return quantize_f<MX_FP8>(x_dtype, p, transpose != 0, s);
    case B200_MX_FP4: return quantize_f<MX_FP4>(x_dtype, p, transpose != 0, s);
    default: return quantize_f<NV_FP4>(x_dtype, p, transpose != 0, s);
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
  rc = b200::gemm_device(nullptr, nullptr, nullptr);
  if (rc != B200_OK) return rc;
  NormParams p{};
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
  p.wide = aligned(a->x, 32) && aligned(a->weight, 32) && (a->ldx * es) % 32 == 0 &&
           (!a->residual || (aligned(a->residual, 32) && aligned(a->h, 32) && (a->ldr * es) % 32 == 0 &&
                             (a->ldh * es) % 32 == 0));
  p.weight_f32 = a->weight_dtype == B200_DT_F32;
  cudaStream_t s = static_cast<cudaStream_t>(stream_v);
  switch (q->format) {
    case B200_MX_FP8: return norm_f<MX_FP8>(a->dtype, p, s);
    case B200_MX_FP4: return norm_f<MX_FP4>(a->dtype, p, s);
    default: return norm_f<NV_FP4>(a->dtype, p, s);
  }
}

}  // extern "C"
