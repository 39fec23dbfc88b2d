// mx_gemm.cu — b200_mx_gemm: checks, kernel choice and launch of the block-scaled
// products (mx_gemm.cuh).
#include <cuda_runtime.h>

#include <cstdint>

#include "b200gemm.h"
#include "gemm_internal.h"
#include "mx_gemm.cuh"

namespace {

using namespace b200;

constexpr uint64_t kWaitNs = 1000000000ull;  // 1 s per device wait

int elem_size(int dt) { return dt == B200_DT_F32 ? 4 : (dt == B200_DT_F16 || dt == B200_DT_BF16) ? 2 : 0; }

struct Call {
  const B200MxTensor* a;
  const B200MxTensor* b;
  void* c;
  int cd;
  int64_t ldc;
  int dev, sms;
  uint32_t* status;
  cudaStream_t stream;
};

template <typename K>
int configure(K kern, int dev, int* configured, uint32_t smem) {
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(smem)) != cudaSuccess) {
      (void)cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev] = 1;
  }
  return B200_OK;
}

template <int FMT, int CD, int NT>
int launch_rows(const Call& k) {
  using Cfg = MxRowsCfg<FMT, NT>;
  auto kern = mx_gemm_rows_kernel<FMT, CD, NT>;
  static int configured[64] = {0};
  int rc = configure(kern, k.dev, configured, Cfg::MAX_SMEM);
  if (rc != B200_OK) return rc;

  MxParams p{};
  p.np = uint32_t(k.b->rows);
  p.nq = uint32_t(k.a->rows);
  p.row_bytes = uint32_t(mx_row_bytes(FMT, k.a->cols));
  p.k_atoms = (p.row_bytes + 127) / 128;
  p.groups = uint32_t(mx_groups(FMT, k.a->cols));
  p.p_tiles = (p.np + 127) / 128;
  p.q_tiles = (p.nq + NT - 1) / NT;
  const uint64_t tiles = uint64_t(p.p_tiles) * p.q_tiles;
  if (tiles > 0x0fffffffull) return B200_ERR_SHAPE;
  // Split K while the tiles leave at least half of the SMs idle, up to a cluster of 8 and
  // no finer than two atoms per CTA.
  p.splits = 1;
  while (p.splits < 8 && tiles * p.splits * 2 <= uint64_t(k.sms) && p.splits * 4 <= p.k_atoms) p.splits *= 2;
  const uint32_t per_cta = (p.k_atoms + p.splits - 1) / p.splits;
  p.stages = per_cta < Cfg::MAX_STAGES ? per_cta : Cfg::MAX_STAGES;
  p.sf_p = static_cast<const uint8_t*>(k.b->scales);
  p.sf_q = static_cast<const uint8_t*>(k.a->scales);
  p.ts_p = k.b->tensor_scale;
  p.ts_q = k.a->tensor_scale;
  p.c = static_cast<uint8_t*>(k.c);
  p.ldc = uint64_t(k.ldc);
  const uint32_t es = uint32_t(elem_size(k.cd));
  p.vec = (reinterpret_cast<uintptr_t>(k.c) % (4 * es)) == 0 && k.ldc % 4 == 0;
  p.status = k.status;
  p.wait_ns = kWaitNs;

  CUtensorMap tp, tq;
  rc = gemm_encode_2d(&tp, k.b->data, B200_DT_E4M3, p.np, p.row_bytes, uint64_t(k.b->ld), 128, 128);
  if (rc != B200_OK) return rc;
  rc = gemm_encode_2d(&tq, k.a->data, B200_DT_E4M3, p.nq, p.row_bytes, uint64_t(k.a->ld), NT, 128);
  if (rc != B200_OK) return rc;

  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(tiles * p.splits), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = Cfg::smem_bytes(p.stages);
  cfg.stream = k.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, tp, tq, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_ERR_LAUNCH;
  }
  return B200_OK;
}

// The narrowest tile that holds A's rows; 128 beyond that.
template <int FMT, int CD>
int run(const Call& k) {
  const int64_t m = k.a->rows;
  if (m <= 16) return launch_rows<FMT, CD, 16>(k);
  if (m <= 32) return launch_rows<FMT, CD, 32>(k);
  if (m <= 64) return launch_rows<FMT, CD, 64>(k);
  if (m <= 128) return launch_rows<FMT, CD, 128>(k);
  return launch_rows<FMT, CD, 256>(k);
}

template <int FMT>
int run_f(const Call& k) {
  switch (k.cd) {
    case B200_DT_F16: return run<FMT, DT_F16>(k);
    case B200_DT_BF16: return run<FMT, DT_BF16>(k);
    default: return run<FMT, DT_F32>(k);
  }
}

}  // namespace

extern "C" int b200_mx_gemm(const B200MxTensor* a, const B200MxTensor* b, void* c, int32_t c_dtype, int64_t ldc,
                            void* stream_v) {
  int rc = b200::mx_validate(a);
  if (rc != B200_OK) return rc;
  rc = b200::mx_validate(b);
  if (rc != B200_OK) return rc;
  const int es = elem_size(c_dtype);
  if (a->format != b->format || !es) return B200_ERR_INVALID_ARG;
  if (a->cols != b->cols) return B200_ERR_SHAPE;
  if (a->rows == 0 || b->rows == 0) return B200_OK;
  if (!c) return B200_ERR_INVALID_ARG;
  if (ldc < b->rows || ldc >= (int64_t(1) << 40)) return B200_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(c) % uintptr_t(es)) return B200_ERR_ALIGN;
  Call k{a, b, c, c_dtype, ldc, 0, 0, nullptr, static_cast<cudaStream_t>(stream_v)};
  rc = b200::gemm_device(&k.dev, &k.sms, &k.status);
  if (rc != B200_OK) return rc;
  if (a->cols == 0) {  // empty sum: C = 0
    return cudaMemset2DAsync(c, size_t(ldc) * es, 0, size_t(b->rows) * es, size_t(a->rows), k.stream) == cudaSuccess
               ? B200_OK
               : B200_ERR_CUDA;
  }
  switch (a->format) {
    case B200_MX_FP8: return run_f<MX_FP8>(k);
    case B200_MX_FP4: return run_f<MX_FP4>(k);
    default: return run_f<NV_FP4>(k);
  }
}
