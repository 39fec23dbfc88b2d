// mx_gemm.cu — b200_mx_gemm: checks, kernel choice and launch of the block-scaled
// products (mx_gemm.cuh).
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "b200gemm.h"
#include "gemm_internal.h"
#include "mx_gemm.cuh"

namespace {

using namespace b200;

// Block-rows of tiles per group of the pair kernel. Back to back, 8192^3 runs at the power
// limit, where what is read again from L2 and DRAM costs clock: NV_FP4 231 us with 16, 236
// with 8, 229 with 32, 250 with 4; MX_FP8 452, 457, 484 and 486.
constexpr uint32_t kGroupM = 16;

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
int configure(K kern, int dev, std::atomic<int>* configured, uint32_t smem) {
  if (!configured[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             int(smem)) != cudaSuccess) {
      (void)cudaGetLastError();
      return B200_ERR_LAUNCH;
    }
    configured[dev].store(1, std::memory_order_release);
  }
  return B200_OK;
}

template <int FMT, int CD, int NT>
int configure_rows(int dev) {
  static std::atomic<int> configured[64];
  return configure(mx_gemm_rows_kernel<FMT, CD, NT>, dev, configured, MxRowsCfg<FMT, NT>::MAX_SMEM);
}

// How many clusters of `size` CTAs of the rows kernel the device holds at once, with the
// ring at its full depth (one CTA per SM) or at half (two). Clusters do not cross GPCs, so
// this is less than SMs / size: 16 tiles in 8 splits each do not fit 148 SMs.
template <int FMT, int CD, int NT>
int clusters_fit(int dev, int size, bool half) {
  using Cfg = MxRowsCfg<FMT, NT>;
  static std::atomic<int> known[64][2][9];
  std::atomic<int>& k = known[dev][half][size];
  int n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(size), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = Cfg::smem_bytes(half ? Cfg::HALF_STAGES : Cfg::MAX_STAGES);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(size);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (configure_rows<FMT, CD, NT>(dev) != B200_OK) return 0;
    if (cudaOccupancyMaxActiveClusters(&n, mx_gemm_rows_kernel<FMT, CD, NT>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      return 0;
    }
    k.store(n < 1 ? -1 : n, std::memory_order_relaxed);
  }
  return n;
}

// K splits and ring depth of the rows kernel. One CTA per SM keeps the deepest ring; a
// second one per SM (half the shared memory each) evens out what whole tiles leave idle
// when few rows make every CTA a stream of weights. One token, NV_FP4, us: 8192 x 8192 (64
// tiles) 8.5 with 4 splits of 4 stages, 9.0 with 2 of 8, 14.3 with 4 of 8 (one per SM, two
// waves); 8 x 28672 x 4096 (224 tiles) 12.5 with 4 stages, 14.9 with 8. Wider tiles lose by
// it (64 x 8192 x 8192: 10.7 with 2 splits of 8 stages, 13.2 with 4 of 2), and shares under
// 5 atoms cost more in joining than they even out (1 x 4096 x 4096: 4.4 with 4 splits, 4.8
// with 8), except that with SMs idle two atoms each are still better (1 x 1024 x 4096: 3.8
// with 8 splits, 4.1 with 4).
struct RowsPlan {
  uint32_t splits, stages;
};
template <int FMT, int CD, int NT>
RowsPlan plan_rows(uint64_t tiles, uint32_t k_atoms, const Call& k) {
  using Cfg = MxRowsCfg<FMT, NT>;
  const auto fill = [&](bool half, uint32_t atoms) {
    uint32_t s = k_atoms / atoms < 8 ? k_atoms / atoms : 8;
    while (s > 1 && (tiles * s > uint64_t(k.sms) * (half ? 2 : 1) ||
                     int64_t(tiles) > clusters_fit<FMT, CD, NT>(k.dev, int(s), half)))
      --s;
    return s < 1 ? 1u : s;
  };
  RowsPlan plan;
  plan.splits = fill(false, 2);
  bool half = tiles * plan.splits > uint64_t(k.sms);
  if (NT <= 32) {
    const uint32_t two = fill(true, 5);
    if (two > plan.splits) {
      plan.splits = two;
      half = true;
    }
  }
  const uint32_t share = (k_atoms + plan.splits - 1) / plan.splits;
  const uint32_t cap = half ? Cfg::HALF_STAGES : Cfg::MAX_STAGES;
  plan.stages = share < cap ? share : cap;
  return plan;
}

template <int FMT, int CD, int NT>
int launch_rows(const Call& k) {
  using Cfg = MxRowsCfg<FMT, NT>;
  auto kern = mx_gemm_rows_kernel<FMT, CD, NT>;
  int rc = configure_rows<FMT, CD, NT>(k.dev);
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
  const RowsPlan plan = plan_rows<FMT, CD, NT>(tiles, p.k_atoms, k);
  p.splits = plan.splits;
  p.stages = plan.stages;
  p.sf_p = static_cast<const uint8_t*>(k.b->scales);
  p.sf_q = static_cast<const uint8_t*>(k.a->scales);
  p.ts_p = k.b->tensor_scale;
  p.ts_q = k.a->tensor_scale;
  p.c = static_cast<uint8_t*>(k.c);
  p.ldc = uint64_t(k.ldc);
  const uint32_t es = uint32_t(elem_size(k.cd));
  p.vec = (reinterpret_cast<uintptr_t>(k.c) % (4 * es)) == 0 && k.ldc % 4 == 0;
  p.status = k.status;
  p.wait_ns = mx_waits().wait_ns;
  p.fault_inject = mx_waits().fault_inject;

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

// Tiled map over the scale tiles of a matrix: 512 bytes x groups x bands, a box of
// `groups_box` x `bands_box` whole tiles; boxes past the end read as zero.
int encode_scales(CUtensorMap* m, const B200MxTensor* t, uint32_t groups_box, uint32_t bands_box) {
  return gemm_encode_tiles(m, t->scales, uint64_t(mx_groups(t->format, t->cols)), uint64_t((t->rows + 127) / 128),
                           groups_box, bands_box);
}

template <int FMT, int CD, int TN>
int launch_pair(const Call& k) {
  using Cfg = MxPairCfg<FMT, TN>;
  auto kern = mx_gemm_pair_kernel<FMT, CD, TN>;
  static std::atomic<int> configured[64];
  int rc = configure(kern, k.dev, configured, Cfg::MAX_SMEM);
  if (rc != B200_OK) return rc;

  MxPairParams p{};
  p.M = uint32_t(k.a->rows);
  p.N = uint32_t(k.b->rows);
  p.row_bytes = uint32_t(mx_row_bytes(FMT, k.a->cols));
  p.m_tiles = (p.M + 255) / 256;
  p.n_tiles = (p.N + TN - 1) / TN;
  const uint64_t tiles = uint64_t(p.m_tiles) * p.n_tiles;
  if (tiles > 0x1fffffffull) return B200_ERR_SHAPE;
  p.num_tiles = uint32_t(tiles);
  p.k_atoms = (p.row_bytes + 127) / 128;
  p.group_m = kGroupM;
  p.ts_a = k.a->tensor_scale;
  p.ts_b = k.b->tensor_scale;
  p.c = static_cast<uint8_t*>(k.c);
  p.ldc = uint64_t(k.ldc);
  const uint64_t bits = reinterpret_cast<uintptr_t>(k.c) | (uint64_t(k.ldc) * uint64_t(elem_size(k.cd)));
  p.align = 32;
  while (bits % p.align) p.align /= 2;
  p.status = k.status;
  p.wait_ns = mx_waits().wait_ns;
  p.fault_inject = mx_waits().fault_inject;

  CUtensorMap ta, tb, tsa, tsb;
  rc = gemm_encode_2d(&ta, k.a->data, B200_DT_E4M3, p.M, p.row_bytes, uint64_t(k.a->ld), 128, 128);
  if (rc != B200_OK) return rc;
  rc = gemm_encode_2d(&tb, k.b->data, B200_DT_E4M3, p.N, p.row_bytes, uint64_t(k.b->ld), Cfg::MMA_N / 2, 128);
  if (rc != B200_OK) return rc;
  rc = encode_scales(&tsa, k.a, Cfg::GROUPS, 1);
  if (rc != B200_OK) return rc;
  rc = encode_scales(&tsb, k.b, Cfg::GROUPS, Cfg::BANDS);
  if (rc != B200_OK) return rc;

  const uint32_t pairs = uint32_t(k.sms) / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (p.num_tiles < pairs ? p.num_tiles : pairs), 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = k.stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, ta, tb, tsa, tsb, p) != cudaSuccess) {
    (void)cudaGetLastError();
    return B200_ERR_LAUNCH;
  }
  return B200_OK;
}

// Up to 128 rows of A: the rows kernel, at the narrowest tile that holds them. Beyond, the
// pair kernel, at the tile width whose waves cost least: a wave of 128-, 192- or 384-wide
// tiles takes time in the ratio 20 : 26 : 47 (8192^3 in 28, 19 and 10 waves: NV_FP4 241,
// 220 and 197 us, MX_FP8 553, 416 and 403; 512 x 8192 x 8192 in 2, 2 and 1: 19.6, 25.3 and
// 22.6 us). That ratio is NV_FP4's and serves all formats: MX_FP8's own figures make 20 : 22 :
// 41, and neither K nor C's type or alignment enters, though an fp32 tile of 384 is drained in
// two parts and odd rows of C take longer. Where the pairs' tiles do not fill one wave and K is
// long, the rows kernel's K splits win: it then has `share` atoms of K per CTA and about 12
// atoms' time for joining, against all of K (256 x 2048 x 8192 NV_FP4: 8.3 us with 4 splits,
// 10.9 in pairs; 1024 x 1024 x 4096, 2 splits of 8 atoms: 8.8 against 7.1); 12 too is one
// number for three formats whose atoms differ in cost.
template <int FMT, int CD>
int run(const Call& k) {
  const int64_t m = k.a->rows, n = k.b->rows;
  if (m <= 16) return launch_rows<FMT, CD, 16>(k);
  if (m <= 32) return launch_rows<FMT, CD, 32>(k);
  if (m <= 64) return launch_rows<FMT, CD, 64>(k);
  if (m <= 128) return launch_rows<FMT, CD, 128>(k);
  const int64_t pairs = k.sms / 2, m_tiles = (m + 255) / 256;
  const auto waves = [&](int64_t tn) { return (m_tiles * ((n + tn - 1) / tn) + pairs - 1) / pairs; };
  if (waves(128) == 1) {
    const uint64_t tiles = uint64_t((n + 127) / 128) * uint64_t((m + 127) / 128);
    const uint32_t atoms = uint32_t((mx_row_bytes(FMT, k.a->cols) + 127) / 128);
    const uint32_t splits = plan_rows<FMT, CD, 128>(tiles, atoms, k).splits;
    if (splits > 1 && atoms / splits + 12 < atoms) return launch_rows<FMT, CD, 128>(k);
  }
  const int64_t c128 = 20 * waves(128), c192 = 26 * waves(192), c384 = 47 * waves(384);
  if (c384 < c192 && c384 < c128) return launch_pair<FMT, CD, 384>(k);
  return c192 < c128 ? launch_pair<FMT, CD, 192>(k) : launch_pair<FMT, CD, 128>(k);
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
