// gemm_internal.h — host-side helpers shared by the C-ABI translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "b200gemm.h"
#include "gemm_sm100.cuh"

namespace b200 {

// Argument checks that need no GPU (same codes as b200_gemm).
int gemm_validate(const B200GemmArgs* a);

// Resolve the driver's tensor-map encoder once per process (allocates nothing).
int gemm_resolve_driver();

// Launch body shared by the entry points: `a` is validated with M, N > 0; `sms`
// and `cc_major` describe the current device; `status` is the device word the
// kernel's bounded waits report into.
// `allow_workspace` = false keeps the launch away from every schedule that needs
// library-owned device memory (stream-K): AUTO never picks it, an explicit request
// returns B200_ERR_SCRATCH_LIMIT.
// Fused all-gather of C (b200_gemm_allgather); validated by the caller.
struct GatherSpec {
  const void* dst;
  uint32_t mode;   // B200_GATHER_MULTICAST or B200_GATHER_PEERS
  uint32_t peers;  // pointers in the array (GATHER_PEERS)
  uint64_t ld;     // row pitch of the gathered matrix, elements
  uint64_t col;    // this GPU's first column, elements
};

int gemm_launch_impl(const B200GemmArgs& a, cudaStream_t stream, int sms, int cc_major,
                     uint32_t* status, bool allow_workspace = true, const GatherSpec* gather = nullptr);

// A launch with everything resolved: variant, tensor maps, kernel parameters, grid.
struct Prepared {
  alignas(64) CUtensorMap tA;
  alignas(64) CUtensorMap tB;
  alignas(64) CUtensorMap tC;
  KParams kp;
  uint32_t grid, smem;
  int ab, cd, cg, sched, tn;
  int dev;
  bool streamk;      // takes a fresh workspace epoch per launch
  bool memset_only;  // K == 0: C = 0
  void* c;
  size_t c_pitch, c_width, c_height;
};

// Set up the current device once and report it: its index, SM count and status word
// (any may be null). B200_ERR_UNSUPPORTED when it is not sm_100.
int gemm_device(int* dev, int* sms, uint32_t** status);

// Tensor map of a row-major [rows x cols] matrix, box [box_rows x box_cols], 128-byte
// swizzle; gemm_device() must have succeeded.
int gemm_encode_2d(CUtensorMap* m, const void* ptr, int dt, uint64_t rows, uint64_t cols, uint64_t ld,
                   uint32_t box_rows, uint32_t box_cols);

// Tensor map of `bands` x `groups` contiguous 512-byte tiles, box bands_box x groups_box
// tiles, no swizzle.
int gemm_encode_tiles(CUtensorMap* m, const void* ptr, uint64_t groups, uint64_t bands, uint32_t groups_box,
                      uint32_t bands_box);

// Checks of one microscaled operand that need no GPU.
int mx_validate(const B200MxTensor* t);

// What b200_mx_wait_limit set for this host thread.
struct MxWaits {
  uint64_t wait_ns;
  uint32_t fault_inject;
};
const MxWaits& mx_waits();

int gemm_prepare(const B200GemmArgs& a, int sms, int cc_major, uint32_t* status, bool allow_workspace,
                 const GatherSpec* gather, Prepared* out);
int gemm_launch_prepared(Prepared& pr, cudaStream_t stream);

}  // namespace b200
