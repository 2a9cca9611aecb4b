// Launchers of the group norm + activation kernels (group_norm.hip). Raw
// pointers only: shapes, types, devices and layouts are checked by the caller
// (small_batch.hip). A launch of 2^32 threads or more, which HIP does not take,
// is hipErrorInvalidConfiguration, before anything has run.
#pragma once

#include <hip/hip_runtime.h>

enum class GnType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

// x, y, residual, dy, dx: [n, hw, c] row-major (channels last), one type.
// weight, bias: [c] of type ptype, or null. mean, rstd: fp32 [n, groups].
// drop: fp32 [n] or null.
constexpr int kGnMaxGroupChannels = 1 << 14;  // their sums are joined in LDS

struct GnArgs {
  long long n, hw;
  int c, groups;
  GnType type;
  int act;  // the values of Act (common.h)
  float eps;
  const void* x;
  GnType ptype;
  const void* weight;
  const void* bias;
  const void* residual;
  const float* drop;
  void* y;
  float* mean;
  float* rstd;
  // backward
  const void* dy;
  void* dx;
  float* dweight;
  float* dbias;
  float* ws;  // gn_fwd_ws / gn_bwd_ws floats
};

long long gn_fwd_ws(const GnArgs& a);
long long gn_bwd_ws(const GnArgs& a);
// Launches the pass that suits the shape: see group_norm.hip.
hipError_t gn_fwd(const GnArgs& a, hipStream_t stream);
hipError_t gn_bwd(const GnArgs& a, hipStream_t stream);

// Slabs held in LDS (group_norm_slab.hip). sums: [n, 2, c] floats, the images'
// parts of dbias and dweight, or null.
bool gn_slab_fits(const GnArgs& a, bool backward);
hipError_t gn_slab_fwd(const GnArgs& a, hipStream_t stream);
hipError_t gn_slab_bwd(const GnArgs& a, float* sums, hipStream_t stream);
