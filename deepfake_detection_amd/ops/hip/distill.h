// Launchers of the top-logits and distillation kernels (distill.hip). Raw
// pointers only: shapes, types, devices and layouts are checked by the caller
// (small_batch.hip).
#pragma once

#include <hip/hip_runtime.h>

enum class LogitType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

constexpr int kMaxTopK = 256;
constexpr int kMaxDistillClasses = 1 << 18;  // one bit each in 32 KB of LDS
constexpr int kDistillStats = 8;             // floats kept a row for the backward pass

struct TopkArgs {
  const void* logits;  // [rows, classes], row_stride elements apart
  long long rows, row_stride;
  int classes, k;
  LogitType type;
  float temperature;
  void* values;        // [rows, k] of type
  long long* indices;  // [rows, k]
  float* rest;         // [rows]
};

struct DistillArgs {
  const void* logits;
  long long rows, row_stride;
  int classes, k;
  LogitType type, vtype;
  float temperature;
  const void* values;        // [rows, k] of vtype
  const long long* indices;  // [rows, k]
  const float* rest;         // [rows] or null
  float* loss;               // [rows]
  float* stats;              // [rows, kDistillStats]
  // backward
  const float* upstream;  // [rows], upstream_stride elements apart
  long long upstream_stride;
  void* grad;  // [rows, classes] of type, contiguous
};

hipError_t topk_logits_launch(const TopkArgs& a, hipStream_t stream);
hipError_t distill_fwd(const DistillArgs& a, hipStream_t stream);
hipError_t distill_bwd(const DistillArgs& a, hipStream_t stream);
