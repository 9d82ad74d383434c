// ppn_policy.h -- what the policy operators' translation units share: element types, errors, launch helpers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/ppn.h"

namespace ppn_policy {

// The text behind ppn_policy_error(): one per host thread, so that two threads' calls do not meet.
int fail(int code, const char* format, ...);
int launched(const char* what);

__device__ inline float to_float(float x) { return x; }
__device__ inline float to_float(__bf16 x) { return (float)x; }
__device__ inline float to_float(_Float16 x) { return (float)x; }

constexpr float LOG2E = 1.44269504088896340736f;

// exp through the hardware's base-2 exponential: one rounding of x * log2 e, so the relative error is |x| half steps plus the unit's own.
__device__ inline float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }
__device__ inline float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }

// log(1 + e^v).  For small e = e^v the sum 1 + e drops e's low digits, so log(u) is corrected by e / (u - 1) (the usual log1p of a rounded u);
// above 20 the result is v to 32 bits.
__device__ inline float softplus(float v) {
  float e = exp_fast(v);
  float u = 1.0f + e;
  float l = 0.693147180559945309f * __builtin_amdgcn_logf(u);
  float r = u == 1.0f ? e : l * (e * __builtin_amdgcn_rcpf(u - 1.0f));
  return v > 20.0f ? v : r;
}

// Which environment's state a row of a step call may touch: read by every workgroup of the row, so that all decide alike.  A row whose
// id an earlier row has (or that is out of range) must not move the state on a second time: it is refused with NaN.  The ids in front of
// the row are compared one a lane; at 4096 rows that is 8 KB a workgroup on average, out of the L2.
// A caller may read the state before it knows (row_env has checked the range); it may not write it.
// Every row is compared with all in front of it, so a call with ids has a most (a minute's work would be 2^24 rows).
constexpr int MOST_IDS = 1 << 18;
enum { ROW_LIVE = 0, ROW_PADDING = 1, ROW_REFUSED = 2 };
__device__ inline int64_t row_env(const int32_t* env_ids, int64_t row, int64_t environments) {      // an environment that exists, the row's if it is live
  const int64_t id = env_ids ? env_ids[row] : row;
  return id >= 0 && id < environments ? id : 0;
}
__device__ inline int row_state(const int32_t* env_ids, int64_t row, int64_t environments) {
  if (!env_ids) return ROW_LIVE;
  const int32_t id = env_ids[row];
  if (id < 0) return ROW_PADDING;
  if (id >= environments) return ROW_REFUSED;
  bool met = false;
  for (int64_t i = threadIdx.x; i < row; i += 4 * (int64_t)blockDim.x) {
    int32_t other[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = i + k * (int64_t)blockDim.x;
      other[k] = env_ids[at < row ? at : i];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) met |= other[k] == id;
  }
  return __syncthreads_or(met) ? ROW_REFUSED : ROW_LIVE;
}

template <typename F>
int by_type(int64_t type, F f) {
  switch (type) {
    case PPN_T_F32: return f((float*)0);
    case PPN_T_BF16: return f((__bf16*)0);
    case PPN_T_F16: return f((_Float16*)0);
  }
  return fail(PPN_E_INVALID, "element type %lld is none of PPN_T_F32, PPN_T_BF16, PPN_T_F16", (long long)type);
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// A launch counts its lanes along an axis in 32 bits.
inline bool too_many(int64_t workgroups, int64_t lanes) { return workgroups > 0xffffffffll / lanes; }
inline int64_t size_of(int64_t type) { return type == PPN_T_F32 ? 4 : 2; }
inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p) % (uint64_t)bytes == 0; }

}  // namespace ppn_policy
