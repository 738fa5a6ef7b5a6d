// What the classifier loss's two ways of working share (gfx950).
#pragma once
#include "rh_gemm.h"

namespace rh {
namespace ce {

using namespace gemm;

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// exp as the loss needs it: for float results the accurate one; for 16-bit ones the hardware exp2 of a
// rounded product (|x| * 6e-8 relative, far below the 2^-9 of the type the result is rounded to).
template <typename T>
__device__ __forceinline__ float exp_for(const float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}
template <>
__device__ __forceinline__ float exp_for<float>(const float x) {
  return expf(x);
}

struct Labels {
  const void* p;
  int wide;             // int64, else int32
  long long ignore;
  int v;
  __device__ __forceinline__ long long at(const long long i) const {
    return wide ? ((const long long*)p)[i] : (long long)((const int*)p)[i];
  }
  __device__ __forceinline__ bool counts(const long long y) const { return y != ignore && y >= 0 && y < v; }
};

// Calls of few rows (rh_ce_few.hip): the weights' bytes are what counts there.
constexpr int kFewRows = 16;
size_t few_workspace_bytes(int n, int d, int v, int dtype, int flags);
int run_few(const rh_linear_ce_args& q, int flags, hipStream_t stream);

}  // namespace ce
}  // namespace rh
