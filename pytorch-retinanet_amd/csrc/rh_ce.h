// What the classifier loss's two ways of working share (gfx950).
#pragma once
#include "rh_gemm.h"

namespace rh {
namespace ce {

using namespace gemm;

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// exp of many logits: the hardware's exp2 of a rounded product, an error of |x| * 2^-24 relative (and of log2 e's own
// rounding, which float's takes back).  That is far below the 2^-9 that a 16-bit result is rounded by; for float it is
// what rounding z itself does to e^z where |x| is no larger than |z|, and e^x is small where it is.
template <typename T>
__device__ __forceinline__ float exp_for(const float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}
template <>
__device__ __forceinline__ float exp_for<float>(const float x) {
  constexpr float kRest = 1.925963033500853e-08f;      // log2 e - kLog2e
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kLog2e, x * kRest));
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

// The upstream gradient that a call's gradients are for: what the host was told, or a value on the device; one that
// is what the host was told already has its gradients.
struct Upstream {
  const float* at;
  float made;
  __device__ __forceinline__ float value() const { return at ? *at : made; }
  __device__ __forceinline__ bool there() const { return at && *at == made; }
};
constexpr int kThere = -1;      // rows counted, of a call whose gradients are there: no kernel has any

// P is the matrix units' operand and so is rounded to the inputs' type.  float16 has no room for
// small probabilities (2^-24 is its smallest value, one of 131 072 equal classes has 2^-17): there P
// is kept times 2^15, which |P| <= 1 allows, and the products' results are scaled back, both exact.
template <typename T>
struct PScale {
  static constexpr float up = 1.0f, down = 1.0f;
};
template <>
struct PScale<_Float16> {
  static constexpr float up = 32768.0f, down = 1.0f / 32768.0f;
};

// Where column `c` of row `r` lies in an array of panels of `rows` rows (in elements).
__device__ __forceinline__ long long in_panels(const int r, const int c, const long long rows) {
  return ((long long)(c / kStepK) * rows + r) * kStepK + c % kStepK;
}

// The rows of a call come in chunks: this chunk's are `first` on, at most `most` of them.
struct Chunk {
  int first, most;
  __device__ __forceinline__ int rows(const int* n_valid) const {
    return min(most, *n_valid - first);
  }
};

// Within each 16 lanes.
template <int kRotate>
__device__ __forceinline__ float rotated(const float x) {
  const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + kRotate, 0xf, 0xf, true);
  return __builtin_bit_cast(float, y);
}
// The sums of both lanes of a pair 32, or 16, lanes apart: of a in the pair's lower lane, of b in its upper one.
__device__ __forceinline__ float fold32(const float a, const float b) {
  const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
  const auto s = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  const unsigned s0 = s[0], s1 = s[1];
  return __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
}
__device__ __forceinline__ float fold16(const float a, const float b) {
  const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
  const auto s = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  const unsigned s0 = s[0], s1 = s[1];
  return __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
}
__device__ __forceinline__ float sum16(float x) {      // over the 16 lanes, in each of them
  x += rotated<8>(x);
  x += rotated<4>(x);
  x += rotated<2>(x);
  return x + rotated<1>(x);
}

// Label sets whose logits a workgroup holds whole (rh_ce_whole.hip): logits, loss, P, its column sums and dX of a
// chunk of placed rows in one launch.
template <typename T>
struct WholeArgs {
  const char* x;            // the chunk's placed rows, in panels of chunk_rows
  long long x_bytes;
  int chunk_rows;
  const char* w;            // rows ldw bytes apart
  long long ldw, w_bytes;
  int steps, w_limit;       // k steps; bytes of a row in the last
  const T* bias;
  int v, d;
  Chunk chunk;
  const int* n_valid;
  const int* label;         // of the chunk's places
  const int* map;
  const float* scale;
  char* p;                  // out: P in panels of chunk_rows, of ldp columns
  int ldp;
  float* column_sums;       // [workgroup][v] or NULL
  T* dx;                    // or NULL
  float* row_loss;
  double* loss;             // [workgroup]
};
constexpr int kWholeRows = 64;          // of a workgroup
// Every 64 rows take the weights through LDS anew, twice, which costs more the larger they are; what it saves is
// the logits' way to memory and back.  A whole call with its gradients, bfloat16, bias, this way / the general one, us:
// 49 104 x 256: 80 classes 61 / 87, 200 classes 65 / 116, 601 classes 125 / 155; 49 104 x 512, 300 classes 129 / 154;
// 196 416 x 256, 80 classes 162 / 238; 8192 x 2048, 80 classes 79 / 89.  Beyond: 8192 x 512, 601 classes 70 / 74,
// 8192 x 1024, 601 classes 100 / 91, 16 384 x 4096, 90 classes 270 / 219.
inline bool whole_pays(int d, int v) { return v <= 640 && (long long)ceil_div(v, 128) * d <= 2048; }
template <typename T>
int run_whole(const WholeArgs<T>& a, hipStream_t stream);

// Calls of few rows (rh_ce_few.hip): the weights' bytes are what counts there.
constexpr int kFewRows = 16;
size_t few_workspace_bytes(int n, int d, int v, int dtype, int flags);
int run_few(const rh_linear_ce_args& q, int flags, hipStream_t stream);

}  // namespace ce
}  // namespace rh
