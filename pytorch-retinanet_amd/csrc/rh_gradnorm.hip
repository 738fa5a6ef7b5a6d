// Global norm of many gradients, and clipping by it, on gfx950.
//
//   total = (sum |g|^2)^(1/2),  sum |g|  or  max |g|   over every value of every tensor of a list
//   c = min(1, max_norm / (total + 1e-6)),   g *= c in place
//
// Both passes are bound by memory: the norm reads every value once, clipping reads and writes it.
// The list travels in the kernels' arguments (no copy to the device, so a call can be captured) and
// is cut into pieces of 32 KiB that a fixed number of workgroups take in runs, whatever the tensors'
// sizes; a piece starts at a 16-byte address, only a tensor's first and last 16 bytes are taken
// value by value.  Sums are float64: the square of any gradient is a normal number there.
// 195 tensors, 38 M float32 values (151 MB): norm 26 us (5.8 TB/s), scaling 49 (6.2 over both ways).  A call whose norm
// is below the bound writes nothing and takes 31 us instead of 76.
#include <algorithm>
#include <vector>
#include "rh_common.h"

namespace rh {
namespace norm {

constexpr int kThreads = 256;
constexpr int kPieceBytes = 32768;
constexpr int kMostTensors = 240;      // of one launch: its table takes 3.8 KiB of the 4 KiB of arguments
constexpr int kMostBlocks = 1024;      // of one launch
constexpr long long kMostValues = 1ll << 29;      // of an entry: a larger tensor takes several

struct Table {
  const char* p[kMostTensors];
  unsigned n[kMostTensors];            // values * 4 + element type
  int end[kMostTensors];               // pieces up to and with this entry
  int tensors;
  int pieces;
};

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
// The tensors' addresses come out of a table, so that they are global memory has to be said.
#define RH_GLOBAL __attribute__((address_space(1)))
typedef RH_GLOBAL char* Global;

template <int kType>
struct Values;
template <>
struct Values<RH_F32> {
  static constexpr int size = 4;
  static __device__ __forceinline__ float get(const u32x4 v, int i) {
    const unsigned w = v[i];      // a copy: the cast of a vector's element takes element 0
    return __builtin_bit_cast(float, w);
  }
  static __device__ __forceinline__ float one(const Global p) { return *(RH_GLOBAL float*)p; }
  static __device__ __forceinline__ void put(const Global p, float v) { *(RH_GLOBAL float*)p = v; }
  static __device__ __forceinline__ u32x4 scaled(u32x4 v, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(unsigned, get(v, i) * c);
    return v;
  }
};
template <>
struct Values<RH_BF16> {
  static constexpr int size = 2;
  static __device__ __forceinline__ float get(const u32x4 v, int i) {
    const unsigned w = v[i >> 1];
    return __builtin_bit_cast(float, i & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ float one(const Global p) { return (float)*(RH_GLOBAL __bf16*)p; }
  static __device__ __forceinline__ void put(const Global p, float v) { *(RH_GLOBAL __bf16*)p = (__bf16)v; }
  static __device__ __forceinline__ u32x4 scaled(u32x4 v, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = __builtin_bit_cast(unsigned short, (__bf16)(get(v, 2 * i) * c));
      const unsigned hi = __builtin_bit_cast(unsigned short, (__bf16)(get(v, 2 * i + 1) * c));
      v[i] = lo | hi << 16;
    }
    return v;
  }
};
template <>
struct Values<RH_F16> {
  static constexpr int size = 2;
  static __device__ __forceinline__ float get(const u32x4 v, int i) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i >> 1] >> (16 * (i & 1))));
  }
  static __device__ __forceinline__ float one(const Global p) { return (float)*(RH_GLOBAL _Float16*)p; }
  static __device__ __forceinline__ void put(const Global p, float v) { *(RH_GLOBAL _Float16*)p = (_Float16)v; }
  static __device__ __forceinline__ u32x4 scaled(u32x4 v, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = __builtin_bit_cast(unsigned short, (_Float16)(get(v, 2 * i) * c));
      const unsigned hi = __builtin_bit_cast(unsigned short, (_Float16)(get(v, 2 * i + 1) * c));
      v[i] = lo | hi << 16;
    }
    return v;
  }
};

// What a value adds to the norm: kSquares and kAbs sums, kMax the largest |g| by its bits (a NaN's are
// larger than infinity's, so a NaN comes through).
enum Kind { kSquares = 0, kAbs = 1, kMax = 2 };

template <int kKind>
struct Sum {
  double sum = 0.0;
  unsigned top = 0;
  __device__ __forceinline__ void add(const float v) {
    if (kKind == kSquares) {
      const double d = v;
      sum = __builtin_fma(d, d, sum);
    } else if (kKind == kAbs) {
      sum += (double)__builtin_fabsf(v);
    } else {
      top = max(top, __builtin_bit_cast(unsigned, v) & 0x7fffffffu);
    }
  }
  __device__ __forceinline__ void join(const double s) {
    if (kKind == kMax) {
      top = max(top, __builtin_bit_cast(unsigned, (float)s));
    } else {
      sum += s;
    }
  }
  __device__ __forceinline__ double value() const {
    return kKind == kMax ? (double)__builtin_bit_cast(float, top) : sum;
  }
  // over the workgroup; every thread gets it
  __device__ __forceinline__ void over_block() {
    __shared__ double s_sum[kThreads / 64];
    __shared__ unsigned s_top[kThreads / 64];
    if (kKind == kMax) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    } else {
      sum = wave_sum(sum);
    }
    if ((threadIdx.x & 63) == 0) {
      s_sum[threadIdx.x >> 6] = sum;
      s_top[threadIdx.x >> 6] = top;
    }
    __syncthreads();
    sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
  }
};

// One piece of a tensor.
struct Range {
  const char* begin;      // of the tensor
  const char* end;
  const char* from;       // of the piece: kPieceBytes from a 16-byte address on, the tensor's part of them
};

template <int kType, typename F, typename G>
__device__ __forceinline__ void walk(const Range r, const F whole, const G single) {
  const Global at = (Global)(r.from + threadIdx.x * 16);
  // eight loads in flight where the piece lies inside the tensor
  if (r.from >= r.begin && r.from + kPieceBytes <= r.end) {
    u32x4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *(RH_GLOBAL u32x4*)(at + i * kThreads * 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) whole(at + i * kThreads * 16, v[i]);
    return;
  }
  const Global begin = (Global)r.begin, end = (Global)r.end;
  const Global stop = r.from + kPieceBytes < r.end ? (Global)(r.from + kPieceBytes) : end;
  for (Global w = at; w < stop; w += kThreads * 16) {
    if (w >= begin && w + 16 <= end) {
      whole(w, *(RH_GLOBAL u32x4*)w);
    } else {
      for (int i = 0; i < 16; i += Values<kType>::size)
        if (w + i >= begin && w + i < end) single(w + i);
    }
  }
}

static_assert(kPieceBytes == 8 * kThreads * 16, "a piece is eight words a thread");

// Calls f(type, range) for every piece of this workgroup's run.  kBack: the runs from the list's end on.
template <bool kBack, typename F>
__device__ __forceinline__ void each_piece(const Table& t, const F f) {
  const int g = kBack ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x;
  const int lo = (int)((long long)t.pieces * g / gridDim.x), hi = (int)((long long)t.pieces * (g + 1) / gridDim.x);
  int a = 0, b = t.tensors - 1;
  while (a < b) {      // the first tensor that ends behind piece lo
    const int m = (a + b) >> 1;
    if (t.end[m] > lo) b = m; else a = m + 1;
  }
  for (int i = lo; i < hi; ++i) {
    while (t.end[a] <= i) ++a;
    const int first = i - (a ? t.end[a - 1] : 0);
    const int type = (int)(t.n[a] & 3u);
    Range r;
    r.begin = t.p[a];
    r.end = r.begin + (unsigned long long)(t.n[a] >> 2) * (type == RH_F32 ? 4 : 2);
    r.from = (const char*)((uintptr_t)r.begin & ~(uintptr_t)15) + (long long)first * kPieceBytes;
    f(type, r);
  }
}

template <int kKind>
__global__ __launch_bounds__(kThreads) void norm_kernel(const Table t, double* __restrict__ partial) {
  Sum<kKind> sum;
  each_piece<false>(t, [&](const int type, const Range& r) {
    if (type == RH_F32) {
      walk<RH_F32>(r, [&](Global, const u32x4 v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sum.add(Values<RH_F32>::get(v, i)); },
        [&](Global p) { sum.add(Values<RH_F32>::one(p)); });
    } else if (type == RH_BF16) {
      walk<RH_BF16>(r, [&](Global, const u32x4 v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum.add(Values<RH_BF16>::get(v, i)); },
        [&](Global p) { sum.add(Values<RH_BF16>::one(p)); });
    } else {
      walk<RH_F16>(r, [&](Global, const u32x4 v) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum.add(Values<RH_F16>::get(v, i)); },
        [&](Global p) { sum.add(Values<RH_F16>::one(p)); });
    }
  });
  sum.over_block();
  if (threadIdx.x == 0) partial[blockIdx.x] = sum.value();
}

// The workgroups' sums, in their order, to the list's.
template <int kKind>
__device__ __forceinline__ double total_of(const double* __restrict__ partial, const int n) {
  Sum<kKind> sum;
  for (int i = threadIdx.x; i < n; i += kThreads) sum.join(partial[i]);
  sum.over_block();
  return sum.value();
}

// partials < 0: the total is there, only the norm is made of it.
template <int kKind>
__global__ __launch_bounds__(kThreads) void total_kernel(const double* __restrict__ partial, const int partials,
                                                         double* __restrict__ total, float* __restrict__ norm) {
  const double s = partials < 0 ? *total : total_of<kKind>(partial, partials);
  if (threadIdx.x == 0) {
    if (partials >= 0) *total = s;
    *norm = (float)(kKind == kSquares ? __builtin_sqrt(s) : s);
  }
}

// partials: how many workgroups' sums `total` is still to be joined from (every workgroup does, in
// the same order: it costs less than a launch); 0: it is there.
template <int kKind>
__global__ __launch_bounds__(kThreads) void clip_kernel(const Table t, const double* __restrict__ partial,
                                                        const int partials, double* __restrict__ total,
                                                        const float max_norm, float* __restrict__ norm) {
  const double s = partials ? total_of<kKind>(partial, partials) : *total;
  const double length = kKind == kSquares ? __builtin_sqrt(s) : s;
  const float rounded = (float)length;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    if (partials) *total = s;
    *norm = rounded;
  }
  // of the unrounded length, unless what is returned is infinity: the factor is rounded once
  const float c = (float)((double)max_norm / ((rounded < __builtin_inff() ? length : (double)rounded) + 1e-6));
  if (c >= 1.0f) return;      // times one: nothing to write (a NaN goes on, and into every gradient)
  // from the list's end, which the norm's pass has read last and the caches still hold
  each_piece<true>(t, [&](const int type, const Range& r) {
    if (type == RH_F32) {
      walk<RH_F32>(r, [&](Global p, const u32x4 v) { *(RH_GLOBAL u32x4*)p = Values<RH_F32>::scaled(v, c); },
                   [&](Global p) { Values<RH_F32>::put(p, Values<RH_F32>::one(p) * c); });
    } else if (type == RH_BF16) {
      walk<RH_BF16>(r, [&](Global p, const u32x4 v) { *(RH_GLOBAL u32x4*)p = Values<RH_BF16>::scaled(v, c); },
                    [&](Global p) { Values<RH_BF16>::put(p, Values<RH_BF16>::one(p) * c); });
    } else {
      walk<RH_F16>(r, [&](Global p, const u32x4 v) { *(RH_GLOBAL u32x4*)p = Values<RH_F16>::scaled(v, c); },
                   [&](Global p) { Values<RH_F16>::put(p, Values<RH_F16>::one(p) * c); });
    }
  });
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
static long long pieces_of(const void* p, long long bytes) {
  return ((long long)((uintptr_t)p & 15) + bytes + kPieceBytes - 1) / kPieceBytes;
}

static int blocks_for(long long pieces) { return (int)(pieces < kMostBlocks ? pieces : kMostBlocks); }

// Cuts the list into launches; f(table, workgroups).
template <typename F>
static int each_table(const rh_tensor_ref* list, int count, const F f) {
  Table t;
  t.tensors = 0;
  long long pieces = 0;
  auto flush = [&]() -> int {
    if (!t.tensors) return RH_OK;
    t.pieces = (int)pieces;
    const int rc = f(t, blocks_for(pieces));
    t.tensors = 0;
    pieces = 0;
    return rc;
  };
  for (int i = 0; i < count; ++i) {
    const int size = list[i].dtype == RH_F32 ? 4 : 2;
    for (long long at = 0; at < list[i].count; at += kMostValues) {
      const long long n = list[i].count - at < kMostValues ? list[i].count - at : kMostValues;
      const char* p = (const char*)list[i].data + at * size;
      const long long more = pieces_of(p, n * size);
      if (t.tensors == kMostTensors || pieces + more > 0x7fffffffll)
        if (int rc = flush()) return rc;
      pieces += more;
      t.p[t.tensors] = p;
      t.n[t.tensors] = (unsigned)(n * 4 + list[i].dtype);
      t.end[t.tensors] = (int)pieces;
      ++t.tensors;
    }
  }
  return flush();
}

static int check_list(const rh_tensor_ref* list, int32_t count, bool written) {
  RH_REQUIRE(count >= 0 && count <= (1 << 24), RH_ESHAPE, "tensor count out of range");
  RH_REQUIRE(list || count == 0, RH_EINVAL, "null list");
  for (int i = 0; i < count; ++i) {
    const rh_tensor_ref& r = list[i];
    RH_REQUIRE(r.dtype == RH_F32 || r.dtype == RH_BF16 || r.dtype == RH_F16, RH_EINVAL,
               "tensor %d: unknown element type %d", i, r.dtype);
    RH_REQUIRE(r.count >= 0 && r.count <= (1ll << 40), RH_ESHAPE, "tensor %d: element count out of range", i);
    RH_REQUIRE(r.data || r.count == 0, RH_EINVAL, "tensor %d: null pointer", i);
    RH_REQUIRE((uintptr_t)r.data % (r.dtype == RH_F32 ? 4 : 2) == 0, RH_EALIGN,
               "tensor %d: not aligned to its elements", i);
  }
  if (written) {      // two workgroups must not scale the same value
    try {
      std::vector<std::pair<uintptr_t, uintptr_t>> spans;
      spans.reserve(count);
      bool sorted = true;
      for (int i = 0; i < count; ++i) {
        if (list[i].count == 0) continue;
        const uintptr_t a = (uintptr_t)list[i].data;
        sorted = sorted && (spans.empty() || spans.back().first <= a);
        spans.emplace_back(a, a + list[i].count * (list[i].dtype == RH_F32 ? 4 : 2));
      }
      if (!sorted) std::sort(spans.begin(), spans.end());
      for (size_t i = 1; i < spans.size(); ++i)
        RH_REQUIRE(spans[i].first >= spans[i - 1].second, RH_EINVAL, "two tensors of the list share memory");
    } catch (...) {
      RH_FAIL(RH_EWORKSPACE, "out of host memory for a list of %d tensors", count);
    }
  }
  return RH_OK;
}

template <int kKind>
static int run(const rh_grad_clip_args& q, hipStream_t stream) {
  double* partial = (double*)q.workspace;
  int blocks = 0;
  if (q.stages & RH_CLIP_NORM) {
    int rc = each_table(q.tensors, q.count, [&](const Table& t, int b) -> int {
      hipLaunchKernelGGL(norm_kernel<kKind>, dim3(b), dim3(kThreads), 0, stream, t, partial + blocks);
      RH_CHECK_LAUNCH("norm_kernel");
      blocks += b;
      return RH_OK;
    });
    if (rc) return rc;
  }
  bool written = false;      // a list without values launches none of these
  if (q.stages & RH_CLIP_SCALE) {
    int rc = each_table(q.tensors, q.count, [&](const Table& t, int b) -> int {
      hipLaunchKernelGGL(clip_kernel<kKind>, dim3(b), dim3(kThreads), 0, stream, t, partial, blocks, q.total, q.max_norm,
                         q.norm);
      RH_CHECK_LAUNCH("clip_kernel");
      written = true;
      return RH_OK;
    });
    if (rc) return rc;
  }
  if (!written) {
    hipLaunchKernelGGL(total_kernel<kKind>, dim3(1), dim3(kThreads), 0, stream, partial,
                       q.stages & RH_CLIP_NORM ? blocks : -1, q.total, q.norm);
    RH_CHECK_LAUNCH("total_kernel");
  }
  return RH_OK;
}

}  // namespace norm
}  // namespace rh

extern "C" {

size_t rh_grad_clip_workspace_bytes(const rh_tensor_ref* tensors, int32_t count) {
  if (rh::norm::check_list(tensors, count, false) != RH_OK) return 0;
  size_t blocks = 0;
  rh::norm::each_table(tensors, count, [&](const rh::norm::Table&, int b) -> int {
    blocks += b;
    return RH_OK;
  });
  return rh::round_up((blocks + 1) * sizeof(double), 256);
}

int rh_grad_clip(const rh_grad_clip_args* args, rh_stream_t stream) {
  RH_REQUIRE(args, RH_EINVAL, "null arguments");
  const rh_grad_clip_args& q = *args;
  RH_REQUIRE(q.stages > 0 && q.stages <= RH_CLIP_ALL, RH_EINVAL, "unknown stages %d", q.stages);
  RH_REQUIRE(q.norm_type >= RH_NORM_2 && q.norm_type <= RH_NORM_INF, RH_EINVAL, "unknown norm %d", q.norm_type);
  RH_REQUIRE(q.total && q.norm, RH_EINVAL, "null pointer");
  if (int rc = rh::norm::check_list(q.tensors, q.count, q.stages & RH_CLIP_SCALE)) return rc;
  if (q.stages & RH_CLIP_NORM) {
    const size_t need = rh_grad_clip_workspace_bytes(q.tensors, q.count);
    RH_REQUIRE(q.workspace && q.workspace_bytes >= need, RH_EWORKSPACE, "workspace of %zu bytes, %zu needed",
               q.workspace_bytes, need);
    RH_REQUIRE((uintptr_t)q.workspace % 256 == 0, RH_EALIGN, "workspace must be 256-byte aligned");
  }
  if (q.norm_type == RH_NORM_2) return rh::norm::run<rh::norm::kSquares>(q, (hipStream_t)stream);
  if (q.norm_type == RH_NORM_1) return rh::norm::run<rh::norm::kAbs>(q, (hipStream_t)stream);
  return rh::norm::run<rh::norm::kMax>(q, (hipStream_t)stream);
}

}  // extern "C"
