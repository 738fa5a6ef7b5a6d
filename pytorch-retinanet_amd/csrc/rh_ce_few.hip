// The classifier loss for a few rows (gfx950).  With so few rows the weights' bytes are what counts.
// Four launches:
//
//   logits      z[row][class] in float32, 16 classes x 16 rows to a matrix instruction that takes the
//               weights straight from memory, and each workgroup's (max, sum of exp) of every row
//   rows        the rows' (max, sum), losses and the call's loss
//   products    one more pass over the weights: dW rows written, dX summed per workgroup; P stays float32
//   features    the workgroups' parts of dX joined
//
// Up to four rows whose sums fit a workgroup's registers read the weights once: see `online`.
#include "rh_ce.h"

namespace rh {
namespace ce {

typedef __attribute__((ext_vector_type(4))) double f64x4;

// A row's largest logit, rounded to float, and the sum of the exponentials of the others' distance to it.
struct TopSum {
  double sum;
  float top;
};

// Logits of so few rows are not averaged over many: float's are held and summed in 64 bits (Z), since rounding a
// logit of 10 to float alone changes its probability by 5e-7.
template <typename T>
struct Mma16;      // 16 classes x 16 rows, 16 bytes of k a lane: lane % 16 is the class / row, lane / 16 the piece
template <>
struct Mma16<float> {
  typedef double Z;
  typedef f64x4 Acc;      // of lane l: row 4 r + l / 16
  static __device__ __forceinline__ int row(const int piece, const int r) { return 4 * r + piece; }
  static __device__ __forceinline__ Acc run(const u32x4 a, const u32x4 b, Acc c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[i], (double)y[i], c, 0, 0, 0);
    return c;
  }
};
template <>
struct Mma16<__bf16> {
  typedef float Z;
  typedef f32x4 Acc;      // row 4 (l / 16) + r
  static __device__ __forceinline__ int row(const int piece, const int r) { return 4 * piece + r; }
  static __device__ __forceinline__ f32x4 run(const u32x4 a, const u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
  }
};
template <>
struct Mma16<_Float16> {
  typedef float Z;
  typedef f32x4 Acc;      // row 4 (l / 16) + r
  static __device__ __forceinline__ int row(const int piece, const int r) { return 4 * piece + r; }
  static __device__ __forceinline__ f32x4 run(const u32x4 a, const u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  }
};

// 16 bytes of values from p on, of which `have` exist (the others read as zero).
template <typename T, bool kWide>
__device__ __forceinline__ u32x4 load_values(const T* p, const int have) {
  constexpr int kV = 16 / (int)sizeof(T);
  if constexpr (kWide) {
    return have >= kV ? *(const u32x4*)p : u32x4{0, 0, 0, 0};      // rows are whole pieces: all or none
  } else {
    union {
      T v[kV];
      u32x4 u;
    } r;
    if (have >= kV) {
      __builtin_memcpy(&r, p, 16);      // aligned to its elements: the card's wide loads ask for no more
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i) r.v[i] = i < have ? p[i] : (T)0.0f;
    }
    return r.u;
  }
}

template <typename T>
__device__ __forceinline__ void to_floats(const u32x4 u, float (&f)[16 / sizeof(T)]) {
  union {
    u32x4 u;
    T v[16 / sizeof(T)];
  } r;
  r.u = u;
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) f[i] = TypeOf<T>::to_float(r.v[i]);
}

// dW is written past the caches where what is read next is not dW: beside the weights that the same kernel reads, if
// the caches cannot hold both, and else where dW alone is more than they hold.  Steps of loss, clipping and an update
// of the weights (each reads dW next), bfloat16, 2048 features, us, past them / into them:
//   16 rows (weights read beside)   160 MiB of dW 305 / 315, 256 MiB 505 / 506, 384 MiB 744 / 778
//   1 row (read before)             160 MiB 236 / 225, 256 MiB 400 / 380, 320 MiB 510 / 499, 384 MiB 618 / 627
//   4 rows, frozen features (the same)   256 MiB 402 / 396, 320 MiB 519 / 514, 384 MiB 620 / 646
// A loss called again and again, its weights still in the caches, gains more and earlier (1 row, 256 MiB: 109 / 141), but
// that is no step.  (In the products of many rows it costs: dW of 32 768 x 2048 578 us instead of 535.)
constexpr long long kPastBeside = 128ll << 20, kPastAlone = 352ll << 20;
template <bool kPast>
__device__ __forceinline__ void store16(void* to, const u32x4 v) {
  if constexpr (kPast) __builtin_nontemporal_store(v, (u32x4*)to);
  else *(u32x4*)to = v;
}

struct FewSpace {
  void* z;             // [n][ldz]  float's are double
  TopSum* part;        // [kFewRows][blocks]
  TopSum* row;         // [kFewRows]  (max, sum), of a row that counts
  float* of_label;     // [kFewRows]  the label's p - 1
  float* scale;        // [1]
  float* dx_part;      // [parts][n][ldpart]
  float* share;        // [n][parts]: what a row's part counts (online)
  size_t bytes;
};

struct FewPlan {
  int groups, waves, blocks;        // logits: groups of 16 classes
  int ldz, z_size;
  // products: 16-lane columns of four waves; weights: threads a row; rows side by side, slices of columns
  int tpr, subsets, slices;
  int grad_blocks, per;             // classes a workgroup takes
  int parts, ldpart;
  bool wide_w, past;                // how the weights are read; dW is written past the caches
  int rows, chunks;                 // online: rows (a power of two) and 16-byte pieces of columns a thread; else 0
};

// Online: dX = sum of p W over the other classes, without P's normalisation, which is not known before the last
// class.  A workgroup takes whole rows of weights, so what a thread read for the logits is still in its registers
// when their exponentials are known: dX's sum is kept relative to the running maximum and joined like a softmax's.
// The weights are read once; dW is written by a pass that reads none.
// 1 x 2048 rows, 65 536 classes, bfloat16 (268 MB of weights, as much of dW): 208 us with two readings, 145 with
// one.  Loads for the next classes issued ahead, more workgroups or contiguous runs of classes for each: no faster.
static void plan_online(FewPlan& p, int n, int d, int v, int vals) {
  p.rows = n <= 1 ? 1 : n <= 2 ? 2 : 4;
  p.chunks = ceil_div(d, kThreads * vals);
  if (p.chunks == 3) p.chunks = 4;
  // 128 registers of rows and their sums at most; or half of the threads idle
  if (n > 4 || p.chunks > 4 || p.rows * p.chunks * vals > 64 || 2 * d < kThreads * vals) {
    p.rows = p.chunks = 0;
    return;
  }
  const int at_once = 16 / (p.rows > p.chunks ? p.rows : p.chunks);
  p.blocks = ceil_div(v, 2 * at_once);
  if (p.blocks > 512) p.blocks = 512;
  p.parts = p.blocks;
  p.ldpart = p.chunks * kThreads * vals;
}

static FewPlan few_plan(int n, int d, int v, int dtype, int flags) {
  FewPlan p = {};
  const int vals = dtype == RH_F32 ? 4 : 8;
  p.groups = ceil_div(v, 16);
  p.waves = p.groups < 2048 ? p.groups : 2048;
  p.blocks = ceil_div(p.waves, 4);
  p.ldz = ceil_div(v, 16) * 16;
  p.z_size = dtype == RH_F32 ? 8 : 4;
  p.wide_w = !(flags & RH_CE_COPY_WEIGHT);      // here that only says how the weights are read
  if (flags & RH_CE_GRAD_X) plan_online(p, n, d, v, vals);
  p.past = (long long)v * d * (16 / vals) >= ((flags & RH_CE_GRAD_X) && !p.rows ? kPastBeside : kPastAlone);
  const int whole = p.rows ? kThreads : 64;      // threads, or sixteen times the waves, of a row of weights
  p.tpr = 16;
  while (p.tpr < whole && p.tpr * vals < d) p.tpr *= 2;
  p.subsets = whole / p.tpr;
  p.slices = ceil_div(d, p.tpr * vals);
  int blocks = (p.rows ? 512 : 1024) / (p.slices < 512 ? p.slices : 512);
  const int step = p.rows ? p.subsets : 16 * p.subsets, most = ceil_div(v, 4 * p.subsets);
  if (blocks > most) blocks = most;
  if (blocks < 1) blocks = 1;
  p.per = ceil_div(ceil_div(v, blocks), step) * step;
  p.grad_blocks = ceil_div(v, p.per);
  if (!p.rows) {
    p.parts = p.grad_blocks * p.subsets;
    p.ldpart = p.slices * p.tpr * vals;
  }
  return p;
}

static FewSpace few_space(void* base, const FewPlan& p, int n, int flags) {
  Carver c(base);
  FewSpace s = {};
  s.z = c.take<char>((size_t)n * p.ldz * p.z_size);
  s.part = c.take<TopSum>((size_t)kFewRows * p.blocks);
  s.row = c.take<TopSum>(kFewRows);
  s.of_label = c.take<float>(kFewRows);
  s.scale = c.take<float>(1);
  if (flags & RH_CE_GRAD_X) s.dx_part = c.take<float>((size_t)p.parts * n * p.ldpart);
  if (p.rows) s.share = c.take<float>((size_t)n * p.parts);
  s.bytes = c.off;
  return s;
}

size_t few_workspace_bytes(int n, int d, int v, int dtype, int flags) {
  return few_space(nullptr, few_plan(n, d, v, dtype, flags), n, flags).bytes;
}

constexpr int kBatch = 8;                 // groups of classes a wave carries through the features
constexpr int kChunkBytes = 4096;         // of a row of features in LDS at a time
constexpr int kPitch = kChunkBytes + 16;  // rows a bank group apart
constexpr int kAhead = 8;                 // loads of weights in flight a lane

// A wave's lanes read 16 bytes of 16 rows of weights each, in the layout the instruction takes, so nothing
// passes through LDS but the features.  Bound by memory: 65 536 x 2048 bfloat16 (268 MB) 62 us, 4.3 TB/s.
template <typename T, bool kWide>
__global__ __launch_bounds__(kThreads) void few_logits_kernel(const T* __restrict__ x, const long long ldx, const int n,
                                                              const int d, const T* __restrict__ w, const long long ldw,
                                                              const int v, const T* __restrict__ bias,
                                                              const int groups, const int waves,
                                                              typename Mma16<T>::Z* __restrict__ z, const int ldz,
                                                              TopSum* __restrict__ part, const Upstream up) {
  if (up.there()) return;
  typedef typename Mma16<T>::Z Z;
  typedef typename Mma16<T>::Acc Acc;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ TopSum s_part[4][16];
  constexpr int kV = 16 / (int)sizeof(T), kStepK = 4 * kV, kChunk = kChunkBytes / (int)sizeof(T);
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, in = lane & 15, piece = lane >> 4;
  const int me = blockIdx.x * 4 + wave;
  float top = -__builtin_inff();      // of row `in`, over this lane's classes
  double sum = 0.0;
  for (int g0 = 0; g0 * waves < groups; g0 += kBatch) {
    Acc acc[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) acc[i] = Acc{0, 0, 0, 0};
    const int mine = me < waves ? min(kBatch, (groups - me + waves - 1) / waves - g0) : 0;
    for (int k0 = 0; k0 < d; k0 += kChunk) {
      const int len = min(kChunk, d - k0);
      __syncthreads();
      for (int i = t; i < 16 * (kChunkBytes / 16); i += kThreads) {
        const int r = i / (kChunkBytes / 16), c = i % (kChunkBytes / 16) * kV;
        if (c < (len + kAhead * kStepK - 1) / (kAhead * kStepK) * (kAhead * kStepK))      // zeros behind the row
          *(u32x4*)(smem + r * kPitch + c * (int)sizeof(T)) =
              r < n ? load_values<T, false>(x + r * ldx + k0 + c, len - c) : u32x4{0, 0, 0, 0};
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (i < mine) {
          const int c = (me + (g0 + i) * waves) * 16 + in;
          const T* row = w + (long long)min(c, v - 1) * ldw + k0 + piece * kV;
          const char* xs = smem + in * kPitch + piece * 16;
          constexpr int kSums = sizeof(Z) == 4 ? kAhead : 1;      // short ones: one over all features rounds more
          Acc sum_of[kSums];
#pragma unroll
          for (int u = 0; u < kSums; ++u) sum_of[u] = Acc{0, 0, 0, 0};
#pragma unroll 1
          for (int k = 0; k < len; k += kAhead * kStepK) {
            u32x4 a[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
              a[u] = load_values<T, kWide>(row + k + u * kStepK, len - k - u * kStepK - piece * kV);
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
              sum_of[u % kSums] =
                  Mma16<T>::run(a[u], *(const u32x4*)(xs + (k + u * kStepK) * (int)sizeof(T)), sum_of[u % kSums]);
          }
#pragma unroll
          for (int half = kSums / 2; half > 0; half >>= 1)
#pragma unroll
            for (int u = 0; u < half; ++u) sum_of[u] += sum_of[u + half];
          acc[i] += sum_of[0];
        }
      }
    }
    // acc: row `in`, classes row(piece, r) of the group
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i < mine) {
        const int c = (me + (g0 + i) * waves) * 16;
        Acc out;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = c + Mma16<T>::row(piece, r);
          const Z b = bias && at < v ? (Z)TypeOf<T>::to_float(bias[at]) : (Z)0;
          out[r] = at < v ? acc[i][r] + b : -(Z)__builtin_inff();
          const float up = fmaxf(top, (float)out[r]), base = up == -__builtin_inff() ? 0.0f : up;
          sum = sum * (double)expf(top - base) + (double)expf((float)(out[r] - (Z)base));
          top = up;
        }
        if (in < n) {
          Z* to = z + (long long)in * ldz + c;
          if constexpr (sizeof(Z) == 4) {
            *(Acc*)(to + 4 * piece) = out;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) to[Mma16<T>::row(piece, r)] = out[r];
          }
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const float other = __shfl_xor(top, o, 64);
    const double more = __shfl_xor(sum, o, 64);
    const float up = fmaxf(top, other), base = up == -__builtin_inff() ? 0.0f : up;
    sum = sum * (double)expf(top - base) + more * (double)expf(other - base);
    top = up;
  }
  if (lane < 16) s_part[wave][lane] = TopSum{sum, top};
  __syncthreads();
  if (t < 16) {
    top = -__builtin_inff();
    sum = 0.0;
    for (int k = 0; k < 4; ++k) top = fmaxf(top, s_part[k][t].top);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    for (int k = 0; k < 4; ++k) sum += s_part[k][t].sum * (double)expf(s_part[k][t].top - base);
    part[t * gridDim.x + blockIdx.x] = TopSum{sum, top};
  }
}

template <int kRotate>
__device__ __forceinline__ double rotated(const double x) {
  const unsigned long long w = __builtin_bit_cast(unsigned long long, x);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)w, 0x120 + kRotate, 0xf, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(w >> 32), 0x120 + kRotate, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (unsigned long long)(unsigned)hi << 32 | (unsigned)lo);
}
// Of every 16 lanes, over those whose number is the same modulo kN.
template <int kN, typename X, typename F>
__device__ __forceinline__ X over_classes(X x, const F f) {
  x = f(x, rotated<8>(x));
  if constexpr (kN <= 4) x = f(x, rotated<4>(x));
  if constexpr (kN <= 2) x = f(x, rotated<2>(x));
  if constexpr (kN <= 1) x = f(x, rotated<1>(x));
  return x;
}
// fold32, fold16 and sum16 for both kinds of logit
template <bool k32>
__device__ __forceinline__ double fold(const double a, const double b) {
  const unsigned long long x = __builtin_bit_cast(unsigned long long, a), y = __builtin_bit_cast(unsigned long long, b);
  const auto swap = [](const unsigned p, const unsigned q) {
    if constexpr (k32) return __builtin_amdgcn_permlane32_swap(p, q, false, false);
    else return __builtin_amdgcn_permlane16_swap(p, q, false, false);
  };
  const auto lo = swap((unsigned)x, (unsigned)y), hi = swap((unsigned)(x >> 32), (unsigned)(y >> 32));
  const unsigned l0 = lo[0], l1 = lo[1], h0 = hi[0], h1 = hi[1];
  return __builtin_bit_cast(double, (unsigned long long)h0 << 32 | l0) +
         __builtin_bit_cast(double, (unsigned long long)h1 << 32 | l1);
}
template <bool k32>
__device__ __forceinline__ float fold(const float a, const float b) {
  return k32 ? fold32(a, b) : fold16(a, b);
}

// kA classes at a time, a value (class, row) each lane of 16: value i = class i / kN, row i % kN.
template <typename T, int kN, int kC, bool kWide>
__global__ __launch_bounds__(kThreads) void few_online_kernel(const T* __restrict__ x, const long long ldx, const int n,
                                                              const int d, const T* __restrict__ w, const long long ldw,
                                                              const int v, const T* __restrict__ bias, const Labels y,
                                                              typename Mma16<T>::Z* __restrict__ z, const int ldz,
                                                              TopSum* __restrict__ part, float* __restrict__ dx_part,
                                                              const int ldpart, const Upstream up) {
  if (up.there()) return;
  constexpr int kV = 16 / (int)sizeof(T), kA = 16 / (kN > kC ? kN : kC), kVals = kA * kN;
  typedef typename Mma16<T>::Z Z;
  typedef typename Mma16<T>::Acc Four;
  __shared__ Four s_z[2][16];      // [value], one sum of each wave
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, in = lane & 15;
  float xs[kN][kC][kV], acc[kN][kC][kV];
#pragma unroll
  for (int r = 0; r < kN; ++r) {
    const bool keep = r < n && y.counts(y.at(r));      // what a row left out holds must not meet its zeros
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      const int c = (j * kThreads + t) * kV;
      to_floats<T>(keep ? load_values<T, false>(x + r * ldx + c, d - c) : u32x4{0, 0, 0, 0}, xs[r][j]);
#pragma unroll
      for (int k = 0; k < kV; ++k) acc[r][j][k] = 0.0f;
    }
  }
  float top = -__builtin_inff();      // of row in % kN, the same in all waves
  double sum = 0.0;
  const long long label = in % kN < n ? y.at(in % kN) : -1;
  int odd = 0;
  for (int v0 = blockIdx.x * kA; v0 < v; v0 += gridDim.x * kA, odd ^= 1) {
    u32x4 ws[kA][kC];
#pragma unroll
    for (int a = 0; a < kA; ++a)
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        const int c = (j * kThreads + t) * kV;
        ws[a][j] = load_values<T, kWide>(w + (long long)min(v0 + a, v - 1) * ldw + c, d - c);
      }
    if constexpr (sizeof(Z) == 8) {      // not to be kept in 64 bits from one round to the next: they take registers
#pragma unroll
      for (int r = 0; r < kN; ++r)
#pragma unroll
        for (int j = 0; j < kC; ++j)
#pragma unroll
          for (int k = 0; k < kV; ++k) asm volatile("" : "+v"(xs[r][j][k]));
    }
    Z part_of[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) part_of[i] = 0;
#pragma unroll
    for (int a = 0; a < kA; ++a)
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        float f[kV];
        to_floats<T>(ws[a][j], f);
#pragma unroll
        for (int r = 0; r < kN; ++r)
#pragma unroll
          for (int k = 0; k < kV; ++k) {
            if constexpr (sizeof(Z) == 4) part_of[a * kN + r] = __builtin_fmaf(f[k], xs[r][j][k], part_of[a * kN + r]);
            else part_of[a * kN + r] = __builtin_fma((double)f[k], (double)xs[r][j][k], part_of[a * kN + r]);
          }
      }
    // sums over the wave: values 4 g .. 4 g + 3 end in the 16 lanes of row g
    Z eight[8], four[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) eight[i] = fold<true>(part_of[i], part_of[i + 8]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      four[i] = over_classes<1>(fold<false>(eight[i], eight[i + 4]), [](const Z p, const Z q) { return p + q; });
    const int value = in + 4 * (lane >> 4);      // of lanes 0 .. 3 of a row
    const Z mine = in == 0 ? four[0] : in == 1 ? four[1] : in == 2 ? four[2] : four[3];
    if (in < 4) ((Z*)&s_z[odd][value])[wave] = mine;
    __syncthreads();      // the other half is written next time, when all have read this one
    const Four of_waves = s_z[odd][in];
    const int a = in / kN, r = in % kN, c = v0 + a;
    const bool real = in < kVals && c < v;
    Z logit = (of_waves[0] + of_waves[1]) + (of_waves[2] + of_waves[3]);
    if (bias && real) logit += (Z)TypeOf<T>::to_float(bias[c]);
    if (!real) logit = -(Z)__builtin_inff();
    if (real && t < 16 && r < n) z[(long long)r * ldz + c] = logit;
    const float up = fmaxf(top, over_classes<kN>((float)logit, [](float p, float q) { return fmaxf(p, q); }));
    const float base = up == -__builtin_inff() ? 0.0f : up;
    const float e = expf((float)(logit - (Z)base)), shrink = expf(top - base);
    sum = sum * (double)shrink + over_classes<kN>((double)e, [](double p, double q) { return p + q; });
    if (__builtin_amdgcn_ballot_w64(top != up)) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, shrink), i));
#pragma unroll
        for (int j = 0; j < kC; ++j)
#pragma unroll
          for (int k = 0; k < kV; ++k) acc[i][j][k] *= f;
      }
    }
    top = up;
    const float e_other = c == label ? 0.0f : e;      // the label's weights join in the end, times p - 1
#pragma unroll
    for (int i = 0; i < kA; ++i)
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        float f[kV];
        to_floats<T>(ws[i][j], f);
#pragma unroll
        for (int q = 0; q < kN; ++q) {
          const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, e_other), i * kN + q));
#pragma unroll
          for (int k = 0; k < kV; ++k) acc[q][j][k] = __builtin_fmaf(p, f[k], acc[q][j][k]);
        }
      }
  }
  if (t < kN) part[t * gridDim.x + blockIdx.x] = TopSum{sum, top};
#pragma unroll
  for (int r = 0; r < kN; ++r)
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      const int c = (j * kThreads + t) * kV;
      if (r < n) {
        float* to = dx_part + ((long long)blockIdx.x * n + r) * ldpart + c;
#pragma unroll
        for (int k = 0; k < kV; k += 4)
          *(f32x4*)(to + k) = f32x4{acc[r][j][k], acc[r][j][k + 1], acc[r][j][k + 2], acc[r][j][k + 3]};
      }
    }
}

// One wave a row.  4 to 8 us, all of it latency.
template <typename Z>
__global__ __launch_bounds__(64 * kFewRows) void few_rows_kernel(const TopSum* __restrict__ part, const int blocks,
                                                                 const Labels y, const int n,
                                                                 const Z* __restrict__ z, const int ldz,
                                                                 const float* __restrict__ divisor, const int mean,
                                                                 const Upstream up_to, TopSum* __restrict__ row,
                                                                 float* __restrict__ scale,
                                                                 float* __restrict__ row_loss,
                                                                 float* __restrict__ small, int* __restrict__ status,
                                                                 float* __restrict__ share,
                                                                 float* __restrict__ of_label) {
  if (up_to.there()) return;
  __shared__ float s_loss[kFewRows];
  __shared__ int s_keep[kFewRows], s_bad[kFewRows];
  const int r = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float top = -__builtin_inff();
  double sum = 0.0;
  if (r < n)
    for (int i = lane; i < blocks; i += 64) {
      const TopSum p = part[r * blocks + i];
      const float up = fmaxf(top, p.top), base = up == -__builtin_inff() ? 0.0f : up;
      sum = sum * (double)expf(top - base) + p.sum * (double)expf(p.top - base);
      top = up;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float other = __shfl_xor(top, o, 64);
    const double more = __shfl_xor(sum, o, 64);
    const float up = fmaxf(top, other), base = up == -__builtin_inff() ? 0.0f : up;
    sum = sum * (double)expf(top - base) + more * (double)expf(other - base);
    top = up;
  }
  const long long label = r < n ? y.at(r) : y.ignore;
  const bool keep = r < n && y.counts(label);
  if (share && r < n) {
    const float base = top == -__builtin_inff() ? 0.0f : top;
    for (int i = lane; i < blocks; i += 64)
      share[r * blocks + i] = keep ? (float)((double)expf(part[r * blocks + i].top - base) / sum) : 0.0f;
  }
  if (lane == 0) {
    float loss = 0.0f;
    if (keep) {
      const Z below = z[(long long)r * ldz + label] - (Z)top;
      loss = (float)(log(sum) - (double)below);
      row[r] = TopSum{sum, top};
      of_label[r] = (float)(((double)expf((float)below) - sum) / sum);
    }
    if (r < n) row_loss[r] = loss;
    s_loss[r] = loss;
    s_keep[r] = keep;
    s_bad[r] = r < n && label != y.ignore && (label < 0 || label >= y.v);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    int count = 0, bad = 0;
    for (int i = 0; i < n; ++i) {
      total += (double)s_loss[i];
      count += s_keep[i];
      bad |= s_bad[i];
    }
    const float div = mean ? fmaxf(divisor ? *divisor : (float)count, 1.0f) : 1.0f;
    *scale = up_to.value() / div;
    small[0] = (float)(total * (double)(1.0f / div));
    small[1] = (float)count;
    small[2] = 1.0f / div;
    *status = bad ? RH_STATUS_LABEL_RANGE : 0;
  }
}

// dW and db of up to four rows whose dX is made online.  A thread has 16 bytes of columns, the rows' features
// beside them in registers; the workgroup's classes are taken `subsets` at a time, a class by tpr threads.  Bound
// by the bytes it writes: 65 536 x 2048 bfloat16 (268 MB) 53 us past the caches, 43 into them.
template <typename T, int kN, bool kPast>
__global__ __launch_bounds__(kThreads) void few_weights_kernel(
    const T* __restrict__ x, const long long ldx, const int n, const int d, const int v, const Labels y,
    const typename Mma16<T>::Z* __restrict__ z, const int ldz, const TopSum* __restrict__ row,
    const float* __restrict__ scale,
    const int per, const int tpr, T* __restrict__ dw, T* __restrict__ db, const Upstream up) {
  if (up.there()) return;
  constexpr int kV = 16 / (int)sizeof(T);
  constexpr int kAtOnce = 128;      // classes whose probabilities wait in LDS
  __shared__ float s_p[kAtOnce][kN];
  __shared__ TopSum s_row[kN];
  __shared__ int s_label[kN];
  const int t = threadIdx.x, subsets = kThreads / tpr, subset = t / tpr;
  const int c = (blockIdx.y * tpr + t % tpr) * kV;
  const float s = *scale;
  if (t < kN) {
    const long long label = t < n ? y.at(t) : y.ignore;
    s_label[t] = t < n && y.counts(label) ? (int)label : -1;
    s_row[t] = s_label[t] >= 0 ? row[t] : TopSum{1.0, 0.0f};
  }
  __syncthreads();
  float xs[kN][kV];
#pragma unroll
  for (int r = 0; r < kN; ++r)      // what a row left out holds must not meet its zeros
    to_floats<T>(s_label[r] >= 0 ? load_values<T, false>(x + r * ldx + c, d - c) : u32x4{0, 0, 0, 0}, xs[r]);
  const int lo = blockIdx.x * per, hi = min(v, lo + per);
  for (int v0 = lo; v0 < hi; v0 += kAtOnce) {
    const int count = min(kAtOnce, hi - v0);
    __syncthreads();
    for (int i = t; i < count * kN; i += kThreads) {
      const int r = i / count, a = i - r * count;
      float p = 0.0f;
      if (s_label[r] >= 0) {
        // the label's p - 1 as (e - sum) / sum, which does not cancel what p was rounded by
        const float e = expf((float)(z[(long long)r * ldz + v0 + a] - (typename Mma16<T>::Z)s_row[r].top));
        p = s_label[r] == v0 + a ? (float)(((double)e - s_row[r].sum) / s_row[r].sum) : e / (float)s_row[r].sum;
        p *= s;
      }
      s_p[a][r] = p;
    }
    __syncthreads();
    if (db && blockIdx.y == 0)
      for (int a = t; a < count; a += kThreads) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < kN; ++r) sum += s_p[a][r];
        db[v0 + a] = TypeOf<T>::from_float(sum);
      }
    if (!dw || c >= d) continue;
#pragma unroll 4
    for (int a = subset; a < count; a += subsets) {
      union {
        T v[kV];
        u32x4 u;
      } out;
#pragma unroll
      for (int k = 0; k < kV; ++k) {
        float g = 0.0f;
#pragma unroll
        for (int r = 0; r < kN; ++r) g = __builtin_fmaf(s_p[a][r], xs[r][k], g);
        out.v[k] = TypeOf<T>::from_float(g);
      }
      T* to = dw + (long long)(v0 + a) * d + c;
      if (d % kV == 0) {
        store16<kPast>(to, out.u);
      } else if (c + kV <= d) {
        __builtin_memcpy(to, &out, 16);
      } else {
#pragma unroll
        for (int k = 0; k < kV; ++k)
          if (c + k < d) to[k] = out.v[k];
      }
    }
  }
}

// The gradients otherwise, by float32 matrix instructions (16 x 16 x 4) where vector ones would take 32
// operations a weight: a wave takes 16 classes by 16 lanes' 16 bytes of columns.  dX = P W needs no transposition: a
// lane's one weight of k is the class of its load, and the columns of its kV instructions are its own kV neighbours.
// dW = P^T X has the rows as k.  P and both products stay float32.  Bound by memory: 16 x 2048 rows, 65 536 classes,
// bfloat16 (268 MB read, 268 written) 139 us; 16 x 572, 62 202 classes, float32 74.  By vector instructions 484, 174.
template <typename T, bool kWide, bool kPast>
__global__ __launch_bounds__(kThreads) void few_products_kernel(
    const T* __restrict__ x, const long long ldx, const int n, const int d, const T* __restrict__ w,
    const long long ldw, const int v, const Labels y, const typename Mma16<T>::Z* __restrict__ z, const int ldz,
    const TopSum* __restrict__ row, const float* __restrict__ scale, const int per, const int waves_a_row,
    T* __restrict__ dw, T* __restrict__ db, float* __restrict__ dx_part, const int ldpart, const Upstream up) {
  if (up.there()) return;
  constexpr int kV = 16 / (int)sizeof(T), kAtOnce = 128, kPitch = kFewRows + 1;      // rows a bank apart
  __shared__ float s_p[kAtOnce * kPitch];
  __shared__ TopSum s_row[kFewRows];
  __shared__ int s_label[kFewRows];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, in = lane & 15, piece = lane >> 4;
  const int subsets = 4 / waves_a_row, subset = wave / waves_a_row;
  const int c = ((blockIdx.y * waves_a_row + wave % waves_a_row) * 16 + in) * kV;
  const float s = *scale;
  if (t < kFewRows) {
    const long long label = t < n ? y.at(t) : y.ignore;
    s_label[t] = t < n && y.counts(label) ? (int)label : -1;
    s_row[t] = s_label[t] >= 0 ? row[t] : TopSum{1.0, 0.0f};
  }
  __syncthreads();
  float xs[4][kV];      // [k / 4]: rows 4 k + piece
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = 4 * k + piece;
    // what a row left out holds must not meet its zeros
    to_floats<T>(s_label[r] >= 0 ? load_values<T, false>(x + r * ldx + c, d - c) : u32x4{0, 0, 0, 0}, xs[k]);
  }
  f32x4 acc[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int lo = blockIdx.x * per, hi = min(v, lo + per);
  for (int v0 = lo; v0 < hi; v0 += kAtOnce) {
    const int count = min(kAtOnce, hi - v0);
    __syncthreads();
    for (int i = t; i < kAtOnce * kFewRows; i += kThreads) {
      const int r = i / kAtOnce, a = i % kAtOnce;
      float p = 0.0f;
      if (a < count && s_label[r] >= 0) {
        // the label's p - 1 as (e - sum) / sum, which does not cancel what p was rounded by
        const float e = expf((float)(z[(long long)r * ldz + v0 + a] - (typename Mma16<T>::Z)s_row[r].top));
        p = s_label[r] == v0 + a ? (float)(((double)e - s_row[r].sum) / s_row[r].sum) : e / (float)s_row[r].sum;
        p *= s;
      }
      s_p[a * kPitch + r] = p;
    }
    __syncthreads();
    if (db && blockIdx.y == 0)
      for (int a = t; a < count; a += kThreads) {
        float sum = 0.0f;
        for (int r = 0; r < n; ++r) sum += s_p[a * kPitch + r];
        db[v0 + a] = TypeOf<T>::from_float(sum);
      }
    for (int a0 = subset * 16; a0 < count; a0 += subsets * 16) {
      u32x4 ws[4];
      if (dx_part) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          ws[k] = load_values<T, kWide>(w + (long long)min(v0 + a0 + 4 * k + piece, v - 1) * ldw + c, d - c);
      }
      if (dw) {
        f32x4 out[kV];
#pragma unroll
        for (int j = 0; j < kV; ++j) out[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = s_p[(a0 + in) * kPitch + 4 * k + piece];
#pragma unroll
          for (int j = 0; j < kV; ++j) out[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(p, xs[k][j], out[j], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int a = a0 + 4 * piece + r;
          union {
            T v[kV];
            u32x4 u;
          } values;
#pragma unroll
          for (int j = 0; j < kV; ++j) values.v[j] = TypeOf<T>::from_float(out[j][r]);
          T* to = dw + (long long)(v0 + a) * d + c;
          if (a < count) {
            if (d % kV == 0) {
              if (c < d) store16<kPast>(to, values.u);
            } else if (c + kV <= d) {
              __builtin_memcpy(to, &values, 16);
            } else {
#pragma unroll
              for (int j = 0; j < kV; ++j)
                if (c + j < d) to[j] = values.v[j];
            }
          }
        }
      }
      if (dx_part) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float p = s_p[(a0 + 4 * k + piece) * kPitch + in];
          float f[kV];
          to_floats<T>(ws[k], f);
#pragma unroll
          for (int j = 0; j < kV; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(p, f[j], acc[j], 0, 0, 0);
        }
      }
    }
  }
  if (dx_part) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = 4 * piece + r;
      float* to = dx_part + ((long long)(blockIdx.x * subsets + subset) * n + at) * ldpart + c;
      if (at < n)
#pragma unroll
        for (int j = 0; j < kV; j += 4) *(f32x4*)(to + j) = f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
    }
  }
}

// Four columns of a row by 64 threads, each every 64th part.  With `share` (online) the parts are weighed
// by it, the label's weights added times p - 1 and the sum scaled here.
template <typename T>
__global__ __launch_bounds__(kThreads) void few_features_kernel(const float* __restrict__ part, const int parts,
                                                                const int n, const int ldpart, const int d,
                                                                const float* __restrict__ share,
                                                                const float* __restrict__ of_label,
                                                                const float* __restrict__ scale, const Labels y,
                                                                const T* __restrict__ w, const long long ldw,
                                                                T* __restrict__ dx, const Upstream up) {
  if (up.there()) return;
  __shared__ f32x4 s_sum[64][4];
  const int quad = threadIdx.x & 3, slice = threadIdx.x >> 2;
  const int c = (blockIdx.x * 4 + quad) * 4, r = blockIdx.y;
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  long long label = 0;
  if (share) {
    label = y.at(r);
    if (!y.counts(label)) {      // its sums may hold anything
      if (slice == 0)
        for (int k = 0; k < 4 && c + k < d; ++k) dx[(long long)r * d + c + k] = TypeOf<T>::from_float(0.0f);
      return;
    }
  }
  if (c < ldpart) {
#pragma unroll 4
    for (int i = slice; i < parts; i += 64) {
      const f32x4 p = *(const f32x4*)(part + ((long long)i * n + r) * ldpart + c);
      const float f = share ? share[r * parts + i] : 1.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] = __builtin_fmaf(p[k], f, sum[k]);
    }
  }
  s_sum[slice][quad] = sum;
  for (int half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (slice < half) s_sum[slice][quad] = sum = sum + s_sum[slice + half][quad];
  }
  if (slice == 0 && c < d) {
    for (int k = 0; k < 4 && c + k < d; ++k) {
      float out = sum[k];
      if (share) out = __builtin_fmaf(of_label[r], TypeOf<T>::to_float(w[label * ldw + c + k]), out) * *scale;
      dx[(long long)r * d + c + k] = TypeOf<T>::from_float(out);
    }
  }
}

static Upstream upstream_of(const rh_linear_ce_args& q) { return Upstream{q.upstream, q.grad}; }

template <typename T, int kN>
static int launch_weights(const rh_linear_ce_args& q, const FewPlan& p, const FewSpace& s, const Labels& y,
                          hipStream_t stream) {
  auto kernel = p.past ? few_weights_kernel<T, kN, true> : few_weights_kernel<T, kN, false>;
  hipLaunchKernelGGL(kernel, dim3(p.grad_blocks, p.slices), dim3(kThreads), 0, stream, (const T*)q.x,
                     (long long)q.ldx, (int)q.n, q.d, (int)q.v, y, (const typename Mma16<T>::Z*)s.z, p.ldz, s.row, s.scale, p.per, p.tpr, (T*)q.dw,
                     (T*)q.db, upstream_of(q));
  RH_CHECK_LAUNCH("few_weights_kernel");
  return RH_OK;
}

template <typename T>
static int launch_products(const rh_linear_ce_args& q, const FewPlan& p, const FewSpace& s, const Labels& y,
                           hipStream_t stream) {
  auto kernel = p.wide_w ? p.past ? few_products_kernel<T, true, true> : few_products_kernel<T, true, false>
                         : few_products_kernel<T, false, false>;
  hipLaunchKernelGGL(kernel, dim3(p.grad_blocks, p.slices), dim3(kThreads), 0, stream, (const T*)q.x, (long long)q.ldx,
                     (int)q.n, q.d, (const T*)q.w, (long long)q.ldw, (int)q.v, y, (const typename Mma16<T>::Z*)s.z, p.ldz, s.row, s.scale, p.per,
                     p.tpr / 16, (T*)q.dw, (T*)q.db, s.dx_part, p.ldpart, upstream_of(q));
  RH_CHECK_LAUNCH("few_products_kernel");
  return RH_OK;
}

template <typename T, int kN, int kC>
static int launch_online(const rh_linear_ce_args& q, const FewPlan& p, const FewSpace& s, const Labels& y,
                         hipStream_t stream) {
  auto kernel = p.wide_w ? few_online_kernel<T, kN, kC, true> : few_online_kernel<T, kN, kC, false>;
  hipLaunchKernelGGL(kernel, dim3(p.blocks), dim3(kThreads), 0, stream, (const T*)q.x, (long long)q.ldx, (int)q.n, q.d,
                     (const T*)q.w, (long long)q.ldw, (int)q.v, (const T*)q.bias, y, (typename Mma16<T>::Z*)s.z, p.ldz, s.part, s.dx_part,
                     p.ldpart, upstream_of(q));
  RH_CHECK_LAUNCH("few_online_kernel");
  return RH_OK;
}

template <typename T, int kN>
static int online_chunks(const rh_linear_ce_args& q, const FewPlan& p, const FewSpace& s, const Labels& y,
                         hipStream_t stream) {
  if (p.chunks == 1) return launch_online<T, kN, 1>(q, p, s, y, stream);
  if (p.chunks == 2) return launch_online<T, kN, 2>(q, p, s, y, stream);
  if constexpr (kN * 4 * (16 / (int)sizeof(T)) <= 64) return launch_online<T, kN, 4>(q, p, s, y, stream);
  return RH_EINVAL;      // no plan leads here
}

template <typename T>
static int run_typed(const rh_linear_ce_args& q, int flags, hipStream_t stream) {
  typedef typename Mma16<T>::Z Z;
  const int n = (int)q.n, v = (int)q.v;
  const FewPlan p = few_plan(n, q.d, v, q.dtype, flags);
  const FewSpace s = few_space(q.workspace, p, n, flags);
  const Labels y{q.labels, q.labels_int64, q.ignore_index, v};
  if (p.rows) {
    if (int rc = p.rows == 1   ? online_chunks<T, 1>(q, p, s, y, stream)
                 : p.rows == 2 ? online_chunks<T, 2>(q, p, s, y, stream)
                               : online_chunks<T, 4>(q, p, s, y, stream))
      return rc;
  } else {
    auto logits = p.wide_w ? few_logits_kernel<T, true> : few_logits_kernel<T, false>;
    hipLaunchKernelGGL(logits, dim3(p.blocks), dim3(kThreads), 16 * kPitch, stream, (const T*)q.x, (long long)q.ldx, n, q.d,
                       (const T*)q.w, (long long)q.ldw, v, (const T*)q.bias, p.groups, p.waves, (Z*)s.z, p.ldz, s.part, upstream_of(q));
    RH_CHECK_LAUNCH("few_logits_kernel");
  }
  hipLaunchKernelGGL(few_rows_kernel<Z>, dim3(1), dim3(64 * kFewRows), 0, stream, s.part, p.blocks, y, n, (const Z*)s.z, p.ldz, q.divisor,
                     q.reduction == RH_CE_MEAN, upstream_of(q), s.row, s.scale, q.row_loss, q.small, (int*)(q.small + 3), s.share,
                     s.of_label);
  RH_CHECK_LAUNCH("few_rows_kernel");
  if (!q.dx && !q.dw && !q.db) return RH_OK;
  if (!p.rows) {
    if (int rc = launch_products<T>(q, p, s, y, stream)) return rc;
  } else if (q.dw || q.db) {
    if (int rc = p.rows == 1   ? launch_weights<T, 1>(q, p, s, y, stream)
                 : p.rows == 2 ? launch_weights<T, 2>(q, p, s, y, stream)
                               : launch_weights<T, 4>(q, p, s, y, stream))
      return rc;
  }
  if (q.dx) {
    hipLaunchKernelGGL(few_features_kernel<T>, dim3(ceil_div(q.d, 16), n), dim3(kThreads), 0, stream, s.dx_part, p.parts, n,
                       p.ldpart, q.d, s.share, s.of_label, s.scale, y, (const T*)q.w, (long long)q.ldw, (T*)q.dx,
                       upstream_of(q));
    RH_CHECK_LAUNCH("few_features_kernel");
  }
  return RH_OK;
}

int run_few(const rh_linear_ce_args& q, int flags, hipStream_t stream) {
  if (q.dtype == RH_F32) return run_typed<float>(q, flags, stream);
  if (q.dtype == RH_BF16) return run_typed<__bf16>(q, flags, stream);
  return run_typed<_Float16>(q, flags, stream);
}

}  // namespace ce
}  // namespace rh
