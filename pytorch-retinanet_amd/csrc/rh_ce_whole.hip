// The classifier loss for label sets that fit a workgroup's registers (gfx950): 64 rows by up to 640 classes.
// The logits are never written: a workgroup makes all of its rows' logits, takes their softmax where they are,
// writes P once (dW's operand) and multiplies it with the weights for dX while it is still in LDS.
//
// 49 104 x 256 against 601 classes, bfloat16: 80 us, where the logits by tiles, the joining of their sums, P
// from the kept logits and dX by tiles took 103.  Of a workgroup's 25 us the logits take 8.5, the exponentials
// 5.5, P 3.6 and dX 7.2: the products are bound by LDS (a wave of 32 rows reads a fragment of weights for every
// instruction; the matrix units are busy 18% of the time), the rest by the vector units.  Up to 256 classes two
// workgroups share a CU and run these against each other (80 classes: 24.5 us, 29.7 one at a time).  The weights
// in panels instead of rows: 79 us, less than laying them out costs.
#include "rh_ce.h"

namespace rh {
namespace ce {

constexpr int kWholeThreads = 512;      // 8 waves: two of 32 rows, by four of kF * 32 classes
constexpr int kLogitRing = 3;
constexpr int kDxColumns = 256;

template <int kF>
struct WholeLds {
  // up to 256 classes two workgroups fit a CU
  static constexpr int kDxRing = kF == 1 ? 3 : kF == 2 ? 2 : 4;
  static constexpr int kX = kWholeRows * kStepBytes, kW = 128 * kF * kStepBytes, kStage = kX + kW;
  static constexpr int kP = kWholeRows * 128 * kF * 2, kDxStage = kDxColumns * kStepBytes;
  static constexpr int kLogits = kLogitRing * kStage + kX, kDx = kP + kDxRing * kDxStage;
  static constexpr int kBytes = kLogits > kDx ? kLogits : kDx;
};

template <typename T, int kF>
__global__ __launch_bounds__(kWholeThreads, kF <= 2 ? 4 : 2) void whole_kernel(const WholeArgs<T> a) {
  typedef WholeLds<kF> L;
  constexpr int kClasses = 128 * kF;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  RH_LDS char* lds = (RH_LDS char*)smem;
  __shared__ __attribute__((aligned(16))) float s_bias[kClasses];
  __shared__ float s_cols[2][kClasses];
  __shared__ __attribute__((aligned(16))) float s_top[4][kWholeRows];
  __shared__ float s_sum[4][kWholeRows], s_zl[kWholeRows];
  __shared__ int s_label[kWholeRows];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wr = wave & 1, wc = wave >> 1, half = lane >> 5;
  const int m0 = blockIdx.x * kWholeRows, rows = a.chunk.rows(a.n_valid) - m0;      // of this workgroup
  if (rows <= 0) {
    if (t == 0) a.loss[blockIdx.x] = 0.0;
    if (a.column_sums)
      for (int c = t; c < a.v; c += kWholeThreads) a.column_sums[(long long)blockIdx.x * a.v + c] = 0.0f;
    return;
  }
  if (t < kWholeRows) s_label[t] = t < rows ? a.label[m0 + t] : -1;
  for (int c = t; c < kClasses; c += kWholeThreads)      // classes that are none: as if masked
    s_bias[c] = c >= a.v ? -__builtin_inff() : a.bias ? TypeOf<T>::to_float(a.bias[c]) : 0.0f;

  // Logits.  A step's loads a thread: 16 bytes of the features (the upper four waves' fall into a spare place)
  // and of kF x 128 rows of weights.
  f32x16 acc[kF];
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[f][r] = 0.0f;
  {
    const int row = t >> 2, chunk = (t & 3) ^ ((row >> 2) & 3);
    const int x_at = row < kWholeRows && row < rows ? row * kStepBytes + chunk * 16 : kNowhere;
    const unsigned base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds);
    const unsigned me = __builtin_amdgcn_readfirstlane((unsigned)(wave * 1024));
    const unsigned spare = base + kLogitRing * L::kStage + me - 4096;
    const char *x = a.x + (long long)m0 * kStepBytes, *w = a.w;
    long long x_left = a.x_bytes - (long long)m0 * kStepBytes, w_left = a.w_bytes;
    const long long x_step = (long long)a.chunk_rows * kStepBytes;
    int to = 0;
    auto load = [&](const int s) {
      u32x4 rx = make_rsrc(x, s < a.steps ? x_left : 0), rw = make_rsrc(w, s < a.steps ? w_left : 0);
      asm volatile("s_nop 4" : "+s"(rx), "+s"(rw));      // see Loader::plan
      const unsigned stage = base + to * L::kStage;
      load_to_lds<0>(rx, me < 4096 ? stage + me : spare, x_at);
      const bool in = s < a.steps - 1 || chunk * 16 < a.w_limit;
      each<kF>([&](auto i) {
        constexpr int k = decltype(i)::value;
        load_to_lds<k * 8192>(rw, stage + L::kX + me, in ? (int)((row + k * 128) * a.ldw) + chunk * 16 : kNowhere);
      });
      x += x_step;
      x_left -= x_step;
      w += kStepBytes;
      w_left -= kStepBytes;
      to = to == kLogitRing - 1 ? 0 : to + 1;
    };
    Fragments<kRows, kWholeRows, 1> fx;
    Fragments<kRows, kClasses, kF> fw;
    fx.init(wr * 32);
    fw.init(wc * kF * 32);
    load(0);
    load(1);
    int at = 0;
    for (int s = 0; s < a.steps; ++s) {
      stage_wait<kF + 1>();      // step s has landed, step s - 1 is read out
      load(s + 2);
      const RH_LDS char* stage = lds + at * L::kStage;
      at = at == kLogitRing - 1 ? 0 : at + 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const u32x4 xv = fx.read(stage, 0, kk);
#pragma unroll
        for (int f = 0; f < kF; ++f) acc[f] = TypeOf<T>::mma(fw.read(stage + L::kX, f, kk), xv, acc[f]);
      }
    }
    stage_wait<0>();
  }

  // dX's weights start on their way
  Loader<kCols, false, kDxColumns, kWholeThreads, 1, 0> lw;
  const int dx_steps = (a.v + kStepK - 1) / kStepK, last = a.v - (dx_steps - 1) * kStepK;
  const unsigned dx_to = __builtin_amdgcn_readfirstlane((unsigned)(size_t)lds + L::kP + wave * 1024);
  int dx_next = 0;
  auto load_dx = [&](const int s) {
    lw.plan(s < dx_steps);
    lw.begin(dx_to + dx_next * L::kDxStage, s == dx_steps - 1 ? last : kStepK);
    lw.template load<true, 0>();
    lw.template load<true, 1>();
    dx_next = dx_next == L::kDxRing - 1 ? 0 : dx_next + 1;
  };
  auto start_dx = [&](const int n0) {
    lw.init(a.w + n0 * (int)sizeof(T), a.ldw, a.w_bytes - n0 * (int)sizeof(T), 0, dx_steps);
    dx_next = 0;
#pragma unroll
    for (int s = 0; s < L::kDxRing - 1; ++s) load_dx(s);
  };
  if (a.dx) start_dx(0);

  // Softmax.  A lane has a row's classes first + 32 f + 8 q + r, its partner 32 lanes on four further.
  const int row = 32 * wr + (lane & 31), first = wc * kF * 32 + 4 * half, y = s_label[row] - first;
  float top = -__builtin_inff(), z_label = 0.0f;
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 b = *(const f32x4*)&s_bias[first + 32 * f + 8 * q];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = acc[f][4 * q + r] + b[r];
        acc[f][4 * q + r] = z;
        top = fmaxf(top, z);
        z_label = y == 32 * f + 8 * q + r ? z : z_label;
      }
    }
  top = fmaxf(top, __shfl_xor(top, 32, 64));
  if (half == 0) s_top[wc][row] = top;
  if (y >= 0 && y < kF * 32 && (y & 7) < 4) s_zl[row] = z_label;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0][row], s_top[1][row]), fmaxf(s_top[2][row], s_top[3][row]));
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int f = 0; f < kF; ++f)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      acc[f][i] = exp_for<T>(acc[f][i] - base);
      sum += acc[f][i];
    }
  sum += __shfl_xor(sum, 32, 64);
  if (half == 0) s_sum[wc][row] = sum;
  __syncthreads();
  sum = (s_sum[0][row] + s_sum[1][row]) + (s_sum[2][row] + s_sum[3][row]);
  if (wc == 0) {      // waves 0 and 1: a row a lane of the lower half
    double loss = 0.0;
    if (half == 0 && row < rows) {
      const float l = (top - s_zl[row]) + logf(sum);
      a.row_loss[a.map[m0 + row]] = l;
      loss = (double)l;
    }
    loss = wave_sum(loss);
    if (lane == 0) ((double*)s_top)[wr] = loss;      // all have read the maxima
  }

  // P; the label's p - 1 as (e - sum) / sum, which does not cancel what p was rounded by
  const float inv = 1.0f / sum;
#pragma unroll
  for (int f = 0; f < kF; ++f) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float less = y == 32 * f + 8 * (i >> 2) + (i & 3) ? sum : 0.0f;
      acc[f][i] = (acc[f][i] - less) * inv;
    }
  }
  if (rows < kWholeRows && row >= rows) {
#pragma unroll
    for (int f = 0; f < kF; ++f)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[f][i] = 0.0f;
  }
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    const int panel = wc * kF + f;
    if (a.column_sums) {
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {      // value i in the first 16 lanes of a half, i + 8 in the others
        const float c = sum16(fold16(acc[f][i], acc[f][i + 8]));
        mine = (lane & 15) == i ? c : mine;
      }
      const int i = (lane & 7) + 8 * ((lane >> 4) & 1);
      if ((lane & 15) < 8) s_cols[wr][panel * 32 + 8 * (i >> 2) + 4 * half + (i & 3)] = mine;
    }
    unsigned long long group[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      Vec4<T> v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v.v[r] = TypeOf<T>::from_float(acc[f][4 * q + r] * PScale<T>::up);
      group[q & 1] = __builtin_bit_cast(unsigned long long, v);
      if (q & 1) {
        const u32x4 eight = whole_group(group[0], group[1]);
        const int chunk = q - 1 + half;
        *(RH_LDS u32x4*)(lds + panel * 4096 + row * kStepBytes + ((chunk ^ ((row >> 2) & 3)) << 4)) = eight;
        if (panel * kStepK < a.ldp && row < rows)
          *(u32x4*)(a.p + in_panels(m0 + row, panel * kStepK + chunk * 8, a.chunk_rows) * 2) = eight;
      }
    }
  }
  __syncthreads();
  if (t == 0) a.loss[blockIdx.x] = ((double*)s_top)[0] + ((double*)s_top)[1];
  if (a.column_sums)
    for (int c = t; c < a.v; c += kWholeThreads)
      a.column_sums[(long long)blockIdx.x * a.v + c] = s_cols[0][c] + s_cols[1][c];
  if (!a.dx) return;

  // dX, 256 columns at a time: a wave 32 rows by 64 of them
  Fragments<kRows, kWholeRows, 1> fp;
  Fragments<kCols, kDxColumns, 2> fw;
  fp.init(wr * 32);
  fw.init(wc * 64);
  const float scale = *a.scale * PScale<T>::down;
  const bool wide = (a.d & 7) == 0;
  for (int n0 = 0; n0 < a.d; n0 += kDxColumns) {
    f32x16 out[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) out[j][r] = 0.0f;
    int at = 0;
    for (int s = 0; s < dx_steps; ++s) {
      stage_wait<2 * (L::kDxRing - 2)>();
      load_dx(s + L::kDxRing - 1);
      const RH_LDS char *p = lds + s * 4096, *stage = lds + L::kP + at * L::kDxStage;
      at = at == L::kDxRing - 1 ? 0 : at + 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const u32x4 pv = fp.read(p, 0, kk);
#pragma unroll
        for (int j = 0; j < 2; ++j) out[j] = TypeOf<T>::mma(fw.read(stage, j, kk), pv, out[j]);
      }
    }
    stage_wait<0>();
    if (n0 + kDxColumns < a.d) start_dx(n0 + kDxColumns);
    if (row >= rows) continue;
    T* to = a.dx + (long long)a.map[m0 + row] * a.d + n0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unsigned long long group[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        Vec4<T> v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v.v[r] = TypeOf<T>::from_float(out[j][4 * q + r] * scale);
        group[q & 1] = __builtin_bit_cast(unsigned long long, v);
        if (q & 1) {
          const u32x4 eight = whole_group(group[0], group[1]);
          const int c = wc * 64 + 32 * j + 8 * (q - 1 + half), left = a.d - n0 - c;
          if (wide) {
            if (left > 0) *(u32x4*)(to + c) = eight;
          } else if (left >= 8) {
            __builtin_memcpy(to + c, &eight, 16);
          } else {
            T single[8];
            __builtin_memcpy(single, &eight, 16);
#pragma unroll
            for (int r = 0; r < 8; ++r)
              if (r < left) to[c + r] = single[r];
          }
        }
      }
    }
  }
}

template <typename T, int kF>
static int launch_whole(const WholeArgs<T>& a, hipStream_t stream) {
  auto kernel = whole_kernel<T, kF>;
  constexpr int kBytes = WholeLds<kF>::kBytes;
  RH_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kBytes));
  hipLaunchKernelGGL(kernel, dim3(ceil_div(a.chunk.most, kWholeRows)), dim3(kWholeThreads), kBytes, stream, a);
  RH_CHECK_LAUNCH("whole_kernel");
  return RH_OK;
}

template <typename T>
int run_whole(const WholeArgs<T>& a, hipStream_t stream) {
  switch (ceil_div(a.v, 128)) {
    case 1: return launch_whole<T, 1>(a, stream);
    case 2: return launch_whole<T, 2>(a, stream);
    case 3: return launch_whole<T, 3>(a, stream);
    case 4: return launch_whole<T, 4>(a, stream);
    default: return launch_whole<T, 5>(a, stream);
  }
}
template int run_whole<__bf16>(const WholeArgs<__bf16>&, hipStream_t);
template int run_whole<_Float16>(const WholeArgs<_Float16>&, hipStream_t);

}  // namespace ce
}  // namespace rh
