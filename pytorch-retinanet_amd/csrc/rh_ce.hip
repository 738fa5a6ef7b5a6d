// Softmax cross entropy of a classifier's last projection over a large label set, forward and
// backward (gfx950).
//
//   z[n][v] = x[n] . w[v] + b[v],   lse[n] = log sum_v exp z[n][v]
//   row[n]  = lse[n] - z[n][y_n],   loss = s sum_n row[n],   s = 1 / max(1, rows counted)  or  1
//   P[n][v] = exp(z[n][v] - lse[n]) - [v == y_n]
//   dX = s P W,   dW = s P^T X,   db = s sum_n P
//
// Rows whose label is ignore_index, or outside [0, V), take no part: the features of the others are
// laid out one after the other in a scratch copy first (its rows padded to whole tile steps), so
// what stands in a row left out never meets a product, not even as 0 * inf, and costs nothing.
//
// The logits of a chunk of rows (2 GiB of them at most) are made once, each tile leaving its rows' (max,
// sum of exponentials) behind and, for the gradients, the logits in 16 bits (float: as they are); P takes
// their place when the rows' sums are known, and two more products make dX and dW: 6 n d v operations.
// Making the logits again instead takes 8 n d v, and P from them no fewer bytes.  Up to 640 classes
// (rh_ce_whole.hip) and up to 16 rows (rh_ce_few.hip) there are other ways.
//
// 4096 x 2048 rows, a twentieth left out, 32 768 classes, bfloat16, us, the least of eight passes: logits 504, P 82,
// dX 426, dW 468, all else 42.  The three products make 1.04, 1.23 and 1.12 PFLOP/s.  The matrix units are busy
// for 57, 70 and 60 % of the CUs' cycles (8192 x 4096: 69, 73 and 66 %): a tile's start and end are not hidden (the
// logits' end, 256 x 256 exponentials a workgroup, takes 14 us).  And the clock is 1.9 GHz there (1.75) where the same
// launches in the same cycles run at 2.4 on zeros.
#include "rh_ce.h"

namespace rh {
namespace ce {

// ---------------------------------------------------------------------------------------------
// Labels, rows
// ---------------------------------------------------------------------------------------------
// Per block of `per` rows: how many count, and whether a label lies outside [0, V).  5 us, all of it latency.
__global__ __launch_bounds__(64) void count_rows_kernel(const Labels y, const int n, const int per,
                                                       int2* __restrict__ blocks) {
  const long long lo = (long long)blockIdx.x * per, hi = min((long long)n, lo + per);
  int count = 0, bad = 0;
  for (long long i = lo + threadIdx.x; i < hi; i += 64) {
    const long long t = y.at(i);
    count += y.counts(t);
    bad |= t != y.ignore && (t < 0 || t >= y.v);
  }
  count = wave_sum(count);
  bad = __any(bad);
  if (threadIdx.x == 0) blocks[blockIdx.x] = make_int2(count, bad);
}

struct RowInfo {
  int* map;        // [n] place -> row
  int* label;      // [n] place -> label
  int* n_valid;    // [1]
  float* scale;    // [1] s * expected upstream gradient
};

// Eight values as the matrix units' operand: the values themselves, or a float's three parts.
template <typename T>
struct Eight {
  u32x4 part[TypeOf<T>::kParts];
};
template <typename T>
__device__ __forceinline__ Eight<T> in_parts(const float (&f)[8]) {
  typedef typename TypeOf<T>::Part P;
  Eight<T> out;
  union {
    P v[8];
    u32x4 u;
  } w[TypeOf<T>::kParts];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float left = f[k];
#pragma unroll
    for (int i = 0; i < TypeOf<T>::kParts; ++i) {
      if constexpr (sizeof(T) == 4) {
        // the nearest bfloat16, but not infinity for a finite number
        const float most = 3.38953139e38f;
        const float near = __builtin_fabsf(left) > most && __builtin_fabsf(left) < __builtin_inff()
                               ? __builtin_copysignf(most, left) : left;
        w[i].v[k] = (P)near;
        left -= (float)w[i].v[k];
      } else {
        w[i].v[k] = (P)left;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TypeOf<T>::kParts; ++i) out.part[i] = w[i].u;
  return out;
}

// Eight values from p on, of which `have` exist (the others are zero), in parts.  p is aligned to its elements only:
// the card's wide loads ask for no more.
template <typename T>
__device__ __forceinline__ Eight<T> load_parts(const T* p, const int have) {
  if constexpr (sizeof(T) == 2) {
    union {
      T v[8];
      Eight<T> e;
    } w;
    if (have >= 8) {
      __builtin_memcpy(&w, p, 16);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w.v[k] = k < have ? p[k] : (T)0.0f;
    }
    return w.e;
  } else {
    float f[8];
    if (have >= 8) {
      __builtin_memcpy(f, p, 32);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = k < have ? p[k] : 0.0f;
    }
    return in_parts<T>(f);
  }
}

// Copies the rows that count to their places in the chunks' panels, padded with zeros to whole panels; sets
// what a row left out gets: no loss, no gradient.  A workgroup takes `per` rows and every gridDim.y-th panel;
// a wave 16 rows of a panel at a time, a kilobyte where they are neighbours.  Bound by memory: 49 104 x 256
// bfloat16, 22 + 22 MB: 13 us.
template <typename T>
__global__ __launch_bounds__(kThreads) void place_rows_kernel(
    const T* __restrict__ x, const long long ldx, const int d, const Labels y, const int n, const int per,
    const int2* __restrict__ blocks, char* __restrict__ xp, const long long part, const int panels, const int chunk,
    const RowInfo info,
    float* __restrict__ row_loss, T* __restrict__ dx, float* __restrict__ small, int* __restrict__ status,
    const float* __restrict__ total, const int mean, const Upstream up) {
  if (up.there()) {
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *info.n_valid = kThere;
    return;
  }
  __shared__ int s_red[4], s_all[4], s_bad[4];
  __shared__ int s_place[kThreads];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  int before = 0, all = 0, bad = 0;
  if (blocks) {
    for (int i = t; i < (int)gridDim.x; i += kThreads) {
      const int2 c = blocks[i];
      if (i < (int)blockIdx.x) before += c.x;
      all += c.x;
      bad |= c.y;
    }
  } else {      // few rows: every workgroup counts them all
    for (int i = t; i < n; i += kThreads) {
      const long long l = y.at(i);
      const int c = y.counts(l);
      if (i < (int)blockIdx.x * per) before += c;
      all += c;
      bad |= l != y.ignore && (l < 0 || l >= y.v);
    }
  }
  before = wave_sum(before);
  all = wave_sum(all);
  bad = __any(bad);
  if (lane == 0) {
    s_red[wave] = before;
    s_all[wave] = all;
    s_bad[wave] = bad;
  }
  __syncthreads();
  before = s_red[0] + s_red[1] + s_red[2] + s_red[3];
  const bool first = blockIdx.y == 0;
  if (first && blockIdx.x == 0 && t == 0) {
    all = s_all[0] + s_all[1] + s_all[2] + s_all[3];
    *info.n_valid = all;
    const float div = mean ? fmaxf(total ? *total : (float)all, 1.0f) : 1.0f;
    *info.scale = up.value() / div;
    small[1] = (float)all;
    small[2] = 1.0f / div;
    *status = (s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3]) ? RH_STATUS_LABEL_RANGE : 0;
  }
  __syncthreads();
  // this block's rows: place within the block by a ballot count (per <= 256)
  const long long lo = (long long)blockIdx.x * per;
  const int rows = (int)min((long long)per, n - lo);
  bool keep = false;
  long long label = 0;
  if (t < rows) {
    label = y.at(lo + t);
    keep = y.counts(label);
  }
  const unsigned long long kept = __ballot(keep);
  if (lane == 0) s_red[wave] = __popcll(kept);
  __syncthreads();
  int at = before + __popcll(kept & ((1ull << lane) - 1ull));
  for (int i = 0; i < wave; ++i) at += s_red[i];
  if (t < rows) {
    s_place[t] = keep ? at : -1;
    if (first) {
      if (keep) {
        info.map[at] = (int)(lo + t);
        info.label[at] = (int)label;
      } else {
        row_loss[lo + t] = 0.0f;
      }
    }
  }
  __syncthreads();
  for (int p = blockIdx.y + gridDim.y * wave; p < panels; p += gridDim.y * 4) {
    const int c = p * kStepK + (lane & 3) * 8;
#pragma unroll 2
    for (int r = lane >> 2; r < rows; r += 16) {
      const int to = s_place[r];
      if (to < 0) continue;
      const Eight<T> w = load_parts<T>(x + (lo + r) * ldx + c, d - c);
      const int in = to / chunk;
      char* dst = xp + ((long long)in * chunk * panels * kStepK + in_panels(to - in * chunk, c, chunk)) * 2;
#pragma unroll
      for (int i = 0; i < TypeOf<T>::kParts; ++i) *(u32x4*)(dst + i * part) = w.part[i];
    }
  }
  if (dx && first)
    for (int r = wave; r < rows; r += 4)
      if (s_place[r] < 0) {
        T* dst = dx + (lo + r) * (long long)d;
        for (int c = lane; c < d; c += 64) dst[c] = (T)0.0f;
      }
}

// A copy of the weights with rows of whole 16-byte pieces (ldp: of whole panels), for a row length or stride that
// has none: the products' loads to LDS need them.  Bound by memory.
template <typename T>
__global__ __launch_bounds__(kThreads) void pad_rows_kernel(const T* __restrict__ w, const long long ldw,
                                                            const int d, const int v, T* __restrict__ out,
                                                            const int ldp, const int* __restrict__ n_valid) {
  if (*n_valid == kThere) return;
  const int lane = threadIdx.x & 63;
  for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < v; r += (long long)gridDim.x * 4)
#pragma unroll 4
    for (int c = lane * 8; c < ldp; c += 512)
      *(u32x4*)(out + r * ldp + c) = load_parts<T>(w + r * ldw + c, d - c).part[0];
}

// The weights in panels and parts (float), by 16 rows of a panel a wave.  Bound by memory: 16 384 x 1024, 67 MB read
// and 101 written: 32 us.
template <typename T>
__global__ __launch_bounds__(kThreads) void take_apart_kernel(const T* __restrict__ w, const long long ldw, const int d,
                                                              const int v, const int panels, char* __restrict__ out,
                                                              const long long part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x * 16 + (lane >> 2);
  if (r >= v) return;
  for (int p = blockIdx.y * 4 + wave; p < panels; p += gridDim.y * 4) {
    const int c = p * kStepK + (lane & 3) * 8;
    const Eight<T> e = load_parts<T>(w + (long long)r * ldw + c, d - c);
    char* dst = out + in_panels(r, c, v) * 2;
#pragma unroll
    for (int i = 0; i < TypeOf<T>::kParts; ++i) *(u32x4*)(dst + i * part) = e.part[i];
  }
}

// ---------------------------------------------------------------------------------------------
// Logits of one tile, and what becomes of them
// ---------------------------------------------------------------------------------------------
struct Grid {
  int m, n;        // tiles
};

// Tiles in groups of eight rows of tiles, down a group's column first: the workgroups that run side
// by side on an XCD share both operands' rows in its L2.
__device__ __forceinline__ int2 tile_at(const Grid g, const int t) {
  const int span = 8 * g.n, first = t / span * 8, rows = min(8, g.m - first), in = t % span;
  return make_int2(first + in % rows, in / rows);
}

// The call's loss from the row blocks' sums, by one workgroup.
__device__ __forceinline__ void add_losses(const double* __restrict__ parts, const int n, float* __restrict__ small) {
  __shared__ double s_red[4];
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) sum += parts[i];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) small[0] = (float)(((s_red[0] + s_red[1]) + (s_red[2] + s_red[3])) * (double)small[2]);
}

// How a logit waits for its row's sum where it is kept: as it is (float), or for the 16-bit types as
// its distance below the largest of its group of columns in the row, in steps of 1 / kSteps of a
// factor of two: an error of at most half a step, which changes p by less than 2^-12 (bfloat16) or
// 2^-13 (float16) relative, a sixteenth and a quarter of what rounding p to the type does.  The last
// code is probability 0; it stands for p < 2^-32 or 2^-23 of the largest.
template <typename T>
struct Kept {
  typedef unsigned short type;
  static constexpr float kSteps = 2048.0f;
};
template <>
struct Kept<_Float16> {
  typedef unsigned short type;
  static constexpr float kSteps = 2840.0f;
};
template <>
struct Kept<float> {
  typedef float type;
  static constexpr float kSteps = 1.0f;
};

// How many splits a product of fewer rows than it was launched for takes: its workgroups share the tiles there are.
struct Sharing {
  int bm, tiles_n;         // of a tile's rows; tiles side by side
  int workgroups;
  int least, most;         // splits
  __device__ __forceinline__ int tiles_m(const int rows) const { return (rows + bm - 1) / bm; }
  __device__ __forceinline__ int splits(const int rows) const {
    return least == most || rows <= 0 ? least : min(most, workgroups / (tiles_m(rows) * tiles_n));
  }
};

template <typename T>
struct LogitArgs {
  const char* x;       // the chunk's placed rows, in panels of chunk_rows
  long long x_bytes, x_part;
  int chunk_rows;
  const char* w;       // the weights: rows ldw bytes apart, or (float) panels, ldw from one to the next
  long long ldw, w_bytes, w_part;
  const T* bias;
  int steps;           // of k
  int w_limit;         // bytes of the last step that are the weights' rows
  int v;
  Grid grid;
  Chunk chunk;
  const int* n_valid;
  const int* label;    // [place], as everything below by the chunk's places
  float2* stats;       // [group of classes][place]  (max, sum of exp above it)
  long long ld_stats;
  float* z_label;      // [place]
  void* z;             // the logits kept, in panels of chunk_rows, of ldp columns
  int ldp;
  Sharing sharing;
  float* part;         // [split][place of whole tiles][ldp]  kParted's sums
};

// kStats: the groups' (max, sum) only, a group being a wave's part of the tile's classes.  kKeep: and the
// logits.  kParted: float sums over a part of the features only, for sum_logits_kernel.
enum What { kStats, kKeep, kParted };

// What becomes of a tile's logits.  kPlain: every class is there and none has a bias; else each column
// gets something, minus infinity where there is no class.
template <typename T, typename S, What kWhat, bool kPlain, typename Acc>
__device__ __forceinline__ void finish_logits(const LogitArgs<T>& a, const Acc& tile, const int m0, const int n0,
                                              const int rows) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5;
  const int wm = (wave / S::kWN) * S::kFM * 32, wn = (wave % S::kWN) * S::kFN * 32;
  const int left = a.v - n0 - wn - 4 * half;      // this lane's columns (32 j + 8 q + r) below it exist
  [[maybe_unused]] const int room = a.ldp - n0 - wn - 4 * half;      // and those below it are stored (float)
  [[maybe_unused]] float bias[S::kFN][16];
  if constexpr (!kPlain) {
#pragma unroll
    for (int j = 0; j < S::kFN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int c = 32 * j + 8 * (r >> 2) + (r & 3), in = min(c, left - 1);       // past the last class: any
        const float b = a.bias ? TypeOf<T>::to_float(a.bias[max(n0 + wn + 4 * half + in, 0)]) : 0.0f;
        bias[j][r] = c < left ? b : -__builtin_inff();
      }
  }
#pragma unroll
  for (int i = 0; i < S::kFM; ++i) {
    const int row = m0 + wm + 32 * i + (lane & 31);
    const bool there = row < rows;
    f32x16 z[S::kFN];
#pragma unroll
    for (int j = 0; j < S::kFN; ++j) {
      z[j] = tile.acc[i][j];
      if constexpr (!kPlain)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[j][r] += bias[j][r];
    }
    const int c = there ? a.label[row] - (n0 + wn + 4 * half) : -1;
    // (kept as 16 bits, z becomes the distance below the group's largest in steps)
    {
      const bool mine = c >= 0 && c < S::kFN * 32 && (c & 7) < 4;
      if (__any(mine)) {
        float zy = 0.0f;
#pragma unroll
        for (int j = 0; j < S::kFN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) zy = c == 32 * j + 8 * (r >> 2) + (r & 3) ? z[j][r] : zy;
        if (mine) a.z_label[row] = zy;
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < S::kFN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[j][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float base = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < S::kFN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if constexpr (sizeof(T) == 4) {
            sum += exp_for<T>(z[j][r] - base);
          } else {
            const float below = z[j][r] - base;      // first: z and base may be the type's lowest
            sum += exp_for<T>(below);
            z[j][r] = below * (-kLog2e * Kept<T>::kSteps / 65535.0f);
          }
        }
      sum += __shfl_xor(sum, 32, 64);
      const int group = (n0 + wn) / (S::kFN * 32);
      if (there && half == 0) a.stats[group * a.ld_stats + row] = make_float2(top, sum);
    }
    if constexpr (kWhat == kKeep) {
      const int c0 = n0 + wn + 4 * half;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < S::kFN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (there && 32 * j + 8 * q < room)
              *(f32x4*)((float*)a.z + in_panels(row, c0 + 32 * j + 8 * q, a.chunk_rows)) =
                  f32x4{z[j][4 * q], z[j][4 * q + 1], z[j][4 * q + 2], z[j][4 * q + 3]};
      } else {
        // eight neighbouring columns a lane: the lower half of the wave takes the even groups of eight; two
        // stores fill a panel's 32 rows
#pragma unroll
        for (int j = 0; j < S::kFN; ++j)
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            unsigned long long half_group[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              unsigned w[2];
#pragma unroll
              for (int k = 0; k < 2; ++k)      // both times 65 535 to the nearest integer, 65 535 at most
                w[k] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16(z[j][4 * (q + g) + 2 * k],
                                                                                    z[j][4 * (q + g) + 2 * k + 1]));
              half_group[g] = (unsigned long long)w[1] << 32 | w[0];
            }
            const u32x4 eight = whole_group(half_group[0], half_group[1]);
            if (there && n0 + wn + 32 * j < a.ldp)
              *(u32x4*)((unsigned short*)a.z + in_panels(row, n0 + wn + 32 * j, a.chunk_rows) + 8 * q +
                        8 * half) = eight;
          }
      }
    }
    __builtin_amdgcn_sched_barrier(0);      // one fragment row's registers at a time
  }
}

template <typename T, typename S, What kWhat>
__global__ __launch_bounds__(S::kThreads, S::kBM == 256 ? 1 : 2) void logits_kernel(const LogitArgs<T> a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  RH_LDS char* lds = (RH_LDS char*)smem;
  const int rows = max(a.chunk.rows(a.n_valid), 0);
  const Grid g = {(rows + S::kBM - 1) / S::kBM, a.grid.n};      // tiles that hold rows
  const int tiles = g.m * g.n, splits = kWhat == kParted ? a.sharing.splits(rows) : 1;
  if ((int)blockIdx.x >= tiles * splits) return;
  const int id = xcd_run(blockIdx.x, tiles * splits), split = kWhat == kParted ? id / tiles : 0;
  const int2 at = tile_at(g, id - split * tiles);
  const int m0 = at.x * S::kBM, n0 = at.y * S::kBN;
  const int most = kWhat == kParted ? (a.steps + splits - 1) / splits : a.steps, k0 = split * most;
  const int steps = max(0, min(most, a.steps - k0));
  constexpr bool kPW = sizeof(T) == 4;
  const long long panel = (long long)a.chunk_rows * kStepBytes, from_x = k0 * panel + (long long)m0 * kStepBytes;
  const long long from = kPW ? k0 * a.ldw + n0 * (long long)kStepBytes : n0 * a.ldw + k0 * kStepBytes;
  Tile<T, kRows, kPanels, kRows, kPW, S> tile;
  tile.run(a.x + from_x, panel, a.x_bytes - from_x, a.x_part, a.w + from, a.ldw, a.w_bytes - from, a.w_part, steps, lds,
           kStepBytes, k0 + steps == a.steps ? a.w_limit : kStepBytes);
  if constexpr (kWhat == kParted) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / S::kWN) * S::kFM * 32, c0 = n0 + (wave % S::kWN) * S::kFN * 32 + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < S::kFM; ++i) {
      const int row = m0 + wm + 32 * i + (lane & 31);
      float* to = a.part + ((long long)split * g.m * S::kBM + row) * a.ldp + c0;
#pragma unroll
      for (int j = 0; j < S::kFN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (row < rows && c0 + 32 * j + 8 * q < a.ldp)
            *(f32x4*)(to + 32 * j + 8 * q) = f32x4{tile.acc[i][j][4 * q], tile.acc[i][j][4 * q + 1],
                                                   tile.acc[i][j][4 * q + 2], tile.acc[i][j][4 * q + 3]};
    }
    return;
  }
  if (!a.bias && n0 + S::kBN <= a.v)
    finish_logits<T, S, kWhat, true>(a, tile, m0, n0, rows);
  else
    finish_logits<T, S, kWhat, false>(a, tile, m0, n0, rows);
}

// The parts' sums, and what finish_logits makes of them, for groups of 64 classes: 16 lanes a row, four classes
// each.  Bound by the parts' bytes.
constexpr int kSumRows = 64;      // of a workgroup
constexpr int kSumGroup = 64;
template <typename T, bool kKeeps>
__global__ __launch_bounds__(kThreads) void sum_logits_kernel(const LogitArgs<T> a) {
  const int rows = max(a.chunk.rows(a.n_valid), 0), splits = a.sharing.splits(rows);
  const long long plane = (long long)a.sharing.tiles_m(rows) * a.sharing.bm * a.ldp;
  const int in = threadIdx.x & 15, c = blockIdx.x * kSumGroup + in * 4;
  f32x4 bias;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    bias[k] = c + k >= a.v ? -__builtin_inff() : a.bias ? TypeOf<T>::to_float(a.bias[c + k]) : 0.0f;
  const int lo = blockIdx.y * kSumRows, hi = min(rows, lo + kSumRows);
  for (int r0 = lo; r0 < hi; r0 += kThreads / 16) {
    const int r = min(r0 + ((int)threadIdx.x >> 4), hi - 1);      // the last row by several: the same values
    const float* from = a.part + (long long)r * a.ldp + c;
    f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
    int k = 0;
    for (; k + 4 <= splits; k += 4) {
      f32x4 p[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) p[u] = *(const f32x4*)(from + (k + u) * plane);
      z += (p[0] + p[1]) + (p[2] + p[3]);
    }
    for (; k < splits; ++k) z += *(const f32x4*)(from + k * plane);
    const int y = a.label[r] - c;
    float top = -__builtin_inff();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      // what stands behind the last class may be anything
      z[u] = c + u >= a.v ? -__builtin_inff() : z[u] + bias[u];
      top = fmaxf(top, z[u]);
      if (y == u) a.z_label[r] = z[u];
    }
    top = fmaxf(top, rotated<8>(top));
    top = fmaxf(top, rotated<4>(top));
    top = fmaxf(top, rotated<2>(top));
    top = fmaxf(top, rotated<1>(top));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) sum += exp_for<T>(z[u] - base);
    sum = sum16(sum);
    if (in == 0) a.stats[blockIdx.x * a.ld_stats + r] = make_float2(top, sum);
    if constexpr (kKeeps) {
      if constexpr (sizeof(T) == 4) {
        *(f32x4*)((float*)a.z + in_panels(r, c, a.chunk_rows)) = z;
      } else {
        constexpr float kCode = -kLog2e * Kept<T>::kSteps / 65535.0f;
        unsigned w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
          w[u] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pknorm_u16((z[2 * u] - base) * kCode,
                                                                              (z[2 * u + 1] - base) * kCode));
        *(unsigned long long*)((unsigned short*)a.z + in_panels(r, c, a.chunk_rows)) =
            (unsigned long long)w[1] << 32 | w[0];
      }
    }
  }
}

constexpr int kProbRows = 256;

// P from the kept logits, in their place (float: beside them, in parts):
//   p = e^(z - group's top) * (e^(group's top - row's top) / row's sum),  the first factor from the code.
// A workgroup takes a group of classes (kPanelsOf panels) of kProbRows places, a thread eight columns of each
// panel's row.  column_sums (or NULL): [row block][v] sums of P over its rows.  The first workgroup of the
// last chunk also adds up the loss (losses > 0).  Bound by memory: 3891 x 32 768 in 16 bits, 255 MB each way:
// 85 us.
template <typename T, int kPanelsOf>
__global__ __launch_bounds__(kThreads) void probs_kernel(const void* __restrict__ kept, char* __restrict__ p_out,
                                                         const long long part, const int chunk_rows, const int ldp,
                                                         const int v, const Chunk chunk,
                                                         const int* __restrict__ n_valid,
                                                         const int* __restrict__ label,
                                                         const float2* __restrict__ row_stats,
                                                         const float2* __restrict__ stats, const long long ld_stats,
                                                         float* __restrict__ column_sums,
                                                         const double* __restrict__ loss_parts, const int losses,
                                                         float* __restrict__ small) {
  constexpr int kWords = sizeof(T) == 4 ? 2 : 1;      // of 16 bytes that hold eight logits
  __shared__ float s_sum[4][kPanelsOf * kStepK];
  if (losses && blockIdx.x == 0 && blockIdx.y == 0) add_losses(loss_parts, losses, small);
  const int rows = chunk.rows(n_valid), lo = blockIdx.y * kProbRows, hi = min(rows, lo + kProbRows);
  const int t = threadIdx.x, first = blockIdx.x * kPanelsOf * kStepK, c = first + (t & 3) * 8;
  const float2* top = stats + (long long)blockIdx.x * ld_stats;
  float sums[kPanelsOf][8];
#pragma unroll
  for (int i = 0; i < kPanelsOf; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) sums[i][k] = 0.0f;
  for (int r = lo + (t >> 2); r < hi; r += kThreads / 4) {
    const long long at = in_panels(r, c, chunk_rows), next = (long long)chunk_rows * kStepK;
    u32x4 z[kPanelsOf][kWords];
#pragma unroll
    for (int i = 0; i < kPanelsOf; ++i)
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        if (first + i * kStepK < ldp) z[i][k] = ((const u32x4*)kept)[(at + i * next) / 8 * kWords + k];
    const float2 of_row = row_stats[r];
    const int y = label[r] - c;
    const float inv = 1.0f / of_row.y, f = sizeof(T) == 4 ? inv : exp_for<T>(top[r].x - of_row.x) * inv;
#pragma unroll
    for (int i = 0; i < kPanelsOf; ++i) {
      if (first + i * kStepK >= ldp) continue;
      float p[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (sizeof(T) == 4) {
          const unsigned w = z[i][k >> 2][k & 3];
          // the label's p - 1 as (e - sum) / sum, which does not cancel what p was rounded by
          p[k] = (exp_for<T>(__builtin_bit_cast(float, w) - of_row.x) - (y == i * kStepK + k ? of_row.y : 0.0f)) * f;
        } else {
          const unsigned w = z[i][0][k >> 1], code = k & 1 ? w >> 16 : w & 0xffffu;
          const float e = __builtin_amdgcn_exp2f((float)code * (-1.0f / Kept<T>::kSteps));
          p[k] = (code == 0xffffu ? 0.0f : e) * f;
          p[k] = y == i * kStepK + k ? p[k] - 1.0f : p[k];
        }
        sums[i][k] += p[k];
        p[k] *= PScale<T>::up;
      }
      const Eight<T> out = in_parts<T>(p);
#pragma unroll
      for (int k = 0; k < TypeOf<T>::kParts; ++k) *(u32x4*)(p_out + k * part + (at + i * next) * 2) = out.part[k];
    }
  }
  if (!column_sums) return;
#pragma unroll
  for (int i = 0; i < kPanelsOf; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float s = sums[i][k];
#pragma unroll
      for (int o = 4; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
      if ((t & 63) < 4) s_sum[t >> 6][i * kStepK + (t & 3) * 8 + k] = s;
    }
  __syncthreads();
  for (int i = t; i < kPanelsOf * kStepK && first + i < v; i += kThreads)
    column_sums[(long long)blockIdx.y * v + first + i] = (s_sum[0][i] + s_sum[1][i]) + (s_sum[2][i] + s_sum[3][i]);
}

// Row loss and (max, sum) of every place from the groups' pairs: 32 threads a row, each a 32nd of the groups.
// 9 us for 3891 rows of 256 pairs.
constexpr int kJoinRows = 8;      // of a workgroup
__global__ __launch_bounds__(kThreads) void join_stats_kernel(const float2* __restrict__ stats,
                                                              const long long ld, const int groups,
                                                              const Chunk chunk, const int* __restrict__ n_valid,
                                                              const int* __restrict__ map,
                                                              const float* __restrict__ z_label,
                                                              float2* __restrict__ row_stats,
                                                              float* __restrict__ row_loss,
                                                              double* __restrict__ partial) {
  constexpr int kParts = kThreads / kJoinRows;
  __shared__ float s_top[kParts][kJoinRows], s_sum[kParts][kJoinRows];
  const int rows = chunk.rows(n_valid), r = threadIdx.x % kJoinRows, part = threadIdx.x / kJoinRows;
  const int row = blockIdx.x * kJoinRows + r;
  float top = -__builtin_inff(), sum = 0.0f;
  if (row < rows) {
    for (int t0 = part; t0 < groups; t0 += 8 * kParts) {      // eight at a time, their loads together
      float2 p[8];
      float up = top;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        p[k] = t0 + kParts * k < groups ? stats[(t0 + kParts * k) * ld + row] : make_float2(-__builtin_inff(), 0.0f);
        up = fmaxf(up, p[k].x);
      }
      const float base = up == -__builtin_inff() ? 0.0f : up;
      sum *= expf(top - base);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += p[k].y * expf(p[k].x - base);
      top = up;
    }
  }
  s_top[part][r] = top;
  s_sum[part][r] = sum;
  __syncthreads();
  if (threadIdx.x < 64) {
    double loss = 0.0;
    if (part == 0 && row < rows) {
      top = -__builtin_inff();
      sum = 0.0f;
      for (int k = 0; k < kParts; ++k) top = fmaxf(top, s_top[k][r]);
      const float base = top == -__builtin_inff() ? 0.0f : top;
      for (int k = 0; k < kParts; ++k) sum += s_sum[k][r] * expf(s_top[k][r] - base);
      const float v = (top - z_label[row]) + logf(sum);
      row_stats[row] = make_float2(top, sum);
      row_loss[map[row]] = v;
      loss = (double)v;
    }
    loss = wave_sum(loss);
    if (threadIdx.x == 0) partial[blockIdx.x] = loss;
  }
}

__global__ __launch_bounds__(kThreads) void finish_loss_kernel(const double* __restrict__ parts, const int n,
                                                               float* __restrict__ small) {
  add_losses(parts, n, small);
}

// ---------------------------------------------------------------------------------------------
// Gradients
// ---------------------------------------------------------------------------------------------
template <typename T>
struct ProductArgs {
  const char* p;               // P in panels of chunk_rows
  long long p_bytes, p_part;
  int chunk_rows;
  const char* b;               // dX: the weights (rows, or panels, ldb bytes apart); dW: the features in panels
  long long ldb, b_bytes, b_part;
  int m, n, k;                 // rows that count bound m (dX) or k (dW) on the device
  const int* n_valid;
  Chunk chunk;
  Sharing sharing;
  const float* scale;
  float down;
  T* out;                      // [map[m] or m][ldo]
  const int* map;
  long long ldo;
  float* part;                 // [split][m][ldpart] instead of out
  long long ldpart;
  int add;                     // part += instead of part =
};

// float parts; the result, in rows of whole 16 bytes or not
enum To { kParts, kWhole, kSingly };

// kLA = kRows: dX = P W, the sum over the classes; kCols: dW = P^T X, over the chunk's rows.  Bound by the matrix
// units (busy 73 and 66 % of the cycles) and their clock where the sums are long (8192 x 4096, 131 072 classes: 1.26 and
// 1.18 PFLOP/s), by filling the card where the result is small; the splits that do so are cut()'s.  Workgroups that follow one another on an XCD
// take the same split's tiles, which read the same rows: dW of 601 x 256 over 49 104 rows 26 us, 37 with a
// split's tiles spread over the XCDs.
template <typename T, Layout kLA, typename S, To kTo>
__global__ __launch_bounds__(S::kThreads, S::kBM == 256 ? 1 : 2) void product_kernel(const ProductArgs<T> a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  RH_LDS char* lds = (RH_LDS char*)smem;
  if (kLA == kCols && *a.n_valid == kThere) return;
  const int rows = max(a.chunk.rows(a.n_valid), 0);
  const int m = kLA == kRows ? rows : a.m, k = kLA == kCols ? rows : a.k;
  const Grid g = {a.sharing.tiles_m(m), a.sharing.tiles_n};
  const int tiles = g.m * g.n, splits = a.sharing.splits(m), k_steps = (k + kStepK - 1) / kStepK;
  if ((int)blockIdx.x >= tiles * splits) return;
  const int id = xcd_run(blockIdx.x, tiles * splits), split = id / tiles;      // a split's tiles share its L2
  const int2 at = tile_at(g, id - split * tiles);
  const int m0 = at.x * S::kBM, n0 = at.y * S::kBN;
  const int split_steps = (k_steps + splits - 1) / splits;
  const int k0 = split * split_steps * kStepK;
  const int steps = max(0, min(split_steps, (k - k0 + kStepK - 1) / kStepK));
  const int last = k - k0 - (steps - 1) * kStepK;      // values of k in the last step
  const long long panel = (long long)a.chunk_rows * kStepBytes;
  const long long from = kLA == kRows ? k0 / kStepK * panel + (long long)m0 * kStepBytes
                                      : m0 / kStepK * panel + (long long)k0 * kStepBytes;
  constexpr bool kPB = kLA == kCols || sizeof(T) == 4;
  const long long from_b = kPB ? n0 / kStepK * a.ldb + (long long)k0 * kStepBytes : k0 * a.ldb + n0 * (int)sizeof(T);
  Tile<T, kLA, kPanels, kCols, kPB, S> tile;
  tile.run(a.p + from, panel, a.p_bytes - from, a.p_part, a.b + from_b, a.ldb, a.b_bytes - from_b, a.b_part, steps, lds, last,
           last);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave / S::kWN) * S::kFM * 32, wn = (wave % S::kWN) * S::kFN * 32 + 4 * (lane >> 5);
  const float s = *a.scale * a.down;
  const int room = a.n - n0 - wn;      // this lane's columns (32 j + 8 q + r) below it exist
#pragma unroll
  for (int i = 0; i < S::kFM; ++i) {
    const int row = m0 + wm + 32 * i + (lane & 31);
    if (row < m) {
      if constexpr (kTo == kParts) {      // ldpart is a multiple of four, 16-byte aligned
        float* part = a.part + ((long long)split * g.m * S::kBM + row) * a.ldpart + n0 + wn;
#pragma unroll
        for (int j = 0; j < S::kFN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (32 * j + 8 * q < room) {
              f32x4 v = {tile.acc[i][j][4 * q], tile.acc[i][j][4 * q + 1], tile.acc[i][j][4 * q + 2],
                         tile.acc[i][j][4 * q + 3]};
              if (a.add) v += *(const f32x4*)(part + 32 * j + 8 * q);
              *(f32x4*)(part + 32 * j + 8 * q) = v;
            }
      } else {
        T* out = a.out + (a.map ? a.map[row] : row) * a.ldo + n0 + wn;
        // 16 bytes a store, eight neighbouring columns of a 16-bit type or four of float; kSingly: of rows of any
        // alignment, and the last of a row one by one
        auto store = [&](T* to, const int left, const auto v) {
          constexpr int kV = 16 / (int)sizeof(T);
          if (kTo == kWhole) {
            if (left > 0) *(u32x4*)to = __builtin_bit_cast(u32x4, v);
          } else if (left >= kV) {
            __builtin_memcpy(to, &v, 16);
          } else {
            T single[kV];
            __builtin_memcpy(single, &v, 16);
#pragma unroll
            for (int r = 0; r < kV; ++r)
              if (r < left) to[r] = single[r];
          }
        };
        [[maybe_unused]] unsigned long long half_group[2];
#pragma unroll
        for (int j = 0; j < S::kFN; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            Vec4<T> v;
#pragma unroll
            for (int r = 0; r < 4; ++r) v.v[r] = TypeOf<T>::from_float(tile.acc[i][j][4 * q + r] * s);
            if constexpr (sizeof(T) == 4) {
              store(out + 32 * j + 8 * q, room - 32 * j - 8 * q, v);
            } else {
              half_group[q & 1] = __builtin_bit_cast(unsigned long long, v);
              if (q & 1) {
                const int c = 32 * j + 8 * (q - 1) + 4 * (lane >> 5);      // from this lane's first column
                store(out + c, room - c, whole_group(half_group[0], half_group[1]));
              }
            }
          }
      }
    }
  }
}

// What is left of a call beside dW: db from the row blocks' column sums (parts [parts][v]), eight columns a workgroup
// and 32 threads a column, and where losses > 0 the call's loss, by the first workgroup.
template <typename T>
struct Rest {
  const float* columns;
  int parts, v;
  const int* n_valid;
  const float* scale;
  T* db;
  const double* loss_parts;
  int losses;
  float* small;
  __device__ __forceinline__ void join(const int block) const {
    if (*n_valid == kThere) return;
    __shared__ float s_sum[32][8];
    if (losses && block == 0) add_losses(loss_parts, losses, small);
    const int in = threadIdx.x & 7, slice = threadIdx.x >> 3, c = block * 8 + in;
    float sum = 0.0f;
    if (c < v)
#pragma unroll 8
      for (int k = slice; k < parts; k += 32) sum += columns[(long long)k * v + c];
    s_sum[slice][in] = sum;
    __syncthreads();
    if (slice == 0 && c < v) {
      for (int k = 1; k < 32; ++k) sum += s_sum[k][in];
      db[c] = TypeOf<T>::from_float(sum * *scale);
    }
  }
  int workgroups() const { return db ? (v + 7) / 8 : 0; }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void join_rest_kernel(const Rest<T> rest) {
  rest.join(blockIdx.x);
}

// out[map[m] or m][:] = scale * sum of the splits' parts, in their order.  The workgroups from `of_rest` on do that.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_parts_kernel(const float* __restrict__ part, const Sharing sharing,
                                                              const long long ldpart, const int m, const int n,
                                                              const Chunk chunk, const int* __restrict__ n_valid,
                                                              const int by_rows,
                                                              const float* __restrict__ scale, const float down,
                                                              const int* __restrict__ map, T* __restrict__ out,
                                                              const long long ldo, const Rest<T> rest,
                                                              const int of_rest) {
  if ((int)blockIdx.x >= of_rest) {
    rest.join(blockIdx.x - of_rest);
    return;
  }
  if (*n_valid == kThere) return;
  const int rows = by_rows ? max(chunk.rows(n_valid), 0) : m, splits = sharing.splits(rows);
  const long long quads = (n + 3) / 4, top = rows * quads;
  const long long plane = (long long)sharing.tiles_m(rows) * sharing.bm * ldpart;
  const float s = *scale * down;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < top; i += (long long)of_rest * kThreads) {
    const long long r = i / quads;
    const int c = (int)(i - r * quads) * 4;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* from = part + r * ldpart + c;
    int k = 0;
    for (; k + 8 <= splits; k += 8) {      // eight loads on their way together
      f32x4 p[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) p[u] = *(const f32x4*)(from + (k + u) * plane);
#pragma unroll
      for (int u = 0; u < 8; ++u) v += p[u];
    }
    for (; k + 2 <= splits; k += 2) {
      const f32x4 p = *(const f32x4*)(from + k * plane), q = *(const f32x4*)(from + (k + 1) * plane);
      v = (v + p) + q;
    }
    if (k < splits) v += *(const f32x4*)(from + k * plane);
    T* to = out + (map ? map[r] : r) * ldo + c;
    if ((n & 3) == 0) {
      Vec4<T> o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o.v[j] = TypeOf<T>::from_float(v[j] * s);
      *(Vec4<T>*)to = o;
    } else {
      for (int j = 0; j < 4 && c + j < n; ++j) to[j] = TypeOf<T>::from_float(v[j] * s);
    }
  }
}

// x *= scale / assumed in place, one rounding; an array whose scale is the assumed one is not touched.  Bound by
// memory: 268 MB of bfloat16 97 us (5.5 TB/s over both ways), of float32 75.
template <typename T>
__global__ __launch_bounds__(kThreads) void upstream_kernel(T* __restrict__ x, const long long n,
                                                            const float* __restrict__ scale, const float assumed) {
  const float s = *scale;
  if (s == assumed) return;
  const float f = s / assumed;
  for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads)
    x[i] = TypeOf<T>::from_float(TypeOf<T>::to_float(x[i]) * f);
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------
typedef Shape<2, 2, 4, 4> Large;      // 256 x 256, 4 waves
typedef Shape<2, 2, 2, 2> Small;      // 128 x 128, 4 waves

constexpr long long kKeptBytes = 2ll << 30;      // of logits at a time, or 256 rows of them
constexpr int kMostChunk = 1 << 22;              // rows; eight panels' offsets stay below 2^31

// How a product is cut up: the tiles' shape, and into how many sums along k its sum is split.
struct Cut {
  bool large;
  int splits, steps;      // k steps of a split
};

// The cut of the least estimated time.  The card takes 256 tiles of 256 x 256 at a time or 512 of 128 x 128;
// a step takes the longer the more of it is at work (the clock sinks, the tiles share the caches): 0.58 to
// 0.88 us in a large tile, 0.26 to 0.56 in a small one.  A tile's start and end take 14 and 6 us, joining
// the splits 4 us and their bytes' way at 4.5 TB/s.  Of 8192 x 8192 logits over 256 features, the first of
// each pair is the small tiles' time: 80 / 94 us; over 1024: 194 / 182.  49 104 x 601 over 256: 40 / 67.
// dX of 2048 x 1024 over 16 384 classes, float: 893 us unsplit, 499 of four splits, large and eight of
// them 380.  200 x 512 over 10 000, bfloat16: 83 unsplit, 18 of sixteen, large 29 at best.
static Cut cut(long long m, long long n, int steps, int terms, int most_splits, float large_end = 14.0f) {
  Cut best = {};
  float least = 0.0f;
  for (int large = 0; large < 2; ++large) {
    const int side = large ? 256 : 128, slots = large ? 256 : 512;
    const long long tiles = (long long)ceil_div(m, side) * ceil_div(n, side);
    for (int splits = 1; splits <= most_splits && (splits == 1 || steps / splits >= 4); ++splits) {
      const Cut c = {large != 0, splits, ceil_div(steps, splits)};
      if (ceil_div(steps, c.steps) < splits) continue;      // the last would be empty
      const long long work = tiles * splits;
      const float filled = work < slots ? (float)work / slots : 1.0f;
      const float end = !large ? 6.0f : splits > 1 ? 14.0f : large_end;
      float us = (float)((work + slots - 1) / slots) *
                 (((large ? 0.58f : 0.26f) + 0.30f * filled) * (float)c.steps * (float)terms + end);
      if (splits > 1) us += 4.0f + (float)splits * (float)m * (float)n * (4.0f / 4.5e6f);
      if (least == 0.0f || us < least) {
        least = us;
        best = c;
      }
    }
  }
  return best;
}

// The call's rows are taken in chunks whose logits take kKeptBytes at most: they are made once (6 n d v
// operations in all), P takes their place, and the chunk's part of the weight's gradient is added to the
// others' in float32 where there are several.
struct Plan {
  int size, parts;              // bytes of a value; numbers that it is taken apart into
  int kept_size;                // bytes of a kept logit
  int per, row_blocks;          // rows a placing block takes
  int panels;                   // of the features
  int ldw_pad;                  // row of the copied weights (0: not copied)
  int chunk, chunks;            // rows at a time
  int ldp;                      // columns of P
  bool whole;                   // a workgroup holds rows of logits whole
  Cut logits;
  int group, groups;            // classes that share a maximum: a wave's of a tile, or kSumGroup
  Cut dx, dw;
  long long ldpart;
};

static Plan make_plan(int n, int d, int v, int dtype, int flags) {
  Plan p = {};
  p.size = dtype == RH_F32 ? 4 : 2;
  p.parts = dtype == RH_F32 ? 3 : 1;
  p.kept_size = dtype == RH_F32 ? 4 : 2;
  p.per = n > 65536 ? 256 : 32;
  p.row_blocks = ceil_div(n, p.per);
  p.panels = ceil_div(d, kStepK);
  p.whole = dtype != RH_F32 && (flags & (RH_CE_GRAD_X | RH_CE_GRAD_W | RH_CE_GRAD_B)) && whole_pays(d, v);
  p.ldw_pad = dtype != RH_F32 && (flags & RH_CE_COPY_WEIGHT) ? p.panels * kStepK : 0;
  p.ldp = ceil_div(v, 64) * 64;
  long long rows = kKeptBytes / ((long long)p.ldp * p.kept_size) / 256 * 256;
  if (rows < 256) rows = 256;
  if (rows > kMostChunk) rows = kMostChunk;
  p.chunk = n;
  p.chunks = 1;
  if (n > rows) {
    p.chunks = ceil_div(n, rows);
    p.chunk = ceil_div(ceil_div(n, p.chunks), 256) * 256;      // of even size
    p.chunks = ceil_div(n, p.chunk);
  }
  const int terms = dtype == RH_F32 ? TypeOf<float>::kTerms : 1;
  // float's logits: more registers than there are at the end of a large tile
  p.logits = cut(p.chunk, v, p.panels, terms, p.whole ? 1 : 64, dtype == RH_F32 ? 30.0f : 14.0f);
  if (p.logits.splits > 1) {
    p.group = kSumGroup;
    p.groups = p.ldp / kSumGroup;
  } else {
    p.group = p.logits.large ? Large::kFN * 32 : Small::kFN * 32;
    p.groups = ceil_div(v, p.logits.large ? Large::kBN : Small::kBN) * (p.logits.large ? Large::kWN : Small::kWN);
  }
  p.dx = cut(p.chunk, d, p.ldp / kStepK, terms, 64);
  p.dw = cut(v, d, ceil_div(p.chunk, kStepK), terms, 64);
  p.ldpart = ceil_div(d, 4) * 4;
  return p;
}

struct Space {
  int2* blocks;
  RowInfo info;
  char* x;
  long long x_part;      // bytes of each of the features' parts, ...
  char* w;
  long long w_part;
  float2* stats;
  float* z_label;
  float2* row_stats;
  double* loss;
  float* z_part;
  char* z;
  char* p;               // z's place for the 16-bit types
  long long p_part;
  float* dx_part;
  float* dw_part;
  float* db_part;
  int db_parts;       // of a column's sum, of all chunks
  size_t bytes;
};

static long long whole_tiles(const Cut& c, int rows) {
  const int side = c.large ? 256 : 128;
  return (long long)ceil_div(rows, side) * side;
}

static Space carve(void* base, const Plan& p, int n, int d, int v, int flags) {
  Carver c(base);
  Space s = {};
  s.blocks = c.take<int2>(p.row_blocks);
  s.info.map = c.take<int>(n);
  s.info.label = c.take<int>(n);
  s.info.n_valid = c.take<int>(1);
  s.info.scale = c.take<float>(1);
  s.x_part = (long long)p.chunks * p.chunk * p.panels * kStepBytes;
  s.x = c.take<char>((size_t)s.x_part * p.parts);
  if (p.ldw_pad) s.w = c.take<char>((size_t)v * p.ldw_pad * p.size);
  if (p.parts > 1) {
    s.w_part = (long long)v * p.panels * kStepBytes;
    s.w = c.take<char>((size_t)s.w_part * p.parts);
  }
  if (!p.whole) {
    s.stats = c.take<float2>((size_t)p.groups * p.chunk);
    s.z_label = c.take<float>(n);
    if (p.logits.splits > 1)
      s.z_part = c.take<float>((size_t)p.logits.splits * whole_tiles(p.logits, p.chunk) * p.ldp);
    s.row_stats = c.take<float2>(n);
  }
  s.loss = c.take<double>(ceil_div(n, kJoinRows));
  if (flags & (RH_CE_GRAD_X | RH_CE_GRAD_W | RH_CE_GRAD_B)) {
    s.z = c.take<char>((size_t)p.chunk * p.ldp * p.kept_size);      // whole rows: P alone
    s.p_part = (long long)p.chunk * p.ldp * 2;
    s.p = p.parts > 1 ? c.take<char>((size_t)s.p_part * p.parts) : s.z;
  }
  if ((flags & RH_CE_GRAD_X) && !p.whole && p.dx.splits > 1)
    s.dx_part = c.take<float>((size_t)p.dx.splits * whole_tiles(p.dx, p.chunk) * p.ldpart);
  if ((flags & RH_CE_GRAD_W) && (p.chunks > 1 || p.dw.splits > 1))
    s.dw_part = c.take<float>((size_t)p.dw.splits * whole_tiles(p.dw, v) * p.ldpart);
  if (flags & RH_CE_GRAD_B) {
    // as many as are written: whole rows' launches have a workgroup for every kWholeRows rows there are (a chunk before
    // the last is a multiple of them), the others' for every kProbRows of every chunk
    s.db_parts = p.whole ? ceil_div(n, kWholeRows) : ceil_div(p.chunk, kProbRows) * p.chunks;
    s.db_part = c.take<float>((size_t)s.db_parts * v);
  }
  s.bytes = c.off;
  return s;
}

template <typename K>
static int raise_lds(K kernel, int bytes) {
  RH_CHECK_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return RH_OK;
}

template <typename T, typename S, What kWhat>
static int launch_logits(LogitArgs<T> a, hipStream_t stream) {
  a.grid = Grid{ceil_div(a.chunk.most, S::kBM), ceil_div(a.v, S::kBN)};
  auto kernel = logits_kernel<T, S, kWhat>;
  if (int rc = raise_lds(kernel, S::kLdsBytes)) return rc;
  const unsigned workgroups = kWhat == kParted ? a.sharing.workgroups : a.grid.m * a.grid.n;
  hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(S::kThreads), S::kLdsBytes, stream, a);
  RH_CHECK_LAUNCH("logits_kernel");
  return RH_OK;
}

template <typename T, What kWhat>
static int launch_logits(const LogitArgs<T>& a, bool large, hipStream_t stream) {
  return large ? launch_logits<T, Large, kWhat>(a, stream) : launch_logits<T, Small, kWhat>(a, stream);
}

// A chunk's logits, in parts where the plan says so.
template <typename T>
static int make_logits(const Plan& p, const LogitArgs<T>& a, bool keep, hipStream_t stream) {
  if (p.logits.splits == 1)
    return keep ? launch_logits<T, kKeep>(a, p.logits.large, stream) : launch_logits<T, kStats>(a, p.logits.large, stream);
  if (int rc = launch_logits<T, kParted>(a, p.logits.large, stream)) return rc;
  const dim3 grid(p.groups, ceil_div(a.chunk.most, kSumRows));
  if (keep) hipLaunchKernelGGL((sum_logits_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((sum_logits_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
  RH_CHECK_LAUNCH("sum_logits_kernel");
  return RH_OK;
}

template <typename T, Layout kLA, typename S>
static int launch_product(const ProductArgs<T>& a, hipStream_t stream) {
  auto kernel = a.part                            ? product_kernel<T, kLA, S, kParts>
                : a.n * (int)sizeof(T) % 16 == 0 ? product_kernel<T, kLA, S, kWhole>
                                                 : product_kernel<T, kLA, S, kSingly>;
  if (int rc = raise_lds(kernel, S::kLdsBytes)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.sharing.workgroups), dim3(S::kThreads), S::kLdsBytes, stream, a);
  RH_CHECK_LAUNCH("product_kernel");
  return RH_OK;
}

template <typename T, int kPanelsOf>
static int launch_probs(const rh_linear_ce_args& q, const Plan& p, const Space& s, const LogitArgs<T>& a, int chunk,
                        hipStream_t stream) {
  const int blocks = ceil_div(p.chunk, kProbRows);
  hipLaunchKernelGGL((probs_kernel<T, kPanelsOf>), dim3(ceil_div(p.ldp, p.group), blocks), dim3(kThreads), 0, stream, s.z,
                     s.p, s.p_part, p.chunk, p.ldp, a.v, a.chunk, a.n_valid, a.label, s.row_stats + a.chunk.first, s.stats,
                     a.ld_stats,
                     s.db_part ? s.db_part + (long long)chunk * blocks * a.v : nullptr, s.loss,
                     chunk == p.chunks - 1 ? ceil_div(q.n, kJoinRows) : 0, q.small);
  RH_CHECK_LAUNCH("probs_kernel");
  return RH_OK;
}

template <typename T>
static int join_parts(const ProductArgs<T>& g, bool by_rows, const Rest<T>& rest, hipStream_t stream) {
  long long blocks = ((long long)g.m * ((g.n + 3) / 4) + kThreads - 1) / kThreads;
  if (blocks > 256 * 8) blocks = 256 * 8;
  hipLaunchKernelGGL(join_parts_kernel<T>, dim3((unsigned)blocks + rest.workgroups()), dim3(kThreads), 0, stream, g.part,
                     g.sharing, g.ldpart, g.m, g.n, g.chunk, g.n_valid, (int)by_rows, g.scale, g.down, g.map, g.out,
                     g.ldo, rest, (int)blocks);
  RH_CHECK_LAUNCH("join_parts_kernel");
  return RH_OK;
}

static Sharing share(const Cut& c, int m, int n, int most) {
  const int side = c.large ? 256 : 128, across = ceil_div(n, side);
  return Sharing{side, across, ceil_div(m, side) * across * c.splits, c.splits, most < c.splits ? c.splits : most};
}

// What the two products share.
template <typename T>
static ProductArgs<T> product_args(const rh_linear_ce_args& q, const Plan& p, const Space& s, const LogitArgs<T>& a) {
  ProductArgs<T> g = {};
  g.p = s.p;
  g.p_bytes = s.p_part;
  g.p_part = s.p_part;
  g.chunk_rows = p.chunk;
  g.n = q.d;
  g.n_valid = a.n_valid;
  g.chunk = a.chunk;
  g.scale = s.info.scale;
  g.down = PScale<T>::down;
  g.ldo = q.d;
  g.ldpart = p.ldpart;
  return g;
}

// dX of a chunk.
template <typename T>
static int features_gradient(const rh_linear_ce_args& q, const Plan& p, const Space& s, const LogitArgs<T>& a,
                             hipStream_t stream) {
  ProductArgs<T> g = product_args(q, p, s, a);
  g.b = a.w;
  g.ldb = a.ldw;
  g.b_bytes = a.w_bytes;
  g.b_part = a.w_part;
  g.m = a.chunk.most;
  g.k = a.v;
  // as many splits as four steps of k each leave, should fewer rows count
  g.sharing = share(p.dx, p.chunk, q.d, s.dx_part ? p.ldp / kStepK / 4 : 1);
  g.out = (T*)q.dx;
  g.map = s.info.map + a.chunk.first;
  g.part = s.dx_part;
  if (int rc = p.dx.large ? launch_product<T, kRows, Large>(g, stream)
                          : launch_product<T, kRows, Small>(g, stream))
    return rc;
  return s.dx_part ? join_parts(g, true, Rest<T>{}, stream) : RH_OK;
}

// dW, or a chunk's part of it; with the last part the rest, of which nothing is left then.
template <typename T>
static int weight_gradient(const rh_linear_ce_args& q, const Plan& p, const Space& s, const LogitArgs<T>& a,
                           int chunk, Rest<T>& rest, hipStream_t stream) {
  ProductArgs<T> g = product_args(q, p, s, a);
  g.b = a.x;
  g.ldb = (long long)p.chunk * kStepBytes;
  g.b_bytes = a.x_bytes;
  g.b_part = a.x_part;
  g.m = a.v;
  g.k = a.chunk.most;
  g.sharing = share(p.dw, a.v, q.d, p.dw.splits);
  g.out = (T*)q.dw;
  g.part = s.dw_part;
  g.add = chunk > 0;
  if (int rc = p.dw.large ? launch_product<T, kCols, Large>(g, stream)
                          : launch_product<T, kCols, Small>(g, stream))
    return rc;
  if (!s.dw_part || chunk < p.chunks - 1) return RH_OK;
  const Rest<T> now = rest;
  rest = Rest<T>{};
  return join_parts(g, false, now, stream);
}

// A chunk's loss, P, column sums and dX by workgroups that hold their rows' logits whole.
template <typename T>
static int whole_rows(const rh_linear_ce_args& q, const Plan& p, const Space& s, const LogitArgs<T>& a, int chunk,
                      hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    WholeArgs<T> g = {};
    g.x = a.x;
    g.x_bytes = a.x_bytes;
    g.chunk_rows = p.chunk;
    g.w = a.w;
    g.ldw = a.ldw;
    g.w_bytes = a.w_bytes;
    g.steps = a.steps;
    g.w_limit = a.w_limit;
    g.bias = a.bias;
    g.v = a.v;
    g.d = q.d;
    g.chunk = a.chunk;
    g.n_valid = a.n_valid;
    g.label = a.label;
    g.map = s.info.map + a.chunk.first;
    g.scale = s.info.scale;
    g.p = s.p;
    g.ldp = p.ldp;
    g.column_sums = s.db_part ? s.db_part + (long long)chunk * ceil_div(p.chunk, kWholeRows) * a.v : nullptr;
    g.dx = (T*)q.dx;
    g.row_loss = q.row_loss;
    g.loss = s.loss + a.chunk.first / kWholeRows;
    return run_whole<T>(g, stream);
  }
  return RH_EINVAL;      // no plan leads here
}

template <typename T>
static int run(const rh_linear_ce_args& q, const Plan& p, const Space& s, hipStream_t stream) {
  const int n = (int)q.n, d = q.d, v = (int)q.v;
  const Labels labels{q.labels, q.labels_int64, q.ignore_index, v};
  // up to 2048 rows counting them takes less than the launch (5 us)
  const bool counted = n > 2048;
  if (counted) {
    hipLaunchKernelGGL(count_rows_kernel, dim3(p.row_blocks), dim3(64), 0, stream, labels, n, p.per, s.blocks);
    RH_CHECK_LAUNCH("count_rows_kernel");
  }
  // a panel a wave where there are few rows
  int side = ceil_div(p.panels, 16) < 8 ? ceil_div(p.panels, 16) : 8;
  if (side < 256 / p.row_blocks) side = 256 / p.row_blocks;
  if (side > ceil_div(p.panels, 4)) side = ceil_div(p.panels, 4);
  hipLaunchKernelGGL(place_rows_kernel<T>, dim3(p.row_blocks, side), dim3(kThreads), 0, stream, (const T*)q.x,
                     (long long)q.ldx, d, labels, n, p.per, counted ? s.blocks : nullptr, s.x, s.x_part, p.panels,
                     p.chunk, s.info, q.row_loss, (T*)q.dx, q.small, (int*)(q.small + 3), q.divisor, q.reduction == RH_CE_MEAN, Upstream{q.upstream, q.grad});
  RH_CHECK_LAUNCH("place_rows_kernel");
  const bool grads = q.dx || q.dw || q.db;
  LogitArgs<T> a = {};
  a.chunk_rows = p.chunk;
  a.x_bytes = (long long)p.chunk * p.panels * kStepBytes;
  a.x_part = s.x_part;
  a.w = (const char*)q.w;
  a.ldw = q.ldw * p.size;
  a.w_bytes = (v - 1) * a.ldw + (long long)d * p.size;
  a.steps = p.panels;
  a.w_limit = d * 2 - (a.steps - 1) * kStepBytes;
  if (p.ldw_pad) {
    hipLaunchKernelGGL(pad_rows_kernel<T>, dim3(v < 8192 ? ceil_div(v, 4) : 2048), dim3(kThreads), 0, stream, (const T*)q.w,
                       (long long)q.ldw, d, v, (T*)s.w, p.ldw_pad, s.info.n_valid);
    RH_CHECK_LAUNCH("pad_rows_kernel");
    a.w = s.w;
    a.ldw = (long long)p.ldw_pad * p.size;
    a.w_bytes = v * a.ldw;
    a.w_limit = kStepBytes;
  }
  if (p.parts > 1) {
    const int across = ceil_div(p.panels, 16) < 16 ? ceil_div(p.panels, 16) : 16;
    hipLaunchKernelGGL(take_apart_kernel<T>, dim3(ceil_div(v, 16), across), dim3(kThreads), 0, stream, (const T*)q.w,
                       (long long)q.ldw, d, v, p.panels, s.w, s.w_part);
    RH_CHECK_LAUNCH("take_apart_kernel");
    a.w = s.w;
    a.ldw = (long long)v * kStepBytes;
    a.w_bytes = s.w_part;
    a.w_part = s.w_part;
    a.w_limit = kStepBytes;
  }
  a.bias = (const T*)q.bias;
  a.v = v;
  a.n_valid = s.info.n_valid;
  a.stats = s.stats;
  a.ld_stats = p.chunk;
  a.z = s.z;
  a.ldp = p.ldp;
  a.sharing = share(p.logits, p.chunk, v, p.logits.splits > 1 ? p.panels / 4 : 1);
  a.part = s.z_part;
  Rest<T> rest = {};
  if (q.db)
    rest = Rest<T>{s.db_part, s.db_parts, v, s.info.n_valid, s.info.scale, (T*)q.db, s.loss, p.whole ? ceil_div(n, kWholeRows) : 0,
                   q.small};
  for (int c = 0; c < p.chunks; ++c) {
    a.chunk = Chunk{c * p.chunk, n - c * p.chunk < p.chunk ? n - c * p.chunk : p.chunk};
    const int first = a.chunk.first;
    a.x = s.x + (long long)first * p.panels * kStepBytes;
    a.label = s.info.label + first;
    if (p.whole) {
      if (int rc = whole_rows(q, p, s, a, c, stream)) return rc;
      if (q.dw)
        if (int rc = weight_gradient(q, p, s, a, c, rest, stream)) return rc;
      continue;
    }
    a.z_label = s.z_label + first;
    if (int rc = make_logits(p, a, grads, stream)) return rc;
    hipLaunchKernelGGL(join_stats_kernel, dim3(ceil_div(a.chunk.most, kJoinRows)), dim3(kThreads), 0, stream, s.stats, a.ld_stats,
                       p.groups, a.chunk, s.info.n_valid, s.info.map + first, a.z_label, s.row_stats + first, q.row_loss,
                       s.loss + first / kJoinRows);
    RH_CHECK_LAUNCH("join_stats_kernel");
    if (!grads) continue;
    if (int rc = p.group == 128 ? launch_probs<T, 128 / kStepK>(q, p, s, a, c, stream)
                                : launch_probs<T, 64 / kStepK>(q, p, s, a, c, stream))
      return rc;
    if (q.dx)
      if (int rc = features_gradient(q, p, s, a, stream)) return rc;
    if (q.dw)
      if (int rc = weight_gradient(q, p, s, a, c, rest, stream)) return rc;
  }
  if (!grads || (p.whole && !q.db)) {
    hipLaunchKernelGGL(finish_loss_kernel, dim3(1), dim3(kThreads), 0, stream, s.loss,
                       ceil_div(n, p.whole ? kWholeRows : kJoinRows), q.small);
    RH_CHECK_LAUNCH("finish_loss_kernel");
  }
  if (rest.db) {
    hipLaunchKernelGGL(join_rest_kernel<T>, dim3(rest.workgroups()), dim3(kThreads), 0, stream, rest);
    RH_CHECK_LAUNCH("join_rest_kernel");
  }
  return RH_OK;
}

static int check_sizes(int64_t n, int32_t d, int64_t v, int32_t dtype) {
  RH_REQUIRE(dtype == RH_F32 || dtype == RH_BF16 || dtype == RH_F16, RH_EINVAL, "unknown element type %d", dtype);
  RH_REQUIRE(n >= 1 && n <= (1 << 26), RH_ESHAPE, "rows must be in 1 .. 2^26 (got %lld)", (long long)n);
  RH_REQUIRE(d >= 1 && d <= (1 << 17), RH_ESHAPE, "features must be in 1 .. 2^17 (got %d)", d);
  RH_REQUIRE(v >= 1 && v <= (1 << 21), RH_ESHAPE, "classes must be in 1 .. 2^21 (got %lld)", (long long)v);
  return RH_OK;
}

}  // namespace ce
}  // namespace rh

extern "C" {

size_t rh_linear_ce_workspace_bytes(int64_t n, int32_t d, int64_t v, int32_t dtype, int32_t flags) {
  if (rh::ce::check_sizes(n, d, v, dtype) != RH_OK) return 0;
  if (n <= rh::ce::kFewRows) return rh::ce::few_workspace_bytes((int)n, d, (int)v, dtype, flags);
  const rh::ce::Plan p = rh::ce::make_plan((int)n, d, (int)v, dtype, flags);
  return rh::ce::carve(nullptr, p, (int)n, d, (int)v, flags).bytes;
}

int rh_linear_ce(const rh_linear_ce_args* args, rh_stream_t stream) {
  RH_REQUIRE(args, RH_EINVAL, "null arguments");
  const rh_linear_ce_args& q = *args;
  if (int rc = rh::ce::check_sizes(q.n, q.d, q.v, q.dtype)) return rc;
  RH_REQUIRE(q.x && q.w && q.labels && q.row_loss && q.small, RH_EINVAL, "null pointer");
  RH_REQUIRE(q.reduction == RH_CE_MEAN || q.reduction == RH_CE_SUM, RH_EINVAL, "unknown reduction %d", q.reduction);
  RH_REQUIRE(q.ldx >= q.d && q.ldw >= q.d, RH_ESHAPE, "row stride smaller than the row");
  RH_REQUIRE(!q.db || q.bias, RH_EINVAL, "a gradient of the bias needs a bias");
  const int size = q.dtype == RH_F32 ? 4 : 2;
  int flags = q.flags & RH_CE_COPY_WEIGHT;
  if (q.dx) flags |= RH_CE_GRAD_X;
  if (q.dw) flags |= RH_CE_GRAD_W;
  if (q.db) flags |= RH_CE_GRAD_B;
  RH_REQUIRE((flags & RH_CE_COPY_WEIGHT) ||
                 (rh::aligned16(q.w) && q.d * size % 16 == 0 && q.ldw * size % 16 == 0 && q.ldw < (1 << 20)),
             RH_EALIGN, "weights whose rows are not whole 16-byte pieces need RH_CE_COPY_WEIGHT");
  RH_REQUIRE(((uintptr_t)q.dx | (uintptr_t)q.dw) % 16 == 0, RH_EALIGN, "gradients must be 16-byte aligned");
  if (q.n <= rh::ce::kFewRows) {
    const size_t need = rh::ce::few_workspace_bytes((int)q.n, q.d, (int)q.v, q.dtype, flags);
    RH_REQUIRE(q.workspace && q.workspace_bytes >= need, RH_EWORKSPACE, "workspace of %zu bytes, %zu needed",
               q.workspace_bytes, need);
    RH_REQUIRE((uintptr_t)q.workspace % 256 == 0, RH_EALIGN, "workspace must be 256-byte aligned");
    return rh::ce::run_few(q, flags, (hipStream_t)stream);
  }
  const rh::ce::Plan p = rh::ce::make_plan((int)q.n, q.d, (int)q.v, q.dtype, flags);
  const rh::ce::Space s = rh::ce::carve(q.workspace, p, (int)q.n, q.d, (int)q.v, flags);
  RH_REQUIRE(q.workspace && q.workspace_bytes >= s.bytes, RH_EWORKSPACE, "workspace of %zu bytes, %zu needed",
             q.workspace_bytes, s.bytes);
  RH_REQUIRE((uintptr_t)q.workspace % 256 == 0, RH_EALIGN, "workspace must be 256-byte aligned");
  if (q.dtype == RH_F32) return rh::ce::run<float>(q, p, s, (hipStream_t)stream);
  if (q.dtype == RH_BF16) return rh::ce::run<__bf16>(q, p, s, (hipStream_t)stream);
  return rh::ce::run<_Float16>(q, p, s, (hipStream_t)stream);
}

int rh_scale_gradient(void* x, int64_t count, int32_t dtype, const float* scale, float assumed, rh_stream_t stream) {
  RH_REQUIRE(count >= 0, RH_ESHAPE, "negative count");
  RH_REQUIRE(assumed != 0.0f, RH_EINVAL, "assumed scale must be non-zero");
  if (count == 0) return RH_OK;
  RH_REQUIRE(x && scale, RH_EINVAL, "null pointer");
  long long blocks = (count + rh::ce::kThreads - 1) / rh::ce::kThreads;
  if (blocks > 256 * 16) blocks = 256 * 16;
  const dim3 grid((unsigned)blocks), block(rh::ce::kThreads);
  if (dtype == RH_F32)
    hipLaunchKernelGGL(rh::ce::upstream_kernel<float>, grid, block, 0, (hipStream_t)stream, (float*)x, (long long)count, scale,
                       assumed);
  else if (dtype == RH_BF16)
    hipLaunchKernelGGL(rh::ce::upstream_kernel<__bf16>, grid, block, 0, (hipStream_t)stream, (__bf16*)x, (long long)count, scale,
                       assumed);
  else if (dtype == RH_F16)
    hipLaunchKernelGGL(rh::ce::upstream_kernel<_Float16>, grid, block, 0, (hipStream_t)stream, (_Float16*)x, (long long)count, scale,
                       assumed);
  else
    RH_FAIL(RH_EINVAL, "unknown element type %d", dtype);
  RH_CHECK_LAUNCH("upstream_kernel");
  return RH_OK;
}

}  // extern "C"
