// Matrix-product core of the classifier loss (gfx950): C[m][n] = sum_k A(m,k) B(n,k) on the matrix
// units, operands staged to LDS by direct loads, two stages deep.
//
// An operand comes in one of two layouts, so that the loss's three products need no transposed
// copies:   kRows  element (i,k) at  base + i*ld + k   (the sum runs along a row)
//           kCols  element (i,k) at  base + k*ld + i   (the sum runs down a column)
// Both are staged as they lie in memory.  A kRows tile holds 128 bytes of k per row and its 16-byte
// fragments are read as they are; a kCols tile of a 16-bit type is read with the transposing LDS
// load, one of a 32-bit type element by element.
//
// Every global read goes through a buffer descriptor whose record count ends at the operand's last
// valid element: what a tile reaches beyond it reads as zero and touches no memory.
#pragma once
#include "rh_common.h"

namespace rh {
namespace gemm {

#define RH_LDS __attribute__((address_space(3)))

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

enum Layout { kRows = 0, kCols = 1 };

// 128 bytes of k per tile step: 64 values of a 16-bit type, 32 of float.
constexpr int kStepBytes = 128;

template <typename T>
struct TypeOf;
template <>
struct TypeOf<float> {
  static __device__ __forceinline__ f32x16 mma(const u32x4 a, const u32x4 b, f32x16 c) {
    // lane half h holds k = 4h .. 4h+3 of eight; both operands agree, so instruction j sums the
    // pair {j, 4+j}
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[0], y[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[1], y[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[2], y[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[3], y[3], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float to_float(float v) { return v; }
  static __device__ __forceinline__ float from_float(float v) { return v; }
};
template <>
struct TypeOf<__bf16> {
  static __device__ __forceinline__ f32x16 mma(const u32x4 a, const u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 from_float(float v) { return (__bf16)v; }
};
template <>
struct TypeOf<_Float16> {
  static __device__ __forceinline__ f32x16 mma(const u32x4 a, const u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from_float(float v) { return (_Float16)v; }
};

// A lane of the lower half of the wave has four values of each of two groups of eight, x of the first
// and y of the second (as 8 bytes), its partner 32 lanes on the other four: afterwards the lower lane
// has the first group whole, the upper one the second.
__device__ __forceinline__ u32x4 whole_group(const unsigned long long x, const unsigned long long y) {
  const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)y, false, false);
  const auto hi = __builtin_amdgcn_permlane32_swap((unsigned)(x >> 32), (unsigned)(y >> 32), false, false);
  return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

template <typename T>
struct Vec4 {
  T v[4];
} __attribute__((aligned(4 * sizeof(T))));

// Workgroups of neighbouring numbers land on different XCDs: number `id` of `total` -> the tile
// number that gives each of the eight XCDs a contiguous run of tiles.
__device__ __forceinline__ int xcd_run(const int id, const int total) {
  const int per = total >> 3, rest = total & 7, x = id & 7, at = id >> 3;
  return x * per + min(x, rest) + at;
}

// One operand's descriptor for a tile: bytes readable from its first element on.
__device__ __forceinline__ u32x4 make_rsrc(const char* base, const long long bytes) {
  const unsigned long long at = (unsigned long long)base;
  const long long top = 0x7fffff00ll;
  u32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((unsigned)at);
  r[1] = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32) & 0xffffu);
  r[2] = __builtin_amdgcn_readfirstlane((unsigned)(bytes <= 0 ? 0 : bytes < top ? bytes : top));
  r[3] = 0x00020000u;
  // a lane instruction may have written these registers: a memory instruction that takes them has to
  // stay five cycles behind, which nobody else sees to for the written-out ones below
  asm volatile("s_nop 4" : "+s"(r));
  return r;
}
constexpr int kNowhere = 0x7fffff80;      // an offset no descriptor reaches: reads as zero

// 16 bytes per lane from the buffer to LDS, lane after lane from `lds` on.  Written out, because
// the compiler waits for every such load of its own before any LDS read; here stage_wait() does.
__device__ __forceinline__ void load_to_lds(const u32x4 rsrc, const unsigned lds, const int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(offset), "s"(rsrc)
               : "memory");
}
// This wave's loads have landed and its LDS reads have returned; then every wave's.
__device__ __forceinline__ void stage_wait() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Moves one stage of an operand's tile (kR rows or columns of the result, kStepBytes of k) to LDS.
template <typename T, Layout kL, int kR, int kThreads>
struct Loader {
  static constexpr int kStepK = kStepBytes / (int)sizeof(T);
  static constexpr int kBytes = kR * kStepBytes;
  static constexpr int kOps = kBytes / (kThreads * 16);
  static constexpr int kRowBytes = kL == kRows ? kStepBytes : kR * (int)sizeof(T);
  static constexpr int kChunks = kRowBytes / 16;             // 16-byte chunks of a staged row
  static constexpr int kRowsPerOp = kThreads / kChunks;      // staged rows one pass of all threads covers
  int offset[kOps];       // this lane's byte offsets from the tile's first element
  const char* base;       // of the coming step
  long long left;         // bytes readable from base on
  long long step;         // bytes from one step to the next

  static __device__ __forceinline__ int chunk_of(const int i) {
    const int row = i * kRowsPerOp + (int)threadIdx.x / kChunks, at = (int)threadIdx.x % kChunks;
    if (kL == kRows) return at ^ ((row >> 1) & 7);
    return sizeof(T) == 2 ? at ^ ((row & 3) << 2) : at;    // 16 bits: 32-byte blocks, block ^ 2*(k & 3)
  }
  // origin: first element of the tile at k = 0; ld in elements; bytes: readable from origin on.
  __device__ __forceinline__ void init(const void* origin, long long ld, long long bytes) {
    base = (const char*)origin;
    left = bytes;
    step = kL == kRows ? kStepBytes : (long long)kStepK * ld * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < kOps; ++i)
      offset[i] = (int)((i * kRowsPerOp + (int)threadIdx.x / kChunks) * ld * (int)sizeof(T)) + chunk_of(i) * 16;
  }
  // The coming step's loads to a stage: begin(), then load<i>() for each of the kOps.  A step that
  // is not `there` reads zeros and touches no memory; limit (kRows): bytes of k that belong to the rows.
  u32x4 rsrc;
  unsigned to;
  int limit;
  __device__ __forceinline__ void begin(RH_LDS char* stage, const bool there, const int k_bytes) {
    rsrc = make_rsrc(base, there ? left : 0);
    to = __builtin_amdgcn_readfirstlane((unsigned)(size_t)stage + (threadIdx.x >> 6) * 1024);
    limit = k_bytes;
    base += step;
    left -= step;
  }
  template <bool kTail>
  __device__ __forceinline__ void load(const int first, const int count) const {
#pragma unroll
    for (int i = first; i < first + count; ++i)
      load_to_lds(rsrc, to + i * kThreads * 16,
                  !kTail || chunk_of(i) * 16 < limit ? offset[i] : kNowhere);
  }
};

// Reads the matrix instructions' fragments of one wave from a staged tile.  `first`: the wave's
// first row / column of the tile (a multiple of 32); fragment f covers 32 from first + 32 f on.
template <typename T, Layout kL, int kR, int kF>
struct Fragments {
  static constexpr int kRowBytes = kR * (int)sizeof(T);      // kCols only
  static constexpr int kAddr = kL == kRows ? 4 : (sizeof(T) == 2 ? kF : 1);
  int addr[kAddr];
  __device__ __forceinline__ void init(const int first) {
    const int l = (int)threadIdx.x & 63;
    if (kL == kRows) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        addr[kk] = (first + (l & 31)) * kStepBytes + (((2 * kk + (l >> 5)) ^ ((l >> 1) & 7)) << 4);
    } else if (sizeof(T) == 2) {
      const int q = (l >> 2) & 3;
#pragma unroll
      for (int f = 0; f < kAddr; ++f)
        addr[f] = (8 * (l >> 5) + q) * kRowBytes + (((first / 32 + f) ^ q) << 6) + ((l >> 4) & 1) * 32 +
                  (l & 3) * 8;
    } else {
      addr[0] = 4 * (l >> 5) * kRowBytes + (first + (l & 31)) * 4;
    }
  }
  __device__ __forceinline__ u32x4 read(const RH_LDS char* stage, const int f, const int kk) const {
    if constexpr (kL == kRows) {
      return *(const RH_LDS u32x4*)(stage + addr[kk] + f * 32 * kStepBytes);
    } else if constexpr (sizeof(T) == 2) {
      union {
        bf16x4 h[2];
        u32x4 u;
      } r;
      const RH_LDS char* p = stage + addr[f] + kk * 16 * kRowBytes;
      r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((RH_LDS bf16x4*)p);
      r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((RH_LDS bf16x4*)(p + 4 * kRowBytes));
      return r.u;
    } else {
      const RH_LDS char* p = stage + addr[0] + f * 128 + kk * 8 * kRowBytes;
      u32x4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = *(const RH_LDS unsigned*)(p + j * kRowBytes);
      return r;
    }
  }
};

// A workgroup's tile: kWM x kWN waves, each kFM x kFN fragments of 32 x 32.
template <int kWM_, int kWN_, int kFM_, int kFN_>
struct Shape {
  static constexpr int kWM = kWM_, kWN = kWN_, kFM = kFM_, kFN = kFN_;
  static constexpr int kBM = kWM * kFM * 32, kBN = kWN * kFN * 32;
  static constexpr int kThreads = kWM * kWN * 64;
  static constexpr int kStage = (kBM + kBN) * kStepBytes;
  static constexpr int kLdsBytes = 2 * kStage;
};

// acc[i][j][r]: result row m = 32 i + lane % 32 and column n = 32 j + 8 (r / 4) + 4 (lane / 32) + r % 4
// of the wave's part: a lane owns rows, four neighbouring columns at a time.
template <typename T, Layout kLA, Layout kLB, typename S>
struct Tile {
  static constexpr int kStepK = kStepBytes / (int)sizeof(T);
  f32x16 acc[S::kFM][S::kFN];

  // a / b: first elements of the tile's operands at the first k; *_bytes: readable from there;
  // steps: k steps (of kStepK values); b_limit (kRows B): bytes of the last step that are b's.
  //
  // A step's fragments are read a quarter ahead of the instructions that take them.  The wait for the
  // next stage stands before the last quarter's instructions, which then cover the barrier, the first
  // reads of that stage and the launch of the loads that refill the one just read out.
  __device__ __forceinline__ void run(const void* a, long long lda, long long a_bytes, const void* b,
                                      long long ldb, long long b_bytes, const int steps,
                                      RH_LDS char* lds, const int b_limit = kStepBytes) {
    Loader<T, kLA, S::kBM, S::kThreads> la;
    Loader<T, kLB, S::kBN, S::kThreads> lb;
    Fragments<T, kLA, S::kBM, S::kFM> fa;
    Fragments<T, kLB, S::kBN, S::kFN> fb;
    constexpr int kOffB = S::kBM * kStepBytes;
    const int wave = (int)threadIdx.x >> 6;
    la.init(a, lda, a_bytes);
    lb.init(b, ldb, b_bytes);
    fa.init((wave / S::kWN) * S::kFM * 32);
    fb.init((wave % S::kWN) * S::kFN * 32);
#pragma unroll
    for (int i = 0; i < S::kFM; ++i)
#pragma unroll
      for (int j = 0; j < S::kFN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (steps <= 0) return;
    constexpr bool kTail = kLB == kRows;      // rows of b may end inside the last step
    constexpr int kOpsA = Loader<T, kLA, S::kBM, S::kThreads>::kOps;
    constexpr int kOpsB = Loader<T, kLB, S::kBN, S::kThreads>::kOps;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      la.begin(lds + s * S::kStage, s < steps, kStepBytes);
      lb.begin(lds + s * S::kStage + kOffB, s < steps, s + 1 == steps ? b_limit : kStepBytes);
      la.template load<false>(0, kOpsA);
      lb.template load<kTail>(0, kOpsB);
      if (s == 0) stage_wait();
    }
    u32x4 x[2][S::kFM], y[2][S::kFN];
    constexpr int kSlots = S::kFM * S::kFN, kFragments = S::kFM + S::kFN;
    // Fragment f of a quarter, in the order the products take them: y0 x0 y1 .. yn x1 .. xm.
    auto read = [&](const int to, const RH_LDS char* stage, const int kk, const int f) {
      if (f == 0) y[to][0] = fb.read(stage + kOffB, 0, kk);
      else if (f == 1) x[to][0] = fa.read(stage, 0, kk);
      else if (f <= S::kFN) y[to][f - 1] = fb.read(stage + kOffB, f - 1, kk);
      else x[to][f - S::kFN] = fa.read(stage, f - S::kFN, kk);
    };
    // A quarter's products, with what comes next issued between them: while one instruction runs on
    // the matrix unit (32 cycles) the wave has time for about seven others.
    auto quarter = [&](const int from, const RH_LDS char* stage, const int kk, const bool load) {
#pragma unroll
      for (int t = 0; t < kSlots; ++t) {
        acc[t / S::kFN][t % S::kFN] =
            TypeOf<T>::mma(y[from][t % S::kFN], x[from][t / S::kFN], acc[t / S::kFN][t % S::kFN]);
        if (t < kFragments) read(from ^ 1, stage, kk, t);
        if (load) {
          constexpr int kA = kOpsA / kSlots, kB = kOpsB / kSlots;
          static_assert(kSlots <= 4 || kOpsA + kOpsB == kSlots, "a load a slot");
          if constexpr (kOpsA + kOpsB == kSlots) {
            if (t < kOpsA) la.template load<false>(t, 1);
            else lb.template load<kTail>(t - kOpsA, 1);
          } else {
            la.template load<false>(t * kA, kA);
            lb.template load<kTail>(t * kB, kB);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
#pragma unroll
    for (int f = 0; f < kFragments; ++f) read(0, lds, 0, f);
    for (int s = 0; s < steps; ++s) {
      RH_LDS char* here = lds + (s & 1) * S::kStage;
      RH_LDS char* next = lds + ((s + 1) & 1) * S::kStage;
      quarter(0, here, 1, false);
      quarter(1, here, 2, false);
      quarter(0, here, 3, false);
      stage_wait();
      la.begin(here, s + 2 < steps, kStepBytes);
      lb.begin(here + kOffB, s + 2 < steps, s + 3 == steps ? b_limit : kStepBytes);
      quarter(1, next, 0, true);
    }
    stage_wait();      // LDS is the caller's again
  }
};

}  // namespace gemm
}  // namespace rh
